"""The fine-tuning operators together, as a user runs them: samples of a small model scored by itself and by a reference, a policy step and a
preference step with clipped gradients and AdamW, against the same steps in plain operations."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F
from nexus_b200.lm.config import LmConfig
from nexus_b200.lm.model import LanguageModel

pytestmark = pytest.mark.gpu


def model(seed, **kw):
    base = dict(vocab_size=500, n_layer=2, d_model=64, n_head=1, d_ff=128, max_position=64, vocab_pad_multiple=64, seed=seed)
    return LanguageModel(LmConfig(**{**base, **kw})).cuda()


def batch(seed=0, B=4, T=24):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, 500, (B, T), generator=g).cuda()
    mask = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    for b in range(B):
        mask[b, 6: T - 2 * b] = True
    return tokens, mask, g


def plain_logp(m, tokens, mask):
    lp = torch.log_softmax(m.logits(tokens)[..., :500].double(), -1)
    one = torch.zeros(tokens.shape, dtype=torch.float64, device=tokens.device)
    one[:, :-1] = lp[:, :-1].gather(2, tokens[:, 1:, None])[..., 0] * mask[:, 1:]
    return one, lp


@pytest.mark.parametrize("tie", [False, True])
def test_fp32_steps(tie):
    """FP32 model: each gradient against autograd's in FP64 from the same FP32 activations; 2e-5 of the whole is the rounding of some hundreds
    of FP32 operations between the logits and the weights."""
    m, ref = model(1, tie_embeddings=tie), model(2, tie_embeddings=tie)
    tokens, mask, g = batch()
    with torch.no_grad():
        old, refl = m.token_logprobs(tokens, mask), ref.token_logprobs(tokens, mask)
    want = plain_logp(m, tokens, mask)[0]
    assert float((old - want).abs().max().detach()) < 1e-5 and bool((old[:, -1] == 0).all()) and bool((old[:, 0] == 0).all())
    old = old + torch.round(torch.randn(old.shape, generator=g).cuda() * 8) / 64
    adv = torch.randn(4, generator=g).cuda()
    params = [p for p in m.parameters()]

    def policy_plain():
        one, lp = plain_logp(m, tokens, mask)
        keep = torch.zeros_like(mask)
        keep[:, :-1] = mask[:, 1:]
        H = -(lp.exp() * lp).sum(-1)
        r = torch.exp(one - old.double())
        gain = torch.minimum(r * adv[:, None].double(), r.clamp(0.8, 1.2) * adv[:, None].double())
        d = refl.double() - one
        per = -gain + 0.05 * (torch.expm1(d) - d) - 0.01 * H
        return (per * keep).sum() / keep.sum()

    def preference_plain():
        s = plain_logp(m, tokens, mask)[0].sum(-1)
        h = (s - refl.double().sum(-1))
        return -torch.nn.functional.logsigmoid(0.1 * (h[:2] - h[2:])).mean()

    fast = [lambda: m.policy_loss(tokens, mask, old, adv, refl, kl_coef=0.05, entropy_coef=0.01).loss,
            lambda: m.preference_loss(tokens, mask, refl.sum(-1)).loss]
    for quick, plain in zip(fast, (policy_plain, preference_plain)):
        a, b = quick(), plain()
        assert float(a.detach()) == pytest.approx(float(b.detach()), abs=2e-5)
        ga, gb = torch.autograd.grad(a, params, allow_unused=True), torch.autograd.grad(b.float(), params, allow_unused=True)
        for x, y in zip(ga, gb):
            assert (x is None) == (y is None)
            if x is not None:
                assert float((x - y).norm()) <= 2e-5 * float(y.norm()) + 1e-9


def test_bf16_training_loop_runs():
    """Score, policy step, preference step, clip, AdamW, three times, in BF16 autocast as the trainer runs it."""
    m, ref = model(3), model(3)
    tokens, mask, g = batch(5)
    adv = torch.tensor([1.0, -1.0, 0.5, -0.5], device="cuda")
    m1 = [torch.zeros_like(p) for p in m.parameters()]
    m2 = [torch.zeros_like(p) for p in m.parameters()]
    ps = list(m.parameters())
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        old, refl = m.token_logprobs(tokens, mask), ref.token_logprobs(tokens, mask)
        h, w = m.hidden(tokens), m.lm_head          # not tied by default
        assert torch.equal(old, F.linear_logprobs(h.bfloat16(), w.bfloat16(), m._next_targets(tokens, mask), vocab=500))
    assert torch.equal(old, refl) and old.dtype == torch.float32
    for step in (1, 2, 3):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            r = m.policy_loss(tokens, mask, old, adv, refl, kl_coef=0.02, reduction="sequence")
            q = m.preference_loss(tokens, mask, refl.sum(-1))
        (r.loss + 0.5 * q.loss).backward()
        grads = [p.grad for p in ps if p.grad is not None]
        before = math.sqrt(sum(float(x.double().pow(2).sum()) for x in grads))
        norm = F.clip_grad_norm_(grads, 0.1)
        assert float(norm) == pytest.approx(before, rel=1e-6) and math.isfinite(before)
        after = math.sqrt(sum(float(x.double().pow(2).sum()) for x in grads))
        assert after == pytest.approx(min(before, 0.1), rel=1e-5)
        idx = [i for i, p in enumerate(ps) if p.grad is not None]
        F.adamw_multi_tensor([ps[i].data for i in idx], grads, [m1[i] for i in idx], [m2[i] for i in idx], step, 1e-3, max_grad_norm=0.1)
        for p in ps:
            p.grad = None
    from nexus_b200.ops import _cuda as K
    K.check_status()


def test_masks_are_checked():
    m = model(4)
    tokens, mask, _ = batch()
    for bad in (mask.long(), mask[:, :-1]):
        with pytest.raises(ValueError):
            m.token_logprobs(tokens, bad)

"""Scores of a language model beside its losses: with unchanged weights the ratio is one, the divergence zero and the margin zero."""
import math

import pytest
import torch
from test_gpu_finetune import batch, model
from test_gpu_objectives import U, logp_error

from nexus_b200.fused import ops as F

pytestmark = pytest.mark.gpu


def loud(seed, **kw):
    """A model whose logits reach some tens, where a step of BF16 is an eighth."""
    m = model(seed, **kw)
    with torch.no_grad():
        (m.wte if m.lm_head is None else m.lm_head).mul_(60.0)
    return m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, None])
@pytest.mark.parametrize("kw", [{}, dict(tie_embeddings=True), dict(init="mup", mup_base_width=32), dict(mxfp8=True)])
def test_unchanged_weights(dtype, kw):
    kw = dict(kw)
    precision = F.linear_precision("mxfp8" if kw.pop("mxfp8", False) and dtype == torch.bfloat16 else "native")
    m = loud(1, **kw)
    tokens, mask, _ = batch()
    adv = torch.ones(4, device="cuda")
    with precision, torch.autocast("cuda", dtype=dtype or torch.bfloat16, enabled=dtype is not None):
        with torch.no_grad():
            old = m.token_logprobs(tokens, mask, temperature=0.9, through_logits=True)
            biggest = float(m.logits(tokens).abs().max())
        r = m.policy_loss(tokens, mask, old, adv, old, kl_coef=0.1, temperature=0.9)
        q = m.preference_loss(tokens, mask, old.double().sum(-1), temperature=0.9)
    assert biggest > 8.0                                   # rounding of logits would show
    # both sides are off by `logp_error` from the same logits' values
    err = 2 * logp_error(old.double(), 500)
    assert bool(((r.logp - old).abs() <= err).all())
    top = float(err.max())
    assert bool((r.kl.abs() <= (1.0 + top) * top).all())
    assert float(r.loss.detach()) == pytest.approx(-1.0, abs=4 * top)
    room = err.sum(-1) + 2 * U * old.double().sum(-1).abs()      # and the sums' roundings to FP32
    assert bool((q.margin.abs() <= room[:2] + room[2:]).all())
    assert float(q.loss.detach()) == pytest.approx(math.log(2.0), abs=0.05 * float((room[:2] + room[2:]).max()) + 4 * U)


def test_gradient_of_scores_through_logits():
    m = loud(2)
    tokens, mask, g = batch(3)
    d = torch.randn(tokens.shape, generator=g).cuda()
    params = list(m.parameters())
    a = torch.autograd.grad(m.token_logprobs(tokens, mask, through_logits=True), params, d, allow_unused=True)
    b = torch.autograd.grad(m.token_logprobs(tokens, mask), params, d, allow_unused=True)
    for x, y in zip(a, b):      # FP32: two orders of the same products
        assert (x is None) == (y is None)
        if x is not None:
            assert float((x - y).norm()) <= 1e-4 * float(y.norm()) + 1e-9

"""`LanguageModel`'s fine-tuning methods on the host, against plain operations."""
import torch

from nexus_b200.lm.config import LmConfig
from nexus_b200.lm.model import LanguageModel


def test_methods_of_the_language_model():
    m = LanguageModel(LmConfig(vocab_size=50, n_layer=1, d_model=16, n_head=2, d_ff=32, max_position=16, vocab_pad_multiple=16, init="mup",
                               mup_base_width=8))
    g = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, 50, (4, 9), generator=g)
    mask = torch.rand(4, 9, generator=g) < 0.6
    lp = torch.log_softmax(m.logits(tokens)[..., :50], -1)
    want = torch.zeros(4, 9)
    want[:, :-1] = lp[:, :-1].gather(2, tokens[:, 1:, None])[..., 0] * mask[:, 1:]
    got = m.token_logprobs(tokens, mask)
    assert torch.allclose(got, want, atol=1e-5)
    assert torch.allclose(m.token_logprobs(tokens)[:, :-1], lp[:, :-1].gather(2, tokens[:, 1:, None])[..., 0], atol=1e-5)
    r = m.policy_loss(tokens, mask, got.detach(), torch.ones(4), got.detach(), kl_coef=0.1)
    assert torch.allclose(r.logp, want, atol=1e-5) and abs(float(r.loss.detach()) + 1.0) < 1e-4 and float(r.kl.abs().max()) < 1e-6
    q = m.preference_loss(tokens, mask)
    h = want.sum(-1)
    assert torch.allclose(q.margin, h[:2] - h[2:], atol=1e-4)
    (r.loss + q.loss).backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)

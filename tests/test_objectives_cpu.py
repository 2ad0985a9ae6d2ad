"""The plain forms of the objectives (gradients against differences in 64 bits) and what the entry points refuse."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F


def inputs(B=4, T=5, W=17, V=15):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(B, T, W, dtype=torch.float64, generator=g, requires_grad=True)
    t = torch.randint(0, V, (B, T), generator=g)
    t[0, :2] = -100
    t[B - 1] = -100
    const = [torch.randn(B, T, generator=g) * 0.1 - 3 for _ in range(2)]
    return x, t, *const, torch.randn(B, generator=g)


def test_gradients_against_differences():
    x, t, old, ref, adv = inputs()
    assert torch.autograd.gradcheck(lambda x: F.token_logprobs(x, t, vocab=15, temperature=0.7), x)
    for reduction in ("token", "sequence", "sum"):
        for kl in ("k1", "k2", "k3"):
            assert torch.autograd.gradcheck(lambda x: F.policy_loss(x, t, old, adv, ref, kl_coef=0.1, kl=kl, entropy_coef=0.02,
                                                                    reduction=reduction, vocab=15).loss, x)
    for kind in ("sigmoid", "hinge", "ipo"):
        assert torch.autograd.gradcheck(lambda x: F.preference_loss(x, t, adv, kind=kind, average=True, vocab=15).loss, x)


def test_policy_clips():
    """Advantage of each sign at ratios inside and outside the borders: value and slope by hand."""
    V = 4
    x = torch.zeros(1, 6, V, dtype=torch.float64, requires_grad=True)
    t = torch.zeros(1, 6, dtype=torch.long)
    ratios = torch.tensor([[0.5, 1.0, 1.5, 0.5, 1.0, 1.5]], dtype=torch.float64)
    adv = torch.tensor([[1.0, 1.0, 1.0, -1.0, -1.0, -1.0]])
    old = math.log(0.25) - torch.log(ratios)
    r = F.policy_loss(x, t, old.double(), adv, clip_low=0.2, clip_high=0.3, reduction="sum")
    assert float(r.loss.detach()) == pytest.approx(-0.5 - 1.0 - 1.3 + 0.8 + 1.0 + 1.5, abs=1e-6)
    r.loss.backward()
    slope = x.grad[0, :, 0] / 0.75
    assert slope.tolist() == pytest.approx([-0.5, -1.0, 0.0, 0.0, 1.0, 1.5], abs=1e-6)


def test_ignored_and_bad_targets():
    x = torch.randn(2, 3, 8)
    x[0, 0] = math.nan
    x.requires_grad_(True)
    t = torch.tensor([[-100, 1, 2], [8, -1, 3]])
    logp = F.token_logprobs(x, t)
    assert float(logp[0, 0].detach()) == 0.0 and torch.isnan(logp).tolist() == [[False] * 3, [True, True, False]]
    logp.sum().backward()
    assert bool((x.grad[0, 0] == 0).all()) and bool((x.grad[1, :2] == 0).all())
    assert math.isnan(float(F.policy_loss(x, t, torch.zeros(2, 3), torch.ones(2)).loss.detach()))


def test_refusals():
    x, t, old, ref, adv = inputs()
    lp, pol, pref = F.token_logprobs, F.policy_loss, F.preference_loss
    bad = [
        lambda: lp(x.long(), t), lambda: lp(x, t.float()), lambda: lp(x, t[:, :-1]), lambda: lp(x, t, vocab=18), lambda: lp(x, t, vocab=0),
        lambda: lp(x, t, temperature=0.0), lambda: lp(x, t, temperature=math.inf), lambda: lp(x, t, temperature=-1.0),
        lambda: pol(x[0], t[0], old[0], adv), lambda: pol(x, t, old[:, :-1], adv), lambda: pol(x, t, old, adv[:-1]), lambda: pol(x, t, old, 1.0),
        lambda: pol(x, t, old.long(), adv), lambda: pol(x, t, old, adv, kl_coef=0.1), lambda: pol(x, t, old, adv, ref[:1], kl_coef=0.1),
        lambda: pol(x, t, old, adv, ref, kl="kl"), lambda: pol(x, t, old, adv, reduction="mean"), lambda: pol(x, t, old, adv, clip_low=-0.1),
        lambda: pol(x, t, old, adv, clip_low=1.1), lambda: pol(x, t, old, adv, clip_high=math.inf), lambda: pol(x, t, old, adv, scale=math.nan),
        lambda: pref(x[:3], t[:3]), lambda: pref(x[0], t[0]), lambda: pref(x, t, adv[:2]), lambda: pref(x, t, kind="dpo"), lambda: pref(x, t, beta=0.0),
        lambda: pref(x, t, label_smoothing=0.5), lambda: pref(x, t, kind="hinge", label_smoothing=0.1), lambda: pref(x, t, kind="ipo", target_margin=1.0),
        lambda: pref(x[:0], t[:0]),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_refuses_temperatures_whose_inverse_is_no_scale():
    x, t, old, _, adv = inputs()
    h, w = torch.randn(*t.shape, 16), torch.randn(x.shape[-1], 16)
    for temperature in (1e-45, 9e-9, 1.1e8, 1e39, math.nan):
        for call in (lambda: F.token_logprobs(x, t, temperature=temperature), lambda: F.linear_logprobs(h, w, t, temperature=temperature),
                     lambda: F.policy_loss(x, t, old, adv, temperature=temperature), lambda: F.preference_loss(x, t, temperature=temperature)):
            with pytest.raises(ValueError, match="temperature"):
                call()
    for temperature in (1e-8, 1e8):
        assert bool(torch.isfinite(F.token_logprobs(x, t, temperature=temperature)).all())


def test_row_layouts():
    """The rows of these views are read where they are; the others are copied first."""
    from nexus_b200.ops._objectives import row_layout
    x = torch.empty(4, 6, 64)
    assert row_layout(x) == (24, 0, 64)
    assert row_layout(x[:, 1:]) == (5, 384, 64) and row_layout(x[..., :50]) == (24, 0, 64)
    assert row_layout(x.transpose(0, 1)) == (4, 64, 384)
    assert row_layout(x[0, 0])[0] == 1 and row_layout(x.view(4, 3, 2, 64)[:, :, 1]) == (12, 0, 128)
    for copied in (x[..., ::2], x[:, :1].expand(4, 6, 64), x[:, -1:], x[..., :20], x.view(4, 3, 2, 64)[:, :2, :1], torch.empty(0, 3, 4)):
        assert row_layout(copied) is None


def test_clip_on_the_host():
    g = torch.Generator().manual_seed(3)
    make = lambda: [torch.randn(n, generator=g) for n in (1, 7, 40)] + [torch.randn(5, 6, generator=g).t(), torch.randn(3, 8, generator=g)[:, :5]]  # noqa: E731
    gs = make()
    want = math.sqrt(sum(float(t.double().pow(2).sum()) for t in gs))
    keep = [t.clone() for t in gs]
    assert F.grad_square_sum(gs) == pytest.approx(want * want, rel=1e-14)
    norm = F.clip_grad_norm_(gs + [None, torch.zeros(0)], 1.5)
    assert norm.dtype == torch.float32 and float(norm) == pytest.approx(want, rel=2 ** -24)
    for a, b in zip(gs, keep):
        assert torch.allclose(a, b * (1.5 / (want + 1e-6)), rtol=2 ** -22, atol=0)
    outs = [torch.empty(t.shape, dtype=torch.bfloat16) for t in keep]
    F.clip_grad_norm_(keep, 1e9, out=outs)
    assert all(torch.equal(o, k.bfloat16()) for o, k in zip(outs, keep))
    bad = [torch.tensor([1.0, math.inf]), torch.tensor([2.0])]
    assert math.isinf(float(F.clip_grad_norm_(bad, 1.0))) and bad[1].item() == 2.0
    tied = torch.ones(4)
    assert float(F.clip_grad_norm_([tied, tied], 1.0)) == 2.0 and float(tied[0]) == pytest.approx(0.5, rel=1e-5)
    assert float(F.clip_grad_norm_([], 1.0)) == 0.0 and float(F.clip_grad_norm_([torch.zeros(0)], 1.0)) == 0.0


def test_clip_refusals():
    a, b = torch.ones(6), torch.ones(6)
    for call in (lambda: F.clip_grad_norm_([a], -1.0), lambda: F.clip_grad_norm_([a], math.nan), lambda: F.clip_grad_norm_([a.long()], 1.0),
                 lambda: F.clip_grad_norm_([a], 1.0, out=[b, b]), lambda: F.clip_grad_norm_([a], 1.0, out=[torch.ones(5)]),
                 lambda: F.clip_grad_norm_([a[:4], a[2:]], 1.0), lambda: F.clip_grad_norm_([torch.ones(1).expand(4)], 1.0),
                 lambda: F.clip_grad_norm_([a, b], 1.0, out=[b, torch.ones(6)]), lambda: F.clip_grad_norm_([a, b], 1.0, out=[torch.ones(6)] + [a]),
                 lambda: F.clip_grad_norm_([a, a], 1.0, out=[torch.ones(6), torch.ones(6)]), lambda: F.clip_grad_norm_([a.to_sparse()], 1.0)):
        with pytest.raises(ValueError):
            call()


def test_linear_logprobs_on_the_host():
    g = torch.Generator().manual_seed(1)
    h = torch.randn(2, 3, 8, dtype=torch.float64, generator=g, requires_grad=True)
    w = torch.randn(11, 8, dtype=torch.float64, generator=g, requires_grad=True)
    t = torch.randint(0, 10, (2, 3), generator=g)
    t[0, 0] = -100
    assert torch.autograd.gradcheck(lambda h, w: F.linear_logprobs(h, w, t, temperature=0.9, vocab=10), (h, w))
    for call in (lambda: F.linear_logprobs(h, w.float(), t), lambda: F.linear_logprobs(h, w[:, :4], t), lambda: F.linear_logprobs(h, w, t[0]),
                 lambda: F.linear_logprobs(h, w, t.float()), lambda: F.linear_logprobs(h, w, t, vocab=12), lambda: F.linear_logprobs(h, w[0], t),
                 lambda: F.linear_logprobs(h, w, t, temperature=0.0), lambda: F.linear_logprobs(h.long(), w.long(), t)):
        with pytest.raises(ValueError):
            call()


def test_slices_of_the_vocabulary():
    from nexus_b200.ops._objectives import head_slices
    assert head_slices(8192, 4096) == 1 and head_slices(609, 896) == 16
    for rows, width in ((1, 64), (256, 4096), (2048, 1024), (4096, 512), (100000, 8)):
        assert 1 <= head_slices(rows, width) <= 16 and (head_slices(rows, width) - 1) * rows * width <= 1 << 25

"""Ends of the ranges that the plain forms of the fine-tuning operators take, and calls that are refused."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F


def test_fp8_gradients_are_refused():
    """A type that the library has codes for and the clipping does not take, first or behind others; an output may have it."""
    a, b = torch.ones(8), torch.ones(8).to(torch.float8_e4m3fn)
    for call in (lambda: F.clip_grad_norm_([a, b], 1.0), lambda: F.clip_grad_norm_([b, a], 1.0), lambda: F.clip_grad_norm_([b], 1.0, out=[a])):
        with pytest.raises(ValueError, match="float8"):
            call()
    assert torch.equal(a, torch.ones(8))
    assert float(F.clip_grad_norm_([2.0 * a], 1e3, out=[b])) == pytest.approx(32.0 ** 0.5) and bool((b.float() == 2.0).all())
    assert F.grad_square_sum([a, b]) == 40.0
    F.clip_grad_norm_([a], 8.0 ** 0.5 / 2, out=[b])
    assert bool((b.float() == 0.5).all())


def test_forward_mode_derivatives():
    """Log-probabilities carry a tangent, constants of a loss none, and the clipping refuses it."""
    from torch.autograd import forward_ad
    g = torch.Generator().manual_seed(0)
    x, v = torch.randn(2, 3, 8, generator=g), torch.randn(2, 3, 8, generator=g)
    t = torch.randint(0, 8, (2, 3), generator=g)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, v)
        got = forward_ad.unpack_dual(F.token_logprobs(d, t)).tangent
        old = forward_ad.make_dual(torch.zeros(2, 3), torch.ones(2, 3))
        assert forward_ad.unpack_dual(F.policy_loss(x, t, old, torch.ones(2)).loss).tangent is None
        for grads, out in (([x, d], None), ([x], [d])):
            with pytest.raises(NotImplementedError):
                F.clip_grad_norm_(grads, 1.0, out=out)
    want = v.gather(2, t[..., None])[..., 0] - (x.softmax(-1) * v).sum(-1)
    assert torch.allclose(got, want, atol=1e-6)


@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0)])
@pytest.mark.parametrize("side", [0, 1])
def test_preference_of_a_sequence_that_cannot_be(kind, smoothing, side):
    """A target whose logit is -inf in the chosen sequence (0) or in the rejected one (1): the loss is its limit, and the gradient finite."""
    x = torch.zeros(4, 2, 4)
    x[2 * side, 1, 0] = -math.inf        # of the first pair, which is rows 0 and 2
    x.requires_grad_(True)
    t = torch.zeros(4, 2, dtype=torch.long)
    r = F.preference_loss(x, t, beta=0.5, kind=kind, label_smoothing=smoothing)
    r.loss.backward()
    other = math.log(2.0) if kind == "sigmoid" else 1.0
    limit = {("sigmoid", 0): math.inf, ("sigmoid", 1): math.inf if smoothing else 0.0, ("hinge", 0): math.inf, ("hinge", 1): 0.0}[kind, side]
    assert float(r.margin[0]) == (math.inf if side else -math.inf) and float(r.margin[1]) == 0.0
    assert float(r.loss.detach()) == pytest.approx((limit + other) / 2)
    slope = {"sigmoid": 0.5 * (smoothing - (0.0 if side else 1.0)), "hinge": 0.0 if side else -0.5}[kind] / 2
    p = torch.softmax(x.detach().double(), -1)
    want = torch.zeros_like(p)
    want[..., 0] = 1.0
    want = (want - p) * slope
    want[2] = -want[2]
    assert torch.allclose(x.grad[[0, 2]].double(), want[[0, 2]], atol=1e-6)
    assert bool(torch.isfinite(x.grad).all())


@pytest.mark.parametrize("kl", ["k1", "k2", "k3"])
def test_an_estimate_of_the_divergence_that_is_only_looked_at(kl):
    """Without a KL term its estimate, which may overflow, is in neither the loss nor the gradient."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 3, 8, generator=g)
    t = torch.randint(0, 7, (2, 3), generator=g)
    x[0, 0, 7] = 200.0                  # a target 200 below: exp(ref - logp) is beyond FP32
    x.requires_grad_(True)
    old = F.token_logprobs(x, t).detach()
    ref = torch.full((2, 3), -1.0)
    grads = []
    for with_ref in (None, ref):
        r = F.policy_loss(x, t, old, torch.ones(2), with_ref, kl=kl)
        grads.append((r.loss.detach(), torch.autograd.grad(r.loss, x)[0]))
    assert bool(torch.isfinite(grads[1][1]).all()) and float(r.kl[0, 0]) == (math.inf if kl == "k3" else pytest.approx(float(r.kl[0, 0])))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("ent", [0.0, 0.05])
def test_masked_vocabulary(ent):
    """Entries of -inf have no weight and no gradient in the policy loss: as the vocabulary without them."""
    g = torch.Generator().manual_seed(3)
    short = torch.randn(2, 4, 9, dtype=torch.float64, generator=g, requires_grad=True)
    t = torch.randint(0, 9, (2, 4), generator=g)
    t[1, 3] = -100
    x = torch.cat([short.detach(), torch.full((2, 4, 5), -math.inf, dtype=torch.float64)], -1).requires_grad_(True)
    old, adv = torch.full((2, 4), -2.0), torch.tensor([1.0, -0.5])
    results = []
    for v in (short, x):
        r = F.policy_loss(v, t, old, adv, entropy_coef=ent)
        results.append((r.loss.detach(), r.entropy, torch.autograd.grad(r.loss, v)[0]))
    (a, ea, ga), (b, eb, gb) = results
    assert torch.allclose(a, b) and torch.allclose(ea, eb) and torch.allclose(ga, gb[..., :9]) and bool((gb[..., 9:] == 0).all())


def test_advantages_of_zero_beside_ratios_beyond_fp32():
    x = torch.zeros(2, 2, 8, requires_grad=True)
    t = torch.zeros(2, 2, dtype=torch.long)
    old = torch.full((2, 2), -100.0)                     # exp(100 - ln 8)
    r = F.policy_loss(x, t, old, torch.zeros(2))
    r.loss.backward()
    assert float(r.loss.detach()) == 0.0 and bool((x.grad == 0).all())
    old[0, 0] = math.nan
    assert math.isnan(float(F.policy_loss(x, t, old, torch.zeros(2)).loss.detach()))
    assert math.isinf(float(F.policy_loss(x, t, torch.full_like(old, -100.0), -torch.ones(2)).loss.detach()))


def test_refuses_an_ignored_index_beyond_64_bits():
    x, t, z = torch.zeros(2, 3, 8), torch.ones(2, 3, dtype=torch.long), torch.zeros(2, 3)
    for index in (2 ** 64 + 1, 2 ** 63, -2 ** 63 - 1):
        for call in (lambda: F.token_logprobs(x, t, ignore_index=index), lambda: F.linear_logprobs(x, torch.zeros(5, 8), t, ignore_index=index),
                     lambda: F.policy_loss(x, t, z, z, ignore_index=index), lambda: F.preference_loss(x, t, ignore_index=index)):
            with pytest.raises(ValueError, match="ignore_index"):
                call()
    assert bool((F.token_logprobs(x, t, ignore_index=2 ** 63 - 1) != 0).all())


@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.float16), (torch.float32, torch.float64)])
def test_clipped_values_of_a_wider_type_are_rounded_once(src, dst):
    g = torch.randn(500, generator=torch.Generator().manual_seed(0)).to(src)
    out = torch.empty(500, dtype=dst)
    F.clip_grad_norm_([g], 1.0, out=[out])
    want = g.double() / (g.double().norm() + 1e-6)
    step = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}[dst]
    # the factor as FP32 or FP64, the product, the type it goes to; half a subnormal step of FP16
    assert bool(((out.double() - want).abs() <= (2 * max(step, 2.0 ** -53) + 2.0 ** -24 * (dst != torch.float64) + 2.0 ** -51) * want.abs() + 2.0 ** -25 * (dst == torch.float16)).all())

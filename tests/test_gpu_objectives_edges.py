"""Ends of the ranges that the fine-tuning operators take, on the GPU: temperatures, rows far below their maximum, infinite margins, derivatives
that are asked for in other ways.  Tolerances as in `test_gpu_objectives.py`, whose helpers are used."""
import math

import pytest
import torch
from test_gpu_objectives import BF16, F16, F32, U, close, grad_error, logp_error, softmax64

from nexus_b200.fused import ops as F

pytestmark = pytest.mark.gpu
STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: U}


# ------------------------------------------------------------------------------------------------ low temperatures
# target logits from which (target / temperature) log2 e is rounded by more than one
LOW = [(1e-8, 4.0, 60.0), (1e-7, 200.0, 600.0), (1e-6, 1500.0, 6000.0), (1e-5, 15000.0, 60000.0), (1e-4, 30000.0, 64000.0)]


def low_rows(dtype, lo, hi, vocab=300):
    """[3, 64] rows at 64 values of the target's logit: alone above all others; beside another of the same value; a step below the largest."""
    g = torch.Generator().manual_seed(int(lo))
    top = torch.linspace(lo, hi, 64).to(dtype)
    x = torch.randn(3, 64, vocab, generator=g).to(dtype)
    t = torch.randint(1, vocab, (3, 64), generator=g)
    x.scatter_(2, t[..., None], top[None, :, None].expand(3, 64, 1))
    x[1:, :, 0] = top
    below = top * (1 - 2 * torch.finfo(dtype).eps)
    x[2].scatter_(1, t[2][:, None], below[:, None])
    return x.cuda(), t.cuda()


def low_expected(x, t, temperature):
    lp = softmax64(x, x.shape[-1], temperature)
    p = lp.exp()
    return lp.gather(2, t[..., None])[..., 0], p, -torch.where(p > 0, p * lp.clamp(min=-1e30), 0.0).sum(-1), torch.where(p > 0, lp, 0.0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("temperature,lo,hi", LOW)
def test_token_logprobs_at_low_temperatures(dtype, temperature, lo, hi):
    x, t = low_rows(dtype, lo, hi)
    want, p, _, _ = low_expected(x, t, temperature)
    x.requires_grad_(True)
    logp = F.token_logprobs(x, t, temperature=temperature)
    close(logp.detach(), want, logp_error(want, 300))
    logp.backward(torch.full_like(logp, temperature))
    delta = torch.nn.functional.one_hot(t, 300).double()
    one = torch.ones(3, 64, 1, dtype=torch.float64, device="cuda")
    # the coefficient is a product with the rounded inverse of the temperature
    close(x.grad, delta - p, grad_error(delta - p, p, one, dtype, 300, coef_rel=4 * U))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("temperature,lo,hi", LOW)
@pytest.mark.parametrize("ent", [0.0, 0.05])
def test_policy_loss_at_low_temperatures(dtype, temperature, lo, hi, ent):
    x, t = low_rows(dtype, lo, hi)
    want, p, H, lp = low_expected(x, t, temperature)
    old = want.float()
    old[2] = 0.0        # far from the old log-probability: the ratio is exp(logp), mostly zero
    adv = torch.ones(3, device="cuda")
    x.requires_grad_(True)
    r = F.policy_loss(x, t, old, adv, entropy_coef=ent, temperature=temperature, reduction="sum", scale=temperature)
    r.loss.backward()
    close(r.logp, want, logp_error(want, 300))
    close(r.entropy, H, U * (8 * H + 40 + 32))
    c = torch.ones(3, 64, 1, dtype=torch.float64, device="cuda")
    c[2] = torch.exp(want[2])[:, None]      # off by logp's own error, of itself
    delta = torch.nn.functional.one_hot(t, 300).double()
    gw = -c * (delta - p) + ent * torch.where(p > 0, p * (lp + H[..., None]), 0.0)
    size = c + ent * (H[..., None] + 20.0)
    rel = 64 * U + logp_error(want, 300)[..., None]
    close(x.grad, gw, grad_error(gw, p, size, dtype, 300, coef_rel=rel) + STEP[dtype] * gw.abs())
    loss = temperature * float((-c[..., 0] - ent * H).sum())
    assert float(r.loss.detach()) == pytest.approx(loss, rel=1e-5)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("temperature,lo,hi", LOW)
def test_preference_loss_at_low_temperatures(dtype, temperature, lo, hi):
    x, t = low_rows(dtype, lo, hi)
    x, t = x[:2].contiguous(), t[:2]          # targets that share the largest value against ones that have it alone
    want, p, _, _ = low_expected(x, t, temperature)
    x.requires_grad_(True)
    r = F.preference_loss(x, t, beta=0.1, temperature=temperature)
    (r.loss * temperature).backward()
    h = float(want[0].sum() - want[1].sum())
    assert h == pytest.approx(64 * math.log(2), rel=1e-6) and float(r.margin) == pytest.approx(h, rel=1e-5)
    assert float(r.loss.detach()) == pytest.approx(math.log1p(math.exp(-0.1 * h)), rel=1e-5)
    slope = 0.1 / (1.0 + math.exp(0.1 * h))
    delta = torch.nn.functional.one_hot(t, 300).double()
    gw = slope * torch.tensor([-1.0, 1.0], device="cuda", dtype=torch.float64)[:, None, None] * (delta - p)
    size = torch.full((2, 64, 1), slope, dtype=torch.float64, device="cuda")
    close(x.grad, gw, grad_error(gw, p, size, dtype, 300, coef_rel=64 * U))


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
def dual_calls(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 5, 24, generator=g).to(dtype).cuda()
    t = torch.randint(0, 24, (4, 5), generator=g).cuda()
    t[0, :2] = -100
    h, w = torch.randn(4, 5, 16, generator=g).to(dtype).cuda(), torch.randn(24, 16, generator=g).to(dtype).cuda()
    old, adv = torch.full((4, 5), -3.0, device="cuda"), torch.ones(4, device="cuda")
    return [(lambda v: F.token_logprobs(v, t), x), (lambda v: F.policy_loss(v, t, old, adv, entropy_coef=0.1).loss, x),
            (lambda v: F.preference_loss(v, t).loss, x), (lambda v: F.linear_logprobs(v, w, t), h), (lambda v: F.linear_logprobs(h, v, t), w)]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_forward_mode_derivatives(dtype):
    """A tangent along v against the product of v with the gradient; values as without one."""
    from torch.autograd import forward_ad
    for call, x in dual_calls(dtype):
        v = torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(dtype)
        leaf = x.clone().requires_grad_(True)
        out = call(leaf)
        up = torch.randn(out.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
        want = float((torch.autograd.grad(out, leaf, up)[0].double() * v.double()).sum())
        with forward_ad.dual_level():
            got = forward_ad.unpack_dual(call(forward_ad.make_dual(x, v)))
            assert got.tangent is not None
            tangent = float((got.tangent.double() * up.double()).sum())
        _, by_func = torch.func.jvp(call, (x,), (v,))
        # the sums have some hundred elements of order one, each rounded to the type
        room = 4 * STEP[dtype] * x.numel() ** 0.5 + 1e-5
        assert abs(tangent - want) < room and abs(float((by_func.double() * up.double()).sum()) - want) < room
        assert torch.allclose(got.primal.detach(), out.detach(), atol=0.1 if dtype == BF16 else 1e-5)


def test_forward_mode_derivatives_of_gradients_are_refused():
    from torch.autograd import forward_ad
    for call, x in dual_calls(F32)[:3]:
        leaf = x.clone().requires_grad_(True)
        with forward_ad.dual_level():
            out = call(leaf)
            up = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, up)


def test_tangents_of_constants_are_dropped():
    from torch.autograd import forward_ad
    x, t = torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda")
    with forward_ad.dual_level():
        old = forward_ad.make_dual(torch.zeros(2, 3, device="cuda"), torch.ones(2, 3, device="cuda"))
        for v in (x, x.double()):
            assert forward_ad.unpack_dual(F.policy_loss(v, t, old, torch.ones(2, device="cuda")).loss).tangent is None


# ------------------------------------------------------------------------------------------------ targets far below the maximum
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("below", [40.0, 60.0, 75.0, 80.0, 83.0, 100.0])
@pytest.mark.parametrize("ent", [0.0, 1e-3])
def test_policy_gradient_of_unlikely_targets(dtype, below, ent):
    """A weight per token of 1e-5 over a sum of exponentials up to e^100 times the target's own: the gradient keeps its digits."""
    g = torch.Generator().manual_seed(int(below))
    x = torch.randn(2, 6, 900, generator=g).to(dtype).cuda()
    t = torch.randint(0, 400, (2, 6), generator=g).cuda()
    x[..., 500:503] = torch.tensor([below, below - 1.0, below - 3.0], dtype=dtype)
    x.scatter_(2, t[..., None], 0.0)
    want = softmax64(x, 900, 1.0)
    p, one = want.exp(), want.gather(2, t[..., None])[..., 0]
    H = -(p * want).sum(-1, keepdim=True)
    x.requires_grad_(True)
    r = F.policy_loss(x, t, one.float(), torch.ones(2, device="cuda"), entropy_coef=ent, reduction="sum", scale=1e-5)
    r.loss.backward()
    close(r.logp, one, logp_error(one, 900))
    delta = torch.nn.functional.one_hot(t, 900).double()
    gw = 1e-5 * (-(delta - p) + ent * p * (want + H))
    # the ratio is off by the errors of logp and of the old one's rounding; log p + H by two roundings of either
    rel = 64 * U + float(logp_error(one, 900).max()) + U * (below + 20)
    size = 1e-5 * (1.0 + ent * (H + 20.0))
    close(x.grad, gw, grad_error(gw, p, size, dtype, 900, coef_rel=rel) + STEP[dtype] * gw.abs())


@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0)])
@pytest.mark.parametrize("side", [0, 1])
def test_preference_of_a_sequence_that_cannot_be(kind, smoothing, side):
    """A target whose logit is -inf in the chosen sequence (0) or in the rejected one (1): the loss is its limit, and the gradient finite."""
    x = torch.zeros(4, 2, 4, device="cuda")
    x[2 * side, 1, 0] = -math.inf        # of the first pair, which is rows 0 and 2
    x.requires_grad_(True)
    t = torch.zeros(4, 2, dtype=torch.long, device="cuda")
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
    x = torch.randn(2, 3, 8, generator=g).cuda()
    t = torch.randint(0, 7, (2, 3), generator=g).cuda()
    x[0, 0, 7] = 200.0                  # a target 200 below: exp(ref - logp) is beyond FP32
    x.requires_grad_(True)
    old = F.token_logprobs(x, t).detach()
    ref = torch.full((2, 3), -1.0, device="cuda")
    grads = []
    for with_ref in (None, ref):
        r = F.policy_loss(x, t, old, torch.ones(2, device="cuda"), with_ref, kl=kl)
        grads.append((r.loss.detach(), torch.autograd.grad(r.loss, x)[0]))
    assert bool(torch.isfinite(grads[1][1]).all()) and float(r.kl[0, 0]) == (math.inf if kl == "k3" else pytest.approx(float(r.kl[0, 0])))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_advantages_of_zero_beside_ratios_beyond_fp32():
    x = torch.zeros(2, 2, 8, device="cuda", requires_grad=True)
    t = torch.zeros(2, 2, dtype=torch.long, device="cuda")
    old = torch.full((2, 2), -100.0, device="cuda")                     # exp(100 - ln 8)
    r = F.policy_loss(x, t, old, torch.zeros(2, device="cuda"))
    r.loss.backward()
    assert float(r.loss.detach()) == 0.0 and bool((x.grad == 0).all())
    old[0, 0] = math.nan
    assert math.isnan(float(F.policy_loss(x, t, old, torch.zeros(2, device="cuda")).loss.detach()))
    assert math.isinf(float(F.policy_loss(x, t, torch.full_like(old, -100.0), -torch.ones(2, device="cuda")).loss.detach()))


@pytest.mark.parametrize("form", ["whole", "view"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_kept_graph_costs_one_copy_of_the_gradient(dtype, form):
    full = torch.randn(2, 65, 8200, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(dtype)
    x = (full if form == "whole" else full[:, 1:, :8100]).detach().requires_grad_(True)
    t = torch.randint(0, 8100, x.shape[:2], device="cuda")
    old, adv = torch.full(x.shape[:2], -9.0, device="cuda"), torch.tensor([1.0, -2.0], device="cuda")
    loss = F.policy_loss(x, t, old, adv, entropy_coef=0.01).loss
    up = torch.tensor(0.3, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    (a,) = torch.autograd.grad(loss, x, up, retain_graph=True)
    assert torch.cuda.max_memory_allocated() - before < 1.1 * full.numel() * full.element_size() + (1 << 21)
    (b,) = torch.autograd.grad(loss, x, up, retain_graph=True)
    (c,) = torch.autograd.grad(loss, x, retain_graph=True)
    (d,) = torch.autograd.grad(loss, x, up)
    assert torch.equal(a, b) and torch.equal(a, d) and torch.equal(a, (c.float() * up).to(dtype))

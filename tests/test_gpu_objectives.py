"""Log-probabilities of given tokens, policy loss and preference loss on the GPU against the definitions in 64 bits.

Tolerances.  u = 2^-24.  A row's exponent is a difference (u of itself), a product (u) and the exponential (2^-22): e^-z is off by
(2 z + 4) u of itself.  Averaged over a row, z is at most ln V.  The sum runs over at most V / 512 + 32 additions in a chain and is off
by u for each.  logp adds the target's own difference and product (2 |z_t| u) and its own rounding.  A gradient element is c (delta - p)
with p off by the same of itself, and rounds once to its type."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def chain(vocab):
    return vocab / 512 + 32


def logp_error(logp, vocab):
    """Bound on the error of FP32 log-probabilities (FP64 tensor of the true ones)."""
    return U * (4 * logp.abs() + 8 + 2 * math.log(max(vocab, 2)) + chain(vocab))


def close(got, want, error):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = torch.isnan(want) | (got == want) | ((got - want).abs() <= error)
    assert bool(ok.all()), (int((~ok).sum()), float(((got - want).abs() / (error + 1e-300))[~ok].max()))


def softmax64(logits, vocab, temperature):
    x = logits.detach().double()[..., :vocab] / temperature
    return torch.log_softmax(x, -1)


def grad_error(want, p, coef, dtype, vocab, coef_rel=0.0):
    """Bound for gradients c (delta - p): `want` [..., V], p the probabilities, coef [..., 1] the rows' |c|."""
    z = -torch.log(p.clamp(min=1e-300)).clamp(max=110.0)
    own = p * U * (4 * z + 12 + 2 * math.log(max(vocab, 2)) + chain(vocab)) + 4 * U * (want != 0) * torch.minimum(torch.ones_like(p), want.abs() / coef.clamp(min=1e-300))
    step = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: U}[dtype]
    least = {BF16: 2.0 ** -126, F16: 2.0 ** -25, F32: 2.0 ** -126}[dtype]  # half a subnormal step of FP16; FP32 exponentials flush
    return step * want.abs() + coef * (1 + step) * own + coef_rel * want.abs() * 2 + least


def make(shape, vocab, dtype, seed=0, spread=2.5, pitch=None):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(*shape, pitch or vocab, generator=g)).to(dtype).cuda()
    t = torch.randint(0, vocab, shape, generator=g).cuda()
    return x, t, g


VOCABS = [1, 2, 7, 33, 1000, 4097, 50257]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", VOCABS)
def test_token_logprobs(dtype, vocab):
    x, t, g = make((3, 5), vocab, dtype, seed=vocab)
    t[0, :2] = -100
    t[2, 4] = -100
    x.requires_grad_(True)
    logp = F.token_logprobs(x, t, temperature=0.8)
    assert logp.dtype == F32 and logp.shape == t.shape
    lp = softmax64(x, vocab, 0.8)
    keep = t != -100
    want = torch.where(keep, lp.gather(2, t.clamp(min=0)[..., None])[..., 0], 0.0)
    close(logp.detach(), want, logp_error(want, vocab))
    assert bool((logp.detach()[~keep] == 0).all())
    d = torch.randn(t.shape, generator=g).cuda()
    logp.backward(d)
    p = lp.exp()
    delta = torch.nn.functional.one_hot(t.clamp(min=0), vocab).double()
    c = torch.where(keep, d.double(), 0.0)[..., None] / 0.8
    gw = c * (delta - p)
    assert x.grad.dtype == dtype
    close(x.grad, gw, grad_error(gw, p, c.abs(), dtype, vocab))
    assert bool((x.grad[~keep] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("form", ["padded", "sliced_time", "time_major", "odd_base", "column_step", "last_token", "expanded", "narrow_vocab_view"])
def test_token_logprobs_strides(dtype, form):
    vocab, B, T = 517, 3, 6
    g = torch.Generator().manual_seed(5)
    full = (2.0 * torch.randn(B, T + 1, 576, generator=g)).to(dtype).cuda()
    leaf = full.clone().requires_grad_(True)
    kw = {}
    if form == "padded":
        view = leaf[:, :T]
        kw = dict(vocab=vocab)
    elif form == "narrow_vocab_view":
        view = leaf[:, :T, :vocab]
    elif form == "sliced_time":
        view = leaf[:, 1:, :vocab]
    elif form == "time_major":
        view = leaf.transpose(0, 1)[:T].contiguous()[..., :vocab].transpose(0, 1)
    elif form == "odd_base":
        view = leaf.view(-1)[1: 1 + B * T * vocab].view(B, T, vocab)
    elif form == "column_step":
        view = leaf[:, :T, ::2][..., :250]
    elif form == "last_token":
        view = leaf[:, -1:, :vocab]
    else:
        view = leaf[:, :1, :vocab].expand(B, T, vocab)
    V = kw.get("vocab", view.shape[-1])
    t = torch.randint(0, V, view.shape[:-1], generator=g).cuda()
    d = torch.randn(view.shape[:-1], generator=g).cuda()
    logp = F.token_logprobs(view, t, **kw)
    (got,) = torch.autograd.grad(logp, leaf, d, retain_graph=True)
    # the same view in 64 bits
    leaf64 = full.double().requires_grad_(True)
    idx = torch.arange(full.numel(), device="cuda").view(full.shape)
    if form == "time_major":
        where = idx.transpose(0, 1)[:T].transpose(0, 1)[..., :vocab]
    elif form == "odd_base":
        where = idx.view(-1)[1: 1 + B * T * vocab].view(B, T, vocab)
    elif form == "column_step":
        where = idx[:, :T, ::2][..., :250]
    elif form == "last_token":
        where = idx[:, -1:, :vocab]
    elif form == "expanded":
        where = idx[:, :1, :vocab].expand(B, T, vocab)
    elif form == "sliced_time":
        where = idx[:, 1:, :vocab]
    else:
        where = idx[:, :T, :vocab]
    lp = torch.log_softmax(leaf64.view(-1)[where], -1)
    want = lp.gather(2, t[..., None])[..., 0]
    close(logp.detach(), want.detach(), logp_error(want.detach(), V))
    (gw,) = torch.autograd.grad(want, leaf64, d.double())
    peak = d.abs().double().amax() * (T if form == "expanded" else 1)
    # a broadcast row is rounded once per use and once per sum; the probability itself is off by p u (4 z + 12 + 2 ln V + chain) as in
    # `grad_error`, with p <= 1 and p z <= 1 / e: FP32 has to count that, BF16's step (2^-8) is far above it
    step = {BF16: 2.0 ** -8, F32: U}[dtype] * (T if form == "expanded" else 1)
    own = U * (2 + 12 + 2 * math.log(V) + chain(V))
    close(got, gw, (step + own) * peak + 0 * gw)
    (again,) = torch.autograd.grad(logp, leaf, d)
    assert torch.equal(got, again)


def test_int32_targets_and_other_ignore_index():
    x, t, _ = make((2, 9), 300, BF16)
    t[1, 3:] = 7
    a = F.token_logprobs(x, t, ignore_index=7)
    b = F.token_logprobs(x, t.int(), ignore_index=7)
    assert torch.equal(a, b) and bool((a[1, 3:] == 0).all()) and bool((a[0] != 0).any())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_masked_vocabulary(dtype):
    """Entries of -inf and of the type's lowest value have no weight and no gradient; a row's weight may lie on one entry."""
    vocab = 2000
    x, t, _ = make((1, 4), vocab, dtype, seed=3)
    x[0, 0, 100:] = -math.inf
    x[0, 1, 100:] = torch.finfo(dtype).min
    x[0, 2, 1:] = -math.inf
    x[0, 3, ::2] = -math.inf
    t[0] = torch.tensor([5, 6, 0, 7])
    x.requires_grad_(True)
    for ent in (0.0, 0.05):
        x.grad = None
        old = torch.full((1, 4), -3.0, device="cuda")
        r = F.policy_loss(x, t, old, torch.ones(1, 4, device="cuda"), entropy_coef=ent, reduction="sum")
        r.loss.backward()
        lp = softmax64(x, vocab, 1.0)
        p = lp.exp()
        plp = torch.where(p > 0, p * lp.clamp(min=-1e30), 0.0)
        H = -plp.sum(-1)
        want = lp.gather(2, t[..., None])[..., 0]
        close(r.logp, want, logp_error(want, vocab))
        close(r.entropy, H, U * (8 * H + 40 + chain(vocab)))
        ratio = torch.exp(want + 3.0)
        c = torch.where(ratio <= 1.2, -ratio, 0.0)[..., None]
        delta = torch.nn.functional.one_hot(t, vocab).double()
        gw = c * (delta - p) + ent * torch.where(p > 0, p * (lp.clamp(min=-1e30) + H[..., None]), 0.0)
        assert bool(torch.isfinite(x.grad).all())
        assert bool((x.grad[p == 0] == 0).all())
        size = c.abs() + ent * (H[..., None] + 20.0)
        close(x.grad, gw, grad_error(gw, p, size, dtype, vocab, coef_rel=64 * U) + {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: U}[dtype] * gw.abs())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("temperature", [1.0, 2.0 ** 14, 1.0e8])
@pytest.mark.parametrize("ent", [0.0, 0.05])
def test_masks_beside_the_lowest_value_and_at_high_temperatures(dtype, temperature, ent):
    """-inf has no weight where the target itself holds the type's lowest value (or lies next to it), nor where a high temperature brings all
    finite logits together."""
    vocab, low = 2000, torch.finfo(dtype).min
    x, t, _ = make((1, 4), vocab, dtype, seed=4)
    x[0, 0] = -math.inf
    x[0, 0, [3, 50, 700, 1999]] = low
    x[0, 1] = -math.inf
    x[0, 1, [3, 50]] = torch.tensor([-65472.0, -65504.0], dtype=dtype, device="cuda")
    x[0, 2, ::2] = -math.inf
    x[0, 3, 1:] = -math.inf
    t[0] = torch.tensor([700, 3, 7, 0])
    lp = softmax64(x, vocab, temperature)
    p = lp.exp()
    want = lp.gather(2, t[..., None])[..., 0]
    H = -torch.where(p > 0, p * lp.clamp(min=-1e30), 0.0).sum(-1)
    x.requires_grad_(True)
    r = F.policy_loss(x, t, want.float(), torch.ones(1, 4, device="cuda"), entropy_coef=ent, reduction="sum", temperature=temperature)
    r.loss.backward()
    close(r.logp, want, logp_error(want, vocab))
    close(F.token_logprobs(x.detach(), t, temperature=temperature), want, logp_error(want, vocab))
    close(r.entropy, H, U * (8 * H + 40 + chain(vocab)))
    delta = torch.nn.functional.one_hot(t, vocab).double()
    gw = (-(delta - p) + ent * torch.where(p > 0, p * (lp.clamp(min=-1e30) + H[..., None]), 0.0)) / temperature
    assert bool((x.grad[torch.isinf(x.detach())] == 0).all())
    size = (1.0 + ent * (H[..., None] + 20.0)) / temperature
    step = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: U}[dtype]
    close(x.grad, gw, grad_error(gw, p, size, dtype, vocab, coef_rel=64 * U) + step * gw.abs())


def test_ignored_rows_are_not_read_and_bad_targets_are_nan():
    x, t, _ = make((2, 3), 64, F32)
    x[0, 0] = math.nan
    t[0, 0] = -100
    t[1, 1] = 64
    t[1, 2] = -1
    x.requires_grad_(True)
    logp = F.token_logprobs(x, t)
    assert float(logp[0, 0].detach()) == 0.0 and bool(torch.isnan(logp[1, 1:]).all()) and bool(torch.isfinite(logp[0]).all())
    logp.sum().backward()
    assert bool((x.grad[0, 0] == 0).all()) and bool((x.grad[1, 1:] == 0).all()) and bool((x.grad[0, 1] != 0).all())
    x.grad = None
    r = F.policy_loss(x, t, torch.zeros(2, 3, device="cuda"), torch.ones(2, device="cuda"))
    assert math.isnan(float(r.loss.detach()))
    q = F.preference_loss(x, t)
    assert math.isnan(float(q.loss.detach()))


def test_nan_logits_show():
    x, t, _ = make((1, 3), 700, BF16)
    x[0, 1, 650] = math.nan
    r = F.policy_loss(x, t, torch.zeros(1, 3, device="cuda"), torch.ones(1, device="cuda"))
    assert torch.isnan(r.logp).tolist() == [[False, True, False]] and torch.isnan(r.entropy).tolist() == [[False, True, False]]
    assert torch.isnan(F.token_logprobs(x, t)).tolist() == [[False, True, False]]
    assert math.isnan(float(r.loss)) and math.isnan(float(F.preference_loss(x.expand(2, 3, 700), t.expand(2, 3)).loss))
    x.requires_grad_(True)
    F.policy_loss(x, t, torch.zeros(1, 3, device="cuda"), torch.ones(1, device="cuda")).loss.backward()
    assert bool(torch.isnan(x.grad[0, 1]).all()) and bool(torch.isfinite(x.grad[0, [0, 2]]).all())
    y = torch.zeros(1, 3, 700, device="cuda", requires_grad=True)
    for adv in (math.nan, math.inf):
        loss = F.policy_loss(y, t, torch.zeros(1, 3, device="cuda"), torch.tensor([adv], device="cuda")).loss
        assert not math.isfinite(float(loss.detach()))


def policy_inputs(B, T, vocab, dtype, pitch=None, seed=1):
    x, t, g = make((B, T), vocab, dtype, seed=seed, pitch=pitch)
    lp = softmax64(x, vocab, 1.0).gather(2, t[..., None])[..., 0]
    # ratios at steps of 1/64 in the logarithm: none within rounding of a border (ln 0.8 = -14.28 / 64, ln 1.28 = 15.8 / 64)
    old = (lp - torch.round(torch.randn(B, T, generator=g) * 12).cuda() / 64).float()
    ref = (lp + 0.2 * torch.randn(B, T, generator=g).cuda()).float()
    return x, t, old, ref, g


def policy64(x, t, old, adv, ref, vocab, kl, reduction, kl_coef, ent_coef, lo, hi, scale=1.0, temperature=1.0):
    leaf = x.detach().double().requires_grad_(True)
    keep = t != -100
    safe = torch.where(keep[..., None], leaf[..., :vocab], 0.0) / temperature
    lp = torch.log_softmax(safe, -1)
    one = lp.gather(2, t.clamp(min=0)[..., None])[..., 0]
    H = -(lp.exp() * lp).sum(-1)
    a = (adv if adv.dim() == 2 else adv[:, None].expand(t.shape)).double()
    r = torch.exp(one - old.double())
    gain = torch.minimum(r * a, r.clamp(1 - lo, 1 + hi) * a)
    d = ref.double() - one
    div = {"k1": -d, "k2": d * d / 2, "k3": torch.expm1(d) - d}[kl]
    per = torch.where(keep, kl_coef * div - gain - ent_coef * H, 0.0)
    n = keep.sum(-1).double()
    if reduction == "token":
        per = per / n.sum().clamp(min=1)
    elif reduction == "sequence":
        per = per / (n.clamp(min=1)[:, None] * (n > 0).sum().clamp(min=1))
    loss = per.sum() * scale
    loss.backward()
    zero = lambda v: torch.where(keep, v, 0.0).detach()  # noqa: E731
    return loss.detach(), zero(one), zero(div), zero(H), leaf.grad


@pytest.mark.parametrize("dtype,vocab,pitch", [(F32, 1000, 1000), (BF16, 4097, 4160), (F16, 333, 333), (BF16, 50257, 50304), (F32, 50257, 50257),
                                               (BF16, 128256, 128256), (BF16, 151936, 151936), (F32, 151936, 151936), (BF16, 600001, 600001)])
@pytest.mark.parametrize("kl,reduction,ent,wide", [("k1", "token", 0.0, False), ("k2", "sequence", 0.01, True), ("k3", "sum", 0.02, False)])
def test_policy_loss(dtype, vocab, pitch, kl, reduction, ent, wide):
    B, T = 3, 5
    x, t, old, ref, g = policy_inputs(B, T, vocab, dtype, pitch)
    t[0, 0] = t[1, 3:] = -100
    t[2] = -100                     # a sequence without tokens
    adv = torch.randn((B, T) if wide else (B,), generator=g).cuda()
    want = policy64(x, t, old, adv, ref, vocab, kl, reduction, 0.1, ent, 0.2, 0.28, scale=0.5)
    x.requires_grad_(True)
    r = F.policy_loss(x, t, old, adv, ref, clip_low=0.2, clip_high=0.28, kl_coef=0.1, kl=kl, entropy_coef=ent, reduction=reduction, scale=0.5,
                      vocab=vocab)
    r.loss.backward()
    err = logp_error(want[1], vocab)
    close(r.logp, want[1], err)
    close(r.kl, want[2], (1.0 + want[2].abs()) * (err + 8 * U))
    close(r.entropy, want[3], U * (8 * want[3] + 40 + 2 * chain(vocab)) * (want[3] != 0))
    n = {"token": float((t != -100).sum()), "sequence": 2.0, "sum": 1.0}[reduction]
    row = float((4 * err.max() + 32 * U) * (1 + adv.abs().max() * 3 + want[2].abs().max() + want[3].max()) * 0.5)
    close(r.loss.detach(), want[0], torch.full_like(want[0], row * (1 if reduction != "sum" else 15) + U * float(want[0].abs())))
    keep = (t != -100)[..., None]
    lp = softmax64(x, vocab, 1.0)
    p = lp.exp()
    weight = 0.5 / n / (1.0 if reduction != "sequence" else 3.0)
    size = torch.full_like(p[..., :1], 0.5 * (float(adv.abs().max()) * 2 + 0.1 * float(want[2].abs().max() + 1) + ent * 40)) * keep
    del weight
    err_g = grad_error(want[4][..., :vocab], p, size, dtype, vocab, coef_rel=float(4 * err.max() + 32 * U))
    close(x.grad[..., :vocab], want[4][..., :vocab], err_g * keep)
    if pitch > vocab:
        assert bool((x.grad[..., vocab:] == 0).all())


@pytest.mark.parametrize("vocab", [20011, 57327, 57344, 57353, 120000, 230001])
@pytest.mark.parametrize("ent", [0.0, 0.02])
def test_policy_many_rows(vocab, ent):
    """Rows for every SM, at both sides of what the shorter ring holds, longer than the longer one, at odd addresses."""
    B, T = 2, 90
    x, t, old, ref, g = policy_inputs(B, T, vocab, BF16, seed=vocab)
    t[0, 5:30] = -100
    adv = torch.randn(B, generator=g).cuda()
    want = policy64(x, t, old, adv, ref, vocab, "k3", "token", 0.1, ent, 0.2, 0.28)
    x.requires_grad_(True)
    r = F.policy_loss(x, t, old, adv, ref, clip_low=0.2, clip_high=0.28, kl_coef=0.1, entropy_coef=ent)
    r.loss.backward()
    err = logp_error(want[1], vocab)
    close(r.logp, want[1], err)
    close(r.entropy, want[3], U * (8 * want[3] + 40 + 2 * chain(vocab)) * (want[3] != 0))
    p = softmax64(x, vocab, 1.0).exp()
    keep = (t != -100)[..., None]
    n = float(keep.sum())
    size = torch.full_like(p[..., :1], (float(adv.abs().max()) * 2 + 0.1 * float(want[2].abs().max() + 1) + ent * 40) / n) * keep
    close(x.grad, want[4], grad_error(want[4], p, size, BF16, vocab, coef_rel=float(4 * err.max() + 32 * U)) * keep)
    a = F.token_logprobs(x.detach(), t)
    close(a, want[1], err)


def test_offsets_beyond_32_bits():
    """Logits of more than 2^31 elements: the last rows and their gradients."""
    vocab, rows = 50257, 43000
    x = torch.empty(1, rows, vocab, dtype=BF16, device="cuda")
    x.view(-1)[: vocab * 1000].normal_()
    x.view(-1)[-vocab * 1000:].normal_()
    t = torch.full((1, rows), -100, device="cuda")
    t[0, :3] = t[0, -3:] = torch.tensor([0, 777, vocab - 1], device="cuda")
    assert x.numel() > 2 ** 31
    x.requires_grad_(True)
    zero = torch.full((1, rows), -11.0, device="cuda")
    logp = F.token_logprobs(x, t)
    logp.backward(torch.ones_like(logp))
    token_grad, x.grad = x.grad, None
    r = F.policy_loss(x, t, zero, torch.ones(1, device="cuda"), reduction="sum")
    r.loss.backward()  # its sums run over other threads than those of `token_logprobs`: each is held against the 64-bit values by itself
    for part in (slice(0, 3), slice(rows - 3, rows)):
        lp = torch.log_softmax(x.detach()[0, part].double(), -1)
        want = lp.gather(1, t[0, part][:, None])[:, 0]
        close(logp.detach()[0, part], want, logp_error(want, vocab))
        close(r.logp[0, part], want, logp_error(want, vocab))
        gw = -lp.exp()
        gw.scatter_add_(1, t[0, part][:, None], torch.ones(3, 1, dtype=torch.float64, device="cuda"))
        one = torch.ones(3, 1, dtype=torch.float64, device="cuda")
        close(token_grad[0, part], gw, grad_error(gw, lp.exp(), one, BF16, vocab))
        ratio = torch.exp(want + 11.0)[:, None]
        c = torch.where(ratio <= 1.2, -ratio, 0.0)
        close(x.grad[0, part], c * gw, grad_error(c * gw, lp.exp(), c.abs(), BF16, vocab, coef_rel=64 * U))
    assert bool((token_grad[0, 3: 1000] == 0).all()) and bool((x.grad[0, rows - 1000: rows - 3] == 0).all())


def test_one_token_without_a_batch():
    x, t, _ = make((1,), 50, F32)
    a = F.token_logprobs(x[0], t[0])
    assert a.shape == () and torch.equal(a, F.token_logprobs(x, t)[0])


def test_saved_tensors_on_the_host():
    """Saved tensors that hooks move away and bring back at other addresses."""
    x, t, old, ref, g = policy_inputs(2, 6, 333, BF16, 336)
    adv = torch.randn(2, generator=g).cuda()
    x.requires_grad_(True)

    def grads():
        a = torch.autograd.grad(F.policy_loss(x, t, old, adv, ref, kl_coef=0.1, vocab=333).loss * 0.5, x)[0]
        b = torch.autograd.grad(F.token_logprobs(x[:, 1:, :333], t[:, 1:]).sum(), x)[0]
        return a, b, torch.autograd.grad(F.preference_loss(x, t, vocab=333).loss, x)[0]

    plain = grads()
    with torch.autograd.graph.save_on_cpu():
        moved = grads()
    assert all(torch.equal(a, b) for a, b in zip(plain, moved))


def test_policy_gradient_against_differences():
    """The gradient in FP32 against central differences of the loss in 64 bits along random directions."""
    B, T, vocab = 2, 6, 257
    x, t, old, ref, g = policy_inputs(B, T, vocab, F32, seed=9)
    adv = torch.randn(B, generator=g).cuda()
    x.requires_grad_(True)
    kw = dict(kl_coef=0.1, entropy_coef=0.01)
    F.policy_loss(x, t, old, adv, ref, **kw).loss.backward()
    for s in range(3):
        v = torch.randn(x.shape, generator=g).cuda().double()
        h = 1e-4  # third-order term: h^2 / 6 of third derivatives of order one, 2e-9
        lo, hi = (F.policy_loss(x.detach().double() + e * h * v, t, old, adv, ref, **kw).loss for e in (-1, 1))
        diff = float((hi - lo) / (2 * h))
        got = float((x.grad.double() * v).sum())
        assert abs(diff - got) <= 1e-6 + 1e-5 * abs(diff)


def test_policy_gradient_of_a_scaled_loss():
    x, t, old, ref, g = policy_inputs(2, 8, 700, F32, 704)
    adv = torch.randn(2, generator=g).cuda()
    x.requires_grad_(True)
    call = lambda **kw: F.policy_loss(x, t, old, adv, ref, kl_coef=0.1, vocab=700, **kw).loss  # noqa: E731
    (one,) = torch.autograd.grad(call(), x)
    (third,) = torch.autograd.grad(call() * 0.375, x)
    assert torch.equal(third, one * 0.375)
    (inside,) = torch.autograd.grad(call(scale=0.375), x)
    assert float((inside - third).abs().max()) <= 4 * U * float(third.abs().max())
    loss = call()
    a = torch.autograd.grad(loss, x, torch.tensor(2.0, device="cuda"), retain_graph=True)[0]
    b = torch.autograd.grad(loss, x, torch.tensor(2.0, device="cuda"))[0]
    assert torch.equal(a, b) and torch.equal(a, one * 2.0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(call(), x, create_graph=True)[0].sum(), x)


@pytest.mark.parametrize("vocab", [333, 50257])
@pytest.mark.parametrize("ent", [0.0, 0.02])
@pytest.mark.parametrize("keep_graph", [False, True])
def test_fp16_gradient_under_loss_scaling(vocab, ent, keep_graph):
    """A loss times 2^14 keeps the gradients that FP16 could not hold without the factor."""
    B, T, factor = 4, 64, 2.0 ** 14
    x, t, old, ref, g = policy_inputs(B, T, vocab, F16, vocab + 7)
    t[1, 40:] = -100
    adv = (1e-3 * torch.randn(B, generator=g)).cuda()
    want = policy64(x, t, old, adv, ref, vocab, "k3", "token", 1e-3, 1e-3 * ent, 0.2, 0.28)
    x.requires_grad_(True)
    r = F.policy_loss(x, t, old, adv, ref, clip_low=0.2, clip_high=0.28, kl_coef=1e-3, entropy_coef=1e-3 * ent, vocab=vocab)
    (got,) = torch.autograd.grad(r.loss * factor, x, retain_graph=keep_graph)
    if keep_graph:
        (again,) = torch.autograd.grad(r.loss * factor, x)
        assert torch.equal(got, again)
    keep = (t != -100)[..., None]
    p = softmax64(x, vocab, 1.0).exp()
    gw = factor * want[4]
    n = float((t != -100).sum())
    size = factor / n * 1e-3 * (2 * adv.abs().max().double() * 1e3 + float(want[2].abs().max()) + 1 + ent * 40) * keep
    err = grad_error(gw[..., :vocab], p, size, F16, vocab, coef_rel=float(4 * logp_error(want[1], vocab).max() + 32 * U))
    close(got[..., :vocab], gw[..., :vocab], err * keep)
    assert bool((got[..., vocab:] == 0).all())
    assert float((got[..., :vocab] != 0).float().mean()) > float(((gw[..., :vocab].abs() > 2.0 ** -24)).float().mean()) - 1e-3


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("temperature", [1e-8, 1e-4, 1e4, 1e8])
def test_entropy_gradient_of_masked_rows_at_extreme_temperatures(dtype, temperature):
    """Entries of -inf have no gradient, and the others a finite one, at both ends of the temperatures that are allowed."""
    vocab = 700
    x, t, _ = make((2, 3), vocab, dtype, seed=8)
    x[0, :, 1::2] = -math.inf
    x[1, :, 1::2] = torch.finfo(dtype).min
    x[1, 1, 2] = -math.inf
    t -= t % 2
    t[1, 1] = 4
    x.requires_grad_(True)
    r = F.policy_loss(x, t, torch.zeros(2, 3, device="cuda"), torch.zeros(2, device="cuda"), entropy_coef=0.05, reduction="sum", temperature=temperature)
    r.loss.backward()
    lp = softmax64(x, vocab, temperature)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp.clamp(min=-1e30), 0.0).sum(-1, keepdim=True)
    gw = 0.05 / temperature * torch.where(p > 0, p * (lp.clamp(min=-1e30) + H), 0.0)
    assert bool(torch.isfinite(x.grad).all())
    assert bool((x.grad[torch.isinf(x.detach())] == 0).all())
    if dtype != F16 or temperature >= 1e4:     # elsewhere FP16 cannot hold an element of the gradient
        # t = (x - x0) k is off by two roundings of itself (z in `grad_error`), and log p + H by as much, absolutely: 20 covers both below
        size = 0.05 / temperature * (H + 20.0)
        step = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: U}[dtype]
        close(x.grad, gw, grad_error(gw, p, size, dtype, vocab, coef_rel=64 * U) + step * gw.abs())


@pytest.mark.parametrize("B,T", [(1, 1), (1, 300), (300, 1), (40, 7)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_shapes(B, T, reduction):
    x, t, old, ref, g = policy_inputs(B, T, 65, BF16, seed=B + T)
    drop = torch.rand(B, T, generator=g).cuda() < 0.3
    t = torch.where(drop, -100, t)
    adv = torch.randn(B, generator=g).cuda()
    want = policy64(x, t, old, adv, ref, 65, "k3", reduction, 0.1, 0.01, 0.2, 0.2)
    x.requires_grad_(True)
    r = F.policy_loss(x, t, old, adv, ref, kl_coef=0.1, entropy_coef=0.01, reduction=reduction)
    r.loss.backward()
    close(r.loss.detach(), want[0], torch.full_like(want[0], 400 * U * (1 + float(adv.abs().max()))))
    # per element: rounding to BF16, and the row's coefficient
    close(x.grad, want[4], (2.0 ** -8 + 400 * U) * want[4].abs() + 400 * U / max(1, int((t != -100).sum())) * 4 * (t != -100)[..., None])


def preference64(x, t, ref, vocab, beta, kind, smoothing, target, average, temperature=1.0):
    leaf = x.detach().double().requires_grad_(True)
    keep = t != -100
    lp = torch.log_softmax(torch.where(keep[..., None], leaf[..., :vocab], 0.0) / temperature, -1)
    one = torch.where(keep, lp.gather(2, t.clamp(min=0)[..., None])[..., 0], 0.0)
    s = one.sum(-1)
    if average:
        s = s / keep.sum(-1).clamp(min=1)
    P = t.shape[0] // 2
    r = s if ref is None else s - ref.double()
    h = r[:P] - r[P:]
    z = beta * h - target
    if kind == "sigmoid":
        each = -(1 - smoothing) * torch.nn.functional.logsigmoid(z) - smoothing * torch.nn.functional.logsigmoid(-z)
    elif kind == "hinge":
        each = (1 - z).clamp(min=0)
    else:
        each = (h - 0.5 / beta) ** 2
    each.mean().backward()
    return each.mean().detach(), s.detach(), h.detach(), leaf.grad, one.detach()


@pytest.mark.parametrize("dtype,pairs,T,vocab,pitch", [(F32, 1, 1, 50, 50), (BF16, 3, 9, 4097, 4160), (F16, 2, 300, 333, 333), (BF16, 40, 3, 128, 128),
                                                      (BF16, 1, 4, 151936, 151936)])
@pytest.mark.parametrize("kind,smoothing,target,average,with_ref", [("sigmoid", 0.0, 0.0, False, True), ("sigmoid", 0.1, 0.5, True, False),
                                                                    ("hinge", 0.0, 0.0, False, True), ("ipo", 0.0, 0.0, True, True)])
def test_preference_loss(dtype, pairs, T, vocab, pitch, kind, smoothing, target, average, with_ref):
    x, t, g = make((2 * pairs, T), vocab, dtype, seed=T + pairs, pitch=pitch)
    if T > 2:
        t[0, :2] = -100
        t[-1, T // 2:] = -100
    if pairs > 1:
        t[1] = -100                 # a sequence without tokens
    lp = softmax64(x, vocab, 1.0).gather(2, t.clamp(min=0)[..., None])[..., 0]
    total = torch.where(t != -100, lp, 0.0).sum(-1)
    if average:
        total = total / (t != -100).sum(-1).clamp(min=1)
    ref = (total + (0.2 if average else 2.0) * torch.randn(2 * pairs, generator=g).cuda()).float() if with_ref else None
    beta = 0.3
    loss, s, h, gw, one = preference64(x, t, ref, vocab, beta, kind, smoothing, target, average)
    x.requires_grad_(True)
    r = F.preference_loss(x, t, ref, beta=beta, kind=kind, label_smoothing=smoothing, target_margin=target, average=average, vocab=vocab)
    (r.loss * 0.5).backward()
    token = logp_error(one, vocab) * (t != -100)
    es = token.sum(-1) + U * s.abs()
    eh = es[:pairs] + es[pairs:] + U * h.abs()
    close(r.logp, s, es)
    close(r.margin, h, eh)
    slope = (2 * (h - 0.5 / beta)).abs().max() if kind == "ipo" else beta
    close(r.loss.detach(), loss, (slope * eh.max() + eh.max() ** 2 + U * loss.abs()))
    bend = 2.0 if kind == "ipo" else beta * beta
    size = 0.5 * torch.full((2 * pairs, 1, 1), float(slope) / pairs, device="cuda", dtype=torch.float64)
    p = softmax64(x, vocab, 1.0).exp()
    keep = (t != -100)[..., None]
    err = grad_error(0.5 * gw[..., :vocab], p, size, dtype, vocab, coef_rel=8 * U) + 0.5 * bend * float(eh.max()) / pairs * (p + (gw[..., :vocab] != 0) * 1.0)
    close(x.grad[..., :vocab], 0.5 * gw[..., :vocab], err * keep)
    assert bool((x.grad[..., vocab:] == 0).all())


def test_extreme_margins():
    """Log-ratios far apart: the sigmoid loss grows linearly on one side and vanishes on the other, without overflow."""
    x, t, _ = make((2, 1), 16, F32)
    for off in (-1e4, 1e4):
        ref = torch.tensor([0.0, off], device="cuda")
        r = F.preference_loss(x, t, ref, beta=1.0)
        h = float(r.margin)
        assert math.isfinite(float(r.loss.detach()))
        assert float(r.loss.detach()) == pytest.approx(max(0.0, -h), rel=4 * U, abs=1e-30)


def test_other_stream_and_two_graphs():
    """Calls captured into two graphs that are replayed in turn, and one on a side stream, give what plain calls give."""
    made = [policy_inputs(2, 40, 3000, BF16, 3008, seed=s) for s in (1, 2)]
    adv = torch.randn(2, 40, device="cuda")

    def step(i):
        x, t, old, ref, _ = made[i]
        x = x.detach().requires_grad_(True)
        r = F.policy_loss(x, t, old, adv, ref, kl_coef=0.1, entropy_coef=0.01, vocab=3000)
        (r.loss * 1.5).backward()
        q = F.preference_loss(x, t, vocab=3000)
        q.loss.backward()
        return r.loss.detach(), q.loss.detach(), x.grad

    plain = [step(i) for i in (0, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = step(0)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(aside, plain[0]):
        assert torch.equal(a, b)
    graphs, outs = [], []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, plain):
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_host_threads_on_streams_of_their_own():
    from concurrent.futures import ThreadPoolExecutor
    made = [policy_inputs(2, 30 + i, 3001, BF16, 3008, seed=i) for i in range(4)]
    adv = [torch.randn(2, 30 + i, device="cuda") for i in range(4)]
    h, w = torch.randn(300, 64, device="cuda", dtype=BF16), torch.randn(3001, 64, device="cuda", dtype=BF16)
    tk = torch.randint(0, 3001, (300,), device="cuda")

    def work(i):
        x, t, old, ref, _ = made[i]
        x = x.detach().requires_grad_(True)
        r = F.policy_loss(x, t, old, adv[i], ref, kl_coef=0.1, vocab=3001)
        (r.loss * 0.5).backward()
        hh, ww = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        g = torch.autograd.grad(F.linear_logprobs(hh, ww, tk).sum(), (hh, ww))
        gs = [x.grad.clone(), g[0].float()]
        n = F.clip_grad_norm_(gs, 0.1)
        return r.loss.detach(), x.grad, *g, n, *gs

    plain = [work(i) for i in range(4)]
    torch.cuda.synchronize()

    def aside(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                out = work(i)
        s.synchronize()
        return out

    with ThreadPoolExecutor(4) as ex:
        for out, want in zip(ex.map(aside, range(4)), plain):
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_no_gradient_asked():
    x, t, old, ref, _ = policy_inputs(2, 5, 100, BF16)
    adv = torch.ones(2, device="cuda")
    a = F.policy_loss(x, t, old, adv, ref, kl_coef=0.1)
    x.requires_grad_(True)
    with torch.no_grad():
        b = F.policy_loss(x, t, old, adv, ref, kl_coef=0.1)
    c = F.policy_loss(x, t, old, adv, ref, kl_coef=0.1)
    assert not a.loss.requires_grad and not b.loss.requires_grad and c.loss.requires_grad and not c.logp.requires_grad
    assert torch.equal(a.loss, b.loss) and torch.equal(a.loss, c.loss.detach())
    x.detach().fill_(0)  # the gradient does not read the logits again
    c.loss.backward()
    assert bool(torch.isfinite(x.grad).all()) and float(x.grad.abs().max()) > 0


def test_empty():
    x = torch.zeros(2, 0, 10, device="cuda", requires_grad=True)
    t = torch.zeros(2, 0, dtype=torch.long, device="cuda")
    assert F.token_logprobs(x, t).shape == (2, 0)
    z = torch.zeros(2, 0, device="cuda")
    r = F.policy_loss(x, t, z, z)
    assert float(r.loss.detach()) == 0.0
    r.loss.backward()
    assert F.preference_loss(x, t).margin.tolist() == [0.0]
    t2 = torch.full((2, 4), -100, device="cuda")
    y = torch.full((2, 4, 10), math.nan, device="cuda", requires_grad=True)
    r = F.policy_loss(y, t2, torch.zeros(2, 4, device="cuda"), torch.zeros(2, device="cuda"), reduction="sequence", entropy_coef=0.1)
    r.loss.backward()
    assert float(r.loss.detach()) == 0.0 and bool((y.grad == 0).all())

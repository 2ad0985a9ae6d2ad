"""Log-probabilities from hidden states and the head's weight on the GPU against the definitions in 64 bits.

Tolerances.  A logit is a sum of d exact products in FP32 on the tensor cores: off by at most (d + 4) 2^-23 of the sum of their
magnitudes (a truncating adder, each addition; in practice far less).  Row sums and logarithms as for logits in memory.  The gradient of the
logits is rounded to the operands' type before its products (half a step of each element), the products are summed in FP32 and rounded once
more; FP16 keeps 2^-24 / 2^15 of the largest coefficient as its smallest step."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
LEAST = {BF16: 2.0 ** -133, F16: 2.0 ** -25}


def make(shape, d, vocab, dtype, seed=0, spread=2.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(*shape, d, generator=g).to(dtype).cuda()
    w = (torch.randn(vocab + pad, d, generator=g) * (spread / math.sqrt(d))).to(dtype).cuda()
    t = torch.randint(0, vocab, shape, generator=g).cuda()
    return h, w, t, g


def expect(h, w, t, vocab, dlogp, temperature=1.0, ignore=-100):
    """In 64 bits: logp, bound on its error, d_hidden, d_weight and bounds on theirs."""
    dtype = h.dtype
    keep = (t != ignore).reshape(-1)
    H = torch.where(keep[:, None], h.detach().reshape(-1, h.shape[-1]).double(), 0.0)
    W = w.detach().double()[:vocab]
    x = H @ W.t() / temperature
    size = H.abs() @ W.abs().t() / temperature
    at = t.reshape(-1).clamp(min=0)[:, None]
    lp = torch.log_softmax(x, -1)
    logp = torch.where(keep, lp.gather(1, at)[:, 0], 0.0)
    ex = (H.shape[1] + 4) * 2 * U * size                      # of a logit
    p = lp.exp()
    mean_ex = (p * ex).sum(-1)
    err = keep * (ex.gather(1, at)[:, 0] + mean_ex + U * (4 * logp.abs() + 48 + 2 * math.log(max(vocab, 2)) + vocab / 4096))
    c = torch.where(keep, dlogp.reshape(-1).double(), 0.0)[:, None] / temperature
    G = c * -p
    G.scatter_add_(1, at, c)
    z = -lp.clamp(min=-110.0)
    # the exponentials and their product with the row's share are both rounded to the type (once, where the logits are made again)
    eg = c.abs() * p * (ex + mean_ex[:, None] + U * (4 * z + 60 + vocab / 4096) + STEP[dtype]) + STEP[dtype] * G.abs() + 4 * U * c.abs() * (G.abs() > 0) * torch.minimum(G.abs() / c.abs().clamp(min=1e-300), torch.ones_like(G))
    if dtype == F16:
        eg = eg + float(c.abs().max()) * 2.0 ** -39
    dh, dw = G @ W, G.t() @ H
    sum_h = (G.abs() + eg) @ W.abs()
    sum_w = (G.abs() + eg).t() @ H.abs()
    n = H.shape[0]
    eh = eg @ W.abs() + (min(vocab, 4096) + 40) * 2 * U * sum_h + STEP[dtype] * dh.abs() + LEAST[dtype]
    ew = eg.t() @ H.abs() + (min(n, 4096) + 40) * 2 * U * sum_w + STEP[dtype] * dw.abs() + LEAST[dtype]
    return logp, err, dh, eh, dw, ew


def close(got, want, error):
    off = (got.double().reshape(want.shape) - want).abs()
    assert bool(torch.isfinite(got).all())
    bad = off > error
    assert not bool(bad.any()), (int(bad.sum()), float((off / error.clamp(min=1e-300))[bad].max()))


def relative(got, want):
    return float((got.double().reshape(want.shape) - want).norm() / want.norm().clamp(min=1e-300))


SIZES = [((1,), 8, 5), ((8,), 64, 300), ((3, 5), 72, 257), ((2, 64), 128, 1000), ((129,), 256, 513), ((2, 128), 96, 4097), ((257,), 64, 128),
         ((3, 203), 160, 1031), ((1300,), 520, 777), ((700,), 264, 5003), ((300,), 2120, 1500)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,d,vocab", SIZES)
def test_forward_and_gradients(dtype, shape, d, vocab, monkeypatch):
    h, w, t, g = make(shape, d, vocab, dtype, seed=d + vocab, pad=3)
    if t.numel() > 4:
        t.view(-1)[::3] = -100
        t.view(-1)[-2:] = -100
    dl = torch.randn(shape, generator=g).cuda() / t.numel()
    want = expect(h, w, t, vocab, dl, 0.7)
    with torch.no_grad():
        plain = F.linear_logprobs(h, w, t, temperature=0.7, vocab=vocab)
    h.requires_grad_(True)
    w.requires_grad_(True)
    logp = F.linear_logprobs(h, w, t, temperature=0.7, vocab=vocab)
    assert logp.dtype == F32 and logp.shape == t.shape
    close(logp.detach(), want[0], want[1])
    close(plain, want[0], want[1])
    logp.backward(dl)
    assert h.grad.dtype == dtype and w.grad.dtype == dtype
    close(h.grad, want[2], want[3])
    close(w.grad[:vocab], want[4], want[5])
    assert bool((w.grad[vocab:] == 0).all())
    assert bool((h.grad.view(-1, d)[t.view(-1) == -100] == 0).all())
    # the other way of the backward pass, which the width alone would not take
    from nexus_b200.ops import _objectives as O
    monkeypatch.setattr(O, "HEAD_KEEP_WIDTH", 0 if d < O.HEAD_KEEP_WIDTH else 1 << 30)
    h2, w2 = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    other = F.linear_logprobs(h2, w2, t, temperature=0.7, vocab=vocab)
    assert torch.equal(other.detach(), logp.detach())
    other.backward(dl)
    close(h2.grad, want[2], want[3])
    close(w2.grad[:vocab], want[4], want[5])
    # as a whole: two roundings to the type, each at most half a step of every element
    assert relative(h.grad, want[2]) <= 2 * STEP[dtype] and relative(w.grad[:vocab], want[4]) <= 2 * STEP[dtype]


@pytest.mark.parametrize("rows", [300, 513])
def test_chunks_of_rows(rows, monkeypatch):
    """The gradient in several chunks of 256 rows, the weight's summed in FP32, some chunks without a row that counts."""
    from nexus_b200.ops import _objectives as O
    monkeypatch.setattr(O, "HEAD_GRAD_ELEMENTS", 1)
    for dtype in (BF16, F16):
        h, w, t, g = make((rows,), 136, 700, dtype, seed=rows)
        for kept in (rows, 270, 256, 100, 0):
            tk = t.clone()
            tk[torch.randperm(rows, generator=g)[kept:].cuda()] = -100
            dl = torch.randn(rows, generator=g).cuda()
            h2, w2 = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
            F.linear_logprobs(h2, w2, tk).backward(dl)
            want = expect(h, w, tk, 700, dl)
            close(h2.grad, want[2], want[3])
            close(w2.grad, want[4], want[5])


def test_forward_in_pieces_of_rows(monkeypatch):
    from nexus_b200.ops import _objectives as O
    h, w, t, g = make((900,), 72, 700, BF16, seed=12)
    t[::5] = -100
    t[7] = -3
    dl = torch.randn(900, generator=g).cuda()
    results = []
    for rows in (1 << 16, 256, 512):
        monkeypatch.setattr(O, "HEAD_ROWS", rows)
        h2, w2 = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        with torch.no_grad():
            plain = F.linear_logprobs(h2, w2, t)
        logp = F.linear_logprobs(h2, w2, t)
        assert torch.equal(plain.nan_to_num(9.0), logp.detach().nan_to_num(9.0)) and int(torch.isnan(plain).sum()) == 1
        results.append((plain.nan_to_num(9.0), *torch.autograd.grad(logp, (h2, w2), dl)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_one_token_without_a_batch():
    h, w, t, _ = make((1,), 64, 50, BF16)
    a = F.linear_logprobs(h[0], w, t[0])
    assert a.shape == () and torch.equal(a, F.linear_logprobs(h, w, t)[0])


def test_slices_of_the_vocabulary():
    from nexus_b200.ops import _objectives as O
    assert O.head_slices(300, 64) > 1 and O.head_slices(8192, 4096) == 1
    for dtype in (BF16, F16):
        h, w, t, g = make((300,), 64, 20000, dtype, seed=1)
        dl = torch.randn(300, generator=g).cuda()
        want = expect(h, w, t, 20000, dl)
        h.requires_grad_(True)
        F.linear_logprobs(h, w, t).backward(dl)        # only the hidden states' gradient
        close(h.grad, want[2], want[3])
        h2 = h.detach().clone()
        w.requires_grad_(True)
        F.linear_logprobs(h2, w, t).backward(dl)       # only the weight's
        close(w.grad, want[4], want[5])


@pytest.mark.parametrize("keep_width", [0, 1 << 30])
def test_backward_twice(keep_width, monkeypatch):
    from nexus_b200.ops import _objectives as O
    monkeypatch.setattr(O, "HEAD_KEEP_WIDTH", keep_width)
    for dtype in (BF16, F16):
        h, w, t, g = make((290,), 64, 800, dtype, seed=6)
        h.requires_grad_(True)
        w.requires_grad_(True)
        logp = F.linear_logprobs(h, w, t)
        d1, d2 = (torch.randn(290, generator=g).cuda() for _ in range(2))
        a = torch.autograd.grad(logp, (h, w), d1, retain_graph=True)
        b = torch.autograd.grad(logp, (h, w), d2, retain_graph=True)
        c = torch.autograd.grad(logp, (h, w), d1)
        assert all(torch.equal(x, y) for x, y in zip(a, c)) and not torch.equal(a[0], b[0])
        with pytest.raises(RuntimeError):
            torch.autograd.grad(logp, h, d1)


def test_small_coefficients_in_fp16():
    """Coefficients far below FP16's smallest step: the products keep their digits."""
    h, w, t, g = make((290,), 128, 3000, F16, seed=2)
    dl = torch.randn(290, generator=g).cuda() * 1e-9
    dl[5] = 1e-3 / 290
    t[7] = -100
    dl[7] = 1e6                                        # of a row that does not count
    want = expect(h, w, t, 3000, dl)
    h.requires_grad_(True)
    w.requires_grad_(True)
    F.linear_logprobs(h, w, t).backward(dl)
    close(h.grad, want[2], want[3])
    close(w.grad, want[4], want[5])


@pytest.mark.parametrize("form", ["pitch", "transposed_rows", "odd_base", "step"])
def test_strides(form):
    d, vocab = 64, 300
    h, w, t, g = make((2, 150), d, vocab, BF16, seed=4)
    wide = torch.randn(2, 150, 200, generator=g).to(BF16).cuda()
    flat = torch.randn(2 * 150 * d + 8, generator=g).to(BF16).cuda()
    view = {"pitch": wide[..., 8: 8 + d], "transposed_rows": h.transpose(0, 1), "odd_base": flat[1: 1 + 300 * d].view(2, 150, d),
            "step": wide[..., : 2 * d: 2]}[form].detach()
    wv = {"pitch": torch.cat([w, w], 1)[:, :d], "transposed_rows": w, "odd_base": torch.cat([w.view(-1)[:1], w.view(-1)])[1:].view(vocab, d),
          "step": w.t().contiguous().t()}[form]
    if form == "transposed_rows":
        t = t.t()
    dl = torch.randn(t.shape, generator=g).cuda()
    want = expect(view.contiguous(), wv.contiguous(), t.contiguous(), vocab, dl.contiguous())
    hv, ww = view.requires_grad_(True), wv.detach().requires_grad_(True)
    logp = F.linear_logprobs(hv, ww, t)
    close(logp.detach().contiguous(), want[0], want[1])
    logp.backward(dl)
    close(hv.grad.contiguous(), want[2], want[3])
    close(ww.grad.contiguous(), want[4], want[5])


def test_rows_that_do_not_count_may_hold_anything():
    for rows in (40, 400):
        h, w, t, g = make((rows,), 64, 500, BF16, seed=rows)
        t[::2] = -100
        t[1] = 500
        t[3] = -7
        clean = h.clone()
        h[::2] = math.nan
        h[1] = math.inf
        dl = torch.ones(rows, device="cuda")
        h.requires_grad_(True)
        w.requires_grad_(True)
        logp = F.linear_logprobs(h, w, t)
        with torch.no_grad():
            again = F.linear_logprobs(h, w, t)
        assert torch.equal(logp.detach().nan_to_num(9.0), again.nan_to_num(9.0))
        assert bool(torch.isnan(logp[[1, 3]]).all()) and bool((logp[::2] == 0).all())
        logp.backward(dl)
        clean[1] = clean[3] = 0
        tk = t.clone()
        tk[1] = tk[3] = -100
        want = expect(clean, w, tk, 500, dl)
        close(h.grad, want[2], want[3])
        close(w.grad, want[4], want[5])
        assert bool((h.grad[[1, 3]] == 0).all())


def test_masked_rows_of_the_weight_and_large_logits():
    """Logits of -inf have no weight; logits in the hundreds neither overflow nor lose the sum."""
    h, w, t, g = make((50,), 64, 700, BF16, seed=8, spread=200.0)
    want = expect(h, w, t, 700, torch.ones(50, device="cuda"))
    close(F.linear_logprobs(h, w, t), want[0], want[1])
    # products with the lowest weights sum to -inf or far below every other logit: the vocabulary without them
    h2 = h.abs()
    w2 = w.clone() / 100
    w2[300:] = torch.finfo(BF16).min
    t2 = t % 300
    short = expect(h2, w2[:300].contiguous(), t2, 300, torch.ones(50, device="cuda"))
    close(F.linear_logprobs(h2, w2, t2), short[0], short[1])


def test_other_types_and_sizes_go_through_the_logits():
    for dtype, d in ((F32, 24), (BF16, 20)):
        h, w, t, _ = make((2, 9), d, 50, dtype)
        a = F.linear_logprobs(h, w, t)
        b = F.token_logprobs(torch.nn.functional.linear(h, w), t)
        assert torch.equal(a, b)
    assert F.linear_logprobs(torch.zeros(0, 64, device="cuda", dtype=BF16), w.new_zeros(5, 64), torch.zeros(0, dtype=torch.long, device="cuda")).shape == (0,)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 3, 16, 17, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("d,vocab", [(8, 1), (72, 31), (1088, 33), (64, 5000), (1600, 20011), (2056, 4737)])
def test_few_rows(dtype, rows, d, vocab):
    """The form for single tokens: runs of the vocabulary per SM, fewer groups than SMs, runs that end inside a tile."""
    h, w, t, _ = make((rows,), d, vocab, dtype, seed=rows + d)
    if rows > 2:
        t[1] = -100
        t[2] = vocab
    logp = F.linear_logprobs(h, w, t, temperature=0.9)
    tk = torch.where(t >= vocab, -100, t)
    want = expect(h, w, tk, vocab, torch.ones(rows, device="cuda"), 0.9)
    bad = t >= vocab
    assert torch.equal(torch.isnan(logp), bad)
    close(logp[~bad], want[0][~bad], want[1][~bad])


def test_agrees_with_logits_in_memory():
    h, w, t, _ = make((4, 100), 256, 2000, BF16, seed=3)
    x = h.float().reshape(-1, 256) @ w.float().t()
    a, b = F.linear_logprobs(h, w, t), F.token_logprobs(x.view(4, 100, 2000), t)
    assert float((a - b).abs().max()) < 260 * 4 * U * 256


@pytest.mark.parametrize("recompute", [False, True])
def test_streams_graphs_and_repeated_backward(recompute):
    made = [make((3, 150), 1024, 900, BF16, seed=s) for s in (1, 2)]
    for h, w, t, _ in made:
        t[:, :40] = -100
    dl = torch.randn(3, 150, device="cuda")

    def step(i):
        h, w, t, _ = made[i]
        h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        logp = F.linear_logprobs(h, w, t, recompute=recompute)
        return (logp.detach(), *torch.autograd.grad(logp, (h, w), dl))

    plain = [step(i) for i in (0, 1)]
    assert all(torch.equal(a, b) for a, b in zip(plain[0], step(0)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = step(0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(aside, plain[0]))
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
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    from nexus_b200.ops import _cuda as K
    K.check_status()

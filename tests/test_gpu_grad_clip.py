"""Global gradient norm over many tensors and clipping on the GPU.  The sum is FP64 (2^-50 of itself here): the FP32 norm is off by half a
step, a clipped element by the rounding of the factor, of the product and of the type it goes to."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: U}
LEAST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}


def true_norm(grads):
    return math.sqrt(sum(float(g.double().pow(2).sum()) for g in grads))


def check(got, grads, norm, max_norm):
    coef = min(1.0, max_norm / (norm + 1e-6))
    for o, g in zip(got, grads):
        want = g.double() * coef
        err = (2 * U + STEP[o.dtype]) * want.abs() * (1 + 2 * U) + LEAST[o.dtype]
        assert bool(((o.double() - want).abs() <= err).all())


def tensors(sizes, types, seed=0, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=g)).to(types[i % len(types)]).cuda() for i, n in enumerate(sizes)]


@pytest.mark.parametrize("types", [[F32], [BF16], [F16], [F32, BF16, F16]])
@pytest.mark.parametrize("sizes", [[1], [3, 1, 8], [16384, 16385, 16383, 5], [1000003, 7, 65536], [17] * 300, [40000] * 600])
@pytest.mark.parametrize("max_norm", [0.0, 0.7, 1e9])
def test_in_place(types, sizes, max_norm):
    grads = tensors(sizes, types)
    before = [g.clone() for g in grads]
    want = true_norm(grads)
    norm = F.clip_grad_norm_(grads, max_norm)
    assert norm.dtype == F32 and norm.is_cuda and norm.dim() == 0
    assert abs(float(norm) - want) <= (U + 1e-12) * want
    check(grads, before, want, max_norm)
    if max_norm > want:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert F.grad_square_sum(before) == pytest.approx(want * want, rel=1e-12)


@pytest.mark.parametrize("src", [F32, BF16, F16])
@pytest.mark.parametrize("dst", [F32, BF16, F16])
@pytest.mark.parametrize("max_norm", [0.5, math.inf])
def test_out(src, dst, max_norm):
    grads = tensors([5, 40000, 333], [src])
    keep = [g.clone() for g in grads]
    out = [torch.full_like(g, 7.0, dtype=dst) for g in grads]
    norm = F.clip_grad_norm_(grads, max_norm, out=out)
    want = true_norm(grads)
    assert abs(float(norm) - want) <= (U + 1e-12) * want
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    check(out, keep, want, max_norm)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_alignment_views_and_neighbours(dtype):
    """Views that start anywhere in a flat buffer, in other orders or with gaps; what lies beside them stays."""
    flat = torch.zeros(400000, dtype=dtype, device="cuda")
    flat.fill_(3.0)
    cuts, at = [], 1
    for n in (1, 2, 9, 31, 64, 1000, 20001, 70000):
        cuts.append((at, n))
        at += n + 1
    views = [flat[a: a + n] for a, n in cuts]
    for i, v in enumerate(views):
        v.copy_(0.1 * torch.randn(v.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)))
    block = torch.randn(64, 96, device="cuda").to(dtype)
    views += [block.t()[:32], torch.randn(33, 17, device="cuda").to(dtype).t(), torch.randn(4, 5, 6, device="cuda").to(dtype).permute(2, 0, 1)]
    before = [v.clone() for v in views]
    whole = block.clone()
    want = true_norm(views)
    outs = [torch.empty(v.shape, dtype=BF16, device="cuda") for v in views]
    F.clip_grad_norm_(views, 0.25, out=outs)
    check(outs, before, want, 0.25)
    norm = F.clip_grad_norm_(views, 0.25)
    assert abs(float(norm) - want) <= (U + 1e-12) * want
    check(views, before, want, 0.25)
    gaps = torch.ones(400000, dtype=torch.bool, device="cuda")
    for a, n in cuts:
        gaps[a: a + n] = False
    assert bool((flat[gaps] == 3.0).all())
    assert torch.equal(block[:, 32:], whole[:, 32:])


def test_not_finite_and_extreme():
    for bad in (math.inf, math.nan):
        grads = tensors([10, 20], [F32])
        grads[1][3] = bad
        before = [g.clone() for g in grads]
        out = [torch.empty_like(g) for g in grads]
        norm = F.clip_grad_norm_(grads, 1.0, out=out)
        assert not math.isfinite(float(norm))
        assert not math.isfinite(float(F.clip_grad_norm_(grads, 1.0)))
        assert not math.isfinite(F.grad_square_sum(grads))
        for a, b, c in zip(grads, before, out):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and torch.equal(c.nan_to_num(7.0), b.nan_to_num(7.0))
    big = [torch.full((100,), 1e25, device="cuda"), torch.full((3,), 1e-30, device="cuda")]
    assert float(F.clip_grad_norm_(big, 1.0)) == pytest.approx(1e26, rel=1e-6)
    assert float(big[0][0]) == pytest.approx(0.1, rel=1e-5)
    small = [torch.full((100,), 1e-25, device="cuda")]
    assert float(F.clip_grad_norm_(small, 1.0)) == pytest.approx(1e-24, rel=1e-6)


def test_lists():
    a, b = torch.ones(4, device="cuda"), torch.full((5,), 2.0, device="cuda")
    assert float(F.clip_grad_norm_([a, None, torch.zeros(0, device="cuda"), b, a], 100.0)) == pytest.approx(math.sqrt(24.0), rel=1e-6)
    F.clip_grad_norm_([a, a], 1.0)
    assert float(a[0]) == pytest.approx(0.5, rel=1e-5)
    for call in (lambda: F.clip_grad_norm_([b[:3], b[2:]], 1.0), lambda: F.clip_grad_norm_([b, a.cpu()], 1.0),
                 lambda: F.clip_grad_norm_([torch.ones(1, device="cuda").expand(3)], 1.0)):
        with pytest.raises(ValueError):
            call()
    d = [torch.ones(3, device="cuda", dtype=torch.float64), torch.ones(1, device="cuda")]
    assert float(F.clip_grad_norm_(d, 1.0)) == 2.0 and float(d[0][0]) == pytest.approx(0.5, rel=1e-5)


def test_captured_and_on_another_stream():
    lists = [tensors([70000, 33, 1], [F32, BF16], seed=s, scale=1.0) for s in (0, 1)]
    keep = [[t.clone() for t in ts] for ts in lists]
    want = []
    for ts in keep:
        copy = [t.clone() for t in ts]
        want.append((F.clip_grad_norm_(copy, 1.0), copy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        copy = [t.clone() for t in keep[0]]
        n = F.clip_grad_norm_(copy, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(n, want[0][0]) and all(torch.equal(a, b) for a, b in zip(copy, want[0][1]))
    graphs, norms = [], []
    for ts in lists:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(F.clip_grad_norm_(ts, 1.0))
        graphs.append(g)
    for _ in range(2):
        for ts, ks in zip(lists, keep):
            for t, k in zip(ts, ks):
                t.copy_(k)
        for g in graphs:
            g.replay()
    for (n, out), ts, m in zip(want, lists, norms):
        assert torch.equal(n, m) and all(torch.equal(a, b) for a, b in zip(ts, out))


def test_trainer_and_adamw_take_the_kernels_norm():
    from nexus_b200.ops import _cuda as K
    ps = tensors([300, 7], [F32], seed=4)
    gs = tensors([300, 7], [F32], seed=5, scale=1.0)
    m, v = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
    before = K.launch_count
    norm = F.adamw_multi_tensor(ps, gs, m, v, 1, 1e-2, max_grad_norm=1.0)
    assert K.launch_count > before and norm == pytest.approx(true_norm(gs), rel=1e-13)


def test_lists_that_are_no_plain_ones():
    """What the quick look over a list leaves to the second one."""
    a = torch.ones(8, device="cuda")
    for call in (lambda: F.clip_grad_norm_([a, 3.0], 1.0), lambda: F.clip_grad_norm_([a, a.to_sparse()], 1.0),
                 lambda: F.clip_grad_norm_([a, a.int()], 1.0), lambda: F.clip_grad_norm_([a.view(2, 4)], 1.0, out=[torch.ones(4, 2, device="cuda")]),
                 lambda: F.clip_grad_norm_([a.view(BF16)[:8], a.view(F16)[:8]], 1.0), lambda: F.clip_grad_norm_([a], 1.0, out=[a.view(BF16)[:8]])):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(a, torch.ones(8, device="cuda"))
    out = [torch.empty(8, device="cuda", dtype=torch.float64)]
    assert float(F.clip_grad_norm_([a], 1.0, out=out)) == pytest.approx(math.sqrt(8.0), rel=1e-6)
    assert float(out[0][0]) == pytest.approx(1 / math.sqrt(8.0), rel=1e-5)
    assert torch.equal(F.clip_grad_norm_(a, 100.0), F.clip_grad_norm_([a], 100.0, out=[a]))

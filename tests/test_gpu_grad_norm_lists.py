"""The gradient norm in the optimizer and the trainer on the GPU: lists of one device (kernels), of two, with sparse gradients."""
import math

import pytest
import torch
from test_grad_norm_lists_cpu import Bag, batch

from nexus_b200.fused import ops as F
from nexus_b200.ops import _cuda as K
from nexus_b200.train import TrainerBuilder

pytestmark = pytest.mark.gpu


def test_gradients_on_two_devices():
    g = torch.Generator().manual_seed(2)
    make = lambda: [torch.randn(n, generator=g) for n in (70, 300, 5)]  # noqa: E731
    ps, gs = make(), make()
    runs = []
    for devices in (("cpu",) * 3, ("cuda", "cpu", "cuda")):
        to = lambda ts: [t.clone().to(d) for t, d in zip(ts, devices)]  # noqa: E731
        p, m, v = to(ps), [torch.zeros_like(t) for t in to(ps)], [torch.zeros_like(t) for t in to(ps)]
        norm = F.adamw_multi_tensor(p, to(gs), m, v, 1, 1e-2, max_grad_norm=1.0)
        assert norm == pytest.approx(math.sqrt(sum(float(t.double().pow(2).sum()) for t in gs)), rel=1e-13)
        runs.append([t.cpu() for t in p])
    for a, b in zip(*runs):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-8)
    with pytest.raises(ValueError):
        F.clip_grad_norm_([gs[0].cuda(), gs[1]], 1.0)


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("clip", [0.0, 0.05, 1e6])
def test_trainer_steps(sparse, clip):
    """Three steps of the trainer against the same steps in plain operations, on the parameters' own device."""
    tr = TrainerBuilder(Bag(sparse)).adamw(lr=0.1).gradient_clip_norm(clip).execution_policy("cuda").build()
    twin = Bag(False).cuda()
    x, y = batch()
    opt = [(torch.zeros_like(p), torch.zeros_like(p)) for p in twin.parameters()]
    for step in (1, 2, 3):
        before = K.launch_count
        tr.fit([(x, y)], epochs=1)
        assert sparse or K.launch_count > before          # one device, dense: the kernels' norm
        twin.zero_grad()
        torch.nn.functional.cross_entropy(twin(x.cuda()), y.cuda()).backward()
        norm = math.sqrt(sum(float(p.grad.double().pow(2).sum()) for p in twin.parameters()))
        coef = min(1.0, clip / (norm + 1e-6)) if clip else 1.0
        with torch.no_grad():
            for p, (m, v) in zip(twin.parameters(), opt):
                g = p.grad * coef
                m.mul_(0.9).add_(0.1 * g)
                v.mul_(0.999).add_(0.001 * g * g)
                p.mul_(1 - 0.1 * 0.01)
                p.sub_(0.1 * (m / (1 - 0.9 ** step)) / ((v / (1 - 0.999 ** step)).sqrt() + 1e-8))
    assert tr.global_step == 3
    for a, b in zip(tr.model.parameters(), twin.parameters()):
        # AdamW divides the first steps' gradients by their own size: rounding of some 1e-6 of a gradient is as much of a step of 0.1
        assert float((a - b).abs().max()) < 1e-5


def test_fp8_gradients_are_refused():
    """A type that the library has codes for and the clipping does not take, first or behind others; an output may have it."""
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda").to(torch.float8_e4m3fn)
    for call in (lambda: F.clip_grad_norm_([a, b], 1.0), lambda: F.clip_grad_norm_([b, a], 1.0), lambda: F.clip_grad_norm_([b], 1.0, out=[a])):
        with pytest.raises(ValueError, match="float8"):
            call()
    assert torch.equal(a, torch.ones(8, device="cuda"))
    assert float(F.clip_grad_norm_([2.0 * a], 1e3, out=[b])) == pytest.approx(32.0 ** 0.5) and bool((b.float() == 2.0).all())
    assert F.grad_square_sum([a, b]) == 40.0
    F.clip_grad_norm_([a], 8.0 ** 0.5 / 2, out=[b])
    assert bool((b.float() == 0.5).all())

"""How often each way of the backward pass of `linear_logprobs` rounds the logits' gradient to 16 bits, seen one element at a time: with the identity
as the head's weight the logits are the hidden states and d_hidden is that gradient (a product with one and zeros: exact)."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("recompute", [False, True])
def test_roundings_of_the_logits_gradient(dtype, rows, recompute):
    d = 512
    g = torch.Generator().manual_seed(rows)
    h = (2.5 * torch.randn(rows, d, generator=g)).to(dtype).cuda().requires_grad_(True)
    w = torch.eye(d, dtype=dtype, device="cuda").requires_grad_(True)
    t = torch.randint(0, d, (rows,), generator=g).cuda()
    t[::4] = -100
    dl = torch.randn(rows, generator=g).cuda()
    (got,) = torch.autograd.grad(F.linear_logprobs(h, w, t, recompute=recompute), h, dl)
    lp = torch.log_softmax(h.detach().double(), -1)
    p = lp.exp()
    c = torch.where(t == -100, 0.0, dl.double())[:, None]
    want = -c * p
    want.scatter_add_(1, t.clamp(min=0)[:, None], c)
    step = STEP[dtype]
    # the exponent's and the sum's roundings in FP32, as for logits in memory; then to the type, the exponential before it where it was held
    err = c.abs() * p * U * (4 * -lp + 60) + step * want.abs() + LEAST[dtype]
    if not recompute:
        err = err + step * (1 + step) * c.abs() * p
    if dtype == torch.float16:      # the smallest step of the scaled gradient
        err = err + float(c.abs().max()) * 2.0 ** -39
    err = err + 4 * U * want.abs()
    off = (got.double() - want).abs()
    assert bool((off <= err).all()), float((off / err).max())
    assert bool((got[t == -100] == 0).all())
    assert math.isfinite(float(off.max()))

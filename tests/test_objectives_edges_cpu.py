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

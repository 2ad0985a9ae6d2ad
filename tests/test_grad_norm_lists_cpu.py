"""Lists of gradients that the optimizer and the trainer take beyond those of the clipping kernels: sparse ones, ones that share memory."""
import math

import pytest
import torch

from nexus_b200.fused import ops as F
from nexus_b200.optim import AdamW
from nexus_b200.train import TrainerBuilder


class Bag(torch.nn.Module):
    def __init__(self, sparse):
        super().__init__()
        g = torch.Generator().manual_seed(0)
        self.emb = torch.nn.Embedding(12, 6, sparse=sparse)
        self.out = torch.nn.Linear(6, 3)
        with torch.no_grad():
            for p in self.parameters():
                p.copy_(torch.randn(p.shape, generator=g))

    def forward(self, tokens):
        return self.out(self.emb(tokens).sum(1))


def batch():
    g = torch.Generator().manual_seed(1)
    return torch.randint(0, 12, (5, 4), generator=g), torch.randint(0, 3, (5,), generator=g)


def test_adamw_with_sparse_gradients():
    after = []
    for sparse in (True, False):
        m = Bag(sparse)
        opt = AdamW(m.parameters(), lr=0.1)
        for _ in range(2):
            opt.zero_grad()
            x, y = batch()
            torch.nn.functional.cross_entropy(m(x), y).backward()
            assert m.emb.weight.grad.is_sparse == sparse
            assert F.grad_square_sum([p.grad for p in m.parameters()]) == pytest.approx(
                sum(float(p.grad.double().to_dense().pow(2).sum()) for p in m.parameters()), rel=1e-12)
            opt.step()
        after.append([p.detach().clone() for p in m.parameters()])
    for a, b in zip(*after):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("clip", [0.0, 0.05, 1e6])
def test_trainer_with_sparse_gradients(clip):
    after = []
    for sparse in (True, False):
        tr = TrainerBuilder(Bag(sparse)).adamw(lr=0.1).gradient_clip_norm(clip).build()
        tr.fit([batch()], epochs=2)
        assert tr.global_step == 2 and tr.skipped_steps == 0
        after.append([p.detach().clone() for p in tr.model.parameters()])
    for a, b in zip(*after):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-7)


def test_trainer_with_gradients_that_share_memory():
    """Views of one buffer that overlap, and one tensor that is the gradient of two parameters: each parameter's is counted and scaled in turn."""
    def grads():
        flat = torch.arange(1.0, 9.0)
        both = torch.full((3,), 2.0)
        return [flat[:5], flat[3:], both, both]

    want = grads()
    sq = sum(float(g.double().pow(2).sum()) for g in want)
    coef = 0.5 / (math.sqrt(sq) + 1e-6)
    for g in want:
        g.mul_(coef)
    model = torch.nn.Module()
    model.ps = torch.nn.ParameterList([torch.nn.Parameter(torch.zeros(n)) for n in (5, 5, 3, 3)])
    tr = TrainerBuilder(model).sgd(lr=1.0).gradient_clip_norm(0.5).build()
    for p, g in zip(model.ps, grads()):
        p.grad = g
    tr._apply_step(1)
    for p, g in zip(model.ps, want):
        assert torch.equal(p.detach(), -g)


def test_clipping_still_refuses_them():
    a = torch.ones(6)
    for gs in ([a, torch.ones(3).to_sparse()], [a[:4], a[2:]]):
        with pytest.raises(ValueError):
            F.clip_grad_norm_(gs, 1.0)

"""What autograd is told of the codebook and clipping operators on the GPU: forward
mode is refused, and what an operator writes in place is a new version."""
import pytest
import torch
from torch.autograd import forward_ad

from cuda_rasterizer import clipping, codebook

pytestmark = pytest.mark.gpu


def test_lookup_refuses_forward_mode():
    table = torch.ones(4, 3, device="cuda")
    index = torch.tensor([0, 2, -1], device="cuda")
    order = codebook.sort_by_code(index, 4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(table, torch.ones_like(table))
        for o in (None, order):
            with pytest.raises(NotImplementedError, match="jvp"):
                codebook.lookup(dual, index, order=o)
        assert forward_ad.unpack_dual(codebook.lookup(table, index)).tangent is None


def test_a_kept_graph_refuses_stale_values():
    """A gradient penalty whose gradient is clipped, a model's graph kept over an update, a destination that is saved."""
    x = torch.randn(300, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(x.pow(3).sum(), x, create_graph=True)
    penalty = g.square().sum()
    clipping.clip_grads([g], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        penalty.backward()
    p = torch.randn(300, device="cuda")
    kept = (torch.ones(300, device="cuda", requires_grad=True) * p).sum()
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    clipping.adam_step_clipped(p, torch.ones_like(p), m, v, [(300, 0.1)], 1, 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    rows, index = torch.randn(50, 8, device="cuda"), torch.randint(0, 6, (50,), device="cuda")
    out = torch.zeros(6, 8, device="cuda")
    kept = (torch.ones(6, 8, device="cuda", requires_grad=True) * out).sum()
    codebook.gradient_sorted(rows, codebook.sort_by_code(index, 6), out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    # what is read only stays as it was
    w = torch.randn(300, device="cuda", requires_grad=True)
    grads = torch.randn(300, device="cuda")
    loss = (w * grads).sum()
    clipping.clip_grads([grads], 1e-3, out=[torch.empty_like(grads)])
    clipping.grad_norm([grads])
    clipping.adam_step_clipped(p, grads, m, v, [(300, 0.1)], 2, 1.0)
    loss.backward()
    assert torch.equal(w.grad, grads)

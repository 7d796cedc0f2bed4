"""What autograd is told of the codebook and clipping operators, without a GPU:
the host side of the calls, with the kernel call replaced by torch."""
import pytest
import torch
from torch.autograd import forward_ad

from cuda_rasterizer import codebook


@pytest.mark.parametrize("mode", ["plain", "no_grad", "leaf"])
def test_lookup_refuses_forward_mode(monkeypatch, mode):
    """A dual table has no requires_grad, and rows without a tangent would be a derivative of zero."""
    monkeypatch.setattr(codebook, "_lookup", lambda table, index, scale, dtype: table.detach()[index] * scale)
    table = torch.ones(4, 3, requires_grad=mode == "leaf")
    index = torch.tensor([0, 2])
    with forward_ad.dual_level(), torch.set_grad_enabled(mode != "no_grad"):
        with pytest.raises(NotImplementedError, match="jvp"):
            codebook.lookup(forward_ad.make_dual(table, torch.ones(4, 3)), index, 2.0)
        assert torch.equal(codebook.lookup(table, index, 2.0), torch.full((2, 3), 2.0))  # not a dual

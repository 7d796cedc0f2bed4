"""What autograd is told of the codebook and clipping operators, without a GPU:
the host side of the calls, with the kernel call replaced by torch."""
import contextlib
from array import array

import pytest
import torch
from torch.autograd import forward_ad

from cuda_rasterizer import _native, clipping, codebook


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


class _Library:
    """Every entry point does nothing and succeeds."""

    def __getattr__(self, name):
        return lambda *a: 0


@pytest.fixture
def no_kernels(monkeypatch):
    monkeypatch.setattr(_native, "lib", lambda: _Library())
    monkeypatch.setattr(_native, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_native, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(_native, "_as_cuda_f32", lambda t, name: t)
    monkeypatch.setattr(clipping, "_workspace", lambda n, dev: torch.empty(256, dtype=torch.uint8))
    monkeypatch.setattr(clipping, "_list", lambda tensors, name: (
        array("Q", [t.data_ptr() for t in tensors]), array("q", [t.numel() for t in tensors]),
        array("i", [0] * len(tensors)), tensors[0].device, True))
    monkeypatch.setattr(codebook, "_size", lambda name, *args: 256)
    monkeypatch.setattr(codebook, "_matrix", lambda t, name: (t, t.shape[1]))


def _saved(*tensors):
    """A graph that has saved each of the tensors."""
    return [(torch.ones_like(t).requires_grad_() * t).sum() for t in tensors]


def _stale(graphs):
    """Which of the graphs refuse their backward, since what they saved has changed."""
    got = []
    for g in graphs:
        try:
            g.backward()
            got.append(False)
        except RuntimeError as e:
            assert "modified by an inplace operation" in str(e)
            got.append(True)
    return got


def test_tensors_written_in_place_are_new_versions(no_kernels):
    a, b, c, d = (torch.ones(6) for _ in range(4))
    graphs = _saved(a, b)
    clipping.clip_grads([a, b], 1.0)
    assert _stale(graphs) == [True, True]
    graphs = _saved(a, b, c, d)
    clipping.clip_grads([a, b], 1.0, out=[c, b])
    assert _stale(graphs) == [False, True, True, False]
    p = torch.nn.Parameter(torch.ones(6))
    p.grad = a
    graphs = _saved(a)
    clipping.clip_grad_norm_([p], 1.0)
    assert _stale(graphs) == [True]
    graphs = _saved(a, b, c, d)
    clipping.adam_step_clipped(a, b, c, d, [(6, 1e-3)], 1, 1.0)
    assert _stale(graphs) == [True, False, True, True]
    graphs = _saved(a, b)
    clipping.grad_norm([a, b])
    assert _stale(graphs) == [False, False]


def test_a_destination_of_the_codebook_is_a_new_version(no_kernels):
    table, rows = torch.ones(3, 2), torch.ones(5, 2)
    order = codebook.SortedCodes(*[torch.zeros(n, dtype=torch.int32) for n in (5, 5, 4)])
    graphs = _saved(table, rows)
    codebook.gradient_sorted(rows, order, out=table)
    assert _stale(graphs) == [True, False]


def test_inference_tensors_have_no_versions(no_kernels):
    with torch.inference_mode():
        a, b = torch.ones(6), torch.ones(6)
        clipping.clip_grads([a], 1.0)
        clipping.clip_grads([a], 1.0, out=[b])

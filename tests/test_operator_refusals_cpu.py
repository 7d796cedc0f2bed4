"""Calls of the codebook and clipping operators that are refused before a kernel runs,
without a GPU: the host side of the calls, with the kernel call replaced by nothing."""
import contextlib
from array import array

import pytest
import torch

from cuda_rasterizer import _native, clipping, codebook


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
    monkeypatch.setattr(codebook, "_size", lambda name, *args: 256)
    monkeypatch.setattr(codebook, "_matrix", lambda t, name: (t, t.stride(0) if t.shape[0] > 1 else t.shape[1]))


def _order(n, codes):
    return codebook.SortedCodes(*[torch.zeros(k, dtype=torch.int32) for k in (n, n, codes + 1)])


def test_a_destination_on_the_rows_is_refused(no_kernels):
    """The sums of one code would be written over rows that another has still to read."""
    wide = torch.zeros(20, 24)
    for rows, out in ((wide[:8, :8], wide[:8, :8]), (wide[:8, :8], wide[7:15, :8]), (wide[:8, :8], wide[3:9, 4:12]),
                      (wide[:8, :8], wide[4:5, 7:15]), (wide[4:5, 4:12], wide[:9, :8]),
                      (wide[:8, 8:16], wide.view(40, 12)[5:9, :8])):
        with pytest.raises(RuntimeError, match="share memory"):
            codebook.gradient_sorted(rows, _order(len(rows), len(out)), out=out)
    for rows, out in ((wide[:8, :8], wide[8:16, :8]), (wide[:8, :8], wide[:8, 8:16]), (wide[:8, 8:16], wide[:8, :8]),
                      (wide[:8, :8], wide[4:5, 8:16]), (wide[4:5, 8:16], wide[:9, :8]), (wide[:0, :8], wide[:9, :8]),
                      (wide[:8, :8], wide[:0, :8])):
        assert codebook.gradient_sorted(rows, _order(len(rows), len(out)), out=out) is out


def test_a_destination_on_the_order_is_refused(no_kernels):
    memory = torch.zeros(64)
    ints = memory.view(torch.int32)
    order = codebook.SortedCodes(ints[:8], ints[8:16], ints[16:21])
    for at in (0, 12, 20):
        with pytest.raises(RuntimeError, match="share memory"):
            codebook.gradient_sorted(torch.zeros(8, 2), order, out=memory[at:at + 8].view(4, 2))
    codebook.gradient_sorted(torch.zeros(8, 2), order, out=memory[24:32].view(4, 2))


def test_adam_buffers_that_overlap_are_refused(no_kernels):
    memory = torch.zeros(64)
    p, g, m, v = memory[:16], memory[16:32], memory[32:48], memory[48:]
    clipping.adam_step_clipped(p, g, m, v, [(16, 1e-3)], 1, 1.0)
    clipping.adam_step_clipped(v, m, g, p, [(16, 1e-3)], 1, 1.0)
    for bad in ((p, p, m, v), (p, g, m, m), (p, g, memory[31:47], v), (p, memory[1:17], m, v), (memory[47:63], g, m, v)):
        with pytest.raises(RuntimeError, match="share memory"):
            clipping.adam_step_clipped(*bad, [(16, 1e-3)], 1, 1.0)
    e = memory[:0]
    clipping.adam_step_clipped(e, e, e, e, [(0, 1e-3)], 1, 1.0)


def test_lookup_with_something_else_as_order():
    table, index = torch.ones(4, 3), torch.zeros(5, dtype=torch.int64)
    for bad in (tuple(_order(5, 4)), torch.zeros(5, dtype=torch.int32), codebook.SortedCodes(None, None, None)):
        with pytest.raises(TypeError, match="order"):
            codebook.lookup(table, index, order=bad)
    for bad in ([[1.0]], None):
        with pytest.raises(TypeError):
            codebook.lookup(bad, index, order=_order(5, 4))
        with pytest.raises(TypeError):
            codebook.lookup(table, bad, order=_order(5, 4))


def test_negated_views(monkeypatch):
    """The imaginary part of a conjugate is a view whose memory holds the values negated."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    z = torch.complex(torch.ones(4, 1), torch.full((4, 1), 2.0)).conj().imag
    assert z.is_neg()
    t, stride = codebook._matrix(z, "table")
    assert not t.is_neg() and torch.equal(t, torch.full((4, 1), -2.0)) and stride == 1
    with pytest.raises(RuntimeError, match="out"):
        codebook._check_out(z, 4, 1, z.device)
    plain = torch.ones(4, 6)[:, :3]
    assert codebook._matrix(plain, "table")[0] is plain


def test_negated_views_in_lists(no_kernels, monkeypatch):
    """In place the values are scaled as they lie; into others the sign would be lost."""
    monkeypatch.setattr(clipping, "_list", lambda tensors, name: (
        array("Q", [t.data_ptr() for t in tensors]), array("q", [t.numel() for t in tensors]),
        array("i", [0] * len(tensors)), tensors[0].device, True))
    z = torch.complex(torch.ones(1), torch.ones(1)).conj().imag
    assert z.is_neg() and z.is_contiguous()
    clipping.clip_grads([torch.ones(1), z], 1.0)
    for grads, out in (([z], [torch.ones(1)]), ([torch.ones(1)], [z])):
        with pytest.raises(RuntimeError, match="negated"):
            clipping.clip_grads(grads, 1.0, out=out)

"""The codebook and clipping operators without a GPU: arguments that the C ABI
and the Python modules refuse before the device is used, and workspace sizes."""
import ctypes
import math

import pytest
import torch

from cuda_rasterizer import _native, clipping, codebook

ARG, WORKSPACE = 1, 2
D = ctypes.c_void_p(256)  # a non-null, aligned pointer that a refused call never reads
BIG = 2 ** 31


def _lookup(**kw):
    a = dict(n=4, codes=8, cols=16, index=D, bits=32, table=D, ttype=0, tstride=16, scale=1.0, rows=D, rtype=0,
             rstride=16)
    a.update(kw)
    return _native.lib().sarr_codebook_lookup(*a.values(), None)


@pytest.mark.parametrize("kw", [
    dict(n=-1), dict(n=BIG), dict(codes=-1), dict(codes=BIG), dict(cols=-1), dict(cols=2 ** 23), dict(bits=16),
    dict(ttype=3), dict(ttype=-1), dict(rtype=1), dict(ttype=1, rtype=2), dict(tstride=15), dict(rstride=15),
    dict(index=None), dict(rows=None), dict(table=None), dict(index=ctypes.c_void_p(258)),
    dict(bits=64, index=ctypes.c_void_p(260)), dict(table=ctypes.c_void_p(258)), dict(rows=ctypes.c_void_p(257))])
def test_lookup_refusals(kw):
    assert _lookup(**kw) == ARG


def test_lookup_of_nothing():
    assert _lookup(n=0, index=None, rows=None) == 0
    assert _lookup(cols=0, tstride=0, rstride=0) == 0


def _sort(**kw):
    a = dict(n=4, codes=8, index=D, bits=32, order=D, sorted=D, offsets=D, ws=D, ws_bytes=1 << 24)
    a.update(kw)
    return _native.lib().sarr_codebook_sort(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), ARG), (dict(n=BIG), ARG), (dict(codes=-1), ARG), (dict(codes=BIG), ARG), (dict(bits=8), ARG),
    (dict(index=None), ARG), (dict(order=None), ARG), (dict(sorted=None), ARG), (dict(offsets=None), ARG),
    (dict(order=ctypes.c_void_p(258)), ARG), (dict(n=20000, ws=None), WORKSPACE), (dict(n=20000, ws_bytes=16), WORKSPACE),
    (dict(n=20000, ws=ctypes.c_void_p(264)), WORKSPACE)])
def test_sort_refusals(kw, status):
    assert _sort(**kw) == status


def _grad(**kw):
    a = dict(n=4, codes=8, cols=16, rows=D, rtype=0, rstride=16, order=D, sorted=D, offsets=D, scale=1.0, table=D,
             ttype=0, tstride=16, ws=D, ws_bytes=1 << 24)
    a.update(kw)
    return _native.lib().sarr_codebook_grad(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), ARG), (dict(codes=-1), ARG), (dict(codes=BIG), ARG), (dict(cols=-1), ARG), (dict(rtype=5), ARG),
    (dict(rtype=1, ttype=2), ARG), (dict(rstride=8), ARG), (dict(tstride=8), ARG), (dict(rows=None), ARG),
    (dict(order=None), ARG), (dict(sorted=None), ARG), (dict(offsets=None), ARG), (dict(table=None), ARG),
    (dict(rows=ctypes.c_void_p(258)), ARG), (dict(ws=None), WORKSPACE), (dict(ws_bytes=0), WORKSPACE)])
def test_gradient_refusals(kw, status):
    assert _grad(**kw) == status


def _gradient(**kw):
    a = dict(n=4, codes=8, cols=16, rows=D, rtype=0, rstride=16, index=D, bits=64, scale=1.0, table=D, ttype=0, tstride=16,
             ws=D, ws_bytes=1 << 24)
    a.update(kw)
    return _native.lib().sarr_codebook_gradient(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), ARG), (dict(n=BIG), ARG), (dict(codes=-1), ARG), (dict(cols=2 ** 22), ARG), (dict(bits=16), ARG),
    (dict(index=None), ARG), (dict(index=ctypes.c_void_p(260)), ARG), (dict(rows=None), ARG), (dict(table=None), ARG),
    (dict(rtype=2, ttype=1), ARG), (dict(rstride=15), ARG), (dict(tstride=0), ARG), (dict(ws=None), WORKSPACE),
    (dict(ws_bytes=64), WORKSPACE), (dict(ws=ctypes.c_void_p(384 + 8)), WORKSPACE)])
def test_gradient_in_one_call_refusals(kw, status):
    assert _gradient(**kw) == status


def test_gradient_of_no_codes():
    assert _grad(codes=0, offsets=None, table=None) == 0
    assert _gradient(codes=0, table=None) == 0
    assert _gradient(cols=0, rstride=0, tstride=0) == 0


def _clip(grads=(4096, 8192), counts=(16, 16), types=(0, 0), outs=(4096, 8192), otypes=(0, 0), kind=0, max_norm=1.0,
          ws=D, ws_bytes=1 << 20, n=None):
    k = len(grads)
    arr = lambda t, x: (t * k)(*x) if x is not None else None  # noqa: E731
    return _native.lib().sarr_clip_grads(
        k if n is None else n, arr(ctypes.c_uint64, grads), arr(ctypes.c_int64, counts), arr(ctypes.c_int32, types),
        arr(ctypes.c_uint64, outs), arr(ctypes.c_int32, otypes), kind, max_norm, D, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), ARG), (dict(counts=(16, -1)), ARG), (dict(types=(0, 7)), ARG), (dict(kind=2), ARG),
    (dict(max_norm=-1.0), ARG), (dict(max_norm=math.nan), ARG), (dict(grads=(4096, 0)), ARG), (dict(outs=(4096, 0)), ARG),
    (dict(outs=None), ARG), (dict(grads=(4096, 8193)), ARG), (dict(otypes=(0, 1)), ARG),
    (dict(types=(1, 1), otypes=(0, 1)), ARG),               # in place into another type
    (dict(ws=None), WORKSPACE), (dict(ws_bytes=8), WORKSPACE), (dict(ws=ctypes.c_void_p(264)), WORKSPACE),
    (dict(grads=(4096, 4096), outs=(4096, 4096)), ARG),     # the same tensor twice
    (dict(grads=(4096, 4128), outs=(4096, 4128)), ARG),     # two that overlap
    (dict(outs=(16384, 16416)), ARG),                       # overlapping destinations
    (dict(outs=(8192, 16384)), ARG),                        # a destination on another tensor's gradient
    (dict(outs=(4100, 16384)), ARG),                        # a destination shifted within its own gradient
    (dict(outs=(8160, 16384)), ARG)])
def test_clip_refusals(kw, status):
    assert _clip(**kw) == status


def _adam(begin=(0, 16), end=(16, 32), first=(0, 16), lr=(1e-3, 1e-3), betas=(0.9, 0.999), step=1, max_norm=1.0, n=None,
          arrays=(D, D, D, D), ws=D, ws_bytes=1 << 20):
    k = len(begin)
    i64 = lambda x: (ctypes.c_int64 * k)(*x)  # noqa: E731
    return _native.lib().sarr_adam_step_clipped(
        k if n is None else n, i64(begin), i64(end), i64(first), (ctypes.c_double * k)(*lr), *arrays, *betas, 1e-8, step,
        max_norm, D, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), ARG), (dict(n=65), ARG), (dict(step=0), ARG), (dict(max_norm=-0.5), ARG), (dict(betas=(1.0, 0.9)), ARG),
    (dict(betas=(0.9, -0.1)), ARG), (dict(begin=(0, -1)), ARG), (dict(end=(16, 15)), ARG), (dict(first=(0, -4)), ARG),
    (dict(begin=(0, 8)), ARG), (dict(arrays=(D, None, D, D)), ARG), (dict(ws=None), WORKSPACE), (dict(ws_bytes=0), WORKSPACE)])
def test_adam_refusals(kw, status):
    assert _adam(**kw) == status


def test_workspace_sizes_grow():
    out = ctypes.c_size_t()
    L = _native.lib()

    def size(fn, *a):
        assert fn(*a, ctypes.byref(out)) == 0
        return out.value

    # two digits need one buffer of keys and places beside the outputs
    assert size(L.sarr_codebook_sort_workspace_size, 1_000_000, 65536) >= 8_000_000
    assert size(L.sarr_codebook_grad_workspace_size, 1_000_000, 16) > size(L.sarr_codebook_grad_workspace_size, 1000, 16)
    assert size(L.sarr_grad_norm_workspace_size, 2000) > size(L.sarr_grad_norm_workspace_size, 1)
    assert L.sarr_codebook_sort_workspace_size(-1, 4, ctypes.byref(out)) == ARG
    assert L.sarr_codebook_grad_workspace_size(4, -1, ctypes.byref(out)) == ARG
    assert L.sarr_grad_norm_workspace_size(-1, ctypes.byref(out)) == ARG


def test_python_refuses_cpu_tensors_and_bad_arguments():
    table, index = torch.zeros(8, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        codebook.lookup(table, index)
    with pytest.raises(RuntimeError, match="CUDA"):
        codebook.sort_by_code(index, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        codebook.gradient(torch.zeros(3, 4), index, 8)
    with pytest.raises(RuntimeError, match="rows"):
        codebook.gradient(torch.zeros(2, 4), index, 8)
    with pytest.raises(TypeError):
        codebook.lookup([[1.0]], index)
    with pytest.raises(RuntimeError, match="CUDA"):
        clipping.grad_norm([table])
    with pytest.raises(RuntimeError, match="CUDA"):
        clipping.clip_grads([table], 1.0)
    with pytest.raises(RuntimeError, match="norm_type"):
        clipping.grad_norm([table], norm_type=1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        clipping.clip_grads([table], -1.0)
    with pytest.raises(RuntimeError, match="destinations"):
        clipping.clip_grads([table], 1.0, out=[])
    with pytest.raises(RuntimeError, match="float32"):
        clipping.grad_norm([table.double()])
    with pytest.raises(TypeError):
        clipping.grad_norm([1.0])
    with pytest.raises(RuntimeError, match="CUDA"):
        clipping.adam_step_clipped(*[torch.zeros(4)] * 4, [(4, 1e-3)], 1, 1.0)
    assert clipping.grad_norm([]).item() == 0.0
    assert clipping.clip_grad_norm_([torch.zeros(3, requires_grad=True)], 1.0, foreach=True).item() == 0.0


def test_clip_grad_norm_takes_torchs_arguments():
    import inspect
    mine = inspect.signature(clipping.clip_grad_norm_).parameters
    assert list(inspect.signature(torch.nn.utils.clip_grad_norm_).parameters) == list(mine)

"""Codebook rows: Gaussians whose parameter rows (the SH coefficients, 16 of a
Gaussian's 20 trained floats) come from a table that they share, by index.

    rows = lookup(table, index, scale)        # rows[i] = scale * table[index[i]]

`lookup` is differentiable with respect to the table. Its gradient sums the
rows' gradients of every code in the order of the Gaussians: `gradient` sorts
the index and sums, `sort_by_code` and `gradient_sorted` are its two halves for
a caller whose index stays the same over many steps (`lookup` takes the order
too; ViewParallelTrainer with `sh_index` keeps one). A Gaussian whose index is outside [0, codes) has no code: its row
is zeros and its gradient reaches no code.

Tables and rows are float32, bfloat16 or float16 CUDA tensors (rows in the
table's type or float32); indexes int32 or int64. Products and sums are formed
in 32 bits and rounded once. Results are bitwise reproducible: a gradient's bits
depend on the sizes, codes, types and strides and on the rows' and the table's
offsets from a 16-byte boundary. No counterpart in the reference, which keeps all
SH coefficients of every Gaussian.
"""
import ctypes
import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _native

__all__ = ["SortedCodes", "lookup", "sort_by_code", "gradient", "gradient_sorted"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INDEX_BITS = {torch.int32: 32, torch.int64: 64}


class SortedCodes(NamedTuple):
    """The Gaussians in the stable order of their codes (sarr_codebook_sort)."""
    order: torch.Tensor    # int32 [n]: the Gaussian at each place, those without a code last
    codes: torch.Tensor    # int32 [n]: the code at each place, `codes` for none
    offsets: torch.Tensor  # int32 [codes + 1]: the first place of each code


def _matrix(t, name):
    """(tensor, row stride) of a [rows, cols] matrix of a supported type."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != 2:
        raise RuntimeError(f"{name} must be a matrix, got shape {tuple(t.shape)}")
    t = t.resolve_neg()
    rows, cols = t.shape
    stride, step = t.stride()
    if (cols > 1 and step != 1) or (rows > 1 and stride < cols):
        t, stride = t.contiguous(), cols
    return t, stride if rows > 1 else cols


def _index(index, name="index"):
    if not isinstance(index, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not index.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if index.dtype not in _INDEX_BITS:
        raise RuntimeError(f"{name} must be int32 or int64, got {index.dtype}")
    return index if index.is_contiguous() else index.contiguous()


def _same_device(dev, name, t):
    if t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, expected {dev}")


def _out_type(dtype, allowed, what):
    if dtype not in allowed:
        raise RuntimeError(f"{what} must be one of {[str(d) for d in allowed]}, got {dtype}")
    return dtype


def _check_out(out, rows, cols, dev, name="out"):
    t, stride = _matrix(out, name)
    if t is not out or t.shape != (rows, cols):
        raise RuntimeError(f"{name} must be a matrix of {rows} x {cols} with contiguous rows")
    _same_device(dev, name, t)
    return stride


def _meet(a, a_stride, b, b_stride):
    """Whether a matrix with contiguous rows (stride in elements) shares memory with
    another, or with a vector."""
    at = b.data_ptr() - a.data_ptr()
    n, cols = a.shape
    a_size = a.element_size()
    if at >= ((n - 1) * a_stride + cols) * a_size:  # the usual answers
        return False
    m, b_cols = b.shape if b.dim() == 2 else (1, b.numel())
    b_size = b.element_size()
    if -at >= ((m - 1) * b_stride + b_cols) * b_size or not (n and cols and m and b_cols):
        return False
    # side by side in rows of one pitch (a single row has that of the other)
    pitch = b_stride * b_size if n == 1 else a_stride * a_size
    if m > 1 and b_stride * b_size != pitch:
        return True
    if n == 1 and m == 1:
        return True
    return at % pitch < cols * a_size or at % pitch + b_cols * b_size > pitch


@functools.lru_cache(maxsize=1024)
def _size(name, *args):
    """Workspace bytes for these sizes."""
    out = ctypes.c_size_t()
    _native._check(getattr(_native.lib(), name)(*args, ctypes.byref(out)), name)
    return out.value


def _lookup(table, index, scale, dtype, out=None):
    table, stride = _matrix(table, "table")
    index = _index(index)
    dev = table.device
    _same_device(dev, "index", index)
    dtype = _out_type(dtype or table.dtype, (table.dtype, torch.float32), "dtype")
    codes, cols = table.shape
    n = index.numel()
    rows_stride = cols
    if out is not None:
        rows_stride = _check_out(out, n, cols, dev)
        if out.dtype != dtype:
            raise RuntimeError(f"out must be {dtype}, got {out.dtype}")
    with _native._on(dev):
        rows = torch.empty((*index.shape, cols), dtype=dtype, device=dev) if out is None else out
        _native._check(_native.lib().sarr_codebook_lookup(
            n, codes, cols, index.data_ptr(), _INDEX_BITS[index.dtype], table.data_ptr(),
            _TYPES[table.dtype], stride, float(scale), rows.data_ptr(), _TYPES[dtype], rows_stride,
            _native._raw_stream(dev)), "sarr_codebook_lookup")
    if out is not None:
        increment_version(out)
    return rows


def sort_by_code(index: torch.Tensor, codes: int) -> SortedCodes:
    """The stable order of the Gaussians by code (`index` flattened)."""
    index = _index(index)
    dev, n, codes = index.device, index.numel(), int(codes)
    size = _size("sarr_codebook_sort_workspace_size", n, codes)
    with _native._on(dev):
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        order = torch.empty(n, dtype=torch.int32, device=dev)
        sorted_codes = torch.empty(n, dtype=torch.int32, device=dev)
        offsets = torch.empty(codes + 1, dtype=torch.int32, device=dev)
        _native._check(_native.lib().sarr_codebook_sort(
            n, codes, index.data_ptr(), _INDEX_BITS[index.dtype], order.data_ptr(),
            sorted_codes.data_ptr(), offsets.data_ptr(), ws.data_ptr() if size else None, size,
            _native._raw_stream(dev)), "sarr_codebook_sort")
    return SortedCodes(order, sorted_codes, offsets)


def _gradient_type(rows, dtype):
    allowed = tuple(_TYPES) if rows.dtype == torch.float32 else (rows.dtype, torch.float32)
    return _out_type(dtype or rows.dtype, allowed, "dtype")


def gradient_sorted(grad_rows: torch.Tensor, sorted_codes: SortedCodes, scale: float = 1.0,
                    dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The table's gradient [codes, cols] from the rows' gradients [n, cols] and
    the order that sort_by_code gave for their index. `dtype`: the result's type
    (the rows' type by default; float32, or any of the three for float32 rows);
    `out`: a matrix to write it into (its rows may be strided; it shares no memory
    with the other arguments)."""
    rows, rows_stride = _matrix(grad_rows, "grad_rows")
    n, cols = rows.shape
    order, places, offsets = sorted_codes
    dev = rows.device
    for name, t in (("order", order), ("codes", places), ("offsets", offsets)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise RuntimeError(f"sorted_codes.{name} must be a contiguous int32 vector")
        _same_device(dev, name, t)
    if order.numel() != n or places.numel() != n or offsets.numel() < 1:
        raise RuntimeError(f"sorted_codes is of {order.numel()} Gaussians, grad_rows of {n}")
    codes = offsets.numel() - 1
    stride = cols
    if out is not None:
        stride = _check_out(out, codes, cols, dev)
        if dtype is not None and dtype != out.dtype:
            raise RuntimeError(f"out is {out.dtype}, dtype {dtype}")
        if _meet(out, stride, rows, rows_stride) or any([
                _meet(out, stride, t, 0) for t in (order, places, offsets)]):
            raise RuntimeError("out must not share memory with grad_rows or sorted_codes")
        dtype = out.dtype
    dtype = _gradient_type(rows, dtype)
    size = _size("sarr_codebook_grad_workspace_size", n, cols)
    with _native._on(dev):
        table = torch.empty((codes, cols), dtype=dtype, device=dev) if out is None else out
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _native._check(_native.lib().sarr_codebook_grad(
            n, codes, cols, rows.data_ptr(), _TYPES[rows.dtype], rows_stride, order.data_ptr(),
            places.data_ptr(), offsets.data_ptr(), float(scale), table.data_ptr(), _TYPES[dtype], stride,
            ws.data_ptr(), size, _native._raw_stream(dev)), "sarr_codebook_grad")
    if out is not None:
        increment_version(out)
    return table


def gradient(grad_rows: torch.Tensor, index: torch.Tensor, codes: int, scale: float = 1.0,
             dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The table's gradient [codes, cols] of lookup(table, index, scale) from the
    rows' gradients [*index.shape, cols] (sort_by_code and gradient_sorted in one
    call)."""
    if isinstance(grad_rows, torch.Tensor) and isinstance(index, torch.Tensor) and grad_rows.dim() not in (0, 2):
        if grad_rows.shape[:-1] != index.shape:
            raise RuntimeError(f"grad_rows is {tuple(grad_rows.shape)}, index {tuple(index.shape)}")
        grad_rows = grad_rows.reshape(index.numel(), grad_rows.shape[-1])
    rows, rows_stride = _matrix(grad_rows, "grad_rows")
    index = _index(index)
    dev, codes = rows.device, int(codes)
    _same_device(dev, "index", index)
    n, cols = rows.shape
    if n != index.numel():
        raise RuntimeError(f"grad_rows has {n} rows, index {index.numel()} elements")
    dtype = _gradient_type(rows, dtype)
    size = _size("sarr_codebook_gradient_workspace_size", n, codes, cols)
    with _native._on(dev):
        table = torch.empty((codes, cols), dtype=dtype, device=dev)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _native._check(_native.lib().sarr_codebook_gradient(
            n, codes, cols, rows.data_ptr(), _TYPES[rows.dtype], rows_stride, index.data_ptr(),
            _INDEX_BITS[index.dtype], float(scale), table.data_ptr(), _TYPES[dtype], cols, ws.data_ptr(), size,
            _native._raw_stream(dev)), "sarr_codebook_gradient")
    return table


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, dtype, order):
        rows = _lookup(table.detach(), index, scale, dtype)
        ctx.save_for_backward(index, *(order or ()))
        ctx.scale, ctx.codes, ctx.dtype = scale, table.shape[0], table.dtype
        return rows

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        index, *order = ctx.saved_tensors
        if order:
            grad = grad.reshape(index.numel(), grad.shape[-1])
            grad_table = gradient_sorted(grad, SortedCodes(*order), ctx.scale, ctx.dtype)
        else:
            grad_table = gradient(grad, index, ctx.codes, ctx.scale, ctx.dtype)
        return grad_table, None, None, None, None


def lookup(table: torch.Tensor, index: torch.Tensor, scale: float = 1.0,
           dtype: Optional[torch.dtype] = None, order: Optional[SortedCodes] = None) -> torch.Tensor:
    """rows[i] = scale * table[index[i]] ([*index.shape, cols]; zeros where
    index[i] is outside [0, codes)), in `dtype` (the table's type by default, or
    float32), with its gradient with respect to the table. `order`: what
    sort_by_code gave for this index, where the caller keeps it; without it the
    gradient sorts the index. Forward-mode differentiation is refused."""
    if order is not None:
        for t, name in ((table, "table"), (index, "index")):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
        if not isinstance(order, SortedCodes) or not all(isinstance(t, torch.Tensor) for t in order):
            raise TypeError("order must be what sort_by_code gave")
        if table.dim() == 2 and (order.order.numel() != index.numel() or order.offsets.numel() != table.shape[0] + 1):
            raise RuntimeError(f"order is of {order.order.numel()} Gaussians and {order.offsets.numel() - 1} codes, "
                               f"the index of {index.numel()} and the table of {table.shape[0]}")
    # a dual table need not require a gradient; apply refuses it
    if isinstance(table, torch.Tensor) and (table.requires_grad and torch.is_grad_enabled()
                                            or forward_ad.unpack_dual(table).tangent is not None):
        return _Lookup.apply(table, index, scale, dtype, order)
    return _lookup(table, index, scale, dtype)

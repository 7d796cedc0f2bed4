"""Global gradient norm over many tensors, clipping by it, and the Adam update
with clipped gradients (one pass for the norm, one for the rest).

    norm = clip_grad_norm_(model_parameters, max_norm)       # in place, on .grad
    norm = clip_grads(grads, max_norm, out=destinations)     # grads untouched
    norm = adam_step_clipped(param, grad, exp_avg, exp_avg_sq, segments, step, max_norm)

with torch.nn.utils.clip_grad_norm_'s rule: every gradient is multiplied by
min(1, max_norm / (norm + 1e-6)). Gradients are dense float32, bfloat16 or
float16 CUDA tensors of one device, types mixed as they come; the norm is summed
in 64 bits and returned as a float32 scalar on the device (no synchronisation).
Results are bitwise reproducible for tensors at the same offsets from a 16-byte
boundary. A tensor written in place is a new version for
autograd, as with torch's in-place operations: a graph that saved it refuses its
backward. The reference trains without clipping.
"""
import ctypes
import functools
import math
from array import array
from operator import attrgetter
from typing import Iterable, Optional, Sequence

import torch
from torch.autograd.graph import increment_version

from . import _native

__all__ = ["grad_norm", "clip_grads", "clip_grad_norm_", "adam_step_clipped"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NORMS = {2.0: 0, math.inf: 1}
_DTYPE = attrgetter("dtype")
MAX_RANGES = 64  # ranges of one clipped Adam step


def _dense(t):
    """Whether the elements fill one stretch of memory (in any order of the axes)."""
    if t.is_contiguous():
        return True
    step = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != step:
            return False
        step *= size
    return True


def _list(tensors, name):
    """(pointers, counts, types, device, whether all are contiguous) of dense CUDA tensors."""
    try:  # unbound methods under map: less host time than a loop, for lists of hundreds
        n, dtypes, dev = len(tensors), list(map(_DTYPE, tensors)), tensors[0].device
        contiguous = all(map(torch.Tensor.is_contiguous, tensors))
        if (dev.type == "cuda" and list(map(torch.Tensor.get_device, tensors)).count(dev.index) == n
                and (contiguous or all(map(_dense, tensors)))):
            if dtypes.count(dtypes[0]) == n:
                types = array("i", [_TYPES[dtypes[0]]]) * n
            else:
                types = array("i", map(_TYPES.__getitem__, dtypes))
            return (array("Q", map(torch.Tensor.data_ptr, tensors)), array("q", map(torch.Tensor.numel, tensors)),
                    types, dev, contiguous)
    except (AttributeError, KeyError, TypeError):
        pass
    dev = None
    for k, t in enumerate(tensors):  # find out which
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}[{k}] must be a torch.Tensor")
        if t.dtype not in _TYPES:
            raise RuntimeError(f"{name}[{k}] must be float32, bfloat16 or float16, got {t.dtype}")
        if not t.is_cuda:
            raise RuntimeError(f"{name}[{k}] must be a CUDA tensor (there is no CPU path)")
        if dev is not None and t.device != dev:
            raise RuntimeError(f"{name}[{k}] is on {t.device}, {name}[0] on {dev}")
        dev = t.device
        if not _dense(t):
            raise RuntimeError(f"{name}[{k}] must be dense, got shape {tuple(t.shape)} with strides {t.stride()}")
    raise RuntimeError(f"{name} cannot be used")


def _at(a):
    return a.buffer_info()[0]


def _norm_kind(norm_type):
    kind = _NORMS.get(float(norm_type))
    if kind is None:
        raise RuntimeError(f"norm_type must be 2 or inf, got {norm_type}")
    return kind


@functools.lru_cache(maxsize=256)
def _ws_size(n):
    out = ctypes.c_size_t()
    _native._check(_native.lib().sarr_grad_norm_workspace_size(n, ctypes.byref(out)), "sarr_grad_norm_workspace_size")
    return out.value


def _workspace(n, dev):
    return torch.empty(_ws_size(n), dtype=torch.uint8, device=dev)


def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of `grads` together: norm_type 2 or inf (the
    largest magnitude). A float32 scalar on the gradients' device."""
    grads = list(grads)
    kind = _norm_kind(norm_type)
    if not grads:
        return torch.zeros(())
    ptrs, counts, types, dev, _ = _list(grads, "grads")
    with _native._on(dev):
        ws = _workspace(len(grads), dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        _native._check(_native.lib().sarr_grad_norm(
            len(grads), _at(ptrs), _at(counts), _at(types), kind, norm.data_ptr(), ws.data_ptr(),
            ws.numel(), _native._raw_stream(dev)), "sarr_grad_norm")
    return norm


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Multiplies `grads` by min(1, max_norm / (norm + 1e-6)), in place or into
    the tensors of `out` (as many elements each, contiguous as the gradients are
    or of their shapes and strides; each of its gradient's type or float32), and returns the norm before clipping. No two
    destinations may overlap, nor a destination another tensor's gradient."""
    grads = list(grads)
    kind = _norm_kind(norm_type)
    if not float(max_norm) >= 0.0:
        raise RuntimeError(f"max_norm must be >= 0, got {max_norm}")
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise RuntimeError(f"{len(grads)} gradients and {len(out)} destinations")
    if not grads:
        return torch.zeros(())
    ptrs, counts, types, dev, flat = _list(grads, "grads")
    optrs, otypes = ptrs, types
    if out is not None:
        optrs, ocounts, otypes, odev, oflat = _list(out, "out")
        # (in place a view of negated values is scaled as any other)
        if any(map(torch.Tensor.is_neg, grads)) or any(map(torch.Tensor.is_neg, out)):
            raise RuntimeError("grads or out has a negated view (resolve_neg makes a tensor of it)")
        if ocounts != counts or odev != dev:
            raise RuntimeError("out must have the gradients' sizes and device")
        if otypes != types:
            for k, (g, o) in enumerate(zip(grads, out)):
                if o.dtype != g.dtype and o.dtype != torch.float32:
                    raise RuntimeError(f"out[{k}] must be {g.dtype} or float32, got {o.dtype}")
        if not (flat and oflat):
            for k, (g, o) in enumerate(zip(grads, out)):
                if o.shape != g.shape or o.stride() != g.stride():
                    raise RuntimeError(f"out[{k}] must have its gradient's shape and strides")
    with _native._on(dev):
        ws = _workspace(len(grads), dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        _native._check(_native.lib().sarr_clip_grads(
            len(grads), _at(ptrs), _at(counts), _at(types), _at(optrs), _at(otypes), kind,
            float(max_norm), norm.data_ptr(), ws.data_ptr(), ws.numel(), _native._raw_stream(dev)),
            "sarr_clip_grads")
    increment_version(grads if out is None else out)
    return norm


def clip_grad_norm_(parameters: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: Optional[bool] = None) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_: clips the .grad of `parameters` (a tensor
    or several) in place and returns their total norm. error_if_nonfinite
    reads the norm on the host before anything is clipped; foreach is accepted
    and changes nothing (the list is always taken as one)."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and grads:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the total norm of order {norm_type} of the gradients is non-finite, so they "
                               "cannot be clipped")
    return clip_grads(grads, max_norm, norm_type)


def adam_step_clipped(param, grad, exp_avg, exp_avg_sq, segments, step, max_norm, betas=(0.9, 0.999),
                      eps=1e-8) -> torch.Tensor:
    """torch.optim.Adam's update over flat float32 buffers of equal length (which
    share no memory) with the gradient clipped by its 2-norm (the gradient itself
    is not rewritten); `segments` = [(end, lr), ...] with ascending ends that cover
    the buffers, as in _native.adam_step; `step` counts from 1. Returns the norm."""
    tensors = (param, grad, exp_avg, exp_avg_sq)
    for t, name in zip(tensors, ("param", "grad", "exp_avg", "exp_avg_sq")):
        _native._as_cuda_f32(t, name)
        if t.numel() != param.numel() or not t.is_contiguous() or t.device != param.device:
            raise RuntimeError("Adam buffers must be contiguous, of equal length and on one device")
    count, dev = param.numel(), param.device
    a, b, c, d = sorted(map(torch.Tensor.data_ptr, tensors))
    if min(b - a, c - b, d - c) < 4 * count:
        raise RuntimeError("Adam buffers must not share memory")
    ranges, at = [], 0
    for end, lr in segments:
        ranges.append((at, int(end), at, lr))
        if end < at:
            break
        at = int(end)
    if not ranges or len(ranges) > MAX_RANGES or at != count or ranges[-1][1] != count:
        raise RuntimeError(f"segments must be 1 to {MAX_RANGES} ascending ends, the last one the buffers' {count}")
    if not max_norm >= 0.0:
        raise RuntimeError(f"max_norm must be >= 0, got {max_norm}")
    with _native._on(dev):
        norm = torch.empty((), dtype=torch.float32, device=dev)
        adam_ranges_clipped(tensors, ranges, step, max_norm, betas, eps, norm, _workspace(MAX_RANGES, dev))
    return norm


def adam_ranges_clipped(tensors, ranges, step, max_norm, betas, eps, norm, ws):
    """sarr_adam_step_clipped on the current device: `tensors` = param, grad,
    exp_avg, exp_avg_sq (flat float32), `ranges` = [(begin, end, first gradient,
    lr), ...], `norm` a float32 scalar to write, `ws` the workspace."""
    begin, end, first, lr = zip(*ranges)
    begin, end, first, lr = array("q", begin), array("q", end), array("q", first), array("d", lr)
    _native._check(_native.lib().sarr_adam_step_clipped(
        len(ranges), _at(begin), _at(end), _at(first), _at(lr), *[t.data_ptr() for t in tensors],
        float(betas[0]), float(betas[1]), float(eps), int(step), float(max_norm), norm.data_ptr(),
        ws.data_ptr(), ws.numel(), _native._raw_stream(tensors[0].device)), "sarr_adam_step_clipped")
    increment_version((tensors[0], tensors[2], tensors[3], norm))

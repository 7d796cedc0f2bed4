"""Norm, clipping and clipped Adam over more elements than one sweep of their grids
holds (19 MB for the norm, 10 MB for clipping, 14.5M elements for Adam), so that each CTA
goes on from tensor to tensor or from range to range.

Whole numbers from -8 to 8 as gradients: the sum of squares is exact, so the norm is the
square root rounded to 64 and then to 32 bits. A clipped gradient is c g, c rounded to 32
bits, the product rounded to 32 bits and to the type."""
import math

import pytest
import torch

from cuda_rasterizer import clipping

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U32 = 2.0 ** -24
HALF_SUBNORMAL = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}
LENGTHS = [(3, F32), (9000003, F32), (5, F16), (8000001, BF16), (0, F32), (20000007, F32), (70, BF16), (12000011, F16), (1, F32)]


def _gradients(shift, seed=1):
    g = torch.Generator("cuda").manual_seed(seed)
    return [torch.randint(-8, 9, (n + shift,), generator=g, device="cuda").to(t)[shift:] for n, t in LENGTHS]


def _norm64(grads):
    return math.sqrt(sum(int(g.long().square().sum()) for g in grads))


def _check(got, grads, coef):
    for y, x in zip(got, grads):
        want = x.double() * coef
        tol = want.abs() * ((1 + U32) * (1 + U32) * (1 + torch.finfo(y.dtype).eps / 2) - 1) + HALF_SUBNORMAL[y.dtype]
        assert bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("shift", [0, 3])
def test_long_lists(shift):
    grads = _gradients(shift)
    keep = [g.clone() for g in grads]
    norm64 = _norm64(grads)
    assert float(clipping.grad_norm(grads)) == torch.tensor(norm64, dtype=torch.float64).float().item()
    assert float(clipping.grad_norm(grads, math.inf)) == 8.0
    # into others: the type's own, and 32 bits
    for outs in ([torch.full_like(g, 9.0) for g in grads], [torch.full((g.numel(),), 9.0, device="cuda") for g in grads]):
        clipping.clip_grads(grads, 0.3 * norm64, out=outs)
        _check(outs, grads, 0.3 * norm64 / (norm64 + 1e-6))
        assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    # nothing to clip: some stay in place, the others are copied
    in_place = (1, 3, 7)
    outs = [g if k in in_place else torch.full((g.numel(),), 9.0, device="cuda") for k, g in enumerate(grads)]
    clipping.clip_grads(grads, 2 * norm64, out=outs)
    assert all(torch.equal(o.float(), k.float()) for o, k in zip(outs, keep))
    # and with a small norm the same list is scaled, the sources of the copies left
    clipping.clip_grads(grads, 0.25 * norm64, out=outs)
    _check(outs, keep, 0.25 * norm64 / (norm64 + 1e-6))
    assert all(torch.equal(g, k) for i, (g, k) in enumerate(zip(grads, keep)) if i not in in_place)
    grads = [k.clone() for k in keep]
    assert float(clipping.clip_grads(grads, 2 * norm64)) == float(clipping.grad_norm(keep))
    assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    clipping.clip_grads(grads, 0.5 * norm64)
    _check(grads, keep, 0.5 * norm64 / (norm64 + 1e-6))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_one_bad_element_of_a_long_list(bad):
    for which in (1, 5, 7):
        for at in (0, 5000001, -1):
            grads = _gradients(0)
            grads[which][at] = bad
            norm = clipping.clip_grads(grads, 1.0)
            assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
            if math.isnan(bad):
                assert all(bool(torch.isnan(g).all()) for g in grads)
            else:
                assert sum(int(torch.isnan(g).sum()) for g in grads) == 1 and all(bool((g[~torch.isnan(g)] == 0).all()) for g in grads)


@pytest.mark.parametrize("sizes", [(16000000,), (9000001, 3000003, 20000009)])
@pytest.mark.parametrize("shifts", [(0, 0, 0, 0), (0, 1, 2, 3)])
@pytest.mark.parametrize("clips", [True, False])
def test_long_adam(sizes, shifts, clips):
    """The bounds of a step: m and v from the roundings of their terms, p from those of the move."""
    total, step = sum(sizes), 7
    g = torch.Generator("cuda").manual_seed(total)
    p, gr, m, v = [torch.empty(total + s, device="cuda")[s:] for s in shifts]
    p.normal_(generator=g), gr.normal_(generator=g), m.normal_(std=0.1, generator=g), v.uniform_(generator=g)
    lrs = [1e-3, 5e-3, 1e-5][:len(sizes)]
    ends = [sum(sizes[:k + 1]) for k in range(len(sizes))]
    lr = torch.cat([torch.full((s,), x, dtype=torch.float64, device="cuda") for s, x in zip(sizes, lrs)])
    p0, m0, v0, keep = p.double(), m.double(), v.double(), gr.clone()
    norm64 = math.sqrt(math.fsum(float(x.double().square().sum()) for x in gr.split(1 << 22)))
    max_norm = 0.7 * norm64 if clips else 2 * norm64
    c = min(1.0, max_norm / (norm64 + 1e-6))
    norm = clipping.adam_step_clipped(p, gr, m, v, list(zip(ends, lrs)), step, max_norm)
    assert abs(float(norm) - norm64) <= U32 * (1 + 2.0 ** -20) * norm64 and torch.equal(gr, keep)
    gc = gr.double() * c
    m64, v64 = 0.9 * m0 + 0.1 * gc, 0.999 * v0 + 0.001 * gc * gc
    gm = gc.abs()
    m_tol = 5 * U32 * (gm + m0.abs())
    v_tol = 6 * U32 * (gm * gm + v0) + 2 * HALF_SUBNORMAL[F32]
    assert bool(((m.double() - m64).abs() <= m_tol).all()) and bool(((v.double() - v64).abs() <= v_tol).all())
    denom = (v64 / (1 - 0.999 ** step)).sqrt() + 1e-8
    rate = lr / (1 - 0.9 ** step)
    move = (rate * m64 / denom).abs()
    tol = (rate * m_tol / denom + move * 12 * U32) * 1.001 + move * 3 * U32 * (gm * gm + v0) / v64.clamp(min=1e-300)
    assert bool(((p.double() - (p0 - rate * m64 / denom)).abs() <= tol + p0.abs() * U32 * 1.01 + HALF_SUBNORMAL[F32]).all())

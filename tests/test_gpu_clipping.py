"""Gradient norm, clipping and the clipped Adam step against the formulas in 64
bits: types, lists from none to more than one launch holds, ragged and unaligned
tensors, extreme and non-finite values, streams and CUDA graphs.

Tolerances. The norm is summed in 64 bits, so only its rounding to 32 bits is
seen: 2^-24 (a few 2^-50 of the sum beside it). A clipped gradient is c g with c
rounded to 32 bits (by 2^-24 of it or half of the smallest subnormal), the product
rounded to 32 bits and to the type: (1 + 2^-24)^2 (1 + eps/2) - 1 of the value, or
half of the type's smallest subnormal."""
import math

import pytest
import torch

from cuda_rasterizer import clipping

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_SUBNORMAL = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}
U32 = 2.0 ** -24
NORM_TOL = U32 * (1 + 2.0 ** -20)


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _list(lengths, types, seed, std=1.0, shift=0):
    g = _gen(seed)
    return [(torch.randn(n + shift, generator=g, device="cuda") * std).to(types[k % len(types)])[shift:]
            for k, n in enumerate(lengths)]


def _norm64(grads, kind=2.0):
    if kind == math.inf:
        return max([float(g.abs().max()) for g in grads if g.numel()], default=0.0)
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def _coef(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))


def _check_clipped(got, grads, coef):
    for y, x in zip(got, grads):
        want = x.double() * coef
        tol = want.abs() * ((1 + U32) * (1 + U32) * (1 + torch.finfo(y.dtype).eps / 2) - 1) + HALF_SUBNORMAL[y.dtype]
        tol = tol + x.double().abs() * HALF_SUBNORMAL[F32]
        assert bool(((y.double() - want).abs() <= tol).all())


LISTS = [[], [0], [1], [3, 0, 5], [4095, 4096, 4097], [1] * 17, [100000], [7, 1000003, 12], [257] * 600, [0] * 513 + [5]]


@pytest.mark.parametrize("lengths", LISTS, ids=lambda x: f"{len(x)}x{sum(x)}")
@pytest.mark.parametrize("types", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("shift", [0, 3])
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_norm_and_clip(lengths, types, shift, kind):
    """shift: tensors that begin 3 elements behind a 16-byte boundary."""
    grads = _list(lengths, types, len(lengths), shift=shift)
    keep = [g.clone() for g in grads]
    norm64 = _norm64(grads, kind)
    norm = clipping.grad_norm(grads, kind)
    assert abs(float(norm) - norm64) <= NORM_TOL * norm64
    for max_norm in (0.5 * norm64, 2 * norm64 + 1):
        coef = _coef(norm64, max_norm)
        # into other tensors: aligned like the gradients, otherwise, and in 32 bits
        for outs in ([torch.full_like(g, 9.0) for g in grads],
                     [torch.full((g.numel() + shift,), 9.0, dtype=g.dtype, device="cuda")[shift:] for g in grads],
                     [torch.full((g.numel(),), 9.0, device="cuda") for g in grads]):
            got = clipping.clip_grads(grads, max_norm, kind, out=outs)
            assert float(got) == float(norm)
            _check_clipped(outs, grads, coef)
        assert all(torch.equal(g, k) for g, k in zip(grads, keep))
        mine = [g.clone() for g in grads]
        assert float(clipping.clip_grads(mine, max_norm, kind)) == float(norm)
        _check_clipped(mine, grads, coef)
        if coef == 1.0:
            assert all(torch.equal(g, k) for g, k in zip(mine, keep))


def test_neighbours_of_unaligned_tensors_are_not_touched():
    """Tensors packed back to back in one buffer, the ones between them not in the list."""
    for dtype in (F32, BF16, F16):
        flat = torch.randn(40000, generator=_gen(1), device="cuda").to(dtype)
        keep = flat.clone()
        cuts = [0, 5, 6, 4103, 4110, 12301, 12308, 39991, 40000]
        parts = [flat[a:b] for a, b in zip(cuts, cuts[1:])]
        mine = parts[1::2]
        norm = clipping.clip_grads(mine, 1e-3)
        assert abs(float(norm) - _norm64([keep[a:b] for a, b in list(zip(cuts, cuts[1:]))[1::2]])) <= NORM_TOL * float(norm)
        for k, (a, b) in enumerate(zip(cuts, cuts[1:])):
            if k % 2 == 0:
                assert torch.equal(flat[a:b], keep[a:b])
            else:
                _check_clipped([flat[a:b]], [keep[a:b]], _coef(_norm64([keep[c:d] for c, d in list(zip(cuts, cuts[1:]))[1::2]]), 1e-3))


@pytest.mark.parametrize("value", [3e38, 1e30, 1e-30, 1e-44, 0.0])
def test_extreme_magnitudes(value):
    """Squares that 32 bits cannot hold."""
    g = torch.full((10001,), value, device="cuda")
    norm64 = float(g[0].double()) * math.sqrt(10001)
    got = float(clipping.grad_norm([g]))
    if norm64 > torch.finfo(F32).max:
        assert got == math.inf
    else:
        assert abs(got - norm64) <= NORM_TOL * norm64 + HALF_SUBNORMAL[F32]
    assert float(clipping.grad_norm([g], math.inf)) == float(g[0])
    mine = g.clone()
    clipping.clip_grads([mine], 1.0)
    _check_clipped([mine], [g], _coef(norm64, 1.0))


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_nonfinite_gradients(kind, dtype):
    """As torch.nn.utils.clip_grad_norm_: a NaN makes all NaN, an infinity makes the rest zeros."""
    for bad in (math.nan, math.inf, -math.inf):
        for at in (0, 4999, 9000):
            grads = _list([5000, 4001], (dtype,), 2)
            (grads[0] if at < 5000 else grads[1])[at % 5000] = bad
            ref = [torch.nn.Parameter(g.float()) for g in grads]
            for r, g in zip(ref, grads):
                r.grad = g.float().clone()
            want = torch.nn.utils.clip_grad_norm_(ref, 1.0, norm_type=kind)
            got = clipping.clip_grads(grads, 1.0, kind)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
            for g, r in zip(grads, ref):
                assert torch.equal(torch.isnan(g), torch.isnan(r.grad))
                if not math.isnan(bad):
                    assert bool((g[~torch.isnan(g)] == 0).all())


def test_clip_grad_norm_matches_torch():
    params = [torch.nn.Parameter(torch.randn(s, generator=_gen(3), device="cuda")) for s in ((300, 3), (300, 16), (300,), (2, 5, 7))]
    ref = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, r in zip(params[:3], ref):
        p.grad = torch.randn(p.shape, generator=_gen(4), device="cuda")
        r.grad = p.grad.clone()
    params[1].grad = params[1].grad.t().contiguous().t()  # dense, columns first
    norm = clipping.clip_grad_norm_(iter(params), 0.25)
    want = torch.nn.utils.clip_grad_norm_(ref, 0.25)
    assert torch.allclose(norm, want, rtol=1e-6, atol=0) and params[3].grad is None
    for p, r in zip(params[:3], ref):
        assert torch.allclose(p.grad, r.grad, rtol=1e-6, atol=0)
    one = torch.nn.Parameter(torch.ones(4, device="cuda"))
    one.grad = torch.full((4,), math.inf, device="cuda")
    with pytest.raises(RuntimeError, match="non-finite"):
        clipping.clip_grad_norm_(one, 1.0, error_if_nonfinite=True)
    assert torch.isinf(one.grad).all()  # untouched
    assert float(clipping.clip_grad_norm_(one, 1.0)) == math.inf


def test_refusals():
    a, b = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    wide = torch.ones(8, 8, device="cuda")
    for call in (lambda: clipping.clip_grads([a, a], 1.0), lambda: clipping.clip_grads([a[:40], a[32:]], 1.0),
                 lambda: clipping.clip_grads([wide[:, :4]], 1.0), lambda: clipping.grad_norm([a[:1].expand(4)]),
                 lambda: clipping.clip_grads([a, b], 1.0, out=[b, a]), lambda: clipping.clip_grads([a], 1.0, out=[b[:32]]),
                 lambda: clipping.clip_grads([a], 1.0, out=[b.half()]), lambda: clipping.clip_grads([a], math.nan),
                 lambda: clipping.clip_grads([a], 1.0, norm_type=3), lambda: clipping.grad_norm([a, b.cpu()]),
                 lambda: clipping.clip_grads([wide], 1.0, out=[wide.clone().t()]),
                 lambda: clipping.adam_step_clipped(a, b, a.clone(), b.clone(), [(32, 1e-3)], 1, 1.0),
                 lambda: clipping.adam_step_clipped(a, b[:32], a.clone(), b.clone(), [(64, 1e-3)], 1, 1.0),
                 lambda: clipping.adam_step_clipped(a, b, a.clone(), b.clone(), [(40, 1e-3), (32, 1e-3), (64, 1.0)], 1, 1.0),
                 lambda: clipping.adam_step_clipped(a, b, a.clone(), b.clone(), [(64, 1e-3)], 0, 1.0),
                 lambda: clipping.adam_step_clipped(a, b, a.clone(), b.clone(), [(64, 1e-3)], 1, -1.0),
                 lambda: clipping.adam_step_clipped(a, b.half(), a.clone(), b.clone(), [(64, 1e-3)], 1, 1.0)):
        with pytest.raises(RuntimeError):
            call()
    assert (a == 1).all() and (b == 1).all() and (wide == 1).all()
    assert float(clipping.grad_norm([a, a])) == math.sqrt(128) or abs(float(clipping.grad_norm([a, a])) - math.sqrt(128)) <= 1e-5


def _adam64(p, g, m, v, lr, step, max_norm, b1=0.9, b2=0.999, eps=1e-8):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    norm = float(g.square().sum().sqrt())
    g = g * _coef(norm, max_norm)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return norm, p - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps), m, v


@pytest.mark.parametrize("sizes", [(1,), (3, 1, 16), (4096,), (30001, 10000, 160003)])
@pytest.mark.parametrize("max_norm", [0.0, 0.7, 1e9, math.inf])
@pytest.mark.parametrize("shifts", [(0, 0, 0, 0), (1, 1, 1, 1), (0, 1, 2, 3)])
def test_adam_step_clipped(sizes, max_norm, shifts):
    """shifts: elements between a 16-byte boundary and the first one of param, grad, exp_avg, exp_avg_sq."""
    total = sum(sizes)
    g = _gen(total)
    buf = [torch.empty(total + s, device="cuda")[s:] for s in shifts]
    p, gr, m, v = buf
    p.normal_(generator=g), gr.normal_(generator=g), m.normal_(std=0.1, generator=g), v.uniform_(generator=g)
    lrs = [1e-3, 5e-3, 1e-5][:len(sizes)]
    ends = [sum(sizes[:k + 1]) for k in range(len(sizes))]
    lr = torch.cat([torch.full((s,), x, dtype=torch.float64, device="cuda") for s, x in zip(sizes, lrs)])
    keep = gr.clone()
    for step in (1, 2, 50):
        old = [x.double() for x in (p, m, v)]
        norm64, p64, m64, v64 = _adam64(p, gr, m, v, lr, step, max_norm)
        norm = clipping.adam_step_clipped(p, gr, m, v, list(zip(ends, lrs)), step, max_norm)
        assert abs(float(norm) - norm64) <= NORM_TOL * norm64
        # m and v: four roundings each (c, c g, the difference or square, the constants), the sum; each term's
        # magnitude bounds its share
        c = _coef(norm64, max_norm)
        gm = (gr.double() * c).abs()
        assert bool(((m.double() - m64).abs() <= 5 * U32 * (gm + old[1].abs())).all())
        assert bool(((v.double() - v64).abs() <= 6 * U32 * (gm * gm + old[2]) + 2 * HALF_SUBNORMAL[F32]).all())
        # the move: m's error over the denominator, whose own terms are rounded seven times, then p's rounding
        denom = (v64 / (1 - 0.999 ** step)).sqrt() + 1e-8
        rate = lr / (1 - 0.9 ** step)
        move = (rate * m64 / denom).abs()
        tol = (rate * 5 * U32 * (gm + old[1].abs()) / denom + move * 12 * U32) * 1.001
        # v's error moves sqrt(v) by half of it, relative
        rel_v = 3 * U32 * (gm * gm + old[2]) / v64.clamp(min=1e-300)
        assert bool(((p.double() - p64).abs() <= tol + move * rel_v + p64.abs() * U32 * 1.001 + HALF_SUBNORMAL[F32]).all())
        assert torch.equal(gr, keep)


def test_adam_step_clipped_matches_torch():
    """Three steps of clip_grad_norm_ and torch.optim.Adam with a rate per group."""
    sizes, lrs = (3000, 1000, 16000), (1e-3, 5e-3, 1e-5)
    g = _gen(5)
    params = [torch.randn(s, device="cuda", generator=g) for s in sizes]
    ref = [p.clone().requires_grad_(True) for p in params]
    opt = torch.optim.Adam([{"params": [r], "lr": lr} for r, lr in zip(ref, lrs)])
    flat = torch.cat(params)
    m, v = torch.zeros_like(flat), torch.zeros_like(flat)
    segments = list(zip([3000, 4000, 20000], lrs))
    for step in range(1, 4):
        grads = [torch.randn(s, device="cuda", generator=g) for s in sizes]
        for r, x in zip(ref, grads):
            r.grad = x.clone()
        torch.nn.utils.clip_grad_norm_(ref, 1.0)
        opt.step()
        clipping.adam_step_clipped(flat, torch.cat(grads), m, v, segments, step, 1.0)
    assert torch.allclose(flat, torch.cat([r.detach() for r in ref]), rtol=1e-6, atol=1e-7)


def test_nonfinite_norm_in_adam():
    p, g, m, v = [torch.ones(100, device="cuda") for _ in range(4)]
    g[7] = math.nan
    assert math.isnan(float(clipping.adam_step_clipped(p, g, m, v, [(100, 0.1)], 1, 1.0)))
    assert torch.isnan(p).all()
    p, g, m, v = [torch.ones(100, device="cuda") for _ in range(4)]
    g[7] = math.inf
    assert float(clipping.adam_step_clipped(p, g, m, v, [(100, 0.1)], 1, 1.0)) == math.inf
    assert torch.isnan(p).sum() == 1 and torch.isfinite(p).sum() == 99  # 0 * inf; the others take a zero gradient


def test_streams_and_graphs():
    """Two captured graphs replayed beside eager calls on another stream."""
    lists = [_list([70001, 5, 300000], (F32, BF16), 10 + k) for k in range(3)]
    outs = [[torch.empty_like(g) for g in gs] for gs in lists]
    want = []
    for gs, os in zip(lists, outs):
        n = clipping.clip_grads(gs, 1.0, out=os)
        want.append((float(n), [o.clone() for o in os]))
    torch.cuda.synchronize()
    graphs, norms = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(clipping.clip_grads(lists[k], 1.0, out=outs[k]))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        for os in outs:
            for o in os:
                o.fill_(math.nan)
        side.wait_stream(torch.cuda.current_stream())
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            last = clipping.clip_grads(lists[2], 1.0, out=outs[2])
        torch.cuda.synchronize()
        for k in range(3):
            assert float((norms + [last])[k]) == want[k][0]
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[k][1]))


def test_more_than_32_bits_of_elements():
    """A tensor of more than 2^32 elements: 2^32 + 9 halves, two of them not zero."""
    n = 2 ** 32 + 9
    if torch.cuda.mem_get_info()[0] < 3 * n:
        pytest.skip("not enough free device memory")
    big = torch.zeros(n, dtype=F16, device="cuda")
    big[3], big[-1] = 3.0, 4.0
    assert float(clipping.clip_grads([big], 1.0)) == 5.0
    assert abs(float(big[-1]) - 0.8) <= 0.8 * 2 ** -11 + 1e-6 and abs(float(big[3]) - 0.6) <= 0.6 * 2 ** -11 + 1e-6


def test_in_place_by_name_and_mixed_destinations():
    """out = the list itself is in place; a list may mix tensors clipped in place and into others."""
    grads = _list([1000, 2003, 70], (F32, BF16), 20)
    keep = [g.clone() for g in grads]
    coef = _coef(_norm64(keep), 0.5)
    clipping.clip_grads(grads, 0.5, out=grads)
    _check_clipped(grads, keep, coef)
    grads = [k.clone() for k in keep]
    outs = [grads[0], torch.empty(2003, device="cuda"), grads[2]]
    clipping.clip_grads(grads, 0.5, out=outs)
    _check_clipped(outs, keep, coef)
    assert torch.equal(grads[1], keep[1])


def test_current_stream_of_the_call():
    side = torch.cuda.Stream()
    grads = _list([300000, 7], (F32,), 21)
    want = clipping.grad_norm(grads)
    torch.cuda.synchronize()
    for _ in range(5):
        for _ in range(4):
            clipping.grad_norm([torch.zeros(1000000, device="cuda")])
        with torch.cuda.stream(side):
            mine = [g.clone() for g in grads]
            norm = clipping.clip_grads(mine, 1.0)
            after = clipping.grad_norm(mine)
            assert torch.equal(norm, want) and abs(float(after) - 1.0) <= 1e-5


def test_clipped_adam_of_nothing():
    e = [torch.zeros(0, device="cuda") for _ in range(4)]
    assert float(clipping.adam_step_clipped(*e, [(0, 1e-3)], 1, 1.0)) == 0.0

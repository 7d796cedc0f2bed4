"""Codebook lookup, sort by code and table gradient against the formulas in 64
bits: types, widths, lengths from none to many, skewed and empty codes, indexes
outside the table, strided and unaligned rows, streams and CUDA graphs.

Tolerances. A rounding to type t is off by at most eps(t)/2 of the value (or half
of the smallest subnormal); a product in 32 bits by 2^-24. A sum of k terms in 32
bits in any order is off by at most (k - 1) 2^-24 of the sum of magnitudes, to
first order; (k + 2) 2^-24 covers the higher orders and the product with scale
for the sizes here (k below 2^17)."""
import math

import numpy as np
import pytest
import torch

from cuda_rasterizer import codebook

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_SUBNORMAL = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}
U32 = 2.0 ** -24


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _index(n, codes, seed, none=0.1, skew=2.0, dtype=torch.int64):
    g = _gen(seed)
    i = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) ** skew * max(codes, 1)).long()
    i = i.clamp(max=max(codes - 1, 0))
    bad = torch.rand(n, generator=g, device="cuda") < none
    # outside in every way: -1, the number of codes, the type's extremes
    out = torch.tensor([-1, codes, torch.iinfo(dtype).min, torch.iinfo(dtype).max], device="cuda")
    return torch.where(bad, out[torch.randint(4, (n,), generator=g, device="cuda")], i).to(dtype)


def _valid(index, codes):
    i = index.reshape(-1).long()
    return (i >= 0) & (i < codes), i


def _lookup64(table, index, scale):
    ok, i = _valid(index, table.shape[0])
    out = torch.zeros(i.numel(), table.shape[1], dtype=torch.float64, device="cuda")
    out[ok] = table.double()[i[ok]] * scale
    return out


def _grad64(rows, index, codes, scale):
    """(gradient, sum of magnitudes, terms per code) in 64 bits."""
    ok, i = _valid(index, codes)
    out = torch.zeros(codes, rows.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    out.index_add_(0, i[ok], rows.double()[ok])
    mag.index_add_(0, i[ok], rows.double()[ok].abs())
    return out * scale, mag * abs(scale), torch.bincount(i[ok], minlength=codes)


def _check_lookup(got, want, dtype):
    tol = want.abs() * ((1 + U32) * (1 + torch.finfo(dtype).eps / 2) - 1) + HALF_SUBNORMAL[dtype]
    assert got.dtype == dtype
    assert bool(((got.double().reshape(want.shape) - want).abs() <= tol).all())


def _check_grad(got, rows, index, codes, scale, dtype):
    want, mag, terms = _grad64(rows, index, codes, scale)
    tol32 = mag * ((terms[:, None] + 2) * U32)
    tol = tol32 + (want.abs() + tol32) * (torch.finfo(dtype).eps / 2) + HALF_SUBNORMAL[dtype]
    assert got.dtype == dtype and got.shape == want.shape
    assert bool(((got.double() - want).abs() <= tol).all())
    assert bool((got[terms == 0] == 0).all())


def _sort_np(index, codes):
    i = index.reshape(-1).cpu().numpy().astype(np.int64)
    keys = np.where((i >= 0) & (i < codes), i, codes)
    order = np.argsort(keys, kind="stable")
    return order, keys[order], np.searchsorted(keys[order], np.arange(codes + 1))


TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]


@pytest.mark.parametrize("n", [0, 1, 2, 31, 257, 4099])
@pytest.mark.parametrize("codes,cols", [(1, 1), (7, 3), (64, 16), (300, 20), (33, 250), (5, 2056)])
def test_lookup_sizes(n, codes, cols):
    index = _index(n, codes, n + cols)
    for k, (tt, rt) in enumerate(TYPES):
        table = torch.randn(codes, cols, generator=_gen(k), device="cuda").to(tt)
        got = codebook.lookup(table, index if k % 2 else index.clamp(-9, 2 ** 31 - 1).int(), scale=0.75, dtype=rt)
        _check_lookup(got, _lookup64(table, index, 0.75), rt)


def test_lookup_shapes_strides_and_special_values():
    table = torch.randn(50, 40, generator=_gen(1), device="cuda")
    index = _index(60, 50, 2).reshape(3, 4, 5)
    got = codebook.lookup(table, index, scale=-2.0)
    assert got.shape == (3, 4, 5, 40)
    _check_lookup(got, _lookup64(table, index, -2.0), F32)
    # column slices (rows that do not start on 16 bytes), a transposed table, a strided index
    for t in (table[:, 1:18], table[:, 4:20], table[::3], table.t(), table.bfloat16()[:, 3:], table.half()[:, 8:24]):
        i = _index(200, t.shape[0], 3)[::2]
        _check_lookup(codebook.lookup(t, i), _lookup64(t, i, 1.0), t.dtype)
    # rows without a code are zeros even where scale or table are not finite
    t = torch.full((4, 8), math.inf, device="cuda")
    out = codebook.lookup(t, torch.tensor([0, -1, 4, 3], device="cuda"), scale=math.nan)
    assert torch.isnan(out[0]).all() and (out[1:3] == 0).all() and torch.isnan(out[3]).all()
    big = torch.full((1, 8), 60000.0, device="cuda", dtype=F16)
    assert torch.isinf(codebook.lookup(big, torch.zeros(1, dtype=torch.int64, device="cuda"), scale=2.0)).all()
    # an empty table: every Gaussian is without a code
    none = codebook.lookup(torch.empty(0, 8, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"))
    assert none.shape == (5, 8) and (none == 0).all()
    assert codebook.lookup(torch.empty(4, 0, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")).shape == (5, 0)


@pytest.mark.parametrize("n,codes", [
    (0, 0), (0, 5), (1, 1), (1, 100000), (33, 2), (1000, 1), (1023, 511), (1024, 512), (1025, 513), (4097, 300),
    (40000, 4096), (65536, 65536), (65537, 1000), (70000, 3), (200003, 70000), (150000, 300000), (300000, 2 ** 27),
    (1000, 2 ** 20)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(n, codes, dtype):
    index = _index(n, codes, n + 1, dtype=dtype, skew=1.5)
    got = codebook.sort_by_code(index, codes)
    for x, y in zip(got, _sort_np(index, codes)):
        assert x.dtype == torch.int32
        assert np.array_equal(x.cpu().numpy(), y)


@pytest.mark.parametrize("n", [20000, 90000])
@pytest.mark.parametrize("kind", ["one", "none", "ascending", "descending"])
def test_sort_extreme_orders(n, kind):
    codes = 1000
    i = torch.arange(n, device="cuda")
    index = {"one": torch.full_like(i, 700), "none": torch.full_like(i, -5), "ascending": i * codes // n,
             "descending": (n - 1 - i) * codes // n}[kind]
    for x, y in zip(codebook.sort_by_code(index, codes), _sort_np(index, codes)):
        assert np.array_equal(x.cpu().numpy(), y)


GRAD_TYPES = TYPES + [(F32, BF16), (F32, F16)]


@pytest.mark.parametrize("n", [0, 1, 9, 257, 5003])
@pytest.mark.parametrize("codes,cols", [(1, 1), (7, 3), (64, 16), (3000, 20), (33, 250), (5, 2056)])
def test_gradient_sizes(n, codes, cols):
    index = _index(n, codes, n + cols)
    for k, (gt, tt) in enumerate(GRAD_TYPES):
        rows = torch.randn(n, cols, generator=_gen(k), device="cuda").to(gt)
        got = codebook.gradient(rows, index, codes, scale=1.5, dtype=tt)
        _check_grad(got, rows, index, codes, 1.5, tt)


@pytest.mark.parametrize("n,codes,cols,skew", [
    (100003, 1, 16, 1.0), (100003, 2, 16, 1.0), (100003, 4096, 16, 4.0), (60001, 100, 1, 3.0), (60001, 100, 5, 3.0),
    (20011, 17, 128, 2.0), (20011, 5000, 1000, 2.0), (3001, 3, 4100, 1.0), (100003, 40000, 16, 1.0)])
def test_gradient_long_and_skewed(n, codes, cols, skew):
    """Codes over many spans (up to all of them), codes that end where a span does, empty codes between them."""
    index = _index(n, codes, n + cols, skew=skew, none=0.01)
    for k, (gt, tt) in enumerate([(F32, F32), (BF16, F32)]):
        rows = torch.randn(n, cols, generator=_gen(k), device="cuda").to(gt)
        got = codebook.gradient(rows, index, codes, scale=0.5, dtype=tt)
        _check_grad(got, rows, index, codes, 0.5, tt)
        assert torch.equal(got, codebook.gradient(rows, index, codes, scale=0.5, dtype=tt))  # the same bits


@pytest.mark.parametrize("length", [1, 7, 8, 16, 32, 64, 511, 512, 513, 2048])
def test_gradient_of_equal_runs(length):
    """Every code has `length` Gaussians, so that codes begin and end at every place of the parts and spans."""
    codes = max(1, 30000 // length)
    index = torch.arange(codes, device="cuda").repeat_interleave(length)
    index = index[torch.randperm(index.numel(), generator=_gen(3), device="cuda")]
    for cols in (4, 16, 1030):
        n = index.numel() if cols < 100 else min(index.numel(), 6000)
        rows = torch.randn(n, cols, generator=_gen(4), device="cuda")
        _check_grad(codebook.gradient(rows, index[:n], codes), rows, index[:n], codes, 1.0, F32)


def test_gradient_strides_and_nonfinite_rows():
    n, codes = 3000, 40
    index = _index(n, codes, 5)
    wide = torch.randn(n, 40, generator=_gen(6), device="cuda")
    order = codebook.sort_by_code(index, codes)
    for rows in (wide[:, 1:18], wide[:, 4:20], wide.bfloat16()[:, 3:11], wide.half()[:, 8:24]):
        _check_grad(codebook.gradient_sorted(rows, order, 1.0, F32), rows, index, codes, 1.0, F32)
    # into the columns of a wider table: the others keep what they held
    table = torch.full((codes, 24), 7.0, device="cuda")
    codebook.gradient_sorted(wide[:, :16], order, 1.0, out=table[:, 3:19])
    _check_grad(table[:, 3:19].contiguous(), wide[:, :16], index, codes, 1.0, F32)
    assert (table[:, :3] == 7).all() and (table[:, 19:] == 7).all()
    # a row without a code does not reach the table, whatever it holds; others do
    ok, i = _valid(index, codes)
    bad = wide[:, :16].clone()
    bad[~ok] = math.nan
    assert torch.equal(codebook.gradient_sorted(bad, order), codebook.gradient_sorted(wide[:, :16].contiguous(), order))
    at = int(torch.nonzero(ok)[0])
    bad[at] = math.inf
    got = codebook.gradient_sorted(bad, order)
    assert torch.isinf(got[i[at]]).all() and torch.isfinite(got).all(dim=1).sum() == codes - 1


def test_offsets_past_32_bits():
    """Rows that begin behind 2^31 and 2^32 elements of a strided matrix."""
    n, stride, cols = 5, 2 ** 30 + 64, 16
    big = torch.empty((n - 1) * stride + cols, dtype=BF16, device="cuda")
    rows = big.as_strided((n, cols), (stride, 1))
    rows.copy_(torch.randn(n, cols, generator=_gen(7), device="cuda"))
    index = torch.tensor([2, 0, 2, 1, 0], device="cuda")
    _check_grad(codebook.gradient(rows, index, 3, dtype=F32), rows, index, 3, 1.0, F32)
    i = torch.tensor([4, 3, 0, -1, 4], device="cuda")
    _check_lookup(codebook.lookup(rows, i), _lookup64(rows, i, 1.0), BF16)


def test_autograd_against_formula_and_differences():
    codes, cols, scale = 9, 5, 1.75
    table = torch.randn(codes, cols, generator=_gen(8), device="cuda", requires_grad=True)
    index = torch.tensor([[3, -1, 3], [8, 0, 3]], device="cuda")
    weight = torch.randn(2, 3, cols, generator=_gen(9), device="cuda")
    rows = codebook.lookup(table, index, scale)
    (rows.square() * weight).sum().backward()
    want, mag, terms = _grad64((2 * rows.detach() * weight).reshape(-1, cols), index, codes, scale)
    # the row gradients are given; only the sum and its rounding differ
    assert bool(((table.grad.double() - want).abs() <= mag * (8 * U32) + 1e-30).all())

    def f(t):
        ok, i = _valid(index, codes)
        r = _lookup64(t, index, scale).reshape(2, 3, cols)
        return float((r.square() * weight.double()).sum())

    # f is quadratic, so central differences are exact but for 64-bit rounding
    t = table.detach().double()
    for c, j in ((3, 0), (8, 4), (0, 2), (5, 1)):
        up, down = t.clone(), t.clone()
        up[c, j] += 0.5
        down[c, j] -= 0.5
        assert abs((f(up) - f(down)) - float(table.grad[c, j])) <= 1e-5 * (1 + abs(float(table.grad[c, j])))
    # half tables get half gradients; no gradient is made where none is asked for
    half = table.detach().half().requires_grad_()
    codebook.lookup(half, index, scale, dtype=F32).sum().backward()
    assert half.grad.dtype == F16
    with torch.no_grad():
        assert codebook.lookup(table, index).grad_fn is None


def test_refusals():
    table = torch.zeros(4, 8, device="cuda")
    index = torch.zeros(3, dtype=torch.int64, device="cuda")
    rows = torch.zeros(3, 8, device="cuda")
    order = codebook.sort_by_code(index, 4)
    for call in (lambda: codebook.lookup(table.double(), index), lambda: codebook.lookup(table, index.short()),
                 lambda: codebook.lookup(table[0], index), lambda: codebook.lookup(table, index.cpu()),
                 lambda: codebook.lookup(table, index, dtype=F16), lambda: codebook.lookup(table.half(), index, dtype=BF16),
                 lambda: codebook.gradient(rows[:2], index, 4), lambda: codebook.gradient(rows, index, -1),
                 lambda: codebook.gradient(rows.half(), index, 4, dtype=BF16),
                 lambda: codebook.gradient_sorted(rows[:2], order),
                 lambda: codebook.gradient_sorted(rows, order, out=torch.zeros(5, 8, device="cuda")),
                 lambda: codebook.gradient_sorted(rows, order, out=torch.zeros(8, 4, device="cuda").t()),
                 lambda: codebook.gradient_sorted(rows, order, out=table, dtype=F16),
                 lambda: codebook.gradient_sorted(rows, codebook.SortedCodes(order.order.long(), order.codes, order.offsets))):
        with pytest.raises(RuntimeError):
            call()


def test_streams_and_graphs():
    """Two captured graphs and eager calls on another stream, interleaved, each with its own results."""
    n, codes, cols = 70000, 600, 16
    index = [_index(n, codes, 10 + k) for k in range(3)]
    rows = [torch.randn(n, cols, generator=_gen(20 + k), device="cuda") for k in range(3)]
    table = torch.randn(codes, cols, generator=_gen(30), device="cuda")
    want = [(codebook.gradient(r, i, codes), codebook.lookup(table, i)) for r, i in zip(rows, index)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((codebook.gradient(rows[k], index[k], codes), codebook.lookup(table, index[k])))
        graphs.append(g)
    side = torch.cuda.Stream()
    eager = []
    for _ in range(3):
        for k, g in enumerate(graphs):
            for t in outs[k]:
                t.fill_(math.nan)
        side.wait_stream(torch.cuda.current_stream())
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            eager.append((codebook.gradient(rows[2], index[2], codes), codebook.lookup(table, index[2])))
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(outs[k][0], want[k][0]) and torch.equal(outs[k][1], want[k][1])
    for e in eager:
        assert torch.equal(e[0], want[2][0]) and torch.equal(e[1], want[2][1])


@pytest.mark.parametrize("shape", [(), (0,), (0, 3), (1,), (2, 0, 4), (2, 3)])
def test_autograd_of_every_index_shape(shape):
    """No axis, no element, several axes; an expanded incoming gradient (of a plain sum)."""
    table = torch.randn(6, 5, generator=_gen(40), device="cuda", requires_grad=True)
    index = torch.randint(-1, 6, shape, generator=_gen(41), device="cuda")
    rows = codebook.lookup(table, index, 0.5)
    assert rows.shape == (*shape, 5)
    rows.sum().backward()
    ok, i = _valid(index, 6)
    want = 0.5 * torch.bincount(i[ok], minlength=6).double()[:, None].expand(6, 5)
    assert torch.equal(table.grad.double(), want)
    with pytest.raises(RuntimeError):
        codebook.gradient(torch.zeros(7, 3, 5, device="cuda"), torch.zeros(7, dtype=torch.int64, device="cuda"), 6)


def test_captured_backward():
    """A whole forward and backward in a graph, replayed on new values."""
    table = torch.randn(300, 16, generator=_gen(42), device="cuda", requires_grad=True)
    index = torch.randint(0, 300, (5000,), generator=_gen(43), device="cuda")
    weight = torch.randn(5000, 16, generator=_gen(44), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad((codebook.lookup(table, index, 2.0) * weight).sum(), table)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad((codebook.lookup(table, index, 2.0) * weight).sum(), table)
    for seed in (45, 46):
        weight.copy_(torch.randn(5000, 16, generator=_gen(seed), device="cuda"))
        graph.replay()
        assert torch.equal(got, codebook.gradient(weight, index, 300, 2.0))


def test_order_of_another_index_stays_inside():
    """An order that was not made for these rows gives wrong sums, and touches nothing outside the table and the rows."""
    n, codes = 5000, 50
    order = codebook.sort_by_code(_index(n, codes, 50), codes)
    rows = torch.randn(n, 16, generator=_gen(51), device="cuda")
    g = _gen(52)
    wild = [torch.randint(-2 ** 31, 2 ** 31 - 1, (t.numel(),), generator=g, device="cuda").int() for t in order]
    around = torch.full((codes + 2, 16), 3.0, device="cuda")
    for bad in (codebook.SortedCodes(wild[0], order.codes, order.offsets), codebook.SortedCodes(order.order, wild[1], order.offsets)):
        codebook.gradient_sorted(rows, bad, out=around[1:-1])
        torch.cuda.synchronize()
        assert (around[0] == 3).all() and (around[-1] == 3).all()
    # places that are not aligned to 16 bytes are refused
    shifted = torch.empty(n + 1, dtype=torch.int32, device="cuda")[1:].copy_(order.order)
    with pytest.raises(RuntimeError):
        codebook.gradient_sorted(rows, codebook.SortedCodes(shifted, order.codes, order.offsets))


def test_current_stream_of_the_call():
    """Inputs made and outputs read on a side stream, while the default stream is busy with other calls."""
    n, codes = 60000, 700
    index, table = _index(n, codes, 60), torch.randn(codes, 16, generator=_gen(61), device="cuda")
    rows = torch.randn(n, 16, generator=_gen(62), device="cuda")
    want = codebook.lookup(table, index, 2.0), codebook.gradient(rows, index, codes)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        for _ in range(4):
            codebook.gradient(rows, index.flip(0).contiguous(), codes)
        with torch.cuda.stream(side):
            i, t, r = index.clone(), table.clone(), rows.clone()
            got = codebook.lookup(t, i, 2.0), codebook.gradient(r, i, codes)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_autograd_with_a_kept_order():
    index = _index(5000, 60, 70).reshape(50, 100)
    order = codebook.sort_by_code(index, 60)
    weight = torch.randn(50, 100, 12, generator=_gen(71), device="cuda")
    grads = []
    for o in (None, order):
        table = torch.randn(60, 12, generator=_gen(72), device="cuda", requires_grad=True)
        (codebook.lookup(table, index, 0.5, order=o) * weight).sum().backward()
        grads.append(table.grad)
    assert torch.equal(grads[0], grads[1]) and float(grads[0].abs().max()) > 0
    for bad in (codebook.sort_by_code(index[:10], 60), codebook.sort_by_code(index, 61)):
        with pytest.raises(RuntimeError):
            codebook.lookup(table, index, order=bad)

"""Sort and table gradient at the sizes of the large scenes (up to 2M Gaussians), and
sums that have to be exact.

Rows of whole numbers from -8 to 8 with a power of two as the scale: every partial sum
is a whole number below 2^24, so 32-bit sums are exact in any order, and a row that is
lost, added twice or taken from another code shows as a difference. Random rows are held
to what the sums' tree can lose: a row's value passes through at most 64 additions in its
part, 255 joins of a span's parts and, in these cases, 313 spans added one after another
(16 columns or less: 16 in a row, or the spans shared by at least 4 groups and a tree
over them); 640 with the scale. Each addition is off by at most 2^-24 of a partial sum,
which the sum of magnitudes bounds."""
import numpy as np
import pytest
import torch

from cuda_rasterizer import codebook

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CHAIN = 640


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _index(n, codes, seed, skew=1.5, none=0.02, dtype=torch.int64):
    g = _gen(seed)
    i = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) ** skew * codes).long().clamp_(max=codes - 1)
    i[torch.rand(n, generator=g, device="cuda") < none] = -1
    return i.to(dtype)


def _check_sort(index, codes):
    got = codebook.sort_by_code(index, codes)
    i = index.cpu().numpy().astype(np.int64)
    keys = np.where((i >= 0) & (i < codes), i, codes)
    order = np.argsort(keys, kind="stable")
    for x, y in zip(got, (order, keys[order], np.searchsorted(keys[order], np.arange(codes + 1)))):
        assert np.array_equal(x.cpu().numpy(), y)


# on both sides of the sizes from which a thread holds 4 and 8 keys, and of more tiles than SMs
@pytest.mark.parametrize("n", [303104, 303105, 606208, 606209, 1000003, 1212417, 2000003])
@pytest.mark.parametrize("codes", [1, 200, 4096, 65536, 2 ** 21 + 5])
def test_sort(n, codes):
    _check_sort(_index(n, codes, n + codes, dtype=torch.int32 if n % 2 else torch.int64), codes)


@pytest.mark.parametrize("n", [400000, 700000, 1500000])
@pytest.mark.parametrize("kind", ["one", "none", "ascending", "descending"])
@pytest.mark.parametrize("codes", [4000, 50000])
def test_sort_extreme_orders(n, kind, codes):
    i = torch.arange(n, device="cuda")
    _check_sort({"one": torch.full_like(i, codes - 1), "none": torch.full_like(i, -5), "ascending": i * codes // n,
                 "descending": (n - 1 - i) * codes // n}[kind], codes)


def _whole_rows(n, cols, dtype, seed):
    return torch.randint(-8, 9, (n, cols), generator=_gen(seed), device="cuda").to(dtype)


def _sums(rows, index, codes):
    ok = (index >= 0) & (index < codes)
    out = torch.zeros(codes, rows.shape[1], dtype=torch.float64, device="cuda")
    return out.index_add_(0, index.long()[ok], rows.double()[ok])


def _check_exact(rows, index, codes, dtype):
    want = _sums(rows, index, codes) * 0.5
    got = codebook.gradient(rows, index, codes, scale=0.5, dtype=dtype)
    assert torch.equal(got, want.float().to(dtype))
    out = torch.full((codes, rows.shape[1] + 4), 9.0, dtype=dtype, device="cuda")
    codebook.gradient_sorted(rows, codebook.sort_by_code(index, codes), 0.5, out=out[:, 3:-1])
    assert torch.equal(out[:, 3:-1], got) and (out[:, :3] == 9).all() and (out[:, -1] == 9).all()


@pytest.mark.parametrize("n,codes,cols,skew", [
    (100003, 1, 16, 1.0), (100003, 2, 16, 1.0), (100003, 4096, 16, 4.0), (60001, 100, 1, 3.0), (60001, 100, 5, 3.0),
    (20011, 17, 128, 2.0), (20011, 5000, 1000, 2.0), (3001, 3, 4100, 1.0), (100003, 40000, 16, 1.0),
    (500009, 1, 16, 1.0), (500009, 4096, 16, 3.0), (1000003, 1, 16, 1.0), (1000003, 7, 16, 1.0), (1000003, 4096, 16, 3.0),
    (1000003, 65536, 9, 1.0), (1000003, 300, 1, 2.0), (2000003, 4096, 16, 2.0), (1000, 256, 16, 2.0), (1025, 3, 16, 1.0),
    (2048, 5, 8, 1.0), (300007, 4096, 64, 2.0)])
def test_exact_sums(n, codes, cols, skew):
    index = _index(n, codes, n + cols, skew=skew)
    for k, (gt, tt) in enumerate([(F32, F32), (BF16, F32), (F16, F16), (F32, BF16)]):
        _check_exact(_whole_rows(n, cols, gt, k), index, codes, tt)


@pytest.mark.parametrize("length", [1, 7, 8, 16, 32, 64, 511, 512, 513, 2047, 2048, 2049, 30000])
@pytest.mark.parametrize("cols", [4, 16, 1030])
def test_exact_sums_of_equal_runs(length, cols):
    """Codes that begin and end at every place of the parts and spans, some of them unused."""
    codes = max(1, (1000000 if cols < 100 else 6000) // length)
    index = (2 * torch.arange(codes, device="cuda")).repeat_interleave(length)
    index = index[torch.randperm(index.numel(), generator=_gen(3), device="cuda")]
    _check_exact(_whole_rows(index.numel(), cols, F32, 4), index, 2 * codes, F32)


@pytest.mark.parametrize("n,codes,cols", [(100003, 1, 16), (100003, 2, 16), (60001, 100, 1), (60001, 100, 5), (20011, 17, 128),
                                          (20011, 5000, 1000), (3001, 3, 4100), (1000003, 1, 16), (1000003, 4096, 16)])
def test_random_rows_to_the_depth_of_the_sum(n, codes, cols):
    index = _index(n, codes, n, skew=2.0)
    for k, dtype in enumerate((F32, BF16)):
        rows = torch.randn(n, cols, generator=_gen(k), device="cuda").to(dtype)
        got = codebook.gradient(rows, index, codes, scale=0.5, dtype=F32)
        bound = _sums(rows.abs(), index, codes) * (0.5 * CHAIN * 2.0 ** -24)
        assert bool(((got.double() - _sums(rows, index, codes) * 0.5).abs() <= bound).all())


def test_wild_offsets_stay_inside():
    """Offsets that no sort made: wrong sums of codes over several spans, nothing outside the table."""
    n, codes = 100003, 50
    index = _index(n, codes, 60)
    order = codebook.sort_by_code(index, codes)
    rows = torch.randn(n, 16, generator=_gen(61), device="cuda")
    around = torch.full((codes + 2, 16), 3.0, device="cuda")
    for wild in (torch.randint(-2 ** 30, 2 ** 30, (codes + 1,), generator=_gen(62), device="cuda").int(), order.offsets.flip(0).contiguous(),
                 torch.full_like(order.offsets, n), torch.zeros_like(order.offsets)):
        codebook.gradient_sorted(rows, codebook.SortedCodes(order.order, order.codes, wild), out=around[1:-1])
        torch.cuda.synchronize()
        assert (around[0] == 3).all() and (around[-1] == 3).all()

"""What the bits of the table gradient, the norm and the clipped gradients may depend
on: sizes, codes, types, strides and how far the arrays lie from a 16-byte boundary, as
the header states. Not on the addresses otherwise, nor on the call, its stream or the
order's origin."""
import pytest
import torch

from cuda_rasterizer import clipping, codebook

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _placed(values, at, pitch):
    """`values` [n, cols] `at` elements into rows of `pitch` elements of a new buffer."""
    wide = torch.zeros(values.shape[0], pitch, dtype=values.dtype, device="cuda")
    wide[:, at:at + values.shape[1]] = values
    return wide[:, at:at + values.shape[1]]


@pytest.mark.parametrize("n,codes,cols", [(100003, 3, 16), (100003, 4096, 16), (20011, 50, 6), (5011, 700, 1000), (900, 40, 16)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_gradient_bits(n, codes, cols, dtype, at):
    index = torch.randint(-1, codes, (n,), generator=_gen(n), device="cuda")
    rows = torch.randn(n, cols, generator=_gen(cols), device="cuda").to(dtype)
    order = codebook.sort_by_code(index, codes)
    pitch = (cols + 7) // 8 * 8 + 32
    per = 16 // rows.element_size()

    def at_places(row_at, table_at):
        out = _placed(torch.zeros(codes, cols, device="cuda"), table_at, pitch)
        codebook.gradient_sorted(_placed(rows, row_at, pitch), order, 0.75, out=out)
        return out

    want = at_places(at, at).clone()
    assert float(want.abs().max()) > 0
    # whole 16-byte steps further on; on another stream; the sort in the same call
    assert torch.equal(at_places(at + per, at + 4), want) and torch.equal(at_places(at + 2 * per, at + 8), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(at_places(at, at), want)
    if at == 0 and cols % per == 0:
        assert torch.equal(codebook.gradient(rows, index, codes, 0.75, dtype=torch.float32), want)
    # elsewhere the sums may be cut otherwise: two sums of k terms, each off by at most (k + 2) 2^-24 of the magnitudes
    other = at_places(at + 1, at)
    ok = index >= 0
    mag = torch.zeros(codes, cols, dtype=torch.float64, device="cuda").index_add_(0, index[ok], rows.double()[ok].abs()) * 0.75
    terms = torch.bincount(index[ok], minlength=codes)[:, None]
    assert bool(((other.double() - want.double()).abs() <= 2 * (terms + 2) * 2.0 ** -24 * mag).all())


@pytest.mark.parametrize("at", [0, 1, 3])
def test_norm_and_clip_bits(at):
    values = [torch.randn(n, generator=_gen(n), device="cuda").to(t) for n, t in
              ((1000003, torch.float32), (70001, torch.bfloat16), (5, torch.float16), (300000, torch.float32))]

    def placed(step):
        return [torch.cat([x.new_zeros(at + step * 16 // x.element_size()), x])[at + step * 16 // x.element_size():] for x in values]

    results = []
    for step in (0, 1, 5):
        grads = placed(step)
        norm = clipping.clip_grads(grads, 0.25)
        results.append([norm, *grads])
    assert float(results[0][0]) > 0.25
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))

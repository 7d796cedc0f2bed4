"""The operators in a training run: ViewParallelTrainer and DensifyingTrainer with
the SH rows in a codebook and the gradients clipped, against the same step
composed from the drop-in modules, torch indexing in 64 bits, torch's clipping
and torch.optim.Adam; the bucketed path of several ranks with the collectives
replaced by a sum of equal ranks; a graph-captured step of the operators."""
import pytest
import torch

from cuda_rasterizer import _native, clipping, codebook, multiview
from cuda_rasterizer import cuda_rasterizer_sar as M
from cuda_rasterizer import rasterizer_autograd as RA
from cuda_rasterizer import synthetic as S

from _helpers import rel_linf

pytestmark = pytest.mark.gpu


def _scene(n, codes, seed, cols=16):
    g = torch.Generator().manual_seed(seed)
    means = (torch.rand((n, 3), generator=g) - 0.5) * torch.tensor([20.0, 20.0, 0.0]) \
        + torch.tensor([0.0, 0.0, 3.0]) * torch.rand((n, 1), generator=g)
    scales = torch.rand((n, 3), generator=g) * 2.3 - 3.0
    rot = torch.randn((n, 4), generator=g)
    rot = rot / rot.norm(dim=1, keepdim=True)
    logits = torch.randn((n,), generator=g)
    table = torch.randn((codes, cols), generator=g) * 0.1
    table[:, 0] += 0.5
    index = torch.randint(-1, codes, (n,), generator=g)
    return [t.cuda() for t in (means, scales, rot, logits, table, index)]


def _targets(views_t):
    t = S.named_scene("target_20k", seed=1, device="cuda")
    return M.render_sar_batched(t["means"], t["cov6"], t["sigma"], t["sh"], views_t)


def _rows(table, index, scale):
    ok = index >= 0
    return torch.where(ok[:, None], table[index.clamp(min=0)] * scale, 0.0)


def _composed_gradients(means, scales, rot, logits, table, index, scale, views_t, targets):
    cov6, sigma = _native.gaussian_params(scales, rot, logits, _native.SARR_COV6)
    rows = _rows(table, index, scale)
    images = M.render_sar_batched(means, cov6, sigma, rows, views_t)
    losses, gimg = _native.combined_loss(images, targets, 1.0, 0.2, 5, "plain")
    gm, _, gs, gsh = M.render_sar_backward_batched(means, cov6, sigma, rows, gimg, views_t)
    gt = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
    ok = index >= 0
    gt.index_add_(0, index[ok], gsh.double()[ok])
    return losses, gm, gs * sigma * (1.0 - sigma), (gt * scale).float()


@pytest.mark.parametrize("max_norm", [None, 1e-4, 1e6])
@pytest.mark.parametrize("ranks", [1, 2])
def test_codebook_and_clipped_step(max_norm, ranks, monkeypatch):
    """Two steps. ranks = 2: the trainer's buckets as with two ranks of equal views, each all-reduce a doubling."""
    n, codes, scale, lr = 20000, 300, 0.5, 1e-3
    means, scales, rot, logits, table, index = _scene(n, codes, 91)
    views_t = S.training_views(8)
    views = [_native.make_view(*v) for v in views_t]
    targets = _targets(views_t)
    reduced = []
    if ranks == 2:
        class Work:
            def __init__(self, t):
                self.t = t

            def wait(self):
                self.t.mul_(2.0)

        monkeypatch.setattr(multiview.dist, "is_initialized", lambda: True)
        monkeypatch.setattr(multiview.dist, "get_world_size", lambda group=None: 2)
        monkeypatch.setattr(multiview.dist, "all_reduce", lambda t, group=None, async_op=False: reduced.append(t) or Work(t))
    tr = multiview.ViewParallelTrainer(means, scales, rot, logits, table, lr=lr, buckets=3, sh_index=index, sh_scale=scale,
                                       max_grad_norm=max_norm)
    ref = [t.clone().requires_grad_(True) for t in (means, logits, table)]
    opt = torch.optim.Adam([{"params": [ref[0]], "lr": lr}, {"params": [ref[1]], "lr": lr}, {"params": [ref[2]], "lr": lr * 0.01}])
    for _ in range(2):
        losses = tr.step(views, targets)
        want, *grads = _composed_gradients(ref[0].detach(), scales, rot, ref[1].detach(), ref[2].detach(), index, scale, views_t,
                                           targets)
        for r, g in zip(ref, grads):
            r.grad = g.reshape(r.shape).clone()
        if max_norm is not None:
            norm = torch.nn.utils.clip_grad_norm_(ref, max_norm)
            assert abs(float(tr.grad_norm) - float(norm)) <= 1e-5 * float(norm)
            assert (float(norm) > 1e-4) and (float(norm) < 1e6)  # one of the two limits clips
        else:
            assert tr.grad_norm is None
        for got, g in zip(tr.gradients(), grads):
            assert rel_linf(got.cpu().numpy(), g.reshape(got.shape).cpu().numpy()) <= 1e-5
        opt.step()
        assert torch.allclose(losses[0] * ranks, want[0], rtol=1e-6, atol=0)  # the total is weighted by 1 / ranks
        assert torch.allclose(losses[1:], want[1:], rtol=1e-6, atol=0)
    for got, r in zip((tr.means, tr.logits, tr.sh), ref):
        assert rel_linf(got.cpu().numpy(), r.detach().cpu().numpy()) <= 1e-6
    assert float((tr.sh - table).abs().max()) > 0
    if ranks == 2:  # three buckets of Gaussians and the table's, each step
        assert len(reduced) == 8 and reduced[3].numel() == codes * 16


def test_unclipped_limit_equals_plain_trainer():
    n = 6000
    means, scales, rot, logits, _, _ = _scene(n, 4, 92)
    sh = torch.randn(n, 16, generator=torch.Generator("cuda").manual_seed(1), device="cuda") * 0.1
    views_t = S.training_views(4)
    views = [_native.make_view(*v) for v in views_t]
    targets = _targets(views_t)
    a = multiview.ViewParallelTrainer(means, scales, rot, logits, sh)
    b = multiview.ViewParallelTrainer(means, scales, rot, logits, sh, max_grad_norm=1e9)
    for t in (a, b):
        t.step(views, targets)
    assert float(b.grad_norm) > 0
    assert all(torch.equal(x, y) for x, y in zip(a.gradients(), b.gradients()))
    # the same update but for 1 - beta rounded to 32 bits from beta in 32 or in 64 bits (up to 2^-24 / 1e-3 of v)
    assert torch.allclose(a.param, b.param, rtol=1e-6, atol=1e-7)


def test_active_degree_leaves_the_other_columns():
    means, scales, rot, logits, table, index = _scene(6000, 50, 93)
    views = [_native.make_view(*v) for v in S.training_views(4)]
    targets = _targets(S.training_views(4))
    tr = multiview.ViewParallelTrainer(means, scales, rot, logits, table, sh_index=index.int(), max_grad_norm=1.0)
    tr.g_sh_rows.fill_(float("nan"))
    tr.sh_active = 4
    tr.step(views, targets)
    assert torch.equal(tr.sh[:, 4:], table[:, 4:]) and not torch.equal(tr.sh[:, :4], table[:, :4])
    assert (tr.gradients()[2][:, 4:] == 0).all() and torch.isfinite(tr.param).all()


def test_densification_keeps_the_codes():
    from cuda_rasterizer import densify
    n, codes = 20000, 70
    means, scales, rot, logits, table, index = _scene(n, codes, 94)
    views_t = S.training_views(8)
    views = [_native.make_view(*v) for v in views_t]
    targets = _targets(views_t)
    dt = multiview.DensifyingTrainer(means, scales, rot, logits, table, buckets=1, densify_interval=2, grad_threshold=0.0,
                                     size_threshold=1.0, sh_interval=1, sh_index=index, max_grad_norm=0.5)
    dt.step(views, targets)
    dt.step(views, targets)
    old = dt.tr
    before = [t.clone() for t in (old.means, old.scales, old.rotations, old.logits)]
    trained = old.sh.clone()
    dt.step(views, targets)
    # the codes of the new set from a copy that carries them as floats
    out, counts = densify.densify_and_prune_tensors(*before, index.float().unsqueeze(1), old.gradients()[0], 0.0, 1.0, 2.0, 0.005,
                                                    2_000_000)
    assert counts[3] > 0 and dt.n == out[0].shape[0] != n
    assert torch.equal(dt.tr.sh_index.float(), out[4].reshape(-1)) and int(dt.tr.sh_index.min()) == -1
    assert torch.equal(dt.tr.sh, trained) and torch.equal(dt.tr.means, out[0])
    dt.step(views, targets)  # the new set trains on
    assert dt.tr.steps_done == 1 and not torch.equal(dt.tr.sh, trained)


def test_trainer_refusals():
    means, scales, rot, logits, table, index = _scene(300, 20, 95)
    args = (means, scales, rot, logits, table)
    for bad in (index[:-1], index.float(), index.clamp(min=19) + 1, torch.full_like(index, -2)):
        with pytest.raises(ValueError):
            multiview.ViewParallelTrainer(*args, sh_index=bad)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            multiview.ViewParallelTrainer(*args, sh_index=index, max_grad_norm=bad)


def test_autograd_training_with_a_codebook():
    """The operators through the autograd module: codebook rows, rasterizer, clip_grad_norm_ on the leaves."""
    n, codes = 3000, 40
    means, scales, rot, logits, table, index = _scene(n, codes, 96)
    cov6, sigma = _native.gaussian_params(scales, rot, logits, _native.SARR_COV6)
    view = S.training_views(4)[1]
    raster = RA.SARRasterizer(*view)
    p_means, p_table = means.clone().requires_grad_(True), table.clone().requires_grad_(True)
    image = raster(p_means, cov6, sigma, codebook.lookup(p_table, index, 0.5))
    w = torch.randn(image.shape, generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    (image * w).sum().backward()
    q_means, q_rows = means.clone().requires_grad_(True), _rows(table, index, 0.5).requires_grad_(True)
    (raster(q_means, cov6, sigma, q_rows) * w).sum().backward()
    want = torch.zeros(codes, 16, dtype=torch.float64, device="cuda")
    ok = index >= 0
    want.index_add_(0, index[ok], q_rows.grad.double()[ok])
    assert torch.equal(p_means.grad, q_means.grad)
    assert rel_linf(p_table.grad.cpu().numpy(), (0.5 * want).cpu().numpy()) <= 1e-5
    norm64 = float(torch.cat([p_means.grad.reshape(-1), p_table.grad.reshape(-1)]).double().norm())
    norm = clipping.clip_grad_norm_([p_means, p_table], 0.5 * norm64)
    assert abs(float(norm) - norm64) <= 1e-6 * norm64
    assert abs(float(clipping.grad_norm([p_means.grad, p_table.grad])) - 0.5 * norm64) <= 1e-5 * norm64


def test_captured_run_of_the_operators():
    """Lookup, table gradient, clipped Adam as one graph, replayed three times, against three eager rounds."""
    n, codes = 30000, 200
    index = torch.randint(0, codes, (n,), generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    aim = torch.randn(n, 16, generator=torch.Generator("cuda").manual_seed(4), device="cuda")

    def state():
        t = torch.zeros(codes * 16, device="cuda")
        return t, torch.zeros_like(t), torch.zeros_like(t)

    def once(table, m, v):
        rows = codebook.lookup(table.view(codes, 16), index, 2.0)
        grad = codebook.gradient(rows - aim, index, codes, 2.0)
        return clipping.adam_step_clipped(table, grad.view(-1), m, v, [(table.numel(), 0.1)], 1, 3.0)

    eager, captured = state(), state()
    once(*state())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = once(*captured)
    for _ in range(3):
        want = once(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
    assert all(torch.equal(a, b) for a, b in zip(eager, captured)) and float(eager[0].abs().max()) > 0

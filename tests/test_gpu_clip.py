"""Gradients clipped in place, against 64 bits."""
import numpy as np
import pytest
import torch

from jax_gs_amd.core.gaussians import Gaussians
from jax_gs_amd.training.adamw import clip_grads_, grad_norms
from jax_gs_amd.training.optimizer import FIELDS, Adam

pytestmark = pytest.mark.gpu


def want_clipped(grads, max_norm, mask=None, scale=1.0):
    g = [x.detach().double().cpu().numpy() for x in grads]
    on = [np.ones(x.shape, bool) if mask is None else np.broadcast_to(mask.reshape(-1, *[1] * (x.ndim - 1)), x.shape) for x in g]
    total = abs(scale) * np.sqrt(sum(float((x[m] ** 2).sum()) for x, m in zip(g, on)))
    factor = scale * min(1.0, max_norm / (total + 1e-6))
    return total, factor, [np.where(m, x * factor, x) for x, m in zip(g, on)]


def check(grads, norms, want):
    total, factor, values = want
    # a float32 result of float64 sums: half a step each; the factor another
    np.testing.assert_allclose(float(norms.total), total, rtol=2.0 ** -23)
    np.testing.assert_allclose(float(norms.scale), factor, rtol=2.0 ** -23)
    for g, x in zip(grads, values):
        # the factor (half a step of float32), the product (another), and one rounding to the type,
        # or half of its smallest value
        info = torch.finfo(g.dtype)
        rtol = info.eps / 2 + 2.0 ** -22
        np.testing.assert_allclose(g.double().cpu().numpy(), x, rtol=rtol, atol=info.tiny * info.eps / 2)


def some(shape, seed, dtype, device):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * torch.exp(torch.randn(shape, generator=gen))).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shapes", [[(1,)], [(3,), (0,), (1,)], [(8191,), (8193,), (4, 5)], [(100003,), (7, 3), (2048,)]])
@pytest.mark.parametrize("scale", [None, 0.25, -3.0])
def test_clip(cuda, dtype, shapes, scale):
    """Views at any element of one buffer; what is between them stays."""
    sizes = [int(np.prod(s)) for s in shapes]
    flat = some((sum(sizes) + 3 * len(sizes),), 1, dtype, cuda)
    grads, at, between = [], 1, torch.ones_like(flat, dtype=torch.bool)
    for s, n in zip(shapes, sizes):
        grads.append(flat[at:at + n].view(s))
        between[at:at + n] = False
        at += n + 3
    rest = flat[between].clone()
    want = want_clipped(grads, 0.7, scale=1.0 if scale is None else scale)
    same = grad_norms(grads, max_norm=0.7, grad_scale=scale)
    version = flat._version
    norms = clip_grads_(grads, 0.7, grad_scale=scale)
    check(grads, norms, want)
    assert torch.equal(norms.total, same.total) and torch.equal(norms.scale, same.scale) and torch.equal(norms.per_tensor, same.per_tensor)
    assert torch.equal(flat[between], rest) and flat._version > version


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, row", [(1, 1), (300, 1), (333, 3), (1000, 48), (3, 5001), (20000, 7)])
def test_masked_rows_keep_what_they_hold(cuda, dtype, rows, row):
    g = [some((rows, row), rows, dtype, cuda), some((rows,), 2, dtype, cuda), None]
    mask = np.random.default_rng(rows).random(rows) < 0.5
    on = torch.from_numpy(mask).to(cuda)
    g[0][~on] = float("nan")
    g[1][~on] = float("inf")
    before = [x.clone() for x in g[:2]]
    norms = clip_grads_(g, 0.1, active_mask=on)
    for x, b in zip(g, before):
        assert torch.equal(x[~on].float().nan_to_num(), b[~on].float().nan_to_num())
    total, factor, values = want_clipped([torch.where(on.view(-1, *[1] * (x.dim() - 1)), x, 0.0) for x in before], 0.1, mask)
    check([torch.where(on.view(-1, *[1] * (x.dim() - 1)), x, 0.0) for x in g[:2]], norms, (total, factor, values))


def test_small_gradients_stay_and_bad_ones_stay(cuda):
    g = [some((5000,), 1, torch.float32, cuda), some((31,), 2, torch.float16, cuda)]
    before = [x.clone() for x in g]
    norms = clip_grads_(g, 1e6)
    assert float(norms.scale) == 1.0 and all(torch.equal(a, b) for a, b in zip(g, before))
    for bad in (float("nan"), float("inf")):
        h = [x.clone() for x in before]
        h[0][4999] = bad
        kept = [x.clone() for x in h]
        norms = clip_grads_(h, 1.0)
        assert bool(torch.isnan(norms.scale)) and all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(h, kept))
    h = [x.clone() for x in before]
    norms = clip_grads_(h, 1.0, grad_scale=torch.full((), float("inf"), device=cuda))
    assert bool(torch.isnan(norms.scale)) and all(torch.equal(a, b) for a, b in zip(h, before))
    z = [torch.zeros(100, device=cuda)]
    assert float(clip_grads_(z, 1.0).total) == 0.0 and not bool(z[0].any())


def test_a_norm_beyond_float32_still_clips(cuda):
    g = [torch.full((1000,), 3e38, device=cuda)]
    norms = clip_grads_(g, 1.0)
    assert torch.isinf(norms.total)
    total = 3e38 * np.sqrt(1000.0)
    # float32 factor below the normal range: steps of 2^-149
    np.testing.assert_allclose(g[0].double().cpu().numpy(), float(np.float32(3e38)) / total, rtol=2.0 ** -149 / (1.0 / total) + 2.0 ** -22)


def test_dense_gradients_of_any_order(cuda):
    g = some((8, 16, 5, 7), 1, torch.float32, cuda).to(memory_format=torch.channels_last)
    t = some((300, 200), 2, torch.bfloat16, cuda).t()
    want = want_clipped([g, t], 0.5)
    check([g, t], clip_grads_([g, t], 0.5), want)
    assert g.is_contiguous(memory_format=torch.channels_last)
    for bad in (torch.zeros(4, 8, device=cuda)[:, :3], torch.zeros(4, device=cuda).expand(3, 4)):
        with pytest.raises(ValueError, match="dense"):
            clip_grads_([bad], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        clip_grads_([g, g], 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        clip_grads_([g], 1.0, active_mask=torch.ones(8, device=cuda))


def test_many_tensors_and_large_ones(cuda):
    rng = np.random.default_rng(0)
    g = [some((int(n),), i, torch.bfloat16 if i % 3 else torch.float32, cuda) for i, n in enumerate(np.exp(rng.uniform(0, 12, 400)))]
    g.append(some((6_000_000, 4), 5, torch.float32, cuda))
    want = want_clipped(g, 3.0)
    check(g, clip_grads_(g, 3.0), want)


def test_very_many_tensors_and_none(cuda):
    """More partial sums than every workgroup would add for itself, and no elements at all."""
    g = [some((1 + i % 7,), i, torch.float32, cuda) for i in range(5000)]
    want = want_clipped(g, 3.0)
    norms = clip_grads_(g, 3.0)
    check(g, norms, want)
    each = grad_norms(g).per_tensor
    assert norms.per_tensor.shape == each.shape and bool(torch.isfinite(norms.per_tensor).all())
    for none in ([torch.zeros(0, device=cuda)], [None, torch.zeros(0, 3, device=cuda), None]):
        norms = clip_grads_(none, 1.0)
        assert float(norms.total) == 0.0 and float(norms.scale) == 1.0 and not bool(norms.per_tensor.any())
    assert float(clip_grads_([g[0]], float("inf")).scale) == 1.0


def test_captured_and_replayed(cuda):
    g = [torch.randn(70_000, device=cuda), torch.randn(333, 3, device=cuda).bfloat16()]
    clip_grads_([x.clone() for x in g], 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = clip_grads_(g, 1.0)
    for k in (1.0, 1e-4, 30.0):
        for x in g:
            x.normal_().mul_(k)
        mine = [x.clone() for x in g]
        graph.replay()
        want = clip_grads_(mine, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(norms.scale, want.scale) and all(torch.equal(a, b) for a, b in zip(g, mine))


def test_a_graph_that_needs_the_gradients_is_refused(cuda):
    w = torch.randn(100, device=cuda, requires_grad=True)
    g = torch.randn(100, device=cuda)
    loss = (w * g).sum()
    clip_grads_([g], 0.1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    kept = torch.randn(100, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        clip_grads_([kept], 0.1)


def test_adam_clips_its_gradients(cuda):
    """The step of Adam(max_grad_norm) is Adam's own on the clipped gradients; train_step reports the norm."""
    from jax_gs_amd import scenes
    from jax_gs_amd.training.density import init_density_state
    from jax_gs_amd.training.trainer import train_step

    sc = scenes.make_scene(1, n=1500, width=96, height=64)
    rates = {f: 1e-3 for f in FIELDS}
    runs = {}
    for name, opt in (("clipped", Adam(rates, max_grad_norm=1e-4)), ("free", Adam(rates, max_grad_norm=1e9)), ("plain", Adam(rates))):
        g, cam, tgt, _ = scenes.to_torch(sc, "cuda:0")
        state = init_density_state(g, opt, 2000)
        for _ in range(2):
            state, _, metrics = train_step(state, tgt, cam.W2C, (cam.W, cam.H, cam.fx, cam.fy, cam.cx, cam.cy), opt, sh_degree=3,
                                           fused=False)
        runs[name] = state, metrics
    assert "grad_norm" not in runs["plain"][1] and runs["plain"][0].opt_state.norms is None
    norm = float(runs["free"][1]["grad_norm"])
    assert norm > 1e-3
    mu = torch.cat([x.reshape(-1) for x in runs["clipped"][0].opt_state.mu.values()])
    # 0.1 g1 0.9 + 0.1 g2, both of norm 1e-4 at most
    assert 0.0 < float(mu.norm()) <= 0.19e-4 * (1.0 + 1e-5)
    g = Gaussians(*[torch.randn(2000, *s, device=cuda) for s in ((3,), (3,), (4,), (1,), (16, 3))])
    state = runs["clipped"][0]
    on = state.active_mask
    before = [getattr(g, f).clone() for f in FIELDS]
    # (the compositing backward's atomics make two runs differ in their last bits: one gradient for both)
    for name, opt in (("free", Adam(rates, max_grad_norm=1e9)), ("plain", Adam(rates))):
        runs[name] = opt.init(g)
        opt.step(Gaussians(*[b.clone() for b in before]), g, runs[name], on)
    assert all(torch.equal(runs["free"].mu[f], runs["plain"].mu[f]) and torch.equal(runs["free"].nu[f], runs["plain"].nu[f]) for f in FIELDS)
    Adam(rates, max_grad_norm=0.5).step(state.gaussians, g, state.opt_state, on)
    check([torch.where(on.bool().view(-1, *[1] * (getattr(g, f).dim() - 1)), getattr(g, f), 0.0) for f in FIELDS], state.opt_state.norms,
          want_clipped([torch.where(on.bool().view(-1, *[1] * (b.dim() - 1)), b, 0.0) for b in before], 0.5))

"""Clipping inside the optimizer's and the trainer's steps."""
import pytest
import torch

from jax_gs_amd.core.gaussians import Gaussians
from jax_gs_amd.training.optimizer import FIELDS, Adam

pytestmark = pytest.mark.gpu
RATES = {f: 1e-3 for f in FIELDS}


def test_norms_are_those_of_the_last_step(cuda):
    """A step that does not clip leaves none behind, in either form of the training step."""
    from jax_gs_amd import scenes
    from jax_gs_amd.training.density import init_density_state
    from jax_gs_amd.training.trainer import train_step

    sc = scenes.make_scene(1, n=1500, width=96, height=64)
    g, cam, tgt, _ = scenes.to_torch(sc, "cuda:0")
    clips, plain = Adam(RATES, max_grad_norm=1e-2), Adam(RATES)
    state = init_density_state(g, clips, 2000)
    static = (cam.W, cam.H, cam.fx, cam.fy, cam.cx, cam.cy)
    for fused in (False, True):
        _, _, metrics = train_step(state, tgt, cam.W2C, static, clips, sh_degree=3, fused=fused)
        assert float(state.opt_state.norms.total) == float(metrics["grad_norm"]) > 0.0
        _, _, metrics = train_step(state, tgt, cam.W2C, static, plain, sh_degree=3, fused=fused)
        assert "grad_norm" not in metrics and state.opt_state.norms is None
    assert state.opt_state.count == 4


def test_a_mask_of_one_column(cuda):
    """Adam takes any mask with an entry for each Gaussian, with clipping too."""
    n = 300
    gen = torch.Generator(device=cuda).manual_seed(1)
    some = lambda: Gaussians(*[torch.randn(n, *s, generator=gen, device=cuda) for s in ((3,), (3,), (4,), (1,), (16, 3))])
    params, grads = some(), some()
    mask = torch.rand(n, generator=gen, device=cuda) < 0.5
    runs = []
    for m in (mask, mask[:, None], mask.view(1, n, 1).to(torch.int32)):
        p, g = [Gaussians(*[getattr(x, f).clone() for f in FIELDS]) for x in (params, grads)]
        opt = Adam(RATES, max_grad_norm=0.5)
        state = opt.step(p, g, opt.init(p), active_mask=m)
        runs.append([state.norms.total, *[getattr(x, f) for x in (p, g) for f in FIELDS]])
    for run in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], run))

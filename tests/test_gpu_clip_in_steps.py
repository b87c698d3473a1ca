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

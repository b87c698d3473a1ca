"""Density control moves the moments of the five arrays, whatever else the optimizer's state is of."""
import contextlib
from array import array

import pytest
import torch

from jax_gs_amd import _lib
from jax_gs_amd.core.gaussians import Gaussians
from jax_gs_amd.training.adamw import AdamW, AdamWState
from jax_gs_amd.training.density import DensityState, densify_and_prune, init_density_state
from jax_gs_amd.training.optimizer import FIELDS

SHAPES = dict(means=(3,), scales=(3,), quaternions=(4,), opacities=(1,), sh_coeffs=(16, 3))
N = 700


def shapes_of(n):
    """The five arrays in an order of their own, a table with a row for each Gaussian and two tensors without."""
    own = {f: (n, *SHAPES[f]) for f in FIELDS}
    return {"exposure": (7,), "sh_coeffs": own.pop("sh_coeffs"), "features": (n, 5), "opacities": own.pop("opacities"), "step": (),
            **own}


def test_the_entry_gets_the_five_arrays_moments(monkeypatch):
    shapes = shapes_of(N)
    opt = AdamWState(list(shapes), shapes.values(), 8)
    opt._allocate(torch.device("cpu"), zero=True)
    calls = {}
    monkeypatch.setattr(_lib, "call", lambda name, *args: calls.update({name: args}))
    monkeypatch.setattr(_lib, "stream_handle", lambda device: None)
    monkeypatch.setattr(_lib, "on", lambda device: contextlib.nullcontext())
    state = DensityState(Gaussians(*[torch.zeros(N, *SHAPES[f]) for f in FIELDS]), opt, torch.ones(N, dtype=torch.uint8), N,
                         torch.zeros(N), torch.zeros(N, dtype=torch.int32), torch.zeros(N))
    densify_and_prune(state, noise=torch.zeros(N, 3))
    _, k, lens, rows, offsets, size, *_ = calls["gs_moments_move"]
    at = {name: o for name, o in zip(shapes, opt.offsets)}
    want = sorted((at[f], torch.Size(SHAPES[f]).numel()) for f in FIELDS)
    assert k == 5 and rows == N and size == opt.size
    assert list(zip(array("q", offsets), array("q", lens))) == want
    nbytes = calls["gs_moments_move"][-1]
    assert nbytes >= _lib.lib().gs_moments_move_workspace_size(k, lens, rows)


@pytest.mark.parametrize("names", [["means", "scales"], ["means", "scales", "quaternions", "opacities", "colours"]])
def test_a_state_of_other_tensors_is_refused(names):
    opt = AdamWState(names, [(N, 3)] * len(names), 8)
    opt._allocate(torch.device("cpu"), zero=True)
    state = DensityState(Gaussians(*[torch.zeros(N, *SHAPES[f]) for f in FIELDS]), opt, torch.ones(N, dtype=torch.uint8), N,
                         torch.zeros(N), torch.zeros(N, dtype=torch.int32), torch.zeros(N))
    with pytest.raises(ValueError, match="sh_coeffs"):
        densify_and_prune(state, noise=torch.zeros(N, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_other_moments_stay(cuda, bits):
    gen = torch.Generator(device=cuda).manual_seed(3)
    g = Gaussians(*[torch.randn(N, *SHAPES[f], generator=gen, device=cuda) for f in FIELDS])
    g.scales.fill_(-2.0)
    state = init_density_state(g, None, 2 * N)
    params = {name: getattr(state.gaussians, name) if name in FIELDS else torch.zeros(s, device=cuda)
              for name, s in shapes_of(2 * N).items()}
    # whole numbers of few bits: blocks hold them exactly, with whatever neighbours
    mu = {name: torch.randint(1, 8, p.shape, generator=gen, device=cuda).float() for name, p in params.items()}
    opt = state.opt_state = AdamW(1e-3, moment_bits=bits).restore(params, mu, {name: m * m for name, m in mu.items()}, 3)
    state.grad_accum[:200], state.denom[:200] = 1.0, 1
    densify_and_prune(state, extent=100.0, sources=True, generator=gen)
    index = state.last_sources.long()
    assert int((index.cpu() != torch.arange(2 * N)).sum()) > 0
    now_mu, now_nu = opt.moments()
    for name, m in mu.items():
        want = m[index] if name in FIELDS else m
        assert torch.equal(now_mu[name], want) and torch.equal(now_nu[name], want * want), name

"""What is changed in place is changed as a whole: an allocation that fails comes before the first launch."""
import contextlib

import pytest
import torch

from jax_gs_amd import _lib
from jax_gs_amd.core.gaussians import Gaussians
from jax_gs_amd.training.adamw import AdamWState
from jax_gs_amd.training.density import DensityState, densify_and_prune
from jax_gs_amd.training.optimizer import FIELDS, AdamState

SHAPES = dict(means=(3,), scales=(3,), quaternions=(4,), opacities=(1,), sh_coeffs=(16, 3))


@pytest.fixture
def host(monkeypatch):
    """The calls that would launch something, by name, and a switch that makes the n-th allocation from now on fail."""

    class Host:
        calls, fail = [], -1

        def until_none_fails(self, call):
            """`call` with its first allocation failing, its second, and so on, and once without; names of what that one calls."""
            for self.fail in range(100):
                self.calls = []
                try:
                    call()
                except torch.OutOfMemoryError:
                    assert self.calls == [], f"allocation {made[0]} fails behind them"
                    made[0] = 0
                else:
                    return self.calls
                finally:
                    made[0] = 0

    h, made, empty = Host(), [0], torch.empty

    def one(*args, **kwargs):
        made[0] += 1
        if made[0] - 1 == h.fail:
            raise torch.OutOfMemoryError("no memory")
        return empty(*args, **kwargs)

    monkeypatch.setattr(torch, "empty", one)
    monkeypatch.setattr(_lib, "call", lambda name, *args: h.calls.append(name))
    monkeypatch.setattr(_lib, "stream_handle", lambda device: None)
    monkeypatch.setattr(_lib, "on", lambda device: contextlib.nullcontext())
    return h


def a_state(bits, masters=False, n=50):
    state = AdamWState(list(FIELDS), [(n, *SHAPES[f]) for f in FIELDS], bits)
    state._allocate(torch.device("cpu"), zero=True)
    if masters:
        state.master_flat = torch.zeros(state.size)
    return state


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("masters", [False, True])
def test_moments_and_masters_move_together(host, bits, masters):
    state = a_state(bits, masters)
    index = torch.arange(50, dtype=torch.int32)
    names = host.until_none_fails(lambda: state.move_rows_(index))
    assert names == ["gs_move_rows"] * (bits == 32 or masters) + ["gs_moments_move"] * (bits == 8)


@pytest.mark.parametrize("kind", ["none", "adam", "32", "8"])
@pytest.mark.parametrize("sources", [False, True])
def test_density_control_moves_all_or_nothing(host, kind, sources):
    n = 50
    zeros = lambda *s: torch.zeros((n, *s))
    opt = None
    if kind == "adam":
        opt = AdamState(mu={f: zeros(*SHAPES[f]) for f in FIELDS}, nu={f: zeros(*SHAPES[f]) for f in FIELDS})
    elif kind != "none":
        opt = a_state(int(kind))
    state = DensityState(Gaussians(*[zeros(*SHAPES[f]) for f in FIELDS]), opt, torch.ones(n, dtype=torch.uint8), n, zeros(),
                         torch.zeros(n, dtype=torch.int32), zeros())
    names = host.until_none_fails(lambda: densify_and_prune(state, noise=zeros(3), sources=sources))
    want = ["gs_densify_and_prune"] + ["gs_densify_sources"] * (sources or kind == "8") + ["gs_moments_move"] * (kind == "8")
    assert names == want
    assert (state.last_sources is not None) == (sources or kind == "8")

"""States that were saved whole before they kept a layout of their rows are moved as others."""
import contextlib
import copy

import torch

from jax_gs_amd import _lib
from jax_gs_amd.training.adamw import AdamWState


def test_a_state_without_a_row_layout(monkeypatch):
    state = AdamWState(["a", "b"], [(6, 3), (6,)], 8)
    state._allocate(torch.device("cpu"), zero=True)
    old = copy.copy(state)
    old.__dict__.pop("_row_layout", None)
    names = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: names.append(name))
    monkeypatch.setattr(_lib, "stream_handle", lambda device: None)
    monkeypatch.setattr(_lib, "on", lambda device: contextlib.nullcontext())
    index = torch.arange(6, dtype=torch.int32)
    old.move_rows_(index)
    assert old.take_rows(index[:2]).shapes == [(2, 3), (2,)]
    assert names == ["gs_moments_move", "gs_moments_take"]
    assert old._rows("take_rows") == state._rows("take_rows")

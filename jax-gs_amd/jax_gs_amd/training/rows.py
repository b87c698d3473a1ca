"""Rows of many tensors by one index: taken into new tensors, moved in place, and the index of the
rows with the best scores.

A row is what one leading index selects in every tensor: a Gaussian in the five arrays, their moments
and whatever else a program keeps of it, or a page of a pool.  Free, copy, fork and compact are one index:

    keep = best_rows(scores, budget, active_mask=state.active_mask)   # int32, ascending, -1 where none is left
    gaussians = take_rows(gaussians, keep)                            # new tensors: compacted, or grown
    move_rows_(features, sources)                                     # in place: row i becomes row sources[i]

Tensors are ``Gaussians``, dicts, lists or tuples of tensors, or one tensor, of any type and with the
same number of rows.  Values arrive as they were, bit by bit.  Nothing waits for the host, and nothing is
differentiated.  The kernels are ``gs_take_rows``, ``gs_move_rows`` and ``gs_best_rows``;
``AdamWState.take_rows`` and ``move_rows_`` do the same for moments in 32 or in 8 bits.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ..core.gaussians import Gaussians
from ..renderer._buffers import as_bytes
from .adamw import _device, _fills, _keys, _tensors, row_index


def _like(tensors, new: list):
    """The new tensors as the given ones came."""
    if isinstance(tensors, torch.Tensor):
        return new[0]
    if isinstance(tensors, Gaussians):
        return Gaussians(*new)
    return dict(zip(tensors, new)) if isinstance(tensors, dict) else new


def take_rows(tensors, index: torch.Tensor, fill=None):
    """New tensors, in the form of the given ones (a list for a tuple), whose row i is row ``index[i]``: an index that comes
    twice forks a row, one that does not come drops it.  Where ``index`` is negative or not a
    row's, the row holds ``fill`` (for each tensor one row or None; zeros without it)."""
    ts = _tensors(tensors)
    if not ts:
        raise ValueError("take_rows: no tensors")
    dev = _device(ts[0], "take_rows")
    index = row_index(index, dev, "take_rows")
    with _lib.on(dev):
        pointers, row_bytes, strides, rows, fills, out, new, kept = _lib.tensors().take(
            ts, None if fill is None else _fills(fill, _keys(tensors), len(ts), "take_rows"), index.numel(), dev.index, "take_rows")
        _lib.call("gs_take_rows", _lib.stream_handle(dev), len(ts), pointers, row_bytes, strides, rows, out, None, fills,
                  index.data_ptr(), 8 * index.element_size(), index.numel())
    return _like(tensors, new)


def move_rows_(tensors, index: torch.Tensor, fill=None, left: Optional[torch.Tensor] = None):
    """In place, row i of every tensor becomes its row ``index[i]``, or ``fill`` (zeros without it) where
    ``index`` is negative; only rows that change are written.  Returns the tensors.

    ``index`` has an entry for every row, i itself where row i stays.  A row can be copied from one that
    stays only: where ``index`` asks for one that changes itself, or for none of the rows, the row is
    left as it is, and ``left`` (one int32 on the device, if given) is raised by one."""
    ts = _tensors(tensors)
    if not ts:
        raise ValueError("move_rows_: no tensors")
    dev = _device(ts[0], "move_rows_")
    index = row_index(index, dev, "move_rows_")
    if left is not None and (left.dtype != torch.int32 or left.numel() != 1 or left.device != dev):
        raise ValueError(f"move_rows_: left must be one int32 on {dev}")
    native = _lib.tensors()
    with _lib.on(dev):
        pointers, row_bytes, strides, rows, fills, kept = native.move(
            ts, None if fill is None else _fills(fill, _keys(tensors), len(ts), "move_rows_"), index, dev.index, "move_rows_")
        if index.numel() != rows:
            raise ValueError(f"move_rows_: {index.numel()} indices for {rows} rows")
        _lib.call("gs_move_rows", _lib.stream_handle(dev), len(ts), pointers, row_bytes, strides, rows, fills,
                  index.data_ptr(), 8 * index.element_size(), None if left is None else left.data_ptr())
    native.written([], [], ts)
    return tensors


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def best_rows(scores: Optional[torch.Tensor], k: int, active_mask=None) -> torch.Tensor:
    """int32 [k]: the numbers of the k rows with the highest scores, ascending, and -1 behind them where
    there are fewer.  Rows whose ``active_mask`` is False are left out; of equal scores the lowest
    rows come first; NaN is below every number.  Without ``scores`` the first k rows of the mask."""
    k = int(k)
    if k < 0 or k >= 1 << 31:
        raise ValueError(f"best_rows: {k} rows")
    given = active_mask if scores is None else scores
    if not isinstance(given, torch.Tensor):
        raise ValueError("best_rows: scores or a mask are needed, on the GPU")
    dev = _device(given, "best_rows")
    if given.dim() != 1:
        raise ValueError(f"best_rows: one score for each row, not a tensor of shape {tuple(given.shape)}")
    rows, type = given.numel(), 0
    if scores is not None:
        if scores.dtype not in _TYPES:
            raise TypeError(f"best_rows: scores must be float32, bfloat16 or float16, not {scores.dtype}")
        type, scores = _TYPES[scores.dtype], scores.resolve_neg().contiguous()
    act = None
    if active_mask is not None:
        act = as_bytes(torch.as_tensor(active_mask, device=dev))
        if act.dim() != 1 or act.numel() != rows:
            raise ValueError(f"best_rows: active_mask has shape {tuple(act.shape)}, there are {rows} rows")
    nbytes = _lib.lib().gs_best_rows_workspace_size(rows)
    with _lib.on(dev):
        out = torch.empty((k,), dtype=torch.int32, device=dev)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        _lib.call("gs_best_rows", _lib.stream_handle(dev), rows, None if scores is None else scores.data_ptr(), type,
                  None if act is None else act.data_ptr(), k, ws.data_ptr(), nbytes, out.data_ptr())
    return out

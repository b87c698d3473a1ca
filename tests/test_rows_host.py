"""Rows by an index, the best rows and clipped gradients: what is refused, on the host."""
import ctypes
from array import array

import numpy as np
import pytest
import torch

from jax_gs_amd import _lib
from jax_gs_amd.core.gaussians import Gaussians
from jax_gs_amd.training.adamw import AdamWState, clip_grads_
from jax_gs_amd.training.optimizer import Adam, FIELDS
from jax_gs_amd.training.rows import best_rows, move_rows_, take_rows


def i64(*x):
    return array("q", x).tobytes()


def refused(name, *args):
    assert getattr(_lib.lib(), name)(*args) == 1
    return _lib.lib().gs_last_error().decode()


P = 4096  # an aligned address; nothing is launched


def test_take_rows_entry_refuses():
    def take(num=1, t=i64(P), row=i64(12), stride=i64(12), rows=10, out=i64(P), size=None, index=P, bits=32, count=5):
        return refused("gs_take_rows", None, num, t, row, stride, rows, out, size, None, index, bits, count)

    assert "-1 tensors" in take(num=-1)
    assert "NULL argument" in take(t=None)
    assert "rows by" in take(rows=-1) and "rows by" in take(rows=1 << 31) and "rows by" in take(count=1 << 31)
    assert "32 or 64" in take(bits=16)
    assert "NULL index" in take(index=None)
    assert "not aligned" in take(index=P + 4, bits=64) and "not aligned" in take(index=P + 2)
    assert "rows of -1 bytes" in take(row=i64(-1)) and "bytes" in take(row=i64(1 << 31))
    assert "output 0 of 59 bytes" in take(size=i64(59))
    assert "output 0" in take(size=i64(256), row=i64(0))  # zeros behind rows of nothing
    assert "output 0" in take(size=i64(1 << 37))
    assert "NULL output" in take(out=i64(0)) and "NULL tensor" in take(t=i64(0))
    assert "16-byte aligned" in take(out=i64(P + 8))


def test_move_rows_entry_refuses():
    def move(num=1, t=i64(P), row=i64(12), stride=i64(12), rows=10, index=P, bits=32):
        return refused("gs_move_rows", None, num, t, row, stride, rows, None, index, bits, None)

    assert "-1 tensors" in move(num=-1)
    assert "NULL argument" in move(stride=None)
    assert "rows" in move(rows=-1) and "rows" in move(rows=1 << 31)
    assert "32 or 64" in move(bits=8)
    assert "NULL index" in move(index=None)
    assert "not aligned" in move(index=P + 4, bits=64)
    assert "rows of -4 bytes" in move(row=i64(-4))
    assert "overlap" in move(stride=i64(8)) and "overlap" in move(stride=i64(0))
    assert "NULL tensor" in move(t=i64(0))


def test_moments_take_entry_refuses():
    def take(num=1, lens=i64(3), rows=100, at=i64(0), size=512, m=P, index=P, bits=32, count=80, to=i64(0), out=256, o=P):
        return refused("gs_moments_take", None, num, lens, rows, at, size, m, P, P, index, bits, count, to, out, o, P, P)

    assert "NULL argument" in take(lens=None)
    assert "rows by" in take(rows=-1) and "rows by" in take(count=-1)
    assert "32 or 64" in take(bits=1)
    assert "NULL index" in take(index=None)
    assert "not aligned" in take(index=P + 4, bits=64)
    assert "states of" in take(size=500) and "states of" in take(out=1 << 40)
    assert "NULL state" in take(m=None) and "NULL state" in take(o=None)
    assert "16-byte aligned" in take(m=P + 8) and "16-byte aligned" in take(o=P + 4)
    assert "rows of" in take(lens=i64(1 << 24))
    assert "outside the state" in take(size=256)  # 300 elements
    assert "outside the state" in take(at=i64(1)) and "outside the state" in take(at=i64(-256))
    assert "outside the state" in take(count=90)  # 270 elements in 256
    # the second tensor's moments on the first's
    assert "tensor 1" in take(num=2, lens=i64(3, 1), at=i64(0, 256), size=1024, to=i64(0, 256), out=1024)


def test_moments_move_entry_refuses():
    size = _lib.lib().gs_moments_move_workspace_size
    assert size(0, None, 0) == 0 and size(-1, None, 5) == 0 and size(1, None, 5) == 0 and size(1, i64(3), -1) == 0
    assert size(1, i64(1 << 24), 5) == 0 and size(1, i64(-1), 5) == 0 and size(1, i64(3), 1 << 31) == 0
    # a bit a row, 4 B an element, or with rows of a multiple of sixteen 2 B and 2 for each sixteen
    assert size(2, i64(3, 48), 1000) >= 125 + 12 * 1000 + (2 * 48 + 6) * 1000

    def move(num=1, lens=i64(3), rows=100, at=i64(0), state=512, m=P, index=P, bits=32, ws=P, nbytes=1 << 20):
        return refused("gs_moments_move", None, num, lens, rows, at, state, m, P, P, index, bits, ws, nbytes)

    assert "NULL argument" in move(at=None)
    assert "rows" in move(rows=-1)
    assert "32 or 64" in move(bits=0)
    assert "NULL index" in move(index=None)
    assert "state of" in move(state=511)
    assert "NULL state" in move(m=None) and "NULL state" in move(ws=None)
    assert "16-byte aligned" in move(ws=P + 8)
    assert "workspace of" in move(nbytes=size(1, i64(3), 100) - 1)
    assert "outside the state" in move(rows=200)


def test_best_rows_entry_refuses():
    def best(rows=100, scores=P, type=0, k=5, ws=P, nbytes=1 << 20, out=P):
        return refused("gs_best_rows", None, rows, scores, type, None, k, ws, nbytes, out)

    assert "rows" in best(rows=-1) and "rows" in best(rows=1 << 31)
    assert "best -1" in best(k=-1) and "best" in best(k=1 << 31)
    assert "type 3" in best(type=3)
    assert "not aligned" in best(scores=P + 2) and "not aligned" in best(scores=P + 1, type=1)
    assert "NULL" in best(out=None) and "NULL" in best(ws=None)
    assert "workspace of" in best(nbytes=_lib.lib().gs_best_rows_workspace_size(100) - 1)
    assert "4-byte aligned" in best(ws=P + 2)
    assert _lib.lib().gs_best_rows(None, 100, P, 0, None, 0, None, 0, None) == 0  # nothing to find


def test_clip_entry_refuses():
    counts, types = i64(10), array("i", [0]).tobytes()

    def clip(max_norm=1.0, at=P, types=types, ws=P, nbytes=1 << 20):
        return refused("gs_clip_grads", None, 1, i64(at), types, counts, None, None, 0, max_norm, None, ws, nbytes, None, P)

    for bad in (0.0, -1.0, float("nan")):
        assert "must be positive" in clip(max_norm=bad)
    assert "not aligned" in clip(at=P + 2)
    assert "type of tensor 0" in clip(types=array("i", [3]).tobytes())
    assert "workspace of" in clip(nbytes=8) and "NULL" in clip(ws=None)


def test_densify_sources_entry_refuses():
    need = _lib.lib().gs_densify_workspace_size(1000)
    assert "capacity" in refused("gs_densify_sources", None, 0, P, need, None, P)
    assert "NULL" in refused("gs_densify_sources", None, 1000, None, need, None, P)
    assert "NULL" in refused("gs_densify_sources", None, 1000, P, need, None, None)
    assert "workspace of" in refused("gs_densify_sources", None, 1000, P, need - 1, None, P)


def test_public_calls_refuse_host_tensors():
    x, index = torch.zeros(4, 3), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: take_rows(x, index), lambda: move_rows_([x], index), lambda: best_rows(x[:, 0], 2),
                 lambda: clip_grads_([x], 1.0)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="no tensors"):
        take_rows([], index)
    with pytest.raises(ValueError, match="no tensors"):
        move_rows_({}, index)
    with pytest.raises(ValueError, match="no gradients"):
        clip_grads_([None, None], 1.0)
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="positive"):
            clip_grads_([x], bad)
        with pytest.raises(ValueError, match="positive"):
            Adam({f: 0.1 for f in FIELDS}, max_grad_norm=bad)
    with pytest.raises(ValueError, match="-1 rows"):
        best_rows(x[:, 0], -1)
    with pytest.raises(ValueError, match="scores or a mask"):
        best_rows(None, 2)


def values(b):
    return list(array("q", b))


def test_rows_of_a_list_are_looked_over():
    take, move, dense = _lib.tensors().take, _lib.tensors().move, _lib.tensors().dense
    index = torch.zeros(6, dtype=torch.int32)
    a = torch.zeros(6, 5, dtype=torch.float16)
    big = torch.zeros(6, 8, 4)
    # a slice of every row: strides stay, nothing is copied
    pointers, row_bytes, strides, rows, fills, out, new, kept = take([a, big[:, 2:5]], None, 9, -1, "take_rows")
    assert values(row_bytes) == [10, 48] and values(strides) == [10, 128] and rows == 6 and values(fills) == [0, 0]
    assert values(pointers) == [a.data_ptr(), big.data_ptr() + 2 * 4 * 4] and kept is None
    assert [x.shape for x in new] == [(9, 5), (9, 3, 4)] and new[0].dtype == torch.float16 and new[1].is_contiguous()
    assert values(out) == [x.data_ptr() for x in new]
    # rows that are not contiguous are copied, in place refused; an expanded row is read as it is
    t = big.transpose(1, 2)
    pointers, row_bytes, strides, _, _, _, _, kept = take([t, a[:1].expand(6, 5)], None, 1, -1, "take_rows")
    assert len(kept) == 1 and kept[0].is_contiguous() and values(strides) == [128, 0]
    for bad in (t, a[:1].expand(6, 5), torch.imag(torch.zeros(6, 5, dtype=torch.complex64).conj())):
        with pytest.raises(ValueError, match="contiguous"):
            move([bad], None, index, -1, "move_rows_")
    with pytest.raises(ValueError, match="7 rows, not 6"):
        take([a, torch.zeros(7)], None, 1, -1, "take_rows")
    with pytest.raises(ValueError, match="no rows"):
        take([torch.zeros(())], None, 1, -1, "take_rows")
    with pytest.raises(TypeError, match="strided"):
        take([torch.zeros(6, 5).to_sparse()], None, 1, -1, "take_rows")
    with pytest.raises(TypeError, match="not a tensor"):
        take([None], None, 1, -1, "take_rows")
    with pytest.raises(ValueError, match="is on cpu"):
        take([a], None, 1, 0, "take_rows")
    leaf = torch.zeros(6, 5, requires_grad=True)
    for call in (lambda: take([leaf], None, 1, -1, "x"), lambda: move([leaf], None, index, -1, "x"),
                 lambda: dense([leaf], -1, "x", False)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad():
            call()


def test_no_memory_is_an_error_of_its_kind():
    """2^31 rows of 2^31 bytes: the allocator's own error, not a process that ends."""
    with pytest.raises(RuntimeError, match="[Mm]emory|alloc"):
        _lib.tensors().take([torch.zeros(1, 1 << 20).expand(1, 1 << 20)], None, 1 << 38, -1, "take_rows")


def test_overlapping_rows_are_refused():
    move, dense = _lib.tensors().move, _lib.tensors().dense
    index = torch.zeros(6, dtype=torch.int32)
    pool = torch.zeros(6, 2, 4)
    # two halves of every page lie between each other and are apart
    move([pool[:, 0], pool[:, 1]], None, index, -1, "move_rows_")
    move([pool[:, 1], pool[:, 0]], None, index, -1, "move_rows_")
    for bad in ([pool, pool], [pool, pool[:, 1]], [pool[:, 0, :3], pool[:, 0, 2:]], [pool[:, 0], pool[:, 0]],
                [pool.view(12, 4)[:6], pool[:, 1]]):
        with pytest.raises(ValueError, match="overlap"):
            move(bad, None, index, -1, "move_rows_")
    flat = torch.zeros(100)
    dense([flat[:50], None, flat[50:]], -1, "clip_grads_", False)
    for bad in ([flat, flat], [flat[:60], flat[50:]]):
        with pytest.raises(ValueError, match="overlap"):
            dense(bad, -1, "clip_grads_", False)
    # what a move reads besides its rows
    ints = torch.zeros(12, dtype=torch.int32)
    with pytest.raises(ValueError, match="index and the fills"):
        move([ints.view(6, 2)], None, ints[:6], -1, "move_rows_")
    with pytest.raises(ValueError, match="index and the fills"):
        move([pool], [pool[0]], index, -1, "move_rows_")
    move([pool[:, 0]], [torch.zeros(4)], index, -1, "move_rows_")


def test_fills_are_rows_of_their_tensors():
    take = _lib.tensors().take
    a, b = torch.zeros(6, 3), torch.zeros(6, dtype=torch.int64)
    fill = torch.ones(3)
    assert values(take([a, b], [fill, None], 2, -1, "take_rows")[4]) == [fill.data_ptr(), 0]
    assert values(take([b], [torch.tensor(7)], 2, -1, "take_rows")[4])[0]
    assert len(take([a], [torch.zeros(3, 2)[:, 0]], 2, -1, "take_rows")[7]) == 1  # strided: copied
    for bad in ([torch.ones(3)], [torch.ones(3), None, None]):
        with pytest.raises(ValueError, match="one fill"):
            take([a, b], bad, 2, -1, "take_rows")
    for bad in (torch.ones(4), torch.ones(1, 3), torch.ones(3, dtype=torch.float64)):
        with pytest.raises(ValueError, match="fill 0 must be one row"):
            take([a], [bad], 2, -1, "take_rows")


def test_gradients_in_place_are_dense():
    dense = _lib.tensors().dense
    last = torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last)
    pointers, types, counts = dense([last, torch.zeros(3, dtype=torch.bfloat16)], -1, "clip_grads_", False)
    assert values(counts) == [120, 3] and list(array("i", types)) == [0, 1]
    with pytest.raises(ValueError, match="contiguous"):
        dense([last], -1, "clip_grads_", True)
    for bad in (torch.zeros(4, 4)[:, :2], torch.zeros(4).expand(3, 4)):
        with pytest.raises(ValueError, match="dense"):
            dense([bad], -1, "clip_grads_", False)
    with pytest.raises(TypeError, match="float64"):
        dense([torch.zeros(3, dtype=torch.float64)], -1, "clip_grads_", False)


def test_states_of_different_rows_have_no_rows():
    for shapes in (((300,), (7,)), ((300, 2), ())):
        with pytest.raises(ValueError, match="same rows"):
            AdamWState(None, shapes, 32)._rows("take_rows")
    rows, lens, *_ = AdamWState(None, ((5, 2, 3), (5,), (5, 0)), 8)._rows("take_rows")
    assert rows == 5 and lens == [6, 1, 0]


def exact(d, magic, largest):
    """Whether the upper half of e * magic is e // d for all e up to the largest."""
    e = np.arange(largest + 1, dtype=np.uint64)
    return np.array_equal((e * np.uint64(magic)) >> np.uint64(32), e // np.uint64(d))


def test_reciprocals_are_exact_where_they_are_used():
    """floor(2^32 / d) + 1 in place of a division: rows of up to 8192 bytes with offsets below a row and a workgroup's 8192;
    up to 256 rows by up to 512 pieces of all tensors, 64 rows by up to 4096 pieces of one, rows by rows that move;
    moments' rows of up to 4096 elements, where it is the upper half of floor(2^64 / d) + 1, plus 1."""
    plain = lambda d: (1 << 32) // d + 1
    for d in [*range(2, 260), *range(260, 8193, 37), 4095, 4096, 4097, 8191, 8192]:
        assert exact(d, plain(d), d + 8192), d
    for m in range(2, 257):
        assert exact(m, 0xFFFFFFFF // m + 1, m * 512 - 1), m
    for pieces in [*range(2, 513, 7), 511, 512]:
        assert exact(pieces, plain(pieces), 256 * pieces - 1), pieces
    for pieces in [*range(2, 4097, 61), 4095, 4096]:
        assert exact(pieces, 0xFFFFFFFF // pieces + 1, 64 * pieces - 1), pieces
    for d in [*range(2, 4097, 13), 4095, 4096]:
        assert exact(d, (((1 << 64) // d + 1 if d & (d - 1) else (1 << 64) // d + 0) >> 32) + 1, d + 256), d

"""Refusals of the AdamW entry points and the format of 8-bit moments, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

import adamw_reference as ref
from jax_gs_amd import _lib
from jax_gs_amd.training.adamw import AdamW, AdamWState, grad_norms

I64, P, I, D = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_double


def step_args(**change):
    """Arguments of gs_adamw_step for one tensor of 300 elements at addresses that are not read."""
    a = dict(stream=None, num=1, params=(P * 1)(4096), ptypes=(I * 1)(0), grads=(P * 1)(8192), gtypes=(I * 1)(0),
             offsets=(I64 * 1)(0), counts=(I64 * 1)(300), row_lens=(I64 * 1)(3), lrs=(D * 1)(0.1), decays=(D * 1)(0.0),
             bits=32, size=512, mu=P(4096), nu=P(8192), fields=P(4096), master=None, active=None, rows=0, scale=None,
             powers=P(64), nxt=P(128), b1=0.9, b2=0.999, eps=1e-8, key=1)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, words", [
    (dict(num=-1), b"tensors"),
    (dict(params=None), b"NULL"),
    (dict(bits=16), b"32 or 8 bits"),
    (dict(size=500), b"state of 500"),
    (dict(mu=None), b"NULL state"),
    (dict(bits=8, fields=None), b"NULL state"),
    (dict(nu=P(8196)), b"aligned"),
    (dict(nxt=P(64)), b"powers"),
    (dict(b1=1.0), b"b1"),
    (dict(b2=-0.1), b"b1"),
    (dict(eps=-1.0), b"eps"),
    (dict(ptypes=(I * 1)(3)), b"type"),
    (dict(gtypes=(I * 1)(-1)), b"type"),
    (dict(counts=(I64 * 1)(-1)), b"elements"),
    (dict(counts=(I64 * 1)(1 << 41)), b"elements"),
    (dict(counts=(I64 * 1)(513)), b"outside the state"),
    (dict(offsets=(I64 * 1)(100)), b"outside the state"),
    (dict(offsets=(I64 * 1)(512)), b"outside the state"),
    (dict(params=(P * 1)(0)), b"NULL tensor"),
    (dict(params=(P * 1)(4098)), b"aligned to its type"),
    (dict(grads=(P * 1)(8193), gtypes=(I * 1)(1)), b"aligned to its type"),
    (dict(active=P(64), rows=100, row_lens=None), b"row lengths"),
    (dict(active=P(64), rows=99), b"rows x row length"),
    (dict(active=P(64), rows=300, row_lens=(I64 * 1)(0)), b"rows x row length"),
])
def test_step_refusals(change, words):
    L = _lib.lib()
    assert L.gs_adamw_step(*step_args(**change)) == 1
    assert words in L.gs_last_error(), L.gs_last_error()


def test_step_refuses_moments_that_overlap():
    L = _lib.lib()
    two = dict(num=2, params=(P * 2)(4096, 8192), ptypes=(I * 2)(), grads=(P * 2)(4096, 8192), gtypes=(I * 2)(),
               counts=(I64 * 2)(300, 100), row_lens=None, lrs=(D * 2)(), decays=(D * 2)(), size=1024)
    for offsets in ((0, 256), (256, 0), (512, 512)):
        assert L.gs_adamw_step(*step_args(offsets=(I64 * 2)(*offsets), **two)) == 1
        assert b"do not lie behind" in L.gs_last_error()


@pytest.mark.parametrize("change, words", [
    (dict(num=-1), b"tensors"), (dict(grads=None), b"NULL"), (dict(out=None), b"NULL"), (dict(ws=None), b"NULL"),
    (dict(nbytes=8), b"workspace"), (dict(ws=P(68)), b"8-byte"), (dict(gtypes=(I * 1)(7)), b"type"),
    (dict(grads=(P * 1)(4097)), b"aligned"), (dict(counts=(I64 * 1)(-3)), b"elements"),
    (dict(max_norm=float("nan")), b"not a number"), (dict(active=P(64), rows=7), b"rows x row length"),
    (dict(active=P(64), rows=100, row_lens=None), b"row lengths"),
])
def test_norm_refusals(change, words):
    L = _lib.lib()
    a = dict(stream=None, num=1, grads=(P * 1)(4096), gtypes=(I * 1)(0), counts=(I64 * 1)(300), row_lens=(I64 * 1)(3),
             active=None, rows=0, max_norm=1.0, scale=None, ws=P(64), nbytes=1 << 20, norms=None, out=P(64))
    a.update(change)
    assert L.gs_grad_norms(*a.values()) == 1
    assert words in L.gs_last_error(), L.gs_last_error()


def test_conversion_refusals_and_sizes():
    L = _lib.lib()
    some = [P(4096)] * 5
    assert L.gs_moments_encode(None, 100, *some) == 1 and b"state of 100" in L.gs_last_error()
    assert L.gs_moments_decode(None, 256, P(4096), None, *some[:3]) == 1 and b"NULL" in L.gs_last_error()
    assert L.gs_moments_encode(None, 256, P(4100), *some[:4]) == 1 and b"aligned" in L.gs_last_error()
    assert L.gs_moments_encode(None, 0, *[None] * 5) == 0 and L.gs_moments_decode(None, 0, *[None] * 5) == 0
    assert L.gs_grad_norms_workspace_size(2, (I64 * 2)(5, -1)) == 0
    assert L.gs_grad_norms_workspace_size(-1, None) == 0
    assert 0 < L.gs_grad_norms_workspace_size(1, (I64 * 1)(5)) < L.gs_grad_norms_workspace_size(1, (I64 * 1)(10 ** 9))


@pytest.mark.parametrize("options", [dict(moment_bits=16), dict(b1=1.0), dict(b2=-1e-3), dict(eps=-1.0),
                                     dict(eps=float("nan")), dict(max_grad_norm=0.0)])
def test_optimizer_refusals(options):
    with pytest.raises(ValueError, match="AdamW"):
        AdamW(1e-3, **options)


def test_there_is_no_cpu_path():
    with pytest.raises(ValueError, match="GPU"):
        AdamW(1e-3).init(torch.zeros(3))
    with pytest.raises(ValueError, match="GPU"):
        grad_norms([torch.zeros(3)])
    with pytest.raises(ValueError, match="no parameters"):
        AdamW(1e-3).init([])


def test_layout_of_the_state():
    s = AdamWState(None, [(3,), (0, 4), (256,), (257,), ()], 8)
    assert s.counts == [3, 0, 256, 257, 1] and s.offsets == [0, 256, 256, 512, 1024] and s.size == 1280


def test_held_values_of_the_reference():
    """The restatement that the GPU tests compare with: steps, range, ties and the largest codes."""
    x = np.zeros(256)
    x[:9] = [1.75, 1.0625, 1.1875, 1.06, -1.07, 2.0 ** -14, 2.0 ** -17, 2.0 ** -18, 1.1 * 2.0 ** -18]
    got, _ = ref.held(x, 3)
    assert list(got[:9]) == [1.75, 1.0, 1.25, 1.0, -1.125, 2.0 ** -14, 2.0 ** -17, 0.0, 2.0 ** -17]
    x[0] = 1.76  # above the largest code: the block's exponent grows, gradual underflow with it
    assert list(ref.held(x, 3)[0][[0, 6]]) == [1.75, 0.0]
    got, _ = ref.held(np.r_[1.875, 1e-9, np.zeros(254)], 4)
    assert list(got[:3]) == [1.875, 2.0 ** -18, 0.0]
    a, b = ref.noise(np.arange(1 << 16), 3, 4)
    assert abs(a.mean() - 0.5) < 0.01 and abs(b.mean() - 0.5) < 0.01 and abs(np.corrcoef(a, b)[0, 1]) < 0.02
    up, _ = ref.held(np.full(1 << 16, 1.03125), 3, a)
    assert abs(up.mean() - 1.03125) < 5 * 0.125 * 0.43 / 256

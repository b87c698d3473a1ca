"""AdamW's kernels for long arrays against float64: tensors of several launch records.

Tolerances as in test_gpu_adamw.py, with e = 2^-24: m and v 8 e of the terms that they are sums of,
w 4 e |w| + 24 e of the update."""
import numpy as np
import pytest
import torch

import adamw_reference as ref
from jax_gs_amd.training.adamw import AdamW

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_of_several_records_under_a_mask(cuda, bits):
    """2^31 + 1281 elements are three records of one launch.  Everywhere: the first step from zero weights and
    moments moves an unmasked weight whose gradient is not zero by the rate, the others not at all.  Around the
    records' ends and at the end: the reference."""
    row = 13
    rows = ((1 << 31) + 1281) // row
    n = rows * row
    gen = torch.Generator(device=cuda).manual_seed(1)
    g = torch.randn(rows, row, dtype=torch.bfloat16, generator=gen, device=cuda)
    on = torch.rand(rows, generator=gen, device=cuda) < 0.75
    p = torch.zeros(rows, row, dtype=torch.bfloat16, device=cuda)
    opt = AdamW(0.5, eps=1e-12, moment_bits=bits, seed=9)
    state = opt.init([p])
    opt.step([p], [g], state, active_mask=on)
    lo, hi = 0.5 - 2.0 ** -9, 0.5 + 2.0 ** -8  # one step of bfloat16 around the rate
    for i in range(0, rows, 1 << 24):
        q, gi = p[i:i + (1 << 24)].abs(), g[i:i + (1 << 24)]
        moved = on[i:i + (1 << 24), None] & (gi != 0)
        assert bool(torch.where(moved, (q >= lo) & (q <= hi) & (torch.sign(p[i:i + (1 << 24)]) == -torch.sign(gi)), q == 0).all())
    flat, grads = p.view(-1), g.view(-1)
    for at in (0, 1 << 30, 1 << 31, n):  # whole blocks around the place
        a, b = max(at - 1024, 0) // 256 * 256, min(at + 1024, n)
        every = np64(on[a // row:-(-b // row)]).repeat(row)[a - a // row * row:][:b - a] > 0
        w, m, v, size = ref.step(np.zeros(b - a), np64(grads[a:b]), np.zeros(b - a), np.zeros(b - a), 1, 0.5, eps=1e-12, on=every)
        if bits == 32:
            got_m, got_v = np64(state.mu_flat[a:b]), np64(state.nu_flat[a:b])
            assert np.all(np.abs(got_m - m) <= 8 * E * size) and np.all(np.abs(got_v - v) <= 8 * E * v)
        else:
            um, ur = ref.noise(np.arange(a, a + len(ref.pad(m))), 9, 1)
            mu, nu = decoded(state, a, b)
            for got, x, mant, u in ((mu, m, 3, um), (np.sqrt(nu), np.sqrt(v), 4, ur)):
                value, near = ref.held(ref.pad(x), mant, u)
                same = got == value[:b - a]
                assert np.all(same | (near[:b - a] < 1e-4)) and np.count_nonzero(~same) <= 1e-3 * len(same) + 1


def decoded(state, a, b):
    """Moments of a short run of an 8-bit state, by way of a state of those blocks alone."""
    import copy

    part = copy.copy(state)
    e = -(-b // 256) * 256
    part.mu_flat, part.nu_flat = state.mu_flat[a:e].clone(), state.nu_flat[a:e].clone()
    part.fields = state.fields[a // 256:e // 256].clone()
    part.size, part.counts, part.offsets, part.shapes = e - a, [e - a], [0], [torch.Size((e - a,))]
    return tuple(np64(x[0])[:b - a] for x in part.moments())

"""AdamW over many tensors with moments in 32 and in 8 bits, against float64.

Tolerances, with e = 2^-24 (half a step of float32):
  m    three roundings a step and the rounded coefficients, each relative to the terms that m is
       the sum of: 8 e per step made, of the largest such size so far.
  v    a sum of terms that are not negative: 8 e relative per step.
  w    its own rounding and that of decay * w: 4 e |w|; the update's: m's error, root, division
       and products, 24 e of lr (size / (1 - b1^t)) / (sqrt(v) / sqrt(1 - b2^t)) per step made.
  half types: the value of theirs nearest to some number within the tolerance for w.
  8 bits: the value held of the float64 result, except where that is within 1e-4 steps of being
       rounded the other way (a float32 error of 8 e in up to 32 steps is 2e-5), where one step
       is allowed."""
import ctypes

import numpy as np
import pytest
import torch

import adamw_reference as ref
from jax_gs_amd.core.gaussians import Gaussians
from jax_gs_amd.training.adamw import AdamW, AdamWState, grad_norms, make_adamw

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = [0, 1, 2, 3, 5, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 2048, 4099]


def np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def rows_like(rng, n):
    """Gradients whose size changes over orders of magnitude, many of them zero."""
    size = np.exp(rng.normal(-7, 2, -(-max(n, 1) // 16))).repeat(16)[:n]
    return (rng.normal(0, 1, n) * size * (rng.random(n) < 0.7)).astype(np.float32)


def tensors(cuda, arrays, dtype, apart=False):
    """The arrays as tensors of the type; `apart`: views into one buffer, one element between."""
    if not apart:
        return [torch.tensor(a, device=cuda).to(dtype) for a in arrays]
    flat = torch.zeros(sum(len(a) + 1 for a in arrays), dtype=dtype, device=cuda)
    out, at = [], 0
    for a in arrays:
        at += 1
        flat[at:at + len(a)] = torch.tensor(a, device=cuda).to(dtype)
        out.append(flat[at:at + len(a)])
        at += len(a)
    return out


def weights_close(got, want, tol, kind):
    """Float32 weights within tol; half weights between the rounded ends of that range."""
    lo, hi = (torch.tensor(x).to(TYPES[kind]).to(torch.float64).numpy() for x in (want - tol, want + tol))
    if kind == "f32":
        lo, hi = want - tol, want + tol
    assert np.all((lo <= got) & (got <= hi))


def check32(got, want, w_size, m_size, kind, t):
    """One tensor's (w, m, v) against the reference's (w, m, v)."""
    (w, m, v), (wr, mr, vr) = got, want
    assert np.all(np.abs(m - mr) <= 8 * E * t * m_size + 1e-44)
    assert np.all(np.abs(v - vr) <= 8 * E * t * vr + 1e-44)
    weights_close(w, wr, t * (4 * E * np.abs(wr) + 24 * E * w_size), kind)


def run32(cuda, sizes, param, grad, master, decay, apart, steps=3, bits=32, on=None, rows=None):
    rng = np.random.default_rng(len(sizes) * 7 + steps)
    w0 = [rng.normal(0, 1, n).astype(np.float32) for n in sizes]
    ps = tensors(cuda, w0, TYPES[param], apart)
    opt = AdamW([1e-2 + 1e-3 * i for i in range(len(sizes))], weight_decay=decay, master_weights=master)
    if rows is not None:
        ps = [p.view(rows, -1) for p in ps]
    state = opt.init(ps)
    refs = [(np64(p).reshape(-1), np.zeros(n), np.zeros(n)) for p, n in zip(ps, sizes)]
    m_size, w_size = [np.zeros(n) for n in sizes], [np.zeros(n) for n in sizes]
    mask = None if on is None else torch.tensor(on, device=cuda)
    for t in range(1, steps + 1):
        gs = tensors(cuda, [rows_like(rng, n) for n in sizes], TYPES[grad], apart)
        if rows is not None:
            gs = [g.view(rows, -1) for g in gs]
        opt.step(ps, gs, state, active_mask=mask)
        for i, n in enumerate(sizes):
            every = None if on is None else np.repeat(on, n // rows)
            w, m, v, size = ref.step(refs[i][0], np64(gs[i]).reshape(-1), refs[i][1], refs[i][2], t, 1e-2 + 1e-3 * i,
                                     decay=decay, on=every)
            m_size[i] = np.maximum(m_size[i], size)
            with np.errstate(divide="ignore", invalid="ignore"):
                unit = np.nan_to_num(m_size[i] / (1 - 0.9 ** t) / np.sqrt(v / (1 - 0.999 ** t)), posinf=0.0)
            w_size[i] = np.maximum(w_size[i], (1e-2 + 1e-3 * i) * unit)
            refs[i] = (w, m, v)
            kind = param
            if master and param != "f32":
                full = np64(state.master[i]).reshape(-1)
                check32((full, np64(state.mu[i]).reshape(-1), np64(state.nu[i]).reshape(-1)), refs[i], w_size[i],
                        m_size[i], "f32", t)
                # the tensor is the master, rounded once
                assert torch.equal(ps[i].reshape(-1), state.master[i].reshape(-1).to(TYPES[param]))
            else:
                check32((np64(ps[i]).reshape(-1), np64(state.mu[i]).reshape(-1), np64(state.nu[i]).reshape(-1)),
                        refs[i], w_size[i], m_size[i], kind, t)
                if kind != "f32":  # the next step starts from the rounded weights
                    refs[i] = (np64(ps[i]).reshape(-1), m, v)
    assert state.count == steps
    # what lies between the tensors stays zero
    used = torch.zeros(state.size, dtype=torch.bool)
    for o, n in zip(state.offsets, state.counts):
        used[o:o + n] = True
    for flat in (state.mu_flat, state.nu_flat):
        assert not flat.cpu()[~used].any()


@pytest.mark.parametrize("param, grad, master", [("f32", "f32", False), ("f32", "bf16", False), ("f32", "f16", False),
                                                 ("bf16", "bf16", False), ("bf16", "bf16", True),
                                                 ("bf16", "f32", True), ("bf16", "f16", False), ("bf16", "f16", True),
                                                 ("bf16", "f32", False), ("f16", "f16", False), ("f16", "f16", True),
                                                 ("f16", "f32", False), ("f16", "f32", True), ("f16", "bf16", False),
                                                 ("f16", "bf16", True)])
@pytest.mark.parametrize("apart", [False, True])
def test_step_in_32_bits(cuda, param, grad, master, apart):
    run32(cuda, SIZES, param, grad, master, 0.1, apart)


def test_step_over_more_tensors_than_a_launch_takes(cuda):
    rng = np.random.default_rng(3)
    run32(cuda, [int(n) for n in rng.integers(0, 700, 131)], "f32", "f32", False, 0.01, True)


@pytest.mark.parametrize("rows, lens", [(1, [1, 7]), (37, [3, 3, 4, 1, 48]), (3, [5000, 4097, 300]), (1000, [64, 65, 9])])
@pytest.mark.parametrize("share", [0.0, 0.5, 1.0])
def test_step_with_a_row_mask(cuda, rows, lens, share):
    on = np.random.default_rng(5).random(rows) < share
    run32(cuda, [rows * n for n in lens], "f32", "f32", False, 0.1, False, on=on, rows=rows)


def test_first_step_is_the_sign_of_the_gradient(cuda):
    """Closed form: with zero moments the update is lr g / (|g| + eps)."""
    g = torch.tensor([3.0, -0.5, 1e-3, 0.0], device=cuda)
    p = torch.zeros(4, device=cuda)
    opt = AdamW(0.1)
    opt.step(p, g, opt.init(p))
    np.testing.assert_allclose(np64(p), [-0.1, 0.1, -0.1 / (1 + 1e-5), 0.0], rtol=1e-6)


def held_close(got, want, near, step):
    """`got` is the held value, or within one step of it where the rounding was that near."""
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    assert np.all(same | ((near < 1e-4) & (np.abs(got - want) <= step))), (got[~same][:5], want[~same][:5], near[~same][:5])
    assert np.count_nonzero(~same) <= 1e-3 * len(same)


def check8(state, i, m, v, t, seed=0):
    """Tensor i's moments after update t against what 8 bits hold of the reference's."""
    n, o = state.counts[i], state.offsets[i]
    um, ur = ref.noise(np.arange(o, o + len(ref.pad(m))), seed, t)
    for got, x, mant, u in ((np64(state.moments()[0][i]), m, 3, um), (np.sqrt(np64(state.moments()[1][i])), np.sqrt(v), 4, ur)):
        value, near = ref.held(ref.pad(x), mant, u)
        step = np.maximum(np.abs(value), np.abs(value).reshape(-1, 256).max(1).repeat(256) * 2.0 ** -13) * 2.0 ** -mant
        held_close(got.reshape(-1), value[:n], near[:n], step[:n])


@pytest.mark.parametrize("param, grad, master", [("f32", "f32", False), ("f32", "bf16", False), ("bf16", "bf16", True),
                                                 ("bf16", "f32", False), ("f16", "f16", True), ("f16", "f16", False)])
@pytest.mark.parametrize("apart", [False, True])
def test_step_in_8_bits(cuda, param, grad, master, apart):
    rng = np.random.default_rng(11)
    sizes = SIZES + [30000]
    ps = tensors(cuda, [rng.normal(0, 1, n).astype(np.float32) for n in sizes], TYPES[param], apart)
    opt = AdamW(1e-2, weight_decay=0.1, moment_bits=8, master_weights=master, seed=77)
    state = opt.init(ps)
    for t in range(1, 5):
        gs = tensors(cuda, [rows_like(rng, n) for n in sizes], TYPES[grad], apart)
        before = [(np64(state.master[i] if state.master_flat is not None else p).reshape(-1), np64(m).reshape(-1), np64(v).reshape(-1))
                  for i, (p, m, v) in enumerate(zip(ps, *state.moments()))]
        opt.step(ps, gs, state)
        for i, n in enumerate(sizes):
            w, m, v, size = ref.step(before[i][0], np64(gs[i]), before[i][1], before[i][2], t, 1e-2, decay=0.1)
            check8(state, i, m, v, t, 77)
            with np.errstate(divide="ignore", invalid="ignore"):
                unit = np.nan_to_num(size / (1 - 0.9 ** t) / np.sqrt(v / (1 - 0.999 ** t)), posinf=0.0)
            got = np64(state.master[i] if state.master_flat is not None else ps[i]).reshape(-1)
            weights_close(got, w, 4 * E * np.abs(w) + 24 * E * 1e-2 * unit, "f32" if master else param)
    for flat in (state.mu_flat, state.nu_flat):  # between the tensors: zero
        used = torch.zeros(state.size, dtype=torch.bool)
        for o, n in zip(state.offsets, state.counts):
            used[o:o + n] = True
        assert not flat.cpu()[~used].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_scale_that_is_not_finite_changes_nothing(cuda, bits):
    rng = np.random.default_rng(2)
    make = lambda: [torch.tensor(rng.normal(0, 1, n).astype(np.float32), device=cuda) for n in (5, 3000)]  # noqa: E731
    ps, grads = make(), [make() for _ in range(3)]
    qs = [p.clone() for p in ps]
    opt = AdamW(1e-2, weight_decay=0.1, moment_bits=bits)
    a, b = opt.init(ps), opt.init(qs)
    opt.step(ps, grads[0], a)
    opt.step(qs, grads[0], b)
    for bad in (float("nan"), float("inf"), -float("inf")):
        keep = [x.clone() for x in (*ps, a.mu_flat, a.nu_flat, a.powers)]
        opt.step(ps, grads[1], a, grad_scale=torch.full((), bad, device=cuda))
        for x, y in zip(keep, (*ps, a.mu_flat, a.nu_flat, a.powers)):
            assert torch.equal(x, y)
    assert a.count == 4
    b.count = 4  # the rounding's random bits follow the count
    opt.step(ps, grads[2], a)
    opt.step(qs, grads[2], b)
    for x, y in zip((*ps, a.mu_flat, a.nu_flat, a.powers), (*qs, b.mu_flat, b.nu_flat, b.powers)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [32, 8])
def test_masked_rows_are_not_read_into_anything(cuda, bits):
    """NaN and infinities in masked rows' gradients: the same bits as with zeros there."""
    rng = np.random.default_rng(4)
    n = 777
    on = torch.tensor(rng.random(n) < 0.6, device=cuda)
    ps = [torch.tensor(rng.normal(0, 1, (n, k)).astype(np.float32), device=cuda) for k in (3, 48)]
    qs = [p.clone() for p in ps]
    g0 = [torch.tensor(rng.normal(0, 1, (n, k)).astype(np.float32), device=cuda) * on[:, None] for k in (3, 48)]
    g1 = [g.clone() for g in g0]
    for g in g1:
        off = (~on).nonzero().flatten()
        g[off[0::3]] = float("nan")
        g[off[1::3]] = float("inf")
        g[off[2::3]] = -3e38
    opt = AdamW(1e-2, weight_decay=0.1, moment_bits=bits, max_grad_norm=0.5)
    a, b = opt.init(ps), opt.init(qs)
    start = [p.clone() for p in ps]
    for _ in range(2):
        opt.step(ps, g0, a, active_mask=on)
        opt.step(qs, g1, b, active_mask=on)
    assert torch.isfinite(b.norms.total)
    for x, y in zip((*ps, a.mu_flat, a.nu_flat), (*qs, b.mu_flat, b.nu_flat)):
        assert torch.equal(x, y)
    for p, s in zip(ps, start):
        assert torch.equal(p[~on], s[~on]) and not torch.equal(p[on], s[on])


def test_values_that_are_not_finite_stay_where_they_are_in_8_bits(cuda):
    rng = np.random.default_rng(6)
    g = torch.tensor(rng.normal(0, 1, 1024).astype(np.float32), device=cuda)
    bad = g.clone()
    where = [3, 256, 511, 1000]
    bad[where] = torch.tensor([float("nan"), float("inf"), -float("inf"), float("nan")], device=cuda)
    zeroed = g.clone()
    zeroed[where] = 0.0
    opt = AdamW(1e-2, moment_bits=8)
    ps = [torch.ones(1024, device=cuda) for _ in range(2)]
    states = [opt.init(p) for p in ps]
    for _ in range(3):
        for p, gr, s in zip(ps, (bad, zeroed), states):
            opt.step(p, gr, s)
    rest = torch.ones(1024, dtype=torch.bool, device=cuda)
    rest[where] = False
    for x, y in zip((ps[0], *[m[0] for m in states[0].moments()]), (ps[1], *[m[0] for m in states[1].moments()])):
        assert torch.equal(x[rest], y[rest])
        assert torch.isnan(x[~rest]).all()


def test_gradients_that_are_not_contiguous_or_missing(cuda):
    rng = np.random.default_rng(8)
    T = lambda *s: torch.tensor(rng.normal(0, 1, s).astype(np.float32), device=cuda)  # noqa: E731
    ps = [T(5, 7), T(4, 4), T(3, 6), T(9)]
    qs = [p.clone() for p in ps]
    gs = [T(7, 5).t(), torch.ones((), device=cuda).expand(4, 4), T(6, 12)[::2, ::2], None]
    opt = AdamW(1e-2, max_grad_norm=1.0)
    a, b = opt.init(ps), opt.init(qs)
    opt.step(ps, gs, a)
    opt.step(qs[:], [g.contiguous() if g is not None else None for g in gs], b)
    for x, y in zip((*ps, a.mu_flat), (*qs, b.mu_flat)):
        assert torch.equal(x, y)
    total = np.sqrt(sum((np64(g) ** 2).sum() for g in gs if g is not None))
    assert abs(float(a.norms.total) - total) <= 4 * E * total
    assert float(a.norms.per_tensor[3]) == 0.0 and not a.mu[3].any()


def test_gradients_that_are_views_of_complex_values(cuda):
    """The imaginary part of a conjugate: strided, and negated only when it is read."""
    z = torch.randn(600, dtype=torch.complex64, device=cuda)
    g = z.conj().imag
    p, q = torch.ones(600, device=cuda), torch.ones(600, device=cuda)
    opt = AdamW(1e-2)
    opt.step(p, g, opt.init(p))
    opt.step(q, -torch.view_as_real(z)[:, 1].contiguous(), opt.init(q))
    assert torch.equal(p, q)
    want = np.sqrt((np64(z.imag) ** 2).sum())
    assert abs(float(grad_norms(g).total) - want) <= 4 * E * want


def test_step_on_a_stream_of_the_callers(cuda):
    g = torch.randn(100_000, device=cuda)
    p, q = torch.ones(100_000, device=cuda), torch.ones(100_000, device=cuda)
    opt = AdamW(1e-2, moment_bits=8, max_grad_norm=0.1)
    a, b = opt.init(p), opt.init(q)
    opt.step(p, g, a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt.step(q, g, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(p, q) and torch.equal(a.mu_flat, b.mu_flat)


def test_more_than_2_to_the_32_elements(cuda):
    """One bfloat16 tensor of 2^32 + 513 elements in 8 bits: its last blocks, beyond a 32-bit
    offset, are those of a short tensor whose elements have the same places' random bits
    switched off by exact values: gradients and moments that 8 bits hold."""
    n = (1 << 32) + 513
    p = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    g = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    tail = torch.tensor(np.resize([1.0, -0.5, 0.25, 0.0, 2.0], 1025).astype(np.float32), device=cuda).to(torch.bfloat16)
    g[-1025:] = tail
    # b1 0.5, b2 0.75: m = g / 2 and sqrt(v) = |g| / 2 of the first step are held exactly
    opt = AdamW(1.0, b1=0.5, b2=0.75, eps=0.5, moment_bits=8, max_grad_norm=1e6)
    state = opt.init(p)
    opt.step(p, g, state)
    short = torch.zeros(1025, dtype=torch.bfloat16, device=cuda)
    other = opt.init(short)
    opt.step(short, tail, other)
    assert torch.equal(p[-1025:], short)
    assert not p[:1 << 20].any() and not p[(1 << 32) - 70000:(1 << 32) - 512].any()
    want = np.sqrt((np64(tail) ** 2).sum())
    assert abs(float(state.norms.total) - want) <= 4 * E * want
    at = state.offsets[0] + n - 1025
    got = state.mu_flat[at:at + 1025]
    fields = state.fields[(at >> 8):]
    # 2^32 + 513 - 1025 is a multiple of 256: the blocks are the short tensor's
    assert at % 256 == 0 and torch.equal(got, other.mu_flat[:1025]) and torch.equal(fields, other.fields)
    del p, g, state


# ---- conversion -----------------------------------------------------------------------------

def values(rng):
    """Blocks of moments at the ends of the range."""
    blocks = [np.zeros(256), rng.normal(0, 1, 256), rng.normal(0, 1, 256) * np.exp(rng.normal(-10, 8, 256)),
              np.full(256, 1e-45), np.full(256, 3.4028235e38), np.r_[3e38, np.full(255, 1e-38)],
              np.r_[np.zeros(255), 1.0], np.r_[1.75, np.full(255, 1.0 / 3)], np.r_[1.7500001, np.full(255, 1.0 / 3)],
              np.r_[1.875, np.full(255, 0.1)], np.r_[1.8750001, np.full(255, 0.1)], 2.0 ** np.arange(0, -256, -1.0),
              rng.normal(0, 1, 256) * 1e-38, rng.normal(0, 1e-41, 256), np.r_[np.nan, np.inf, -np.inf, rng.normal(0, 1, 253)],
              np.full(256, np.nan), 1.0 + np.arange(256) / 256.0]
    return np.concatenate(blocks).astype(np.float32)


def state_of(cuda, opt, m, v, count=0):
    p = torch.zeros(len(m), device=cuda)
    return opt.restore(p, torch.tensor(m, device=cuda), torch.tensor(v, device=cuda), count)


def test_conversion_to_nearest(cuda):
    rng = np.random.default_rng(0)
    m = values(rng)
    with np.errstate(over="ignore", invalid="ignore"):
        v = np.square(m).astype(np.float32)
    s32 = state_of(cuda, AdamW(1e-3), m, v)
    s8 = s32.convert(8)
    back = s8.convert(32)
    got_m, got_r = np64(back.mu_flat), np64(back.nu_flat)
    want, near = ref.held(m.astype(np.float64), 3)
    tie = near < 2.0 ** -30
    same = (got_m == want) | (np.isnan(got_m) & np.isnan(want))
    assert np.all(same), (m[~same][:9], got_m[~same][:9], want[~same][:9])
    assert tie.any()  # ties are among the values
    # the root is a float32 root: within 1e-4 steps of a threshold it may go either way
    with np.errstate(invalid="ignore"):
        want, near = ref.held(np.sqrt(v.astype(np.float64)), 4)
        square = np.float32(np.float32(want) ** 2).astype(np.float64)
    same = (got_r == square) | (np.isnan(got_r) & np.isnan(square))
    assert np.all(same | (near < 1e-4)), (v[~same][:9], got_r[~same][:9], square[~same][:9])
    assert np.mean(~same) < 0.02
    # what 8 bits hold is held again
    again = back.convert(8)
    assert torch.equal(again.convert(32).mu_flat.view(torch.int32), back.mu_flat.view(torch.int32))
    assert torch.equal(again.convert(32).nu_flat.nan_to_num(7.0), back.nu_flat.nan_to_num(7.0))


def test_conversion_keeps_roots_above_zero(cuda):
    v = np.r_[1.0, np.full(255, 1e-30)].astype(np.float32)
    s = state_of(cuda, AdamW(1e-3, moment_bits=8), np.zeros(256, np.float32), v)
    r = np.sqrt(np64(s.moments()[1][0] if isinstance(s.moments()[1], list) else s.moments()[1]))
    assert r[0] == 1.0 and np.all(r[1:] == 2.0 ** -18)


def test_stochastic_rounding_is_unbiased(cuda):
    """A moment between two codes: the mean over elements is the moment, within five standard
    deviations (a step of 1/8 of a power of two, rounded up with probability f)."""
    n, x = 1 << 20, 1.09375  # 3/4 of the way from 1 to 1.125
    opt = AdamW(0.0, b1=0.0, b2=0.0, moment_bits=8, seed=5)
    p = torch.zeros(n, device=cuda)
    state = opt.init(p)
    opt.step(p, torch.full((n,), x, device=cuda), state)
    m, v = (np64(t[0] if isinstance(t, list) else t) for t in state.moments())
    assert set(np.unique(m)) == {1.0, 1.125} and abs(m.mean() - x) <= 5 * 0.125 * np.sqrt(0.75 * 0.25 / n)
    r = np.sqrt(v)
    assert set(np.unique(r)) == {1.0625, 1.125} and abs(r.mean() - x) <= 5 * 0.0625 * 0.5 / np.sqrt(n)


def test_an_8_bit_run_follows_a_32_bit_run(cuda):
    """A quadratic bowl with noisy gradients over 400 steps: both reach the bottom; the 8-bit
    run's distance is at most 1.5 times the 32-bit run's."""
    n = 20_000
    gen = torch.Generator(device=cuda).manual_seed(1)
    goal = torch.randn(n, generator=gen, device=cuda)
    size = torch.exp(torch.randn(n, generator=gen, device=cuda))
    far = {}
    for bits in (32, 8):
        noise = torch.Generator(device=cuda).manual_seed(2)
        p = torch.zeros(n, device=cuda)
        opt = AdamW(lambda c: 0.05 * 0.99 ** c, moment_bits=bits)
        state = opt.init(p)
        for _ in range(400):
            g = size * ((p - goal) + 0.3 * torch.randn(n, generator=noise, device=cuda))
            opt.step(p, g, state)
        far[bits] = float((p - goal).norm() / goal.norm())
    assert far[32] < 0.1 and far[8] <= 1.5 * far[32], far


# ---- norms ----------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("apart", [False, True])
def test_norms(cuda, kind, apart):
    """float64 sums: the float32 results are within one rounding, 2 e relative with the root's."""
    rng = np.random.default_rng(9)
    sizes = SIZES + [70_001, 3_000_003] + [int(n) for n in rng.integers(0, 300, 120)]
    gs = tensors(cuda, [rng.normal(0, 1, n).astype(np.float32) * np.float32(10.0 ** rng.integers(-3, 3)) for n in sizes],
                 TYPES[kind], apart)
    each = np.array([np.sqrt((np64(g) ** 2).sum()) for g in gs])
    total = np.sqrt((each ** 2).sum())
    got = grad_norms(gs, max_norm=2.0)
    np.testing.assert_allclose(np64(got.per_tensor), each, rtol=2 * E)
    assert abs(float(got.total) - total) <= 2 * E * total
    assert abs(float(got.scale) - 2.0 / (total + 1e-6)) <= 2 * E
    # not clipped below the norm, and a scale that comes along
    s = torch.full((), -0.25, device=cuda)
    got = grad_norms(gs, max_norm=1e9, grad_scale=s)
    assert abs(float(got.total) - 0.25 * total) <= 2 * E * total and float(got.scale) == -0.25
    assert float(grad_norms(gs, grad_scale=s).scale) == -0.25
    assert torch.equal(grad_norms(gs).per_tensor, grad_norms(gs).per_tensor)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", [[1], [8191, 8192, 8193], [131_072], [131_073], [0, 131_071, 0, 1], [8192] * 16,
                                   [100] * 17, [0] * 16])
def test_norms_of_few_and_of_empty_tensors(cuda, kind, sizes):
    """Around whole runs of a workgroup (8192 elements) and with empty tensors between."""
    rng = np.random.default_rng(12)
    gs = tensors(cuda, [rng.normal(0, 1, n).astype(np.float32) for n in sizes], TYPES[kind], apart=True)
    each = np.array([np.sqrt((np64(g) ** 2).sum()) for g in gs])
    total = np.sqrt((each ** 2).sum())
    got = grad_norms(gs, max_norm=3.0, grad_scale=torch.full((), 0.5, device=cuda))
    np.testing.assert_allclose(np64(got.per_tensor), 0.5 * each, rtol=2 * E)
    assert abs(float(got.total) - 0.5 * total) <= 2 * E * total
    assert abs(float(got.scale) - 0.5 * min(1.0, 3.0 / (0.5 * total + 1e-6))) <= 2 * E


def test_norms_of_very_large_and_very_small_values(cuda):
    for x in (1e30, 3e38, 1e-30, 1e-44):
        g = torch.full((1000,), x, device=cuda)
        want = np.float64(np.float32(x)) * np.sqrt(1000.0)
        got = grad_norms([g], max_norm=1.0)
        if want < 3.4e38:
            assert abs(float(got.total) - want) <= 2 * E * want + 1e-45
        assert abs(float(got.scale) - min(1.0, 1.0 / (want + 1e-6))) <= 2 * E * float(got.scale) + 1e-45


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_norms_that_are_not_finite(cuda, bad):
    g = torch.ones(5000, device=cuda)
    g[4321] = bad
    got = grad_norms([torch.ones(3, device=cuda), g], max_norm=1.0)
    assert not torch.isfinite(got.total) and torch.isnan(got.scale)
    assert float(got.per_tensor[0]) == pytest.approx(3 ** 0.5)
    keep = torch.ones(5000, dtype=torch.bool, device=cuda)
    keep[4321] = False
    ok = grad_norms(g, max_norm=1.0, active_mask=keep)
    assert float(ok.total) == pytest.approx(4999 ** 0.5)


@pytest.mark.parametrize("rows, lens", [(1, [1, 7]), (379, [3, 48, 1]), (3, [5000, 4097]), (20_000, [48, 9]),
                                        (41, [5000, 8191, 8193, 9001]), (70_003, [1, 2, 3, 5, 6, 7, 8])])
def test_norms_with_a_row_mask(cuda, rows, lens):
    rng = np.random.default_rng(10)
    on = rng.random(rows) < 0.5
    gs = [torch.tensor(rng.normal(0, 1, (rows, n)).astype(np.float32), device=cuda) for n in lens]
    for m in (on, np.zeros(rows, bool), np.ones(rows, bool)):
        each = [np.sqrt((np64(g)[m] ** 2).sum()) for g in gs]
        got = grad_norms(gs, max_norm=0.1, active_mask=torch.tensor(m, device=cuda))
        np.testing.assert_allclose(np64(got.per_tensor), each, rtol=2 * E)
        want = min(1.0, 0.1 / (np.linalg.norm(each) + 1e-6))
        assert abs(float(got.scale) - want) <= 2 * E


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows, lens", [(500, [1, 2, 3, 7, 8, 9, 48]), (9000, [1, 3, 5, 6, 16, 31])])
def test_norms_of_half_types_with_a_row_mask(cuda, kind, rows, lens):
    """Eight elements a lane, over up to eight rows; NaN in the masked ones."""
    rng = np.random.default_rng(13)
    on = rng.random(rows) < 0.4
    gs = [torch.tensor(rng.normal(0, 1, (rows, n)).astype(np.float32), device=cuda).to(TYPES[kind]) for n in lens]
    for g in gs:
        g[torch.tensor(~on, device=cuda)] = float("nan")
    each = [np.sqrt((np64(g)[on] ** 2).sum()) for g in gs]
    got = grad_norms(gs, active_mask=torch.tensor(on, device=cuda))
    np.testing.assert_allclose(np64(got.per_tensor), each, rtol=2 * E)


def test_norms_of_nothing(cuda):
    got = grad_norms([torch.zeros(0, device=cuda), torch.zeros(0, 3, device=cuda)], max_norm=1.0)
    assert float(got.total) == 0.0 and float(got.scale) == 1.0


# ---- the state ------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_goes_on_with_the_same_bits(cuda, bits):
    make = lambda: {"a": torch.randn(300, 5, device=cuda), "b": torch.randn(7, device=cuda).to(torch.bfloat16)}  # noqa: E731
    p, grads = make(), [make() for _ in range(3)]
    opt = AdamW({"a": 1e-2, "b": lambda c: 1e-2 / (c + 1)}, weight_decay={"a": 0.1, "b": 0.0}, moment_bits=bits,
                master_weights=True)
    a = opt.init(p)
    opt.step(p, grads[0], a)
    q = {k: v.clone() for k, v in p.items()}
    saved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in a.state_dict().items()}
    b = opt.load_state_dict(q, saved)
    for g in grads[1:]:
        opt.step(p, g, a)
        opt.step(q, g, b)
    for k in p:
        assert torch.equal(p[k], q[k])
    assert torch.equal(a.mu_flat, b.mu_flat) and torch.equal(a.nu_flat, b.nu_flat) and a.count == b.count == 3


def gaussians(cuda, n, k=4, seed=0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device=cuda)  # noqa: E731
    return Gaussians(r(n, 3), r(n, 3), r(n, 4), r(n, 1), r(n, k, 3))


def test_restored_from_an_adam_run(cuda):
    """The state after two steps of Adam, gone on with: the third step is the formula's from
    Adam's moments at t = 3, with the schedule's rate at count 2."""
    from jax_gs_amd.training.optimizer import FIELDS, make_optimizer

    opt, new = make_optimizer(1.0, 100), make_adamw(1.0, 100)
    p = gaussians(cuda, 321)
    grads = [gaussians(cuda, 321, seed=s) for s in range(1, 4)]
    state = opt.init(p)
    opt.step(p, grads[0], state)
    opt.step(p, grads[1], state)
    other = new.restore(p, state.mu, state.nu, state.count)
    before = {f: (np64(getattr(p, f)), np64(state.mu[f]), np64(state.nu[f])) for f in FIELDS}
    new.step(p, grads[2], other)
    for f in FIELDS:
        lr = opt.lr_at(f, 2)
        w, m, v, size = ref.step(before[f][0], np64(getattr(grads[2], f)), *before[f][1:], 3, lr)
        unit = size / (1 - 0.9 ** 3) / np.sqrt(v / (1 - 0.999 ** 3))
        check32((np64(getattr(p, f)), np64(other.mu[f]), np64(other.nu[f])), (w, m, v), lr * unit, size, "f32", 1)


def test_refusals(cuda):
    p, g = torch.zeros(8, device=cuda), torch.zeros(8, device=cuda)
    opt = AdamW(1e-3)
    state = opt.init([p, p.clone()])
    with pytest.raises(ValueError, match="not those of the state"):
        opt.step([p], [g], state)
    with pytest.raises(ValueError, match="given twice"):
        opt.step([p, p], [g, g], state)
    both = torch.zeros(12, device=cuda)
    with pytest.raises(ValueError, match="overlap"):
        opt.step([both[:8], both[4:]], [g, g], state)
    with pytest.raises(TypeError, match="entry 1 is not a tensor"):
        opt.step([p, 3.0], [g, g], state)
    with pytest.raises(TypeError, match="int64"):
        grad_norms([g, torch.zeros(3, dtype=torch.int64, device=cuda)])
    with pytest.raises(ValueError, match="is on cpu"):
        grad_norms([g, torch.zeros(3)])
    with pytest.raises(ValueError, match="contiguous"):
        opt.init([torch.zeros(4, 6, device=cuda).t()])
    with pytest.raises(ValueError, match="2 tensors"):
        opt.step([p, p.clone()], [g], state)
    with pytest.raises(ValueError, match="shaped like"):
        opt.step([p, p.clone()], [g, g[:4]], state)
    with pytest.raises(ValueError, match="shaped like"):
        opt.step([p, p.clone()], [g, g.cpu()], state)
    with pytest.raises(TypeError, match="float64"):
        opt.step([p, p.clone()], [g, g.double()], state)
    with pytest.raises(ValueError, match="contiguous"):
        opt.step([torch.zeros(16, device=cuda)[::2], p], [g, g], state)
    with pytest.raises(ValueError, match="active_mask"):
        opt.step([p, p.clone()], [g, g], state, active_mask=torch.ones(7, dtype=torch.bool, device=cuda))
    with pytest.raises(ValueError, match="grad_scale"):
        opt.step([p, p.clone()], [g, g], state, grad_scale=torch.ones(2, device=cuda))
    with pytest.raises(ValueError, match="8 bits"):
        AdamW(1e-3, moment_bits=8).init(p).mu
    with pytest.raises(ValueError, match="32 or 8"):
        state.convert(16)
    with pytest.raises(ValueError, match="other tensors"):
        opt.load_state_dict(p, state.state_dict())
    with pytest.raises(ValueError, match="values of"):
        AdamW([1e-3]).init([p, g])
    with pytest.raises(ValueError, match="missing"):
        AdamW({"a": 1e-3}).init({"a": p, "b": g})
    with pytest.raises(ValueError, match="not those of the parameters"):
        opt.restore([p], [p[:3]], [p], 1)
    with pytest.raises(ValueError, match="no gradients"):
        grad_norms([None])
    with pytest.raises(ValueError, match="max_norm"):
        grad_norms([g], max_norm=0.0)
    named = AdamW(1e-3).init({"a": p, "b": p.clone()})
    with pytest.raises(ValueError, match="no tensor for"):
        opt.step({"a": p, "b": p.clone()}, {"a": g}, named)
    assert state.count == 0 and named.count == 0 and not p.any()


# ---- as it is used: the training step and density control -------------------------------------

def training_state(cuda, optimizer, n=1500, capacity=2000):
    from jax_gs_amd import scenes
    from jax_gs_amd.training.density import init_density_state

    sc = scenes.make_scene(1, n=n, width=96, height=64)
    g, cam, tgt, _ = scenes.to_torch(sc, cuda)
    static = (cam.W, cam.H, cam.fx, cam.fy, cam.cx, cam.cy)
    return init_density_state(g, optimizer, capacity), tgt, cam.W2C, static


@pytest.mark.parametrize("bits", [32, 8])
def test_train_steps(cuda, bits):
    """train_step with AdamW: the loss falls, inactive rows stay, the norm is reported, and the
    fused and the autograd entry agree bit for bit (they are one path)."""
    from jax_gs_amd.training.trainer import train_step

    opt = make_adamw(1.0, 200, weight_decay=0.0, moment_bits=bits, max_grad_norm=10.0)
    state, tgt, w2c, static = training_state(cuda, opt)
    off = state.active_mask == 0
    keep = state.gaussians.sh_coeffs[off].clone()
    losses = []
    for _ in range(30):
        state, loss, metrics = train_step(state, tgt, w2c, static, opt, sh_degree=3)
        losses.append(float(loss))
    assert losses[-1] < 0.9 * losses[0], losses
    assert torch.isfinite(metrics["grad_norm"]) and state.opt_state.count == 30
    assert torch.equal(state.gaussians.sh_coeffs[off], keep)


@pytest.mark.parametrize("bits", [32, 8])
def test_density_control_moves_the_moments(cuda, bits):
    """Clones and splits take their source's moments along; every other row keeps its own."""
    from jax_gs_amd.training.density import densify_and_prune
    from jax_gs_amd.training.optimizer import FIELDS
    from jax_gs_amd.training.trainer import train_step

    opt = make_adamw(1.0, 200, moment_bits=bits)
    state, tgt, w2c, static = training_state(cuda, opt)
    for _ in range(3):
        train_step(state, tgt, w2c, static, opt, sh_degree=3)
    state.grad_accum.zero_()
    state.grad_accum[:300], state.denom[:300] = 1.0, 1  # above the threshold, and fewer than the empty slots
    was_on = state.active_mask.clone().bool()
    before = [{f: t.clone() for f, t in m.items()} for m in state.opt_state.moments()]
    densify_and_prune(state, grad_threshold=0.0002, extent=5.0, generator=torch.Generator(device=cuda).manual_seed(0))
    filled = state.active_mask.bool() & ~was_on
    assert int(filled.sum()) > 0
    after = state.opt_state.moments()
    for was, now in zip(before, after):
        for f in FIELDS:
            a, b = was[f].reshape(len(filled), -1), now[f].reshape(len(filled), -1)
            tol = 0.0 if bits == 32 else 2.0 ** -3
            # 8 bits: a filled row can raise its block's exponent, which costs its neighbours at most a step
            floor = 0.0 if bits == 32 else 2.0 ** -13 * float(b.abs().max())
            assert torch.all((a - b).abs()[~filled] <= tol * a.abs()[~filled] + floor)
            if bits == 32:
                rows = {tuple(r.tolist()) for r in a}
                assert all(tuple(r.tolist()) in rows for r in b[filled][:50])
            else:
                assert torch.isfinite(b).all() and b[filled].abs().sum() > 0
    train_step(state, tgt, w2c, static, opt, sh_degree=3)
    assert all(torch.isfinite(getattr(state.gaussians, f)).all() for f in FIELDS)


def test_gradients_agree_with_differences_of_the_loss(cuda):
    """The direction of one AdamW step from zero moments is minus the sign of the loss's
    differences: p moves by lr wherever a coordinate's difference is clear."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    a = torch.randn(40, 12, generator=gen, device=cuda, dtype=torch.float64)
    x0 = torch.randn(12, generator=gen, device=cuda, dtype=torch.float64)
    loss = lambda x: (a @ x).square().mean()  # noqa: E731
    x = x0.float().requires_grad_(True)
    loss(x.double()).backward()
    h = 1e-5
    diff = np.array([float(loss(x0 + h * e) - loss(x0 - h * e)) / (2 * h) for e in torch.eye(12, device=cuda, dtype=torch.float64)])
    opt = AdamW(0.01)
    p = x.detach().clone()
    opt.step(p, x.grad, opt.init(p))
    np.testing.assert_allclose(np64(p) - np64(x0.float()), -0.01 * np.sign(diff), rtol=1e-3)

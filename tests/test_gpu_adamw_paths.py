"""AdamW's paths against float64: scales and clip factors, masks with every type, arrays that go past the
caches (from 128 MB on), tensors of several launch records.

Tolerances as in test_gpu_adamw.py, with e = 2^-24: m and v 8 e of the terms that they are sums of (a scale adds
one rounding to the gradient, two to its square: 4 and 6 in all), w 4 e |w| + 24 e of the update; 8 bits: the value
held of the float64 result, one step beside it where that is within 1e-4 steps of being rounded the other way;
where many elements are compared, and sums that cancel are among them, exactly the value held of the same operations
in float32, those within 8 e of float64.
A clip factor is compared with its formula (2 e) and the step then with the factor that was used."""
import numpy as np
import pytest
import torch

import adamw_reference as ref
from jax_gs_amd.training.adamw import AdamW, grad_norms
from test_gpu_adamw import SIZES, TYPES, check32, check8, rows_like, run32, tensors, weights_close

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


# ---- scales and clip factors ------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param, grad, master", [("f32", "f32", False), ("bf16", "bf16", True), ("f16", "f16", False)])
@pytest.mark.parametrize("scale, clip", [(0.37, None), (torch.tensor(-0.25), None), (None, 0.01), (1.0 / 64.0, 0.002),
                                         (torch.tensor(8.0), 1e6)])
def test_step_with_a_scale_and_a_clip_factor(cuda, bits, param, grad, master, scale, clip):
    rng = np.random.default_rng(21)
    sizes = SIZES + [5000]
    ps = tensors(cuda, [rng.normal(0, 1, n).astype(np.float32) for n in sizes], TYPES[param])
    opt = AdamW(1e-2, weight_decay=0.1, moment_bits=bits, master_weights=master, max_grad_norm=clip, seed=5)
    state = opt.init(ps)
    given = scale.to(cuda) if isinstance(scale, torch.Tensor) else scale
    for t in (1, 2):
        gs = tensors(cuda, [rows_like(rng, n) for n in sizes], TYPES[grad])
        before = [[np64(x).reshape(-1) for x in (state.master[i] if master else ps[i], *(m[i] for m in state.moments()))]
                  for i in range(len(sizes))]
        opt.step(ps, gs, state, grad_scale=given)
        s = 1.0 if scale is None else float(np.float32(float(scale)))
        if clip is not None:
            total = abs(s) * np.sqrt(sum((np64(g) ** 2).sum() for g in gs))
            want = s * min(1.0, clip / (total + 1e-6))
            assert (want != s) == (clip < 1.0)  # the case clips, or does not
            s = float(state.norms.scale)
            assert abs(s - want) <= 2 * E * abs(want)
        for i, n in enumerate(sizes):
            w0, m0, v0 = before[i]
            w, m, v, size = ref.step(w0, np64(gs[i]), m0, v0, t, 1e-2, decay=0.1, scale=s)
            with np.errstate(divide="ignore", invalid="ignore"):
                unit = np.nan_to_num(size / (1 - 0.9 ** t) / np.sqrt(v / (1 - 0.999 ** t)), posinf=0.0)
            got = np64(state.master[i] if master else ps[i]).reshape(-1)
            if bits == 8:
                check8(state, i, m, v, t, 5)
                weights_close(got, w, 4 * E * np.abs(w) + 24 * E * 1e-2 * unit, "f32" if master else param)
            else:
                check32((got, np64(state.mu[i]), np64(state.nu[i])), (w, m, v), 1e-2 * unit, size, "f32" if master else param, 1)


# ---- masks ------------------------------------------------------------------------------------

HALF = [("f32", "bf16", False), ("bf16", "bf16", False), ("bf16", "bf16", True), ("bf16", "f32", True), ("f16", "f16", False),
        ("f16", "f16", True), ("f16", "bf16", True)]


@pytest.mark.parametrize("param, grad, master", HALF)
@pytest.mark.parametrize("rows, lens", [(1, [1, 7]), (37, [3, 4, 1, 48, 2]), (3, [5000, 4097, 300]), (1000, [64, 65, 9])])
def test_step_of_half_types_with_a_row_mask(cuda, param, grad, master, rows, lens):
    on = np.random.default_rng(5).random(rows) < 0.5
    run32(cuda, [rows * n for n in lens], param, grad, master, 0.1, True, on=on, rows=rows)


@pytest.mark.parametrize("param, grad, master", [("f32", "f32", False), *HALF])
@pytest.mark.parametrize("rows, lens", [(37, [3, 4, 1, 48, 2]), (3, [5000, 4097, 300]), (1000, [64, 65, 9])])
def test_step_in_8_bits_with_a_row_mask(cuda, param, grad, master, rows, lens):
    rng = np.random.default_rng(6)
    on = rng.random(rows) < 0.5
    ps = [p.view(rows, -1) for p in tensors(cuda, [rng.normal(0, 1, rows * n).astype(np.float32) for n in lens], TYPES[param], True)]
    opt = AdamW(1e-2, weight_decay=0.1, moment_bits=8, master_weights=master, seed=7)
    state = opt.init(ps)
    for t in range(1, 4):
        gs = [g.view(rows, -1) for g in tensors(cuda, [rows_like(rng, rows * n) for n in lens], TYPES[grad], True)]
        before = [[np64(x).reshape(-1) for x in (state.master[i] if state.master_flat is not None else ps[i], *(m[i] for m in state.moments()))]
                  for i in range(len(lens))]
        opt.step(ps, gs, state, active_mask=torch.tensor(on, device=cuda))
        for i, n in enumerate(lens):
            w0, m0, v0 = before[i]
            w, m, v, size = ref.step(w0, np64(gs[i]).reshape(-1), m0, v0, t, 1e-2, decay=0.1, on=on.repeat(n))
            check8(state, i, m, v, t, 7)
            with np.errstate(divide="ignore", invalid="ignore"):
                unit = np.nan_to_num(size / (1 - 0.9 ** t) / np.sqrt(v / (1 - 0.999 ** t)), posinf=0.0)
            got = np64(state.master[i] if state.master_flat is not None else ps[i]).reshape(-1)
            weights_close(got, w, 4 * E * np.abs(w) + 24 * E * 1e-2 * unit, "f32" if master else param)


# ---- past the caches, on the device -----------------------------------------------------------

def pow2(e):
    """2^e exactly (torch.ldexp multiplies by a rounded power on the device)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def held64(x, mantissa, u=None):
    """adamw_reference.held for finite float64 values on the device."""
    x = x.view(-1, 256)
    a = x.abs()
    f, e = torch.frexp(a.amax(1, keepdim=True))
    e = torch.where(f > 1.0 - 2.0 ** -mantissa, e, e - 1).clamp(-127, 127)
    q = a * pow2(-e)
    own = (torch.frexp(q)[1] - 1).clamp(min=-14)
    at = q * pow2(mantissa - own)
    if u is None:
        near, k = (at - at.floor() - 0.5).abs(), at.round()
    else:
        w = at + u.view(-1, 256)
        near, k = (w - w.round()).abs(), w.floor()
    if mantissa == 4:
        k = torch.where((a > 0) & (k == 0), 1.0, k)
    value = (k * pow2(own - mantissa)).clamp(max=2.0 - 2.0 / 2 ** mantissa) * pow2(e)
    value = value * torch.where(torch.signbit(x), -1.0, 1.0)
    edge = (f / (1.0 - 2.0 ** -mantissa) - 1.0).abs() < 1e-5
    return value.view(-1), torch.where(edge, 0.0, near).view(-1), pow2(own - mantissa + e).view(-1)


def noise64(n, start, seed, step):
    low = 0xFFFFFFFF
    p = torch.arange(start, start + n, device="cuda")
    key = (seed * 0x85EBCA6B + step * 0xC2B2AE3D + 0x27D4EB2F) & low
    h = (p * 0x9E3779B1 + key) & low  # places below 2^32
    h ^= h >> 15
    h = (h * 0xD1B54A35) & low
    h ^= h >> 13
    return (h >> 16).double() / 65536, (h & 0xFFFF).double() / 65536


def held_close(got, want, mantissa, u=None):
    value, near, step = held64(want, mantissa, u)
    same = got == value
    assert bool((same | ((near < 1e-4) & ((got - value).abs() <= 2 * step))).all())
    assert int((~same).sum()) <= 1e-3 * len(same)


def padded(t, n):
    out = torch.zeros(-(-n // 256) * 256, dtype=torch.float64, device=t.device)
    out[:n] = t.double().reshape(-1)
    return out


# elements so that parameters, gradients and moments are above 128 MB, or the parameters alone are
@pytest.mark.parametrize("bits, param, grad, master, row, rows", [
    (32, "f32", "f32", False, 1, 9_000_001), (32, "f32", "f32", False, 7, 1_300_003), (32, "bf16", "bf16", True, 1, 9_000_003),
    (32, "bf16", "f16", True, 3, 3_100_001), (32, "f16", "f16", False, 5, 2_300_001), (32, "f32", "bf16", False, 1, 34_000_001),
    (32, "f32", "f32", False, 48, 710_003), (8, "f32", "f32", False, 1, 14_000_001), (8, "f32", "bf16", False, 48, 300_011),
    (8, "bf16", "bf16", True, 1, 14_000_005), (8, "bf16", "bf16", True, 3, 4_700_001), (8, "f16", "f32", False, 7, 2_100_001),
    (8, "f32", "f32", False, 3, 11_400_001)])
def test_steps_past_the_caches(cuda, bits, param, grad, master, row, rows):
    """Three tensors at odd places of one buffer, a short one on each side; rows of more than one element under a
    mask, with NaN where it is off; a scale and a clip factor; two steps from moments in the middle of a run."""
    gen = torch.Generator(device=cuda).manual_seed(rows)
    sizes = [rows * row] if row > 1 else [5, rows, 257]
    rnd = lambda n: torch.randn(n, generator=gen, device=cuda)  # noqa: E731

    def buffer(parts, dtype):
        flat = torch.zeros(sum(sizes) + 1, dtype=dtype, device=cuda)
        flat[1:] = torch.cat(parts).to(dtype)
        return [x.view(rows, row) if row > 1 else x for x in flat[1:].split(sizes)]

    ps = buffer([rnd(n) for n in sizes], TYPES[param])
    on = torch.rand(rows, generator=gen, device=cuda) < 0.6 if row > 1 else None
    opt = AdamW(1e-2, weight_decay=0.1, moment_bits=bits, master_weights=master, max_grad_norm=1.0, seed=3)
    m0 = [rnd(n) * 1e-3 for n in sizes]
    state = opt.restore(ps, m0, [(x.abs() + 1e-4) ** 2 for x in m0], 40)
    first = ps[-1].clone()
    for t in (41, 42):
        gs = buffer([rnd(n) * torch.exp(rnd(n) - 7.0) for n in sizes], TYPES[grad])
        if on is not None:
            gs[0][~on] = float("nan")
        mu, nu = state.moments()
        before = [[x.reshape(-1).double() for x in (state.master[i] if master else ps[i], mu[i], nu[i])] for i in range(len(sizes))]
        opt.step(ps, gs, state, active_mask=on, grad_scale=0.5)
        live = [g.double() if on is None else torch.where(on[:, None], g.double(), 0.0) for g in gs]
        total = 0.5 * float(torch.stack([g.square().sum() for g in live]).sum().sqrt())
        s = float(state.norms.scale)
        assert abs(float(state.norms.total) - total) <= 4 * E * total and abs(s - 0.5 / (total + 1e-6)) <= 4 * E * s
        mu, nu = state.moments()
        for i, n in enumerate(sizes):
            w0, m, v = before[i]
            g = live[i].reshape(-1) * s
            size = 0.9 * m.abs() + (1 - 0.9) * g.abs()
            m = 0.9 * m + (1 - 0.9) * g
            v = 0.999 * v + (1 - 0.999) * g * g
            unit = 1.0 / (1 - 0.9 ** t) / (v / (1 - 0.999 ** t)).sqrt()  # v > 0 here
            w = w0 - 1e-2 * (m / (1 - 0.9 ** t) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8) + 0.1 * w0)
            got_m, got_v = mu[i].double().reshape(-1), nu[i].double().reshape(-1)
            if bits == 32:
                assert bool(((got_m - m).abs() <= 8 * E * size).all()) and bool(((got_v - v).abs() <= 8 * E * v).all())
            else:
                um, ur = noise64(-(-n // 256) * 256, state.offsets[i], 3, state.count)
                x = live[i].float().reshape(-1) * state.norms.scale
                m32 = before[i][1].float() * 0.9 + x * (1 - 0.9)
                v32 = before[i][2].float() * 0.999 + (x * x) * (1 - 0.999)
                assert bool(((m32 - m).abs() <= 8 * E * size).all()) and bool(((v32 - v).abs() <= 8 * E * v).all())
                assert torch.equal(padded(got_m, n), held64(padded(m32, n), 3, um)[0])
                assert torch.equal(padded(got_v, n).sqrt(), held64(padded(v32.sqrt(), n), 4, ur)[0])
            got = (state.master[i] if master else ps[i]).reshape(-1)
            tol = 4 * E * w.abs() + 24 * E * 1e-2 * size * unit
            lo, hi = w - tol, w + tol
            if not master and param != "f32":  # half of its type's nearest values of the range's ends
                lo, hi = lo.float().to(TYPES[param]).double(), hi.float().to(TYPES[param]).double()
            close = (got.double() >= lo) & (got.double() <= hi)
            if on is not None:
                off = (~on).repeat_interleave(row)
                close = torch.where(off, got.double() == w0, close)
            assert bool(close.all())
            if master:
                assert torch.equal(ps[i].reshape(-1), got.to(TYPES[param]))
    if on is not None:
        assert torch.equal(ps[0][~on], first[~on]) and not torch.equal(ps[0][on], first[on])


@pytest.mark.parametrize("n", [14_000_001, 40_000_000])
def test_conversions_past_the_caches(cuda, n):
    gen = torch.Generator(device=cuda).manual_seed(n)
    size = torch.exp(3.0 * torch.randn(n, generator=gen, device=cuda) - 9.0)
    m = torch.randn(n, generator=gen, device=cuda) * size
    v = (torch.rand(n, generator=gen, device=cuda) + 0.05) * size * size
    s8 = AdamW(1e-3, moment_bits=8).restore([torch.empty(n, device=cuda)], [m], [v], 5)
    got_m, got_v = (x[0].double() for x in s8.moments())
    held_close(padded(got_m, n), padded(m, n), 3)
    held_close(padded(got_v, n).sqrt(), padded(v, n).sqrt(), 4)
    again = s8.convert(32).convert(8)  # the same values (a block whose largest was rounded down takes other codes)
    for x, y in zip(again.moments(), s8.moments()):
        assert torch.equal(x[0], y[0])


# ---- as it is used ----------------------------------------------------------------------------

def test_both_entries_of_the_training_step_are_one_path(cuda, monkeypatch):
    """With an AdamW, fused=True and fused=False both compose the step from autograd."""
    from jax_gs_amd.training import trainer
    from jax_gs_amd.training.adamw import make_adamw
    from test_gpu_adamw import training_state

    taken = []
    compose = trainer._train_step_autograd
    monkeypatch.setattr(trainer, "_train_step_autograd", lambda *a: (taken.append(len(a)), compose(*a))[1])
    for fused in (True, False):
        opt = make_adamw(1.0, 200)
        state, tgt, w2c, static = training_state(cuda, opt)
        trainer.train_step(state, tgt, w2c, static, opt, sh_degree=3, fused=fused)
        assert state.opt_state.count == 1
    assert len(taken) == 2


def test_a_norm_beyond_float32_still_clips(cuda):
    """The sums are float64: 100 gradients of 2e38 have the norm 2e39, which float32 does not hold, and a factor of
    5e-40, which it holds to half of 2^-149.  The step is made; gradients that are not finite make none."""
    g = torch.full((100,), 2e38, device=cuda)
    norms = grad_norms([g], max_norm=1.0)
    assert float(norms.total) == float("inf") == float(norms.per_tensor[0])
    want = 1.0 / (float(g[0].double()) * 10.0)
    assert abs(float(norms.scale.double()) - want) <= 2.0 ** -150
    p = torch.zeros(100, device=cuda)
    opt = AdamW(1e-2, max_grad_norm=1.0)
    state = opt.init([p])
    opt.step([p], [g], state)
    # g * scale: half of 2^-149 of 5e-40, 1.5e-6, and one rounding; three more in m
    np.testing.assert_allclose(np64(state.mu[0]), 0.1 * np64(g) * want, rtol=2e-6)
    before = p.clone()
    g[3] = float("inf")
    opt.step([p], [g], state)
    assert torch.equal(p, before) and bool(p.lt(0).all()) and torch.isnan(state.norms.scale)

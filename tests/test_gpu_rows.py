"""Rows by an index on the device: every value arrives bit by bit; 8-bit moments against 64 bits."""
import numpy as np
import pytest
import torch

from adamw_reference import held, pad
from jax_gs_amd.core.gaussians import Gaussians
from jax_gs_amd.training.adamw import AdamW
from jax_gs_amd.training.optimizer import FIELDS, Adam
from jax_gs_amd.training.rows import best_rows, move_rows_, take_rows

pytestmark = pytest.mark.gpu


def bits(shape, dtype, seed, device):
    """Any bits, NaNs with payloads among them."""
    gen = torch.Generator().manual_seed(seed)
    size = torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 256, (int(np.prod(shape)) * size,), generator=gen, dtype=torch.uint8)
    if dtype == torch.bool:
        raw &= 1
    return raw.to(device).view(dtype).reshape(shape)


def raw(t):
    return t.detach().contiguous().reshape(-1).view(torch.uint8).cpu().numpy()


def want_taken(t, index, fill=None):
    """Row by row on the host."""
    rows = t.detach().cpu().contiguous()
    out = torch.zeros((len(index), *t.shape[1:]), dtype=t.dtype) if fill is None else \
        fill.detach().cpu().expand((len(index), *t.shape[1:])).clone()
    index = index.cpu().long()
    there = (index >= 0) & (index < t.shape[0])
    out[there] = rows[index[there]]
    return out


def an_index(n, count, seed, dtype):
    """Repeats, rows that do not come, and entries that are no rows."""
    gen = torch.Generator().manual_seed(seed)
    index = torch.randint(0, max(n, 1), (count,), generator=gen)
    odd = torch.rand(count, generator=gen)
    index[odd < 0.1] = -1
    index[(odd >= 0.1) & (odd < 0.13)] = n
    index[(odd >= 0.13) & (odd < 0.15)] = -(1 << 31)
    index[(odd >= 0.15) & (odd < 0.17)] = (1 << 31) - 1
    if n == 0:
        index[:] = -1
    if dtype == torch.int64 and count > 2:
        index[0], index[1] = (1 << 32), -(1 << 40)  # row 0's and another's lower 32 bits
    return index.to(dtype)


SHAPES = [((), torch.float32), ((1,), torch.uint8), ((3,), torch.float32), ((3,), torch.uint8), ((7,), torch.float16),
          ((4,), torch.float32), ((5,), torch.float64), ((16, 3), torch.float32), ((2, 3, 4), torch.bfloat16),
          ((45,), torch.int8), ((0,), torch.float32), ((2, 0, 3), torch.int32), ((1000,), torch.bool),
          ((2049,), torch.complex64), ((16385,), torch.uint8), ((20001,), torch.float16), ((33333,), torch.int64)]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n, count", [(1, 1), (1, 300), (300, 1), (300, 411), (41, 0), (0, 5)])
def test_take_rows(cuda, n, count, dtype):
    """Rows of no, one and many elements, up to more than a workgroup's, of every type's size."""
    index = an_index(n, count, 7 * n + count, dtype).to(cuda)
    tensors = [bits((n, *shape), t, i, cuda) for i, (shape, t) in enumerate(SHAPES)]
    for x, got in zip(tensors, take_rows(tensors, index)):
        assert got.shape == (count, *x.shape[1:]) and got.dtype == x.dtype and got.is_contiguous()
        np.testing.assert_array_equal(raw(got), raw(want_taken(x, index)))


def test_take_rows_of_strided_and_odd_tensors(cuda):
    """Slices of rows and of their elements, addresses of every alignment, an expanded row, a transposed tensor, a
    lazily negated and a conjugated one; fills of all kinds."""
    gen = torch.Generator().manual_seed(3)
    index = an_index(97, 250, 5, torch.int32).to(cuda)
    tensors, fills = [], []
    for at in (1, 2, 3, 4, 8, 12, 16):
        buffer = bits((97 * 24 + at,), torch.uint8, at, cuda)
        tensors.append(buffer[at:].view(97, 24))
    wide = bits((200, 40), torch.int16, 9, cuda)
    tensors += [wide[3:100, 5:12], wide[::2][:97, 8:16], wide[:97, :1], wide[:97, ::3]]
    tensors.append(torch.randn(1, 9, generator=gen).to(cuda).expand(97, 9))
    tensors.append(torch.randn(30, 97, generator=gen).to(cuda).t())
    c = torch.randn(97, 5, dtype=torch.complex64, generator=gen).to(cuda)
    tensors += [c.conj(), c.conj().imag]
    for i, t in enumerate(tensors):
        assert t.shape[0] == 97
        fills.append(None if i % 3 == 0 else (t.resolve_conj().resolve_neg()[i] if i % 3 == 1 else t[i + 1]))
    before = [t.resolve_conj().resolve_neg().clone() for t in tensors]
    got = take_rows(tensors, index, fill=fills)
    for x, f, g in zip(before, fills, got):
        np.testing.assert_array_equal(raw(g), raw(want_taken(x, index, None if f is None else f.resolve_conj().resolve_neg())))
    # an index that is a strided view
    two = torch.stack([index, index.flip(0)], 1)
    np.testing.assert_array_equal(raw(take_rows(tensors[0], two[:, 1])), raw(want_taken(before[0], index.flip(0))))


def test_take_rows_of_many_tensors(cuda):
    """More than one launch, and the forms of the answer."""
    ts = {f"t{i}": bits((61, i % 9), torch.float32, i, cuda) for i in range(150)}
    index = an_index(61, 70, 1, torch.int64).to(cuda)
    got = take_rows(ts, index, fill={**dict.fromkeys(ts), "t4": torch.ones(4, device=cuda)})
    assert list(got) == list(ts)
    for k in ts:
        np.testing.assert_array_equal(raw(got[k]), raw(want_taken(ts[k], index, torch.ones(4) if k == "t4" else None)))
    g = Gaussians(*[bits((61, *s), torch.float32, 1, cuda) for s in ((3,), (3,), (4,), (1,), (16, 3))])
    new = take_rows(g, index)
    assert isinstance(new, Gaussians)
    for f in FIELDS:
        np.testing.assert_array_equal(raw(getattr(new, f)), raw(want_taken(getattr(g, f), index)))
    assert isinstance(take_rows(tuple(ts.values())[:2], index), list)


def test_take_rows_beyond_4_gib(cuda):
    """Offsets above 32 bits on both sides."""
    n, row = 300_000, 16 * 1024
    x = torch.empty((n, row), dtype=torch.uint8, device=cuda)
    x[:, 0] = (torch.arange(n, device=cuda) % 251).to(torch.uint8)
    x[:, -1] = (torch.arange(n, device=cuda) // 251 % 251).to(torch.uint8)
    index = torch.arange(n - 1, -1, -1, device=cuda, dtype=torch.int32)
    got = take_rows(x, index)
    assert torch.equal(got[:, 0], x[:, 0].flip(0)) and torch.equal(got[:, -1], x[:, -1].flip(0))
    stay = torch.arange(n, device=cuda, dtype=torch.int64)
    stay[-3:] = torch.tensor([1, -1, n - 100], device=cuda)
    move_rows_(x, stay)
    assert torch.equal(x[-3, ::16383], x[1, ::16383]) and not bool(x[-2].any()) and torch.equal(x[-1], x[n - 100])


def a_move(n, seed, dtype, moved=0.3, freed=0.1):
    """An index whose sources stay."""
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(n, generator=gen)
    m, f = int(moved * n), int(freed * n)
    index = torch.arange(n)
    stay = order[m + f:]
    if len(stay):
        index[order[:m]] = stay[torch.randint(0, len(stay), (m,), generator=gen)]
    index[order[m:m + f]] = -1
    return index.to(dtype)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [1, 2, 63, 1024, 1025, 5000])
def test_move_rows(cuda, n, dtype):
    index = a_move(n, n, dtype).to(cuda)
    tensors = [bits((n, *shape), t, i, cuda) for i, (shape, t) in enumerate(SHAPES) if n * np.prod(shape, dtype=int) < 1 << 25]
    before = [t.clone() for t in tensors]
    versions = [t._version for t in tensors]
    left = torch.full((), 5, dtype=torch.int32, device=cuda)
    assert move_rows_(tensors, index, left=left) is tensors
    for x, got, v in zip(before, tensors, versions):
        np.testing.assert_array_equal(raw(got), raw(want_taken(x, index)))
        assert got._version > v
    assert int(left) == 5
    # moved once more nothing changes but what is freed
    move_rows_(tensors, torch.arange(n, device=cuda, dtype=dtype))
    for x, got in zip(before, tensors):
        np.testing.assert_array_equal(raw(got), raw(want_taken(x, index)))


@pytest.mark.parametrize("n, row", [(300, 2048), (300, 8000), (70, 9000), (5, 70_000), (1025, 700)])
def test_wide_rows_move(cuda, n, row):
    """Rows of up to many workgroups' pieces, by themselves and beside short ones, all changed rows together and scattered."""
    tensors = [bits((n, row), torch.uint8, 1, cuda), bits((n, 3), torch.float32, 2, cuda), bits((n, row + 1), torch.uint8, 3, cuda),
               bits((n,), torch.float16, 4, cuda)]
    end = torch.arange(n)
    end[n - n // 3:] = torch.arange(n // 3)
    for index in (a_move(n, row, torch.int32), end):
        for some in (tensors[:1], tensors):
            before = [t.clone() for t in some]
            move_rows_(some, index.to(cuda))
            for x, got in zip(before, some):
                np.testing.assert_array_equal(raw(got), raw(want_taken(x, index)))


def test_move_rows_between_others(cuda):
    """Halves of a pool's pages with other pages between: what is not theirs stays; fills."""
    pool = bits((400, 3, 10), torch.float16, 1, cuda)
    before = pool.clone()
    index = a_move(200, 8, torch.int32).to(cuda)
    fill = bits((10,), torch.float16, 2, cuda)
    move_rows_([pool[::2, 0], pool[::2, 2]], index, fill=[fill, None])
    want = before.cpu().clone()
    want[::2, 0] = want_taken(before[::2, 0], index, fill)
    want[::2, 2] = want_taken(before[::2, 2], index)
    np.testing.assert_array_equal(raw(pool), raw(want))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rows_whose_sources_change_stay(cuda, dtype):
    """Swaps, chains, copies of freed rows and indices beyond the rows: each such row stays and is counted; the others move."""
    n = 3000
    index = a_move(n, 4, dtype, moved=0.1)
    want = index.clone()
    bad = 0
    gen = torch.Generator().manual_seed(1)
    stays = (index == torch.arange(n)).nonzero().reshape(-1)
    used = set(index[index != torch.arange(n)].tolist())
    spare = [i for i in stays.tolist() if i not in used]
    changed = ((index != torch.arange(n)) & (index >= 0)).nonzero().reshape(-1).tolist()
    freed = (index < 0).nonzero().reshape(-1).tolist()
    a, b, c, d, e = spare[:5]
    index[a], index[b] = b, a            # a swap
    index[c] = changed[0]                # a chain
    index[d] = freed[0]                  # a row that is freed
    index[e] = n                         # no row
    bad = 5
    if dtype == torch.int64:
        f = spare[5]
        index[f] = (1 << 32) + stays[0]
        bad += 1
    x = bits((n, 5), torch.float32, 3, cuda)
    before, left = x.clone(), torch.zeros(1, dtype=torch.int32, device=cuda)
    move_rows_({"x": x}, index.to(cuda), left=left)
    np.testing.assert_array_equal(raw(x), raw(want_taken(before, want)))
    assert int(left) == bad
    # the moments follow the same rule
    for moment_bits in (32, 8):
        p = torch.zeros(n, 5, device=cuda)
        m = torch.randint(1, 8, (n, 5), generator=gen).float().to(cuda)  # held exactly in 8 bits
        state = AdamW(1e-3, moment_bits=moment_bits).restore([p], [m], [m * m], 3)
        state.move_rows_(index.to(cuda))
        mu, nu = state.moments()
        assert torch.equal(mu[0].cpu(), want_taken(m, want)) and torch.equal(nu[0].cpu(), want_taken(m * m, want))


def moments(shapes, seed, device):
    gen = torch.Generator().manual_seed(seed)
    size = [torch.exp(torch.randn(s[0], *[1] * (len(s) - 1), generator=gen) * 2.0 - 9.0) for s in shapes]
    mu = [(torch.randn(*s, generator=gen) * z).to(device) for s, z in zip(shapes, size)]
    nu = [((torch.rand(*s, generator=gen) + 0.05) * z * z).to(device) for s, z in zip(shapes, size)]
    return mu, nu


ROWS = [((), (3,), (4,), (16, 3)), ((1,), (255,), (256,), (257,), (0,)), ((5000,), (2, 2), (7,))]


@pytest.mark.parametrize("n, count", [(1, 1), (1, 700), (700, 1), (333, 500), (20, 0)])
@pytest.mark.parametrize("shapes", ROWS)
def test_moments_are_taken(cuda, shapes, n, count):
    """In 32 bits as they are; in 8 bits the values that 64 bits would hold of the rows taken, and zeros behind them."""
    shapes = [(n, *s) for s in shapes]
    mu, nu = moments(shapes, n + count, cuda)
    params = [torch.zeros(s, device=cuda) for s in shapes]
    index = an_index(n, count, n, torch.int32).to(cuda)
    wide = AdamW(1e-3).restore(params, mu, nu, 7)
    eight = wide.convert(8)
    taken = wide.take_rows(index)
    assert taken.count == 7 and taken.bits == 32 and torch.equal(taken.powers, wide.powers)
    for own, flat in ((mu, taken.mu_flat), (nu, taken.nu_flat)):
        want = np.concatenate([pad(want_taken(x, index).numpy()) for x in own] or [np.zeros(0)])
        np.testing.assert_array_equal(flat.cpu().numpy(), want.astype(np.float32))
    got = eight.take_rows(index)
    assert got.shapes == taken.shapes and got.bits == 8 and got.count == 7
    now = got.convert(32)
    for i, (m, v) in enumerate(zip(*eight.moments())):
        at, size = got.offsets[i], len(pad(np.zeros(got.counts[i])))
        if not size:
            continue
        want_m, _ = held(pad(want_taken(m, index).double().numpy()), 3)
        want_r, _ = held(pad(want_taken(v, index).double().sqrt().numpy()), 4)
        np.testing.assert_array_equal(now.mu_flat[at:at + size].double().cpu().numpy(), want_m)
        np.testing.assert_array_equal(now.nu_flat[at:at + size].double().cpu().numpy(), want_r ** 2)


@pytest.mark.parametrize("n", [1, 6, 333, 4000])
@pytest.mark.parametrize("shapes", ROWS)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_moments_are_moved(cuda, shapes, n, dtype):
    shapes = [(n, *s) for s in shapes]
    mu, nu = moments(shapes, n, cuda)
    params = [torch.zeros(s, device=cuda) for s in shapes]
    index = a_move(n, n, dtype, moved=0.1, freed=0.02).to(cuda)
    wide = AdamW(1e-3).restore(params, mu, nu, 7)
    eight = wide.convert(8)
    was = eight.moments()
    addresses = eight.mu_flat.data_ptr(), eight.nu_flat.data_ptr(), eight.fields.data_ptr()
    assert wide.move_rows_(index) is wide and eight.move_rows_(index) is eight
    assert addresses == (eight.mu_flat.data_ptr(), eight.nu_flat.data_ptr(), eight.fields.data_ptr())
    now = eight.convert(32)
    for i in range(len(shapes)):
        np.testing.assert_array_equal(raw(wide.mu[i]), raw(want_taken(mu[i], index)))
        np.testing.assert_array_equal(raw(wide.nu[i]), raw(want_taken(nu[i], index)))
        at, size = eight.offsets[i], len(pad(np.zeros(eight.counts[i])))
        if not size:
            continue
        want_m, _ = held(pad(want_taken(was[0][i], index).double().numpy()), 3)
        want_r, _ = held(pad(want_taken(was[1][i], index).double().sqrt().numpy()), 4)
        np.testing.assert_array_equal(now.mu_flat[at:at + size].double().cpu().numpy(), want_m)
        np.testing.assert_array_equal(now.nu_flat[at:at + size].double().cpu().numpy(), want_r ** 2)


def test_moments_that_are_not_finite_and_tiny_ones_move(cuda):
    """A NaN moves with its row and spreads to nobody; a root above zero stays above zero, the largest and the smallest exponents too."""
    n = 512
    m = torch.ones(n, 3, device=cuda)
    v = torch.ones(n, 3, device=cuda)
    m[5, 1], v[6, 2] = float("inf"), float("nan")
    m[7], v[7] = 3e38, 3e38
    v[300:] = 1e-38
    m[300:] = 1e-38
    state = AdamW(1e-3, moment_bits=8).restore([torch.zeros(n, 3, device=cuda)], [m], [v], 1)
    before = [x[0].cpu() for x in state.moments()]
    index = torch.arange(n, dtype=torch.int32)
    index[10:13] = torch.tensor([5, 6, 7])
    state.move_rows_(index.to(cuda))
    mu, nu = [x[0].cpu() for x in state.moments()]
    assert bool(torch.isnan(mu[5, 1])) and bool(torch.isnan(mu[10, 1])) and bool(torch.isnan(nu[6, 2])) and bool(torch.isnan(nu[11, 2]))
    assert torch.equal(mu[12], before[0][7]) and torch.equal(nu[12], before[1][7])
    assert int(torch.isnan(mu).sum()) == 2 and int(torch.isnan(nu).sum()) == 2
    assert bool((nu[300:] > 0).all()) and torch.equal(mu[300:], before[0][300:])


@pytest.mark.parametrize("row", [16, 48, 64, 272, 3, 4, 1, 45])
@pytest.mark.parametrize("kind", ["near", "wide", "tiny", "odd"])
def test_moments_of_all_sizes_side_by_side(cuda, row, kind):
    """Rows whose exponents differ a little, by all of float32's range, lie at its lower end, and with values that are not finite
    and rows of zeros between: what the way by 32 bits gives, value by value."""
    n = 1200
    gen = torch.Generator().manual_seed(row)
    low, high = {"near": (-2, 2), "wide": (-37, 37), "tiny": (-44, -30), "odd": (-20, 20)}[kind]
    size = 10.0 ** (torch.rand(n, 1, generator=gen).double() * (high - low) + low)
    m = (torch.randn(n, row, generator=gen).double() * size).float()
    # roots whose squares are float32s: the way by 32 bits goes through them
    size = 10.0 ** (torch.rand(n, 1, generator=gen).double() * (min(high, 18) - max(low, -18)) + max(low, -18))
    v = ((torch.rand(n, row, generator=gen).double() * size) ** 2).clamp(max=1e37).float()
    zero = torch.rand(n, generator=gen) < 0.2
    m[zero], v[zero] = 0.0, 0.0
    if kind == "odd":
        for value in (float("nan"), float("inf"), -float("inf")):
            m[torch.rand(n, row, generator=gen) < 3e-4] = value
        v[torch.rand(n, row, generator=gen) < 3e-4] = float("inf")
    opt = AdamW(1e-3, moment_bits=8)
    state = opt.restore([torch.zeros(n, row, device=cuda)], [m.to(cuda)], [v.to(cuda)], 1)
    was = [x[0].cpu() for x in state.moments()]

    def check(got, index):
        rows = [want_taken(x, index).to(cuda) for x in was]
        want = opt.restore([torch.zeros_like(rows[0])], [rows[0]], [rows[1]], 1)
        for a, b in zip(got.moments(), want.moments()):
            a, b = a[0].cpu(), b[0].cpu()
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())

    for index in (an_index(n, 1500, row, torch.int32), torch.randperm(n, generator=gen)):
        check(state.take_rows(index.to(cuda)), index)
    index = a_move(n, row, torch.int32, moved=0.1, freed=0.05)
    check(state.move_rows_(index.to(cuda)), index)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n, shapes", [
    (40, [(8208,), (20000,), (3,), (8192,)]),           # long rows, dealt out piece by piece
    (130, [(1 + i % 19,) for i in range(150)]),         # more tensors than a launch holds
    (600_001, [(1,), (2,), (3,), (16,)]),               # more than 512 rows a CU
    (262_145, [(5,), (32,), (0,)])])
def test_moments_of_long_rows_many_tensors_and_many_rows(cuda, n, shapes, dtype):
    """Taken and moved against the way by 32 bits."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    mu, nu = [], []
    for s in shapes:
        size = torch.exp(torch.randn(n, 1, generator=gen, device=cuda) * 2.0 - 9.0)
        mu.append(torch.randn(n, *s, generator=gen, device=cuda) * size)
        nu.append((torch.rand(n, *s, generator=gen, device=cuda) * size) ** 2)
    opt = AdamW(1e-3, moment_bits=8)
    state = opt.restore([torch.zeros_like(x) for x in mu], mu, nu, 1)
    was = state.moments()

    def check(got, index):
        index = index.to(cuda).long()
        there = ((index >= 0) & (index < n))[:, None]
        rows = [[torch.where(there, x[index.clamp(0, n - 1)], 0.0) for x in xs] for xs in was]
        want = opt.restore([torch.zeros_like(x) for x in rows[0]], *rows, 1)
        # (the values: blocks that a move leaves alone may hold them under a larger exponent than a new encoding)
        for xs, ys in zip(got.moments(), want.moments()):
            assert all([torch.equal(a, b) for a, b in zip(xs, ys)])

    index = an_index(n, n + 77, 3, dtype)
    check(state.take_rows(index.to(cuda)), index)
    index = a_move(n, 5, dtype, moved=0.2, freed=0.05)
    check(state.move_rows_(index.to(cuda)), index)


def test_masters_follow(cuda):
    for moment_bits in (32, 8):
        p = [torch.randn(200, 3, device=cuda).bfloat16(), torch.randn(200, device=cuda).half()]
        opt = AdamW(1e-2, moment_bits=moment_bits, master_weights=True)
        state = opt.init(p)
        for _ in range(2):
            opt.step(p, [torch.randn_like(x) for x in p], state)
        index = an_index(200, 300, 2, torch.int32).to(cuda)
        q, taken = take_rows(p, index), state.take_rows(index)
        for a, b in zip(state.master, taken.master):
            np.testing.assert_array_equal(raw(b), raw(want_taken(a, index)))
        assert bool((taken.master_flat[taken.counts[0]:taken.offsets[1]] == 0).all())
        opt.step(q, [torch.randn_like(x) for x in q], taken)  # a state like any other
        assert taken.count == 3 and state.count == 2
        index = a_move(200, 6, torch.int32).to(cuda)
        before = [x.clone() for x in state.master]
        state.move_rows_(index)
        for a, b in zip(before, state.master):
            np.testing.assert_array_equal(raw(b), raw(want_taken(a, index)))


def a_state(cuda, opt, n=2500, capacity=4000, seed=0):
    from jax_gs_amd.training.density import init_density_state

    gen = torch.Generator().manual_seed(seed)
    g = Gaussians(*[torch.randn(n, *s, generator=gen).to(cuda) for s in ((3,), (3,), (4,), (1,), (16, 3))])
    state = init_density_state(g, opt, capacity)
    # holes, as pruning leaves them
    state.active_mask[torch.randperm(n, generator=gen)[:n // 5].to(cuda)] = 0
    state.grad_accum.uniform_(0, 4e-4)
    state.denom.random_(0, 5)
    state.max_radii.uniform_(0, 500)
    return state


RATES = {f: 1e-2 for f in FIELDS}


@pytest.mark.parametrize("opt", [Adam(RATES), AdamW(RATES), AdamW(RATES, moment_bits=8), None], ids=["adam", "32", "8", "none"])
@pytest.mark.parametrize("capacity", [1500, 2000, 6000])
def test_resize_density_state(cuda, opt, capacity):
    """Compacted, cut to a budget or grown: everything of a Gaussian stays together, in its order, padding as
    init_density_state's, and training goes on."""
    from jax_gs_amd.training.density import resize_density_state

    state = a_state(cuda, opt)
    gen = torch.Generator(device=cuda).manual_seed(1)
    grads = lambda s: Gaussians(*[torch.randn(getattr(s.gaussians, f).shape, generator=gen, device=cuda) for f in FIELDS])
    if opt is not None:
        opt.step(state.gaussians, grads(state), state.opt_state, state.active_mask)
    on = state.active_mask.cpu().bool()
    logits = state.gaussians.opacities.cpu().reshape(-1).numpy()
    keep = on.nonzero().reshape(-1).numpy()
    if len(keep) > capacity:
        keep = np.sort(keep[np.argsort(-logits[keep], kind="stable")[:capacity]])
    k = len(keep)
    assert k == min(capacity, int(on.sum()))
    new = resize_density_state(state, capacity)
    assert new.num_active == k == int(new.active_mask.sum()) and new.active_mask.dtype == torch.uint8
    assert bool(new.active_mask[:k].all())
    for f in FIELDS:
        a, b = getattr(state.gaussians, f).cpu(), getattr(new.gaussians, f).cpu()
        assert b.shape == (capacity, *a.shape[1:]) and torch.equal(b[:k], a[keep])
        rest = torch.zeros_like(b[k:])
        if f == "quaternions":
            rest[:, 0] = 1.0
        assert torch.equal(b[k:], rest)
    for f in ("grad_accum", "denom", "max_radii"):
        a, b = getattr(state, f).cpu(), getattr(new, f).cpu()
        assert a.dtype == b.dtype and torch.equal(b[:k], a[keep]) and not bool(b[k:].any())
    if opt is None:
        assert new.opt_state is None
        return
    s, t = state.opt_state, new.opt_state
    assert t.count == 1
    if getattr(s, "bits", 32) == 32:
        for a, b in ((s.mu, t.mu), (s.nu, t.nu)):
            for f in FIELDS:
                assert torch.equal(b[f][:k].cpu(), a[f].cpu()[keep]) and not bool(b[f][k:].any())
    else:
        index = torch.from_numpy(np.concatenate([keep, np.full(capacity - k, -1)])).to(cuda)
        again = s.take_rows(index)
        assert torch.equal(again.mu_flat, t.mu_flat) and torch.equal(again.nu_flat, t.nu_flat)
    opt.step(new.gaussians, grads(new), t, new.active_mask)
    assert all(bool(torch.isfinite(getattr(new.gaussians, f)).all()) for f in FIELDS)


@pytest.mark.parametrize("opt", [Adam(RATES), AdamW(RATES, moment_bits=8)], ids=["adam", "8"])
def test_what_else_a_program_keeps_follows_density_control(cuda, opt):
    """densify_and_prune's sources move a table of features as they moved the Gaussians; the 8-bit moments are those of their sources."""
    from jax_gs_amd.training.density import densify_and_prune

    state = a_state(cuda, opt)
    state.gaussians.scales.fill_(-2.0)
    state.gaussians.scales[::3] = -5.0
    gen = torch.Generator(device=cuda).manual_seed(1)
    grads = Gaussians(*[torch.randn(getattr(state.gaussians, f).shape, generator=gen, device=cuda) for f in FIELDS])
    opt.step(state.gaussians, grads, state.opt_state, state.active_mask)
    features = state.gaussians.quaternions.clone()  # nothing but the moves changes quaternions
    was = [x.reshape(4000, -1).cpu() for m in state.opt_state.moments() for x in m.values()] if opt.__class__ is AdamW else None
    densify_and_prune(state, grad_threshold=1e-4, extent=5.0, sources=True, generator=gen)
    clones, splits = state.last_counts[:2].tolist()
    index = state.last_sources
    assert clones > 0 and splits > 0 and int((index.cpu() != torch.arange(4000)).sum()) == clones + splits
    move_rows_([features], index)
    assert torch.equal(features, state.gaussians.quaternions)
    if was is None:
        return
    now = [x.reshape(4000, -1).cpu() for m in state.opt_state.moments() for x in m.values()]
    for i, (a, b) in enumerate(zip(was, now)):
        want, _ = held(pad(want_taken(a, index).double().numpy() ** (1.0 if i < 5 else 0.5)), 3 if i < 5 else 4)
        np.testing.assert_array_equal(b.reshape(-1).double().numpy(), want[:b.numel()] ** (1 if i < 5 else 2))
    assert densify_and_prune(state, densify_enabled=False).last_sources is not None


@pytest.mark.parametrize("kind", ["adam", "8"])
def test_a_run_with_all_of_them(cuda, kind):
    """Clipped steps, density control with a table of features, a cut to a budget and a larger capacity, in turn: training
    goes on, the features stay with their Gaussians, and what is rendered does not change by a resize."""
    from jax_gs_amd import render, scenes
    from jax_gs_amd.training.adamw import make_adamw
    from jax_gs_amd.training.density import densify_and_prune, init_density_state, resize_density_state
    from jax_gs_amd.training.optimizer import make_optimizer
    from jax_gs_amd.training.trainer import train_step

    sc = scenes.make_scene(1, n=1500, width=96, height=64)
    g, cam, tgt, _ = scenes.to_torch(sc, "cuda:0")
    opt = make_optimizer(1.0, 100, max_grad_norm=0.01) if kind == "adam" else make_adamw(1.0, 100, moment_bits=8, max_grad_norm=0.01)
    static = (cam.W, cam.H, cam.fx, cam.fy, cam.cx, cam.cy)
    state = init_density_state(g, opt, 2000)
    features = torch.randn(2000, 5, device=cuda).half()
    for round in range(3):
        for _ in range(3):
            state, loss, metrics = train_step(state, tgt, cam.W2C, static, opt, sh_degree=3)
            assert bool(torch.isfinite(loss)) and bool(torch.isfinite(metrics["grad_norm"]))
        state.grad_accum.zero_()
        state.grad_accum[:200], state.denom[:200] = 1.0, 1
        tag = state.gaussians.quaternions.clone()
        densify_and_prune(state, extent=5.0, sources=True, generator=torch.Generator(device=cuda).manual_seed(round))
        assert int(state.last_counts[0] + state.last_counts[1]) > 0
        move_rows_([features, tag], state.last_sources)
        assert torch.equal(tag, state.gaussians.quaternions)
        active = int(state.active_mask.sum())
        # to a capacity that holds them all, then to a smaller budget, then to a larger capacity
        for capacity in (active, 1200, 2500):
            keep = best_rows(state.gaussians.opacities.reshape(-1), capacity, state.active_mask)
            before = render(state.gaussians, cam, mask=state.active_mask.bool(), sh_degree=3)[0]
            state, features, old = resize_density_state(state, capacity), take_rows(features, keep), features
            k = state.num_active
            assert torch.equal(features[:k], old[keep[:k].long()]) and not bool(features[k:].any())
            if capacity != 1200:
                after = render(state.gaussians, cam, mask=state.active_mask.bool(), sh_degree=3)[0]
                assert torch.equal(before, after)
    assert state.opt_state.count == 9 and state.gaussians.means.shape[0] == 2500


def test_sources_only_where_they_are_asked_for(cuda):
    from jax_gs_amd.training.density import densify_and_prune

    state = a_state(cuda, Adam(RATES))
    assert densify_and_prune(state, densify_enabled=False).last_sources is None
    densify_and_prune(state, densify_enabled=False, sources=True)
    assert torch.equal(state.last_sources.cpu(), torch.arange(4000, dtype=torch.int32))


def test_captured_and_replayed_with_other_inputs(cuda):
    """Every call into one graph: replays between eager work give the eager results for the index and values of the moment."""
    n = 5000
    x, pool = torch.randn(n, 7, device=cuda), torch.randn(n, 3, device=cuda)
    scores = torch.randn(n, device=cuda)
    index = a_move(n, 1, torch.int32).to(cuda)
    opt = AdamW(1e-3, moment_bits=8)
    state = opt.restore([pool], [torch.randn(n, 3, device=cuda)], [torch.rand(n, 3, device=cuda)], 5)

    def run():
        keep = best_rows(scores, 3000)
        taken = take_rows([x, scores], keep)
        move_rows_([pool], index)
        state.move_rows_(index)
        return [keep, *taken, state.take_rows(keep).mu_flat]

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for k in range(4):
        x.normal_()
        scores.normal_()
        pool.normal_()
        index.copy_(a_move(n, 10 + k, torch.int32))
        saved = pool.clone(), state.mu_flat.clone(), state.nu_flat.clone(), state.fields.clone()
        graph.replay()
        got = [t.clone() for t in captured] + [pool.clone(), state.mu_flat.clone()]
        for a, b in zip((pool, state.mu_flat, state.nu_flat, state.fields), saved):
            a.copy_(b)
        want = run() + [pool, state.mu_flat]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_on_another_stream(cuda):
    """Work queued on a side stream, with its inputs made there."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn(3_000_000, 8, device=cuda)
        scores = x[:, 0].contiguous()
        keep = best_rows(scores, 1_000_000)
        got = take_rows(x, keep)
        y = x.clone()
        index = torch.arange(3_000_000, device=cuda, dtype=torch.int32)
        index[5::7] = 0
        move_rows_(y, index)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, x[keep.long()]) and torch.equal(y, x[index.long()])


def test_device_refusals(cuda):
    x = torch.zeros(5, 3, device=cuda)
    index = torch.zeros(5, dtype=torch.int32, device=cuda)
    with pytest.raises(TypeError, match="int32 or int64"):
        take_rows(x, index.short())
    with pytest.raises(ValueError, match="one dimension"):
        take_rows(x, index.view(5, 1))
    with pytest.raises(ValueError, match="the index is on cpu"):
        take_rows(x, index.cpu())
    with pytest.raises(ValueError, match="4 indices for 5 rows"):
        move_rows_(x, index[:4])
    with pytest.raises(ValueError, match="left must be"):
        move_rows_(x, index, left=torch.zeros(1, device=cuda))
    with pytest.raises(ValueError, match="5 rows, not 4"):
        take_rows([x[:4], x], index)
    leaf = torch.zeros(5, 3, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        take_rows(leaf, index)
    state = AdamW(1e-3).init([x, torch.zeros(4, device=cuda)])
    with pytest.raises(ValueError, match="same rows"):
        state.take_rows(index)
    state = AdamW(1e-3, moment_bits=8).init([x])
    with pytest.raises(ValueError, match="4 indices for 5 rows"):
        state.move_rows_(index[:4])
    other = a_state(cuda, AdamW(RATES, moment_bits=8))
    other.opt_state = AdamW(RATES, moment_bits=8).init(take_rows(other.gaussians, index))
    before = other.active_mask.clone()
    with pytest.raises(ValueError, match="capacity rows"):
        from jax_gs_amd.training.density import densify_and_prune

        densify_and_prune(other, extent=1e-3)
    assert torch.equal(other.active_mask, before)
    with pytest.raises(ValueError, match="capacity 0"):
        from jax_gs_amd.training.density import resize_density_state

        resize_density_state(a_state(cuda, None), 0)

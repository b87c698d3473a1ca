"""The paths that are taken from a size on: outputs and gradients past the caches (160 MiB together), tables of so many rows that
workgroups look at more of them."""
import pytest
import torch

from jax_gs_amd.training.adamw import AdamW, clip_grads_
from jax_gs_amd.training.rows import move_rows_, take_rows

pytestmark = pytest.mark.gpu
PAST = 160 << 20


def raw(t):
    """A tensor's rows as bytes."""
    return t.contiguous().view(torch.uint8) if t.dim() > 1 else t.contiguous().view(torch.uint8).view(len(t), -1)


def some_bytes(n, row, gen, device):
    return torch.randint(0, 256, (n, row), generator=gen, device=device, dtype=torch.uint8)


def rows_of(t, index, fill=None):
    """Row by row by torch's own indexing, as bytes."""
    there = (index >= 0) & (index < len(t))
    got = raw(t)[torch.where(there, index, 0)]
    return torch.where(there[:, None], got, 0 if fill is None else fill.reshape(1, -1).view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rows_taken_past_the_caches(cuda, dtype):
    """Rows of fewer than 16 bytes, of 16 and of more that are multiples of it and not, at even and odd addresses, with fills, entries
    that are no rows, and outputs that end inside a vector and inside a workgroup's part."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    n, count = 1_500_001, 1_300_003
    index = torch.randint(0, n, (count,), generator=gen, device=cuda)
    odd = torch.rand(count, generator=gen, device=cuda)
    index[odd < 0.05] = -1
    index[(odd >= 0.05) & (odd < 0.08)] = n
    index[-1] = n - 1
    tensors, fills = [], []
    for i, row in enumerate((1, 2, 5, 12, 15, 16, 17, 48, 90)):
        tensors.append(some_bytes(n, row, gen, cuda))
        fills.append(some_bytes(1, row, gen, cuda)[0] if i % 2 else None)
    wide = some_bytes(n, 31, gen, cuda)
    tensors += [wide[:, 3:16], wide[:, 1:20]]  # rows of 13 and 19 bytes, apart
    fills += [None, some_bytes(1, 19, gen, cuda)[0]]
    assert sum(count * t.shape[1] for t in tensors) >= PAST
    got = take_rows(tensors, index.to(dtype), fill=fills)
    for t, f, g in zip(tensors, fills, got):
        assert torch.equal(g, rows_of(t, index, f)), t.shape
    # each kind of rows by itself
    for row in (12, 90, 192):
        t = some_bytes(n, row, gen, cuda)
        more = torch.cat([index] * -(-PAST // (row * count))).to(dtype)
        (g,) = take_rows([t], more)
        assert g.nbytes >= PAST and torch.equal(g, rows_of(t, more.long())), row


@pytest.mark.parametrize("masters", [False, True])
def test_a_large_state_taken(cuda, masters):
    """Moments and masters in 32 bits: the last 256 elements of every tensor end in zeros."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    n, count = 400_001, 390_011
    params = [torch.zeros(n, *s, device=cuda, dtype=torch.bfloat16 if masters else torch.float32) for s in ((16, 3), (45,), (3,), ())]
    mu = [torch.randn(p.shape, generator=gen, device=cuda) for p in params]
    nu = [torch.rand(p.shape, generator=gen, device=cuda) for p in params]
    state = AdamW(1e-3, master_weights=masters).restore(params, mu, nu, 2, master=mu if masters else None)
    index = torch.randint(-1000, n, (count,), generator=gen, device=cuda)
    taken = state.take_rows(index)
    assert taken.mu_flat.nbytes + taken.nu_flat.nbytes >= PAST
    for flat, own in ((taken.mu_flat, mu), (taken.nu_flat, nu), (taken.master_flat, mu if masters else [])):
        for i, x in enumerate(own):
            at, size = taken.offsets[i], taken.counts[i]
            assert torch.equal(flat[at:at + size].view(count, -1).view(torch.uint8), rows_of(x.view(n, -1), index))
            end = taken.offsets[i + 1] if i + 1 < len(own) else taken.size
            assert not bool(flat[at + size:end].any())


def check_clipped(grads, before, norms, max_norm, on=None):
    """As one rounding of the factor, one of the product and one to the type."""
    keep = [slice(None) if on is None else on] * len(grads)
    total = torch.stack([b[k].double().square().sum() for b, k in zip(before, keep)]).sum().sqrt()
    factor = torch.clamp(max_norm / (total + 1e-6), max=1.0)
    assert abs(float(norms.total) / float(total) - 1.0) <= 2.0 ** -23 and abs(float(norms.scale) / float(factor) - 1.0) <= 2.0 ** -23
    for g, b, k in zip(grads, before, keep):
        info = torch.finfo(g.dtype)
        want = b[k].double() * factor
        bound = want.abs() * (info.eps / 2 + 2.0 ** -22) + info.tiny * info.eps / 2
        assert bool(((g[k].double() - want).abs() <= bound).all()), g.dtype


@pytest.mark.parametrize("of", [[torch.float32], [torch.bfloat16], [torch.float16], [torch.float32, torch.bfloat16, torch.float16]])
def test_gradients_clipped_past_the_caches(cuda, of):
    """Views from an odd element on, of a length that is no multiple of a vector or of a run; what is around them stays."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    buffers, grads = [], []
    for i, dtype in enumerate(of):
        size = PAST // (len(of) * (4 if dtype == torch.float32 else 2)) + 5003 + i
        buffers.append((torch.randn(size + 4, generator=gen, device=cuda) * 0.1).to(dtype))
        grads.append(buffers[-1][1:1 + size])
    grads.append((torch.randn(7, generator=gen, device=cuda)).to(of[0]))
    before, around = [g.clone() for g in grads], [b[[0, -3, -2, -1]].clone() for b in buffers]
    assert sum(g.nbytes for g in grads) >= PAST
    norms = clip_grads_(grads, 3.0)
    check_clipped(grads, before, norms, 3.0)
    assert all(torch.equal(b[[0, -3, -2, -1]], a) for b, a in zip(buffers, around))
    for i in range(len(grads)):
        assert abs(float(norms.per_tensor[i]) / float(before[i].double().norm()) - 1.0) <= 2.0 ** -23


@pytest.mark.parametrize("row", [48, 45])
def test_masked_gradients_of_that_size(cuda, row):
    gen = torch.Generator(device=cuda).manual_seed(4)
    n = PAST // (4 * row) + 1001
    on = torch.rand(n, generator=gen, device=cuda) < 0.7
    grads = [torch.randn(n, row, generator=gen, device=cuda), torch.randn(n, generator=gen, device=cuda).bfloat16()]
    for g in grads:
        g[~on] = float("nan")
    before = [g.clone() for g in grads]
    check_clipped(grads, before, clip_grads_(grads, 3.0, active_mask=on), 3.0, on)
    assert all(bool(torch.isnan(g[~on]).all()) for g in grads)


@pytest.mark.parametrize("n", [1 << 18, (1 << 18) + 1, (1 << 19) + 1, 1_100_003])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rows_moved_in_large_tables(cuda, n, dtype):
    """Up to 2^18 rows a workgroup looks at 64 of them, up to 2^19 at 128, beyond at 256; rows that change lie scattered and together."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    scattered = torch.arange(n, device=cuda)
    change = torch.rand(n, generator=gen, device=cuda) < 0.3
    stay = (~change).nonzero().reshape(-1)
    scattered[change] = stay[torch.randint(0, len(stay), (int(change.sum()),), generator=gen, device=cuda)]
    scattered[change & (torch.rand(n, generator=gen, device=cuda) < 0.2)] = -1
    together = torch.arange(n, device=cuda)
    together[n // 2:n // 2 + 20_000] = torch.arange(20_000, device=cuda)
    for index in (scattered, together):
        tensors = [some_bytes(n, row, gen, cuda) for row in (1, 12, 16, 59, 80)]
        fills = [None, None, some_bytes(1, 16, gen, cuda)[0], some_bytes(1, 59, gen, cuda)[0], None]
        want = [rows_of(t, index, f) for t, f in zip(tensors, fills)]
        left = torch.zeros(1, dtype=torch.int32, device=cuda)
        move_rows_(tensors, index.to(dtype), fill=fills, left=left)
        assert all(torch.equal(t, w) for t, w in zip(tensors, want)) and int(left) == 0

"""What clipping leaves alone it leaves bit by bit: masked rows beside others in one vector, and everything where some gradient is
not finite."""
import pytest
import torch

from jax_gs_amd.training.adamw import clip_grads_

pytestmark = pytest.mark.gpu
INTS = {torch.float32: torch.int32, torch.bfloat16: torch.int16, torch.float16: torch.int16}


def any_bits(shape, dtype, gen, device):
    """Any value of the type, NaNs with payloads, quiet and signalling, and gradual underflow among them."""
    size = torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * size), generator=gen, device=device, dtype=torch.uint8)
    return raw.view(dtype)


@pytest.mark.parametrize("dtype", list(INTS))
@pytest.mark.parametrize("row", [1, 2, 3, 5, 7, 8, 16, 48, 4099])
def test_masked_rows_keep_their_bits(cuda, dtype, row):
    gen = torch.Generator(device=cuda).manual_seed(row)
    n = 40_000 // row + 3
    on = torch.rand(n, generator=gen, device=cuda) < 0.5
    g = any_bits((n, row), dtype, gen, cuda)
    g[on] = torch.randn(int(on.sum()), row, generator=gen, device=cuda).to(dtype)
    before = g.clone()
    norms = clip_grads_([g], 0.25, active_mask=on)
    assert 0.0 < float(norms.scale) < 1.0
    assert torch.equal(g[~on].view(INTS[dtype]), before[~on].view(INTS[dtype]))
    assert not torch.equal(g[on], before[on])


@pytest.mark.parametrize("dtype", list(INTS))
def test_gradients_that_are_not_finite_stay(cuda, dtype):
    gen = torch.Generator(device=cuda).manual_seed(1)
    grads = [any_bits((1, 70_001), dtype, gen, cuda), torch.randn(333, generator=gen, device=cuda).to(dtype)]
    before = [g.clone() for g in grads]
    for mask in (None, torch.ones(1, device=cuda)):
        some = grads[:1] if mask is not None else grads
        norms = clip_grads_(some, 1.0, active_mask=mask)
        assert bool(torch.isnan(norms.scale))
        assert all(torch.equal(g.view(INTS[dtype]), b.view(INTS[dtype])) for g, b in zip(grads, before))

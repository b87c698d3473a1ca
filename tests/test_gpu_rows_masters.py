"""Rows that come from nowhere: the float32 masters of half-typed parameters hold the parameters' fill, so that the next step
goes on from it."""
import pytest
import torch

from jax_gs_amd.training.adamw import AdamW
from jax_gs_amd.training.rows import move_rows_, take_rows

N = 300


def a_model(cuda, bits):
    gen = torch.Generator(device=cuda).manual_seed(bits)
    shapes = {"w": ((N, 3, 2), torch.bfloat16), "q": ((N, 4), torch.float16), "s": ((N,), torch.bfloat16), "e": ((N, 0), torch.float16)}
    params = {k: torch.randn(s, generator=gen, device=cuda).to(t) for k, (s, t) in shapes.items()}
    opt = AdamW(1e-2, moment_bits=bits, master_weights=True)
    state = opt.init(params)
    for _ in range(2):
        opt.step(params, {k: torch.randn(p.shape, generator=gen, device=cuda).to(p.dtype) for k, p in params.items()}, state)
    fill = {"w": torch.randn(3, 2, generator=gen, device=cuda).bfloat16(),
            "q": torch.tensor([1.0, 0, 0, 0], device=cuda).half(), "s": None, "e": None}
    return params, opt, state, fill


def check(params, opt, state, nowhere, fill):
    nowhere = nowhere.to(params["w"].device)
    assert int(nowhere.sum()) > 0
    for k, p in params.items():
        want = torch.zeros(p.shape[1:], device=p.device) if fill[k] is None else fill[k].float()
        assert torch.equal(state.master[k][nowhere], want.expand(state.master[k][nowhere].shape)), k
        assert torch.equal(state.master[k].to(p.dtype), p), k
    before = {k: p.clone() for k, p in params.items()}
    # nothing moves what has no gradient and no moments
    opt.step(params, {k: torch.zeros_like(p) for k, p in params.items()}, state)
    for k, p in params.items():
        assert torch.equal(p[nowhere], before[k][nowhere]), k


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_masters_of_rows_taken_from_nowhere(cuda, bits, dtype):
    params, opt, state, fill = a_model(cuda, bits)
    index = torch.randint(-N // 3, N + 20, (N + 57,), generator=torch.Generator().manual_seed(1)).to(dtype)
    taken = state.take_rows(index.to(cuda), fill=fill)
    check(take_rows(params, index.to(cuda), fill=fill), opt, taken, (index < 0) | (index >= N), fill)
    # without a fill the masters are zero there, as the parameters are
    none = dict.fromkeys(fill)
    check(take_rows(params, index.to(cuda)), opt, state.take_rows(index.to(cuda)), (index < 0) | (index >= N), none)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_masters_of_rows_that_are_freed(cuda, bits):
    params, opt, state, fill = a_model(cuda, bits)
    index = torch.arange(N, dtype=torch.int32)
    index[5::7] = -1
    index[6::7] = 0
    move_rows_(params, index.to(cuda), fill=fill)
    assert state.move_rows_(index.to(cuda), fill=fill) is state
    check(params, opt, state, index < 0, fill)
    # a fill that lies in the masters themselves, of a row that changes
    index = torch.arange(N, dtype=torch.int32)
    index[::2] = -1
    row = state.master["w"][0].clone()
    state.move_rows_(index.to(cuda), fill={**fill, "w": state.master["w"][0]})
    assert torch.equal(state.master["w"][::2], row.expand(N // 2, 3, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_lazily_negated_or_strided_fill(cuda, bits):
    params, opt, state, fill = a_model(cuda, bits)
    fill["q"] = torch._neg_view(torch.arange(8.0, device=cuda).half()[::2])
    fill["w"] = torch.randn(2, 3, device=cuda).bfloat16().t()
    index = torch.full((5,), -1, device=cuda)
    check(take_rows(params, index, fill=fill), opt, state.take_rows(index, fill=fill), torch.ones(5, dtype=torch.bool), fill)


@pytest.mark.gpu
def test_fills_that_are_no_rows_are_refused(cuda):
    params, opt, state, fill = a_model(cuda, 32)
    index = torch.full((N,), -1, device=cuda)
    masters = state.master_flat.clone()
    for bad in (torch.ones(3, device=cuda), torch.ones(1, 4, device=cuda), torch.ones(4), torch.ones(4, dtype=torch.int32, device=cuda), 1.0):
        for call in (state.take_rows, state.move_rows_):
            with pytest.raises((ValueError, TypeError), match="fill"):
                call(index, fill={**fill, "q": bad})
    for call in (state.take_rows, state.move_rows_):
        with pytest.raises(ValueError, match="w"):
            call(index, fill={"q": fill["q"]})
        with pytest.raises(ValueError, match="1 fills for 4"):
            call(index, fill=[fill["q"]])
    assert torch.equal(state.master_flat, masters)
    # a state without masters takes and checks the same fill, and has no use for it
    plain = AdamW(1e-2).init(params)
    assert not bool(plain.take_rows(index, fill=fill).mu_flat.any())
    with pytest.raises((ValueError, TypeError), match="fill"):
        plain.take_rows(index, fill={**fill, "q": torch.ones(3, device=cuda)})

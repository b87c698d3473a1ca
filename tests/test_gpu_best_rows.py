"""The best rows against a stable sort on the host."""
import numpy as np
import pytest
import torch

from jax_gs_amd.training.rows import best_rows

pytestmark = pytest.mark.gpu


def want_best(scores, k, mask=None):
    n = len(scores if scores is not None else mask)
    rows = np.arange(n) if mask is None else np.flatnonzero(mask)
    x = np.zeros(n) if scores is None else scores.detach().cpu().double().numpy()
    x = x[rows]
    # NaN below everything, the lowest row first among equals
    order = np.lexsort((rows, -np.where(np.isnan(x), 0.0, x), np.isnan(x)))
    out = np.full(k, -1)
    best = np.sort(rows[order[:k]])
    out[:len(best)] = best
    return out


def check(scores, k, mask, cuda):
    got = best_rows(None if scores is None else scores.to(cuda), k, None if mask is None else torch.as_tensor(mask).to(cuda))
    assert got.dtype == torch.int32 and got.shape == (k,)
    np.testing.assert_array_equal(got.cpu().numpy(), want_best(scores, k, mask))


def some_scores(n, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=gen)
    if kind == "equal":
        x = torch.full((n,), -2.5)
    elif kind == "few":
        x = torch.randint(-2, 3, (n,), generator=gen).float()
    elif kind == "zeros":
        x = x * (torch.rand(n, generator=gen) < 0.3)  # zeros of both signs
    elif kind == "odd":
        odd = torch.tensor([float("nan"), -float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-45, -1e-45, 3e38, -3e38])
        x = odd[torch.randint(0, len(odd), (n,), generator=gen)]
    elif kind == "wide":
        x = x * torch.exp(torch.randn(n, generator=gen) * 20.0)
    elif kind == "close":
        x = 1.0 + torch.randint(0, 200, (n,), generator=gen) * 2.0 ** -23
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["normal", "equal", "few", "zeros", "odd", "wide", "close"])
@pytest.mark.parametrize("n", [1, 2, 65, 1000, 16384, 16385, 70001])
def test_best_rows(cuda, dtype, kind, n):
    scores = some_scores(n, kind, n).to(dtype)
    mask = torch.rand(n, generator=torch.Generator().manual_seed(n)) < 0.6
    for k in sorted({0, 1, n // 3, n - 1, n, n + 5}):
        check(scores, k, None, cuda)
        check(scores, k, mask.numpy(), cuda)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, k", [(3_000_000, 1_000_000), (1_048_576, 1), (2_000_003, 2_000_002)])
def test_best_of_many(cuda, dtype, n, k):
    scores = some_scores(n, "zeros", 1).to(dtype)
    check(scores, k, None, cuda)
    check(scores, k, (torch.rand(n, generator=torch.Generator().manual_seed(2)) < 0.8).numpy(), cuda)


@pytest.mark.parametrize("n", [1, 100, 40_000, 1_000_000])
def test_first_rows_of_a_mask(cuda, n):
    mask = torch.rand(n, generator=torch.Generator().manual_seed(n)) < 0.3
    for m in (mask, torch.zeros(n, dtype=torch.bool), torch.ones(n, dtype=torch.uint8)):
        for k in (0, 1, n // 4, n, n + 3):
            check(None, k, m.numpy(), cuda)


def test_masked_scores_do_not_count_whatever_they_are(cuda):
    scores = torch.arange(5000.0)
    mask = np.ones(5000, bool)
    mask[2000:] = False
    scores[2000:4000], scores[4000:] = float("nan"), float("inf")
    check(scores, 10, mask, cuda)
    check(scores, 3000, mask, cuda)


def test_no_rows_and_strided_scores(cuda):
    assert best_rows(torch.zeros(0, device=cuda), 3).tolist() == [-1, -1, -1]
    x = torch.randn(1000, 4)
    got = best_rows(x.to(cuda)[:, 2], 100)
    np.testing.assert_array_equal(got.cpu().numpy(), want_best(x[:, 2], 100))
    with pytest.raises(ValueError, match="one score"):
        best_rows(x.to(cuda), 5)
    with pytest.raises(TypeError, match="float64"):
        best_rows(x.double().to(cuda)[:, 0], 5)
    with pytest.raises(ValueError, match="active_mask"):
        best_rows(x.to(cuda)[:, 0], 5, active_mask=torch.ones(999, device=cuda))


@pytest.mark.parametrize("n", [0, 3, 5000, 40_000])
def test_many_more_than_there_are(cuda, n):
    """What lies behind the last row is written by many workgroups."""
    scores = some_scores(n, "normal", 1) if n else torch.zeros(0)
    for k in (300_000, 20_000_001):
        for x, mask in ((scores, None), (None, torch.arange(n) % 3 > 0)):
            got = best_rows(None if x is None else x.to(cuda), k, None if mask is None else mask.to(cuda))
            rows = torch.arange(n, device=cuda, dtype=torch.int32)
            rows = rows if mask is None else rows[mask.to(cuda)]
            assert torch.equal(got[:len(rows)], rows) and bool((got[len(rows):] == -1).all())

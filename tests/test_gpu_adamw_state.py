"""AdamW's state: streams, checkpoints, masters, and what a step leaves alone."""
import numpy as np
import pytest
import torch

from jax_gs_amd.training.adamw import AdamW, grad_norms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_on_a_stream_while_another_allocates(cuda, bits):
    """The state is made on one stream and stepped on another, while the first allocates and fills arrays of
    the powers' size: the bits of a run on one stream."""
    n = 4_000_000
    gen = torch.Generator(device=cuda).manual_seed(0)
    p = torch.randn(n, generator=gen, device=cuda)
    g = torch.randn(n, generator=gen, device=cuda)
    q = p.clone()
    opt = AdamW(1e-2, weight_decay=0.1, moment_bits=bits, max_grad_norm=1.0)
    a, b = opt.init(p), opt.init(q)
    for _ in range(8):
        opt.step(p, g, a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    filled = []
    for _ in range(8):
        with torch.cuda.stream(side):
            opt.step(q, g, b)
        filled += [torch.full((4,), 0.5, dtype=torch.float64, device=cuda) for _ in range(16)]
        del filled[:-8]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a.powers, b.powers) and a.count == b.count == 8
    np.testing.assert_allclose(a.powers.cpu().numpy()[:2], [0.9 ** 8, 0.999 ** 8], rtol=1e-14)
    assert torch.equal(p, q) and torch.equal(a.mu_flat, b.mu_flat) and torch.equal(a.nu_flat, b.nu_flat)


def test_a_converted_state_goes_on_by_itself(cuda):
    """Steps of the one leave the other's powers, which were the same."""
    g = torch.ones(1000, device=cuda)
    opt = AdamW(1e-2)
    p = torch.zeros(1000, device=cuda)
    a = opt.init(p)
    opt.step(p, g, a)
    b = a.convert(8)
    q = p.clone()
    for _ in range(3):
        opt.step(p, g, a)
    np.testing.assert_allclose(b.powers.cpu().numpy()[:2], [0.9, 0.999], rtol=1e-15)
    opt.step(q, g, b)
    np.testing.assert_allclose(b.powers.cpu().numpy()[:2], [0.9 ** 2, 0.999 ** 2], rtol=1e-15)
    np.testing.assert_allclose(a.powers.cpu().numpy()[:2], [0.9 ** 4, 0.999 ** 4], rtol=1e-14)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, row", [(400, 1), (333, 3), (100, 2), (9, 301), (7, 4)])
def test_masked_rows_keep_what_the_program_wrote(cuda, bits, dtype, rows, row):
    """Half parameters with masters: a program writes its tensor, not the masters.  Rows whose mask is off keep what
    it wrote, whoever their neighbours are, and their masters stay too; the others follow their masters."""
    gen = torch.Generator(device=cuda).manual_seed(rows)
    p = torch.randn(rows, row, generator=gen, device=cuda).to(dtype)
    on = torch.rand(rows, generator=gen, device=cuda) < 0.5
    on[:2] = torch.tensor([True, False], device=cuda)
    opt = AdamW(1e-2, moment_bits=bits, master_weights=True)
    state = opt.init([p])
    p.fill_(3.0)
    master = state.master[0].clone()
    opt.step([p], [torch.ones(rows, row, device=cuda).to(dtype)], state, active_mask=on)
    assert bool((p[~on] == 3.0).all()) and torch.equal(state.master[0][~on], master[~on])
    assert torch.equal(p[on], state.master[0][on].to(dtype)) and not bool((state.master[0][on] == master[on]).any())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_from_before_the_step_is_refused(cuda, bits):
    """A graph that saved a parameter would give its gradient with the values after the step."""
    p, q = (torch.randn(1000, device=cuda, requires_grad=True) for _ in range(2))
    opt = AdamW(1e-2, moment_bits=bits, max_grad_norm=1.0)
    state = opt.init([p, q])
    loss, other = (p * p).sum(), (q * q).sum()
    opt.step([p, q], [torch.ones_like(p), None], state)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    other.backward()
    assert torch.equal(q.grad, 2.0 * q.detach())
    (p * p).sum().backward()
    assert torch.equal(p.grad, 2.0 * p.detach())


def test_a_step_is_not_captured_but_the_norms_are(cuda):
    """The refusal under a real capture leaves the state as it was; gradient norms are replayed."""
    p = torch.zeros(5000, device=cuda)
    g = torch.randn(5000, device=cuda)
    opt = AdamW(1e-2)
    state = opt.init([p])
    opt.step([p], [g], state)
    grad_norms([g], max_norm=1.0)
    before = p.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = grad_norms([g], max_norm=1.0)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step([p], [g], state)
    assert state.count == 1
    for k in (1.0, 3.0, 0.5):
        g.normal_().mul_(k)
        graph.replay()
        want = grad_norms([g], max_norm=1.0)
        torch.cuda.synchronize()
        assert torch.equal(norms.total, want.total) and torch.equal(norms.scale, want.scale)
    assert torch.equal(p, before)
    opt.step([p], [g], state)
    assert state.count == 2 and not torch.equal(p, before)
    np.testing.assert_allclose(state.powers.cpu().numpy()[:2], [0.9 ** 2, 0.999 ** 2], rtol=1e-14)

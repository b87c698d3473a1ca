"""What AdamW hands to the native step, on the host: the device calls are recorded, not made."""
import ctypes
from array import array

import pytest
import torch

from jax_gs_amd import _lib
from jax_gs_amd.training import adamw
from jax_gs_amd.training.adamw import AdamW, AdamWState


class Recorder:
    """Stands in for the native library and for streams: keeps the arguments of every call, and which
    memory was recorded on which stream."""

    def __init__(self, monkeypatch):
        self.calls, self.recorded, self.stream = [], [], 0
        monkeypatch.setattr(_lib, "call", lambda name, *args: self.calls.append((name, args)))
        monkeypatch.setattr(_lib, "stream_handle", lambda device: ctypes.c_void_p(self.stream))
        monkeypatch.setattr(_lib, "tensors", lambda: self)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.stream)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: self.recorded.append((t.data_ptr(), s)))

    @staticmethod
    def pair(ps, gs, shapes, device):
        counts = array("q", [p.numel() for p in ps]).tobytes()
        return b"", b"", b"", b"", counts, None

    def __getattr__(self, name):  # whatever else the list module offers
        return lambda *args: None

    def steps(self):
        return [args for name, args in self.calls if name == "gs_adamw_step"]


def host_state(opt, shapes=((300,), (7,))):
    state = AdamWState(None, shapes, opt.moment_bits)
    state._allocate(torch.device("cpu"), zero=True)
    state._set_powers(opt._powers(0, torch.device("cpu")))
    return state


POWERS, NEXT = 20, 21  # places of powers and powers_next among gs_adamw_step's arguments


def test_powers_are_not_handed_back_while_another_stream_reads_them(monkeypatch):
    """A step on another stream than the one its powers were allocated on: their memory is recorded on the
    step's stream, so that the allocator's next user waits for it.  On one stream nothing is to be done."""
    native = Recorder(monkeypatch)
    opt = AdamW(1e-3)
    state = host_state(opt)
    ps = [torch.zeros(s) for s in state.shapes]
    held, want, owner = [], [], 0
    for stream in (0, 0, 64, 64, 64, 0, 96, 96):
        native.stream = stream
        held.append(state.powers)  # so that an address cannot come back
        if stream != owner:
            want.append((state.powers.data_ptr(), stream))
        owner = stream
        opt.step(ps, ps, state)
    assert native.recorded == want and len(want) == 3
    args = native.steps()
    assert [a[NEXT] for a in args[:-1]] == [a[POWERS] for a in args[1:]]
    assert state.powers.data_ptr() == args[-1][NEXT]


def test_powers_of_a_converted_state(monkeypatch):
    """Two states share the powers until each steps; neither step writes what the other reads."""
    native = Recorder(monkeypatch)
    opt = AdamW(1e-3)
    a = host_state(opt)
    native.stream = 64
    b = a.convert(8)
    ps = [torch.zeros(s) for s in a.shapes]
    held, shared = [a.powers], a.powers.data_ptr()
    for s in (a, b, a, b):
        opt.step(ps, ps, s)
        held.append(s.powers)
    args = native.steps()
    assert args[0][POWERS] == args[1][POWERS] == shared and len({x[NEXT] for x in args} | {shared}) == 5
    assert native.recorded == [(shared, 64), (shared, 64)]


@pytest.fixture
def on_host(monkeypatch):
    """States may be made of host tensors."""
    native = Recorder(monkeypatch)
    monkeypatch.setattr(adamw, "_device", lambda t, what: t.device)
    native.gather = lambda ts, device, what: (b"", b"", b"", None)
    return native


def checkpoint(opt, params):
    state = opt.init(params)
    return {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in state.state_dict().items()}


@pytest.mark.parametrize("bits, name, length", [
    (32, "mu_flat", 1), (32, "nu_flat", 511), (32, "powers", 3), (32, "powers", 1), (32, "master_flat", 511), (32, "master_flat", 1),
    (8, "mu_flat", 513), (8, "nu_flat", 1), (8, "powers", 8), (8, "master_flat", 513), (8, "fields", 1)])
def test_buffers_of_another_length_are_not_loaded(on_host, bits, name, length):
    """The native step takes their addresses alone: a short one would be read and written out of range."""
    params = [torch.zeros(300, dtype=torch.bfloat16)]
    opt = AdamW(1e-3, moment_bits=bits, master_weights=True)
    saved = checkpoint(opt, params)
    assert saved[name].shape[0] != length
    opt.load_state_dict(params, saved)
    bad = torch.zeros((length, *saved[name].shape[1:]), dtype=saved[name].dtype)
    with pytest.raises(ValueError, match=name):
        opt.load_state_dict(params, {**saved, name: bad})


def test_a_checkpoint_without_a_buffer_is_refused(on_host):
    params = [torch.zeros(300)]
    opt = AdamW(1e-3, moment_bits=8)
    saved = checkpoint(opt, params)
    for name in ("mu_flat", "nu_flat", "fields", "powers"):
        with pytest.raises(ValueError, match=name):
            opt.load_state_dict(params, {**saved, name: None})
    with pytest.raises(ValueError, match="32 or 8"):
        opt.load_state_dict(params, {**saved, "bits": 16})


def test_loaded_buffers_are_whole_and_the_states_own(on_host):
    """Strided and lazily negated tensors of the right length are loaded as their values."""
    params = [torch.zeros(300, dtype=torch.float16)]
    opt = AdamW(1e-3, master_weights=True)
    saved = checkpoint(opt, params)
    z = torch.complex(torch.zeros(512), torch.arange(512.0))
    saved["master_flat"] = z.conj().imag
    saved["mu_flat"] = torch.arange(1024.0)[::2]
    state = opt.load_state_dict(params, saved)
    for t, want in ((state.master_flat, -torch.arange(512.0)), (state.mu_flat, torch.arange(0.0, 1024.0, 2.0))):
        assert t.is_contiguous() and not t.is_neg() and torch.equal(t, want)
    state.powers.fill_(7.0)
    assert not (saved["powers"] == 7.0).any()


def test_masters_must_be_those_of_the_parameters(on_host):
    """Too few of them, or one value for a whole tensor, would leave weights to be computed from zeros or from
    that value."""
    params = [torch.ones(300, dtype=torch.bfloat16), torch.ones(7, dtype=torch.bfloat16)]
    zeros = [torch.zeros(300), torch.zeros(7)]
    opt = AdamW(1e-3, master_weights=True)
    good = [torch.full((300,), 1.001), torch.full((7,), 0.999)]
    state = opt.restore(params, zeros, zeros, 3, master=good)
    assert all(torch.equal(a, b) for a, b in zip(state.master, good))
    for bad in (good[:1], [good[0], good[1][:1]], [good[0], torch.ones(())], good + good, [good[0], torch.ones(8)]):
        with pytest.raises(ValueError, match="masters are not those"):
            opt.restore(params, zeros, zeros, 3, master=bad)
    with pytest.raises(ValueError, match="keeps none"):
        AdamW(1e-3).restore(params, zeros, zeros, 3, master=good)


@pytest.mark.parametrize("bits", [32, 8])
def test_masters_of_a_checkpoint_without_any(on_host, bits):
    """An optimizer that keeps masters makes them from the parameters, as init does; one that keeps none goes on
    with those that a checkpoint has."""
    params = [torch.randn(300).to(torch.bfloat16), torch.randn(7), torch.zeros(0, dtype=torch.float16)]
    without, keeps = AdamW(1e-3, moment_bits=bits), AdamW(1e-3, moment_bits=bits, master_weights=True)
    saved = checkpoint(without, params)
    assert saved["master_flat"] is None
    state = keeps.load_state_dict(params, saved)
    assert state.master_flat is not None and torch.equal(state.master_flat, keeps.init(params).master_flat)
    assert torch.equal(state.master[0], params[0].float())
    assert without.load_state_dict(params, saved).master_flat is None
    saved = checkpoint(keeps, params)
    saved["master_flat"] += 2.0 ** -12
    for opt in (keeps, without):
        assert torch.equal(opt.load_state_dict(params, saved).master_flat, saved["master_flat"])
    full = [p.float() for p in params]
    assert keeps.load_state_dict(full, checkpoint(keeps, full)).master_flat is None


SCALE = 19  # place of grad_scale among gs_adamw_step's arguments


def test_a_lazily_negated_scale_is_handed_on_as_its_value(on_host):
    """The imaginary part of a conjugate is float32 and reads as minus what lies in memory."""
    opt = AdamW(1e-3)
    ps = [torch.zeros(300)]
    state = opt.init(ps)
    scale = torch.tensor(complex(0.0, -0.5), dtype=torch.complex64).conj().imag
    assert scale.is_neg() and float(scale) == 0.5
    seen = []
    call = _lib.call
    _lib.call = lambda name, *args: (call(name, *args), seen.append(ctypes.c_float.from_address(args[SCALE]).value))
    try:
        opt.step(ps, ps, state, grad_scale=scale)
    finally:
        _lib.call = call
    assert seen == [0.5]


def test_norms_are_those_of_the_last_step(on_host):
    """A step that takes no norm leaves none behind from an earlier one."""
    clips, plain = AdamW(1e-3, max_grad_norm=1.0), AdamW(1e-3)
    ps = [torch.zeros(300)]
    state = clips.init(ps)
    clips.step(ps, ps, state)
    assert state.norms is not None
    plain.step(ps, ps, state)
    assert state.norms is None


@pytest.fixture
def counting(on_host, module=_lib.tensors):
    """The module that tells autograd of what was written is the built one."""
    on_host.written = module().written
    return on_host


def test_autograd_knows_that_a_step_writes(counting):
    """A graph that saved a parameter's or a master's values from before the step gives no gradient from those after
    it; one that saved a tensor without a gradient in the step goes on."""
    opt = AdamW(1e-3, master_weights=True)
    ps = [torch.randn(300, requires_grad=True), torch.randn(7, requires_grad=True), torch.randn(9).to(torch.bfloat16)]
    state = opt.init([p.detach() for p in ps])
    first, second = (ps[0] * ps[0]).sum(), (ps[1] * ps[1]).sum()
    scale = torch.ones((), requires_grad=True)
    third = (state.master[2] * scale).sum()
    opt.step(ps, [torch.zeros(300), None, torch.zeros(9)], state)
    for y in (first, third):
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
    second.backward()
    assert torch.equal(ps[1].grad, 2.0 * ps[1].detach())


def test_versions_of_what_a_step_writes(counting):
    opt = AdamW(1e-3, moment_bits=8)
    ps = [torch.zeros(300), torch.zeros(7)]
    state = opt.init(ps)
    count = lambda: [t._version for t in (*ps, state.mu_flat, state.nu_flat, state.fields)]  # noqa: E731
    before = count()
    opt.step(ps, [ps[0], None], state)
    assert [a - b for a, b in zip(count(), before)] == [1, 0, 1, 1, 1]
    before = count()
    state.set_moments(AdamW(1e-3).init(ps))
    assert [a > b for a, b in zip(count(), before)] == [False, False, True, True, True]
    with torch.inference_mode():
        qs = [torch.zeros(300), torch.zeros(7)]
    opt.step(qs, qs, opt.init(qs))  # they count none


def test_a_refused_step_writes_nothing(counting, monkeypatch):
    opt = AdamW(1e-3)
    ps = [torch.zeros(300)]
    state = opt.init(ps)

    def refuse(name, *args):
        raise ValueError("refused")

    monkeypatch.setattr(_lib, "call", refuse)
    with pytest.raises(ValueError, match="refused"):
        opt.step(ps, ps, state)
    assert ps[0]._version == 0 and state.count == 0


def test_a_step_under_graph_capture_is_refused(on_host, monkeypatch):
    """A captured step holds the addresses of the powers that the state lets go of, one t and one rounding key."""
    opt = AdamW(1e-3, max_grad_norm=1.0)
    ps = [torch.zeros(300)]
    state = opt.init(ps)
    powers = state.powers
    made = len(on_host.calls)
    monkeypatch.setattr(_lib, "capturing", lambda device: True, raising=False)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step(ps, ps, state)
    assert len(on_host.calls) == made and state.powers is powers and state.count == 0 and state.norms is None


@pytest.mark.parametrize("bits, entry", [(32, "gs_moments_decode"), (8, "gs_moments_encode")])
def test_moments_of_a_state_on_another_device(on_host, monkeypatch, bits, entry):
    """The conversions take addresses of their own device: another device's moments are brought over first."""
    ps = [torch.zeros(300)]
    state, other = AdamW(1e-3, moment_bits=bits).init(ps), AdamW(1e-3, moment_bits=40 - bits).init(ps)
    names = ["mu_flat", "nu_flat"] + (["fields"] if other.bits == 8 else [])
    brought = {}
    for name in names:
        here = getattr(other, name)
        there = torch.empty_like(here, device="meta")
        setattr(other, name, there)
        brought[id(there)] = here
    to = torch.Tensor.to
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *a: brought[id(t)] if t.is_meta else to(t, *a))
    state.set_moments(other)
    name, args = on_host.calls[-1]
    assert name == entry
    assert list(args[2:2 + len(names)]) == [t.data_ptr() for t in brought.values()] and all(args[2:])

"""AdamW over many tensors at once, with moments in 32 or in 8 bits, and gradient norms with
the factor that clips them.

For models of any number of tensors of any sizes (the five Gaussian arrays, and whatever is
trained next to them); ``optimizer.Adam`` stays the reference trainer's own step.  One launch
updates up to 76 tensors, nothing waits for the host, and a step whose gradients are not finite
changes nothing when its scale comes from ``grad_norms``:

    optimizer = AdamW(1e-3, weight_decay=0.01, moment_bits=8, max_grad_norm=1.0)
    state = optimizer.init(params)
    optimizer.step(params, grads, state)

``params`` and ``grads`` are ``Gaussians``, dicts, lists or tuples of tensors, or one tensor:
float32, bfloat16 or float16, gradients of a type of their own (``None``: the tensor is left
alone).  The arithmetic is float32; the kernels are ``gs_adamw_step``, ``gs_grad_norms``,
``gs_moments_encode`` and ``gs_moments_decode``.
"""
from __future__ import annotations

from array import array
from typing import Callable, Optional, Union

import torch

from .. import _lib
from ..core.gaussians import Gaussians
from ..renderer._buffers import as_bytes
from .optimizer import FIELDS, make_optimizer

LearningRate = Union[float, Callable[[int], float]]
BLOCK = 256  # elements that share an exponent in 8 bits; each tensor's moments begin at a multiple


class GradNorms:
    """Device float32: ``total``, the norm of all gradients; ``per_tensor``, each one's (infinite beyond
    float32's range); ``scale``, the factor for the step."""
    __slots__ = ("_out", "_k")

    def __init__(self, out: torch.Tensor, k: int):
        self._out, self._k = out, k  # total, scale, one for each of k tensors, the call's workspace

    @property
    def total(self) -> torch.Tensor:
        return self._out[0]

    @property
    def scale(self) -> torch.Tensor:
        return self._out[1]

    @property
    def per_tensor(self) -> torch.Tensor:
        return self._out[2:2 + self._k]


def _keys(x) -> Optional[list]:
    if isinstance(x, Gaussians):
        return list(FIELDS)
    return list(x) if isinstance(x, dict) else None


def _tensors(x, keys=None) -> list:
    if isinstance(x, torch.Tensor):
        return [x]
    if isinstance(x, Gaussians):
        return [getattr(x, f) for f in FIELDS]
    if isinstance(x, dict):
        missing = [k for k in keys or () if k not in x]
        if missing:
            raise ValueError(f"AdamW: no tensor for {missing}")
        return [x[k] for k in (x if keys is None else keys)]
    return list(x)


def _fills(fill, keys, count: int, what: str) -> list:
    """The rows (or None) that new rows of `count` tensors get."""
    fills = _tensors(fill, keys)
    if len(fills) != count:
        raise ValueError(f"{what}: {len(fills)} fills for {count} tensors")
    return fills


def _like(keys, values):
    return list(values) if keys is None else dict(zip(keys, values))


def _device(tensor, what: str) -> torch.device:
    if not isinstance(tensor, torch.Tensor) or tensor.device.type != "cuda":
        raise ValueError(f"{what}: tensors must live on the GPU (there is no CPU path)")
    return tensor.device


def _mask(active_mask, tensors, dev, what: str):
    """(mask bytes, rows, elements per row of each tensor) for a mask over leading rows."""
    act = as_bytes(torch.as_tensor(active_mask, device=dev))
    rows = act.numel()
    if act.dim() != 1:
        raise ValueError(f"{what}: active_mask must have one dimension")
    for i, t in enumerate(tensors):
        if t is not None and (t.dim() == 0 or t.shape[0] != rows):
            raise ValueError(f"{what}: active_mask has {rows} entries, tensor {i} has shape {tuple(t.shape)}")
    lens = [1 if t is None else max(t.numel() // max(rows, 1), 1) for t in tensors]
    return act, rows, array("q", lens).tobytes()


def _scalar(grad_scale, dev, what: str):
    if grad_scale is None:
        return None
    if not isinstance(grad_scale, torch.Tensor):
        return torch.full((), float(grad_scale), device=dev)
    if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != dev:
        raise ValueError(f"{what}: grad_scale must be one float32 on {dev}")
    return grad_scale.resolve_neg() if grad_scale.is_neg() else grad_scale


def row_index(index, dev, what: str) -> torch.Tensor:
    """The index of rows, contiguous."""
    if not isinstance(index, torch.Tensor) or index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: the index must be an int32 or int64 tensor")
    if index.dim() != 1:
        raise ValueError(f"{what}: the index must have one dimension, not {index.dim()}")
    if index.device != dev:
        raise ValueError(f"{what}: the index is on {index.device}, the tensors are on {dev}")
    return index if index.is_contiguous() and not index.is_neg() else index.resolve_neg().contiguous()


def _address(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _norms(dev, k: int, pointers: bytes, types: bytes, counts: bytes, mask, max_norm, scale,
           entry: str = "gs_grad_norms") -> GradNorms:
    act, rows, lens = mask or (None, 0, None)
    nbytes = _lib.lib().gs_grad_norms_workspace_size(k, counts)
    # one allocation: the results, and from the next multiple of 8 bytes on the workspace
    head = (k + 3) // 2 * 2
    out = torch.empty((head + (nbytes + 3) // 4,), dtype=torch.float32, device=dev)
    at = out.data_ptr()
    _lib.call(entry, _lib.stream_handle(dev), k, pointers, types, counts, lens, _address(act), rows,
              0.0 if max_norm is None else float(max_norm), _address(scale), at + 4 * head, nbytes, at + 8, at)
    return GradNorms(out, k)


def grad_norms(grads, max_norm: Optional[float] = None, active_mask=None, grad_scale=None) -> GradNorms:
    """2-norms of grad_scale times the gradients, per tensor and of all, and the factor
    ``grad_scale * min(1, max_norm / (total + 1e-6))`` (``grad_scale`` without ``max_norm``),
    NaN when a gradient or ``grad_scale`` is not finite, all on the device (the sums are float64, so
    that a norm beyond float32's range still clips).  Rows where ``active_mask`` is False
    are left out, whatever they hold; ``None`` gradients count as empty."""
    if max_norm is not None and not max_norm > 0.0:
        raise ValueError(f"grad_norms: max_norm must be positive, not {max_norm}")
    gs = _tensors(grads)
    first = next((g for g in gs if g is not None), None)
    if first is None:
        raise ValueError("grad_norms: no gradients")
    dev = _device(first, "grad_norms")
    pointers, types, counts, kept = _lib.tensors().gather(gs, dev.index, "grad_norms")
    mask = None if active_mask is None else _mask(active_mask, gs, dev, "grad_norms")
    return _norms(dev, len(gs), pointers, types, counts, mask, max_norm, _scalar(grad_scale, dev, "grad_norms"))


def clip_grads_(grads, max_norm: float, active_mask=None, grad_scale=None) -> GradNorms:
    """``grad_norms``, and every gradient multiplied in place by its factor, ``grad_scale * min(1, max_norm /
    (total + 1e-6))``, rounded once to the gradient's type.  Rows where ``active_mask`` is False keep
    what they hold, and where a gradient (of the other rows) or ``grad_scale`` is not finite all do: ``scale`` is NaN then.  For
    optimizers that take no factor; ``AdamW(max_grad_norm=...)`` clips without writing the gradients."""
    if not max_norm > 0.0:
        raise ValueError(f"clip_grads_: max_norm must be positive, not {max_norm}")
    gs = _tensors(grads)
    first = next((g for g in gs if g is not None), None)
    if first is None:
        raise ValueError("clip_grads_: no gradients")
    dev = _device(first, "clip_grads_")
    native = _lib.tensors()
    pointers, types, counts = native.dense(gs, dev.index, "clip_grads_", active_mask is not None)
    mask = None if active_mask is None else _mask(active_mask, gs, dev, "clip_grads_")
    with _lib.on(dev):
        norms = _norms(dev, len(gs), pointers, types, counts, mask, max_norm, _scalar(grad_scale, dev, "clip_grads_"),
                       "gs_clip_grads")
    native.written([], [], gs)
    return norms


def _load(own: torch.Tensor, d: dict, name: str) -> torch.Tensor:
    """A checkpoint's array into the state's own, which the kernels take to be whole."""
    given = d[name]
    if not isinstance(given, torch.Tensor) or given.shape != own.shape:
        raise ValueError(f"AdamW.load_state_dict: {name} must be a tensor of shape {tuple(own.shape)}")
    return own.copy_(given)


class AdamWState:
    """Moments and step count of one model's parameters.

    ``mu_flat`` and ``nu_flat`` hold all moments: tensor i's from ``offsets[i]`` on, a multiple
    of 256, zeros between.  With ``bits`` 32 they are float32 and ``mu``/``nu`` give them tensor
    by tensor, as views.  With ``bits`` 8 they are bytes with two exponent bytes per 256 elements
    in ``fields``: ``mu_flat`` a sign, four exponent and three mantissa bits, ``nu_flat`` four
    exponent and four mantissa bits of the root of the second moment (``gs_moments_encode``).
    ``master_flat`` holds float32 weights of half-typed tensors, if asked for.  ``count`` is the
    number of steps asked for; ``powers`` (device float64) belongs to the updates made, which
    are fewer if a scale was not finite."""

    _row_layout = None  # _rows; of the class, as states that were saved whole may not have one

    def __init__(self, keys, shapes, bits: int):
        self.keys, self.shapes, self.bits = keys, [torch.Size(s) for s in shapes], bits
        self._lay_out([s.numel() for s in self.shapes])
        self.mu_flat = self.nu_flat = self.fields = self.master_flat = self.powers = None
        self._powers_stream: Optional[int] = None  # that the powers were allocated on
        self.count = 0
        self.norms: Optional[GradNorms] = None

    def _lay_out(self, counts: list) -> None:
        self.counts, self.offsets, at = counts, [], 0
        for n in counts:
            self.offsets.append(at)
            at += -(-n // BLOCK) * BLOCK
        self.size = at
        self._offsets = array("q", self.offsets).tobytes()

    def _allocate(self, dev, zero: bool):
        new = torch.zeros if zero else torch.empty
        dtype = torch.float32 if self.bits == 32 else torch.uint8
        self.mu_flat, self.nu_flat = (new((self.size,), dtype=dtype, device=dev) for _ in range(2))
        self.fields = new((self.size // BLOCK, 2), dtype=torch.uint8, device=dev) if self.bits == 8 else None

    def _set_powers(self, powers: torch.Tensor) -> None:
        """Take over powers that were allocated on the current stream."""
        self.powers, self._powers_stream = powers, _lib.stream_handle(powers.device).value

    def _views(self, flat):
        return _like(self.keys, [flat[o:o + n].view(s) for o, n, s in zip(self.offsets, self.counts, self.shapes)])

    @property
    def mu(self):
        """First moments, tensor by tensor: views of a 32-bit state."""
        return self.moments()[0] if self._is32("mu") else None

    @property
    def nu(self):
        """Second moments, tensor by tensor: views of a 32-bit state."""
        return self.moments()[1] if self._is32("nu") else None

    @property
    def master(self):
        """Float32 weights, tensor by tensor (those of float32 tensors are not kept up), or None."""
        return None if self.master_flat is None else self._views(self.master_flat)

    def _is32(self, name):
        if self.bits != 32:
            raise ValueError(f"AdamWState.{name}: this state is in 8 bits: moments() has its values")
        return True

    def moments(self):
        """(first, second) moments in float32, tensor by tensor: views of a 32-bit state, the
        values that an 8-bit state stands for."""
        s = self if self.bits == 32 else self.convert(32)
        return s._views(s.mu_flat), s._views(s.nu_flat)

    def convert(self, bits: int) -> "AdamWState":
        """A state of its own with the same moments in ``bits`` (32 or 8), to nearest."""
        if bits not in (32, 8):
            raise ValueError(f"AdamWState.convert: 32 or 8 bits, not {bits}")
        to = AdamWState.__new__(AdamWState)
        to.__dict__.update(self.__dict__)  # the layout and the powers are never written in place
        to.bits, to.norms = bits, None
        to.master_flat = None if self.master_flat is None else self.master_flat.clone()
        to._allocate(self.mu_flat.device, zero=False)
        to._take(self.bits, self.mu_flat, self.nu_flat, self.fields)
        return to

    def set_moments(self, other: "AdamWState") -> None:
        """Take over another state's moments (of the same tensors), to nearest."""
        if other.shapes != self.shapes:
            raise ValueError("AdamWState.set_moments: states of different tensors")
        given, dev = (other.mu_flat, other.nu_flat, other.fields), self.mu_flat.device
        if other.mu_flat.device != dev:  # the kernels take addresses of their own device
            given = [None if x is None else x.to(dev) for x in given]
        self._take(other.bits, *given)
        _lib.tensors().written([], [], [self.mu_flat, self.nu_flat, self.fields])

    def _take(self, bits: int, mu, nu, fields) -> None:
        """Moments in ``bits`` on this device, laid out as these, into this state's."""
        dev = self.mu_flat.device
        if self.bits == bits:
            for own, given in ((self.mu_flat, mu), (self.nu_flat, nu), (self.fields, fields)):
                if own is not None:
                    own.copy_(given)
        elif self.bits == 8:
            _lib.call("gs_moments_encode", _lib.stream_handle(dev), self.size, *map(_address, (
                mu, nu, self.mu_flat, self.nu_flat, self.fields)))
        else:
            _lib.call("gs_moments_decode", _lib.stream_handle(dev), self.size, *map(_address, (
                mu, nu, fields, self.mu_flat, self.nu_flat)))

    def _rows(self, what: str, only: Optional[list] = None):
        """(rows, elements per row of each tensor, the same as int64, bytes per row in 32 bits, a row's shapes) of a
        state whose tensors have the same rows; of the tensors with the numbers `only`, if given."""
        if only is None and self._row_layout is not None:
            return self._row_layout
        shapes = self.shapes if only is None else [self.shapes[i] for i in only]
        rows = shapes[0][0] if len(shapes[0]) else None
        if any([not len(s) or s[0] != rows for s in shapes]):
            raise ValueError(f"AdamWState.{what}: the state's tensors do not have the same rows")
        lens = [s[1:].numel() for s in shapes]
        layout = (rows, lens, array("q", lens).tobytes(), array("q", [4 * n for n in lens]).tobytes(),
                  [tuple(s[1:]) for s in shapes])
        if only is None:
            self._row_layout = layout
        return layout

    def _flats(self) -> list:
        """The float32 arrays."""
        flats = [self.mu_flat, self.nu_flat] if self.bits == 32 else []
        return flats if self.master_flat is None else flats + [self.master_flat]

    def _addresses(self, flats, only: Optional[list] = None) -> bytes:
        """Of every tensor (of `only`) in each of the float32 arrays."""
        offsets = self.offsets if only is None else [self.offsets[i] for i in only]
        return array("q", [at + 4 * o for at in [x.data_ptr() for x in flats] for o in offsets]).tobytes()

    def _master_fills(self, fill, row_shapes: list, what: str) -> Optional[list]:
        """The masters' new rows, copies in float32 of the parameters' `fill`; None without masters or fills."""
        if fill is None:
            return None
        dev, rows = self.mu_flat.device, []
        for i, (f, s) in enumerate(zip(_fills(fill, self.keys, len(row_shapes), what), row_shapes)):
            if f is not None:
                if not isinstance(f, torch.Tensor) or not f.is_floating_point() or f.device != dev or tuple(f.shape) != s:
                    raise ValueError(f"{what}: fill {i} must be one row of its tensor, of shape {s} on {dev}")
                if self.master_flat is not None:
                    f = torch.empty(s, dtype=torch.float32, device=dev).copy_(f.detach())
            rows.append(f)
        return None if self.master_flat is None else rows

    @staticmethod
    def _fill_addresses(fills: Optional[list], each: int) -> Optional[bytes]:
        """Of the masters' new rows, behind none for the moments: the masters are the last of `each` float32 arrays."""
        if fills is None:
            return None
        rows = [0 if f is None else f.data_ptr() for f in fills]
        return array("q", [0] * (len(rows) * (each - 1)) + rows).tobytes()

    def take_rows(self, index, fill=None) -> "AdamWState":
        """A state of its own for tensors whose row i is these tensors' row ``index[i]`` (``rows.take_rows``
        of the parameters): moments and masters of those rows.  Where ``index`` is no row's the moments are
        zero and the masters hold ``fill``, which is that of the parameters (zeros without it).  8-bit
        moments are rounded to nearest where a new neighbour raises the exponent of their block."""
        dev = self.mu_flat.device
        index = row_index(index, dev, "AdamWState.take_rows")
        rows, lens, lens_bytes, row_bytes, row_shapes = self._rows("take_rows")
        fills = self._master_fills(fill, row_shapes, "AdamWState.take_rows")
        count, k = index.numel(), len(lens)
        to = AdamWState.__new__(AdamWState)
        to.__dict__.update(self.__dict__)  # the powers are never written in place
        to.norms = None
        to.shapes = [torch.Size((count, *s)) for s in row_shapes]
        to._lay_out([n * count for n in lens])
        to._row_layout = count, lens, lens_bytes, row_bytes, row_shapes
        with _lib.on(dev):
            to._allocate(dev, zero=False)
            if self.master_flat is not None:
                to.master_flat = torch.empty((to.size,), dtype=torch.float32, device=dev)
            stream, of = _lib.stream_handle(dev), (index.data_ptr(), 8 * index.element_size(), count)
            flats = self._flats()
            if flats:
                each = len(flats)
                padded = array("q", [4 * (b - a) for a, b in zip(to.offsets, to.offsets[1:] + [to.size])]).tobytes()
                _lib.call("gs_take_rows", stream, each * k, self._addresses(flats), row_bytes * each, row_bytes * each,
                          rows, to._addresses(to._flats()), padded * each,
                          self._fill_addresses(fills, each), *of)
            if self.bits == 8:
                _lib.call("gs_moments_take", stream, k, lens_bytes, rows, self._offsets, self.size,
                          self.mu_flat.data_ptr(), self.nu_flat.data_ptr(), self.fields.data_ptr(), *of, to._offsets,
                          to.size, to.mu_flat.data_ptr(), to.nu_flat.data_ptr(), to.fields.data_ptr())
        return to

    def move_rows_(self, index, fill=None) -> "AdamWState":
        """In place, the moments and masters of row i become those of row ``index[i]``, as ``rows.move_rows_``
        moves the parameters.  Where ``index`` is negative the moments become zero and the masters ``fill``, which is
        that of the parameters (zero without it).  Returns the state."""
        dev = self.mu_flat.device
        index = row_index(index, dev, "AdamWState.move_rows_")
        rows, _, _, _, row_shapes = self._rows("move_rows_")
        if index.numel() != rows:
            raise ValueError(f"AdamWState.move_rows_: {index.numel()} indices for {rows} rows")
        fills = self._master_fills(fill, row_shapes, "AdamWState.move_rows_")
        with _lib.on(dev):
            self._move(index, self._move_workspace(), fills=fills)
        return self

    def _move_workspace(self, only: Optional[list] = None) -> Optional[torch.Tensor]:
        """What ``_move`` needs beside the state, so that it is there before anything is written."""
        if self.bits != 8:
            return None
        rows, lens, lens_bytes, _, _ = self._rows("move_rows_", only)
        nbytes = _lib.lib().gs_moments_move_workspace_size(len(lens), lens_bytes, rows)
        return torch.empty((nbytes,), dtype=torch.uint8, device=self.mu_flat.device)

    def _move(self, index: torch.Tensor, ws: Optional[torch.Tensor], only: Optional[list] = None,
              fills: Optional[list] = None) -> None:
        """``move_rows_`` by an index that was looked over, on the current device: allocates nothing there.  `only`:
        the numbers of the tensors that it is for, ascending, if not all."""
        dev = self.mu_flat.device
        rows, lens, lens_bytes, row_bytes, _ = self._rows("move_rows_", only)
        k, stream, bits = len(lens), _lib.stream_handle(dev), 8 * index.element_size()
        flats = self._flats()
        if flats:
            each = len(flats)
            _lib.call("gs_move_rows", stream, each * k, self._addresses(flats, only), row_bytes * each, row_bytes * each,
                      rows, self._fill_addresses(fills, each), index.data_ptr(), bits, None)
        if self.bits == 8:
            offsets = self._offsets if only is None else array("q", [self.offsets[i] for i in only]).tobytes()
            _lib.call("gs_moments_move", stream, k, lens_bytes, rows, offsets, self.size,
                      self.mu_flat.data_ptr(), self.nu_flat.data_ptr(), self.fields.data_ptr(), index.data_ptr(), bits,
                      ws.data_ptr(), ws.numel())
        _lib.tensors().written([], [], [self.mu_flat, self.nu_flat, self.fields, self.master_flat])

    def state_dict(self) -> dict:
        """The state as a dict of tensors (the state's own) and plain values, for a checkpoint."""
        return {"bits": self.bits, "shapes": [tuple(s) for s in self.shapes], "count": self.count, "mu_flat": self.mu_flat,
                "nu_flat": self.nu_flat, "fields": self.fields, "master_flat": self.master_flat,
                "powers": self.powers}


class AdamW:
    """w -= lr ((m / (1 - b1^t)) / (sqrt(v) / sqrt(1 - b2^t) + eps) + weight_decay w).

    ``learning_rates`` and ``weight_decay`` are one value for all tensors, or a list or dict
    like the parameters; a rate may be a schedule of the step count (``exponential_decay``).
    ``moment_bits`` 8 holds the moments in 8 bits, rounded stochastically with random bits that
    follow from ``seed``, the step and the element.  ``master_weights`` keeps float32 weights of
    half-typed parameters in the state.  With ``max_grad_norm`` every step takes the gradients'
    norm first (``state.norms``), scales them down to it, and leaves everything as it is when
    some gradient is not finite."""

    def __init__(self, learning_rates, b1: float = 0.9, b2: float = 0.999, eps: float = 1e-8, weight_decay=0.0,
                 moment_bits: int = 32, master_weights: bool = False, max_grad_norm: Optional[float] = None,
                 seed: int = 0):
        if moment_bits not in (32, 8):
            raise ValueError(f"AdamW: moments in 32 or 8 bits, not {moment_bits}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: b1 and b2 must be in [0, 1), not {b1}, {b2}")
        if not eps >= 0.0:
            raise ValueError(f"AdamW: eps must not be negative, not {eps}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"AdamW: max_grad_norm must be positive, not {max_grad_norm}")
        self.lrs, self.decay = learning_rates, weight_decay
        self.b1, self.b2, self.eps = float(b1), float(b2), float(eps)
        self.moment_bits, self.master_weights = moment_bits, bool(master_weights)
        self.max_grad_norm, self.seed = max_grad_norm, int(seed)

    def _powers(self, t: int, dev) -> torch.Tensor:
        p1, p2 = self.b1 ** t, self.b2 ** t
        return torch.tensor([p1, p2, 1.0 / (1.0 - p1 * self.b1), (1.0 - p2 * self.b2) ** -0.5], dtype=torch.float64,
                            device=dev)

    @staticmethod
    def _each(values, state: AdamWState, what: str) -> list:
        k = len(state.shapes)
        if isinstance(values, dict):
            missing = [x for x in (state.keys or ()) if x not in values]
            if state.keys is None or missing:
                raise ValueError(f"AdamW: {what} for {missing or 'parameters without names'} missing")
            return [values[x] for x in state.keys]
        if isinstance(values, (list, tuple)):
            if len(values) != k:
                raise ValueError(f"AdamW: {len(values)} values of {what} for {k} tensors")
            return list(values)
        return [values] * k

    def _state(self, params, bits) -> AdamWState:
        ps = _tensors(params)
        if not ps:
            raise ValueError("AdamW: no parameters")
        if _lib.tensors().gather(ps, _device(ps[0], "AdamW").index, "AdamW")[3] is not None:
            raise ValueError("AdamW: parameters must be contiguous")
        state = AdamWState(_keys(params), [p.shape for p in ps], bits)
        self._each(self.lrs, state, "the learning rate")
        self._each(self.decay, state, "weight_decay")
        return state

    def _masters(self, state: AdamWState, ps, master) -> None:
        if all([p.dtype == torch.float32 for p in ps]):
            return
        if not self.master_weights:
            if master is not None:
                raise ValueError("AdamW.restore: masters given to an optimizer that keeps none (master_weights)")
            return
        given = ps if master is None else _tensors(master, state.keys)
        if [x.numel() for x in given] != state.counts:
            raise ValueError("AdamW.restore: the masters are not those of the parameters")
        state.master_flat = torch.zeros((state.size,), dtype=torch.float32, device=ps[0].device)
        for o, n, x in zip(state.offsets, state.counts, given):
            state.master_flat[o:o + n].copy_(x.detach().reshape(-1))

    def init(self, params) -> AdamWState:
        """Zero moments for these parameters, no step made."""
        state = self._state(params, self.moment_bits)
        ps = _tensors(params)
        state._allocate(ps[0].device, zero=True)
        state._set_powers(self._powers(0, ps[0].device))
        self._masters(state, ps, None)
        return state

    def restore(self, params, mu, nu, count: int, master=None) -> AdamWState:
        """The state after ``count`` updates from first and second moments in 32 bits given
        tensor by tensor (an ``AdamState``'s ``mu`` and ``nu``, for one), and float32 masters if the
        optimizer keeps them (the parameters' values where none are given)."""
        full = self._state(params, 32)
        ps = _tensors(params)
        full._allocate(ps[0].device, zero=True)
        for flat, given in ((full.mu_flat, mu), (full.nu_flat, nu)):
            given = _tensors(given, full.keys)
            if [x.numel() for x in given] != full.counts:
                raise ValueError("AdamW.restore: the moments are not those of the parameters")
            for o, n, x in zip(full.offsets, full.counts, given):
                flat[o:o + n].copy_(x.detach().reshape(-1))
        full.count = int(count)
        full._set_powers(self._powers(full.count, ps[0].device))
        state = full if self.moment_bits == 32 else full.convert(8)
        self._masters(state, ps, master)
        return state

    def load_state_dict(self, params, d: dict) -> AdamWState:
        """The state of a checkpoint (``AdamWState.state_dict``) for these parameters: with its bits and its
        master weights.  Where it has none and the optimizer keeps them, they are the parameters' values."""
        bits = int(d["bits"])
        if bits not in (32, 8):
            raise ValueError(f"AdamW.load_state_dict: moments in 32 or 8 bits, not {bits}")
        state = self._state(params, bits)
        dev = _tensors(params)[0].device
        if [tuple(s) for s in d["shapes"]] != [tuple(s) for s in state.shapes]:
            raise ValueError("AdamW.load_state_dict: the checkpoint is of other tensors")
        state._allocate(dev, zero=True)
        for name in ("mu_flat", "nu_flat", "fields"):
            if getattr(state, name) is not None:
                _load(getattr(state, name), d, name)
        state.count = int(d["count"])
        state._set_powers(_load(torch.empty((4,), dtype=torch.float64, device=dev), d, "powers"))
        if d["master_flat"] is not None:
            state.master_flat = _load(torch.empty((state.size,), dtype=torch.float32, device=dev), d, "master_flat")
        else:
            self._masters(state, _tensors(params), None)
        return state

    def lr_at(self, lr: LearningRate, count: int) -> float:
        return float(lr(count)) if callable(lr) else float(lr)

    def step(self, params, grads, state: AdamWState, active_mask=None, grad_scale=None) -> AdamWState:
        """Update the parameters, the moments and the count in place; returns the state.  As after any
        in-place operation, autograd refuses a backward pass that needs the values from before.

        ``grad_scale`` (one float32 on the device, or a number) multiplies the gradients; when it
        is not finite nothing changes.  Rows whose ``active_mask`` entry is False keep their
        parameters and take a zero gradient, whatever theirs holds."""
        ps, gs = _tensors(params, state.keys), _tensors(grads, state.keys)
        k, dev = len(ps), state.mu_flat.device
        if _lib.capturing(dev):
            # replays would read powers that the state has let go of, and repeat one step's t and random bits
            raise RuntimeError("AdamW: a step cannot be captured into a graph")
        native = _lib.tensors()
        to, to_types, of, of_types, counts, kept = native.pair(ps, gs, state.shapes, dev.index)
        mask = None if active_mask is None else _mask(active_mask, ps, dev, "AdamW")
        act, rows, lens = mask or (None, 0, None)
        scale = _scalar(grad_scale, dev, "AdamW")
        state.norms = None
        if self.max_grad_norm is not None:
            state.norms = _norms(dev, k, of, of_types, counts, mask, self.max_grad_norm, scale)
            scale = state.norms.scale
        rates = self._each(self.lrs, state, "the learning rate")
        try:
            rates = array("d", rates)
        except TypeError:  # schedules among them
            rates = array("d", [self.lr_at(x, state.count) for x in rates])
        decays = array("d", self._each(self.decay, state, "weight_decay"))
        powers = torch.empty_like(state.powers)
        key = (self.seed * 0x85EBCA6B + (state.count + 1) * 0xC2B2AE3D + 0x27D4EB2F) & 0xFFFFFFFF
        stream = _lib.stream_handle(dev)
        _lib.call("gs_adamw_step", stream, k, to, to_types, of, of_types, state._offsets, counts,
                  lens, rates.tobytes(), decays.tobytes(), state.bits, state.size, state.mu_flat.data_ptr(),
                  state.nu_flat.data_ptr(), _address(state.fields), _address(state.master_flat), _address(act), rows,
                  _address(scale), state.powers.data_ptr(), powers.data_ptr(), self.b1, self.b2, self.eps, key)
        native.written(ps, gs, [state.mu_flat, state.nu_flat, state.fields, state.master_flat])
        if stream.value != state._powers_stream:
            # read here, and about to be let go of: whoever the allocator gives them to on the stream
            # that they come from waits for this step
            state.powers.record_stream(torch.cuda.current_stream(dev))
        state.powers, state._powers_stream = powers, stream.value
        state.count += 1
        return state


def make_adamw(extent: float, num_iterations: int, **options) -> AdamW:
    """AdamW with the trainer's learning rates (``make_optimizer``) for the five Gaussian arrays."""
    return AdamW(dict(make_optimizer(extent, num_iterations).lrs), **options)

"""Operators over the rows of a training state: rows taken by an index into new tensors, rows moved in
place, both of AdamW's moments in 32 and in 8 bits as well, the rows with the best scores, and
gradients clipped in place.

A row is what one leading index selects: a Gaussian in the five arrays and their moments, a page of a
pool, a line of a table.

Operators ("op") and what a case of each holds:
  "take"  row index[i] of every tensor as row i of a new one, zeros for index -1.
          "gaussians": five float32 arrays of n Gaussians and AdamW's moments (`bits`);
          "pages": `tensors` tensors of n rows of `row` elements of one type
  "move"  the same in place, most rows staying where they are
          "gaussians" as above; "table": tensors of n rows of odd lengths, drawn from `shapes`
  "best"  the k rows with the highest scores, in index order, the lowest index first among equals
  "clip"  gradients times scale * min(1, c / (norm + 1e-6)), in place
          "gaussians": five float32 arrays; "list": tensors of 1 to `most` elements, drawn from `shapes`

Moments lie in one flat array, each tensor from a multiple of 256 elements on.  Their 8-bit form, per
block of 256: values m = +-f 2^e with f of 4 exponent and 3 mantissa bits, and roots r = sqrt(v) = f 2^e
with f of 4 exponent and 4 mantissa bits, e the block's own for each, rounded to nearest even.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

BLOCK = 256
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "u8": 1}
FIELDS = ("means", "scales", "quaternions", "opacities", "sh_coeffs")


def _take(name, n, rows, k=16, bits=32, active=0.7, order="compact"):
    return {"name": name, "op": "take", "kind": "gaussians", "n": n, "rows": rows, "k": k, "bits": bits, "active": active,
            "order": order}


def _pages(name, n, rows, tensors, row, type, order):
    return {"name": name, "op": "take", "kind": "pages", "n": n, "rows": rows, "tensors": tensors, "row": row, "type": type,
            "order": order}


def _move(name, n, moved, freed, k=16, bits=32):
    return {"name": name, "op": "move", "kind": "gaussians", "n": n, "moved": moved, "freed": freed, "k": k, "bits": bits}


def _table(name, n, moved, freed, tensors, shapes, type):
    return {"name": name, "op": "move", "kind": "table", "n": n, "moved": moved, "freed": freed, "tensors": tensors,
            "shapes": shapes, "type": type}


def _best(name, n, k, type="f32", active=1.0):
    return {"name": name, "op": "best", "n": n, "k": k, "type": type, "active": active}


def _clip(name, n, k=16, active=1.0):
    return {"name": name, "op": "clip", "kind": "gaussians", "n": n, "k": k, "active": active, "type": "f32"}


def _clip_list(name, tensors, most, shapes, type):
    return {"name": name, "op": "clip", "kind": "list", "tensors": tensors, "most": most, "shapes": shapes, "type": type,
            "active": 1.0}


def listed():
    return [
        # a unit-test sized scene into its padded capacity: launches only
        _take("take_2k", 2000, 4096),
        # the trainer's padded capacity, compacted in the middle of a run
        _take("take_2m", 2_097_152, 1_500_000, active=0.6),
        # a pool of pages, forked: some pages taken many times, others not at all
        _pages("take_pages", 4099, 4096, 24, 8192, "bf16", "repeat"),
        # the headline scene with moments in 8 bits, its capacity raised
        _take("take8_1m", 1_000_000, 1_500_000, bits=8),
        # density control of an object-sized scene: clones into free slots
        _move("move_200k", 200_000, 0.05, 0.0),
        # a table of learned features of odd lengths beside the largest scene: rows moved and freed
        _table("move_3m", 3_000_000, 0.1, 0.05, 4, 11, "f16"),
        # density control at full capacity with moments in 8 bits
        _move("move8_2m", 2_097_152, 0.08, 0.0, bits=8),
        # a unit-test sized scene's budget
        _best("best_2k", 2000, 1500),
        # the largest scene, padded, cut to a budget by half-precision scores: many equal ones
        _best("best_3m", 3_000_000, 1_000_000, "bf16", 0.8),
        # gradients of a unit-test sized scene
        _clip("clip_2k", 2000),
        # gradients of the headline scene
        _clip("clip_1m", 1_000_000),
        # gradients of a network of many layers as they leave a half-precision backward
        _clip_list("clip_list_bf16", 148, 3_000_000, 1, "bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    op = rng.choice(("take", "take", "move", "move", "best", "clip"))
    if op == "take" and rng.random() < 0.4:
        row, tensors = log(1, 20_000), log(1, 32)
        n = min(log(64, 100_000), 1 + 400_000_000 // (row * tensors))
        c = _pages("", n, log(max(1, n // 4), 1 + n), tensors, row, rng.choice(("f32", "bf16", "f16", "u8")),
                   rng.choice(("repeat", "shuffle", "compact")))
    elif op == "take":
        n = log(1000, 2_000_000)
        c = _take("", n, min(int(n * rng.uniform(0.4, 1.5)), 1_900_000), rng.choice((1, 4, 9, 16)), rng.choice((32, 8)),
                  rng.uniform(0.3, 1.0), rng.choice(("compact", "shuffle", "repeat")))
    elif op == "move" and rng.random() < 0.4:
        c = _table("", log(64, 2_500_000), rng.uniform(0.0, 0.3), rng.uniform(0.0, 0.2), log(1, 6), rng.randrange(1 << 20),
                   rng.choice(("f32", "bf16", "f16", "u8")))
    elif op == "move":
        c = _move("", log(1000, 2_000_000), rng.uniform(0.0, 0.3), rng.choice((0.0, 0.1)), rng.choice((1, 4, 9, 16)),
                  rng.choice((32, 8)))
    elif op == "best":
        n = log(1000, 5_000_000)
        c = _best("", n, max(1, int(n * rng.uniform(0.01, 1.2))), rng.choice(("f32", "bf16", "f16")), rng.choice((1.0, 0.5, 0.9)))
    elif rng.random() < 0.5:
        c = _clip("", log(1000, 1_200_000), rng.choice((1, 4, 9, 16)), rng.choice((1.0, 0.6)))
    else:
        c = _clip_list("", log(1, 200), log(1000, 2_000_000), rng.randrange(1 << 20), rng.choice(("f32", "bf16", "f16")))
    del c["name"]
    return c


def _rows(case):
    """Elements per row of each tensor."""
    if case["kind"] == "gaussians":
        return [3, 3, 4, 1, 3 * case["k"]]
    if case["kind"] == "pages":
        return [case["row"]] * case["tensors"]
    rng = random.Random(case["shapes"])
    return [int(math.exp(rng.uniform(0.0, math.log(65)))) for _ in range(case["tensors"])]


def _sizes(case):
    """Elements of each gradient."""
    if case["kind"] == "gaussians":
        return [case["n"] * r for r in _rows(case)]
    rng = random.Random(case["shapes"])
    return [int(math.exp(rng.uniform(0.0, math.log(case["most"] + 1)))) for _ in range(case["tensors"])]


def _padded(count):
    return -(-count // BLOCK) * BLOCK


def work(case):
    op, n = case["op"], case.get("n", 0)
    if op == "best":
        return {"bytes": n * SIZE[case["type"]] + (n if case["active"] < 1.0 else 0) + 4 * case["k"], "flops": n}
    if op == "clip":
        count = sum(_sizes(case))
        return {"bytes": (2 * SIZE[case["type"]]) * count + (n if case["active"] < 1.0 else 0), "flops": 3 * count}
    row = sum(_rows(case))
    if op == "take":
        there = min(int(n * case["active"]), case["rows"]) if case["kind"] == "gaussians" else min(n, case["rows"])
        if case["kind"] == "pages":
            return {"bytes": 4 * case["rows"] + row * SIZE[case["type"]] * (there + case["rows"]), "flops": 0}
        if case["bits"] == 32:
            return {"bytes": 4 * case["rows"] + 12 * row * (there + case["rows"]), "flops": 0}
        # the values that the moved state stands for come back in 32 bits
        return {"bytes": 4 * case["rows"] + 6 * row * (there + case["rows"]) + 8 * row * case["rows"],
                "flops": 40 * row * case["rows"]}
    moved, freed = int(case["moved"] * n), int(case["freed"] * n)
    if case["kind"] == "table":
        return {"bytes": 4 * n + row * SIZE[case["type"]] * (2 * moved + freed), "flops": 0}
    if case["bits"] == 32:
        return {"bytes": 4 * n + 12 * row * (2 * moved + freed), "flops": 0}
    # of the 8-bit state the moved rows, and all of it once more for the values that come back
    return {"bytes": 4 * n + 6 * row * (2 * moved + freed) + (2 + 8) * row * n, "flops": 40 * row * (moved + freed)}


# ---- inputs -------------------------------------------------------------------------------------

def _values(gen, n, row, type):
    """Rows whose sizes vary over orders of magnitude, two in five of them zero."""
    if type == "u8":
        return torch.randint(0, 256, (n, row), generator=gen, device="cuda", dtype=torch.uint8)
    size = torch.exp(torch.randn(n, 1, generator=gen, device="cuda") * 1.5 - 9.0)
    seen = torch.rand(n, 1, generator=gen, device="cuda") < 0.6
    if type != "f32":
        return (torch.randn(n, row, generator=gen, device="cuda", dtype=torch.float32) * (seen * 1024.0) * size).to(TYPES[type])
    return torch.randn(n, row, generator=gen, device="cuda") * (size * seen)


def _index(case, gen):
    """int32 row numbers, as a user's program has them from its own bookkeeping."""
    n = case["n"]
    if case["op"] == "move":
        index = torch.arange(n, device="cuda", dtype=torch.int32)
        order = torch.randperm(n, generator=gen, device="cuda")
        moved, freed = int(case["moved"] * n), int(case["freed"] * n)
        to, stay = order[:moved].sort()[0], order[moved + freed:].sort()[0]
        if stay.numel():  # free slots take copies in order
            pick = torch.randint(0, stay.numel(), (moved,), generator=gen, device="cuda").sort()[0]
            index[to] = stay[pick].int()
        index[order[moved:moved + freed]] = -1
        return index
    rows = case["rows"]
    if case["order"] == "repeat":  # a quarter of the rows, most of them several times
        few = torch.randperm(n, generator=gen, device="cuda")[:max(1, n // 4)]
        there = few[torch.randint(0, few.numel(), (rows,), generator=gen, device="cuda")]
    elif case["order"] == "shuffle":
        there = torch.randperm(n, generator=gen, device="cuda")[:rows]
    else:
        there = torch.nonzero(torch.rand(n, generator=gen, device="cuda") < case.get("active", 0.7)).reshape(-1)[:rows]
    index = torch.full((rows,), -1, device="cuda", dtype=torch.int32)
    index[:there.numel()] = there.int()
    return index


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case, "pass": 0}
    op, n = case["op"], case.get("n", 0)
    if op == "best":
        # scores as density control has them: mean gradients, zero where a row was not seen
        s["scores"] = _values(gen, n, 1, "f32").reshape(-1).abs().to(TYPES[case["type"]]) if case["type"] != "f16" \
            else (_values(gen, n, 1, "f32").reshape(-1).abs() * 1024.0).half()
    elif op == "clip":
        sizes = _sizes(case)
        wide = _rows(case) if case["kind"] == "gaussians" else [64] * len(sizes)
        grads = [_values(gen, -(-c // w), w, case["type"]).reshape(-1)[:c] for c, w in zip(sizes, wide)]
        if case["kind"] == "gaussians":
            s["grads"] = [g.reshape(n, -1, 3) if i == 4 else g.reshape(n, -1) for i, g in enumerate(grads)]
        else:  # views into one buffer: they begin at any element
            s["flat"] = torch.cat(grads)
            s["grads"] = list(s["flat"].split(sizes))
        # gradients of four steps' sum go down to a norm of 0.1, the next time to 0.05, and so on: what was
        # clipped is clipped again
        s["scale"] = torch.full((), 4.0, device="cuda")
    else:
        rows = _rows(case)
        type = "f32" if case["kind"] == "gaussians" else case["type"]
        s["tensors"] = [_values(gen, n, row, type) for row in rows]
        if case["kind"] == "gaussians":
            s["tensors"][4] = s["tensors"][4].reshape(n, case["k"], 3)
            size = torch.exp(torch.randn(n, 1, generator=gen, device="cuda") * 1.5 - 9.0)
            mu = [torch.randn(n, row, generator=gen, device="cuda") * (0.3 * size) for row in rows]
            nu = [(torch.rand(n, row, generator=gen, device="cuda") + 0.05) * size * size for row in rows]
            s["mu"], s["nu"] = _pad(mu), _pad(nu)
        s["index"] = _index(case, gen)
    s["mask"] = torch.rand(n, generator=gen, device="cuda") < case["active"] if op in ("best", "clip") and case["active"] < 1.0 else None
    return s


def _pad(tensors):
    """The tensors one after another, each from a multiple of BLOCK on, zeros between."""
    gap = tensors[0].new_zeros(BLOCK)
    return torch.cat([x for t in tensors for x in (t.reshape(-1), gap[:_padded(t.numel()) - t.numel()])])


def _unpad(flat, n, rows):
    """The tensors of a padded array, as views of n rows."""
    out, at = [], 0
    for row in rows:
        out.append(flat[at:at + n * row].reshape(n, row))
        at += _padded(n * row)
    return out


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jax-gs_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        from jax_gs_amd.core.gaussians import Gaussians
        from jax_gs_amd.training import adamw, rows

        s["adamw"], s["rows"] = adamw, rows
        if case["op"] in ("take", "move") and case["kind"] == "gaussians":
            s["gaussians"] = Gaussians(*s["tensors"])
            s["state"] = adamw.AdamW(1e-3, moment_bits=case["bits"]).restore(
                s["gaussians"], _unpad(s["mu"], case["n"], _rows(case)), _unpad(s["nu"], case["n"], _rows(case)), 100)
            del s["mu"], s["nu"]
    else:
        s["pow2"] = torch.tensor([2.0 ** (e - 127) for e in range(255)], device="cuda")
        if case["op"] in ("take", "move") and case["kind"] == "gaussians" and case["bits"] == 8:
            s["m8"] = _encode(s, s.pop("mu"), 3)
            s["r8"] = _encode(s, s.pop("nu").sqrt(), 4)
    return s


def run(s):
    with torch.no_grad():
        return _run_own(s) if own else _run_plain(s)


def _norm_to(s):
    s["pass"] += 1
    return 0.1 if s["pass"] % 2 else 0.05


def _run_own(s):
    case, rows = s["case"], s["rows"]
    if case["op"] == "best":
        return rows.best_rows(s["scores"], case["k"], active_mask=s["mask"])
    if case["op"] == "clip":
        norms = s["adamw"].clip_grads_(s["grads"], _norm_to(s), active_mask=s["mask"], grad_scale=s["scale"])
        return [norms.total, norms.scale] + (s["grads"] if case["kind"] == "gaussians" else [s["flat"]])
    if case["kind"] != "gaussians":
        if case["op"] == "take":
            return rows.take_rows(s["tensors"], s["index"])
        rows.move_rows_(s["tensors"], s["index"])
        return s["tensors"]
    if case["op"] == "take":
        g, state = rows.take_rows(s["gaussians"], s["index"]), s["state"].take_rows(s["index"])
    else:
        g, state = s["gaussians"], s["state"]
        rows.move_rows_(g, s["index"])
        state.move_rows_(s["index"])
    if case["bits"] == 8:
        state = state.convert(32)
    return [getattr(g, f) for f in FIELDS] + [state.mu_flat, state.nu_flat]


# ---- the plain form: elementary torch operations in 32 bits ---------------------------------------

def _encode(s, x, mantissa):
    """8-bit codes (of the type uint8) and the exponent of each block, to nearest even.  Four exponent bits and
    `mantissa` mantissa bits: with the block's exponent taken out and the range moved to the bottom of
    float32's, the code is the top of the value's bits, gradual underflow included."""
    top = (16 << mantissa) - 1
    x = x.reshape(-1, BLOCK)
    size = x.abs()
    finite = size < math.inf
    most = torch.where(finite, size, 0.0).amax(1)
    exponent = ((most.view(torch.int32) + (1 << (24 - mantissa)) - 1) >> 23).clamp(max=254)
    bits = (size * s["pow2"][254 - exponent][:, None] * 2.0 ** -112).view(torch.int32)
    drop = 23 - mantissa
    code = ((bits + (1 << (drop - 1)) - 1 + ((bits >> drop) & 1)) >> drop).clamp(max=top - 1)
    if mantissa == 4:  # a root that is not zero stays so
        code = torch.maximum(code, (size > 0).int())
    code = torch.where(finite, code, top)
    if mantissa == 3:
        code = code | ((x.view(torch.int32) >> 31) & 128)
    return code.to(torch.uint8), exponent.to(torch.uint8)


def _decode(s, code, exponent, mantissa):
    top = (16 << mantissa) - 1
    code = code.int()
    size = code & top
    value = (size << (23 - mantissa)).view(torch.float32) * 2.0 ** 112 * s["pow2"][exponent.int()][:, None]
    value = torch.where(size == top, math.nan, value)
    if mantissa == 3:
        value = torch.where(code > 127, -value, value)
    return value.reshape(-1)


def _taken(t, index):
    there = (index >= 0).reshape(-1, *[1] * (t.dim() - 1))
    return torch.where(there, t[index.long().clamp(min=0)], torch.zeros((), dtype=t.dtype, device=t.device))


def _taken_flat(flat, s):
    return _pad([_taken(t, s["index"]) for t in _unpad(flat, s["case"]["n"], _rows(s["case"]))])


def _run_plain(s):
    case = s["case"]
    if case["op"] == "best":
        x = s["scores"].float()
        if s["mask"] is not None:
            x = torch.where(s["mask"], x, -math.inf)
        order = torch.sort(x, descending=True, stable=True)[1][:case["k"]]
        if s["mask"] is not None:  # masked rows go last
            order = torch.where(s["mask"][order], order, case["n"])
        order = torch.sort(order)[0]
        index = torch.full((case["k"],), -1, device="cuda", dtype=torch.int32)
        index[:order.numel()] = torch.where(order < case["n"], order, -1).int()
        return index
    if case["op"] == "clip":
        kept = s["grads"]
        if s["mask"] is not None:
            on = [s["mask"].reshape(-1, *[1] * (g.dim() - 1)) for g in kept]
            kept = [torch.where(m, g, 0.0) for m, g in zip(on, kept)]
        total = torch.stack([g.double().square().sum() for g in kept]).sum().sqrt() * s["scale"].abs()
        scale = (s["scale"] * (_norm_to(s) / (total + 1e-6)).clamp(max=1.0)).float()
        for i, g in enumerate(s["grads"]):
            new = (g.float() * scale).to(g.dtype)
            g.copy_(new if s["mask"] is None else torch.where(on[i], new, g))
        return [total.float(), scale] + (s["grads"] if case["kind"] == "gaussians" else [s["flat"]])
    new = [_taken(t, s["index"]) for t in s["tensors"]]
    if case["op"] == "move":
        s["tensors"] = new
    if case["kind"] != "gaussians":
        return new
    if case["bits"] == 32:
        moments = [_taken_flat(s["mu"], s), _taken_flat(s["nu"], s)]
        if case["op"] == "move":
            s["mu"], s["nu"] = moments
        return new + moments
    m8 = _encode(s, _taken_flat(_decode(s, *s["m8"], 3), s), 3)
    r8 = _encode(s, _taken_flat(_decode(s, *s["r8"], 4), s), 4)
    if case["op"] == "move":
        s["m8"], s["r8"] = m8, r8
    return new + [_decode(s, *m8, 3), _decode(s, *r8, 4).square()]


# ---- the definition in 64 bits --------------------------------------------------------------------

def _held(x, mantissa):
    """The values that 8 bits hold of x (float64, whole blocks): per block the least 2^e with all values at
    most (2 - 2 / 2^mantissa) 2^e; steps of 2^-mantissa of a value's own power of two, none below
    2^(e - 14), to nearest, ties to even; of the roots (mantissa 4) none that is above zero becomes zero."""
    x = x.reshape(-1, BLOCK)
    most = x.abs().amax(1, keepdim=True)
    f, e = torch.frexp(most)  # most = f 2^e, f in [1/2, 1)
    e = torch.where(f > 1.0 - 2.0 ** -mantissa, e, e - 1).clamp(min=-127)
    q = torch.ldexp(x.abs(), -e.double())
    power = (torch.frexp(q)[1] - 1).clamp(min=-14)
    step = torch.ldexp(torch.ones_like(q), power.double() - mantissa)
    at = torch.round(q / step)
    if mantissa == 4:
        at = torch.where((q > 0) & (at == 0), 1.0, at)
    return (torch.ldexp(at * step, e.double()) * x.sign()).reshape(-1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "best":
        return None  # whole numbers
    if case["op"] == "clip":
        g = [x.double() for x in s["grads"]]
        on = [torch.ones_like(x, dtype=torch.bool) for x in g]
        if s["mask"] is not None:
            on = [s["mask"].reshape(-1, *[1] * (x.dim() - 1)).expand_as(x) for x in g]
        total = 4.0 * math.sqrt(sum(float((x[m] ** 2).sum()) for x, m in zip(g, on)))
        scale = 4.0 * min(1.0, 0.1 / (total + 1e-6))
        new = [torch.where(m, x * scale, x) for x, m in zip(g, on)]
        return [torch.tensor(total, dtype=torch.float64), torch.tensor(scale, dtype=torch.float64)] + \
            (new if case["kind"] == "gaussians" else [torch.cat(new)])

    index = s["index"].long()

    def taken(t):  # an empty row behind the last is what -1 selects
        t = t.double() if t.is_floating_point() else t
        return torch.cat([t, torch.zeros_like(t[:1])]).index_select(0, torch.where(index < 0, t.shape[0], index))

    new = [taken(t) for t in s["tensors"]]
    if case["kind"] != "gaussians":
        return new
    moments = []
    for flat, mantissa in ((s["mu"].double(), 3), (s["nu"].double(), 4)):
        if case["bits"] == 8:
            flat = _held(flat if mantissa == 3 else flat.sqrt(), mantissa)
        flat = _pad([taken(t) for t in _unpad(flat, case["n"], _rows(case))])
        if case["bits"] == 8:
            flat = _held(flat, mantissa) ** (1 if mantissa == 3 else 2)
        moments.append(flat)
    return new + moments

"""AdamW and its 8-bit moments from their definitions, float64 numpy, on the host.

Also the random bits that the stochastic rounding takes, which are defined bit by bit."""
import numpy as np

BLOCK = 256
LOW = np.uint64(0xFFFFFFFF)


def pad(x):
    """A flat float64 array with zeros up to a whole block."""
    x = np.asarray(x, np.float64).reshape(-1)
    return np.concatenate([x, np.zeros(-len(x) % BLOCK)])


def noise(places, seed, step):
    """(16 bits for m, 16 bits for r) of each place, as fractions of 1."""
    p = np.asarray(places, np.uint64)
    x = ((p & LOW) + (p >> np.uint64(32)) * np.uint64(0x632BE5AB)) & LOW
    key = np.uint64((seed * 0x85EBCA6B + step * 0xC2B2AE3D + 0x27D4EB2F) & 0xFFFFFFFF)
    h = (x * np.uint64(0x9E3779B1) + key) & LOW
    h ^= h >> np.uint64(15)
    h = (h * np.uint64(0xD1B54A35)) & LOW
    h ^= h >> np.uint64(13)
    return (h >> np.uint64(16)).astype(np.float64) / 65536, (h & np.uint64(0xFFFF)).astype(np.float64) / 65536


def held(x, mantissa, u=None):
    """(the values 8 bits hold of x, how near each was to being rounded the other way).

    Whole blocks.  u None: to nearest, ties to even; else the value goes up when its fraction
    of a step plus u reaches 1.  The second result is the distance to the nearest threshold in
    steps of the value's own size (infinite where the value cannot move)."""
    x = np.asarray(x, np.float64).reshape(-1, BLOCK)
    finite = np.isfinite(x)
    a = np.where(finite, np.abs(x), 0.0)
    most = a.max(1, keepdims=True)
    f, e = np.frexp(most)
    e = np.clip(np.where(f > 1.0 - 2.0 ** -mantissa, e, e - 1), -127, 127)
    q = np.ldexp(a, -e)
    own = np.maximum(np.frexp(q)[1] - 1, -14)
    at = np.ldexp(q, mantissa - own)
    if u is None:
        near = np.abs(at - np.floor(at) - 0.5)
        k = np.rint(at)
    else:
        w = at + np.asarray(u).reshape(-1, BLOCK)
        near = np.abs(w - np.rint(w))
        k = np.floor(w)
    if mantissa == 4:
        k = np.where((a > 0) & (k == 0), 1.0, k)
    value = np.minimum(np.ldexp(k, own - mantissa), 2.0 - 2.0 / 2 ** mantissa)
    value = np.where(finite, np.ldexp(value, e) * np.where(np.signbit(x), -1.0, 1.0), np.nan)
    # a block whose largest value is about to move the exponent
    edge = np.abs(f / (1.0 - 2.0 ** -mantissa) - 1.0) < 1e-5
    return value.reshape(-1), np.where(edge, 0.0, near).reshape(-1)


def step(w, g, m, v, t, lr, b1=0.9, b2=0.999, eps=1e-8, decay=0.0, scale=1.0, on=None):
    """(w, m, v) after update t, and the size of what m is a sum of."""
    w, g, m, v = (np.asarray(x, np.float64) for x in (w, g, m, v))
    g = g * scale
    if on is not None:
        g = np.where(on, g, 0.0)
    size = np.abs(b1 * m) + np.abs((1 - b1) * g)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    u = (m / (1 - b1 ** t)) / (np.sqrt(v) / np.sqrt(1 - b2 ** t) + eps)
    new = w - lr * (u + decay * w)
    return (new if on is None else np.where(on, new, w)), m, v, size

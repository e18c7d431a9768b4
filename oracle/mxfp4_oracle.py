"""MXFP4 in numpy, float64: the format, its quantisation, products and the expert layer, from their definitions.  Test infrastructure."""
from __future__ import annotations

import numpy as np

BLOCK = 32
VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode(v: np.ndarray) -> np.ndarray:
    """Finite values -> codes 0 .. 15: the nearest of VALUES, of two equally near ones the even code; beyond 6 the largest."""
    d = np.abs(np.abs(v)[..., None] - VALUES)
    best = d.min(-1, keepdims=True)
    code = np.where(d == best, np.where(np.arange(8) % 2 == 0, 0, 1), 9).argmin(-1)
    return (code + 8 * np.signbit(v)).astype(np.uint8)


def decode(code: np.ndarray) -> np.ndarray:
    return np.where(code & 8, -VALUES[code & 7], VALUES[code & 7])


def scale_byte(amax: np.ndarray) -> np.ndarray:
    """Largest magnitudes (float64) -> scale bytes."""
    finite = np.isfinite(amax)
    mant, ex = np.frexp(np.where(finite, amax, 1.0))  # amax = mant * 2^ex, mant in [0.5, 1)
    top = ex - 1 + (mant >= 0.875)
    top = np.where(amax == 0, -1000, np.minimum(top, 127))  # a float32 exponent
    return np.where(finite, np.maximum(top - 2 + 127, 0), 255).astype(np.uint8)


def quant(x: np.ndarray):
    """x [m, k] -> codes [m, k], scale bytes [m, k / 32]."""
    g = x.astype(np.float64).reshape(x.shape[0], -1, BLOCK)
    with np.errstate(invalid="ignore"):
        byte = scale_byte(np.where(np.isfinite(g).all(-1), np.abs(g).max(-1), np.inf))
        v = np.where((byte == 255)[..., None], 0.0, g) * 2.0 ** (127.0 - np.where(byte == 255, 127, byte))[..., None]
    code = encode(v)
    code[byte == 255] = 0
    return code.reshape(x.shape), byte


def values(code: np.ndarray, byte: np.ndarray) -> np.ndarray:
    scale = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127.0))
    return decode(code) * np.repeat(scale, BLOCK, axis=-1)


def pack(code: np.ndarray) -> np.ndarray:
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def unpack(q: np.ndarray) -> np.ndarray:
    return np.stack((q & 15, q >> 4), axis=-1).reshape(q.shape[:-1] + (-1,))


def act(v: np.ndarray, kind: str) -> np.ndarray:
    if kind == "silu":
        with np.errstate(over="ignore"):
            return v / (1.0 + np.exp(-v))
    from math import erf

    return v * 0.5 * (1.0 + np.vectorize(erf)(v / np.sqrt(2.0)))


def experts(x, w1, w2, weights, ids, kind="silu", on_input=False, scaling=1.0):
    """(out, size): the layer in float64 on values w1 [E, 2I, H], w2 [E, H, I], and the sum of the magnitudes of the second stage's terms."""
    out, size = np.zeros(x.shape), np.zeros(x.shape)
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < w1.shape[0]:
                continue
            a = w1[e] @ x[t]
            if on_input:
                a = a * weights[t, j]
            half = a.shape[0] // 2
            h = act(a[:half], kind) * a[half:]
            f = scaling * (1.0 if on_input else weights[t, j])
            out[t] += f * (w2[e] @ h)
            size[t] += np.abs(f) * (np.abs(w2[e]) @ np.abs(h))
    return out, size

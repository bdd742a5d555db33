"""The operators behind one shared prefix in 64 bits, from their definitions: rotary positions, the cache's
codes, attention over a cached prefix and a sequence's own keys.  Test infrastructure only."""
import math

import numpy as np

NAN_CODE = 0x7F


# ---- 16-bit types as numpy sees them: bf16 by its bits ------------------------------------------


def to_bits(x, bf16):
    """Nearest-even 16-bit elements (uint16) of float values."""
    if not bf16:
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float64).astype(np.float16).view(np.uint16)
    x = np.asarray(x, np.float64)
    f = x.astype(np.float32)
    # to f32 by rounding to odd, so that the second rounding sees what the first left out
    b = f.view(np.uint32).copy()
    inexact = (f.astype(np.float64) != x) & np.isfinite(f)
    beyond = inexact & (np.abs(f.astype(np.float64)) > np.abs(x))
    b = np.where(beyond, b - 1, b)
    b = np.where(inexact, b | 1, b).astype(np.uint32)
    out = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def from_bits(b, bf16):
    b = np.asarray(b, np.uint16)
    if not bf16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def half_step(x, bf16):
    """The most that rounding x to the type moves it."""
    least = 2.0 ** -134 if bf16 else 2.0 ** -25
    return np.maximum(np.abs(x) * (2.0 ** -9 if bf16 else 2.0 ** -12) * 2, least)  # eps / 2: 2^-8, 2^-11


# ---- rotary positions ---------------------------------------------------------------------------


def rope_frequencies(rotary, theta, scaling="plain", factor=1.0, context=32768, fast=32.0, slow=1.0):
    i = np.arange(rotary // 2, dtype=np.float64)
    f = theta ** (-2 * i / rotary)
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        edge = [rotary * math.log(context / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (fast, slow)]
        low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rotary - 1)
        r = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        return f * (1 - r) + f / factor * r
    return f


def rope(x, positions, f, layout, magnitude=1.0, inverse=False):
    """x [tokens, heads, dim] f64 rotated."""
    n = len(f)
    angle = np.asarray(positions, np.float64)[:, None] * f * (-1 if inverse else 1)
    c, s = (magnitude * g(angle)[:, None, :] for g in (np.cos, np.sin))
    ia, ib = (np.arange(n), np.arange(n) + n) if layout == "half" else (2 * np.arange(n), 2 * np.arange(n) + 1)
    out = x.copy()
    out[..., ia] = x[..., ia] * c - x[..., ib] * s
    out[..., ib] = x[..., ib] * c + x[..., ia] * s
    return out


# ---- cache codes ----------------------------------------------------------------------------------


def e4m3_values():
    """The value of each of the 256 codes."""
    c = np.arange(256)
    sign, e, m = np.where(c & 128, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = sign * np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    return np.where((c & 127) == NAN_CODE, np.nan, v)


def e4m3_code(y):
    """Nearest code (ties to the even one) of values within +-448."""
    grid = e4m3_values()[:NAN_CODE]
    a = np.abs(y)
    at = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    low, high = grid[at - 1], grid[at]
    up = (a - low > high - a) | ((a - low == high - a) & (at % 2 == 0))
    code = np.where(up, at, at - 1)
    code = np.where(np.isnan(y), NAN_CODE, code)
    return (code | np.where(np.signbit(y) & ~np.isnan(y), 128, 0)).astype(np.uint8)


def quantise(x, form, bf16):
    """(codes uint8, scales f32) of f64 vectors along the last axis, bit for bit."""
    finite = np.where(np.isfinite(x), np.abs(x), 0).max(-1)
    zeros = finite < 2.0 ** -100
    safe = np.where(zeros, 1.0, finite)
    flat = np.where(np.isfinite(x) & zeros[..., None], 0, x)
    if form == "int8":
        amax = safe.astype(np.float32)
        scale = np.where(zeros, np.float32(1), amax / np.float32(127)).astype(np.float32)
        inv = np.where(zeros, np.float32(1), np.float32(127) / amax).astype(np.float32)
        with np.errstate(invalid="ignore"):
            y = np.clip(np.rint(flat.astype(np.float32) * inv[..., None]), -127, 127)
        return np.where(np.isnan(y), 0, y).astype(np.int8).view(np.uint8), scale
    e = np.ceil(np.log2(safe / 448.0))
    e = np.where(safe <= 448.0 * 2.0 ** (e - 1), e - 1, e)
    e = np.where(safe > 448.0 * 2.0 ** e, e + 1, e)
    scale = np.where(zeros, 1.0, 2.0 ** e)
    most = np.where(scale >= (2.0 ** 120 if bf16 else 2.0 ** 8), 240, 448)[..., None]
    y = np.clip(flat / scale[..., None], -most, most)
    return e4m3_code(y), scale.astype(np.float32)


def values(codes, scale, form):
    """What codes and scales stand for, in 64 bits."""
    v = codes.view(np.int8).astype(np.float64) if form == "int8" else e4m3_values()[codes]
    return v * np.asarray(scale, np.float64)[..., None]


# ---- attention --------------------------------------------------------------------------------------


def visible(query, keys, mask, prefix, window):
    """Which of the positions 0 .. keys - 1 the position `query` sees."""
    k = np.arange(keys)
    keep = k <= query
    if mask:
        keep &= (k < prefix) | (query - k < window)
    return keep


def attend(q, shared, own, lengths_q, mask=0, prefix=176, window=432, scale=None):
    """q [tokens, heads, dim]; shared (K, V) [P, kv, dim]; own: a (K, V) pair per sequence.  A row that
    sees no key gives zeros, and a key that a row does not see adds nothing, whatever it holds."""
    heads, dim = q.shape[1:]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, t = np.zeros(q.shape, np.float64), 0
    for m, (k, v) in zip(lengths_q, own):
        keys, vals = np.concatenate([shared[0], k]), np.concatenate([shared[1], v])
        group = heads // keys.shape[1]
        for j in range(m):
            keep = visible(len(keys) - m + j, len(keys), mask, prefix, window)
            if keep.any():
                for g in range(keys.shape[1]):
                    rows = q[t, g * group:(g + 1) * group]
                    s = rows @ keys[keep, g].T * scale
                    p = np.exp(s - s.max(-1, keepdims=True))
                    out[t, g * group:(g + 1) * group] = p @ vals[keep, g] / p.sum(-1, keepdims=True)
            t += 1
    return out

"""The operators of a forward with 8-bit activations from their definitions: rows into 8-bit codes, 4-bit weights
with whole-number group scales and their image, the products.  Test infrastructure only."""
import numpy as np

import shared_ref as ref

LEAST = np.float32(2.0 ** -100)

# ---- rows into 8 bits ---------------------------------------------------------------------------


def q8_codes(t):
    """(codes, amax, lost, none) of rows t (f32), every operation rounded to f32."""
    t = np.asarray(t, np.float32)
    amax = np.abs(t).max(-1)
    lost = ~np.isfinite(t).all(-1)
    none = ~lost & (amax < LEAST)
    with np.errstate(all="ignore"):
        factor = np.where(lost | none, np.float32(0), np.float32(127) / amax).astype(np.float32)
        codes = np.where((lost | none)[:, None], np.float32(0), np.rint(t * factor[:, None]))
    return codes.astype(np.int8), amax, lost, none


def quantize_q8(bits, bf16):
    """Codes, and scales in 64 bits, of rows of 16-bit elements."""
    codes, amax, lost, none = q8_codes(ref.from_bits(bits, bf16))
    return codes, np.where(lost, np.nan, np.where(none, 0.0, amax.astype(np.float64) / 127))


def rmsnorm_q8(x, residual, weight, bf16, eps):
    """(codes, scales in 64 bits, the sum's bits or None) of rows of 16-bit elements."""
    x = ref.from_bits(x, bf16)
    total = None
    with np.errstate(all="ignore"):
        v = x.astype(np.float32)
        if residual is not None:
            v = v + ref.from_bits(residual, bf16).astype(np.float32)
            total = ref.to_bits(v, bf16)
            x = ref.from_bits(total, bf16)
        codes, amax, lost, none = q8_codes(x.astype(np.float32) * np.asarray(weight, np.float32))
        squares = (v.astype(np.float64) ** 2).sum(-1)
        lost = lost | ~(squares < 2.0 ** 128)
        codes[lost] = 0
        inv = 1 / np.sqrt(squares / x.shape[1] + eps)
        scales = np.where(lost, np.nan, np.where(none, 0.0, amax.astype(np.float64) / 127 * inv))
    return codes, scales, total


# ---- 4-bit weights ------------------------------------------------------------------------------


def values(codes, groups, scales=None):
    """(code - zero) * multiplier of codes [N, K], groups [N, K / 32]: whole numbers; times the row scales."""
    codes = np.asarray(codes, np.int64)
    mult, zero = (np.repeat(np.asarray(g, np.int64), 32, 1) for g in (groups & 15, groups >> 4))
    w = (codes - zero) * mult
    return w if scales is None else w * np.asarray(scales, np.float64)[:, None]


def pairs():
    """Every (multiplier, zero point) whose weights fit 8 bits, as group bytes."""
    return np.array([m | z << 4 for m in range(16) for z in range(16) if z * m <= 128 and (15 - z) * m <= 127], np.uint8)


def nibbles(codes):
    """Codes [N, K] two to a byte, even columns low."""
    codes = np.asarray(codes, np.uint8)
    return codes[:, 0::2] | codes[:, 1::2] << 4


def image(codes, groups, scales):
    """The image, element by element from its description: tiles of 16 rows, blocks of 128 columns."""
    N, K = codes.shape
    tiles, blocks = -(-N // 16), -(-K // 128)
    c = np.zeros((tiles, 16, blocks, 4, 32), np.uint8)
    g = np.zeros((tiles, 16, blocks, 4), np.uint8)
    s = np.zeros(tiles * 16, np.float32)
    s[:N] = scales
    pad = np.zeros((tiles * 16, blocks * 128), np.uint8)
    pad[:N, :K] = codes
    c[:] = pad.reshape(c.shape)
    padg = np.zeros((tiles * 16, blocks * 4), np.uint8)
    padg[:N, :K // 32] = groups
    g[:] = padg.reshape(g.shape)
    records = (c[..., :16] | c[..., 16:] << 4).transpose(0, 2, 3, 1, 4)  # [tile, block, group, row, byte]
    return np.concatenate([records.ravel(), g.transpose(0, 2, 1, 3).ravel(), s.view(np.uint8)])


def taken_apart(packed, K, N):
    """(codes, groups, scales) of an image."""
    tiles, blocks = -(-N // 16), -(-K // 128)
    at = tiles * blocks * 1024
    records = packed[:at].reshape(tiles, blocks, 4, 16, 16).transpose(0, 3, 1, 2, 4)
    codes = np.concatenate([records & 15, records >> 4], -1).reshape(tiles * 16, blocks * 128)
    groups = packed[at:at + tiles * blocks * 64].reshape(tiles, blocks, 16, 4).transpose(0, 2, 1, 3).reshape(tiles * 16, -1)
    return codes[:N, :K], groups[:N, :K // 32], packed[at + tiles * blocks * 64:].view(np.float32)[:N]


def quantize(w):
    """(codes, groups, scales) of float rows [N, K], by the library's definition in 64 bits."""
    w = np.asarray(w, np.float32).astype(np.float64)
    N, K = w.shape
    codes, groups = np.zeros((N, K), np.uint8), np.zeros((N, K // 32), np.uint8)
    scales = np.zeros(N, np.float32)
    for n in range(N):
        top = np.abs(w[n]).max()
        if top < 2.0 ** -100:
            continue
        scales[n] = np.float32(top / 120)
        s = float(scales[n])
        for g in range(K // 32):
            x = w[n, 32 * g:32 * g + 32]
            a = x[np.abs(x).argmax()]
            if a == 0:
                continue
            zero = 8 if a < 0 else 7
            least = int(np.floor(abs(a) / 8 / s))
            best = None
            for m in sorted({min(max(least, 1), 15), min(max(least + 1, 1), 15)}):
                q = np.clip(np.rint(x / (s * m)), -zero, 15 - zero)
                d = x - q * (s * m)
                error = 0.0
                for e in d * d:  # in turn, as written
                    error += e
                if best is None or error < best[0]:
                    best = (error, m, q)
            codes[n, 32 * g:32 * g + 32] = best[2] + zero
            groups[n, g] = best[1] | zero << 4
    return codes, groups, scales


def random_weights(rng, N, K):
    """Codes of all values, groups of every allowed pair, row scales of both signs."""
    return (rng.integers(0, 16, (N, K)).astype(np.uint8), rng.choice(pairs(), (N, K // 32)),
            (rng.standard_normal(N) * 0.01).astype(np.float32))


# ---- products -----------------------------------------------------------------------------------


def product(x, x_scale, codes, groups, scales):
    """y in 64 bits; the sums are exact."""
    sums = np.asarray(x, np.float64) @ values(codes, groups).astype(np.float64).T
    return sums * np.asarray(x_scale, np.float64)[:, None] * np.asarray(scales, np.float64)


def product_bound(want, bf16):
    """The sum's conversion to f32 and two products, 2^-24 each, then the result's rounding."""
    err = np.abs(want) * 3.01 * 2.0 ** -24
    return err + ref.half_step(np.abs(want) + err, bf16)


def swiglu(g, u):
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u


def swiglu_bound(g, u, bf16):
    """g and u are off by 3 * 2^-24 each.  exp2's argument is off by that and two roundings (the constant's and the
    product's), so the sigmoid by |g| * 5 * 2^-24 of it, and by exp2, the sum and the reciprocal, 2^-23 each; then
    two products.  exp2 beyond 2^127 or a reciprocal below 2^-126 give 0: |g u| 2^-126 at most."""
    want = np.abs(swiglu(g, u))
    err = want * (2.0 ** -24 * (6 + 6 + 2 + 6 * np.abs(g))) * 1.01 + np.abs(g * u) * 2.0 ** -125
    return err + ref.half_step(want + err, bf16)

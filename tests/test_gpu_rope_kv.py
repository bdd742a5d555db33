"""Rotary positions (qattn_rope) and the paged cache's write and read (qattn_kv_write, qattn_kv_read)
against their definitions in 64 bits, on the GPU."""
import ctypes

import numpy as np
import pytest

import shared_ref as ref

pytestmark = pytest.mark.gpu
rng_of = np.random.default_rng


def upload(ctx, a):
    return ctx.upload(np.ascontiguousarray(a))


def rope_bound(x, positions, f, layout, magnitude, out, bf16):
    """The turn is a product in f64 (a few roundings of 2^-53 of it, the frequency's among them: 2^-50), its
    fraction in f32 within 2^-25 turns, sincospi within 2^-23 of the value, the magnitude one rounding more:
    cos and sin are off by at most 2^-21 + 2^-50 angle.  The two products and their sum round to f32."""
    n = len(f)
    angle = np.abs(np.asarray(positions, np.float64)[:, None] * f)[:, None, :]
    ia, ib = (np.arange(n), np.arange(n) + n) if layout == "half" else (2 * np.arange(n), 2 * np.arange(n) + 1)
    size = (np.abs(x[..., ia]) + np.abs(x[..., ib])) * abs(magnitude)
    err = size * (2.0 ** -21 + 2.0 ** -50 * angle + 2.0 ** -22)
    bound = np.zeros_like(out)
    bound[..., ia] = bound[..., ib] = err
    return bound + ref.half_step(np.abs(out) + bound, bf16)


ROPE_CASES = [
    # tokens, q heads, k heads, dim, rotary, layout, bf16, scaling, factor, far, inverse, stride pad, offset
    (1, 16, 8, 128, 128, "half", False, "plain", 1.0, 0, False, 0, 0),
    (5, 16, 8, 128, 128, "half", False, "yarn", 4.0, 131072, False, 1024, 0),
    (67, 28, 4, 128, 64, "interleaved", True, "linear", 4.0, 30000, False, 0, 0),
    (33, 3, 1, 64, 64, "interleaved", False, "plain", 1.0, 1 << 20, True, 8, 0),
    (33, 3, 0, 64, 32, "half", True, "yarn", 8.0, 500, True, 8, 0),
    (300, 2, 2, 128, 48, "half", True, "plain", 1.0, 77, False, 0, 0),
    (9, 5, 1, 80, 20, "half", False, "linear", 2.0, 1000, False, 0, 0),       # pairs no multiple of eight
    (9, 5, 1, 80, 20, "interleaved", True, "yarn", 2.0, 1000, True, 3, 1),    # and an odd stride and address
    (7, 1, 1, 2, 2, "half", False, "plain", 1.0, 10, False, 0, 0),            # the smallest head
    (4, 2, 1, 512, 512, "half", True, "plain", 1.0, (1 << 31) - 5, False, 0, 0),  # the widest, the farthest
    (3, 2, 1, 17, 16, "interleaved", False, "plain", 1.0, 100, False, 0, 0),  # odd head
    (3000, 2, 1, 128, 128, "half", False, "plain", 1.0, 100, False, 0, 0),
    (2500, 3, 1, 96, 6, "interleaved", True, "plain", 1.0, 5000, False, 0, 0),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", ROPE_CASES, ids=lambda c: "-".join(map(str, c[:9])))
def test_rope(ctx, qattn, case, in_place):
    tokens, hq, hk, dim, rotary, layout, bf16, scaling, factor, far, inverse, pad, offset = case
    print("rope", case, in_place, flush=True)
    rng = rng_of(tokens * 31 + dim)
    positions = (far + rng.permutation(tokens)).clip(0, (1 << 31) - 1).astype(np.int32)
    f = ref.rope_frequencies(rotary, 1e4, scaling, factor)
    magnitude = 0.1 * np.log(factor) + 1 if scaling == "yarn" else 1.0
    bp, blocks, rows = upload(ctx, positions), [], []
    for heads in (hq, hk):
        stride = heads * dim + pad
        x = ref.to_bits(rng.standard_normal((tokens, max(stride, 1))) * 3, bf16)
        flat = np.concatenate([np.zeros(offset, np.uint16), x.ravel()])
        bx = upload(ctx, flat)
        bo = bx if in_place else upload(ctx, np.full(len(flat), 0x7E11, np.uint16))
        blocks.append((bx, bo))
        rows.append(x)
    part = lambda i, heads: (blocks[i][0].ptr + 2 * offset, blocks[i][1].ptr + 2 * offset, heads)  # noqa: E731
    desc = qattn.make_rope_desc(bp.ptr, tokens, part(0, hq), part(1, hk) if hk else None, dim, rotary,
                                qattn.ROPE_HALF if layout == "half" else qattn.ROPE_INTERLEAVED,
                                qattn.BF16 if bf16 else qattn.F16, hq * dim + pad, hk * dim + pad, hq * dim + pad,
                                hk * dim + pad, theta=1e4, factor=factor, inverse=inverse,
                                scaling={"plain": 0, "linear": 1, "yarn": 2}[scaling])
    ctx.rope(desc)
    ctx.synchronize()
    for (bx, bo), heads, x in zip(blocks, (hq, hk), rows):
        if not heads:
            continue
        got = bo.read(np.uint16, (offset + x.size,))
        head = x[:, :heads * dim].reshape(tokens, heads, dim)
        value = ref.from_bits(head, bf16)
        want = ref.rope(value, positions, f, layout, magnitude, inverse)
        out = got[offset:].reshape(x.shape)
        y = out[:, :heads * dim].reshape(tokens, heads, dim)
        err = np.abs(ref.from_bits(y, bf16) - want)
        bound = rope_bound(value, positions, f, layout, magnitude, want, bf16)
        assert (err <= bound).all(), float((err / bound).max())
        assert np.array_equal(y[..., rotary:], head[..., rotary:])
        # what lies between the rows stays
        assert np.array_equal(out[:, heads * dim:], x[:, heads * dim:] if in_place else np.full_like(x[:, heads * dim:], 0x7E11))
        assert (got[:offset] == (0 if in_place else 0x7E11)).all()
    for pair in blocks:
        for b in set(pair):
            b.free()
    bp.free()


def test_rope_inverse_is_the_gradient(ctx, qattn):
    """The rotation is linear, so the inner product of an output gradient with a rotated difference is the
    one of the inverse rotation of the gradient with the difference; both sides in 64 bits over the
    device's bf16 results, whose roundings (2^-8 each of 128 terms) bound the difference."""
    tokens, dim = 12, 128
    rng = rng_of(4)
    positions = rng.integers(0, 5000, tokens).astype(np.int32)
    x, g = (ref.to_bits(rng.standard_normal((tokens, dim)), True) for _ in range(2))
    bp, bufs = upload(ctx, positions), [upload(ctx, a) for a in (x, g)]
    for b, inverse in zip(bufs, (False, True)):
        ctx.rope(qattn.make_rope_desc(bp.ptr, tokens, (b.ptr, b.ptr, 1), layout=qattn.ROPE_INTERLEAVED,
                                      dtype=qattn.BF16, scaling=qattn.ROPE_YARN, factor=4.0, inverse=inverse))
    ctx.synchronize()
    y, gx = (ref.from_bits(b.read(np.uint16, (tokens, dim)), True) for b in bufs)
    x, g = ref.from_bits(x, True), ref.from_bits(g, True)
    bound = 2.0 ** -8 * (np.abs(g * y).sum(-1) + np.abs(x * gx).sum(-1)) * 1.01
    assert (np.abs((g * y).sum(-1) - (x * gx).sum(-1)) <= bound).all()
    for b in bufs + [bp]:
        b.free()


# ---- the cache ------------------------------------------------------------------------------------


class Pool:
    """A cache whose memory holds a pattern, on the device."""

    def __init__(self, ctx, qattn, pages, page, heads, dim, bf16, form):
        self.shape, self.form, self.bf16 = (pages, heads, page, dim), form, bf16
        width = 2 if form == "16bit" else 1
        self.fill = np.full((pages, heads, page, dim * width), 0x5A, np.uint8)
        self.codes = [upload(ctx, self.fill) for _ in range(2)]
        self.scales = [upload(ctx, np.full((pages, heads, page), 7.0, np.float32)) for _ in range(2)]
        self.desc = qattn.make_kv_cache(self.codes[0].ptr, self.codes[1].ptr, pages, page, heads, dim,
                                        qattn.BF16 if bf16 else qattn.F16,
                                        {"16bit": qattn.KV_16BIT, "e4m3": qattn.KV_E4M3, "int8": qattn.KV_INT8}[form],
                                        self.scales[0].ptr, self.scales[1].ptr)

    def read(self, which):
        return (self.codes[which].read(np.uint8, self.fill.shape),
                self.scales[which].read(np.float32, self.fill.shape[:3]))

    def free(self):
        for b in self.codes + self.scales:
            b.free()


def special_rows(rng, tokens, heads, dim, bf16):
    """Ordinary vectors, and among them the ones where a quantiser goes wrong."""
    x = rng.standard_normal((tokens, heads, dim)) * np.exp(2 * rng.standard_normal((tokens, heads, 1)))
    kinds = [np.zeros(dim), np.full(dim, 1e-7 if not bf16 else 1e-35), np.full(dim, -448.0), np.full(dim, 449.0),
             np.where(np.arange(dim) == 3, np.inf, 1.0), np.where(np.arange(dim) % 2, np.nan, -2.5),
             np.full(dim, -np.inf), np.where(np.arange(dim) < 2, 60000.0, 1e-4),
             np.linspace(-127, 127, dim), np.full(dim, 3.3e38 if bf16 else 65504.0),
             np.where(np.arange(dim) == 0, 448.0, np.arange(dim) * 2.0 ** -9 + 2.0 ** -10),
             np.full(dim, 2.0 ** -101 if bf16 else 2.0 ** -24)]
    for i in range(min(tokens, len(kinds))):
        x[i, i % heads] = kinds[i]
    return ref.to_bits(x, bf16)


@pytest.mark.parametrize("tokens,heads,dim,page,bf16,form,pad", [
    (1, 8, 128, 64, False, "e4m3", 0), (1, 1, 64, 16, True, "int8", 0), (77, 8, 128, 64, False, "int8", 0),
    (77, 3, 64, 16, True, "e4m3", 8), (200, 4, 128, 32, True, "e4m3", 0), (200, 8, 64, 128, False, "e4m3", 1024),
    (130, 5, 128, 16, True, "int8", 24), (64, 2, 64, 4096, False, "int8", 0), (90, 8, 128, 64, False, "16bit", 0),
    (90, 3, 64, 16, True, "16bit", 8), (3000, 8, 128, 64, False, "e4m3", 0)])
def test_kv_write_and_read(ctx, qattn, tokens, heads, dim, page, bf16, form, pad):
    print("kv", tokens, heads, dim, page, bf16, form, pad, flush=True)
    rng = rng_of(tokens + dim + page)
    pages = tokens // page + 3
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    padded = slots.copy()
    if tokens > 5:  # padding rows: nothing written
        padded[::5] = rng.choice([-1, pages * page, 1 << 40, -(1 << 62)], len(padded[::5]))
    pool = Pool(ctx, qattn, pages, page, heads, dim, bf16, form)
    stride = heads * dim + pad
    rows = []
    for _ in range(2):
        x = np.zeros((tokens, stride), np.uint16)
        x[:, :heads * dim] = special_rows(rng, tokens, heads, dim, bf16).reshape(tokens, -1)
        rows.append(x)
    bufs = [upload(ctx, x) for x in rows]
    bs = upload(ctx, padded)
    ctx.kv_write(pool.desc, bufs[0].ptr, bufs[1].ptr, bs.ptr, tokens, stride, stride)
    ctx.synchronize()
    kept = (padded >= 0) & (padded < pages * page)
    at = (padded[kept] // page, slice(None), padded[kept] % page)
    want = []
    for which, x in enumerate(rows):
        codes, scales = pool.read(which)
        bits = x[:, :heads * dim].reshape(tokens, heads, dim)
        expect, expect_scale = pool.fill.copy(), np.full(codes.shape[:3], 7.0, np.float32)
        if form == "16bit":
            expect[at] = bits[kept].view(np.uint8)
            value = ref.from_bits(bits, bf16)
        else:
            c, s = ref.quantise(ref.from_bits(bits, bf16), form, bf16)
            expect[at], expect_scale[at] = c[kept], s[kept]
            product = np.float32(1) * (c.view(np.int8).astype(np.float32) if form == "int8" else
                                       ref.e4m3_values()[c].astype(np.float32)) * s[..., None]
            value = product.astype(np.float64)
        codes_nan = codes.copy()
        if form == "e4m3":  # a NaN code has either sign
            codes_nan = np.where(codes & 127 == ref.NAN_CODE, ref.NAN_CODE, codes)
        assert np.array_equal(codes_nan, expect)
        assert np.array_equal(scales, expect_scale)
        out = ref.to_bits(np.where(kept[:, None, None], value, 0), bf16)
        held = np.isfinite(ref.from_bits(bits, bf16)) & kept[:, None, None]
        assert np.isfinite(ref.from_bits(out, bf16)[held]).all()
        want.append(np.where(kept[:, None, None], bits, 0) if form == "16bit" else out)
    outs = [upload(ctx, np.full((tokens, stride), 0x7E11, np.uint16)) for _ in range(2)]
    ctx.kv_read(pool.desc, bs.ptr, tokens, outs[0].ptr, outs[1].ptr, stride, stride)
    ctx.synchronize()
    for b, expect in zip(outs, want):
        got = b.read(np.uint16, (tokens, stride))
        assert (got[:, heads * dim:] == 0x7E11).all()
        got = got[:, :heads * dim].reshape(tokens, heads, dim)
        same = got == expect
        if form == "e4m3":
            same |= np.isnan(ref.from_bits(got, bf16)) & np.isnan(ref.from_bits(expect, bf16))
        assert same.all(), (got[~same][:5], expect[~same][:5])
    for b in bufs + outs + [bs]:
        b.free()
    pool.free()


def test_kv_read_repeats_slots_and_zero_tokens(ctx, qattn):
    pool = Pool(ctx, qattn, 2, 16, 2, 64, False, "16bit")
    rows = ref.to_bits(rng_of(1).standard_normal((2, 128)), False)
    b, slots, out = upload(ctx, rows), upload(ctx, np.array([5, 30, 5, 5], np.int64)), ctx.alloc(4 * 256)
    ctx.kv_write(pool.desc, b.ptr, b.ptr, slots.ptr, 2)
    ctx.kv_write(pool.desc, None, None, None, 0)
    ctx.kv_read(pool.desc, slots.ptr, 4, out.ptr, out.ptr)
    ctx.synchronize()
    assert np.array_equal(out.read(np.uint16, (4, 128)), rows[[0, 1, 0, 0]])
    for x in (b, slots, out):
        x.free()
    pool.free()

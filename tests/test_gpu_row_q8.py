"""Rows into 8 bits (qattn_quantize_q8, qattn_rmsnorm_q8) against their definitions, on the GPU."""
import numpy as np
import pytest

import shared_ref as ref
import w4_ref

pytestmark = pytest.mark.gpu
rng_of = np.random.default_rng
PATTERN = 0x5A


def half_words(a):
    return np.ascontiguousarray(a, np.uint16)


class Rows:
    """Rows in device memory, `pad` elements apart, between guards whose bytes have to stay."""

    def __init__(self, ctx, rows, width, pad, size):
        self.shape, self.stride, self.size = (rows, width), width + pad, size
        self.fill = np.full((rows * self.stride + 64) * size, PATTERN, np.uint8)
        self.buf = ctx.upload(self.fill)
        self.ptr = self.buf.ptr + 32 * size

    def write(self, values):
        image = self.fill.copy()
        self._view(image, values.dtype)[:] = values
        self.buf.write(image)
        self.fill = image

    def _view(self, image, dtype):
        body = image[32 * self.size:32 * self.size + self.shape[0] * self.stride * self.size]
        return body.view(dtype).reshape(self.shape[0], self.stride)[:, :self.shape[1]]

    def read(self, dtype):
        """The rows; what lies around them has to be as it was."""
        image = self.buf.read(np.uint8, self.fill.shape)
        values = self._view(image, dtype).copy()
        self._view(image, dtype)[:] = self._view(self.fill, dtype)
        assert np.array_equal(image, self.fill), "bytes between or around the rows changed"
        return values

    def free(self):
        self.buf.free()


def some_rows(rng, rows, width, bf16):
    x = rng.standard_normal((rows, width)) * np.exp(0.7 * rng.standard_normal(width)) * np.exp(rng.standard_normal((rows, 1)))
    return ref.to_bits(x, bf16)


def scale_bound(width, norm):
    """amax / 127 rounds once.  With the norm: t's product; the sum of squares (each of a sum rounded once) passes
    at most 32 fused additions in a lane, 6 between lanes and 16 between wavefronts, all terms positive, and a root
    halves its error; the quotient by the width, eps, the root (1 ulp) and the reciprocal; the last product."""
    roundings = 1 if not norm else 1 + 1 + (32 + 6 + 16 + 2) / 2 + 0.5 + 0.5 + 2 + 1 + 1
    return roundings * 1.01 * 2.0 ** -24


def check_scales(got, want, width, norm):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(got - want)[fine] <= want[fine] * scale_bound(width, norm) + 2.0 ** -149).all()


WIDTHS = [8, 64, 72, 128, 136, 256, 264, 512, 520, 1000, 1024, 1032, 2048, 2056, 4096, 5000, 8192, 8200, 16384, 32760, 32768]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,width", [(3, w) for w in WIDTHS] + [(1, 1024), (5, 1024), (2000, 1024), (777, 136), (301, 2560), (2001, 64), (1003, 128), (513, 256), (33, 8)])
def test_quantize(ctx, qattn, rows, width, bf16):
    print("quantize", rows, width, bf16, flush=True)
    rng = rng_of(rows * 7 + width)
    bits = some_rows(rng, rows, width, bf16)
    for pad in (0, 24):
        x, codes, scales = Rows(ctx, rows, width, pad, 2), Rows(ctx, rows, width, pad, 1), Rows(ctx, 1, rows, 0, 4)
        x.write(bits)
        ctx.quantize_q8(x.ptr, codes.ptr, scales.ptr, rows, width, qattn.BF16 if bf16 else qattn.F16, x.stride, codes.stride)
        ctx.synchronize()
        want, scale = w4_ref.quantize_q8(bits, bf16)
        got = codes.read(np.int8)
        assert np.array_equal(got, want)
        check_scales(scales.read(np.float32)[0], scale, width, False)
        assert np.array_equal(x.read(np.uint16), bits)
        # The value that a code stands for is half a step away at most, and two roundings of 127.
        value = ref.from_bits(bits, bf16)
        assert (np.abs(got * scale[:, None] - value) <= scale[:, None] * (0.5 + 127 * 2.0 ** -23)).all()
        for b in (x, codes, scales):
            b.free()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,width", [(3, w) for w in WIDTHS] + [(1, 1024), (5, 1024), (1419, 1024), (777, 136), (2001, 64), (1003, 128), (513, 256), (33, 8)])
@pytest.mark.parametrize("sum_in", [None, "own", "x", "residual"])
def test_rmsnorm(ctx, qattn, rows, width, bf16, sum_in):
    print("rmsnorm", rows, width, bf16, sum_in, flush=True)
    rng = rng_of(rows * 5 + width)
    bits, more = some_rows(rng, rows, width, bf16), some_rows(rng, rows, width, bf16)
    weight = (1 + 0.3 * rng.standard_normal(width)).astype(np.float32)
    weight[rng.integers(0, width)] = 0
    eps = 1e-6 if width % 16 else 1e-3
    w = ctx.upload(weight)
    x, r, s = (Rows(ctx, rows, width, pad, 2) for pad in (8, 0, 16))
    codes, scales = Rows(ctx, rows, width, 16, 1), Rows(ctx, 1, rows, 0, 4)
    x.write(bits)
    r.write(more)
    out = {None: None, "own": s, "x": x, "residual": r}[sum_in]
    ctx.rmsnorm_q8(x.ptr, w.ptr, codes.ptr, scales.ptr, rows, width, None if out is None else r.ptr,
                   None if out is None else out.ptr, eps, qattn.BF16 if bf16 else qattn.F16, x.stride, r.stride,
                   0 if out is None else out.stride, codes.stride)
    ctx.synchronize()
    want, scale, total = w4_ref.rmsnorm_q8(bits, None if out is None else more, weight, bf16, eps)
    assert np.array_equal(codes.read(np.int8), want)
    check_scales(scales.read(np.float32)[0], scale, width, True)
    for rows_of, before in ((x, bits), (r, more)):
        assert np.array_equal(rows_of.read(np.uint16), total if out is rows_of else before)
    if out is s:
        assert np.array_equal(s.read(np.uint16), total)
    for b in (w, x, r, s, codes, scales):
        b.free()


def odd_rows(width, bf16):
    """Zeros, an infinity, a NaN, next to nothing, subnormals, the largest values, one value among zeros, ties."""
    rng = rng_of(width)
    x = rng.standard_normal((16, width))
    x[0] = 0
    x[1, width // 2] = np.inf
    x[2, -1] = -np.inf
    x[3, 0] = np.nan
    x[4] *= 2.0 ** -24
    x[5] = np.where(x[5] > 0, 1, -1) * (3.38e38 if bf16 else 65504.0)
    x[6] = 0
    x[6, width - 1] = -3.0
    x[7] = (np.arange(width) % 255 - 127) / 2  # amax 63.5: factor 2, every value a whole number
    x[8] = (np.arange(width) % 128) / 2
    x[8, 0] = 127.0                            # factor 1: halves are ties
    x[9] = -0.0
    if bf16:
        x[10] *= 2.0 ** -120
        x[11] *= 2.0 ** -100
        x[12] *= 2.0 ** -126
        x[13] *= 2.0 ** 66                     # squares pass f32's range
        x[14] *= 2.0 ** 60
    return ref.to_bits(x, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("width", [64, 1024, 2560, 9000])
def test_rows_that_hold_little_or_too_much(ctx, qattn, width, bf16):
    bits = odd_rows(width, bf16)
    rows, dtype = len(bits), qattn.BF16 if bf16 else qattn.F16
    weight, none = np.ones(width, np.float32), ref.to_bits(np.zeros((rows, width)), bf16)
    x, r, s, w = ctx.upload(bits), ctx.upload(none), ctx.upload(none), ctx.upload(weight)
    codes, scales = ctx.alloc(rows * width), ctx.alloc(rows * 4)
    calls = [(lambda: ctx.quantize_q8(x.ptr, codes.ptr, scales.ptr, rows, width, dtype), w4_ref.quantize_q8(bits, bf16), False)]
    for eps in (1e-6, 0.0):
        calls.append((lambda eps=eps: ctx.rmsnorm_q8(x.ptr, w.ptr, codes.ptr, scales.ptr, rows, width, eps=eps, dtype=dtype),
                      w4_ref.rmsnorm_q8(bits, None, weight, bf16, eps), True))
        calls.append((lambda eps=eps: ctx.rmsnorm_q8(x.ptr, w.ptr, codes.ptr, scales.ptr, rows, width, r.ptr, s.ptr, eps, dtype),
                      w4_ref.rmsnorm_q8(bits, none, weight, bf16, eps), True))
    for call, want, norm in calls:
        call()
        ctx.synchronize()
        got, scale = codes.read(np.int8, (rows, width)), scales.read(np.float32, (rows,)).astype(np.float64)
        assert np.array_equal(got, want[0])
        assert np.isnan(scale[[1, 2, 3]]).all() and (got[[1, 2, 3]] == 0).all()
        assert scale[0] == 0 and scale[9] == 0
        if not norm:
            check_scales(scale, want[1], width, False)
        else:
            # Squares below f32's normal range lose their digits: rows that small are held to 2^-6 where eps is 0.
            normal = np.isnan(want[1]) | (np.abs(ref.from_bits(bits, bf16)).max(-1) > 2.0 ** -50)
            check_scales(scale[normal], want[1][normal], width, True)
    for b in (x, r, s, w, codes, scales):
        b.free()


def test_norm_is_the_frameworks_own(ctx, qattn):
    """The values that the codes stand for are those of qattn_rmsnorm before its rounding: half a step away from it,
    and its half step.  The stored sums are equal."""
    rng = rng_of(3)
    rows, width = 50, 1024
    x, r = (rng.standard_normal((rows, width)).astype(np.float16) for _ in range(2))
    weight = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32)
    bx, bs, br, bw = ctx.upload(x), ctx.upload(x), ctx.upload(r), ctx.upload(weight)
    out, codes, scales = ctx.alloc(rows * width * 2), ctx.alloc(rows * width), ctx.alloc(rows * 4)
    ctx.rmsnorm(bx.ptr, bw.ptr, out.ptr, rows, width, br.ptr)
    ctx.rmsnorm_q8(bs.ptr, bw.ptr, codes.ptr, scales.ptr, rows, width, br.ptr, bs.ptr)
    ctx.synchronize()
    assert np.array_equal(bx.read(np.uint16, (rows, width)), bs.read(np.uint16, (rows, width)))
    y = out.read(np.float16, (rows, width)).astype(np.float64)
    scale = scales.read(np.float32, (rows,)).astype(np.float64)[:, None]
    got = codes.read(np.int8, (rows, width)) * scale
    assert (np.abs(got - y) <= scale * 0.5001 + ref.half_step(y, False) * 1.01).all()
    for b in (bx, bs, br, bw, out, codes, scales):
        b.free()

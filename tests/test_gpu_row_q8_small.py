"""The norm's scales of rows whose squares leave f32's range downwards, on the GPU: as right as any other row's,
whatever eps is."""
import numpy as np
import pytest

import shared_ref as ref
import w4_ref
from test_gpu_row_q8 import check_scales, odd_rows

pytestmark = pytest.mark.gpu
rng_of = np.random.default_rng

# Exponents of a row's largest values and of the gains: next to nothing, about the sizes where squares leave f32,
# subnormal values that their gains raise, and ordinary rows.
SIZES = [(-98, 0), (-90, 0), (-76, 0), (-75, 0), (-66, 0), (-63, 0), (-50, 0), (-42, -50), (-41, -40), (-38, 0), (-126, 60),
         (-132, 100), (-120, 126), (0, 0), (40, -60), (45, 0)]
EPS = [0.0, 2.0 ** -140, 1e-38, 2.0 ** -101, 2.0 ** -100, 1e-20, 1e-6]


def small_rows(rng, width, top):
    x = rng.standard_normal((4, width)) * 2.0 ** (top - 2)
    x[1, 1:] = 0                                   # one value
    x[1, 0] = 2.0 ** top
    x[2, :] = -2.0 ** (top - 3)                    # all alike
    x[3, ::2] *= 2.0 ** -20                        # squares far apart
    return ref.to_bits(x, True)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("width", [8, 64, 120, 256, 512, 1024, 2048, 2560, 8192, 9000, 32768])
def test_rows_whose_squares_vanish(ctx, qattn, width, residual):
    rng = rng_of(width)
    for top, gain in SIZES:
        bits = small_rows(rng, width, top)
        rows = len(bits)
        more = ref.to_bits(rng.standard_normal((rows, width)) * 2.0 ** (top - 3), True) if residual else None
        weight = ((1 + 0.2 * rng.standard_normal(width)) * 2.0 ** gain).astype(np.float32)
        x, w = ctx.upload(bits), ctx.upload(weight)
        r, s = (ctx.upload(more), ctx.upload(more)) if residual else (None, None)
        codes, scales = ctx.alloc(rows * width), ctx.alloc(rows * 4)
        for eps in EPS:
            want, scale, total = w4_ref.rmsnorm_q8(bits, more, weight, True, float(np.float32(eps)))
            ctx.rmsnorm_q8(x.ptr, w.ptr, codes.ptr, scales.ptr, rows, width, r.ptr if residual else None,
                           s.ptr if residual else None, eps, qattn.BF16)
            ctx.synchronize()
            got = scales.read(np.float32, (rows,))
            assert np.isfinite(scale).all() and np.isfinite(got).all(), (top, gain, eps, got)
            assert np.array_equal(codes.read(np.int8, (rows, width)), want), (top, gain, eps)
            check_scales(got, scale, width, True)
            if residual:
                assert np.array_equal(s.read(np.uint16, (rows, width)), total)
        for b in (x, w, r, s, codes, scales):
            if b is not None:
                b.free()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("width", [64, 1024, 2560, 9000])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_odd_rows_are_held_to_the_same_bound(ctx, qattn, width, bf16, eps):
    """Rows of zeros, next to nothing, subnormals, the largest values: every scale, the smallest rows' too."""
    bits = odd_rows(width, bf16)
    rows, weight = len(bits), np.ones(width, np.float32)
    x, w, codes, scales = ctx.upload(bits), ctx.upload(weight), ctx.alloc(rows * width), ctx.alloc(rows * 4)
    want = w4_ref.rmsnorm_q8(bits, None, weight, bf16, float(np.float32(eps)))
    ctx.rmsnorm_q8(x.ptr, w.ptr, codes.ptr, scales.ptr, rows, width, eps=eps, dtype=qattn.BF16 if bf16 else qattn.F16)
    ctx.synchronize()
    assert np.array_equal(codes.read(np.int8, (rows, width)), want[0])
    got = scales.read(np.float32, (rows,))
    assert not np.isinf(got).any()
    check_scales(got, want[1], width, True)
    for b in (x, w, codes, scales):
        b.free()

"""The operators of a forward with 8-bit activations over tensors whose offsets pass 32 bits: rows 2^22 elements apart,
weights of 2^22 rows."""
import numpy as np
import pytest

import shared_ref as ref
import w4_ref
from test_gpu_row_q8 import check_scales, some_rows
from test_gpu_w4 import check

pytestmark = pytest.mark.gpu
rng_of = np.random.default_rng
FAR = 1 << 22


def some(M):
    """Rows about the tiles' edges and beyond 32 bits."""
    return sorted({r for e in (0, 32, 64, 128, 256, 512, 1024, 2048, M) for r in (e - 1, e) if 0 <= r < M})


def put(buf, rows, values, stride):
    for r, v in zip(rows, values):
        buf.write(np.ascontiguousarray(v), r * stride)


def get(buf, rows, width, dtype, stride):
    size = np.dtype(dtype).itemsize
    return np.stack([buf.read(np.uint8, (width * size,), r * stride * size).view(dtype) for r in rows])


# Sizes of every kernel of the products.
@pytest.mark.parametrize("M,K,N,swiglu", [(2500, 1056, 4090, False), (2500, 1024, 2048, True), (3000, 160, 4090, False), (3000, 160, 2048, True),
                                          (3000, 128, 2040, False), (1500, 128, 1400, False), (2200, 64, 2050, False),
                                          (1419, 2048, 1020, False), (1500, 256, 512, True), (700, 96, 1023, False), (333, 2080, 999, False),
                                          (1000, 288, 1000, False)])
def test_products_of_rows_far_apart(ctx, qattn, M, K, N, swiglu):
    print("far", M, K, N, swiglu, flush=True)
    rng = rng_of(M + K + N)
    codes, groups, scales = w4_ref.random_weights(rng, 2 * N if swiglu else N, K)
    image = qattn.w4_pack(w4_ref.nibbles(codes), groups, scales)
    rows = some(M)
    x, x_scale = rng.integers(-128, 128, (len(rows), K)).astype(np.int8), np.zeros(M, np.float32)
    x_scale[rows] = rng.random(len(rows)) / (40 * np.sqrt(K)) * (20 if swiglu else 1)
    w, s = ctx.upload(image), ctx.upload(x_scale)
    bx, y = ctx.alloc((M - 1) * FAR + K), ctx.alloc(((M - 1) * FAR + N) * 2)
    put(bx, rows, x, FAR)
    call = ctx.w4_matmul_swiglu if swiglu else ctx.w4_matmul
    call(bx.ptr, s.ptr, M, K, w.ptr, image.nbytes, N, y.ptr, qattn.F16, FAR, FAR)
    ctx.synchronize()
    got = ref.from_bits(get(y, rows, N, np.uint16, FAR), False)
    want = w4_ref.product(x, x_scale[rows], codes, groups, scales)
    if swiglu:
        g, u = want[:, :N], want[:, N:]
        check(got, w4_ref.swiglu(g, u), w4_ref.swiglu_bound(g, u, False), x_scale[rows], False)
    else:
        check(got, want, w4_ref.product_bound(want, False), x_scale[rows], False)
    for b in (w, s, bx, y):
        b.free()


def test_rows_into_8_bits_far_apart(ctx, qattn):
    M, width = 1100, 264
    rng = rng_of(4)
    rows = some(M)
    bits, more = (some_rows(rng, len(rows), width, False) for _ in range(2))
    weight = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32)
    x, r, total = (ctx.alloc(((M - 1) * FAR + width) * 2) for _ in range(3))
    codes, scales, w = ctx.alloc((M - 1) * FAR + width), ctx.alloc(M * 4), ctx.upload(weight)
    put(x, rows, bits, 2 * FAR)
    put(r, rows, more, 2 * FAR)
    ctx.quantize_q8(x.ptr, codes.ptr, scales.ptr, M, width, qattn.F16, FAR, FAR)
    ctx.synchronize()
    want = w4_ref.quantize_q8(bits, False)
    assert np.array_equal(get(codes, rows, width, np.int8, FAR), want[0])
    check_scales(scales.read(np.float32, (M,))[rows], want[1], width, False)
    ctx.rmsnorm_q8(x.ptr, w.ptr, codes.ptr, scales.ptr, M, width, r.ptr, total.ptr, 1e-6, qattn.F16, FAR, FAR, FAR, FAR)
    ctx.synchronize()
    want = w4_ref.rmsnorm_q8(bits, more, weight, False, 1e-6)
    assert np.array_equal(get(codes, rows, width, np.int8, FAR), want[0])
    assert np.array_equal(get(total, rows, width, np.uint16, FAR), want[2])
    check_scales(scales.read(np.float32, (M,))[rows], want[1], width, True)
    for b in (x, r, total, codes, scales, w):
        b.free()


def test_rows_into_8_bits_beyond_a_grids_dimension(ctx, qattn):
    """A workgroup to a row, and more rows than a launch has workgroups in one dimension."""
    M, width = (1 << 20) + 7, 2056
    rng = rng_of(8)
    rows = [0, 1, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, M - 1]
    bits = some_rows(rng, len(rows), width, True)
    x, codes, scales = ctx.alloc(M * width * 2), ctx.alloc(M * width), ctx.alloc(M * 4)
    put(x, rows, bits, 2 * width)
    ctx.quantize_q8(x.ptr, codes.ptr, scales.ptr, M, width, qattn.BF16)
    ctx.synchronize()
    want = w4_ref.quantize_q8(bits, True)
    assert np.array_equal(get(codes, rows, width, np.int8, width), want[0])
    check_scales(scales.read(np.float32, (M,))[rows], want[1], width, False)
    for b in (x, codes, scales):
        b.free()


def test_weights_of_most_rows(ctx, qattn):
    """2^22 weight rows, whose codes take 4 GiB and more: the last columns are those of the last rows by themselves."""
    K, N, last = 2080, 1 << 22, 528
    blocks, tiles = -(-K // 128), N // 16
    size = qattn.lib().qattn_w4_bytes(K, N)
    assert tiles * blocks * 1024 > 1 << 32 and size == tiles * blocks * 1088 + 4 * N
    rng = rng_of(6)
    w = ctx.alloc(size)
    chunk = rng.integers(0, 256, 1 << 26).astype(np.uint8)
    for at in range(0, tiles * blocks * 1024, chunk.nbytes):
        chunk[:8] = rng.integers(0, 256, 8)
        w.write(chunk[:min(chunk.nbytes, tiles * blocks * 1024 - at)], at)
    # Every pair of a multiplier and a zero point that fits; columns past K hold nothing.
    groups = np.resize(w4_ref.pairs(), 1 << 20)
    part = groups.reshape(-1, 16, 4)[:blocks * 256].reshape(-1, blocks, 16, 4)
    part[:, -1, :, 1:] = 0
    part = np.ascontiguousarray(part).reshape(-1)
    start = tiles * blocks * 1024
    for at in range(0, tiles * blocks * 64, part.nbytes):
        w.write(part[:min(part.nbytes, tiles * blocks * 64 - at)], start + at)
    scales = (rng.standard_normal(N) * 0.01).astype(np.float32)
    w.write(scales, start + tiles * blocks * 64)
    few = last // 16
    take = lambda first, length: w.read(np.uint8, (length,), first)  # noqa: E731
    alone = np.concatenate([take((tiles - few) * blocks * 1024, few * blocks * 1024), take(start + (tiles - few) * blocks * 64, few * blocks * 64),
                            scales[-last:].view(np.uint8)])
    codes, group_bytes, s = w4_ref.taken_apart(alone, K, last)
    b_alone = ctx.upload(alone)
    for M in (3, 40, 300):
        x, x_scale = rng.integers(-128, 128, (M, K)).astype(np.int8), (rng.random(M) / 2000).astype(np.float32)
        bx, bs = ctx.upload(x), ctx.upload(x_scale)
        y, y_alone = ctx.alloc(M * N * 2), ctx.alloc(M * last * 2)
        ctx.w4_matmul(bx.ptr, bs.ptr, M, K, w.ptr, size, N, y.ptr)
        ctx.w4_matmul(bx.ptr, bs.ptr, M, K, b_alone.ptr, alone.nbytes, last, y_alone.ptr)
        ctx.synchronize()
        few_bits = y_alone.read(np.uint16, (M, last))
        want = w4_ref.product(x, x_scale, codes, group_bytes, s)
        check(ref.from_bits(few_bits, False), want, w4_ref.product_bound(want, False), x_scale, False)
        for m in (0, 1, M // 2, M - 1):
            row = y.read(np.uint16, (last,), (m * N + N - last) * 2)
            assert np.array_equal(row, few_bits[m]), (M, m)
        for b in (bx, bs, y, y_alone):
            b.free()
    w.free()
    b_alone.free()


@pytest.mark.parametrize("N", [8, 112])
def test_most_rows(ctx, qattn, N):
    """2^24 - 1 rows: as many workgroups as a call may have, and results past 2^31 bytes."""
    M, K = (1 << 24) - 1, 32
    rng = rng_of(N)
    codes, groups, scales = w4_ref.random_weights(rng, N, K)
    image = qattn.w4_pack(w4_ref.nibbles(codes), groups, scales)
    block, block_scale = rng.integers(-128, 128, (1 << 20, K)).astype(np.int8), (rng.random(1 << 20) / 300).astype(np.float32)
    bx, bs, w, y = ctx.alloc(M * K), ctx.alloc(M * 4), ctx.upload(image), ctx.alloc(M * N * 2)
    for at in range(0, M, 1 << 20):
        bx.write(block[:M - at], at * K)
        bs.write(block_scale[:M - at], at * 4)
    ctx.w4_matmul(bx.ptr, bs.ptr, M, K, w.ptr, image.nbytes, N, y.ptr)
    ctx.synchronize()
    rows = np.concatenate([np.arange(300), np.arange(M - 300, M), rng.integers(0, M, 50)])
    got = np.stack([y.read(np.uint16, (N,), int(r) * N * 2) for r in rows])
    at = rows % (1 << 20)
    want = w4_ref.product(block[at], block_scale[at], codes, groups, scales)
    check(ref.from_bits(got, False), want, w4_ref.product_bound(want, False), block_scale[at], False)
    for b in (bx, bs, w, y):
        b.free()

"""Products of 8-bit rows with 4-bit weights (qattn_w4_matmul, qattn_w4_matmul_swiglu) against their definitions in
64 bits, on the GPU."""
import numpy as np
import pytest

import shared_ref as ref
import w4_ref
from test_gpu_row_q8 import Rows

pytestmark = pytest.mark.gpu
rng_of = np.random.default_rng


class Weights:
    def __init__(self, ctx, qattn, rng, N, K):
        self.codes, self.groups, self.scales = w4_ref.random_weights(rng, N, K)
        image = qattn.w4_pack(w4_ref.nibbles(self.codes), self.groups, self.scales)
        # Behind the image, and so behind every read of it, lies something that is no weight.
        self.bytes, self.buf = image.nbytes, ctx.upload(np.concatenate([image, np.full(4096, 0xA5, np.uint8)]))
        self.ptr = self.buf.ptr

    def product(self, x, x_scale):
        return w4_ref.product(x, x_scale, self.codes, self.groups, self.scales)

    def free(self):
        self.buf.free()


def check(got, want, bound, x_scale, bf16):
    bad = np.isnan(x_scale)
    assert np.isnan(got[bad]).all()
    got, want, bound = got[~bad], want[~bad], bound[~bad]
    # fp16 ends at 65504: from half a step above, 65520, a value rounds to infinity.
    most, over = (np.inf if bf16 else 65520.0), np.isinf(got)
    assert (np.abs(want) + bound >= most)[over].all() and (np.sign(got) == np.sign(want))[over].all()
    assert over[np.abs(want) - bound >= most].all()
    off = np.abs(got - want)[~over] / bound[~over]
    assert (off <= 1).all(), float(off.max())


def run_case(ctx, qattn, M, K, N, bf16, swiglu, pad=(0, 0), seed=0):
    print("w4", M, K, N, "bf16" if bf16 else "f16", "swiglu" if swiglu else "", pad, flush=True)
    rng = rng_of(seed + 31 * M + 7 * K + N)
    w = Weights(ctx, qattn, rng, 2 * N if swiglu else N, K)
    x = rng.integers(-128, 128, (M, K)).astype(np.int8)
    x_scale = (np.abs(rng.standard_normal(M)) / (40 * np.sqrt(K))).astype(np.float32)
    if M > 4:
        x_scale[1], x_scale[3], x[2] = np.nan, 0, -128
    if swiglu:
        x_scale *= 20  # gates of several units
    rows, y, s = Rows(ctx, M, K, pad[0], 1), Rows(ctx, M, N, -N % 8 + pad[1], 2), ctx.upload(x_scale)
    rows.write(x)
    call = ctx.w4_matmul_swiglu if swiglu else ctx.w4_matmul
    call(rows.ptr, s.ptr, M, K, w.ptr, w.bytes, N, y.ptr, qattn.BF16 if bf16 else qattn.F16, rows.stride, y.stride)
    ctx.synchronize()
    got = ref.from_bits(y.read(np.uint16), bf16)
    want = w.product(x, x_scale)
    if swiglu:
        g, u = want[:, :N], want[:, N:]
        check(got, w4_ref.swiglu(g, u), w4_ref.swiglu_bound(g, u, bf16), x_scale, bf16)
    else:
        check(got, want, w4_ref.product_bound(want, bf16), x_scale, bf16)
    for b in (rows, y, s, w):
        b.free()


# Rows and columns about the tiles' edges, K about the blocks' (32 and 128), and the sizes of real projections.
CASES = [(1, 32, 1), (1, 64, 17), (2, 96, 16), (15, 128, 33), (16, 160, 48), (17, 256, 31), (1, 4096, 1000), (1, 8192, 64),
         (16, 1024, 4096), (31, 1024, 100), (33, 992, 129), (50, 2048, 1024), (64, 224, 257), (65, 512, 513), (100, 1024, 1001),
         (129, 1056, 640), (255, 288, 1024), (257, 384, 250), (333, 2592, 1001), (500, 1024, 1024), (1000, 96, 77),
         (1419, 2048, 1024), (2049, 1120, 1000), (4000, 128, 4096), (8000, 64, 40)]
# Each kernel with a last tile of few rows, and columns that end inside its last 16 or its last 8.
CASES += [(1300, 320, 1003), (1500, 2080, 1023), (4097, 160, 2052), (3841, 288, 4085), (20000, 64, 130), (2400, 256, 2049),
          (33, 96, 40001), (60, 4096, 1025), (100, 8192, 290), (7, 16384, 50), (2401, 1056, 4090), (1900, 96, 2003),
          (999, 2080, 1021), (195, 288, 4090), (64, 1024, 20001), (64, 2080, 2045)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,K,N", CASES)
def test_product(ctx, qattn, M, K, N, bf16):
    run_case(ctx, qattn, M, K, N, bf16, False)


GATE_CASES = [(1, 32, 32), (1, 4096, 96), (5, 160, 64), (16, 1024, 2816), (17, 96, 32), (50, 1024, 1024), (64, 256, 96),
              (130, 1056, 160), (257, 128, 2816), (700, 512, 416), (1500, 1024, 1024), (3000, 64, 288), (3900, 192, 1952),
              (5001, 288, 2080), (40, 4096, 2048), (90, 4096, 1056), (9, 8224, 64), (2401, 1056, 2048), (199, 1056, 2048),
              (100, 2080, 2016), (1411, 2080, 512), (1900, 96, 1024)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,K,N", GATE_CASES)
def test_swiglu(ctx, qattn, M, K, N, bf16):
    run_case(ctx, qattn, M, K, N, bf16, True)


@pytest.mark.parametrize("M,K,N,swiglu", [(3, 96, 50, False), (70, 1024, 200, False), (600, 160, 320, False), (2100, 256, 1024, False),
                                          (40, 128, 64, True), (900, 96, 320, True)])
def test_rows_apart(ctx, qattn, M, K, N, swiglu):
    """Strides beyond the width: what lies between the rows is not read into sums and stays as it was."""
    run_case(ctx, qattn, M, K, N, False, swiglu, pad=(48, 40))


def test_extreme_sums(ctx, qattn):
    """The largest sums there are: K = 65536 of -128 * -128 and -128 * 127, and zero points at both ends."""
    M, K, N = 3, 65536, 20
    groups = np.full((N, K // 32), 15 | 8 << 4, np.uint8)
    groups[1] = 8                  # zero point 0: weights 0 .. 120
    groups[2] = 8 | 15 << 4        # zero point 15: weights -120 .. 0
    codes = np.zeros((N, K), np.uint8)
    codes[1], codes[3:] = 15, 15
    scales = np.ones(N, np.float32)
    x = np.full((M, K), -128, np.int8)
    x[1], x[2, ::2] = 127, 127
    image = qattn.w4_pack(w4_ref.nibbles(codes), groups, scales)
    x_scale = np.full(M, 2.0 ** -20, np.float32)
    w, bx, bs, y = ctx.upload(image), ctx.upload(x), ctx.upload(x_scale), ctx.alloc(M * 24 * 2)
    ctx.w4_matmul(bx.ptr, bs.ptr, M, K, w.ptr, image.nbytes, N, y.ptr, qattn.BF16, ldy=24)
    ctx.synchronize()
    got = ref.from_bits(y.read(np.uint16, (M, 24))[:, :N], True)
    want = w4_ref.product(x, x_scale, codes, groups, scales)
    assert np.abs(want).max() > 2.0 ** 9
    assert (np.abs(got - want) <= w4_ref.product_bound(want, True)).all()
    for b in (w, bx, bs, y):
        b.free()


def test_swiglu_of_far_gates(ctx, qattn):
    """Gates beyond the exponential's range on both sides: the gate itself, or nothing."""
    M, K, n = 5, 32, 32
    codes, groups = np.full((2 * n, K), 8, np.uint8), np.full((2 * n, 1), 1 | 7 << 4, np.uint8)  # weights of 1
    scales = np.ones(2 * n, np.float32)
    scales[n:] = 0.5
    x = np.ones((M, K), np.int8) * np.array([[1], [-1], [1], [-1], [0]], np.int8)
    x_scale = np.array([10, 10, 2, 3, 1], np.float32)  # gates of 320, -320, 64, -96, 0
    image = qattn.w4_pack(w4_ref.nibbles(codes), groups, scales)
    w, bx, bs, y = ctx.upload(image), ctx.upload(x), ctx.upload(x_scale), ctx.alloc(M * n * 2)
    for bf16 in (False, True):
        ctx.w4_matmul_swiglu(bx.ptr, bs.ptr, M, K, w.ptr, image.nbytes, n, y.ptr, qattn.BF16 if bf16 else qattn.F16)
        ctx.synchronize()
        got = ref.from_bits(y.read(np.uint16, (M, n)), bf16)
        both = w4_ref.product(x, x_scale, codes, groups, scales)
        g, u = both[:, :n], both[:, n:]
        assert (np.abs(got - w4_ref.swiglu(g, u)) <= w4_ref.swiglu_bound(g, u, bf16)).all()
    for b in (w, bx, bs, y):
        b.free()


@pytest.mark.parametrize("K,N,swiglu", [(1024, 1024, False), (2048, 96, False), (256, 2080, False), (1024, 512, True)])
def test_a_row_does_not_depend_on_its_batch(ctx, qattn, K, N, swiglu):
    """Bit for bit the same in launches of 1 to 3,000 rows, whichever kernel takes them."""
    rng = rng_of(K + N)
    w = Weights(ctx, qattn, rng, 2 * N if swiglu else N, K)
    M = 3000
    x = rng.integers(-127, 128, (M, K)).astype(np.int8)
    x_scale = (rng.random(M) / 1000).astype(np.float32)
    bx, bs, y = ctx.upload(x), ctx.upload(x_scale), ctx.alloc(M * N * 2)
    call = ctx.w4_matmul_swiglu if swiglu else ctx.w4_matmul
    call(bx.ptr, bs.ptr, M, K, w.ptr, w.bytes, N, y.ptr)
    ctx.synchronize()
    whole = y.read(np.uint16, (M, N))
    for first, count in ((0, 1), (5, 16), (100, 40), (7, 90), (1000, 300), (64, 700), (2000, 999), (2999, 1), (16, 2000)):
        y.fill_u16(0x7E00)
        call(bx.ptr + first * K, bs.ptr + 4 * first, count, K, w.ptr, w.bytes, N, y.ptr)
        ctx.synchronize()
        assert np.array_equal(y.read(np.uint16, (count, N)), whole[first:first + count]), (first, count)
    for b in (bx, bs, y, w):
        b.free()


def halves(M):
    """(t, scale) whose f32 products lie next to a border of fp16: rounded to f32 first they go one way, at once the other."""
    rng = rng_of(11)
    t, scale = np.zeros(0, np.int64), np.zeros(0, np.float32)
    while len(t) < M:
        a, b = rng.integers(1, 128, 1 << 20), (1 + rng.random(1 << 20)).astype(np.float32)
        exact = a.astype(np.float64) * b.astype(np.float64)
        twice = exact.astype(np.float32).astype(np.float16)
        hit = twice != exact.astype(np.float16)
        t, scale = np.concatenate([t, a[hit]]), np.concatenate([scale, b[hit]])
    return t[:M], scale[:M]


@pytest.mark.parametrize("swiglu", [False, True])
def test_a_rounding_does_not_depend_on_the_kernel(ctx, qattn, swiglu):
    """Products are rounded to f32, then to 16 bits, in every kernel and at every place of a column in it."""
    M, K, N = 6000, 32, 800 if swiglu else 795
    t, scale = halves(M)
    x = np.zeros((M, K), np.int8)
    x[:, 0], x[:, 1] = t, 1
    codes = np.full((2 * N if swiglu else N, K), 8, np.uint8)
    codes[:, 0] += 1                                   # weights of 1 in the first column
    if swiglu:
        codes[N:, 0], codes[N:, 1] = 8, 9              # the up product is the row's scale
    groups, scales = np.full((len(codes), 1), 1 | 8 << 4, np.uint8), np.ones(len(codes), np.float32)
    image = qattn.w4_pack(w4_ref.nibbles(codes), groups, scales)
    ldy = -(-N // 8) * 8
    w, bx, bs, y = ctx.upload(image), ctx.upload(x), ctx.upload(scale), ctx.alloc(M * ldy * 2)
    call = ctx.w4_matmul_swiglu if swiglu else ctx.w4_matmul
    seen = []
    for count in (M, 3000, 1200, 300, 40, 9):
        call(bx.ptr, bs.ptr, count, K, w.ptr, image.nbytes, N, y.ptr, ldy=ldy)
        ctx.synchronize()
        seen.append(y.read(np.uint16, (M, ldy))[:count, :N])
        assert np.array_equal(seen[-1], seen[0][:count]), count
    assert (seen[0] == seen[0][:, :1]).all()           # a row's columns are all alike
    if not swiglu:
        want = (t.astype(np.float32) * scale).astype(np.float16)
        assert np.array_equal(seen[0][:, 0], want.view(np.uint16))
    for b in (w, bx, bs, y):
        b.free()

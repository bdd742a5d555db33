"""Every kernel of the products of 8-bit rows with 4-bit weights, on the GPU: against the definition, bit for bit against
another kernel, in a captured layer and after another call's error.  KERNELS names the kernel that each size takes;
test_w4_launches.py holds them to it."""
import numpy as np
import pytest

import shared_ref as ref
import test_gpu_w4_chain as chain
import w4_ref
from test_gpu_shared import Graph
from test_gpu_w4 import Weights, check, halves

pytestmark = pytest.mark.gpu
rng_of = np.random.default_rng

# (M, K, N, SwiGLU's features): the kernel and its sizes.  Columns end inside a last 16 or a last 8.
KERNELS = [((9, 8224, 195, 96), "small", (1, 2, 8, 2)), ((9, 1056, 163, 96), "small", (1, 2, 8, 1)), ((60, 2080, 1603, 800), "small", (2, 2, 4, 2)),
           ((100, 288, 1003, 512), "small", (2, 2, 4, 1)), ((333, 2080, 1001, 512), "small", (4, 2, 8, 1)),
           ((1000, 288, 1003, 512), "small", (4, 2, 4, 1)), ((1411, 288, 1019, 512), "mid", (4, 1)), ((1411, 2080, 1019, 512), "mid", (4, 2)),
           ((2000, 288, 2043, 1024), "mid", (8, 1)), ((2401, 288, 4090, 2048), "tile", (8, 2)), ((2401, 1056, 4090, 2048), "tile", (8, 4))]
IDS = ["-".join([kind, *map(str, sizes)]) for _, kind, sizes in KERNELS]


def other_rows(M):
    """A count of rows that takes another kernel."""
    return 9 if M > 16 else 700


class Product:
    def __init__(self, ctx, qattn, K, N, swiglu, bf16, image, x, x_scale):
        self.ctx, self.K, self.N, self.bf16, self.dtype = ctx, K, N, bf16, qattn.BF16 if bf16 else qattn.F16
        self.call = ctx.w4_matmul_swiglu if swiglu else ctx.w4_matmul
        self.ldy, self.bytes = -(-N // 8) * 8, image.nbytes
        self.w, self.x, self.s, self.y = ctx.upload(image), ctx.upload(x), ctx.upload(x_scale), ctx.alloc(len(x) * self.ldy * 2)

    def bits(self, M):
        self.y.fill_u16(0x7E55)
        self.call(self.x.ptr, self.s.ptr, M, self.K, self.w.ptr, self.bytes, self.N, self.y.ptr, self.dtype, ldy=self.ldy)
        self.ctx.synchronize()
        y = self.y.read(np.uint16, (M, self.ldy))
        assert (y[:, self.N:] == 0x7E55).all()
        return y[:, :self.N]

    def free(self):
        for b in (self.w, self.x, self.s, self.y):
            b.free()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("sizes", [k[0] for k in KERNELS], ids=IDS)
def test_every_kernel(ctx, qattn, sizes, swiglu, bf16):
    """The definition in 64 bits, and the same bits from another kernel."""
    (M, K), N = sizes[:2], sizes[3 if swiglu else 2]
    print("kernel", M, K, N, swiglu, bf16, flush=True)
    rng = rng_of(M + K + N)
    w = Weights(ctx, qattn, rng, 2 * N if swiglu else N, K)
    rows = max(M, other_rows(M))
    x = rng.integers(-128, 128, (rows, K)).astype(np.int8)
    x_scale = (np.abs(rng.standard_normal(rows)) * (0.5 if swiglu else 0.025) / np.sqrt(K)).astype(np.float32)
    x_scale[1], x_scale[3] = np.nan, 0
    image = qattn.w4_pack(w4_ref.nibbles(w.codes), w.groups, w.scales)
    p = Product(ctx, qattn, K, N, swiglu, bf16, image, x, x_scale)
    whole, other = p.bits(M), p.bits(other_rows(M))
    both = min(M, other_rows(M))
    assert np.array_equal(whole[:both], other[:both])
    want = w.product(x[:M], x_scale[:M])
    got = ref.from_bits(whole, bf16)
    if swiglu:
        g, u = want[:, :N], want[:, N:]
        check(got, w4_ref.swiglu(g, u), w4_ref.swiglu_bound(g, u, bf16), x_scale[:M], bf16)
    else:
        check(got, want, w4_ref.product_bound(want, bf16), x_scale[:M], bf16)
    p.free()
    w.free()


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("sizes", [k[0] for k in KERNELS], ids=IDS)
def test_every_kernel_rounds_alike(ctx, qattn, sizes, swiglu):
    """Values next to a border of fp16: products are rounded to f32, then to 16 bits, in every kernel and at every place
    of a column in it.  Columns of x past the second are zero, their weights are not."""
    (M, K), N = sizes[:2], sizes[3 if swiglu else 2]
    print("rounding", M, K, N, swiglu, flush=True)
    rows = max(M, other_rows(M))
    t, scale = halves(rows)
    x = np.zeros((rows, K), np.int8)
    x[:, 0], x[:, 1] = t, 1
    codes, groups, _ = w4_ref.random_weights(rng_of(K), 2 * N if swiglu else N, K)
    groups[:, 0] = 1 | 8 << 4
    codes[:, 0], codes[:, 1] = 9, 8                    # the first column weighs 1
    if swiglu:
        codes[N:, 0], codes[N:, 1] = 8, 9              # the up product is the row's scale
    image = qattn.w4_pack(w4_ref.nibbles(codes), groups, np.ones(len(codes), np.float32))
    p = Product(ctx, qattn, K, N, swiglu, False, image, x, scale)
    whole, other = p.bits(M), p.bits(other_rows(M))
    both = min(M, other_rows(M))
    assert (whole == whole[:, :1]).all()               # a row's columns are all alike
    assert np.array_equal(whole[:both], other[:both])
    if not swiglu:
        want = (t.astype(np.float32) * scale).astype(np.float16).view(np.uint16)
        assert np.array_equal(whole[:, 0], want[:M])
    p.free()


@pytest.fixture
def wide(monkeypatch):
    """A layer whose projections take the kernels of many rows."""
    for name, value in dict(HIDDEN=1024, QKV=4096, VALUE=2048, INTER=2048).items():
        monkeypatch.setattr(chain, name, value)
    return chain.Layer


@pytest.mark.parametrize("tokens", [1419, 2401])
def test_a_wide_layer_captured(ctx, qattn, wide, tokens):
    """Replays on new inputs, with eager work between them, each compared with the eager layer."""
    layer = wide(ctx, qattn, tokens, False, tokens)
    layer.encode()
    ctx.synchronize()
    layer.verify()
    graph = Graph(ctx.stream, layer.encode)
    for _ in range(3):
        layer.fresh()
        graph.replay()
        ctx.synchronize()
        replayed = layer.results()
        layer.encode()
        ctx.synchronize()
        assert chain.alike(replayed, layer.results())
    layer.verify()
    graph.destroy()
    layer.free()


def test_two_wide_layers_at_once(ctx, qattn, wide):
    layers = [wide(ctx, qattn, 2401, False, 7), wide(ctx, qattn, 1419, True, 8)]
    want = []
    for layer in layers:
        layer.encode()
        ctx.synchronize()
        want.append(layer.results())
    with qattn.Context(0) as other:
        for b in (layers[0].y, layers[1].y, layers[0].ffn, layers[1].ffn):
            b.fill_u16(0x7E55)
        ctx.synchronize()
        for _ in range(5):
            layers[0].encode(ctx.stream)
            layers[1].encode(other.stream)
        ctx.synchronize()
        other.synchronize()
        assert chain.alike(layers[0].results(), want[0]) and chain.alike(layers[1].results(), want[1])
    for layer in layers:
        layer.free()


def test_a_failed_allocation_is_no_later_launch_s_error(ctx, qattn):
    """Device memory that runs out leaves an error in the HIP runtime, per thread; a launch after it is checked for
    its own."""
    layer = chain.Layer(ctx, qattn, 9, False, 1)
    with pytest.raises(qattn.QattnError) as e:
        ctx.alloc(1 << 50)
    assert e.value.code == qattn.ENOMEM
    a, (ptr, size, _, K, N) = layer.q8[0], layer.weights["qkv"]
    calls = {
        "norm": lambda: ctx.rmsnorm_q8(layer.x.ptr, layer.d_gains[0].ptr, a[0].ptr, a[1].ptr, 9, K),
        "rows": lambda: ctx.quantize_q8(layer.x.ptr, a[0].ptr, a[1].ptr, 9, K),
        "product": lambda: ctx.w4_matmul(a[0].ptr, a[1].ptr, 9, K, ptr, size, N, layer.qkv.ptr),
        "gate/up": lambda: ctx.w4_matmul_swiglu(a[0].ptr, a[1].ptr, 9, K, *layer.weights["gate_up"][:2], chain.INTER, layer.ffn.ptr),
    }
    for name, call in calls.items():
        print("after a failed allocation:", name, flush=True)
        with pytest.raises(qattn.QattnError):
            ctx.alloc(1 << 50)
        call()
    ctx.synchronize()
    layer.encode()
    ctx.synchronize()
    layer.verify()
    layer.free()

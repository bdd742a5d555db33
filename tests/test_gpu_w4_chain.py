"""The operators of a forward with 8-bit activations as they are used together: the projections and norms of a layer,
eagerly, captured and replayed, and on two streams at once."""
import numpy as np
import pytest

import shared_ref as ref
import w4_ref
from test_gpu_row_q8 import check_scales, some_rows
from test_gpu_shared import Graph
from test_gpu_w4 import check

pytestmark = pytest.mark.gpu
rng_of = np.random.default_rng
HIDDEN, QKV, VALUE, INTER = 256, 640, 384, 288  # the "attention output" is the last 384 columns of the QKV rows


class Layer:
    """rmsnorm_q8 -> product -> quantize_q8 of some of its columns -> product -> rmsnorm_q8 with the residual's sum ->
    gate/up product and SwiGLU -> quantize_q8 -> product."""

    def __init__(self, ctx, qattn, tokens, bf16, seed):
        self.ctx, self.tokens, self.bf16, self.rng = ctx, tokens, bf16, rng_of(seed)
        self.dtype = qattn.BF16 if bf16 else qattn.F16
        self.bufs, self.weights = [], {}
        for name, N, K in (("qkv", QKV, HIDDEN), ("out", HIDDEN, VALUE), ("gate_up", 2 * INTER, HIDDEN), ("down", HIDDEN, INTER)):
            image = qattn.w4_quantize((self.rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32))
            self.weights[name] = (self.up(image).ptr, image.nbytes, w4_ref.taken_apart(image, K, N), K, N)
        self.gains = [(1 + 0.2 * self.rng.standard_normal(HIDDEN)).astype(np.float32) for _ in range(2)]
        self.d_gains = [self.up(g) for g in self.gains]
        T = tokens
        self.x, self.r, self.sum = (self.alloc(T * HIDDEN * 2) for _ in range(3))
        self.qkv, self.out, self.ffn, self.y = (self.alloc(T * n * 2) for n in (QKV, HIDDEN, INTER, HIDDEN))
        self.q8 = [(self.alloc(T * n), self.alloc(T * 4), n) for n in (HIDDEN, VALUE, HIDDEN, INTER)]
        self.fresh()

    def up(self, a):
        self.bufs.append(self.ctx.upload(np.ascontiguousarray(a)))
        return self.bufs[-1]

    def alloc(self, size):
        self.bufs.append(self.ctx.alloc(size))
        return self.bufs[-1]

    def fresh(self):
        """New inputs, and something else where the results will be."""
        self.inputs = [some_rows(self.rng, self.tokens, HIDDEN, self.bf16) for _ in range(2)]
        for b, bits in zip((self.x, self.r), self.inputs):
            b.write(bits)
        for b in (self.sum, self.qkv, self.out, self.ffn, self.y):
            b.fill_u16(0x7E55)

    def encode(self, stream=None):
        ctx, T, dt = self.ctx, self.tokens, self.dtype

        def product(name, rows, y, call=ctx.w4_matmul):
            ptr, size, _, K, N = self.weights[name]
            call(rows[0].ptr, rows[1].ptr, T, K, ptr, size, INTER if name == "gate_up" else N, y.ptr, dt, stream=stream)

        a, b, c, d = self.q8
        ctx.rmsnorm_q8(self.x.ptr, self.d_gains[0].ptr, a[0].ptr, a[1].ptr, T, HIDDEN, dtype=dt, stream=stream)
        product("qkv", a, self.qkv)
        ctx.quantize_q8(self.qkv.ptr + 2 * (QKV - VALUE), b[0].ptr, b[1].ptr, T, VALUE, dt, QKV, stream=stream)
        product("out", b, self.out)
        ctx.rmsnorm_q8(self.out.ptr, self.d_gains[1].ptr, c[0].ptr, c[1].ptr, T, HIDDEN, self.r.ptr, self.sum.ptr, dtype=dt,
                       stream=stream)
        product("gate_up", c, self.ffn, ctx.w4_matmul_swiglu)
        ctx.quantize_q8(self.ffn.ptr, d[0].ptr, d[1].ptr, T, INTER, dt, stream=stream)
        product("down", d, self.y)

    def results(self):
        T = self.tokens
        tensors = [b.read(np.uint16, (T, n)) for b, n in
                   ((self.sum, HIDDEN), (self.qkv, QKV), (self.out, HIDDEN), (self.ffn, INTER), (self.y, HIDDEN))]
        return tensors + [v for codes, scales, n in self.q8 for v in (codes.read(np.int8, (T, n)), scales.read(np.float32, (T,)))]

    def verify(self):
        """Every stage against its definition in 64 bits, on what the stage before it wrote."""
        total, qkv, out, ffn, y = self.results()[:5]
        q8 = [(c.read(np.int8, (self.tokens, n)), s.read(np.float32, (self.tokens,))) for c, s, n in self.q8]
        bits = lambda b: ref.from_bits(b, self.bf16)  # noqa: E731

        def rows(got, want, width, norm):
            assert np.array_equal(got[0], want[0])
            check_scales(got[1], want[1], width, norm)

        def product(name, given):
            return w4_ref.product(given[0], given[1], *self.weights[name][2])

        rows(q8[0], w4_ref.rmsnorm_q8(self.inputs[0], None, self.gains[0], self.bf16, 1e-6)[:2], HIDDEN, True)
        for name, given, got in (("qkv", q8[0], qkv), ("out", q8[1], out), ("down", q8[3], y)):
            want = product(name, given)
            check(bits(got), want, w4_ref.product_bound(want, self.bf16), given[1], self.bf16)
        rows(q8[1], w4_ref.quantize_q8(np.ascontiguousarray(qkv[:, QKV - VALUE:]), self.bf16), VALUE, False)
        codes, scales, sums = w4_ref.rmsnorm_q8(out, self.inputs[1], self.gains[1], self.bf16, 1e-6)
        rows(q8[2], (codes, scales), HIDDEN, True)
        assert np.array_equal(total, sums)
        g, u = np.split(product("gate_up", q8[2]), 2, axis=1)
        check(bits(ffn), w4_ref.swiglu(g, u), w4_ref.swiglu_bound(g, u, self.bf16), q8[2][1], self.bf16)
        rows(q8[3], w4_ref.quantize_q8(ffn, self.bf16), INTER, False)

    def free(self):
        for b in self.bufs:
            b.free()


def alike(a, b):
    return all(np.array_equal(x.view(np.uint32) if x.dtype == np.float32 else x, y.view(np.uint32) if y.dtype == np.float32 else y)
               for x, y in zip(a, b))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("tokens", [1, 9, 50, 333, 2500])
def test_a_layer(ctx, qattn, tokens, bf16):
    layer = Layer(ctx, qattn, tokens, bf16, tokens)
    layer.encode()
    ctx.synchronize()
    layer.verify()
    layer.free()


@pytest.mark.parametrize("tokens", [3, 400])
def test_a_layer_captured(ctx, qattn, tokens):
    """Replays on new inputs, with eager work between them, each compared with the eager layer."""
    layer = Layer(ctx, qattn, tokens, False, 5)
    layer.encode()
    ctx.synchronize()
    graph = Graph(ctx.stream, layer.encode)
    for _ in range(4):
        layer.fresh()
        graph.replay()
        ctx.synchronize()
        replayed = layer.results()
        layer.verify()
        layer.encode()
        ctx.synchronize()
        assert alike(replayed, layer.results())
    graph.destroy()
    layer.free()


def test_two_layers_at_once(ctx, qattn):
    """Two streams, launches in turn: neither call leaves anything that the other would find."""
    layers = [Layer(ctx, qattn, 700, False, 7), Layer(ctx, qattn, 61, False, 8)]
    want = []
    for layer in layers:
        layer.encode()
        ctx.synchronize()
        layer.verify()
        want.append(layer.results())
    with qattn.Context(0) as other:
        for _ in range(3):
            for b in (layers[0].y, layers[1].y, layers[0].ffn, layers[1].ffn):
                b.fill_u16(0x7E55)
            ctx.synchronize()
            for _ in range(5):
                layers[0].encode(ctx.stream)
                layers[1].encode(other.stream)
            ctx.synchronize()
            other.synchronize()
            assert alike(layers[0].results(), want[0]) and alike(layers[1].results(), want[1])
    for layer in layers:
        layer.free()

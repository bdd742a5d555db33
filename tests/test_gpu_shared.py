"""Attention behind one shared prefix (qattn_shared_run_*) against its definition in 64 bits, on the GPU.

The bound on a row's error, from the roundings the kernel makes (u: half a step of the 16-bit type, D the
head dim, n the keys): a score is off by at most d = scale sum |q k| (D + 2) 2^-24; a weight then by a factor
within exp(2 d), plus its own rounding u (an int8 key's weight times its scale's factor, in f32, is rounded
once), plus f32's exp2 and sums (2^-20 + n 2^-24); fp16 weights below the normal range by at most 2^-25 of the
largest; the result by u.  Codes are exact."""
import ctypes

import numpy as np
import pytest

import shared_ref as ref

pytestmark = pytest.mark.gpu
GARBAGE = 0x7E11  # a NaN in fp16, a large number in bf16


def error_bound(q, keys, vals, keep, scale, bf16, form, out):
    """Per (head, dim) of one query: q [group, dim], keys / vals [n, dim] of one KV head."""
    u, n = (2.0 ** -8 if bf16 else 2.0 ** -11), int(keep.sum())
    k, v = keys[keep], np.abs(vals[keep])
    s = q @ k.T * scale
    d = (np.abs(q) @ np.abs(k).T * scale).max(-1, keepdims=True) * (q.shape[1] + 2) * 2.0 ** -24
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    small = 0.0 if bf16 else n * 2.0 ** -25
    size = p @ v * (np.expm1(2 * d) + u + 2.0 ** -20 + n * 2.0 ** -24) + small * v.max(0)
    return size + ref.half_step(np.abs(out) + size, bf16)


class Case:
    """One batch on the device, and its tensors in 64 bits."""

    def __init__(self, ctx, qattn, prefix, queries, own, heads=16, kv=8, dim=128, page=64, bf16=False, form="16bit",
                 paged=True, mask=0, always=176, window=432, scale=0.0, pad=0, seed=0, spread=1.0, pages=0):
        self.ctx, self.qattn, self.bf16, self.form, self.args = ctx, qattn, bf16, form, (mask, always, window)
        self.prefix, self.queries, self.own = prefix, list(queries), list(own)
        self.heads, self.kv, self.dim, self.page, self.paged = heads, kv, dim, page, paged
        self.scale = scale
        rng = self.rng = np.random.default_rng(seed + 1000 * prefix + sum(queries))
        T, self.pad = sum(queries), pad
        bits = lambda *shape: ref.to_bits(rng.standard_normal(shape) * spread, bf16)  # noqa: E731
        self.q = bits(T, heads * dim + pad)
        need = [-(-prefix // page)] + ([-(-n // page) for n in own] if paged else [])
        pages = pages or max(sum(need), 1) + 3
        order = rng.permutation(pages).astype(np.int32)
        ends = np.cumsum(need)
        self.tables = [order[a:b] for a, b in zip(ends - need, ends)]
        # The pool: garbage everywhere (NaN in 16-bit and e4m3 pools, and NaN scales), then the keys.
        shape = (pages, kv, page, dim)
        stored = np.uint16 if form == "16bit" else np.uint8
        self.pool = [np.full(shape, 0x7FC1 if form == "16bit" else 0x7F, stored) for _ in range(2)]
        self.scales = [np.full(shape[:3], np.nan, np.float32) for _ in range(2)]
        self.shared = [self.fill(w, self.tables[0], prefix, bits) for w in range(2)]
        if paged:
            self.mine = [[self.fill(w, t, n, bits) for w in range(2)] for t, n in zip(self.tables[1:], own)]
            self.rows = [None, None]
        else:
            self.rows = [bits(max(sum(own), 1), kv * dim + pad) for _ in range(2)]
            values = [ref.from_bits(r[:, :kv * dim], bf16).reshape(-1, kv, dim) for r in self.rows]
            starts = np.concatenate([[0], np.cumsum(own)])
            self.mine = [[x[a:b] for x in values] for a, b in zip(starts[:-1], starts[1:])]
        self.upload()

    def fill(self, which, table, n, bits):
        """n new keys through a page table; their values in 64 bits [n, kv, dim]."""
        x = bits(n, self.kv, self.dim)
        at = (np.asarray(table, np.int64)[np.arange(n) // self.page], slice(None), np.arange(n) % self.page)
        if self.form == "16bit":
            self.pool[which][at] = x
            return ref.from_bits(x, self.bf16)
        codes, scale = ref.quantise(ref.from_bits(x, self.bf16), self.form, self.bf16)
        self.pool[which][at], self.scales[which][at] = codes, scale
        return ref.values(codes, scale, self.form)

    def upload(self):
        up = self.ctx.upload
        self.buf = {"q": up(self.q), "k": up(self.pool[0]), "v": up(self.pool[1]), "ks": up(self.scales[0]),
                    "vs": up(self.scales[1]), "o": up(np.full((len(self.q) + 2, self.q.shape[1]), GARBAGE, np.uint16))}
        if not self.paged:
            self.buf.update(rk=up(self.rows[0]), rv=up(self.rows[1]))
        q, b = self.qattn, self.buf
        self.cache = q.make_kv_cache(b["k"].ptr, b["v"].ptr, len(self.pool[0]), self.page, self.kv, self.dim,
                                     q.BF16 if self.bf16 else q.F16,
                                     {"16bit": q.KV_16BIT, "e4m3": q.KV_E4M3, "int8": q.KV_INT8}[self.form],
                                     b["ks"].ptr, b["vs"].ptr)

    def lists(self):
        return dict(cu_q=np.concatenate([[0], np.cumsum(self.queries)]), own_len=self.own, prefix_pages=self.tables[0],
                    prefix_len=self.prefix, own_pages=np.concatenate(self.tables[1:]) if self.paged else None)

    def desc(self):
        q, b, stride = self.qattn, self.buf, self.q.shape[1]
        kv_stride = self.kv * self.dim + self.pad
        return q.make_shared_desc(b["q"].ptr, b["o"].ptr, self.cache, q_heads=self.heads, q_row_stride=stride,
                                  o_row_stride=stride, k=None if self.paged else b["rk"].ptr,
                                  v=None if self.paged else b["rv"].ptr, k_row_stride=kv_stride, v_row_stride=kv_stride,
                                  mask=self.args[0], prefix=self.args[1], window=self.args[2], scale=self.scale,
                                  **self.lists())

    def output(self):
        return self.buf["o"].read(np.uint16, (len(self.q) + 2, self.q.shape[1]))

    def run(self):
        r = self.ctx.shared_run(self.desc())
        r.encode()
        self.ctx.synchronize()
        info = r.info()
        r.destroy()
        return self.check(), info

    def check(self):
        """The output rows against the definition; returns the greatest error over its bound."""
        T, width = len(self.q), self.heads * self.dim
        out = self.output()
        assert (out[T:] == GARBAGE).all() and (out[:, width:] == GARBAGE).all()  # rows behind, columns between
        got = ref.from_bits(out[:T, :width], self.bf16).reshape(T, self.heads, self.dim)
        q = ref.from_bits(self.q[:, :width], self.bf16).reshape(T, self.heads, self.dim)
        mask, always, window = self.args
        scale = self.scale or self.dim ** -0.5
        want = ref.attend(q, self.shared, self.mine, self.queries, mask, always, window, scale)
        worst, t, group = 0.0, 0, self.heads // self.kv
        for m, (k, v) in zip(self.queries, self.mine):
            keys, vals = np.concatenate([self.shared[0], k]), np.concatenate([self.shared[1], v])
            for j in range(m):
                keep = ref.visible(len(keys) - m + j, len(keys), mask, always, window)
                if not keep.any():
                    assert not out[t, :width].any(), t
                else:
                    for g in range(self.kv):
                        h = slice(g * group, (g + 1) * group)
                        bound = error_bound(q[t, h], keys[:, g], vals[:, g], keep, scale, self.bf16, self.form, want[t, h])
                        err = np.abs(got[t, h] - want[t, h])
                        assert np.isfinite(got[t, h]).all(), (t, g)
                        worst = max(worst, float((err / bound).max()))
                t += 1
        assert worst <= 1.0, worst
        return worst

    def free(self):
        for b in self.buf.values():
            b.free()


SMALL = [
    dict(prefix=0, queries=[1], own=[1]),
    dict(prefix=0, queries=[1], own=[0]),
    dict(prefix=0, queries=[3], own=[1]),
    dict(prefix=5, queries=[9], own=[2], paged=False),
    dict(prefix=65, queries=[0, 4, 0], own=[3, 4, 0]),
    dict(prefix=500, queries=[1] * 16, own=list(range(16)), page=16),
    dict(prefix=1000, queries=[1] * 40, own=[37 * i % 301 for i in range(40)]),
    dict(prefix=300, queries=[1] * 3, own=[250, 33, 32], heads=5, kv=5),
    dict(prefix=300, queries=[2, 1, 5, 8, 9, 1], own=[40, 50, 5, 8, 100, 600], page=32),
    dict(prefix=200, queries=[36, 84, 150, 10, 67], own=[36, 84, 150, 10, 67], paged=False),
    dict(prefix=130, queries=[70], own=[90], heads=12, kv=1, pad=8),
    dict(prefix=700, queries=[1, 1], own=[900, 0], heads=28, kv=4, page=128),
    dict(prefix=0, queries=[130, 1, 40], own=[130, 500, 41], paged=False, pad=64),
]


@pytest.mark.parametrize("dim,bf16,form", [(128, False, "16bit"), (128, False, "e4m3"), (128, True, "int8"),
                                           (64, True, "16bit"), (64, True, "e4m3"), (64, False, "int8")])
@pytest.mark.parametrize("case", SMALL, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items())[:60])
def test_shared_attention(ctx, qattn, case, dim, bf16, form):
    print("shared", case, dim, bf16, form, flush=True)
    c = Case(ctx, qattn, dim=dim, bf16=bf16, form=form, **case)
    worst, info = c.run()
    print(f"  error / bound {worst:.3f}  {info.as_dict()}", flush=True)
    c.free()


@pytest.mark.parametrize("form", ["16bit", "e4m3", "int8"])
@pytest.mark.parametrize("always,window", [(176, 432), (0, 33), (100, 1), (64, 0), (0, 0), (10, 200)])
@pytest.mark.parametrize("case", [SMALL[5], SMALL[8], SMALL[9], SMALL[11]], ids=["step", "few", "prompts", "long"])
def test_local_mask(ctx, qattn, case, always, window, form):
    print("local", case, always, window, form, flush=True)
    c = Case(ctx, qattn, form=form, mask=1, always=always, window=window, **case)
    c.run()
    c.free()


@pytest.mark.parametrize("spread,scale", [(6.0, 0.0), (1.0, 1e-3), (4.0, 1.0)])
def test_sharp_and_flat_scores(ctx, qattn, spread, scale):
    """Scores of hundreds (one key takes all, the running reference moves) and near-uniform weights."""
    for case in (SMALL[6], SMALL[9]):
        c = Case(ctx, qattn, spread=spread, scale=scale, **case)
        c.run()
        c.free()
    # ascending scores: every tile exceeds the one before
    c = Case(ctx, qattn, 0, [1, 100], [900, 900], paged=False)
    width = c.kv * c.dim
    ramp = np.concatenate([np.arange(900), np.arange(900)])[:, None] * np.full((1, width), 0.02)
    c.rows[0][:, :width] = ref.to_bits(ramp, False)
    c.q[:, :] = ref.to_bits(np.abs(ref.from_bits(c.q, False)), False)
    c.mine = [[ref.from_bits(c.rows[0][a:a + 900, :width], False).reshape(900, c.kv, c.dim), m[1]]
              for a, m in zip((0, 900), c.mine)]
    c.free()
    c.upload()
    c.run()
    c.free()


@pytest.mark.parametrize("form", ["16bit", "e4m3"])
@pytest.mark.parametrize("mask,always,window", [(0, 0, 0), (1, 8, 40)])
def test_what_a_row_does_not_see_adds_nothing(ctx, qattn, form, mask, always, window):
    """Infinities and NaN in K and V of keys that some rows see and others do not."""
    bf16 = form == "e4m3"
    c = Case(ctx, qattn, 100, [1, 70, 6], [90, 130, 6], bf16=bf16, form=form, mask=mask, always=always, window=window)
    # own key 100 of the long prompt (seen by its later rows), key 3 of the short one, a prefix key (seen
    # under the local mask by no row with a position past the window)
    targets = [(c.tables[2], 1, 100), (c.tables[3], 2, 3)] + ([(c.tables[0], -1, 30)] if mask else [])
    for table, i, key in targets:
        values = c.shared if i < 0 else c.mine[i]
        for which in range(2):
            at = (table[key // c.page], slice(None), key % c.page)
            if form == "16bit":
                c.pool[which][at] = 0x7E01 if which == 0 else 0x7C00  # K NaN, V infinite
                values[which][key] = np.nan if which == 0 else np.inf
            else:
                c.pool[which][at] = ref.NAN_CODE
                values[which][key] = np.nan
    c.free()
    c.upload()
    r = ctx.shared_run(c.desc())
    r.encode()
    ctx.synchronize()
    r.destroy()
    got = ref.from_bits(c.output()[:len(c.q)], bf16).reshape(len(c.q), c.heads, c.dim)
    q = ref.from_bits(c.q, bf16).reshape(got.shape)
    want = ref.attend(q, c.shared, c.mine, c.queries, mask, always, window)
    clean = np.isfinite(want).all((1, 2))
    assert 20 < clean.sum() < len(clean)  # both kinds of rows
    assert np.isnan(got[~clean]).all()
    assert np.abs(got[clean] - want[clean]).max() < 0.05
    c.free()


@pytest.mark.parametrize("form", ["16bit", "e4m3"])
def test_infinite_value_reaches_the_rows_that_see_it(ctx, qattn, form):
    """K finite, V infinite (or NaN) in some dims of a key: those dims of the rows that see it, no others."""
    c = Case(ctx, qattn, 40, [70, 1], [100, 40], form=form)
    for table, i, key in ((c.tables[1], 0, 80), (c.tables[2], 1, 39), (c.tables[2], 1, 7)):
        at = (table[key // c.page], slice(None), key % c.page, slice(3, 90, 29))
        c.pool[1][at] = 0xFC00 if form == "16bit" else ref.NAN_CODE
        c.mine[i][1][key, :, 3:90:29] = -np.inf if form == "16bit" else np.nan
    c.free()
    c.upload()
    r = ctx.shared_run(c.desc())
    r.encode()
    ctx.synchronize()
    r.destroy()
    got = ref.from_bits(c.output()[:71], False).reshape(71, c.heads, c.dim)
    want = ref.attend(ref.from_bits(c.q, False).reshape(got.shape), c.shared, c.mine, c.queries)
    fine = np.isfinite(want)
    assert 0 < (~fine).sum() < fine.size / 2 and fine[:50].all()
    if form == "16bit":
        assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.abs(got[fine] - want[fine]).max() < 0.02
    c.free()


def test_update_steps_and_rebind_layers(ctx, qattn):
    """A run of single-token steps over two layers' caches: the lengths grow, pages are added, the batch
    changes, a refused update leaves the plan."""
    first = Case(ctx, qattn, 200, [1] * 5, [15, 16, 1, 63, 40], page=16, form="e4m3", seed=1, pages=40)
    run = ctx.shared_run(first.desc())
    for own in ([16, 17, 2, 64, 41], [17, 18, 3, 65, 42]):
        for layer in range(2):
            c = Case(ctx, qattn, 200, [1] * 5, own, page=16, form="e4m3", seed=7 + layer, pages=40)
            run.rebind(c.buf["q"].ptr, c.buf["o"].ptr, c.cache)
            run.update(**c.lists())
            run.encode()
            ctx.synchronize()
            c.check()
            bad = dict(c.lists(), prefix_pages=np.full(13, 10 ** 6))
            with pytest.raises(qattn.QattnError):
                run.update(**bad)
            with pytest.raises(qattn.QattnError):
                run.rebind(c.buf["q"].ptr, c.buf["o"].ptr + 2, c.cache)
            run.encode()
            ctx.synchronize()
            c.check()
            c.free()
    # another packing, larger than every one before
    c = Case(ctx, qattn, 900, [30, 1, 200], [90, 700, 260], page=16, form="e4m3")
    with pytest.raises(qattn.QattnError):  # another number of pages
        run.rebind(c.buf["q"].ptr, c.buf["o"].ptr, c.cache)
    run.destroy()
    run = ctx.shared_run(c.desc())
    run.update(**first_step(c))
    run.update(**c.lists())
    run.encode()
    ctx.synchronize()
    c.check()
    run.destroy()
    c.free()
    first.free()


def first_step(c):
    lists = c.lists()
    return dict(lists, cu_q=[0, 1], own_len=[5], own_pages=lists["own_pages"][:1])


def test_same_result_every_time_and_on_another_stream(ctx, qattn):
    c = Case(ctx, qattn, 1500, [1] * 9 + [50], [300] * 9 + [77], form="int8")
    run = ctx.shared_run(c.desc())
    run.encode()
    ctx.synchronize()
    c.check()
    want = c.output()
    with qattn.Context(0) as other:
        for _ in range(3):
            run.encode(other.stream)
            other.synchronize()
            assert np.array_equal(c.output(), want)
        run.update(**c.lists())  # records its fence on the other stream
        run.encode()
        ctx.synchronize()
        assert np.array_equal(c.output(), want)
        run.destroy()
    c.free()


class Graph:
    """What a function enqueues on a stream, captured (the HIP runtime that the library has loaded)."""

    def __init__(self, stream, enqueue):
        self.hip, self.stream = ctypes.CDLL("libamdhip64.so.7"), ctypes.c_void_p(stream)
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self.do("hipStreamBeginCapture", self.stream, 2)  # relaxed
        enqueue(stream)
        self.do("hipStreamEndCapture", self.stream, ctypes.byref(graph))
        self.do("hipGraphInstantiate", ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0))
        self.do("hipGraphDestroy", graph)

    def do(self, name, *args):
        assert getattr(self.hip, name)(*args) == 0, name

    def replay(self):
        self.do("hipGraphLaunch", self.exec, self.stream)

    def destroy(self):
        self.do("hipGraphExecDestroy", self.exec)


def test_captured_launches(ctx, qattn):
    """A graph of a step's launches (rope, cache write, attention, merge), replayed on new inputs and
    compared with the eager step every time."""
    heads, kv, dim, page, n, P = 16, 8, 128, 16, 6, 4000
    rng = np.random.default_rng(3)
    f16 = lambda *shape: rng.standard_normal(shape).astype(np.float16).view(np.uint16)  # noqa: E731
    pages = P // page + n
    pool = [ctx.upload(np.zeros((pages, kv, page, dim), np.uint16)) for _ in range(2)]
    cache = qattn.make_kv_cache(pool[0].ptr, pool[1].ptr, pages, page, kv, dim)
    row = (heads + 2 * kv) * dim
    qkv, q, k, o = ctx.alloc(n * row * 2), ctx.alloc(n * heads * dim * 2), ctx.alloc(n * kv * dim * 2), ctx.alloc(n * heads * dim * 2)
    positions, slots = ctx.upload(np.full(n, P, np.int32)), ctx.upload((np.arange(n) * page + P).astype(np.int64))
    keys, prefix_slots = ctx.upload(f16(P, 2 * kv * dim)), ctx.upload(np.arange(P))
    ctx.kv_write(cache, keys.ptr, keys.ptr + 2 * kv * dim, prefix_slots.ptr, P, 2 * kv * dim, 2 * kv * dim)
    rope = qattn.make_rope_desc(positions.ptr, n, (qkv.ptr, q.ptr, heads), (qkv.ptr + 2 * heads * dim, k.ptr, kv),
                                q_row_stride=row, k_row_stride=row)
    run = ctx.shared_run(qattn.make_shared_desc(q.ptr, o.ptr, cache, np.arange(n + 1), [1] * n,
                                                prefix_pages=np.arange(P // page), prefix_len=P,
                                                own_pages=P // page + np.arange(n)))
    assert run.info().merged_rows > 0  # both launches are in the graph

    def step(stream):
        ctx.rope(rope, stream)
        ctx.kv_write(cache, k.ptr, qkv.ptr + 2 * (heads + kv) * dim, slots.ptr, n, None, row, stream)
        run.encode(stream)

    def outcome(launch):
        o.fill_u16(GARBAGE)
        launch()
        ctx.synchronize()
        return o.read(np.uint16, (n, heads * dim))

    qkv.write(f16(n, row))
    first = outcome(lambda: step(ctx.stream))
    graph = Graph(ctx.stream, step)
    for _ in range(4):
        qkv.write(f16(n, row))
        replayed = outcome(graph.replay)
        assert np.array_equal(replayed, outcome(lambda: step(ctx.stream))) and not np.array_equal(replayed, first)
        assert np.isfinite(replayed.view(np.float16)).all()
    graph.destroy()
    run.destroy()
    for b in pool + [qkv, q, k, o, positions, slots, keys, prefix_slots]:
        b.free()


@pytest.mark.parametrize("form,bound", [("16bit", 2e-3), ("int8", 2e-2), ("e4m3", 8e-2)])
def test_prefix_kept_once_equals_whole_prompts(ctx, qattn, oracle, form, bound):
    """As a service uses them together: the instruction's tokens run once and their keys cached, then each
    request's own tokens behind them, against whole prompts through the framework's own path (QK
    RMSNorm + RoPE and prefill).  16-bit caches differ by roundings; int8 and e4m3 by their codes: half
    a step of 1/127 of a vector's largest value (about 3 sigma), or 2^-4 of each value, averaged over
    the weights."""
    P, lengths = 150, [40, 1, 77, 13]
    rng = np.random.default_rng(5)
    f16 = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
    instruction, requests = f16(P, 4096), [f16(n, 4096) for n in lengths]
    whole = np.concatenate([np.concatenate([instruction, r]) for r in requests])
    cu = np.concatenate([[0], np.cumsum([P + n for n in lengths])]).astype(np.int32)
    up = lambda a: ctx.upload(np.ascontiguousarray(a).view(np.uint16))  # noqa: E731
    bw, T = up(whole), len(whole)
    bq, bk, bo = ctx.alloc(T * 4096), ctx.alloc(T * 2048), ctx.alloc(T * 4096)
    ctx.qk_norm_rope_qkv(bw.ptr, bq.ptr, bk.ptr, cu)
    ctx.prefill(qattn.make_desc(bq.ptr, bk.ptr, bw.ptr, bo.ptr, cu, 0, v_row_stride=4096, v_offset=2048 + 1024))
    want = bo.read(np.uint16, (T, 2048)).view(np.float16).astype(np.float64)
    want = np.concatenate([want[a + P:b] for a, b in zip(cu[:-1], cu[1:])])
    # the instruction once, at positions 0 .. P - 1
    own = np.concatenate(requests)
    n = len(own)
    page, pages = 32, 6
    width = 1024
    codes = [ctx.alloc(pages * page * width * 2) for _ in range(2)]
    scales = [ctx.alloc(pages * page * 8 * 4) for _ in range(2)]
    cache = qattn.make_kv_cache(codes[0].ptr, codes[1].ptr, pages, page,
                                format={"16bit": 0, "e4m3": 1, "int8": 2}[form], k_scale=scales[0].ptr, v_scale=scales[1].ptr)
    table = np.array([4, 1, 5, 0, 2], np.int32)
    slots = ctx.upload((table[np.arange(P) // page] * page + np.arange(P) % page).astype(np.int64))
    bi = up(instruction)
    iq, ik = ctx.alloc(P * 4096), ctx.alloc(P * 2048)
    ctx.qk_norm_rope_qkv(bi.ptr, iq.ptr, ik.ptr, np.array([0, P], np.int32))
    ctx.kv_write(cache, ik.ptr, bi.ptr + 2 * (2048 + 1024), slots.ptr, P, v_row_stride=4096)
    # the requests: normalised and rotated to positions that restart, then P further: rotations add
    br = up(own)
    rq, rk, ro = ctx.alloc(n * 4096), ctx.alloc(n * 2048), ctx.alloc(n * 4096)
    ctx.qk_norm_rope_qkv(br.ptr, rq.ptr, rk.ptr, np.concatenate([[0], np.cumsum(lengths)]))
    shift = ctx.upload(np.full(n, P, np.int32))
    ctx.rope(qattn.make_rope_desc(shift.ptr, n, (rq.ptr, rq.ptr, 16), (rk.ptr, rk.ptr, 8)))
    run = ctx.shared_run(qattn.make_shared_desc(rq.ptr, ro.ptr, cache, np.concatenate([[0], np.cumsum(lengths)]), lengths,
                                                prefix_pages=table, prefix_len=P, k=rk.ptr, v=br.ptr + 2 * (2048 + 1024),
                                                v_row_stride=4096))
    run.encode()
    ctx.synchronize()
    got = ro.read(np.uint16, (n, 2048)).view(np.float16).astype(np.float64)
    err = np.linalg.norm(got - want) / np.linalg.norm(want)
    print(f"{form}: relative difference {err:.2e}", flush=True)
    assert err <= bound
    run.destroy()
    for b in [bw, bq, bk, bo, bi, iq, ik, br, rq, rk, ro, shift, slots] + codes + scales:
        b.free()

"""Attention behind one shared prefix on the GPU: blocks of 256 and 128 rows, with what no row or only some
rows may see in the cache (garbage codes and scales, infinities, NaN), against the definition in 64 bits.
Bounds: as in test_gpu_shared.py."""
import numpy as np
import pytest

import shared_ref as ref
from test_gpu_shared import GARBAGE, Case, error_bound

pytestmark = pytest.mark.gpu
FORMS = [(128, False, "16bit"), (128, False, "e4m3"), (128, True, "int8"), (64, True, "16bit"), (64, True, "e4m3"), (64, False, "int8")]


class Sampled(Case):
    """Many heads fill the chip with 256-row blocks; three KV heads are checked."""

    def sample(self):
        group, self.some = self.heads // self.kv, [0, self.kv // 2, self.kv - 1]
        return np.concatenate([np.arange(g * group, (g + 1) * group) for g in self.some])

    def outputs(self):
        heads, T, width = self.sample(), len(self.q), self.heads * self.dim
        out = self.output()
        assert (out[T:] == GARBAGE).all() and (out[:, width:] == GARBAGE).all()
        got, q = (ref.from_bits(x, self.bf16).reshape(T, self.heads, self.dim)[:, heads] for x in (out[:T, :width], self.q[:, :width]))
        shared, mine = [x[:, self.some] for x in self.shared], [[x[:, self.some] for x in m] for m in self.mine]
        return got, q, shared, mine

    def check(self):
        got, q, shared, mine = self.outputs()
        mask, always, window = self.args
        scale, group = self.dim ** -0.5, self.heads // self.kv
        want = ref.attend(q, shared, mine, self.queries, mask, always, window, scale)
        t = 0
        for m, (k, v) in zip(self.queries, mine):
            keys, vals = np.concatenate([shared[0], k]), np.concatenate([shared[1], v])
            for j in range(m):
                keep = ref.visible(len(keys) - m + j, len(keys), mask, always, window)
                assert np.isfinite(got[t]).all(), t
                for g in range(3):
                    h = slice(g * group, (g + 1) * group)
                    bound = error_bound(q[t, h], keys[:, g], vals[:, g], keep, scale, self.bf16, self.form, want[t, h])
                    assert (np.abs(got[t, h] - want[t, h]) <= bound).all(), (t, g)
                t += 1
        return 0.0


def tall(ctx, qattn, **kw):
    c = Sampled(ctx, qattn, 200, [170, 1, 300, 30], [170, 400, 350, 30], heads=128, kv=32, page=32, **kw)
    kinds = set(qattn.shared_plan(c.desc())[0]["items"][:, 6].tolist())
    assert 0 in kinds or c.args[0], kinds  # short windows leave little to share: 128 rows then
    return c


def blocks(ctx, qattn, **kw):
    """128-row blocks, and single tokens by themselves."""
    c = Case(ctx, qattn, 150, [170, 1, 90, 30], [200, 300, 90, 30], page=16, **kw)
    assert 1 in set(qattn.shared_plan(c.desc())[0]["items"][:, 6].tolist())
    return c


def steps(ctx, qattn, **kw):
    return Case(ctx, qattn, 150, [1] * 20, [1 + 37 * i % 90 for i in range(20)], page=16, **kw)


@pytest.mark.parametrize("dim,bf16,form", FORMS)
@pytest.mark.parametrize("mask,always,window", [(0, 0, 0), (1, 176, 432), (1, 176, 132), (1, 0, 40)])
@pytest.mark.parametrize("paged", [True, False])
def test_tall_blocks(ctx, qattn, dim, bf16, form, mask, always, window, paged):
    c = tall(ctx, qattn, dim=dim, bf16=bf16, form=form, mask=mask, always=always, window=window, paged=paged)
    print("tall", dim, bf16, form, mask, paged, flush=True)
    c.run()
    c.free()


@pytest.mark.parametrize("make", [tall, blocks, steps])
@pytest.mark.parametrize("dim,bf16,form", [f for f in FORMS if f[2] != "16bit"])
@pytest.mark.parametrize("mask,always,window", [(0, 0, 0), (1, 70, 50)])
def test_garbage_in_unused_slots(ctx, qattn, make, dim, bf16, form, mask, always, window):
    """Slots that hold no key may share a tile with ones that do: any codes, and any scales."""
    c = make(ctx, qattn, dim=dim, bf16=bf16, form=form, mask=mask, always=always, window=window)
    rng = np.random.default_rng(2)
    for pool, scales in zip(c.pool, c.scales):
        unused = np.isnan(scales)
        assert unused.any()
        pool[unused] = rng.choice(np.array([0x80, 0x7F, 0xFF, 0x81, 0x00, 0x7E], np.uint8), (int(unused.sum()), c.dim))
        scales[unused] = rng.choice(np.array([np.nan, np.inf, -np.inf, 3e38, -3e38, 0, 1e-38, -1], np.float32), int(unused.sum()))
    c.free()
    c.upload()
    print("garbage", make.__name__, dim, bf16, form, mask, flush=True)
    c.run()
    c.free()


@pytest.mark.parametrize("make", [tall, blocks, steps])
@pytest.mark.parametrize("form", ["16bit", "e4m3", "int8"])
@pytest.mark.parametrize("prefix_key", [False, True])
def test_infinities_and_nan_reach_the_rows_that_see_them(ctx, qattn, make, form, prefix_key):
    """K finite, V infinite or NaN in a key, of an own sequence or of the prefix (seen by every row): an int8
    key's scale is infinite, then its codes of 0 give NaN."""
    c = make(ctx, qattn, form=form)
    i, key = (-1, 5) if prefix_key else (2, 27)
    table, values = (c.tables[0], c.shared) if prefix_key else (c.tables[1 + i], c.mine[i])
    at = (table[key // c.page], slice(None), key % c.page)
    if form == "int8":
        c.pool[1][at][:, ::5] = 0
        c.scales[1][at] = np.inf
        with np.errstate(invalid="ignore"):
            values[1][key] = c.pool[1][at].view(np.int8).astype(np.float64) * np.inf
    else:
        at += (slice(3, 60, 9),)
        c.pool[1][at] = 0x7C00 if form == "16bit" else ref.NAN_CODE
        values[1][key, :, 3:60:9] = np.inf if form == "16bit" else np.nan
    c.free()
    c.upload()
    r = ctx.shared_run(c.desc())
    r.encode()
    ctx.synchronize()
    r.destroy()
    if make is tall:
        got, q, shared, mine = c.outputs()
    else:
        T = len(c.q)
        got, q = (ref.from_bits(x, False).reshape(T, c.heads, c.dim) for x in (c.output()[:T], c.q))
        shared, mine = c.shared, c.mine
    with np.errstate(invalid="ignore"):
        want = ref.attend(q, shared, mine, c.queries)
    fine = np.isfinite(want)
    assert 0 < (~fine).sum() and (prefix_key or fine[:100].all() if make is not steps else True)
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert not fine.any() or np.abs(got[fine] - want[fine]).max() < 0.02
    c.free()


@pytest.mark.parametrize("make", [tall, blocks, steps])
@pytest.mark.parametrize("bf16,form", [(False, "16bit"), (False, "e4m3"), (False, "int8"), (True, "int8")])
def test_values_near_the_type_s_least(ctx, qattn, make, bf16, form):
    """fp16 elements below the normal range, bf16 ones far below 1: V's codes and their scales too."""
    c = make(ctx, qattn, bf16=bf16, form=form, spread=1e-25 if bf16 else 2.0 ** -18)
    c.run()
    c.free()


def test_two_runs_at_once(ctx, qattn):
    """Runs on two streams, in flight together: each has a workspace of its own."""
    a, b = steps(ctx, qattn, form="e4m3"), blocks(ctx, qattn, form="int8", bf16=True)
    with qattn.Context(0) as other:
        runs = [ctx.shared_run(a.desc()), ctx.shared_run(b.desc())]
        streams = [ctx.stream, other.stream]
        for _ in range(20):
            for run, stream in zip(runs, streams):
                run.encode(stream)
        ctx.synchronize()
        other.synchronize()
        a.check()
        b.check()
        # one run after itself on another stream, with an update between
        runs[0].update(**a.lists())
        runs[0].encode(other.stream)
        other.synchronize()
        a.check()
        for run in runs:
            run.destroy()
    a.free()
    b.free()

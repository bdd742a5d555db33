"""Attention behind one shared prefix on the GPU: the edges of scales, infinities and unused slots, against the
definition in 64 bits.  Bounds: as in test_gpu_shared.py."""
import time

import numpy as np
import pytest

import shared_ref as ref
from test_gpu_shared import Case, error_bound
from test_gpu_shared_blocks import FORMS, Sampled, blocks, steps, tall

pytestmark = pytest.mark.gpu


def outputs(c):
    """(outputs, queries, the prefix's K and V, the sequences') of the checked heads in 64 bits."""
    if isinstance(c, Sampled):
        return c.outputs()
    T, width = len(c.q), c.heads * c.dim
    got, q = (ref.from_bits(x[:T, :width], c.bf16).reshape(T, c.heads, c.dim) for x in (c.output(), c.q))
    return got, q, c.shared, c.mine


def launched(ctx, c):
    r = ctx.shared_run(c.desc())
    r.encode()
    ctx.synchronize()
    r.destroy()
    return outputs(c)


def check(c, seen, scale=None):
    """Outputs against the definition: infinities and NaN where it has them, else within the bound.  Returns the
    definition's."""
    got, q, shared, mine = seen
    scale = c.dim ** -0.5 if scale is None else scale
    with np.errstate(invalid="ignore"):
        want = ref.attend(q, shared, mine, c.queries, *c.args, scale)
    group, t = c.heads // c.kv, 0
    for m, (k, v) in zip(c.queries, mine):
        keys, vals = np.concatenate([shared[0], k]), np.concatenate([shared[1], v])
        for j in range(m):
            keep = ref.visible(len(keys) - m + j, len(keys), *c.args)
            assert keep.any(), t
            for g in range(keys.shape[1]):
                h = slice(g * group, (g + 1) * group)
                x, y = got[t, h], want[t, h]
                fine = np.isfinite(y)
                assert np.array_equal(x[~fine], y[~fine], equal_nan=True) and np.isfinite(x[fine]).all(), (t, g, x[~fine], y[~fine])
                finite = np.where(np.isfinite(vals[:, g]), vals[:, g], 0)  # an infinity's dim is not in `fine`
                bound = error_bound(q[t, h], keys[:, g], finite, keep, scale, c.bf16, c.form, np.where(fine, y, 0))
                assert (np.abs(x[fine] - y[fine]) <= bound[fine]).all(), (t, g)
            t += 1
    return want


@pytest.mark.parametrize("make", [tall, blocks, steps])
@pytest.mark.parametrize("dim,bf16,form", FORMS)
@pytest.mark.parametrize("mask,always,window", [(0, 0, 0), (1, 70, 50)])
def test_least_scale_averages(ctx, qattn, make, dim, bf16, form, mask, always, window):
    """The least scale that f32 holds: every seen key weighs the same, a masked one nothing."""
    c = make(ctx, qattn, dim=dim, bf16=bf16, form=form, mask=mask, always=always, window=window, scale=4.9e-46)
    print("least scale", make.__name__, dim, bf16, form, mask, flush=True)
    assert np.isfinite(check(c, launched(ctx, c), 4.9e-46)).all()
    c.free()


@pytest.mark.parametrize("make", [tall, blocks, steps])
@pytest.mark.parametrize("dim,bf16,form", [(128, False, "16bit"), (128, False, "int8"), (64, True, "16bit"), (64, True, "int8")])
@pytest.mark.parametrize("always,window", [(0, 40), (8, 24)])
@pytest.mark.parametrize("key", [100, 45])
def test_an_infinity_among_few_keys_of_a_tile(ctx, qattn, make, dim, bf16, form, always, window, key):
    """Rows whose window covers only one half of a tile see the infinity in it: the half that sees nothing must
    not turn it into NaN."""
    c = make(ctx, qattn, dim=dim, bf16=bf16, form=form, mask=1, always=always, window=window)
    key, i = (key % 64, next(i for i, n in enumerate(c.own) if key % 64 < n <= key % 64 + window)) if make is steps else (key, 0)
    at = (c.tables[1 + i][key // c.page], slice(None), key % c.page)
    c.pool[1][at][:, ::5] = 77 if form == "int8" else 0x7F80 if bf16 else 0x7C00
    if form == "int8":
        c.pool[1][at] |= 1  # no code of 0, which would give NaN
        c.scales[1][at] = np.inf
        c.mine[i][1][key] = c.pool[1][at].view(np.int8) * np.inf
    else:
        c.mine[i][1][key] = ref.from_bits(c.pool[1][at], bf16)
    c.free()
    c.upload()
    print("few keys", make.__name__, dim, bf16, form, always, window, key, flush=True)
    want = check(c, launched(ctx, c))
    assert np.isposinf(want).any() and not np.isnan(want).any() and np.isfinite(want).sum() > want.size // 2
    c.free()


LONG = dict(prefix=8190, queries=[1] * 64, own=[1 + 37 * i % 300 for i in range(64)])  # flat items, and blocks for the prefix
CHUNK = dict(prefix=4999, queries=[200] * 4, own=[203] * 4)


@pytest.mark.parametrize("case", [LONG, CHUNK], ids=["steps", "prompts"])
@pytest.mark.parametrize("bf16,form", [(False, "16bit"), (True, "e4m3"), (False, "int8")])
def test_unused_slots_cost_nothing(ctx, qattn, case, bf16, form):
    """What lies in slots that hold no key (a page's end that nothing has written) changes neither the results nor
    the time: NaN codes and scales against zeros, launches in turn.  The repair that infinities of seen keys
    need takes many times a launch, so half as much again is between the two."""
    c = Case(ctx, qattn, bf16=bf16, form=form, **case)  # its unused slots hold NaN
    clean = Case(ctx, qattn, bf16=bf16, form=form, **case)
    for which in range(2):
        unused = clean.pool[which] == 0x7FC1 if form == "16bit" else np.isnan(clean.scales[which])
        assert unused.any()
        clean.pool[which][unused] = 0
        clean.scales[which][np.isnan(clean.scales[which])] = 1
    clean.free()
    clean.upload()
    runs, least = [ctx.shared_run(x.desc()) for x in (c, clean)], [np.inf, np.inf]
    for _ in range(12):
        for i, run in enumerate(runs):
            ctx.synchronize()
            start = time.perf_counter()
            for _ in range(20):
                run.encode()
            ctx.synchronize()
            least[i] = min(least[i], (time.perf_counter() - start) / 20 * 1e6)
    print(f"unused {len(c.q)} {form}: {least[0]:.1f} us, clean {least[1]:.1f}", flush=True)
    assert np.array_equal(c.output(), clean.output())
    assert least[0] < 1.5 * least[1], least
    for run in runs:
        run.destroy()
    for x in (c, clean):
        x.free()

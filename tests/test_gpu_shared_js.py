"""The operators behind one shared prefix through Node, as a program uses them together: a prefix's keys into
a paged cache, a batch rotated to the positions behind them, attention over both."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import shared_ref as ref
from test_gpu_shared import error_bound

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
@pytest.mark.parametrize("form", ["16bit", "e4m3", "int8"])
def test_node_requests_behind_a_prefix(tmp_path, form):
    prefix, lengths, page = 75, [1, 40, 7], 16
    rng = np.random.default_rng(11)
    pages = rng.permutation(9).tolist()
    T = sum(lengths)
    half = lambda *s: rng.standard_normal(s).astype(np.float16)  # noqa: E731
    kept, qkv = [half(prefix, 8, 128) for _ in range(2)], half(T, 4096)
    for name, a in (("prefix_k", kept[0]), ("prefix_v", kept[1]), ("qkv", qkv)):
        a.tofile(str(tmp_path / f"{name}.bin"))
    (tmp_path / "case.json").write_text(json.dumps(dict(prefix=prefix, lengths=lengths, pageSize=page, pages=pages, format=form)))
    r = subprocess.run(["node", os.path.join(HERE, "js", "shared.gpu.js"), str(tmp_path)], capture_output=True, text=True,
                       timeout=180)
    print(r.stdout, r.stderr[-2000:])
    assert r.returncode == 0, r.stdout + r.stderr
    load = lambda name, *s: np.fromfile(str(tmp_path / f"{name}.bin"), np.float16).reshape(s).astype(np.float64)  # noqa: E731
    # rotation: f32 arithmetic, one rounding to the type
    q, k, out = load("q", T, 16, 128), load("k", T, 8, 128), load("o", T, 16, 128)
    positions = np.concatenate([prefix + np.arange(n) for n in lengths])
    f = ref.rope_frequencies(128, 1e6)
    for got, x in ((q, qkv[:, :2048].reshape(T, 16, 128)), (k, qkv[:, 2048:2048 + 1024].reshape(T, 8, 128))):
        x = x.astype(np.float64)
        want = ref.rope(x, positions, f, "half")
        size = np.abs(x[..., :64]) + np.abs(x[..., 64:])
        assert (np.abs(got - want) <= ref.half_step(want, False) + np.concatenate([size, size], -1) * 2.0 ** -20).all()
    # the cache gives back the rows as they are, or within its codes' rounding
    back = [load("back_k", prefix, 8, 128), load("back_v", prefix, 8, 128)]
    for a, b in zip(kept, back):
        a = a.astype(np.float64)
        amax = np.abs(a).max(-1, keepdims=True)
        if form == "16bit":
            assert np.array_equal(a, b)
        elif form == "e4m3":  # half a step of a normal code, or of the subnormal ones below amax 2^-14
            assert (np.abs(a - b) <= np.maximum(np.abs(a) * 2.0 ** -4, amax * 2.0 ** -17)).all()
        else:  # half a step, the scale's and the value's roundings
            assert (np.abs(a - b) <= amax / 127 / 2 * (1 + 2.0 ** -10) + ref.half_step(a, False)).all()
    # attention over what the kernels themselves wrote
    own_v = qkv[:, 2048 + 1024:].reshape(T, 8, 128).astype(np.float64)
    scale, at = 128 ** -0.5, 0
    for n in lengths:
        rows = slice(at, at + n)
        keys, vals = (np.concatenate([b, x[rows]]) for b, x in zip(back, (k, own_v)))
        for i in range(n):
            keep = np.arange(prefix + n) <= prefix + i
            for h in range(8):
                qh = q[at + i, 2 * h:2 * h + 2]
                p = qh @ keys[keep, h].T * scale
                p = np.exp(p - p.max(-1, keepdims=True))
                want = p / p.sum(-1, keepdims=True) @ vals[keep, h]
                bound = error_bound(qh, keys[:, h], vals[:, h], keep, scale, False, form, want)
                assert (np.abs(out[at + i, 2 * h:2 * h + 2] - want) <= bound).all(), (at, i, h)
        at += n

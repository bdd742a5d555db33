"""A forward's operators with 8-bit activations through Node: an FFN from its norm to its result."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import shared_ref as ref
import w4_ref
from test_gpu_row_q8 import check_scales, some_rows
from test_gpu_w4 import check

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
@pytest.mark.parametrize("bf16", [False, True])
def test_node_ffn(tmp_path, qattn, bf16):
    tokens, width, features, n = 37, 256, 96, 77
    rng = np.random.default_rng(2)
    x, r = some_rows(rng, tokens, width, bf16), some_rows(rng, tokens, width, bf16)
    gains = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32)
    weights = {"gate_up": (2 * features, width), "down": (n, features)}
    taken = {}
    for name, (N, K) in weights.items():
        w = (rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32)
        w.tofile(str(tmp_path / f"{name}.bin"))
        taken[name] = w4_ref.taken_apart(qattn.w4_quantize(w), K, N)
    for name, a in (("x", x), ("r", r), ("gains", gains)):
        a.tofile(str(tmp_path / f"{name}.bin"))
    (tmp_path / "case.json").write_text(json.dumps(dict(tokens=tokens, width=width, features=features, n=n,
                                                        dtype="bf16" if bf16 else "f16")))
    out = subprocess.run(["node", os.path.join(HERE, "js", "w4.gpu.js"), str(tmp_path)], capture_output=True, text=True, timeout=180)
    print(out.stdout, out.stderr[-2000:])
    assert out.returncode == 0, out.stdout + out.stderr
    load = lambda name, dtype, *s: np.fromfile(str(tmp_path / f"{name}.bin"), dtype).reshape(s)  # noqa: E731
    codes, scales = load("codes", np.int8, tokens, width), load("scales", np.float32, tokens)
    want = w4_ref.rmsnorm_q8(x, r, gains, bf16, 1e-6)
    assert np.array_equal(codes, want[0]) and np.array_equal(load("sum", np.uint16, tokens, width), want[2])
    check_scales(scales, want[1], width, True)
    g, u = np.split(w4_ref.product(codes, scales, *taken["gate_up"]), 2, axis=1)
    ffn = load("ffn", np.uint16, tokens, features)
    check(ref.from_bits(ffn, bf16), w4_ref.swiglu(g, u), w4_ref.swiglu_bound(g, u, bf16), scales, bf16)
    codes, scales = load("inner_codes", np.int8, tokens, features), load("inner_scales", np.float32, tokens)
    want = w4_ref.quantize_q8(ffn, bf16)
    assert np.array_equal(codes, want[0])
    check_scales(scales, want[1], features, False)
    y = load("y", np.uint16, tokens, 80)
    want = w4_ref.product(codes, scales, *taken["down"])
    check(ref.from_bits(y[:, :n], bf16), want, w4_ref.product_bound(want, bf16), scales, bf16)
    assert (y[:, n:] == 0).all()

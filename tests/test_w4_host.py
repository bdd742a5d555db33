"""The operators of a forward with 8-bit activations on the CPU: what their entry points refuse, before any launch,
and what they launch.  The library runs over a stand-in for the HIP runtime (fake_hip.cc, preloaded into a child
process)."""
import json
import os
import shutil
import subprocess
import sys

import pytest

from test_host_launches import HERE, ROCM, Launches
from test_shared_host import attempt

X, R, S, W, C, F, Y = (1 << 40) * 1, (1 << 40) * 2, (1 << 40) * 3, (1 << 40) * 4, (1 << 40) * 5, (1 << 40) * 6, (1 << 40) * 7


def row_refusals():
    h = Launches()
    L, q = h.qattn.lib(), h.qattn

    def quantize(x=X, xs=64, codes=C, cs=64, scales=F, rows=5, width=64, dtype=0, ctx=h.ctx.handle):
        return attempt(h, lambda: q._check(L.qattn_quantize_q8(ctx, x, xs, codes, cs, scales, rows, width, dtype, None)))

    def norm(x=X, xs=64, r=R, rs=64, s=S, ss=64, w=W, codes=C, cs=64, scales=F, rows=5, width=64, dtype=0, eps=1e-6,
             ctx=h.ctx.handle):
        return attempt(h, lambda: q._check(L.qattn_rmsnorm_q8(ctx, x, xs, r, rs, s, ss, w, codes, cs, scales, rows, width,
                                                              dtype, eps, None)))

    both = [dict(x=None), dict(codes=None), dict(scales=None), dict(x=X + 8), dict(codes=C + 4), dict(scales=F + 2),
            dict(xs=56), dict(xs=68), dict(cs=56), dict(cs=66), dict(xs=(1 << 22) + 8), dict(cs=(1 << 22) + 8),
            dict(width=0), dict(width=4), dict(width=60), dict(width=32776, xs=32776, cs=32776), dict(rows=-1),
            dict(rows=1 << 24), dict(dtype=2), dict(dtype=-1), dict(ctx=None), dict(codes=X), dict(codes=X + 632),
            dict(scales=X + 4), dict(scales=C + 316)]
    alone = [dict(w=None), dict(w=W + 4), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=1e40),
             dict(r=None), dict(s=None), dict(r=R + 2), dict(s=S + 2), dict(rs=56), dict(ss=60), dict(codes=S + 64),
             dict(codes=W), dict(scales=R), dict(s=X + 16), dict(s=X, ss=72), dict(s=R, ss=128, rs=64), dict(s=C)]
    return {"fine": [quantize(), quantize(dtype=1), quantize(rows=0), quantize(codes=X + 640), norm(), norm(dtype=1),
                     norm(r=None, s=None), norm(s=X), norm(s=R), norm(rows=0), norm(eps=0.0),
                     norm(width=32768, xs=32768, rs=32768, ss=32768, cs=32768)],
            "bad": [["quantize " + str(c), *quantize(**c)] for c in both] + [["norm " + str(c), *norm(**c)] for c in both + alone]}


def product_refusals():
    h = Launches()
    L, q = h.qattn.lib(), h.qattn
    need = L.qattn_w4_bytes(64, 96)

    def product(x=X, ldx=64, s=S, M=5, K=64, w=W, w_bytes=need, N=96, y=Y, ldy=96, dtype=0, ctx=h.ctx.handle, swiglu=False):
        call = L.qattn_w4_matmul_swiglu if swiglu else L.qattn_w4_matmul
        return attempt(h, lambda: q._check(call(ctx, x, ldx, s, M, K, w, w_bytes, N, y, ldy, dtype, None)))

    both = [dict(x=None), dict(s=None), dict(w=None), dict(y=None), dict(x=X + 8), dict(s=S + 2), dict(w=W + 8), dict(y=Y + 8),
            dict(ldx=48), dict(ldx=72), dict(ldx=(1 << 22) + 16), dict(M=-1), dict(M=1 << 24), dict(K=0), dict(K=48),
            dict(K=65568, ldx=65568, w_bytes=1 << 40), dict(w_bytes=100), dict(dtype=2), dict(ctx=None), dict(y=X + 16),
            dict(y=W), dict(y=S - 16), dict(ldy=(1 << 22) + 8)]
    alone = [dict(N=0), dict(N=-4), dict(N=(1 << 22) + 1, w_bytes=1 << 40), dict(ldy=88), dict(ldy=100),
             dict(M=1 << 20, N=4096, ldy=4096, w_bytes=1 << 40)]
    gate = [dict(N=0), dict(N=16), dict(N=40), dict(N=-32), dict(N=(1 << 21) + 32, w_bytes=1 << 40, ldy=1 << 22), dict(N=64, w_bytes=1 << 30, ldy=56)]
    swiglu = dict(N=32, ldy=32, w_bytes=L.qattn_w4_bytes(64, 64), swiglu=True)
    return {"fine": [product(), product(dtype=1), product(M=0), product(N=1, ldy=8), product(**swiglu), product(**dict(swiglu, M=0)),
                     product(y=X + 5 * 64)],
            "bad": [[str(c), *product(**c)] for c in both + alone] + [["swiglu " + str(c), *product(**{**swiglu, **c})] for c in both + gate]}


def largest_launches():
    """[what, workgroups, threads] of the first dimension of the largest calls there are."""
    h, out = Launches(), []
    now = [""]
    h.on = lambda name, grid, block, args: out.append([now[0], grid, block])
    most = (1 << 24) - 1
    for width in (8, 72, 136, 264, 520, 1032, 2056, 4104, 8200, 16384):
        now[0] = f"rows of {width}"
        h.ctx.quantize_q8(X, C, F, most, width)
        h.ctx.rmsnorm_q8(X, W, C, F, most, width, R, S)
    for M, K, N in ((1, 32, 1 << 22), (16, 65536, 1 << 22), (32, 2048, 1 << 22), (most, 32, 1), (most, 32, 112), (200, 1024, 1 << 22),
                    (480, 1024, 1 << 22), (most, 4096, 100), (1 << 19, 1024, 4080)):
        now[0] = f"{M} x {K} -> {N}"
        h.ctx.w4_matmul(X, S, M, K, W, 1 << 40, N, Y, ldy=-(-N // 8) * 8)
        if N % 64 == 0:
            h.ctx.w4_matmul_swiglu(X, S, M, K, W, 1 << 40, N // 2, Y)
    return out


CASES = {f.__name__: f for f in (row_refusals, product_refusals, largest_launches)}


@pytest.fixture(scope="module")
def w4_child(tmp_path_factory):
    compiler = shutil.which("g++")
    if not compiler or not os.path.isdir(os.path.join(ROCM, "include", "hip")):
        pytest.skip("no g++ or HIP headers")
    lib = str(tmp_path_factory.mktemp("fake") / "libfake_hip.so")
    subprocess.run([compiler, "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-I" + os.path.join(ROCM, "include"), "-o", lib,
                    os.path.join(HERE, "fake_hip.cc")], check=True)

    def run(case):
        preload = " ".join(v for v in (os.environ.get("LD_PRELOAD"), lib) if v)
        out = subprocess.run([sys.executable, os.path.abspath(__file__), case], check=True, capture_output=True, text=True,
                             env=dict(os.environ, LD_PRELOAD=preload, FAKE_HIP=lib), timeout=120)
        return json.loads(out.stdout)

    return run


def test_the_largest_launches_fit_a_grid(w4_child):
    launches = w4_child("largest_launches")
    assert len(launches) > 30
    for what, grid, block in launches:
        assert 0 < grid and grid * block < 1 << 32 and block <= 1024, what


@pytest.mark.parametrize("case", ["row_refusals", "product_refusals"])
def test_refusals_on_the_host(w4_child, case):
    got = w4_child(case)
    for i, (code, message, launches) in enumerate(got["fine"]):
        assert code == 0 and len(launches) <= 1, (i, message)
    assert any(f[2] for f in got["fine"]) and any(not f[2] for f in got["fine"])  # no rows: no launch
    for name, code, message, launches in got["bad"]:
        assert code == -1 and not launches and len(message) > 20, (name, code, message)


if __name__ == "__main__":
    print(json.dumps(CASES[sys.argv[1]]()))

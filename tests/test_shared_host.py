"""The operators behind one shared prefix on the CPU: what their entry points refuse, before any launch.
The library runs over a stand-in for the HIP runtime (fake_hip.cc, preloaded into a child process)."""
import json
import os
import shutil
import subprocess
import sys

import pytest

from test_host_launches import HERE, ROCM, Launches

X, Y, Z, P = 1 << 20, 1 << 30, 1 << 31, 1 << 32  # stand-in device addresses


def attempt(h, call):
    """[error code, message, launches] of one call."""
    names = []
    h.on = lambda name, *rest: names.append(name)
    try:
        call()
    except h.qattn.QattnError as e:
        return [e.code, str(e), names]
    return [0, "", names]


def rope_refusals():
    h = Launches()
    q = h.qattn

    def desc(part=None, **changes):
        d = q.make_rope_desc(P, 5, (X, Y, 4), (X, Z, 2))
        for name, value in changes.items():
            setattr(getattr(d, part) if part else d, name, value)
        return attempt(h, lambda: h.ctx.rope(d))

    out = {"fine": desc(), "no tokens": desc(tokens=0), "k alone is none": desc("k", heads=0),
           "odd address": desc("q", x=X + 2), "null": attempt(h, lambda: q._check(q.lib().qattn_rope(h.ctx.handle, None, None)))}
    bad = [("", dict(dtype=2)), ("", dict(head_dim=514)), ("", dict(head_dim=64)), ("", dict(rotary_dim=3)),
           ("", dict(rotary_dim=0)), ("", dict(rotary_dim=130)), ("", dict(layout=2)), ("", dict(scaling=3)),
           ("", dict(theta=0.0)), ("", dict(theta=float("nan"))), ("", dict(theta=float("inf"))),
           ("", dict(theta=5e-324)), ("", dict(scaling=1, factor=1e-320)), ("", dict(magnitude=float("inf"))), ("", dict(scaling=1, factor=0.0)), ("", dict(scaling=2, factor=float("nan"))),
           ("", dict(scaling=2, factor=4.0, beta_slow=64.0)), ("", dict(scaling=2, factor=4.0, original_context=0.0)),
           ("", dict(scaling=2, factor=4.0, theta=1.0)), ("", dict(tokens=-1)), ("", dict(tokens=1 << 24)),
           ("", dict(positions=None)), ("", dict(positions=P + 2)), ("q", dict(heads=0)), ("k", dict(heads=-1)),
           ("q", dict(heads=5000)), ("q", dict(x=None)), ("k", dict(out=None)), ("q", dict(x=X + 1)),
           ("q", dict(x_row_stride=511)), ("k", dict(out_row_stride=255)), ("k", dict(out=X, out_row_stride=512))]
    out["bad"] = [[str((p, c)), *desc(p, **c)] for p, c in bad if c != dict(head_dim=64)]
    out["head below rotary"] = desc(head_dim=64)
    return out


def kv_refusals():
    h = Launches()
    q = h.qattn

    def write(k=X, v=X, slots=P, tokens=5, ks=None, vs=None, read=False, **changes):
        c = q.make_kv_cache(X, Y, 4, 64, format=q.KV_E4M3, k_scale=Z, v_scale=P)
        for name, value in changes.items():
            setattr(c, name, value)
        if read:
            return attempt(h, lambda: h.ctx.kv_read(c, slots, tokens, k, v, ks, vs))
        return attempt(h, lambda: h.ctx.kv_write(c, k, v, slots, tokens, ks, vs))

    null = attempt(h, lambda: q._check(q.lib().qattn_kv_write(h.ctx.handle, None, X, 1024, X, 1024, P, 4, None)))
    fine = [write(), write(read=True), write(tokens=0, k=None), write(format=q.KV_16BIT, k_scale=None, v_scale=None),
            write(kv_heads=1, head_dim=64, page_size=16)]
    bad = [dict(dtype=7), dict(head_dim=96), dict(kv_heads=0), dict(kv_heads=257), dict(format=3), dict(page_size=48),
           dict(page_size=8), dict(page_size=8192), dict(pages=0), dict(k=None), dict(v=X + 4), dict(slots=None),
           dict(slots=P + 4), dict(tokens=-1), dict(tokens=1 << 24), dict(ks=1016), dict(vs=1028),
           dict(k_scale=None), dict(v_scale=Z + 4), dict(tokens=(1 << 24) - 1, kv_heads=128, ks=1 << 20, vs=1 << 20)]
    return {"fine": fine, "null": null,
            "bad": [[str(c), *write(**c)] for c in bad] + [[str(c), *write(read=True, **c)] for c in bad]}


CASES = {f.__name__: f for f in (rope_refusals, kv_refusals)}


@pytest.fixture(scope="module")
def shared_child(tmp_path_factory):
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


def test_rope_refuses_on_the_host(shared_child):
    got = shared_child("rope_refusals")
    for name in ("fine", "k alone is none", "odd address"):
        code, message, launches = got[name]
        assert code == 0 and len(launches) == 1, (name, message)
    assert "Lb1EEE" in got["fine"][2][0] and "Lb0EEE" in got["odd address"][2][0]  # wide and narrow accesses
    assert got["no tokens"][0] == 0 and not got["no tokens"][2]
    for name, code, message, launches in got["bad"] + [["null", *got["null"]], ["head", *got["head below rotary"]]]:
        assert code == -1 and not launches and len(message) > 20, name


def test_cache_refuses_on_the_host(shared_child):
    got = shared_child("kv_refusals")
    assert [f[0] for f in got["fine"]] == [0] * 5 and [len(f[2]) for f in got["fine"]] == [1, 1, 0, 1, 1]
    for name, code, message, launches in got["bad"] + [["null", *got["null"]]]:
        assert code == -1 and not launches and len(message) > 20, name


if __name__ == "__main__":
    print(json.dumps(CASES[sys.argv[1]]()))

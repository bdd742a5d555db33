"""The Node classes of the operators behind one shared prefix, on the CPU (tests/js/shared.test.js)."""
import os
import shutil
import subprocess

import pytest

from test_host_launches import HERE, ROCM


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
def test_node_extents_and_lifetimes(tmp_path):
    if not shutil.which("g++") or not os.path.isdir(os.path.join(ROCM, "include", "hip")):
        pytest.skip("no g++ or HIP headers")
    lib = str(tmp_path / "libfake_hip.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-I" + os.path.join(ROCM, "include"), "-o", lib,
                    os.path.join(HERE, "fake_hip.cc")], check=True)
    preload = " ".join(v for v in (os.environ.get("LD_PRELOAD"), lib) if v)
    r = subprocess.run(["node", os.path.join(HERE, "js", "shared.test.js")], capture_output=True, text=True, timeout=120,
                       env=dict(os.environ, LD_PRELOAD=preload))
    print(r.stdout, r.stderr[-2000:])
    assert r.returncode == 0, r.stdout + r.stderr

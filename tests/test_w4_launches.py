"""What the products of 8-bit rows with 4-bit weights launch, on the CPU: the library runs over a stand-in for the HIP
runtime (fake_hip.cc, preloaded into a child process), whose launches only call a hook here."""
import ctypes
import json
import os
import re
import shutil
import subprocess
import sys

import pytest

from test_host_launches import HERE, ROCM, Launches

X, S, W, Y = (1 << 40) * 1, (1 << 40) * 2, (1 << 40) * 3, (1 << 40) * 4


def launch(h, M, K, N, swiglu, bf16=False):
    call = h.ctx.w4_matmul_swiglu if swiglu else h.ctx.w4_matmul
    call(X, S, M, K, W, 1 << 40, N, Y, dtype=h.qattn.BF16 if bf16 else h.qattn.F16, ldy=-(-N // 8) * 8)


STORES = [(1500, 1024, 4096, False), (2400, 1024, 4096, False), (2900, 1024, 4096, False), (3200, 1024, 4096, False), (8000, 1024, 4096, False),
          (20000, 1024, 4096, False), (2401, 1056, 2048, True), (20000, 1024, 2816, True), (8000, 2048, 1024, False)]


def stores():
    """[(M, K, N, swiglu, whether the tiles of many rows store past the L2s)]"""
    h, out = Launches(), []
    now = []

    def on(name, grid, block, args):
        assert "w4_tile_kernel" in name, (now, name)
        out.append([*now, h.word(args, 4)])  # product, tiles_n, tiles_total, per_xcd, far
    h.on = on
    for now in STORES:
        launch(h, *now)
    return out


def kernels():
    """The products' kernels that the library holds, and those that the sizes of test_gpu_w4_kernels.py take, with the
    kernel that each is compared with: [[all], [[size's index, swiglu, bf16, kernel, other]]]."""
    import test_gpu_w4_kernels as gpu
    h, held, out, seen = Launches(), [], [], []
    each = ctypes.CFUNCTYPE(None, ctypes.c_char_p)(lambda name: held.append(name.decode()))
    h.fake.fake_hip_kernels(each)
    h.on = lambda name, *rest: seen.append(name)
    for i, ((M, K, N, features), *_) in enumerate(gpu.KERNELS):
        for swiglu in (False, True):
            for bf16 in (False, True):
                for rows in (M, gpu.other_rows(M)):
                    launch(h, rows, K, features if swiglu else N, swiglu, bf16)
                out.append([i, swiglu, bf16, *seen[-2:]])
    return [[k for k in held if re.search(r"w4_(small|mid|tile)_kernel", k)], out]


CASES = {f.__name__: f for f in (stores, kernels)}


@pytest.fixture(scope="module")
def child(tmp_path_factory):
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


def test_large_results_stay_where_their_reader_finds_them(child):
    """A product's result of more than 24 MiB is stored plainly: past the L2s the product itself gains less than the call
    that reads the result loses.  SwiGLU's results, where both are alike, go past them."""
    seen = child("stores")
    assert len(seen) == len(STORES)
    for M, K, N, swiglu, far in seen:
        assert far == (swiglu or 2 * M * N <= 24 << 20), (M, K, N, swiglu)
    assert {far for *_, far in seen} == {0, 1}


def test_every_kernel_is_taken_by_the_size_that_names_it(child):
    """The library holds no kernel of the products that nothing launches, and the GPU tests compare each with the
    definition and with another kernel's bits."""
    import test_gpu_w4_kernels as gpu
    held, taken = child("kernels")
    assert len(held) == 4 * len(gpu.KERNELS) and {k for *_, k, _ in taken} == set(held)
    for i, swiglu, bf16, kernel, other in taken:
        _, kind, sizes = gpu.KERNELS[i]
        template = f"w4_{kind}_kernelILb{int(bf16)}ELb{int(swiglu)}E" + "".join(f"Li{n}E" for n in sizes) + "E"
        assert template in kernel and other != kernel, (kernel, template, other)


if __name__ == "__main__":
    print(json.dumps(CASES[sys.argv[1]]()))

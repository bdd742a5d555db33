"""The hand-counted waits of the tiled kernels for 8-bit rows and 4-bit weights, followed through the gfx950 assembly
on the CPU, as test_q4_waits.py does for the Q4_0 kernels: by barrier b every load of the b-th X tile must have
landed on the strength of the explicit waits alone."""
import os
import re
import subprocess

import pytest

from test_q4_waits import HIPCC, PASSES, ROOT

SOURCE = os.path.join(ROOT, "qwen3-embedding-webgpu-prepacked_amd", "csrc", "w4_matmul.hip")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = str(tmp_path_factory.mktemp("asm") / "w4.s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", "-o", out, SOURCE], check=True, capture_output=True)
    found, name = {}, None
    for line in open(out):
        start = re.match(r"(_ZN5qattn\w*w4_(?:tile|mid|small)_kernel\w+):", line)
        if start:
            name = start.group(1)
            found[name] = []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name:
            found[name].append(line.split(";")[0].strip() if "#ASM" not in line else line.strip())
    return found


def events(lines):
    """"load", "dma" and explicit ("wait", V) events of the prologue and of the main loop: of the backward branches over
    LDS-DMA loads, the one whose target comes last (others leave blocks that the compiler has moved out of line)."""
    flat, labels, loops, asm = [], {}, [], False
    for line in lines:
        if "#ASMSTART" in line or "#ASMEND" in line:
            asm = "#ASMSTART" in line
            continue
        label = re.match(r"(\.LBB\w+):", line)
        if label:
            labels[label.group(1)] = len(flat)
        elif re.match(r"(buffer|global|flat|scratch)_", line):
            flat.append(("dma",) if line.endswith(" lds") else ("load",))
        elif asm and "vmcnt(" in line:
            flat.append(("wait", int(re.search(r"vmcnt\((\d+)\)", line).group(1))))
        branch = re.match(r"s_c?branch\w*\s+(\.LBB\w+)", line)
        if branch and branch.group(1) in labels and ("dma",) in flat[labels[branch.group(1)]:]:
            loops.append((labels[branch.group(1)], len(flat)))
    first, last = max(loops)
    return flat[:first], flat[first:last]


def test_every_published_x_tile_has_landed(kernels):
    assert [sum("w4_" + kind in name for name in kernels) for kind in ("tile", "mid", "small")] == [8, 12, 24]
    for name, lines in kernels.items():
        prologue, loop = events(lines)
        sizes = [int(v) for v in re.findall(r"Li(\d+)E", name)]
        # LDS-DMA loads of an X tile, per wavefront, and the waits ahead of the loop and in it: the first kernel reads X
        # tile 0 before its loop, the others in it; a wavefront of the last waits for its own X alone.
        if "w4_tile" in name:
            group, ahead, waits = sizes[0] // sizes[1], 1, 4
        elif "w4_mid" in name:
            group, ahead, waits = sizes[0] // 2, 0, 4
        else:
            group, ahead, waits = 2 * sizes[0], 0, sizes[3]
        assert sum(e[0] == "wait" for e in prologue) == ahead and sum(e[0] == "wait" for e in loop) == waits, name
        issued, dma, barrier = 0, [], 0  # dma: issue numbers of the LDS-DMA loads
        for event in prologue + PASSES * loop:
            if event[0] == "wait":
                newer = issued - 1 - dma[group * (barrier + 1) - 1]
                assert newer >= event[1], (
                    f"{name}: barrier {barrier} waits with vmcnt({event[1]}), but only {newer} operations are newer "
                    f"than the X tile it publishes")
                barrier += 1
            else:
                if event[0] == "dma":
                    dma.append(issued)
                issued += 1


def test_nothing_spills(kernels):
    """Scratch accesses would count among the loads in flight, and cost more than they hide."""
    for name, lines in kernels.items():
        assert not any(re.match(r"scratch_", line) for line in lines), name

"""Code-generation checks of the dense-layer kernels that need no GPU (hipcc cross-compiles)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
needs_hipcc = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")

# One product kernel of every tile, so that this takes seconds; all types and layouts share the code.
SOURCE = """
#include "kernels/linear_tile.h"
namespace dtf {
#define KERNEL(KIND, V) template __global__ void linear_tile_kernel<KIND, LinLoopOf<KIND, true, false, V>::type, kLinTiles[V].tm, kLinTiles[V].tn, \\
    kLinTiles[V].wgm, kLinTiles[V].wgn>(LinTileArgs);
KERNEL(MM_BF16, LIN_REGS) KERNEL(MM_BF16, LIN_64) KERNEL(MM_BF16, LIN_128) KERNEL(MM_BF16, LIN_256) KERNEL(MM_BF16, LIN_32) KERNEL(MM_F32, LIN_64)
}
"""


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Kernel name -> lines of its LLVM IR."""
    d = tmp_path_factory.mktemp("dense")
    src = d / "k.hip"
    src.write_text(SOURCE)
    out = d / "k.ll"
    r = subprocess.run([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-fno-fast-math", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                        "-I", os.path.join(ROOT, "csrc"), "--cuda-device-only", "-S", "-emit-llvm", "-o", str(out), str(src)],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    found, name = {}, None
    for line in out.read_text().splitlines():
        m = re.match(r"define .*amdgpu_kernel void @(\w+)\(", line)
        if m:
            name = m.group(1)
            found[name] = []
        elif line == "}":
            name = None
        elif name:
            found[name].append(line)
    assert len(found) == 6
    return found


@needs_hipcc
def test_lanes_that_exchange_sums_through_lds_are_kept_in_step(kernels):
    """The epilogue stores a lane's sums into LDS and reads other lanes': between stores and reads, and between reads and the next stores, the
    wave has to come together, or lanes that have nothing to write to the output may run ahead. Only the epilogue stores <4 x float> in LDS
    (fp32 fragments are read as such, in front of a barrier)."""
    for name, lines in kernels.items():
        events = ""
        for line in lines:
            if re.search(r"store <4 x float> .*addrspace\(3\)", line):
                events += "S"
            elif re.search(r"load <4 x float>, .*addrspace\(3\)", line):
                events += "L"
            elif "@llvm.amdgcn.wave.barrier" in line or "s_barrier" in line or "@llvm.amdgcn.s.barrier" in line:
                events += "B"
        assert "S" in events and "L" in events, name
        assert "SL" not in events and "LS" not in events, f"{name}: {events}"


@needs_hipcc
def test_asm_that_writes_m0_says_so(kernels):
    """The compiler uses M0 for instructions of its own: a block that writes it has to be in its list."""
    seen = 0
    for name, lines in kernels.items():
        for line in lines:
            if " asm " in line and re.search(r"\bm0\b", line.split('"')[1]):
                seen += 1
                assert "~{m0}" in line, f"{name}: {line.strip()}"
    assert seen > 0

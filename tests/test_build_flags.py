"""Device code is built without packed fp32 instructions wherever this repository builds it or says how to."""
import glob
import os
import subprocess

import pytest

from conftest import ROOT
from loops_amd._lib import DEVICE_FLAGS

SOURCE = """
#include <hip/hip_runtime.h>
__global__ void two(const float2* a, const float2* b, float2* c) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  c[i] = make_float2(a[i].x * b[i].x + c[i].x, a[i].y * b[i].y + c[i].y);
}
"""


@pytest.mark.parametrize("flags", [DEVICE_FLAGS, []])
def test_device_code_of_the_tests_own_builds(tmp_path, flags):
    """A kernel that -O3 would pack, with the library's flags and with none (what the C++ tests pass: conftest adds them)."""
    src, out = tmp_path / "two.hip", tmp_path / "two.s"
    src.write_text(SOURCE)
    subprocess.check_call(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-std=c++17", "-O3", *flags, "--cuda-device-only", "-S", str(src), "-o", str(out)],
                          stderr=subprocess.DEVNULL)
    text = out.read_text()
    assert "v_fma" in text and "v_pk_" not in text


def test_written_commands():
    """Every hipcc command line of the build scripts, the integration guide and the sources' build notes."""
    files = ["INTEGRATION.md", "oracle/Makefile", "loops_amd/csrc/loops_c_abi.hip", *glob.glob("scripts/build_*.sh", root_dir=ROOT),
             *glob.glob("tests/perf/*.hip", root_dir=ROOT)]
    seen = 0
    for name in files:
        for line in open(os.path.join(ROOT, name), encoding="utf-8"):
            if "--offload-arch=gfx950" in line and ("hipcc" in line or "FLAGS" in line):
                seen += 1
                assert " ".join(DEVICE_FLAGS) in line, (name, line)
    assert seen >= 9

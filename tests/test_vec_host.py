"""What the vectors of csrc/vec.h promise the compiler of their addresses: the callers check
16 bytes at most, so no access may be declared at more (no GPU needed: the device code is
compiled, not run)."""
import re
import subprocess

import pytest

from ssla_amd import build

SOURCE = """
#include "vec.h"
using namespace ssla;
template <int DT, int W>
__global__ void copy(const void *x, void *y) { store_vec<DT, W>(y, threadIdx.x * W, load_vec<DT, W>(x, threadIdx.x * W)); }
template <int DT, int W>
__global__ void held(const void *x, uint32_t *y) { y[threadIdx.x] = load_held<DT, W>(x, threadIdx.x * W).w[0]; }
#define FORMS(W) \\
  template __global__ void copy<SSLA_F32, W>(const void *, void *); \\
  template __global__ void copy<SSLA_BF16, W>(const void *, void *); \\
  template __global__ void copy<SSLA_F16, W>(const void *, void *); \\
  template __global__ void held<SSLA_F32, W>(const void *, uint32_t *); \\
  template __global__ void held<SSLA_BF16, W>(const void *, uint32_t *); \\
  template __global__ void held<SSLA_F16, W>(const void *, uint32_t *);
FORMS(1) FORMS(2) FORMS(4) FORMS(8)
"""


def test_no_access_is_declared_past_16_bytes(tmp_path):
    src = tmp_path / "vectors.hip"
    src.write_text(SOURCE)
    cmd = [build._hipcc(), *build.HIPCC_FLAGS, f"-I{build.CSRC}", "--cuda-device-only", "-emit-llvm", "-S", str(src), "-o", "-"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        pytest.fail(res.stderr)
    accesses = [line for line in res.stdout.splitlines() if re.search(r"\b(load|store|memcpy)\b.* addrspace\(1\)", line)]
    aligned = [int(a) for line in accesses for a in re.findall(r"align (\d+)", line)]
    assert len(accesses) >= 36 and max(aligned) == 16, max(aligned)

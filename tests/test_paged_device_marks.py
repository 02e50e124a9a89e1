"""The mark by which tests/test_paged_device_code.py finds a split spill is one that
this compiler writes: a kernel that holds too many four-register operands of matrix
instructions gets it, under the flags of the paged attention's sources. A compiler
that words it otherwise fails here, instead of passing there."""

import concurrent.futures as cf
import os
import subprocess

import pytest

from mtplx_amd import build

KERNEL = """
#include <hip/hip_runtime.h>
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__global__ __launch_bounds__(256, 1) void crowded(const bf16x8* in, float* out, int n) {
  bf16x8 x[HELD];   // four registers each, beside 192 of sums: 512 are there
  f32x16 sum[12] = {};
#pragma unroll
  for (int i = 0; i < HELD; ++i) x[i] = in[i * 256 + threadIdx.x];
  for (int k = 0; k < n; ++k) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      sum[i % 12] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[i], x[(7 * i + 3) % HELD], sum[i % 12], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 12; ++i)
    for (int j = 0; j < 16; ++j) out[(i * 16 + j) * 256 + threadIdx.x] = sum[i][j];
}
"""


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc")
def test_a_split_spill_is_marked(tmp_path):
    src = tmp_path / "crowded.hip"
    src.write_text(KERNEL)

    def assembly(held):
        out = tmp_path / f"{held}.s"
        subprocess.run([build.HIPCC, *build.flags_for("paged_attn.hip"), "--cuda-device-only", "-S", f"-DHELD={held}",
                        str(src), "-o", str(out)], check=True, capture_output=True)
        return out.read_text()

    sizes = (74, 78, 82)   # (which of them split a tuple is the allocator's choice)
    with cf.ThreadPoolExecutor(len(sizes)) as pool:
        texts = list(pool.map(assembly, sizes))
    assert all("mfma" in t for t in texts) and any("Reload Reuse" in t for t in texts)

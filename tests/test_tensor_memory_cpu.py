"""CTAs of a cluster wait for one another while they hold tensor memory. Two clusters whose CTAs could come up on one SM although their
columns of it exceed 512 could wait for each other's without end, so no two such CTAs may fit one SM's shared memory. Sizes only, from
the headers that the launches take them from, over everything that the launches can ask for."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tracea_b200", "csrc")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

PROGRAM = """
#include <cstdio>
#include <algorithm>
#include "conv2d_sm100.cuh"
#include "conv2d_window_sm100.cuh"
#include "mx_gemm_sm100.cuh"
#include "mx_tokens_sm100.cuh"
using namespace tb200;
int main() {
  const long long sm = 228 * 1024, most = 227 * 1024, reserved = 1024;    // of an SM; of a CTA; what a CTA takes besides
  long long tokens = most, pair = most;
  for (int cols = 16; cols <= kTokMaxRows; cols += 16)
    for (int stages = 1; stages <= kTokMaxStages; ++stages)
      for (int fused = 0; fused <= kTokFusedSteps; ++fused) tokens = std::min<long long>(tokens, tok_smem_bytes(cols, stages, fused));
  // the resident-filter kernel: every filter, pitch and number of 128-pixel blocks that its plan may have
  for (long long R = 1; R <= 3; ++R)
    for (long long S = 1; S <= 3; ++S)
      for (long long Wp = 1; Wp <= 256 && R * S >= 4; ++Wp)
        for (long long nb = 1; nb <= kWinMaxBlocks; ++nb)
          for (long long ht = 1; ht * Wp <= 128 * nb + Wp; ++ht) {
            const long long reach = 128 * nb + (R - 1) * Wp + (S - 1), slot = (std::max((ht + R - 1) * Wp, reach) * 128 + 1023) / 1024 * 1024;
            const long long n = window_smem_bytes(static_cast<uint32_t>(R * S) * 4096u, static_cast<uint32_t>(slot));
            if (n <= most) pair = std::min(pair, n);
          }
  printf("%lld %lld\\n", tokens, pair);
  // the general convolution's pairs, with as few stages as a knob may ask for
  for (int depth = 0; depth <= 2; ++depth) pair = std::min<long long>(pair, conv_launch_smem_bytes(256, 2, true, false, depth, 0));
  // the 4-bit product's pairs
  for (int bn = 192; bn <= 256; bn += 64)
    for (int store = kMxStoreTma; store <= kMxStoreMx; ++store)
      pair = std::min<long long>(pair, mx_smem_bytes(bn, mx_num_stages(bn, true, store), true, store));
  // 256 columns twice, 512 alone: two CTAs of the form for few rows fit beside each other, and nothing else
  const bool three = 3 * (tokens + reserved) > sm, mixed = tokens + pair + 2 * reserved > sm, two = 2 * (pair + reserved) > sm;
  printf("%lld %lld %d %d %d\\n", tokens, pair, three, mixed, two);
  return three && mixed && two ? 0 : 1;
}
"""


@pytest.mark.skipif(shutil.which(NVCC) is None, reason="needs nvcc")
def test_no_two_clusters_can_wait_for_each_others_tensor_memory(tmp_path):
    source, program = tmp_path / "sizes.cu", tmp_path / "sizes"
    source.write_text(PROGRAM)
    subprocess.run([NVCC, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, "-o", str(program), str(source)], check=True)
    r = subprocess.run([str(program)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout

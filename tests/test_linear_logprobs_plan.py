"""The regions of linear_token_logprobs' backward workspace hold what every piece of the vocabulary puts there.

The plan is host arithmetic in a header of its own: it is compiled by itself, and walked over rows, widths,
vocabularies and types with products that ask for no workspace, so that nothing behind a region hides that it is short.
"""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "wayfinder_attention_b200" / "csrc"

PROGRAM = r"""
#include "wf_linear_logprobs_plan.h"
#include <cstdio>

namespace wf {
// A product's workspace is never less than this.
size_t gemm_workspace_bytes(int64_t, int64_t, int64_t, int, int) { return 0; }
}

int main() {
  using namespace wf;
  const int64_t rows[] = {1, 16, 64, 65, 512, 1531, 2048, 4096, 8192, 8193, 16384, 32768, 65536, 200000};
  const int64_t widths[] = {1, 64, 256, 768, 1001, 1024, 2048, 4096, 8192};
  const int64_t vocabularies[] = {1, 128, 2047, 2049, 10007, 32000, 50001, 50257, 65537, 128000, 128256, 131072, 151936, 262144};
  long calls = 0, short_ones = 0;
  for (int64_t M : rows)
    for (int64_t K : widths)
      for (int64_t N : vocabularies)
        for (int dtype : {(int)kBF16, (int)kF16, (int)kF32}) {
          const BwdPlan b = make_bwd_plan(M, N, K, dtype);
          ++calls;
          for (int64_t first = 0; first < N; first += b.columns) {
            const int64_t n = std::min(b.columns, N - first);
            // blocks over the rows times columns partial sums, as dz_columns_kernel stores them
            const size_t sums = (size_t)column_shares(M, n) * n * sizeof(float);
            const size_t dz = (size_t)M * round8(n) * (dtype == kF32 ? 4 : 2) * b.layers;
            const size_t operand = dtype == kF32 ? (size_t)M * round8(n) * 6 : 0;
            const size_t dw = b.dw_apart ? (size_t)n * round8(K) * sizeof(float) : 0;
            const size_t dx = b.dx_apart ? (size_t)M * round8(K) * sizeof(float) : 0;
            const size_t x = b.scaled ? (size_t)M * round8(K) * 2 : 0;
            if (sums > b.sums || dz > b.dz || operand > b.dz_operand || dw > b.dw || dx > b.dx || x > b.scaled_x) {
              if (++short_ones <= 5)
                std::printf("%ld x %ld -> %ld, type %d, piece of %ld: sums %zu of %zu, dz %zu of %zu, operand %zu of %zu, "
                            "dw %zu of %zu\n", (long)M, (long)K, (long)N, dtype, (long)n, sums, b.sums, dz, b.dz, operand,
                            b.dz_operand, dw, b.dw);
            }
          }
        }
  std::printf("%ld calls, %ld short pieces\n", calls, short_ones);
  return short_ones != 0;
}
"""


def test_every_piece_fits_its_regions(tmp_path):
    from wayfinder_attention_b200 import build

    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    source, program = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text(PROGRAM)
    cuda = Path(build.nvcc_path()).resolve().parent.parent / "include"
    subprocess.run([gxx, "-std=c++17", "-O1", "-I", str(CSRC), "-isystem", str(cuda), str(source), "-o", str(program)], check=True)
    r = subprocess.run([str(program)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout

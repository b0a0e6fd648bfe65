// What a backward of linear_token_logprobs (wf_linear_logprobs.cu) cuts the vocabulary into, and the regions of its
// workspace.  Host arithmetic alone, which the tests compile by themselves.
#pragma once

#include "wf_gemm.h"
#include "wf_kernels.h"

#include <algorithm>

namespace wf {
namespace {

// Blocks over the rows that sum a bias's gradient, and the partial sums that they leave.  A shorter piece has more
// blocks and may leave more: 12 x 25344 of a full piece, 13 x 24913 of the last one (8192 rows -> 50257).
inline int column_shares(int64_t M, int64_t N) {
  const int64_t by = (N + 255) / 256, want = (8 * kSms + by - 1) / by, most = (M + 15) / 16;
  return (int)std::max<int64_t>(1, std::min(want, most));
}
inline size_t column_sum_bytes(int64_t M, int64_t N) {
  return round256((size_t)column_shares(M, N) * N * sizeof(float));
}

// Columns of the vocabulary that a piece has: as many as 512 MB of dz hold, but 2048 at least
// (shorter ones leave the products' tiles idle) and all of them where they are few.  More are cut into pieces of
// like size, in the least number or one of the next few, whichever leaves the pairs of blocks idle
// least: each product of a piece takes whole waves of tiles.  (Training at 8192 x 1024 -> 50001: 256 MB
// 2.68 ms, 512 MB 2.61; pieces of 64 MB, which L2 would hold, 2.87.)
constexpr int64_t kPieceBytes = 512ll << 20, kPieceLeast = 2048;
inline int64_t piece_columns(int64_t M, int64_t N, int64_t K, int dtype, int layers) {
  int64_t fit = kPieceBytes / (M * (dtype == kF32 ? 10 : 2 * layers)) / 256 * 256;
  if (dtype == kF16) fit = std::min(fit, kPieceBytes / (4 * round8(K)) / 256 * 256);  // the piece's rows of dW in fp32
  const int64_t most = std::max(fit, kPieceLeast);
  if (N <= most) return N;
  auto waves = [](int64_t tiles) { return (tiles + kSms / 2 - 1) / (kSms / 2); };
  const int64_t tm = (M + 255) / 256, tk = (K + 255) / 256;
  auto stages = [&](int64_t n) {  // of a piece's three products
    const int64_t tn = (n + 255) / 256;
    return waves(tm * tn) * ((K + 63) / 64) + waves(tm * tk) * ((n + 63) / 64) + waves(tn * tk) * ((M + 63) / 64) + 12;
  };
  int64_t best = 0, least = 0;
  const int64_t fewest = (N + most - 1) / most;
  for (int64_t pieces = fewest; pieces < fewest + 6; ++pieces) {
    const int64_t columns = ((N + pieces - 1) / pieces + 255) / 256 * 256;
    if (columns > most || (pieces > fewest && columns < kPieceLeast)) continue;
    const int64_t whole = N / columns, rest = N % columns;
    const int64_t cost = whole * stages(columns) + (rest ? stages(rest) : 0);
    if (!best || cost < least) {
      least = cost;
      best = columns;
    }
  }
  return best ? best : most;
}
// Pieces of a 16-bit dz, as in wf_linear.cu: two where the products are small, so that rounding it
// adds nothing to the gradients' own rounding.  And up to 64 rows, where a row of dW is a row or
// two of x and one rounding makes much of its error: the products are bound by the weight's bytes
// there and pay a sixth for it (64 rows, 1024 -> 50001: 86 -> 100 us; at 512 rows it would be 162 -> 251).
inline int dz_layers(int64_t M, int64_t N, int64_t K, int dtype) {
  return dtype != kF32 && ((double)M * N * K <= (double)(1 << 30) || M <= 64) ? 2 : 1;
}

struct BwdPlan {
  int64_t columns;
  int layers, pieces;
  bool scaled, dx_apart, dw_apart;
  size_t exponents, factor, dz, dz_operand, dx, dw, sums, scaled_x, gemm;
};
inline BwdPlan make_bwd_plan(int64_t M, int64_t N, int64_t K, int dtype) {
  BwdPlan b{};
  b.layers = dz_layers(M, N, K, dtype);
  b.columns = piece_columns(M, N, K, dtype, b.layers);
  b.pieces = dtype == kF32 ? 3 : 1;
  b.scaled = dtype == kF16;
  b.dx_apart = dtype != kF32 && (b.scaled || b.columns < N);  // fp32 sums, rounded at the end
  b.dw_apart = b.scaled;
  b.exponents = b.scaled ? round256((M + 1) * sizeof(int)) : 0;
  b.factor = dtype != kF32 && b.layers == 1 ? round256(2 * sizeof(float)) : 0;
  b.dz = round256((size_t)M * round8(b.columns) * (dtype == kF32 ? 4 : 2) * b.layers);
  b.dz_operand = dtype == kF32 ? operand_bytes(M, b.columns, dtype) : 0;
  b.dx = b.dx_apart ? round256((size_t)M * round8(K) * sizeof(float)) : 0;
  b.dw = b.dw_apart ? round256((size_t)b.columns * round8(K) * sizeof(float)) : 0;
  b.scaled_x = b.scaled ? operand_bytes(M, K, dtype) : 0;
  const int64_t last = N - (N - 1) / b.columns * b.columns;
  for (int64_t n : {b.columns, last}) {
    b.sums = std::max(b.sums, column_sum_bytes(M, n));
    b.gemm = std::max({b.gemm, gemm_workspace_bytes(M, K, n, b.pieces, b.layers),
                       gemm_workspace_bytes(n, K, M, b.pieces, b.layers)});
  }
  return b;
}

}  // namespace
}  // namespace wf

// Linear layer with its epilogue, forward and backward, on the tensor-core product.
//
//   forward   z = x W^T + b,  y = act(z) + residual
//   backward  dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_rows dz
//
// act: none, gelu (z Phi(z), Phi by erf), relu, silu (z sigmoid(z)).  Products and sums
// are fp32; y is rounded once.  The backward reads z as the forward kept it (fp16 for both
// 16-bit types), and takes dz in the activations' type to the two products, in one piece or
// (small products, see dz_turns) two; db sums the unrounded values.
//
#include "wf_activation.cuh"
#include "wf_columns.cuh"
#include "wf_gemm.h"
#include "wf_linear_few.h"
#include "wf_operand.cuh"
#include "wf_rowio.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>
#include <utility>

namespace wf {
namespace {

// dz = dy act'(z) into the operand's layout, and partial column sums: a block takes 256
// columns (8 a lane) of a share of the rows, its 8 warps a row each.  Bound by the bytes (dy, z
// and dz each once): a row's registers take the next one's loads as soon as they are unpacked,
// and four blocks an SM keep enough of them under way.  8192 x 4096, gelu, bf16: 41 us (4.9
// TB/s); two rows loaded and then computed at two blocks an SM took 53, two rows ahead at
// three blocks 43.  fp32 holds one row ahead (78 us; two of them spill: 97).
template <typename T>
constexpr int kRowsAhead = sizeof(T) == 4 ? 1 : 2;
template <typename T, int ACT>
__global__ void __launch_bounds__(256, 4) linear_dz_kernel(const T* dy, int64_t dy_stride, bool dy_vec,
                                                        const typename Kept<T>::type* z, void* out, int64_t pitch,
                                                        int64_t piece, int64_t M, int64_t N, float* partials) {
  __shared__ float red[8][32][9];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + lane) * 8;
  float s[8] = {};
  const int64_t z_pitch = (N + 7) / 8 * 8;
  if (c < N) {
    constexpr int kAhead = kRowsAhead<T>;
    Raw8<T> rg[kAhead];
    Raw8<typename Kept<T>::type> rz[kAhead];
    const int64_t step = (int64_t)gridDim.y * 8;
    auto load = [&](int i, int64_t m) {
      if (m < M) {
        rg[i].load(dy + m * dy_stride, c, N, dy_vec);
        if constexpr (ACT != kActNone) rz[i].load(z + m * z_pitch, c, N, true);
      }
    };
    int64_t m = (int64_t)blockIdx.y * 8 + warp;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(i, m + i * step);
    while (m < M) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i, m += step) {
        if (m >= M) break;
        float g[8], f[8];
        rg[i].unpack(g);
        if constexpr (ACT != kActNone) rz[i].unpack(f);
        load(i, m + kAhead * step);
        if constexpr (ACT != kActNone) times_slope<ACT, T, 8>(f, g);
        if (out) store_operand<T>(out, m * pitch + c, piece, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += g[j];
      }
    }
  }
  if (!partials) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[warp][lane][j] = s[j];
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col < N) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += red[i][threadIdx.x / 8][threadIdx.x % 8];
    partials[(size_t)blockIdx.y * N + col] = v;
  }
}

// Row shares of the column sums: eight blocks an SM over all columns, 16 rows at least.
int row_shares(int64_t M, int64_t N) {
  const int64_t by = (N + 255) / 256, want = (8 * kSms + by - 1) / by, most = (M + 15) / 16;
  return (int)(want < most ? want : most);
}

template <typename T>
int launch_fwd(const LinearParams& p, int dtype, cudaStream_t stream) {
  if (linear_few_takes(p, dtype)) return launch_linear_few(p, dtype, stream);
  unsigned char* ws = static_cast<unsigned char*>(p.ws);
  GemmOperand o[2];
  if (int rc = operands<T>({{p.x, p.M, p.K, p.x_stride}, {p.w, p.N, p.K, p.w_stride}}, dtype, &ws, o, stream)) return rc;
  GemmProblem g = problem<T>(o[0], o[1], p.M, p.N, p.K, dtype, ws, p.status);
  g.out = GemmEpilogue{p.bias, p.residual, p.z, p.y, p.r_stride, round8(p.N), p.N, p.act};
  return launch_gemm(g, stream);
}

template <typename T, int ACT>
cudaError_t launch_dz(const LinearBwdParams& p, const GemmOperand& o, bool write, float* partials,
                      cudaStream_t stream) {
  return launch_pdl(linear_dz_kernel<T, ACT>, dim3((unsigned)((p.N + 255) / 256), row_shares(p.M, p.N)), dim3(256), 0,
                    stream, static_cast<const T*>(p.dy), p.dy_stride, on_16_bytes<T>(p.dy, p.dy_stride),
                    static_cast<const typename Kept<T>::type*>(p.z), write ? const_cast<void*>(o.ptr) : nullptr, o.pitch, o.piece_stride,
                    p.M, p.N, partials);
}

// Pieces of a 16-bit dz.  gelu's and silu's has more bits than its type, and rounding it
// leaves dx and dW with 1.4 times the error of their own rounding (more by chance where they
// have few elements).  Small products take what is left as a second piece, walk the depth twice
// and are exact but for their own rounding.  That is 23.2 -> 25.3 us of a step's kernels (forward
// and backward, in a captured graph) at 256 x 1024 x 256, 28.4 -> 30.2 at 1024 x 1024 x 256 and
// 32.7 -> 43.2 at 1024^3, where an eager step takes 83 us either way, the host's; past 2^30
// multiplications the products are what a step waits for (4096 x 4096 x 1024: eager 134 -> 190 us).
int dz_turns(int64_t M, int64_t N, int64_t K, int dtype, int act) {
  const bool rounded = dtype != kF32 && (act == kActGelu || act == kActSilu);
  return rounded && (double)M * N * K <= (double)(1 << 30) ? 2 : 1;
}

template <typename T>
int launch_bwd(const LinearBwdParams& p, int dtype, cudaStream_t stream) {
  if (p.M == 0) {  // sums over no rows
    for (auto [ptr, n] : {std::pair<void*, size_t>{p.dw, (size_t)p.N * p.K}, {p.db, (size_t)p.N}})
      if (ptr)
        if (cudaError_t e = cudaMemsetAsync(ptr, 0, n * sizeof(T), stream)) return (int)e;
    return 0;
  }
  unsigned char* ws = static_cast<unsigned char*>(p.ws);
  const bool products = p.dx || p.dw;
  const bool direct = p.act == kActNone && dtype != kF32 && on_16_bytes<T>(p.dy, p.dy_stride);
  GemmOperand dz{p.dy, p.M, p.N, p.dy_stride, 0, false};
  const int turns = dz_turns(p.M, p.N, p.K, dtype, p.act);
  if (products && !direct) dz = blank_operand<T>(p.M, p.N, dtype, &ws, turns);
  float* partials = nullptr;
  if (p.db) {
    partials = reinterpret_cast<float*>(ws);
    ws += round256((size_t)row_shares(p.M, p.N) * p.N * sizeof(float));
  }
  if (p.db || (products && !direct)) {
    const bool write = products && !direct;
    cudaError_t e;
    switch (p.act) {
      case kActGelu: e = launch_dz<T, kActGelu>(p, dz, write, partials, stream); break;
      case kActRelu: e = launch_dz<T, kActRelu>(p, dz, write, partials, stream); break;
      case kActSilu: e = launch_dz<T, kActSilu>(p, dz, write, partials, stream); break;
      default: e = launch_dz<T, kActNone>(p, dz, write, partials, stream); break;
    }
    if (e) return (int)e;
  }
  if (p.db)
    if (cudaError_t e = join_columns<T>(partials, row_shares(p.M, p.N), p.N, p.N, p.db, nullptr, stream)) return (int)e;
  GemmOperand o[2];  // w for dx, x for dw
  if (int rc = operands<T>({{p.dx ? p.w : nullptr, p.N, p.K, p.w_stride}, {p.dw ? p.x : nullptr, p.M, p.K, p.x_stride}},
                           dtype, &ws, o, stream))
    return rc;
  if (p.dx) {
    o[0].mn_major = true;  // its columns are dx's, its rows the depth
    GemmProblem g = problem<T>(dz, o[0], p.M, p.K, p.N, dtype, ws, p.status);
    g.turns = turns;
    g.out.y = p.dx;
    g.out.y_stride = p.K;
    if (int rc = launch_gemm(g, stream)) return rc;
  }
  if (p.dw) {
    dz.mn_major = o[1].mn_major = true;  // the rows of both are the depth
    GemmProblem g = problem<T>(dz, o[1], p.N, p.K, p.M, dtype, ws, p.status);
    g.turns = turns;
    g.out.y = p.dw;
    g.out.y_stride = p.K;
    if (int rc = launch_gemm(g, stream)) return rc;
  }
  return 0;
}

}  // namespace

size_t linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, bool x_direct, bool w_direct) {
  if (M <= kFewRows) return 0;  // linear_few_takes them, whatever their type and alignment
  const int pieces = dtype == kF32 ? 3 : 1;
  return (x_direct && pieces == 1 ? 0 : operand_bytes(M, K, dtype)) +
         (w_direct && pieces == 1 ? 0 : operand_bytes(N, K, dtype)) + gemm_workspace_bytes(M, N, K, pieces);
}

size_t linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int act, bool x_direct,
                                       bool w_direct, bool dy_direct) {
  const int pieces = dtype == kF32 ? 3 : 1;
  const int turns = dz_turns(M, N, K, dtype, act);
  const size_t dz = act == kActNone && pieces == 1 && dy_direct ? 0 : operand_bytes(M, N, dtype, turns);
  const size_t sums = round256((size_t)row_shares(M, N) * N * sizeof(float));
  const size_t laid_out = (w_direct && pieces == 1 ? 0 : operand_bytes(N, K, dtype)) +
                          (x_direct && pieces == 1 ? 0 : operand_bytes(M, K, dtype));
  const size_t dx = gemm_workspace_bytes(M, K, N, pieces, turns), dw = gemm_workspace_bytes(N, K, M, pieces, turns);
  return dz + sums + laid_out + std::max(dx, dw);  // the products' parts, one after the other
}

int launch_linear(const LinearParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_fwd<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_fwd<__half>(p, dtype, stream);
  return launch_fwd<float>(p, dtype, stream);
}

int launch_linear_backward(const LinearBwdParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_bwd<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_bwd<__half>(p, dtype, stream);
  return launch_bwd<float>(p, dtype, stream);
}

}  // namespace wf

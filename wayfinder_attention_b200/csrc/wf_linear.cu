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
// The product reads 16-bit matrices whose rows start on 16 bytes.  Others are laid out in
// the workspace first: 16-bit rows of any width or offset are copied to such rows, and an
// fp32 matrix becomes three bf16 pieces, x = x0 + x1 + x2 to fp32's last bit.
#include "wf_activation.cuh"
#include "wf_columns.cuh"
#include "wf_gemm.h"
#include "wf_linear_few.h"
#include "wf_rowio.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>
#include <utility>

namespace wf {
namespace {

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// x = p[0] + p[1] + p[2], each a rounding of what the ones before leave.  Infinities and
// NaN stay in p[0] alone; what would round to infinity is cut instead.
__device__ __forceinline__ void split3(float x, __nv_bfloat16* p) {
  p[0] = __float2bfloat16_rn(x);
  if (isinf(__bfloat162float(p[0])) && !isinf(x)) p[0] = __float2bfloat16_rz(x);
  float r = isfinite(x) ? x - __bfloat162float(p[0]) : 0.f;
  p[1] = __float2bfloat16_rn(r);
  p[2] = __float2bfloat16_rn(r - __bfloat162float(p[1]));
}

// 8 fp32 values to the operand at column c of a row: one 16-byte store a piece (the
// operand's rows are padded to whole vectors).
template <typename T>
__device__ __forceinline__ void store_operand(void* out, int64_t at, int64_t piece, const float* f) {
  if constexpr (std::is_same<T, float>::value) {
    __nv_bfloat16 p[8][3];
#pragma unroll
    for (int j = 0; j < 8; ++j) split3(f[j], p[j]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint4 v;
      uint32_t* u = &v.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __nv_bfloat162 h;
        h.x = p[2 * j][k];
        h.y = p[2 * j + 1][k];
        u[j] = *reinterpret_cast<uint32_t*>(&h);
      }
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + k * piece + at) = v;
    }
  } else {
    store_vec<T, 8>(static_cast<T*>(out) + at, f);
    if (piece) {  // what that rounding leaves, where the operand has a second piece
      float left[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float r = to_f32(from_f32<T>(f[j]));
        left[j] = isfinite(r) ? f[j] - r : 0.f;
      }
      store_vec<T, 8>(static_cast<T*>(out) + piece + at, left);
    }
  }
}

// 8 values of a row from column c (zeros past the end), by vectors where the row allows it.
template <typename T>
struct Raw8 {
  static constexpr int V = Vec16<T>::N;
  uint4 raw[8 / V];
  __device__ __forceinline__ void load(const T* row, int64_t c, int64_t cols, bool vec) {
    if (vec && c + 8 <= cols) {
#pragma unroll
      for (int j = 0; j < 8 / V; ++j) raw[j] = ldg16(row + c + j * V);
    } else {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = c + j < cols ? row[c + j] : from_f32<T>(0.f);
      memcpy(raw, e, sizeof(e));
    }
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) Vec16<T>::unpack(raw[j], f + j * V);
  }
};

// Lays matrices out as operands: the blocks are shared between up to two of them.
template <typename T>
struct LayOut {
  const T* x;
  void* out;
  int64_t rows, cols, stride, pitch, piece;
  int blocks;
  bool vec;
};
template <typename T>
__global__ void __launch_bounds__(256) lay_out_kernel(LayOut<T> first, LayOut<T> second) {
  pdl_wait();
  const bool one = (int)blockIdx.x < first.blocks;
  const LayOut<T>& j = one ? first : second;
  const int64_t block = one ? blockIdx.x : blockIdx.x - first.blocks;
  const int64_t groups = j.pitch / 8, total = j.rows * groups;
  for (int64_t i = block * 256 + threadIdx.x; i < total; i += (int64_t)j.blocks * 256) {
    const int64_t r = i / groups, c = i % groups * 8;
    Raw8<T> raw;
    raw.load(j.x + r * j.stride, c, j.cols, j.vec);
    float f[8];
    raw.unpack(f);
    store_operand<T>(j.out, r * j.pitch + c, j.piece, f);
  }
}

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
constexpr int kPieces = std::is_same<T, float>::value ? 3 : 1;

template <typename T>
bool on_16_bytes(const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
}

// A (rows, cols) matrix as the product reads it: itself, or laid out at *ws, which moves on.
size_t operand_bytes(int64_t rows, int64_t cols, int dtype, int turns = 1) {
  return round256((size_t)rows * round8(cols) * 2 * (dtype == kF32 ? 3 : turns));
}
template <typename T>
GemmOperand blank_operand(int64_t rows, int64_t cols, int dtype, unsigned char** ws, int turns = 1) {
  GemmOperand o{};
  o.ptr = *ws;
  o.rows = rows;
  o.cols = cols;
  o.pitch = round8(cols);
  o.piece_stride = dtype == kF32 || turns > 1 ? rows * o.pitch : 0;
  *ws += operand_bytes(rows, cols, dtype, turns);
  return o;
}
// Two matrices as operands, either of which may be missing (no pointer); what has to be laid
// out goes in one launch.
struct Matrix {
  const void* ptr;
  int64_t rows, cols, stride;
};
template <typename T>
int operands(const Matrix (&m)[2], int dtype, unsigned char** ws, GemmOperand (&o)[2], cudaStream_t stream) {
  LayOut<T> jobs[2] = {};
  for (int i = 0; i < 2; ++i) {
    if (!m[i].ptr) continue;
    const bool vec = on_16_bytes<T>(m[i].ptr, m[i].stride);
    if (dtype != kF32 && vec) {
      o[i] = GemmOperand{m[i].ptr, m[i].rows, m[i].cols, m[i].stride, 0, false};
      continue;
    }
    o[i] = blank_operand<T>(m[i].rows, m[i].cols, dtype, ws);
    const int64_t blocks = (m[i].rows * (o[i].pitch / 8) + 255) / 256;
    jobs[i] = LayOut<T>{static_cast<const T*>(m[i].ptr), const_cast<void*>(o[i].ptr), m[i].rows, m[i].cols,
                        m[i].stride, o[i].pitch, o[i].piece_stride, (int)std::min<int64_t>(blocks, 16 * kSms), vec};
  }
  const int blocks = jobs[0].blocks + jobs[1].blocks;
  return blocks ? (int)launch_pdl(lay_out_kernel<T>, dim3(blocks), dim3(256), 0, stream, jobs[0], jobs[1]) : 0;
}

template <typename T>
GemmProblem problem(const GemmOperand& a, const GemmOperand& b, int64_t M, int64_t N, int64_t K, int dtype, void* ws,
                    int32_t* status) {
  GemmProblem g{};
  g.a = a;
  g.b = b;
  g.M = M;
  g.N = N;
  g.K = K;
  g.pieces = kPieces<T>;
  g.turns = 1;
  g.op_dtype = dtype == kF16 ? kF16 : kBF16;
  g.out_dtype = dtype;
  g.ws = ws;
  g.status = status;
  return g;
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

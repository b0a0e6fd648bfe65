// Linear layer with its epilogue, forward and backward.
//
//   forward   z = x W^T + b,  y = act(z) + residual
//   backward  dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_rows dz
//
// act: none, gelu (z Phi(z), Phi by erf), relu, silu (z sigmoid(z)).  Products and sums
// are fp32; y is rounded once.  The backward reads z as the forward rounded it to the
// activations' type, and rounds dz to that type before the two products, as operands of
// that type are what the products take.
#include "wf_columns.cuh"
#include "wf_kernels.h"
#include "wf_rowio.cuh"

namespace wf {
namespace {

__device__ __forceinline__ float gelu_cdf(float z) { return 0.5f * (1.f + erff(z * 0.70710678118654752f)); }
__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }

__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case kActGelu: return z * gelu_cdf(z);
    case kActRelu: return z < 0.f ? 0.f : z;  // NaN stays
    case kActSilu: return z * sigmoid(z);
    default: return z;
  }
}
__device__ __forceinline__ float activation_slope(int act, float z) {
  switch (act) {
    case kActGelu: return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), gelu_cdf(z));
    case kActRelu: return z > 0.f ? 1.f : 0.f;
    case kActSilu: {
      const float s = sigmoid(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    default: return 1.f;
  }
}

// C[m][n] = sum_k A(m, k) B(n, k) over any element strides, then the epilogue.
struct GemmParams {
  const void* a;
  const void* b;
  int64_t am, ak, bn, bk;
  int64_t M, N, K;
  const void* bias;
  const void* residual;
  void* z;
  void* y;
  int64_t r_stride, z_stride, y_stride;
  int act;
};

constexpr int kTile = 64, kDepth = 16;
template <typename T>
__global__ void __launch_bounds__(256) gemm_kernel(GemmParams p) {
  __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);
  // two levels of sums: a long one loses bits with its length
  float acc[4][4] = {}, sum[4][4] = {};
  for (int64_t k0 = 0; k0 < p.K; k0 += kDepth) {
    if (k0 % 256 == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[i][j] += acc[i][j];
          acc[i][j] = 0.f;
        }
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      // the unit-strided axis runs over the threads
      const int ka = p.ak == 1 ? i % kDepth : i / kTile, ma = p.ak == 1 ? i / kDepth : i % kTile;
      const int kb = p.bk == 1 ? i % kDepth : i / kTile, nb = p.bk == 1 ? i / kDepth : i % kTile;
      as[ka][ma] = m0 + ma < p.M && k0 + ka < p.K ? to_f32(a[(m0 + ma) * p.am + (k0 + ka) * p.ak]) : 0.f;
      bs[kb][nb] = n0 + nb < p.N && k0 + kb < p.K ? to_f32(b[(n0 + nb) * p.bn + (k0 + kb) * p.bk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[k][ty * 4 + i], bs[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= p.M || n >= p.N) continue;
      float v = sum[i][j] + acc[i][j];
      if (p.bias) v += to_f32(static_cast<const T*>(p.bias)[n]);
      if (p.z) static_cast<T*>(p.z)[m * p.z_stride + n] = from_f32<T>(v);
      v = activate(p.act, v);
      if (p.residual) v += to_f32(static_cast<const T*>(p.residual)[m * p.r_stride + n]);
      static_cast<T*>(p.y)[m * p.y_stride + n] = from_f32<T>(v);
    }
}

template <typename T>
int launch_gemm(const GemmParams& p, cudaStream_t stream) {
  if (p.M == 0 || p.N == 0) return 0;
  gemm_kernel<T><<<dim3((unsigned)((p.N + kTile - 1) / kTile), (unsigned)((p.M + kTile - 1) / kTile)), 256, 0,
                   stream>>>(p);
  return (int)cudaGetLastError();
}

// dz = dy act'(z) and the partial column sums of dz (of the unrounded values): a warp
// owns a column a lane, the block's 8 warps and the grid's y share the rows.
template <typename T>
__global__ void __launch_bounds__(256) linear_dz_kernel(const T* dy, int64_t dy_stride, const T* z, T* dz, int64_t M,
                                                        int64_t N, int act, float* partials) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < N)
    for (int64_t m = (int64_t)blockIdx.y * 8 + warp; m < M; m += (int64_t)gridDim.y * 8) {
      float g = to_f32(dy[m * dy_stride + c]);
      if (z) {
        g *= activation_slope(act, to_f32(z[m * N + c]));
        dz[m * N + c] = from_f32<T>(g);
      }
      s += g;
    }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < N && partials) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][lane];
    partials[(size_t)blockIdx.y * N + c] = s;
  }
}

int row_shares(int64_t M) { return (int)(M <= 64 ? 1 : M / 64 < 64 ? M / 64 : 64); }
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

template <typename T>
int launch_fwd(const LinearParams& p, cudaStream_t stream) {
  GemmParams g{};
  g.a = p.x; g.am = p.x_stride; g.ak = 1;
  g.b = p.w; g.bn = p.w_stride; g.bk = 1;
  g.M = p.M; g.N = p.N; g.K = p.K;
  g.bias = p.bias; g.residual = p.residual; g.r_stride = p.r_stride;
  g.z = p.z; g.z_stride = p.N;
  g.y = p.y; g.y_stride = p.N;
  g.act = p.act;
  return launch_gemm<T>(g, stream);
}

template <typename T>
int launch_bwd(const LinearBwdParams& p, cudaStream_t stream) {
  const T* dz = static_cast<const T*>(p.dy);
  int64_t dz_stride = p.dy_stride;
  unsigned char* ws = static_cast<unsigned char*>(p.ws);
  if (p.M > 0 && (p.act != kActNone || p.db)) {
    T* out = nullptr;
    if (p.act != kActNone) {
      out = reinterpret_cast<T*>(ws);
      ws += round256((size_t)p.M * p.N * sizeof(T));
      dz = out;
      dz_stride = p.N;
    }
    float* partials = p.db ? reinterpret_cast<float*>(ws) : nullptr;
    const int shares = row_shares(p.M);
    linear_dz_kernel<T><<<dim3((unsigned)((p.N + 31) / 32), shares), 256, 0, stream>>>(
        static_cast<const T*>(p.dy), p.dy_stride, p.act != kActNone ? static_cast<const T*>(p.z) : nullptr, out, p.M,
        p.N, p.act, partials);
    if (cudaError_t e = cudaGetLastError()) return (int)e;
    if (p.db)
      if (cudaError_t e = join_columns<T>(partials, shares, p.N, p.N, p.db, nullptr, stream)) return (int)e;
  } else if (p.db) {
    if (cudaError_t e = cudaMemsetAsync(p.db, 0, (size_t)p.N * sizeof(T), stream)) return (int)e;
  }
  if (p.dx) {
    GemmParams g{};
    g.a = dz; g.am = dz_stride; g.ak = 1;
    g.b = p.w; g.bn = 1; g.bk = p.w_stride;
    g.M = p.M; g.N = p.K; g.K = p.N;
    g.y = p.dx; g.y_stride = p.K;
    if (int rc = launch_gemm<T>(g, stream)) return rc;
  }
  if (p.dw) {
    GemmParams g{};
    g.a = dz; g.am = 1; g.ak = dz_stride;
    g.b = p.x; g.bn = 1; g.bk = p.x_stride;
    g.M = p.N; g.N = p.K; g.K = p.M;
    g.y = p.dw; g.y_stride = p.K;
    if (int rc = launch_gemm<T>(g, stream)) return rc;
  }
  return 0;
}

}  // namespace

size_t linear_workspace_bytes(int64_t, int64_t, int64_t, int) { return 0; }

size_t linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t, int dtype, int act) {
  const size_t dz = act == kActNone ? 0 : round256((size_t)M * N * (dtype == kF32 ? 4 : 2));
  return dz + (size_t)row_shares(M) * N * sizeof(float);
}

int launch_linear(const LinearParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_fwd<__nv_bfloat16>(p, stream);
  if (dtype == kF16) return launch_fwd<__half>(p, stream);
  return launch_fwd<float>(p, stream);
}

int launch_linear_backward(const LinearBwdParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_bwd<__nv_bfloat16>(p, stream);
  if (dtype == kF16) return launch_bwd<__half>(p, stream);
  return launch_bwd<float>(p, stream);
}

}  // namespace wf

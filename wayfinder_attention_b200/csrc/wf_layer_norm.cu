// Layer norm over the last axis, forward and backward, with the reduction of the
// parameters' gradients.
//
//   forward   mu = mean(x), var = mean((x - mu)^2), r = 1 / sqrt(var + eps),
//             y = (x - mu) r w + b
//   backward  with h = (x - mu) r and g = dy w:
//             dx = r (g - mean(g) - h mean(g h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Both are bound by bytes: x in and y out, or x and dy in and dx out.  A row is held
// in registers by the group of W warps that owns it, so each element crosses HBM
// once; the variance is a second pass over those registers (no cancellation of large
// means).  All statistics and sums are fp32; y, dx, dw and db are rounded once.
//
// Backward: groups walk rows with a stride of the grid and keep the column sums of
// their own columns in registers; the next row's vectors are requested before the
// current one is reduced, so a group always has loads in flight.  The groups of a
// block add their sums in shared memory, each block writes one row of partials, and a
// second kernel adds the blocks' rows in a fixed order (no atomics: the same inputs
// give the same bits).
#include "wf_columns.cuh"
#include "wf_kernels.h"
#include "wf_rowio.cuh"

#include <initializer_list>

namespace wf {
namespace {

// fp32 or the activations' type
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, bool f32, float absent, int64_t c, float* f) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = absent;
  } else if (f32) {
    const float* q = static_cast<const float*>(p) + c;
    if constexpr (VEC == 1) {
      f[0] = __ldg(q);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) Vec16<float>::unpack(ldg16(q + j), f + j);
    }
  } else {
    const T* q = static_cast<const T*>(p) + c;
    if constexpr (VEC == 1) f[0] = to_f32(*q);
    else Vec16<T>::unpack(ldg16(q), f);
  }
}

// Sums a pair over the W warps of a group; every thread gets the result.  `buf` holds
// 2 * W floats of the group; the caller alternates two of them so that one barrier a
// call suffices.
template <int W>
__device__ __forceinline__ float2 group_sum2(float a, float b, float2* buf, int warp_in_group) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (W == 1) return make_float2(a, b);
  if ((threadIdx.x & 31) == 0) buf[warp_in_group] = make_float2(a, b);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float2 v = buf[i];
    s.x += v.x;
    s.y += v.y;
  }
  return s;
}

// W warps a row; W = 1: eight rows a block, otherwise one row a block.
__host__ __device__ constexpr int threads_of(int W) { return W == 1 ? 256 : 32 * W; }

template <typename T, int VEC, int W, int NV>
__global__ void __launch_bounds__(threads_of(W)) layer_norm_kernel(LayerNormParams p) {
  constexpr int G = 32 * W;
  __shared__ float2 red[2][W];
  const int t = threadIdx.x % G, wig = t >> 5;
  const int64_t row = (int64_t)blockIdx.x * (threads_of(W) / G) + threadIdx.x / G;
  if (W == 1 && row >= p.rows) return;  // whole warps; W > 1 has one row a block, always in range
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  RawVec<T, VEC> raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * VEC;
    if (c < p.d) raw[i].load(x + c);
    else raw[i].clear();
  }
  float v[NV][VEC];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    raw[i].unpack(v[i]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += v[i][j];
  }
  const float inv_d = 1.f / (float)p.d;
  const float mean = group_sum2<W>(s, 0.f, red[0], wig).x * inv_d;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * G + t) * VEC < p.d) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] -= mean;
        q = fmaf(v[i][j], v[i][j], q);
      }
    }
  }
  const float var = group_sum2<W>(q, 0.f, red[1], wig).x * inv_d;
  const float rstd = 1.f / sqrtf(var + p.eps);
  T* y = static_cast<T*>(p.y) + row * p.y_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * VEC;
    if (c < p.d) {
      float w[VEC], b[VEC];
      load_param<T, VEC>(p.weight, p.param_f32, 1.f, c, w);
      load_param<T, VEC>(p.bias, p.param_f32, 0.f, c, b);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf(v[i][j] * rstd, w[j], b[j]);
      store_vec<T, VEC>(y + c, v[i]);
    }
  }
  if (t == 0 && p.mean) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
}

// Rows too long for registers: one block a row, three passes over it (the second and
// third find it in L2).
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(LayerNormParams p) {
  __shared__ float2 red[2][32];
  const int wig = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  T* y = static_cast<T*>(p.y) + row * p.y_stride;
  float s = 0.f;
  for (int c = threadIdx.x; c < p.d; c += 1024) s += to_f32(x[c]);
  const float inv_d = 1.f / (float)p.d;
  const float mean = group_sum2<32>(s, 0.f, red[0], wig).x * inv_d;
  float q = 0.f;
  for (int c = threadIdx.x; c < p.d; c += 1024) {
    const float e = to_f32(x[c]) - mean;
    q = fmaf(e, e, q);
  }
  const float var = group_sum2<32>(q, 0.f, red[1], wig).x * inv_d;
  const float rstd = 1.f / sqrtf(var + p.eps);
  for (int c = threadIdx.x; c < p.d; c += 1024) {
    float w, b;
    load_param<T, 1>(p.weight, p.param_f32, 1.f, c, &w);
    load_param<T, 1>(p.bias, p.param_f32, 0.f, c, &b);
    y[c] = from_f32<T>(fmaf((to_f32(x[c]) - mean) * rstd, w, b));
  }
  if (threadIdx.x == 0 && p.mean) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
}

// Partials of the column sums: [blocks][2][d] fp32, dw first.
template <typename T, int VEC, int W, int NV>
__global__ void __launch_bounds__(threads_of(W)) layer_norm_backward_kernel(LayerNormBwdParams p) {
  constexpr int G = 32 * W, ROWS = threads_of(W) / G;
  __shared__ float2 red[2][W];
  extern __shared__ float part[];  // W = 1: [ROWS][2 d]
  const int t = threadIdx.x % G, wig = t >> 5, grp = threadIdx.x / G;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  const float inv_d = 1.f / (float)p.d;
  float sw[NV][VEC], sb[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) sw[i][j] = sb[i][j] = 0.f;

  RawVec<T, VEC> rx[NV], rd[NV];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * VEC;
      if (c < p.d) {
        rx[i].load(x + row * p.x_stride + c);
        rd[i].load(dy + row * p.dy_stride + c);
      } else {
        rx[i].clear();
        rd[i].clear();
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + grp;
  if (row < p.rows) fetch(row);
  int flip = 0;
  // W > 1: all threads of the block share the row, so the barriers inside are met by all
  for (; row < p.rows; row += step) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    float h[NV][VEC], g[NV][VEC];
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * VEC;
      rx[i].unpack(h[i]);
      rd[i].unpack(g[i]);
      if (c < p.d) {
        float w[VEC];
        load_param<T, VEC>(p.weight, p.param_f32, 1.f, c, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          h[i][j] = (h[i][j] - mean) * rstd;
          sw[i][j] = fmaf(g[i][j], h[i][j], sw[i][j]);
          sb[i][j] += g[i][j];
          g[i][j] *= w[j];
          sg += g[i][j];
          sgh = fmaf(g[i][j], h[i][j], sgh);
        }
      }
    }
    if (row + step < p.rows) fetch(row + step);
    const float2 s = group_sum2<W>(sg, sgh, red[flip], wig);
    flip ^= 1;
    if (p.dx) {
      const float mg = s.x * inv_d, mgh = s.y * inv_d;
      T* dx = static_cast<T*>(p.dx) + row * p.d;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if (c < p.d) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[i][j] = rstd * (g[i][j] - mg - h[i][j] * mgh);
          store_vec<T, VEC>(dx + c, g[i]);
        }
      }
    }
  }
  if (!p.partials) return;
  float* out = p.partials + (size_t)blockIdx.x * 2 * p.d;
  if constexpr (W == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (i * G + t) * VEC + j;
        if (c < p.d) {
          part[(size_t)grp * 2 * p.d + c] = sw[i][j];
          part[(size_t)grp * 2 * p.d + p.d + c] = sb[i][j];
        }
      }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.d; c += blockDim.x) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) s += part[(size_t)r * 2 * p.d + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (i * G + t) * VEC + j;
        if (c < p.d) {
          out[c] = sw[i][j];
          out[p.d + c] = sb[i][j];
        }
      }
  }
}

// Rows too long for registers: dx by one block a row in two passes ...
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_backward_long_kernel(LayerNormBwdParams p) {
  __shared__ float2 red[32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
  T* dx = static_cast<T*>(p.dx) + row * p.d;
  const float mean = p.mean[row], rstd = p.rstd[row], inv_d = 1.f / (float)p.d;
  float sg = 0.f, sgh = 0.f;
  for (int c = threadIdx.x; c < p.d; c += 1024) {
    float w;
    load_param<T, 1>(p.weight, p.param_f32, 1.f, c, &w);
    const float g = to_f32(dy[c]) * w;
    sg += g;
    sgh = fmaf(g, (to_f32(x[c]) - mean) * rstd, sgh);
  }
  const float2 s = group_sum2<32>(sg, sgh, red, threadIdx.x >> 5);
  for (int c = threadIdx.x; c < p.d; c += 1024) {
    float w;
    load_param<T, 1>(p.weight, p.param_f32, 1.f, c, &w);
    const float g = to_f32(dy[c]) * w;
    dx[c] = from_f32<T>(rstd * (g - s.x * inv_d - (to_f32(x[c]) - mean) * rstd * (s.y * inv_d)));
  }
}
// ... and the column sums by threads that each walk one column of a share of the rows.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(LayerNormBwdParams p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.d) return;
  const T* x = static_cast<const T*>(p.x) + c;
  const T* dy = static_cast<const T*>(p.dy) + c;
  float sw = 0.f, sb = 0.f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float g = to_f32(dy[row * p.dy_stride]);
    sw = fmaf(g, (to_f32(x[row * p.x_stride]) - p.mean[row]) * p.rstd[row], sw);
    sb += g;
  }
  float* out = p.partials + (size_t)blockIdx.y * 2 * p.d;
  out[c] = sw;
  out[p.d + c] = sb;
}

// Group shapes.  A thread holds at most 16 elements of a row (the backward keeps four
// fp32 values for each, 64 of the 128 registers that 512 threads leave a thread): one
// warp a row up to 512 columns, then the fewest of 4, 8 or 16 warps that hold it, and
// the long form above 8192 columns.
struct Shape {
  int warps, nv;  // nv = 0: the long form
};
Shape shape_of(int64_t d, int vec) {
  const int64_t per = 16 / vec;  // vectors a thread
  auto nv_for = [&](int w) {
    const int64_t n = (d + 32 * w * vec - 1) / (32 * w * vec);
    int64_t v = 1;
    while (v < n) v *= 2;
    return v;
  };
  for (int w : {1, 4, 8, 16})
    if (nv_for(w) <= per) return {w, (int)nv_for(w)};
  return {0, 0};
}
constexpr int kLongRowShares = 64;

// W = 1 shares its column sums in shared memory: 8 rows x 2 x 512 floats = 32 KB at most.
int backward_blocks(int64_t rows, const Shape& s) {
  const int64_t groups = s.warps == 1 ? (rows + 7) / 8 : rows;
  // resident blocks an SM: 2048 threads' worth at about 64 registers each is half of that
  const int per_sm = s.warps == 1 ? 4 : s.warps == 4 ? 8 : s.warps == 8 ? 4 : 2;
  const int64_t most = kSms * per_sm;
  return (int)(groups < most ? groups : most);
}

// Elements a load: 16 bytes where every row and parameter starts on 16 bytes, else 1.
template <typename T>
int vec_of(int64_t d, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  const int vec = 16 / (int)sizeof(T);
  if (d % vec) return 1;
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % 16) return 1;
  for (int64_t s : strides)
    if ((s * (int64_t)sizeof(T)) % 16) return 1;
  return vec;
}

#define WF_LN_NV(KERNEL, VEC_, W_, ...)                                                    \
  switch (s.nv) {                                                                          \
    case 1: KERNEL<T, VEC_, W_, 1> __VA_ARGS__; break;                                     \
    case 2: KERNEL<T, VEC_, W_, 2> __VA_ARGS__; break;                                     \
    default:                                                                               \
      if constexpr (16 / VEC_ >= 4) {                                                      \
        if (s.nv == 4) { KERNEL<T, VEC_, W_, 4> __VA_ARGS__; break; }                      \
        if constexpr (16 / VEC_ >= 16) {                                                   \
          if (s.nv == 8) { KERNEL<T, VEC_, W_, 8> __VA_ARGS__; break; }                    \
          KERNEL<T, VEC_, W_, 16> __VA_ARGS__;                                             \
        }                                                                                  \
      }                                                                                    \
  }
#define WF_LN_W(KERNEL, VEC_, ...)                                   \
  switch (s.warps) {                                                 \
    case 1: WF_LN_NV(KERNEL, VEC_, 1, __VA_ARGS__) break;            \
    case 4: WF_LN_NV(KERNEL, VEC_, 4, __VA_ARGS__) break;            \
    case 8: WF_LN_NV(KERNEL, VEC_, 8, __VA_ARGS__) break;            \
    default: WF_LN_NV(KERNEL, VEC_, 16, __VA_ARGS__) break;          \
  }

template <typename T>
int launch_fwd(const LayerNormParams& p, cudaStream_t stream) {
  const int vec = vec_of<T>(p.d, {p.x, p.y, p.weight, p.bias}, {p.x_stride, p.y_stride});
  const Shape s = shape_of(p.d, vec);
  if (s.nv == 0) {
    layer_norm_long_kernel<T><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
    return (int)cudaGetLastError();
  }
  const unsigned grid = (unsigned)(s.warps == 1 ? (p.rows + 7) / 8 : p.rows);
  const int threads = threads_of(s.warps);
  if (vec == 1) {
    WF_LN_W(layer_norm_kernel, 1, <<<grid, threads, 0, stream>>>(p))
  } else {
    constexpr int V = 16 / (int)sizeof(T);
    WF_LN_W(layer_norm_kernel, V, <<<grid, threads, 0, stream>>>(p))
  }
  return (int)cudaGetLastError();
}

template <typename T>
int launch_bwd(LayerNormBwdParams p, cudaStream_t stream) {
  const int vec = vec_of<T>(p.d, {p.x, p.dy, p.dx, p.weight}, {p.x_stride, p.dy_stride});
  const Shape s = shape_of(p.d, vec);
  int blocks;
  if (s.nv == 0) {
    blocks = (int)(p.rows < kLongRowShares ? p.rows : kLongRowShares);
    if (p.dx) layer_norm_backward_long_kernel<T><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
    if (p.partials)
      layer_norm_columns_kernel<T><<<dim3((unsigned)((p.d + 255) / 256), (unsigned)blocks), 256, 0, stream>>>(p);
  } else {
    blocks = backward_blocks(p.rows, s);
    const int threads = threads_of(s.warps);
    const size_t smem = s.warps == 1 && p.partials ? (size_t)8 * 2 * p.d * 4 : 0;
    if (vec == 1) {
      WF_LN_W(layer_norm_backward_kernel, 1, <<<blocks, threads, smem, stream>>>(p))
    } else {
      constexpr int V = 16 / (int)sizeof(T);
      WF_LN_W(layer_norm_backward_kernel, V, <<<blocks, threads, smem, stream>>>(p))
    }
  }
  if (cudaError_t e = cudaGetLastError()) return (int)e;
  if (!p.partials) return 0;
  return (int)(p.param_f32 ? join_columns<float>(p.partials, blocks, 2 * (int64_t)p.d, p.d, p.dweight, p.dbias, stream)
                           : join_columns<T>(p.partials, blocks, 2 * (int64_t)p.d, p.d, p.dweight, p.dbias, stream));
}

}  // namespace

size_t layer_norm_backward_workspace_bytes(int64_t rows, int64_t d, int dtype) {
  // the block count of the vector or the scalar form, whichever has more
  size_t most = 0;
  for (int vec : {1, dtype == kF32 ? 4 : 8}) {
    const Shape s = shape_of(d, vec);
    const size_t blocks = s.nv == 0 ? (size_t)(rows < kLongRowShares ? rows : kLongRowShares)
                                    : (size_t)backward_blocks(rows, s);
    if (blocks > most) most = blocks;
  }
  return most * 2 * (size_t)d * sizeof(float);
}

int launch_layer_norm(const LayerNormParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_fwd<__nv_bfloat16>(p, stream);
  if (dtype == kF16) return launch_fwd<__half>(p, stream);
  return launch_fwd<float>(p, stream);
}

int launch_layer_norm_backward(const LayerNormBwdParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_bwd<__nv_bfloat16>(p, stream);
  if (dtype == kF16) return launch_bwd<__half>(p, stream);
  return launch_bwd<float>(p, stream);
}

}  // namespace wf

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
// means).  The mean is rounded once and x - mean is taken before rstd multiplies, so that the
// deviations of equal values are 0: x rstd - mean rstd leaves its rounding, 316 |mean| 2^-24
// at the usual eps, in each.  All statistics and sums are fp32; y, dx, dw and db are rounded once.
//
// Backward: groups walk rows with a stride of the grid and keep the column sums of
// their own columns in registers, with the next rows on their way to shared memory.
// The groups of a block add their sums in shared memory, each block writes one row of partials, and a
// second kernel adds the blocks' rows in a fixed order (no atomics: the same inputs
// give the same bits).
#include "wf_columns.cuh"
#include "wf_kernels.h"
#include "wf_pair.cuh"
#include "wf_rowio.cuh"

#include <algorithm>
#include <initializer_list>

namespace wf {
namespace {

// VEC parameters from column c: fp32 or of the activations' type.
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, bool f32, float absent, int64_t c, float* f) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = absent;
  } else if (f32) {
    const float* q = static_cast<const float*>(p) + c;
    if constexpr (VEC < 4) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = __ldg(q + j);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) Vec16<float>::unpack(ldg16(q + j), f + j);
    }
  } else {
    RawVec<T, VEC> raw;
    raw.load(static_cast<const T*>(p) + c);
    raw.unpack(f);
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

// sum / d: the product with 1 / d and what that leaves of the sum, which is 0 where the quotient
// is representable (a division's own instructions cost 32768 rows of 256 a tenth of their time).
__device__ __forceinline__ float mean_of(float sum, float d, float inv_d) {
  const float m = sum * inv_d;
  return fmaf(fmaf(-m, d, sum), inv_d, m);
}

// W warps a row; W = 1: eight rows a block at a time, otherwise one.
__host__ __device__ constexpr int threads_of(int W) { return W == 1 ? 256 : 32 * W; }

// Rows on their way: a thread's vectors of the next kAhead rows go to slots of its own in
// shared memory with asynchronous copies, so that a block has that many rows in flight
// whatever its registers hold, and no thread waits for another.  M matrices of NV vectors.
// (Single 16-bit elements cannot be copied so: the next row's wait in registers.)
constexpr int kAhead = 3;
template <typename T, int VEC, int NV, int M, int G, int THREADS>
struct RowRing {
  static constexpr int SIZE = VEC * (int)sizeof(T);
  static constexpr bool ASYNC = SIZE >= 4;
  static constexpr size_t bytes = ASYNC ? (size_t)kAhead * M * NV * THREADS * SIZE : 0;
  RawVec<T, VEC> raw[M][NV];
  uint32_t slots;  // of this thread
  int slot = 0;
  __device__ __forceinline__ explicit RowRing(void* smem)
      : slots((uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * SIZE) {}
  // Asks for this thread's part of a row (nothing past column d, nothing at all without a row).
  __device__ __forceinline__ void ask(const T* const (&row)[M], bool there, int t, int d) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if constexpr (ASYNC) {
          if (there && c < d) copy_async<SIZE>(slots + ((slot * M + m) * NV + i) * THREADS * SIZE, row[m] + c);
        } else {
          if (there && c < d) raw[m][i].load(row[m] + c);
          else raw[m][i].clear();
        }
      }
    if constexpr (ASYNC) {
      copy_async_commit();
      slot = slot == kAhead - 1 ? 0 : slot + 1;
    }
  }
  // The oldest row asked for, as fp32 (zeros past column d).
  __device__ __forceinline__ void get(float (&f)[M][NV][VEC], int t, int d) {
    if constexpr (ASYNC) copy_async_wait<kAhead - 1>();
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (ASYNC) {
          raw[m][i].clear();
          if ((i * G + t) * VEC < d) {
            const uint32_t at = slots + ((slot * M + m) * NV + i) * THREADS * SIZE;
            if constexpr (SIZE == 16) {
              uint4& v = raw[m][i].v;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                           : "r"(at)
                           : "memory");
            } else {
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(*reinterpret_cast<uint32_t*>(&raw[m][i].v)) : "r"(at) : "memory");
            }
          }
        }
        raw[m][i].unpack(f[m][i]);
      }
  }
  static constexpr int ahead = ASYNC ? kAhead : 1;
};

// The forward has nothing to keep between rows: a group takes one row and is gone (a warp R
// of them side by side, so that more is in flight and a parameter is loaded once for R rows).
template <typename T, int VEC, int W, int NV, int R>
__global__ void __launch_bounds__(threads_of(W)) layer_norm_kernel(LayerNormParams p) {
  pdl_wait();
  static_assert(R == 1 || W == 1, "rows of a block share its barriers");
  constexpr int G = 32 * W;
  __shared__ float2 red[2][W];
  const int t = threadIdx.x % G, wig = t >> 5;
  const int64_t row0 = ((int64_t)blockIdx.x * (threads_of(W) / G) + threadIdx.x / G) * R;
  if (W == 1 && row0 >= p.rows) return;  // whole warps; W > 1 has one row a block, always in range
  const T* x = static_cast<const T*>(p.x) + row0 * p.x_stride;
  RawVec<T, VEC> raw[R][NV];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * VEC;
      if (c < p.d && (R == 1 || row0 + r < p.rows)) raw[r][i].load(x + r * p.x_stride + c);
      else raw[r][i].clear();
    }
  const float inv_d = 1.f / (float)p.d;
  float v[R][NV][VEC], mean[R], rstd[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[r][i].unpack(v[r][i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += v[r][i][j];
    }
    mean[r] = mean_of(group_sum2<W>(s, 0.f, red[0], wig).x, (float)p.d, inv_d);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * G + t) * VEC < p.d) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[r][i][j] -= mean[r];
          q = fmaf(v[r][i][j], v[r][i][j], q);
        }
      }
    }
    rstd[r] = 1.f / sqrtf(group_sum2<W>(q, 0.f, red[1], wig).x * inv_d + p.eps);
  }
  T* y = static_cast<T*>(p.y) + row0 * p.y_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * VEC;
    if (c < p.d) {
      float w[VEC], b[VEC];
      load_param<T, VEC>(p.weight, p.param_f32, 1.f, c, w);
      load_param<T, VEC>(p.bias, p.param_f32, 0.f, c, b);
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[r][i][j] = fmaf(v[r][i][j] * rstd[r], w[j], b[j]);
        if (R == 1 || row0 + r < p.rows) store_vec<T, VEC>(y + r * p.y_stride + c, v[r][i]);
      }
    }
  }
  if (t == 0 && p.mean) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (R == 1 || row0 + r < p.rows) {
        p.mean[row0 + r] = mean[r];
        p.rstd[row0 + r] = rstd[r];
      }
  }
}

// Rows too long for registers: one block a row, three passes over it (the second and
// third find it in L2).
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(LayerNormParams p) {
  pdl_wait();
  __shared__ float2 red[2][32];
  const int wig = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  T* y = static_cast<T*>(p.y) + row * p.y_stride;
  float s = 0.f;
  for (int c = threadIdx.x; c < p.d; c += 1024) s += to_f32(x[c]);
  const float inv_d = 1.f / (float)p.d;
  const float mean = mean_of(group_sum2<32>(s, 0.f, red[0], wig).x, (float)p.d, inv_d);
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
__global__ void __launch_bounds__(threads_of(W), W == 1 ? 2 : 16 / W) layer_norm_backward_kernel(LayerNormBwdParams p) {
  pdl_wait();
  constexpr int G = 32 * W, ROWS = threads_of(W) / G;
  __shared__ float2 red[2][W];
  extern __shared__ uint4 ring_smem[];
  RowRing<T, VEC, NV, 2, G, threads_of(W)> ring(ring_smem);
  const int t = threadIdx.x % G, wig = t >> 5, grp = threadIdx.x / G;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  const float inv_d = 1.f / (float)p.d;
  float sw[NV][VEC], sb[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) sw[i][j] = sb[i][j] = 0.f;

  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + grp;
  auto ask = [&](int64_t r) { ring.ask({x + r * p.x_stride, dy + r * p.dy_stride}, r < p.rows, t, p.d); };
#pragma unroll
  for (int i = 0; i < ring.ahead; ++i) ask(row + i * step);
  float mean = 0.f, rstd = 0.f;
  if (row < p.rows) {
    mean = p.mean[row];
    rstd = p.rstd[row];
  }
  int flip = 0;
  // W > 1: all threads of the block share the row, so the barriers inside are met by all
  for (; row < p.rows; row += step) {
    // columns past d hold x = dy = 0: they add (h of 0) times 0 to every sum
    const float minus_mean = -mean, scale = rstd;
    float f[2][NV][VEC];
    ring.get(f, t, p.d);
    float(&h)[NV][VEC] = f[0];
    float(&g)[NV][VEC] = f[1];
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * VEC;
      float w[VEC];
      load_param<T, VEC>(c < p.d ? p.weight : nullptr, p.param_f32, 1.f, c, w);
      if constexpr (VEC == 1) {
        h[i][0] = (h[i][0] + minus_mean) * scale;
        sw[i][0] = fmaf(g[i][0], h[i][0], sw[i][0]);
        sb[i][0] += g[i][0];
        g[i][0] *= w[0];
        sg += g[i][0];
        sgh = fmaf(g[i][0], h[i][0], sgh);
      } else {
        Pair pg(0.f), pgh(0.f);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          const Pair y(g[i][j], g[i][j + 1]);
          const Pair x2 = mul2(add2(Pair(h[i][j], h[i][j + 1]), Pair(minus_mean)), Pair(scale));
          x2.get(h[i][j], h[i][j + 1]);
          fma2(y, x2, Pair(sw[i][j], sw[i][j + 1])).get(sw[i][j], sw[i][j + 1]);
          add2(y, Pair(sb[i][j], sb[i][j + 1])).get(sb[i][j], sb[i][j + 1]);
          const Pair yw = mul2(y, Pair(w[j], w[j + 1]));
          yw.get(g[i][j], g[i][j + 1]);
          pg = add2(pg, yw);
          pgh = fma2(yw, x2, pgh);
        }
        float a, b;
        pg.get(a, b);
        sg += a + b;
        pgh.get(a, b);
        sgh += a + b;
      }
    }
    ask(row + ring.ahead * step);
    if (row + step < p.rows) {
      mean = p.mean[row + step];
      rstd = p.rstd[row + step];
    }
    const float2 s = group_sum2<W>(sg, sgh, red[flip], wig);
    flip ^= 1;
    if (p.dx) {
      // dx = r g - r mean(g) - (r mean(g h)) h
      const float a = -scale * (s.x * inv_d), b = -scale * (s.y * inv_d);
      T* dx = static_cast<T*>(p.dx) + row * p.d;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * G + t) * VEC;
        if constexpr (VEC == 1) {
          g[i][0] = fmaf(g[i][0], scale, fmaf(h[i][0], b, a));
        } else {
#pragma unroll
          for (int j = 0; j < VEC; j += 2)
            fma2(Pair(g[i][j], g[i][j + 1]), Pair(scale), fma2(Pair(h[i][j], h[i][j + 1]), Pair(b), Pair(a)))
                .get(g[i][j], g[i][j + 1]);
        }
        if (c < p.d) store_vec<T, VEC>(dx + c, g[i]);
      }
    }
  }
  if (!p.partials) return;
  float* out = p.partials + (size_t)blockIdx.x * 2 * p.d;
  if constexpr (W == 1) {
    float* part = reinterpret_cast<float*>(ring_smem);  // [ROWS][2 d], in the ring's place
    if constexpr (ring.ASYNC) copy_async_wait<0>();
    __syncthreads();
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
  pdl_wait();
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
  pdl_wait();
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

// Group shapes: the fewest warps that hold a row with at most `most` elements a thread, up
// to 16; nv = 0 is the long form.  The forward keeps one fp32 value an element: 32, so one
// warp up to 1024 columns.  The backward keeps up to four (its sums, and what it has
// loaded): 16 elements, of the 128 registers that 512 threads leave a thread.
struct Shape {
  int warps, nv;
};
Shape shape_of(int64_t d, int vec, int most) {
  for (int w : {1, 4, 8, 16}) {
    const int64_t n = (d + 32 * w * vec - 1) / (32 * w * vec);
    int64_t v = 1;
    while (v < n) v *= 2;
    // single elements are many loads: spread them over more warps first
    if (v * vec <= (vec == 1 && w < 16 ? 8 : most)) return {w, (int)v};
  }
  return {0, 0};
}
constexpr int kForwardElements = 32, kBackwardElements = 16;
constexpr int kLongRowShares = 64;

// Blocks of the backward: what is resident at once (128 registers a thread), but eight rows a
// group at least, since each block costs a row of partial sums.
int backward_blocks(int64_t rows, const Shape& s) {
  const int64_t groups = s.warps == 1 ? (rows + 63) / 64 : (rows + 7) / 8;
  const int64_t most = (int64_t)kSms * (s.warps == 1 ? 2 : 16 / s.warps);
  return (int)(groups < most ? groups : most);
}

// Elements a load: 16 bytes where every row and parameter starts on 16 bytes, two 16-bit
// ones where they start on 4, else 1.
template <typename T>
int vec_of(int64_t d, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides) {
  for (int vec : {16 / (int)sizeof(T), 2}) {
    const int64_t bytes = vec * (int64_t)sizeof(T);
    if (bytes != 16 && bytes != 4) continue;
    bool fits = d % vec == 0;
    for (const void* q : ptrs) fits = fits && reinterpret_cast<uintptr_t>(q) % bytes == 0;
    for (int64_t s : strides) fits = fits && s % vec == 0;
    if (fits) return vec;
  }
  return 1;
}

// A kernel's instance for (T, VEC, W, NV) with its ring's bytes, and at least `smem`.
template <typename P>
int launch_rows(void (*kern)(P), int blocks, int threads, size_t smem, const P& p, cudaStream_t stream) {
  if (smem > 40 * 1024)  // 48 KB without asking, static shared memory included
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem))
      return (int)e;
  return (int)launch_pdl(kern, dim3(blocks), dim3(threads), smem, stream, p);
}
template <bool BACKWARD, typename T, int VEC, int W, int NV, typename P>
int launch_shape(int blocks, const P& p, cudaStream_t stream) {
  if constexpr (BACKWARD) {
    if constexpr (NV * VEC <= kBackwardElements) {
      size_t smem = RowRing<T, VEC, NV, 2, 32 * W, threads_of(W)>::bytes;
      if (W == 1 && p.partials) smem = std::max(smem, (size_t)8 * 2 * p.d * sizeof(float));
      return launch_rows<P>(layer_norm_backward_kernel<T, VEC, W, NV>, blocks, threads_of(W), smem, p, stream);
    }
  } else if constexpr (NV * VEC <= kForwardElements) {
    const int64_t groups = threads_of(W) / (32 * W);
    // several rows a warp once that still leaves every SM two blocks
    constexpr int R = W == 1 && NV * VEC <= 16 ? (NV * VEC <= 8 ? 4 : 2) : 1;
    if (R > 1 && p.rows >= groups * R * 2 * kSms)
      return launch_rows<P>(layer_norm_kernel<T, VEC, W, NV, R>, (int)((p.rows + groups * R - 1) / (groups * R)),
                            threads_of(W), 0, p, stream);
    return launch_rows<P>(layer_norm_kernel<T, VEC, W, NV, 1>, (int)((p.rows + groups - 1) / groups), threads_of(W), 0,
                          p, stream);
  }
  return -1;
}
template <bool BACKWARD, typename T, int VEC, int W, typename P>
int launch_warps(int nv, int blocks, const P& p, cudaStream_t stream) {
  switch (nv) {
    case 1: return launch_shape<BACKWARD, T, VEC, W, 1>(blocks, p, stream);
    case 2: return launch_shape<BACKWARD, T, VEC, W, 2>(blocks, p, stream);
    case 4: return launch_shape<BACKWARD, T, VEC, W, 4>(blocks, p, stream);
    case 8: return launch_shape<BACKWARD, T, VEC, W, 8>(blocks, p, stream);
    case 16: return launch_shape<BACKWARD, T, VEC, W, 16>(blocks, p, stream);
    default: return launch_shape<BACKWARD, T, VEC, W, 32>(blocks, p, stream);
  }
}
template <bool BACKWARD, typename T, int VEC, typename P>
int launch_vec(const Shape& s, int blocks, const P& p, cudaStream_t stream) {
  switch (s.warps) {
    case 1: return launch_warps<BACKWARD, T, VEC, 1>(s.nv, blocks, p, stream);
    case 4: return launch_warps<BACKWARD, T, VEC, 4>(s.nv, blocks, p, stream);
    case 8: return launch_warps<BACKWARD, T, VEC, 8>(s.nv, blocks, p, stream);
    default: return launch_warps<BACKWARD, T, VEC, 16>(s.nv, blocks, p, stream);
  }
}

template <bool BACKWARD, typename T, typename P>
int launch_any(int vec, const Shape& s, int blocks, const P& p, cudaStream_t stream) {
  if (vec == 1) return launch_vec<BACKWARD, T, 1>(s, blocks, p, stream);
  if constexpr (sizeof(T) == 2)
    if (vec == 2) return launch_vec<BACKWARD, T, 2>(s, blocks, p, stream);
  return launch_vec<BACKWARD, T, 16 / (int)sizeof(T)>(s, blocks, p, stream);
}

template <typename T>
int launch_fwd(const LayerNormParams& p, cudaStream_t stream) {
  const int vec = vec_of<T>(p.d, {p.x, p.y, p.weight, p.bias}, {p.x_stride, p.y_stride});
  const Shape s = shape_of(p.d, vec, kForwardElements);
  if (s.nv == 0) {
    layer_norm_long_kernel<T><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
    return (int)cudaGetLastError();
  }
  return launch_any<false, T>(vec, s, 0, p, stream);
}

template <typename T>
int launch_bwd(LayerNormBwdParams p, cudaStream_t stream) {
  const int vec = vec_of<T>(p.d, {p.x, p.dy, p.dx, p.weight}, {p.x_stride, p.dy_stride});
  const Shape s = shape_of(p.d, vec, kBackwardElements);
  int blocks;
  if (s.nv == 0) {
    blocks = (int)(p.rows < kLongRowShares ? p.rows : kLongRowShares);
    if (p.dx) layer_norm_backward_long_kernel<T><<<(unsigned)p.rows, 1024, 0, stream>>>(p);
    if (p.partials)
      layer_norm_columns_kernel<T><<<dim3((unsigned)((p.d + 255) / 256), (unsigned)blocks), 256, 0, stream>>>(p);
  } else {
    blocks = backward_blocks(p.rows, s);
    if (int rc = launch_any<true, T>(vec, s, blocks, p, stream)) return rc;
  }
  if (cudaError_t e = cudaGetLastError()) return (int)e;
  if (!p.partials) return 0;
  return (int)(p.param_f32 ? join_columns<float>(p.partials, blocks, 2 * (int64_t)p.d, p.d, p.dweight, p.dbias, stream)
                           : join_columns<T>(p.partials, blocks, 2 * (int64_t)p.d, p.d, p.dweight, p.dbias, stream));
}

}  // namespace

size_t layer_norm_backward_workspace_bytes(int64_t rows, int64_t d, int dtype) {
  // the block count of whichever load width has the most
  size_t most = 0;
  for (int vec : {1, 2, 4, 8}) {
    const Shape s = shape_of(d, vec, kBackwardElements);
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

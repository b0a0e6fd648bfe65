// Linear layer over few rows (new tokens of a batch): y = act(x W^T + b) + residual without a
// tile of 128 rows.
//
// Bound by W's bytes: each is used M times only.  A block's warps take columns of y and parts
// of the depth; a lane's 16-byte pieces of several rows of W are on their way together, and
// the parts of the depth are added through shared memory in order before the block applies
// the epilogue: one launch, where the tiled product splits the depth over the SMs and joins
// it in a second kernel.  Products and sums are fp32.
//
// 16-bit rows on 16 bytes, M <= 16: warp-level matrix instructions (16 columns of y by 8 rows
// of x), whose depth index is free to be any order as long as W and x agree: a lane's 16
// contiguous bytes of a W row serve two instructions, so that operands go from memory to
// registers without a shuffle or a shared-memory pass.  (The fifth-generation instructions
// read shared memory; staging W there would add a pass over what is used once.)
// Other rows, M <= 8: fused multiply-adds, 8 columns a warp (4 from three rows on); the sums
// of a lane are halved lane by lane (62 exchanges for 64 sums, not 320).
//
// 8 x 4096 x 4096 takes 8.3 us in fp16 (33.5 MB at 4.0 TB/s; 8192 x 8192 5.0 TB/s) and 29 us
// in fp32.  The next step's pieces of W are asked for before a step is computed (10.1 and 40 us
// without), and two blocks fit an SM (fp32's 8 rows then spill some registers: 40 us at one
// block, 62 us at three).
#include "wf_activation.cuh"
#include "wf_linear_few.h"
#include "wf_rowio.cuh"

#include <type_traits>

namespace wf {
namespace {

constexpr int kWarps = 8;  // of a block

// What becomes of a finished sum.
template <typename T>
__device__ __forceinline__ void put(const LinearParams& p, int64_t m, int64_t n, float v) {
  if (p.bias) v += to_f32(static_cast<const T*>(p.bias)[n]);
  using Z = typename Kept<T>::type;
  if (p.z) static_cast<Z*>(p.z)[m * ((p.N + 7) / 8 * 8) + n] = from_f32<Z>(kept_z(p.act, v));
  float a[2] = {v, 0.f};
  activate_all<T, 2>(p.act, a);
  if (p.residual) a[0] += to_f32(static_cast<const T*>(p.residual)[m * p.r_stride + n]);
  static_cast<T*>(p.y)[m * p.N + n] = from_f32<T>(a[0]);
}

// ---------------------------------------------------------------- matrix instructions
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Lane l: rows l / 4 and l / 4 + 8 of the warp's 16 columns of y (rows of W), row l / 4 of
// each 8 of x, and 8 elements of the depth from 8 (l % 4) on in every 32.
constexpr int kMmaCols = 16, kAhead = 4;
template <typename T, int TILES>
__global__ void __launch_bounds__(32 * kWarps, TILES == 1 ? 2 : 0) linear_few_mma_kernel(LinearParams p, int parts) {
  __shared__ float sums[kWarps][kMmaCols][8 * TILES + 1];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % parts, group = warp / parts, groups = kWarps / parts;
  const int64_t n0 = ((int64_t)blockIdx.x * groups + group) * kMmaCols;
  const int r = lane / 4, k_lane = lane % 4 * 8;
  const int M = (int)p.M;
  const T* w = static_cast<const T*>(p.w) + (n0 + r) * p.w_stride;
  const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
  const bool live0 = n0 + r < p.N, live1 = n0 + r + 8 < p.N;
  float d[TILES][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // kAhead steps of 32 of the depth are under way: a step's registers take the loads of the
  // same step of the part's next piece as soon as the instructions have read them
  uint4 a[kAhead][2], b[kAhead][TILES];
  const int64_t stride = (int64_t)parts * 32 * kAhead;
  auto load = [&](int i, int64_t k) {  // p.K is a multiple of 8: a piece is there or not
    const bool there = k < p.K;
    a[i][0] = there && live0 ? ldg16(w + k) : zero;
    a[i][1] = there && live1 ? ldg16(w + 8 * p.w_stride + k) : zero;
#pragma unroll
    for (int t = 0; t < TILES; ++t) b[i][t] = there && r + 8 * t < M ? ldg16(x + 8 * t * p.x_stride + k) : zero;
  };
  int64_t k = (int64_t)part * 32 * kAhead + k_lane;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(i, k + 32 * i);
  // The instructions' own adds round towards 0, 2^-24 of the sum each.  Up to 8 rows every
  // iteration's 128 of depth is summed apart and added with rounding: z's error at a depth of 4096
  // falls from 6.5e-7 to 2.0e-7 (an fp32 product's: 4.2e-7) in the same time.  The 16-row form has
  // no registers for it (10.0 -> 11.3 us at 4096 x 4096).
  constexpr bool APART = TILES == 1;
  for (; k - k_lane < p.K; k += stride) {
    float apart[4] = {};
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        float(&to)[4] = APART ? apart : d[t];
        mma_16x8x16<T>(to, a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y, b[i][t].x, b[i][t].y);
        mma_16x8x16<T>(to, a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w, b[i][t].z, b[i][t].w);
      }
      load(i, k + stride + 32 * i);
    }
    if constexpr (APART)
#pragma unroll
      for (int j = 0; j < 4; ++j) d[0][j] += apart[j];
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[warp][r + 8 * (j / 2)][8 * t + lane % 4 * 2 + j % 2] = d[t][j];
  __syncthreads();
  for (int i = threadIdx.x; i < groups * kMmaCols * M; i += 32 * kWarps) {
    // consecutive threads take consecutive columns
    const int c = i % kMmaCols, g = i / kMmaCols % groups, m = i / (kMmaCols * groups);
    const int64_t n = ((int64_t)blockIdx.x * groups + g) * kMmaCols + c;
    if (n >= p.N) continue;
    float v = 0.f;
    for (int q = 0; q < parts; ++q) v += sums[g * parts + q][c][m];
    put<T>(p, m, n, v);
  }
}

// ---------------------------------------------------------------- multiply-adds

// Sums v[0 .. N) over the warp: afterwards lane l's v[i] is the sum of value
// i + (N / 32) * (the bits of l in the order of the halvings).
template <int N, int O>
__device__ __forceinline__ void halve(float* v, int lane) {
  if constexpr (O > 0) {
    if constexpr (N > 1) {
      const bool upper = lane & O;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float send = upper ? v[i] : v[i + N / 2], keep = upper ? v[i + N / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, O);
      }
      halve<N / 2, O / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], O);
      halve<1, O / 2>(v, lane);
    }
  }
}

// VEC elements a lane and load; MB >= M rows; `parts` warps share a group of columns.
template <typename T, int VEC, int MB, int kCols>
__global__ void __launch_bounds__(32 * kWarps, 2) linear_few_kernel(LinearParams p, int parts) {
  constexpr int SUMS = MB * kCols;
  __shared__ float sums[kWarps][SUMS];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % parts, group = warp / parts, groups = kWarps / parts;
  const int64_t n0 = ((int64_t)blockIdx.x * groups + group) * kCols;
  const int M = (int)p.M;
  const T* w = static_cast<const T*>(p.w);
  const T* x = static_cast<const T*>(p.x);
  float acc[SUMS];
#pragma unroll
  for (int i = 0; i < SUMS; ++i) acc[i] = 0.f;
  // W's vectors of a step of the depth; x's come from the caches
  auto fetch = [&](auto& rw, int64_t k) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      if (n0 + c < p.N) rw[c].load(w + (n0 + c) * p.w_stride + k);
      else rw[c].clear();
    }
  };
  auto multiply = [&](auto& rw, int64_t k, auto refill) {
    constexpr int V = sizeof(rw[0]) / sizeof(T);
    float fw[kCols][V];
    RawVec<T, V> rx[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      if (m < M) rx[m].load(x + m * p.x_stride + k);
      else rx[m].clear();
    }
#pragma unroll
    for (int c = 0; c < kCols; ++c) rw[c].unpack(fw[c]);
    refill();
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      float fx[V];
      rx[m].unpack(fx);
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        float& a = acc[m * kCols + c];
        if constexpr (V == 1) {
          a = fmaf(fw[c][0], fx[0], a);
        } else {
          Pair q(a, 0.f);
#pragma unroll
          for (int j = 0; j < V; j += 2) q = fma2(Pair(fw[c][j], fw[c][j + 1]), Pair(fx[j], fx[j + 1]), q);
          float lo, hi;
          q.get(lo, hi);
          a = lo + hi;
        }
      }
    }
  };
  // whole vectors of the depth first, kSteps of them on their way, then its end by elements
  const int64_t whole = p.K / VEC * VEC, step = (int64_t)parts * 32 * VEC;
  if (n0 < p.N) {
    constexpr int kSteps = MB == 4 ? 2 : 1;
    RawVec<T, VEC> rw[kSteps][kCols];
    int64_t k = (int64_t)(part * 32 + lane) * VEC;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      if (k + i * step < whole) fetch(rw[i], k + i * step);
    while (k < whole) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i, k += step) {
        if (k >= whole) break;
        multiply(rw[i], k, [&] {
          if (k + kSteps * step < whole) fetch(rw[i], k + kSteps * step);
        });
      }
    }
    const int64_t last = whole + lane;
    if (part == parts - 1 && last < p.K) {
      RawVec<T, 1> one[kCols];
      fetch(one, last);
      multiply(one, last, [] {});
    }
  }
  halve<SUMS, 16>(acc, lane);
  if constexpr (SUMS >= 32) {
    // the first halving splits the values in two, the next in four, ...: bit 16 of the lane is
    // the highest bit of the value's index
#pragma unroll
    for (int i = 0; i < SUMS / 32; ++i) sums[warp][lane * (SUMS / 32) + i] = acc[i];
  } else {
    if (lane % (32 / SUMS) == 0) sums[warp][lane / (32 / SUMS)] = acc[0];
  }
  __syncthreads();
  // a thread an output
  for (int i = threadIdx.x; i < groups * SUMS; i += 32 * kWarps) {
    const int g = i / SUMS, s = i % SUMS, m = s / kCols;
    const int64_t n = ((int64_t)blockIdx.x * groups + g) * kCols + s % kCols;
    if (m >= M || n >= p.N) continue;
    float v = 0.f;
    for (int q = 0; q < parts; ++q) v += sums[g * parts + q][s];
    put<T>(p, m, n, v);
  }
}

// Warps that share a group of columns, each with a part of the depth: until the SMs have 16
// warps each, while a part is at least `least` deep.
int parts_of(int64_t groups, int64_t K, int64_t least) {
  int parts = 1;
  while (parts < kWarps && K >= 2 * parts * least && groups * parts < 16 * kSms) parts *= 2;
  return parts;
}

template <typename T, int VEC, int MB, int COLS>
int launch_rows(const LinearParams& p, cudaStream_t stream) {
  const int64_t groups = (p.N + COLS - 1) / COLS;
  const int parts = parts_of(groups, p.K, 64 * VEC);
  return (int)launch_pdl(linear_few_kernel<T, VEC, MB, COLS>, dim3((unsigned)((groups * parts + kWarps - 1) / kWarps)),
                         dim3(32 * kWarps), 0, stream, p, parts);
}
template <typename T, int VEC>
int launch_vec(const LinearParams& p, cudaStream_t stream) {
  if (p.M == 1) return launch_rows<T, VEC, 1, 8>(p, stream);
  if (p.M == 2) return launch_rows<T, VEC, 2, 8>(p, stream);
  if (p.M <= 4) return launch_rows<T, VEC, 4, 4>(p, stream);
  return launch_rows<T, VEC, 8, 4>(p, stream);
}

bool on_16_bytes(const LinearParams& p, int size) {
  return reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0 &&
         p.x_stride * size % 16 == 0 && p.w_stride * size % 16 == 0;
}
bool takes_mma(const LinearParams& p, int dtype) { return dtype != kF32 && p.K % 8 == 0 && on_16_bytes(p, 2); }

template <typename T>
int launch(const LinearParams& p, int dtype, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (takes_mma(p, dtype)) {
      const int64_t groups = (p.N + kMmaCols - 1) / kMmaCols;
      const int parts = parts_of(groups, p.K, 128);
      const unsigned grid = (unsigned)((groups * parts + kWarps - 1) / kWarps);
      return (int)launch_pdl(p.M <= 8 ? linear_few_mma_kernel<T, 1> : linear_few_mma_kernel<T, 2>, dim3(grid),
                             dim3(32 * kWarps), 0, stream, p, parts);
    }
  }
  return on_16_bytes(p, sizeof(T)) ? launch_vec<T, Vec16<T>::N>(p, stream) : launch_vec<T, 1>(p, stream);
}

}  // namespace

bool linear_few_takes(const LinearParams& p, int dtype) { return p.M <= (takes_mma(p, dtype) ? 16 : kFewRows); }

int launch_linear_few(const LinearParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch<__half>(p, dtype, stream);
  return launch<float>(p, dtype, stream);
}

}  // namespace wf

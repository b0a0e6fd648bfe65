// Tensor-core product with an epilogue: C = act(A B^T + bias) + residual.
//
// A persistent kernel, one block an SM, each block walking 128 x BN tiles of C.  Warp 8
// streams 64-deep slices of A and B into a ring of shared-memory stages with TMA; warp 9
// issues tcgen05.mma (128 x BN x 16, fp32 accumulators in TMEM) on them; warps 0-7 read a
// finished accumulator back, apply the epilogue and store.  Two accumulators alternate, so
// the epilogue of one tile runs under the products of the next.
//
// Operands are K-major or MN-major as they lie in memory: nothing is transposed.  The TMA
// box of a K-major operand is 64 of depth by all its rows; of an MN-major one, 64 rows of
// the product by 64 of depth, side by side.  Both use the 128-byte swizzle.
//
// fp32 operands come as three bf16 pieces (8 + 8 + 8 bits of mantissa).  The six products
// of pieces that reach fp32's last bit go into one accumulator, smallest first; the other
// three are below 2^-24 of the whole.  The tensor cores' own adds lose more with the
// length of a sum than fp32 rounding would, so every kChunk of depth the accumulator is
// added to fp32 registers and begun anew.
//
// Few tiles with a deep sum (a weight's gradient over many rows) are split along the
// depth: each part writes fp32 partials, and a second kernel adds them in order and
// applies the epilogue.
#include "wf_activation.cuh"
#include "wf_gemm.h"
#include "wf_rowio.cuh"
#include "wf_sm100.cuh"

#include <type_traits>

namespace wf {
namespace {

using namespace sm100;

constexpr int kBM = 128;
constexpr int kBK = 64;                 // depth of a stage: 128 bytes
constexpr int kChunk = 4;               // stages between additions to fp32 registers (three-piece form)
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (kEpilogueWarps + 2);
constexpr uint64_t kWaitNs = 1000000000ull;
constexpr int kMaxSplits = 32;

struct GemmParams {
  int M, N, tiles_n, units, splits, k_blocks, pieces;
  bool a_mn, b_mn, vec;
  GemmEpilogue out;
  float* partial;  // [splits][M][N] when splits > 1
  int32_t* status;
  uint32_t idesc;
};

template <int BN>
struct Layout {
  static constexpr uint32_t A_BYTES = kBM * 128, B_BYTES = BN * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr size_t off_bar = (size_t)STAGES * STAGE;
  static constexpr size_t off_misc = off_bar + 8 * (2 * STAGES + 5);
  static constexpr size_t smem = off_misc + 16 + 1024;
  static constexpr uint32_t TMEM_COLS = 2 * BN;
};

// Pieces of a and b multiplied in this order: (0,2) (1,1) (2,0) (0,1) (1,0) (0,0).
__device__ __forceinline__ int piece_a(int pair) { return (0x010210 >> (4 * pair)) & 3; }
__device__ __forceinline__ int piece_b(int pair) { return (0x001012 >> (4 * pair)) & 3; }

// Descriptor of an MN-major operand with the 128-byte swizzle: 64 rows of the product are
// 128 bytes, 8 of depth 1024 bytes apart, the next 64 rows 64 of depth further.
__device__ __forceinline__ uint64_t smem_desc_mnmajor(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3fff);
  d |= (uint64_t)((kBK * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

struct Ring {
  uint32_t stage = 0, phase = 0;
  template <int STAGES>
  __device__ __forceinline__ void next() {
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// Units of work: a tile and a share of the depth.
struct Unit {
  int m0, n0, kb0, kb1, split;
  __device__ __forceinline__ Unit(const GemmParams& p, int u, int BN) {
    split = u % p.splits;
    const int tile = u / p.splits;
    m0 = tile / p.tiles_n * kBM;
    n0 = tile % p.tiles_n * BN;
    kb0 = (int)((int64_t)p.k_blocks * split / p.splits);
    kb1 = (int)((int64_t)p.k_blocks * (split + 1) / p.splits);
  }
};

// 32 columns of one row: bias, activation, residual, stores.
template <typename T>
__device__ __forceinline__ void finish_row(const GemmEpilogue& o, int64_t m, int n, int N, bool vec, float* v) {
  constexpr int V = Vec16<T>::N;
  if (vec && n + 32 <= N) {
    if (o.bias) {
      const T* b = static_cast<const T*>(o.bias) + n;
#pragma unroll
      for (int j = 0; j < 32; j += V) {
        float f[V];
        Vec16<T>::unpack(ldg16(b + j), f);
#pragma unroll
        for (int i = 0; i < V; ++i) v[j + i] += f[i];
      }
    }
    if (o.z) {
      T* z = static_cast<T*>(o.z) + m * o.z_stride + n;
#pragma unroll
      for (int j = 0; j < 32; j += V) store_vec<T, V>(z + j, v + j);
    }
    activate_all<32>(o.act, v);
    if (o.residual) {
      const T* r = static_cast<const T*>(o.residual) + m * o.r_stride + n;
#pragma unroll
      for (int j = 0; j < 32; j += V) {
        float f[V];
        Vec16<T>::unpack(ldg16(r + j), f);
#pragma unroll
        for (int i = 0; i < V; ++i) v[j + i] += f[i];
      }
    }
    T* y = static_cast<T*>(o.y) + m * o.y_stride + n;
#pragma unroll
    for (int j = 0; j < 32; j += V) store_vec<T, V>(y + j, v + j);
    return;
  }
  if (o.bias) {
    const T* b = static_cast<const T*>(o.bias) + n;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n + j < N) v[j] += to_f32(b[j]);
  }
  if (o.z) {
    T* z = static_cast<T*>(o.z) + m * o.z_stride + n;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n + j < N) z[j] = from_f32<T>(v[j]);
  }
  activate_all<32>(o.act, v);
  if (o.residual) {
    const T* r = static_cast<const T*>(o.residual) + m * o.r_stride + n;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n + j < N) v[j] += to_f32(r[j]);
  }
  T* y = static_cast<T*>(o.y) + m * o.y_stride + n;
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (n + j < N) y[j] = from_f32<T>(v[j]);
}

template <typename T, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                const GemmParams p) {
  using L = Layout<BN>;
  constexpr bool PIECES = std::is_same<T, float>::value;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + L::off_bar);
  uint64_t* empty = full + L::STAGES;
  uint64_t* acc_full = empty + L::STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2]
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(base + L::off_misc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpilogueWarps);
    }
    mbar_init(drained, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_s, L::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_s;
  const int pairs = PIECES ? 6 : 1;
  uint32_t why = 0;

  if (warp == kEpilogueWarps) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      prefetch_tmap(&amap);
      prefetch_tmap(&bmap);
      Ring r;
      uint32_t issued = 0;
      for (int u = blockIdx.x; u < p.units && !why; u += gridDim.x) {
        const Unit w(p, u, BN);
        for (int c0 = w.kb0; c0 < w.kb1 && !why; c0 += PIECES ? kChunk : w.kb1 - w.kb0) {
          const int c1 = PIECES ? min(c0 + kChunk, w.kb1) : w.kb1;
          for (int pair = 0; pair < pairs && !why; ++pair) {
            const int pa = PIECES ? piece_a(pair) : 0, pb = PIECES ? piece_b(pair) : 0;
            for (int kb = c0; kb < c1; ++kb) {
              if (!mbar_wait(&empty[r.stage], r.phase ^ 1, kWaitNs)) { why = 4; break; }
              unsigned char* st = base + (size_t)r.stage * L::STAGE;
              uint64_t* bar = &full[r.stage];
              mbar_arrive_expect_tx(bar, L::STAGE);
              if (p.a_mn) {
#pragma unroll
                for (int i = 0; i < kBM / 64; ++i)
                  tma_load_3d(st + i * kBK * 128, &amap, bar, w.m0 + 64 * i, kb * kBK, pa);
              } else {
                tma_load_3d(st, &amap, bar, kb * kBK, w.m0, pa);
              }
              st += L::A_BYTES;
              if (p.b_mn) {
#pragma unroll
                for (int i = 0; i < BN / 64; ++i)
                  tma_load_3d(st + i * kBK * 128, &bmap, bar, w.n0 + 64 * i, kb * kBK, pb);
              } else {
                tma_load_3d(st, &bmap, bar, kb * kBK, w.n0, pb);
              }
              ++issued;
              r.next<L::STAGES>();
            }
          }
        }
      }
      // after a wait that gave up, loads may be in flight that no product will wait for
      if (why)
        for (uint32_t s = 0; s < (uint32_t)L::STAGES && s < issued; ++s) {
          const uint32_t last = (issued - 1 - s) / L::STAGES * L::STAGES + s;  // newest load of stage s
          mbar_wait(&full[s], (last / L::STAGES) & 1, kWaitNs);
        }
    }
  } else if (warp == kEpilogueWarps + 1) {
    // ------------------------------------------------------------ products
    if (lane == 0) {
      Ring r;
      uint32_t acc = 0, acc_phase = 0;
      const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;
      for (int u = blockIdx.x; u < p.units && !why; u += gridDim.x) {
        const Unit w(p, u, BN);
        for (int c0 = w.kb0; c0 < w.kb1 && !why; c0 += PIECES ? kChunk : w.kb1 - w.kb0) {
          const int c1 = PIECES ? min(c0 + kChunk, w.kb1) : w.kb1;
          if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1, kWaitNs)) { why = 8; break; }
          tc_fence_after();
          const uint32_t d = tmem + acc * BN;
          const int n = (c1 - c0) * pairs;
          for (int i = 0; i < n; ++i) {
            if (!mbar_wait(&full[r.stage], r.phase, kWaitNs)) { why = 16; break; }
            tc_fence_after();
            const uint32_t as = smem_u32(base + (size_t)r.stage * L::STAGE), bs = as + L::A_BYTES;
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              const uint32_t aa = as + k * a_step, bb = bs + k * b_step;
              mma_f16(d, p.a_mn ? smem_desc_mnmajor(aa) : smem_desc_kmajor(aa, 128),
                      p.b_mn ? smem_desc_mnmajor(bb) : smem_desc_kmajor(bb, 128), p.idesc, i > 0 || k > 0);
            }
            mma_commit(&empty[r.stage]);
            r.next<L::STAGES>();
          }
          mma_commit(&acc_full[acc]);
          acc ^= 1;
          acc_phase ^= acc == 0;
        }
      }
      mma_commit(drained);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    // warp w reads TMEM lanes 32 (w % 4) .. + 31 (a row a lane) and half w / 4 of the columns
    constexpr int COLS = BN / 2;
    const uint32_t lbase = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (warp >> 2) * COLS;
    uint32_t acc = 0, acc_phase = 0;
    for (int u = blockIdx.x; u < p.units; u += gridDim.x) {
      const Unit w(p, u, BN);
      const int64_t m = w.m0 + 32 * (warp & 3) + lane;
      const int n0 = w.n0 + (warp >> 2) * COLS;
      float sum[PIECES ? COLS : 1];
      if constexpr (PIECES) {
#pragma unroll
        for (int j = 0; j < COLS; ++j) sum[j] = 0.f;
      }
      for (int c0 = w.kb0; c0 < w.kb1; c0 += PIECES ? kChunk : w.kb1 - w.kb0) {
        const bool there = __all_sync(0xffffffffu, mbar_wait(&acc_full[acc], acc_phase, kWaitNs));
        if (!there) { why = 32; break; }
        tc_fence_after();
        const uint32_t src = lbase + acc * BN;
        if constexpr (PIECES) {
#pragma unroll
          for (int c = 0; c < COLS; c += 32) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(src + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[c + j] += __uint_as_float(r[j]);
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < COLS; c += 32) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(src + c, r);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
            const int n = n0 + c;
            if (m < p.M && n < p.N) {
              if (p.splits > 1) {
                GemmEpilogue o{};
                o.y = p.partial;
                o.y_stride = p.N;
                finish_row<float>(o, (int64_t)w.split * p.M + m, n, p.N, p.N % 4 == 0, v);
              } else {
                finish_row<T>(p.out, m, n, p.N, p.vec, v);
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
        acc ^= 1;
        acc_phase ^= acc == 0;
      }
      if (why) break;
      if constexpr (PIECES) {
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          const int n = n0 + c;
          if (m < p.M && n < p.N) {
            if (p.splits > 1) {
              GemmEpilogue o{};
              o.y = p.partial;
              o.y_stride = p.N;
              finish_row<float>(o, (int64_t)w.split * p.M + m, n, p.N, p.N % 4 == 0, sum + c);
            } else {
              finish_row<float>(p.out, m, n, p.N, p.vec, sum + c);
            }
          }
        }
      }
    }
  }
  __syncwarp();
  if (why && p.status && lane == 0) atomicOr(p.status, 2 | (int)why);
  // TMEM is given back once no product writes to it
  const bool done = mbar_wait(drained, 0, kWaitNs);
  if (!done && p.status && threadIdx.x == 0) atomicOr(p.status, 2 | 64);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
}

// Adds the parts of a split depth and applies the epilogue: a thread takes 4 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) gemm_join_kernel(const float* partial, int splits, int64_t M, int64_t N,
                                                        GemmEpilogue o) {
  const int64_t groups = (N + 3) / 4, total = M * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / groups, n = i % groups * 4;
    const int live = (int)min((int64_t)4, N - n);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float* q = partial + ((int64_t)s * M + m) * N + n;
      if (N % 4 == 0) {
        const float4 f = *reinterpret_cast<const float4*>(q);
        v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
      } else {
        for (int j = 0; j < live; ++j) v[j] += q[j];
      }
    }
    if (o.bias)
      for (int j = 0; j < live; ++j) v[j] += to_f32(static_cast<const T*>(o.bias)[n + j]);
    if (o.z)
      for (int j = 0; j < live; ++j) static_cast<T*>(o.z)[m * o.z_stride + n + j] = from_f32<T>(v[j]);
    activate_all<4>(o.act, v);
    if (o.residual)
      for (int j = 0; j < live; ++j) v[j] += to_f32(static_cast<const T*>(o.residual)[m * o.r_stride + n + j]);
    for (int j = 0; j < live; ++j) static_cast<T*>(o.y)[m * o.y_stride + n + j] = from_f32<T>(v[j]);
  }
}

typedef CUresult (*EncodeTiledFnG)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFnG encode_fn() {
  static const EncodeTiledFnG fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeTiledFnG>(ptr);
  }();
  return fn;
}

bool make_map(CUtensorMap* map, const GemmOperand& o, int pieces, int op_dtype, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)pieces};
  const int64_t piece = pieces > 1 ? o.piece_stride : o.pitch * o.rows;
  const cuuint64_t strides[2] = {(cuuint64_t)(o.pitch * 2), (cuuint64_t)(piece * 2)};
  const cuuint32_t box[3] = {64, (cuuint32_t)(o.mn_major ? kBK : box_rows), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  EncodeTiledFnG fn = encode_fn();
  return fn && fn(map, op_dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(o.ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tile width and depth shares.  The widest tile that still gives every SM one (wider tiles
// read A less often); below that, narrower tiles and then shares of at least kMinShare
// stages of depth until the SMs are busy.
struct Plan {
  int bn, tiles_n, tiles, splits, k_blocks;
};
constexpr int kMinShare = 4;
Plan plan_of(int64_t M, int64_t N, int64_t K, int pieces) {
  Plan p{};
  p.k_blocks = (int)((K + kBK - 1) / kBK);
  auto tiles = [&](int bn) { return (M + kBM - 1) / kBM * ((N + bn - 1) / bn); };
  p.bn = pieces == 1 && N > 128 && tiles(256) >= kSms ? 256 : N > 64 && tiles(128) * 2 >= kSms ? 128 : 64;
  p.tiles_n = (int)((N + p.bn - 1) / p.bn);
  const int64_t t = tiles(p.bn);
  p.tiles = (int)t;
  p.splits = 1;
  if (t * 2 <= kSms) {
    const int64_t most = p.k_blocks / kMinShare, fill = kSms / t;
    const int64_t s = most < fill ? most : fill;
    p.splits = (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
  }
  return p;
}

template <typename T, int BN>
int launch_tile(const GemmProblem& g, const Plan& plan, cudaStream_t stream) {
  using L = Layout<BN>;
  CUtensorMap amap, bmap;
  if (!make_map(&amap, g.a, g.pieces, g.op_dtype, kBM) || !make_map(&bmap, g.b, g.pieces, g.op_dtype, BN)) return -1;
  GemmParams p{};
  p.M = (int)g.M;
  p.N = (int)g.N;
  p.tiles_n = plan.tiles_n;
  p.splits = plan.splits;
  p.units = plan.tiles * plan.splits;
  p.k_blocks = plan.k_blocks;
  p.pieces = g.pieces;
  p.a_mn = g.a.mn_major;
  p.b_mn = g.b.mn_major;
  p.out = g.out;
  p.partial = static_cast<float*>(g.ws);
  p.status = g.status;
  p.idesc = idesc_f16(g.op_dtype == kBF16, kBM, BN) | (g.a.mn_major ? 1u << 15 : 0u) | (g.b.mn_major ? 1u << 16 : 0u);
  auto on16 = [](const void* q, int64_t stride) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
  };
  p.vec = on16(g.out.y, g.out.y_stride) && on16(g.out.z, g.out.z_stride) && on16(g.out.residual, g.out.r_stride) &&
          on16(g.out.bias, 0);
  auto kern = gemm_kernel<T, BN>;
  if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem))
    return (int)e;
  const int grid = p.units < kSms ? p.units : kSms;
  kern<<<grid, kThreads, L::smem, stream>>>(amap, bmap, p);
  if (cudaError_t e = cudaGetLastError()) return (int)e;
  if (plan.splits > 1) {
    const int64_t work = (g.M * ((g.N + 3) / 4) + 255) / 256;
    gemm_join_kernel<T><<<(unsigned)(work < 8 * kSms ? work : 8 * kSms), 256, 0, stream>>>(p.partial, plan.splits, g.M,
                                                                                        g.N, g.out);
    return (int)cudaGetLastError();
  }
  return 0;
}

template <typename T>
int launch_type(const GemmProblem& g, cudaStream_t stream) {
  const Plan plan = plan_of(g.M, g.N, g.K, g.pieces);
  if (plan.bn == 64) return launch_tile<T, 64>(g, plan, stream);
  if (plan.bn == 128) return launch_tile<T, 128>(g, plan, stream);
  if constexpr (!std::is_same<T, float>::value) return launch_tile<T, 256>(g, plan, stream);
  return -1;
}

}  // namespace

size_t gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, int pieces) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = plan_of(M, N, K, pieces);
  return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) : 0;
}

int launch_gemm(const GemmProblem& g, cudaStream_t stream) {
  if (g.M == 0 || g.N == 0) return 0;
  if (g.out_dtype == kBF16) return launch_type<__nv_bfloat16>(g, stream);
  if (g.out_dtype == kF16) return launch_type<__half>(g, stream);
  return launch_type<float>(g, stream);
}

}  // namespace wf

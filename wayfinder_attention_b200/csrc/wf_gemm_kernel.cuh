// Tensor-core product with an epilogue: C = act(A B^T + bias) + residual.
//
// A persistent kernel, one block an SM.  CG = 2: two blocks of a cluster work on a
// 256 x BN tile together, each loading its 128 rows of A and its half of B's rows and
// keeping its 128 rows of the accumulator; the leader issues tcgen05.mma.cta_group::2 for
// both, so each B element is read from L2 once for 256 rows.  CG = 1: 128 x BN tiles.
//
// Warp 16 streams 64-deep slices of A and B into a ring of shared-memory stages with TMA;
// warp 17 issues the products (fp32 accumulators in TMEM) on them; warps 0-15 read a
// finished accumulator back, apply the epilogue and store.  Two accumulators alternate, so
// the epilogue of one tile runs under the products of the next.
//
// Operands are K-major or MN-major as they lie in memory: nothing is transposed.  The TMA
// box of a K-major operand is 64 of depth by all its rows; of an MN-major one, 64 rows of
// the product by 64 of depth, side by side.  Both use the 128-byte swizzle.
//
// fp32 operands come as three bf16 pieces (8 + 8 + 8 bits of mantissa).  Six of the nine
// products of pieces reach fp32's last bit; the others are below 2^-24 of the whole.  A stage
// holds one piece of A and of B, each is loaded once and the six products of a depth are made
// from three stages.  The tensor cores' own adds lose more with the length of a sum than fp32
// rounding would: the product of the first pieces has an accumulator of its own, apart from
// the five small ones, and every kChunk of depth both are added to fp32 registers and begun
// anew.
//
// Epilogue: a warp owns 32 rows (its TMEM lanes, a row a lane) and walks them in slices of
// 64 bytes of output, through two swizzled shared-memory buffers in turn that TMA stores
// write out (and TMA loads fill with the residual first).  The next slice's accumulator,
// the next tile's too, is on its way while one is computed.  (Stores from registers, 32
// bytes a lane and row, took half as long again: 32 lines an instruction.)  Outputs whose
// rows do not start on 16 bytes go from the buffers with coalesced element stores instead.
//
// Few tiles with a deep sum (a weight's gradient over many rows) are split along the
// depth: each part writes fp32 partials, and a second kernel adds them in order and
// applies the epilogue.
#pragma once

#include "wf_activation.cuh"
#include "wf_gemm.h"
#include "wf_rowio.cuh"
#include "wf_sm100.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

namespace wf {
namespace {

using namespace sm100;

constexpr int kBM = 128;                // rows of a block
constexpr int kBK = 64;                 // depth of a stage: 128 bytes
constexpr int kChunk = 4;               // stages between additions to fp32 registers (three-piece form)
// The same for runs of 16-bit operands, whose logits nothing rounds: the tensor cores' adds truncate,
// by 2^-24 of the sum each on average, which at a depth of 4096 had log probabilities off by 4e-6
// of their size, and has them by 3e-7 in chunks of 512.
constexpr int kDeepChunk = 8;
// A run of up to so many stages of depth keeps its rows of A in shared memory and streams B alone.  The
// products of a 256-wide pair read 64 bytes a cycle of an SM's shared memory and their loads
// write 64, which is all it can do: with half the loads 32768 x 256 -> 50001 goes from 725 to 700 us.
constexpr int kResident = 4;
constexpr int kEpilogueWarps = 16;
constexpr int kThreads = 32 * (kEpilogueWarps + 2);
constexpr int kSliceBytes = 64;         // of a row of output
constexpr uint32_t kBuffer = 32 * kSliceBytes;  // staging: two a warp
constexpr uint64_t kWaitNs = 1000000000ull;
constexpr int kMaxSplits = 32;

struct GemmParams {
  int M, N, tiles_n, units, splits, k_blocks;
  int tiles_m, group, ranges;  // of runs (see Unit)
  bool resident;               // A stays for a run (see kResident)
  int turn_blocks;  // of k_blocks: past them the depth is walked again, with a's second piece
  bool a_mn, b_mn;
  bool y_tma, residual_tma;  // y, the residual start and step on 16 bytes (z always does)
  bool bias_vec;                 // so does the bias
  GemmEpilogue out;
  int32_t* status;
  uint32_t idesc;
};

// BUFFERS: of staging, an epilogue warp (the stages take what they leave).
template <typename T, int BN, int CG, bool PIECES, int BUFFERS>
struct Layout {
  static constexpr uint32_t A_BYTES = kBM * 128, B_BYTES = BN / CG * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr uint32_t STAGING = kEpilogueWarps * BUFFERS * kBuffer;
  static constexpr int FIT = (227 * 1024 - 2048 - (int)STAGING) / (int)STAGE;
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  // a run's A where it stays (see kResident), and the stages of B alone that this leaves room for
  static constexpr int B_FIT = (STAGES * (int)STAGE - kResident * (int)A_BYTES) / (int)B_BYTES;
  static constexpr int B_STAGES = B_FIT < 8 ? B_FIT : 8;
  static constexpr int RING = STAGES > B_STAGES ? STAGES : B_STAGES;
  static constexpr size_t off_staging = (size_t)STAGES * STAGE;
  static constexpr size_t off_bar = off_staging + STAGING;
  static constexpr size_t off_misc = off_bar + 8 * (2 * RING + 5 + 2 * kEpilogueWarps + 2 * kResident);
  static constexpr size_t smem = off_misc + 16 + 1024;
  static constexpr int ACC = PIECES ? 2 * BN : BN;  // TMEM columns of an accumulator (main and small products)
  static constexpr uint32_t TMEM_COLS = 2 * ACC;
  static_assert(!PIECES || STAGES >= 6, "two depths of three pieces");
  // columns of a slice, and of an epilogue warp (a quarter of the tile, or a slice's where
  // that is more: then fewer warps work)
  static constexpr int SC = kSliceBytes / (int)sizeof(T);
  static constexpr int COLS = BN / 4 < SC ? SC : BN / 4;
  static constexpr int WARPS = 4 * (BN / COLS);
};

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

// Units of work: a tile and a share of the depth; or a run of tiles of the same rows, next to
// each other (a range of the columns).  The units of a range of columns follow one another, so
// that the blocks at work share B's rows, in groups of as many tiles of rows as L2 holds of A.
template <bool RUNS>
struct Unit {
  int m0, n0, kb0, kb1, split, run;
  __device__ __forceinline__ int tiles() const { return RUNS ? run : 1; }
  __device__ __forceinline__ Unit(const GemmParams& p, uint32_t u, int BM, int BN) {
    if constexpr (RUNS) {
      const uint32_t whole = (uint32_t)p.group * p.ranges, g = u / whole, at = u - g * whole;
      const uint32_t first = g * p.group, rows = min((uint32_t)p.group, (uint32_t)p.tiles_m - first);
      split = at / rows;
      m0 = (first + at - split * rows) * BM;
      const int t0 = (int)((int64_t)p.tiles_n * split / p.ranges);
      run = (int)((int64_t)p.tiles_n * (split + 1) / p.ranges) - t0;
      n0 = t0 * BN;
      kb0 = 0;
      kb1 = p.k_blocks;
      return;
    }
    // shares of the depth differ by one stage at most; products stay below 2^30 * 32 / 64
    const uint32_t kb = p.k_blocks;
    split = 0;
    kb0 = 0;
    kb1 = kb;
    if (p.splits > 1) {
      const uint32_t splits = p.splits, tile = u / splits;
      split = u - tile * splits;
      kb0 = kb * split / splits;
      kb1 = kb * (split + 1) / splits;
      u = tile;
    }
    const uint32_t tm = u / (uint32_t)p.tiles_n;
    m0 = tm * BM;
    n0 = (u - tm * p.tiles_n) * BN;
  }
};

// Byte of a staging buffer that holds byte `at` of row r's 64: the 64-byte swizzle.
__device__ __forceinline__ uint32_t staged(int r, int at) {
  return r * kSliceBytes + ((at ^ (r << 3)) & 0x30) + (at & 15);
}

// Between a staging buffer and rows that start anywhere: 32 lanes take consecutive elements
// of a row, or of two rows of 16.  For fp32 all sixteen accesses are under way at once; the
// 16-bit types' usual way would pay for that in spilled registers (40 -> 45 us at 32768 x
// 1024), so they have four.
template <typename T>
__device__ __forceinline__ void copy_rows_out(const unsigned char* buf, T* y, int64_t stride, int64_t m, int64_t M,
                                              int n, int N, int lane) {
  constexpr int SC = kSliceBytes / (int)sizeof(T), PER = 32 / SC;  // rows an access
  constexpr int AT = sizeof(T) == 4 ? 16 : 4;
  const int c = lane % SC;
#pragma unroll(AT)
  for (int r = lane / SC; r < 32; r += PER)
    if (m + r < M && n + c < N)
      y[(m + r) * stride + n + c] = *reinterpret_cast<const T*>(buf + staged(r, c * (int)sizeof(T)));
}
template <typename T>
__device__ __forceinline__ void copy_rows_in(unsigned char* buf, const T* x, int64_t stride, int64_t m, int64_t M,
                                             int n, int N, int lane) {
  constexpr int SC = kSliceBytes / (int)sizeof(T), PER = 32 / SC;
  const int c = lane % SC;
  if constexpr (sizeof(T) == 4) {
    T v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = lane / SC + PER * i;
      if (m + r < M && n + c < N) v[i] = x[(m + r) * stride + n + c];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = lane / SC + PER * i;
      if (m + r < M && n + c < N) *reinterpret_cast<T*>(buf + staged(r, c * (int)sizeof(T))) = v[i];
    }
  } else {
#pragma unroll 4
    for (int r = lane / SC; r < 32; r += PER)
      if (m + r < M && n + c < N)
        *reinterpret_cast<T*>(buf + staged(r, c * (int)sizeof(T))) = x[(m + r) * stride + n + c];
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else
    return make_uint4(pack2(T(), v[0], v[1]), pack2(T(), v[2], v[3]), pack2(T(), v[4], v[5]), pack2(T(), v[6], v[7]));
}
// A lane's slice to its staging row.
template <typename T>
__device__ __forceinline__ void stage_slice(uint32_t buf, int lane, const float* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) st_shared_16(buf + staged(lane, 16 * j), pack16<T>(v + j * Vec16<T>::N));
}
__device__ __forceinline__ void add_pairs(const float* f, int n, float* v) {
#pragma unroll
  for (int i = 0; i < n; i += 2) add2(Pair(v[i], v[i + 1]), Pair(f[i], f[i + 1])).get(v[i], v[i + 1]);
}
template <typename T>
__device__ __forceinline__ void add_staged_slice(uint32_t buf, int lane, float* v) {
  constexpr int V = Vec16<T>::N;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float f[V];
    Vec16<T>::unpack(ld_shared_16(buf + staged(lane, 16 * j)), f);
    add_pairs(f, V, v + j * V);
  }
}
// The bias of a slice's columns, from column n on.
template <typename T>
__device__ __forceinline__ void add_bias(const GemmParams& p, int n, float* v) {
  constexpr int V = Vec16<T>::N, SC = kSliceBytes / (int)sizeof(T);
  if (!p.out.bias) return;
  const T* b = static_cast<const T*>(p.out.bias) + n;
  if (p.bias_vec && n + SC <= p.N) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[V];
      Vec16<T>::unpack(ldg16(b + j * V), f);
      add_pairs(f, V, v + j * V);
    }
  } else {
#pragma unroll
    for (int j = 0; j < SC; ++j)
      if (n + j < p.N) v[j] += to_f32(b[j]);
  }
}

// What becomes of a finished accumulator.  Finish: the epilogue above, a tile at a time.  Others
// (wf_linear_logprobs.cu) take runs of tiles of the same rows: begin() a run with a row a lane,
// slice() by slice of it, and end(); where STORES is set, what a slice became goes to ymap, in
// `layers` pieces.
struct Finish {
  static constexpr bool kRuns = false, kStores = false, kFactor = false;
  static constexpr int kBuffers = 2;
};
struct FinishByFactor : Finish {  // with a factor: apart, since its registers spill 16 bytes more
  static constexpr bool kFactor = true;
};

template <typename T, int BN, int CG, bool PIECES, class E>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                const __grid_constant__ CUtensorMap ymap, const __grid_constant__ CUtensorMap zmap,
                const __grid_constant__ CUtensorMap rmap, const GemmParams p, const E e) {
  using L = Layout<T, BN, CG, PIECES, E::kBuffers>;
  using Work = Unit<E::kRuns>;
  // stages between additions to fp32 registers in runs
  constexpr int kRunChunk = PIECES ? kChunk : kDeepChunk;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + L::off_bar);
  uint64_t* empty = full + L::RING;
  uint64_t* acc_full = empty + L::RING;    // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2]
  uint64_t* drained = acc_empty + 2;
  uint64_t* res_full = drained + 1;        // [kEpilogueWarps][2]
  uint64_t* a_full = res_full + 2 * kEpilogueWarps;  // [kResident]
  uint64_t* a_empty = a_full + kResident;            // [kResident]
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(base + L::off_misc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
  constexpr int BM = kBM * CG;
  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;

  // Pair: `full` and `acc_empty` are the leader's alone; the leader's products arrive on
  // `empty`, `acc_full` and `drained` of both.
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::RING; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kResident; ++s) {
      mbar_init(&a_full[s], 1);
      mbar_init(&a_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], CG * L::WARPS);
    }
    mbar_init(drained, 1);
    for (int i = 0; i < 2 * kEpilogueWarps; ++i) mbar_init(&res_full[i], 1);
    fence_mbarrier_init();
  }
  if (warp == 0) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_s, L::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_s, L::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2) {
    __syncthreads();
    cluster_sync();
  } else {
    __syncthreads();
  }
  tc_fence_after();
  pdl_wait();  // what comes before this kernel on its stream is done; nothing above touched global memory
  const uint32_t tmem = *tmem_s;
  uint32_t why = 0;

  if (warp == kEpilogueWarps) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      prefetch_tmap(&amap);
      prefetch_tmap(&bmap);
      Ring r;
      uint32_t issued = 0;
      if constexpr (E::kRuns && !PIECES) {
        if (p.resident) {
          auto load = [&](uint64_t* bar, void* dst, const CUtensorMap* map, int x, int y, uint32_t bytes) {
            if (rank == 0) mbar_arrive_expect_tx(bar, CG * bytes);
            if constexpr (CG == 2) tma_load_3d_pair(dst, map, map_peer(bar, 0), x, y, 0);
            else tma_load_3d(dst, map, bar, x, y, 0);
          };
          uint32_t runs = 0, a_issued = 0;  // a_issued: of this run
          for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step, ++runs) {
            const Work w(p, u, BM, BN);
            a_issued = 0;
            for (int t = 0; t < w.tiles() && !why; ++t)
              for (int kb = 0; kb < p.k_blocks && !why; ++kb) {
                if (t == 0) {
                  if (!mbar_wait_asleep(&a_empty[kb], (runs & 1) ^ 1, kWaitNs)) { why = 4; break; }
                  load(&a_full[kb], base + (size_t)kb * L::A_BYTES, &amap, kb * kBK, w.m0 + (int)rank * kBM, L::A_BYTES);
                  ++a_issued;
                }
                if (!mbar_wait_asleep(&empty[r.stage], r.phase ^ 1, kWaitNs)) { why = 4; break; }
                load(&full[r.stage], base + (size_t)kResident * L::A_BYTES + (size_t)r.stage * L::B_BYTES, &bmap, kb * kBK,
                     w.n0 + t * BN + (int)rank * (BN / CG), L::B_BYTES);
                ++issued;
                r.next<L::B_STAGES>();
              }
          }
          // as below: what is in flight lands before the block ends
          if (rank == 0) {
            for (uint32_t s = 0; s < (uint32_t)L::B_STAGES && s < issued; ++s)
              mbar_wait_asleep(&full[s], (issued - 1 - s) / L::B_STAGES & 1, kWaitNs);
            for (uint32_t s = 0; s < a_issued; ++s) mbar_wait_asleep(&a_full[s], runs - 1 & 1, kWaitNs);
          }
        }
      }
      if (!(E::kRuns && !PIECES && p.resident))
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Work w(p, u, BM, BN);
        const int am = w.m0 + (int)rank * kBM;
        for (int t = 0; t < w.tiles() && !why; ++t)
        for (int kb = w.kb0, bn = w.n0 + t * BN + (int)rank * (BN / CG); kb < w.kb1 && !why; ++kb) {
#pragma unroll 1
          for (int piece = 0; piece < (PIECES ? 3 : 1); ++piece) {
            if (!mbar_wait_asleep(&empty[r.stage], r.phase ^ 1, kWaitNs)) { why = 4; break; }
            unsigned char* st = base + (size_t)r.stage * L::STAGE;
            uint64_t* bar = &full[r.stage];
            if (rank == 0) mbar_arrive_expect_tx(bar, CG * L::STAGE);
            const uint32_t on = CG == 2 ? map_peer(bar, 0) : 0;
            auto load = [&](void* dst, const CUtensorMap* map, int x, int y, int layer) {
              if constexpr (CG == 2) tma_load_3d_pair(dst, map, on, x, y, layer);
              else tma_load_3d(dst, map, bar, x, y, layer);
            };
            const int turn = !PIECES && kb >= p.turn_blocks ? 1 : 0, k = (kb - turn * p.turn_blocks) * kBK;
            if (p.a_mn) {
#pragma unroll
              for (int i = 0; i < kBM / 64; ++i) load(st + i * kBK * 128, &amap, am + 64 * i, k, piece + turn);
            } else {
              load(st, &amap, k, am, piece + turn);
            }
            st += L::A_BYTES;
            if (p.b_mn) {
#pragma unroll
              for (int i = 0; i < BN / CG / 64; ++i) load(st + i * kBK * 128, &bmap, bn + 64 * i, k, piece);
            } else {
              load(st, &bmap, k, bn, piece);
            }
            ++issued;
            r.next<L::STAGES>();
          }
        }
      }
      // where a wait gave up, here or in the products, loads may be in flight that no product will wait for
      if (rank == 0 && !(E::kRuns && !PIECES && p.resident))
        for (uint32_t s = 0; s < (uint32_t)L::STAGES && s < issued; ++s) {
          const uint32_t last = (issued - 1 - s) / L::STAGES;  // round of the newest load of stage s
          mbar_wait_asleep(&full[s], last & 1, kWaitNs);
        }
    }
  } else if (warp == kEpilogueWarps + 1) {
    // ------------------------------------------------------------ products
    if (lane == 0 && rank == 0) {
      Ring r;
      uint32_t acc = 0, acc_phase = 0;
      const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;
      auto commit = [&](uint64_t* bar) {
        if constexpr (CG == 2) mma_commit_pair(bar);
        else mma_commit(bar);
      };
      if constexpr (E::kRuns && !PIECES) {
        if (p.resident) {
          uint32_t runs = 0;
          auto wait = [&](uint64_t* bar, uint32_t phase, uint32_t site) {
            if (mbar_wait_asleep(bar, phase, kWaitNs)) return true;
            why = site;
            return false;
          };
          for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step, ++runs) {
            const Work w(p, u, BM, BN);
            for (int t = 0; t < w.tiles() && !why; ++t) {
              if (!wait(&acc_empty[acc], acc_phase ^ 1, 8)) break;
              tc_fence_after();
              for (int kb = 0; kb < p.k_blocks; ++kb) {
                if ((t == 0 && !wait(&a_full[kb], runs & 1, 16)) || !wait(&full[r.stage], r.phase, 16)) break;
                tc_fence_after();
                const uint32_t as = smem_u32(base + (size_t)kb * L::A_BYTES);
                const uint32_t bs = smem_u32(base + (size_t)kResident * L::A_BYTES + (size_t)r.stage * L::B_BYTES);
#pragma unroll
                for (int k = 0; k < kBK / 16; ++k) {
                  const uint64_t da = smem_desc_kmajor(as + k * 32, 128), db = smem_desc_kmajor(bs + k * 32, 128);
                  if constexpr (CG == 2) mma_f16_pair(tmem + acc * L::ACC, da, db, p.idesc, kb > 0 || k > 0);
                  else mma_f16(tmem + acc * L::ACC, da, db, p.idesc, kb > 0 || k > 0);
                }
                commit(&empty[r.stage]);
                if (t + 1 == w.tiles()) commit(&a_empty[kb]);
                r.next<L::B_STAGES>();
              }
              commit(&acc_full[acc]);
              acc ^= 1;
              acc_phase ^= acc == 0;
            }
          }
        }
      }
      if (!(E::kRuns && !PIECES && p.resident))
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Work w(p, u, BM, BN);
        for (int t = 0; t < w.tiles() && !why; ++t)
        for (int c0 = w.kb0, c1; c0 < w.kb1 && !why; c0 = c1) {
          c1 = E::kRuns ? min(c0 + kRunChunk, w.kb1) : PIECES ? min(c0 + kChunk, w.kb1) : w.kb1;
          if (!mbar_wait_asleep(&acc_empty[acc], acc_phase ^ 1, kWaitNs)) { why = 8; break; }
          tc_fence_after();
          const uint32_t d = tmem + acc * L::ACC;
          // the products of a stage's A with a stage's B
          auto multiply = [&](uint32_t to, uint32_t a_stage, uint32_t b_stage, bool onto) {
            const uint32_t as = smem_u32(base + (size_t)a_stage * L::STAGE);
            const uint32_t bs = smem_u32(base + (size_t)b_stage * L::STAGE) + L::A_BYTES;
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              const uint32_t aa = as + k * a_step, bb = bs + k * b_step;
              const uint64_t da = p.a_mn ? smem_desc_mnmajor(aa) : smem_desc_kmajor(aa, 128);
              const uint64_t db = p.b_mn ? smem_desc_mnmajor(bb) : smem_desc_kmajor(bb, 128);
              if constexpr (CG == 2) mma_f16_pair(to, da, db, p.idesc, onto || k > 0);
              else mma_f16(to, da, db, p.idesc, onto || k > 0);
            }
          };
          auto arrived = [&](const Ring& at) {
            if (!mbar_wait_asleep(&full[at.stage], at.phase, kWaitNs)) {
              why = 16;
              return false;
            }
            tc_fence_after();
            return true;
          };
          for (int kb = c0; kb < c1; ++kb) {
            const bool onto = kb > c0;
            const Ring r0 = r;
            if (!arrived(r0)) break;
            multiply(d, r0.stage, r0.stage, onto);
            r.next<L::STAGES>();
            if constexpr (PIECES) {
              const uint32_t small = d + BN;
              const Ring r1 = r;
              if (!arrived(r1)) break;
              multiply(small, r0.stage, r1.stage, onto);
              multiply(small, r1.stage, r0.stage, true);
              multiply(small, r1.stage, r1.stage, true);
              commit(&empty[r1.stage]);
              r.next<L::STAGES>();
              const Ring r2 = r;
              if (!arrived(r2)) break;
              multiply(small, r0.stage, r2.stage, true);
              multiply(small, r2.stage, r0.stage, true);
              commit(&empty[r2.stage]);
              r.next<L::STAGES>();
            }
            commit(&empty[r0.stage]);
          }
          commit(&acc_full[acc]);
          acc ^= 1;
          acc_phase ^= acc == 0;
        }
      }
      commit(drained);
    }
  } else if (warp < L::WARPS) {
    // ------------------------------------------------------------ epilogue
    // warp w reads TMEM lanes 32 (w % 4) .. + 31 (a row a lane) and share w / 4 of the columns
    constexpr int COLS = L::COLS, SC = L::SC;
    const uint32_t lbase = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (warp >> 2) * COLS;
    constexpr int kBuffers = E::kBuffers;
    unsigned char* bufs = base + L::off_staging + (size_t)warp * kBuffers * kBuffer;
    const GemmEpilogue& o = p.out;
    uint32_t acc = 0, acc_phase = 0, turn = 0, res_phase = 0;
    auto buffer = [&](uint32_t i) { return bufs + (kBuffers > 1 ? i & 1 : 0) * kBuffer; };
    auto release = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) mbar_arrive(&acc_empty[acc]);
        else mbar_arrive_peer_relaxed(map_peer(&acc_empty[acc], 0));
      }
      acc ^= 1;
      acc_phase ^= acc == 0;
    };
    auto store = [&](bool tma, const CUtensorMap* map, void* to, int64_t stride, int m, int n, int layer) {
      unsigned char* buf = buffer(turn++);
      if (tma) {
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(map, buf, n, m, layer);
          bulk_commit();
        }
      } else {
        __syncwarp();
        copy_rows_out<T>(buf, static_cast<T*>(to) + (int64_t)layer * p.M * stride, stride, m, p.M, n, p.N, lane);
        fence_async_shared();  // a residual's load may fill the buffer next
        __syncwarp();
      }
    };
    // z, activation, residual and y of one slice; the buffers take turns.  A buffer may be
    // written again once the copy engine has read what it held: where every use is a TMA store,
    // that is the last but one group.  y's element stores make no group, so z's store of the
    // slice before, from the same buffer, is then the newest one and has to be waited for.
    auto out = [&](float* v, int m, int n, int layer) {
      if (o.z) {
        if (lane == 0) {
          if (p.y_tma) bulk_wait_read<1>();
          else bulk_wait_read<0>();
        }
        __syncwarp();
        float kept[SC];
#pragma unroll
        for (int j = 0; j < SC; ++j) kept[j] = kept_z(o.act, v[j]);
        stage_slice<typename Kept<T>::type>(smem_u32(buffer(turn)), lane, kept);
        store(true, &zmap, nullptr, 0, m, n, 0);
      }
      if (lane == 0) bulk_wait_read<1>();
      __syncwarp();
      const uint32_t i = turn & 1;
      if (o.residual) {
        if (p.residual_tma) {
          if (lane == 0) {
            mbar_arrive_expect_tx(&res_full[2 * warp + i], kBuffer);
            tma_load_3d(buffer(turn), &rmap, &res_full[2 * warp + i], n, m, 0);
          }
        } else {
          copy_rows_in<T>(buffer(turn), static_cast<const T*>(o.residual), o.r_stride, m, p.M, n, p.N, lane);
          __syncwarp();
        }
      }
      activate_all<T, SC>(o.act, v);
      if (o.residual) {
        if (p.residual_tma) {
          if (!__all_sync(0xffffffffu, mbar_wait_asleep(&res_full[2 * warp + i], res_phase >> i & 1, kWaitNs)))
            why = 128;
          res_phase ^= 1u << i;
        }
        add_staged_slice<T>(smem_u32(buffer(turn)), lane, v);
      }
      stage_slice<T>(smem_u32(buffer(turn)), lane, v);
      store(p.y_tma, &ymap, o.y, o.y_stride, m, n, layer);
    };
    auto ready = [&] {
      if (!__all_sync(0xffffffffu, mbar_wait_asleep(&acc_full[acc], acc_phase, kWaitNs))) why = 32;
      tc_fence_after();
      return why == 0;
    };
    if constexpr (E::kRuns) {
      // a slice of a run, at column n; all lanes, whether or not their row is in range
      typename E::Row row;
      auto take = [&](float* v, int m, int n) {
        add_bias<T>(p, n, v);
        e.template slice<SC>(row, v, m + lane, n, p.N);
        if constexpr (E::kStores) {
          for (int layer = 0;; ++layer) {
            if (lane == 0) bulk_wait_read<kBuffers - 1>();
            __syncwarp();
            stage_slice<T>(smem_u32(buffer(turn)), lane, v);
            store(true, &ymap, nullptr, 0, m, n, layer);
            if (layer + 1 == e.layers) break;
#pragma unroll
            for (int j = 0; j < SC; ++j) {  // what the rounding leaves
              const float r = to_f32(from_f32<T>(v[j]));
              v[j] = isfinite(r) ? v[j] - r : 0.f;
            }
          }
        }
      };
      // The accumulator of a tile goes to registers as soon as it is finished, and the tensor
      // memory back: what is done with it runs under the next products.
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Work w(p, u, BM, BN);
        const int m = w.m0 + (int)rank * kBM + 32 * (warp & 3), share = warp >> 2;
        e.begin(row, m + lane, p.M, p.N);
        for (int t = 0; t < w.tiles() && !why; ++t) {
          const int n0 = w.n0 + t * BN + share * COLS;
          float sum[COLS];
          for (int c0 = w.kb0; c0 < w.kb1; c0 += kRunChunk) {
            if (!ready()) break;
            if (c0 == w.kb0) {
              uint32_t r[COLS];
#pragma unroll
              for (int c = 0; c < COLS; c += SC)
                tmem_ld(lbase + acc * L::ACC + c, reinterpret_cast<uint32_t(&)[SC]>(r[c]));
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < COLS; ++j) sum[j] = __uint_as_float(r[j]);
            } else {
#pragma unroll
              for (int c = 0; c < COLS; c += 16) {
                uint32_t r[16];
                tmem_ld(lbase + acc * L::ACC + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(r[j]);
              }
            }
            if constexpr (PIECES) {
#pragma unroll
              for (int c = 0; c < COLS; c += 16) {
                uint32_t r[16];
                tmem_ld(lbase + acc * L::ACC + BN + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(r[j]);
              }
            }
            release();
          }
#pragma unroll
          for (int c = 0; c < COLS; c += SC)
            if (m < p.M && n0 + c < p.N && !why) take(sum + c, m, n0 + c);
        }
        if (!why) e.end(row, m + lane, p.M, w.split * (L::WARPS / 4) + share);
      }
    } else if constexpr (PIECES) {
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Work w(p, u, BM, BN);
        const int m = w.m0 + (int)rank * kBM + 32 * (warp & 3), n0 = w.n0 + (warp >> 2) * COLS;
        float sum[COLS];
#pragma unroll
        for (int j = 0; j < COLS; ++j) sum[j] = 0.f;
        for (int c0 = w.kb0; c0 < w.kb1; c0 += kChunk) {
          if (!ready()) break;
#pragma unroll
          for (int c = 0; c < COLS; c += SC) {
            uint32_t r[SC], s[SC];
            tmem_ld(lbase + acc * L::ACC + c, r);
            tmem_ld(lbase + acc * L::ACC + BN + c, s);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < SC; ++j) sum[c + j] += __uint_as_float(r[j]) + __uint_as_float(s[j]);
          }
          release();
        }
#pragma unroll
        for (int c = 0; c < COLS; c += SC)
          if (m < p.M && n0 + c < p.N && !why) {
            add_bias<T>(p, n0 + c, sum + c);
            out(sum + c, m, n0 + c, w.split);
          }
      }
    } else {
      // slices come in order over the units; the one after the current is asked for before
      // the current is computed, across units where its accumulator is finished by then
      uint32_t r[SC];
      bool asked = false;
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Work w(p, u, BM, BN);
        const int m = w.m0 + (int)rank * kBM + 32 * (warp & 3), n0 = w.n0 + (warp >> 2) * COLS;
        if (!asked) {
          if (!ready()) break;
          tmem_ld(lbase + acc * L::ACC, r);
        }
        asked = false;
#pragma unroll 1
        for (int c = 0; c < COLS && !why; c += SC) {
          float v[SC];
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < SC; ++j) v[j] = __uint_as_float(r[j]);
          if constexpr (E::kFactor) {
            const float factor = __ldg(o.factor);
#pragma unroll
            for (int j = 0; j < SC; j += 2) mul2(Pair(v[j], v[j + 1]), Pair(factor)).get(v[j], v[j + 1]);
          }
          add_bias<T>(p, n0 + c, v);
          if (c + SC < COLS) {
            tmem_ld(lbase + acc * L::ACC + c + SC, r);
          } else {
            release();
            if (u + step < (uint32_t)p.units && __all_sync(0xffffffffu, mbar_try_wait(&acc_full[acc], acc_phase))) {
              tc_fence_after();
              tmem_ld(lbase + acc * L::ACC, r);
              asked = true;
            }
          }
          if (m < p.M && n0 + c < p.N) out(v, m, n0 + c, w.split);
        }
      }
      if (asked) tmem_ld_wait();
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncwarp();
  if (why && p.status && lane == 0) atomicOr(p.status, 2 | (int)why);
  // TMEM is given back, and a pair parts, once no product writes to it
  if (warp == 0 && !__all_sync(0xffffffffu, mbar_wait_asleep(drained, 0, kWaitNs)) && p.status && lane == 0)
    atomicOr(p.status, 2 | 64);
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  if (warp == 0) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem, L::TMEM_COLS);
    else tmem_dealloc(tmem, L::TMEM_COLS);
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

bool encode(CUtensorMap* map, int dtype, const void* ptr, const int64_t (&dims)[3], int64_t pitch, int64_t layer_pitch,
            int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
  const int64_t size = dtype == kF32 ? 4 : 2;
  const cuuint64_t d[3] = {(cuuint64_t)dims[0], (cuuint64_t)dims[1], (cuuint64_t)dims[2]};
  const cuuint64_t strides[2] = {(cuuint64_t)(pitch * size), (cuuint64_t)(layer_pitch * size)};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  EncodeTiledFnG fn = encode_fn();
  return fn && fn(map,
                  dtype == kBF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                  : dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                  3, const_cast<void*>(ptr), d, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// An operand in boxes of 64 columns (128 bytes); its pieces are the third axis.
bool make_map(CUtensorMap* map, const GemmOperand& o, int pieces, int op_dtype, int box_rows) {
  return encode(map, op_dtype, o.ptr, {o.cols, o.rows, pieces}, o.pitch,
                pieces > 1 ? o.piece_stride : o.pitch * o.rows, 64, o.mn_major ? kBK : box_rows,
                CU_TENSOR_MAP_SWIZZLE_128B);
}
// An epilogue's matrix in slices of 32 rows; the parts of a split depth are the third axis.
template <typename T>
bool make_out_map(CUtensorMap* map, const void* ptr, int64_t cols, int64_t rows, int64_t layers, int64_t pitch) {
  constexpr int dtype = std::is_same<T, float>::value ? kF32 : std::is_same<T, __half>::value ? kF16 : kBF16;
  return encode(map, dtype, ptr, {cols, rows, layers}, pitch, pitch * rows, kSliceBytes / (int)sizeof(T), 32,
                CU_TENSOR_MAP_SWIZZLE_64B);
}

struct Shape {
  int bn, cg;
  // 64 of depth: the products' time, or the loads' at about 64 bytes a cycle an SM; of one
  // piece, and of three with their six products (0: no room for the stages or the sums)
  int cycles, cycles3;
};
struct Plan {
  Shape shape;
  int tiles_n, tiles, splits, k_blocks;
  int layers;                  // of y: the parts of a split depth, or the pieces of what a run stores
  int tiles_m, group, ranges;  // of runs (see Unit)
};

template <typename T, int BN, int CG, bool PIECES, class E>
int launch_tile(const GemmProblem& g, const GemmEpilogue& out, const Plan& plan, const E& e, cudaStream_t stream) {
  using L = Layout<T, BN, CG, PIECES, E::kBuffers>;
  // encoding a tensor map is a driver call: it needs the device's context current in this thread,
  // which the runtime sees to at a launch, and this may be a thread's first (a backward's)
  int device = 0;
  if (cudaError_t rc = cudaGetDevice(&device)) return (int)rc;
  if (cudaError_t rc = cudaSetDevice(device)) return (int)rc;
  CUtensorMap amap, bmap, ymap{}, zmap{}, rmap{};
  if (!make_map(&amap, g.a, g.pieces * g.turns, g.op_dtype, kBM) ||
      !make_map(&bmap, g.b, g.pieces, g.op_dtype, BN / CG))
    return -1;
  GemmParams p{};
  p.M = (int)g.M;
  p.N = (int)g.N;
  p.tiles_n = plan.tiles_n;
  p.splits = plan.splits;
  p.units = E::kRuns ? plan.tiles_m * plan.ranges : plan.tiles * plan.splits;
  p.tiles_m = plan.tiles_m;
  p.group = plan.group;
  p.ranges = plan.ranges;
  p.resident = E::kRuns && !PIECES && !g.a.mn_major && !g.b.mn_major && g.turns == 1 && plan.k_blocks <= kResident;
  p.k_blocks = plan.k_blocks;
  p.turn_blocks = plan.k_blocks / g.turns;
  p.a_mn = g.a.mn_major;
  p.b_mn = g.b.mn_major;
  p.out = out;
  p.status = g.status;
  p.idesc = idesc_f16(g.op_dtype == kBF16, kBM * CG, BN) | (g.a.mn_major ? 1u << 15 : 0u) |
            (g.b.mn_major ? 1u << 16 : 0u);
  auto on16 = [](const void* q, int64_t stride) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
  };
  p.y_tma = out.y && on16(out.y, out.y_stride);
  // rows that overlap (a broadcast residual) are not a tensor map's
  p.residual_tma = out.residual && on16(out.residual, out.r_stride) && out.r_stride >= g.N;
  if (p.y_tma && !make_out_map<T>(&ymap, out.y, g.N, g.M, plan.layers, out.y_stride)) return -1;
  if (out.z && !make_out_map<T>(&zmap, out.z, g.N, g.M, 1, out.z_stride)) return -1;
  if (p.residual_tma && !make_out_map<T>(&rmap, out.residual, g.N, g.M, 1, out.r_stride)) return -1;
  p.bias_vec = reinterpret_cast<uintptr_t>(out.bias) % 16 == 0;
  auto kern = gemm_kernel<T, BN, CG, PIECES, E>;
  static std::atomic<uint64_t> allowed{0};  // devices whose limit has been raised for this kernel
  if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
    if (cudaError_t rc = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem))
      return (int)rc;
    if (device < 64) allowed.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CG * std::min(p.units, kSms / CG)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, kern, amap, bmap, ymap, zmap, rmap, p, e);
}


}  // namespace
}  // namespace wf

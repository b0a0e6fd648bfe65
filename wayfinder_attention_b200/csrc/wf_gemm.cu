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
constexpr int kEpilogueWarps = 16;
constexpr int kThreads = 32 * (kEpilogueWarps + 2);
constexpr int kSliceBytes = 64;         // of a row of output
constexpr uint32_t kBuffer = 32 * kSliceBytes;  // staging: two a warp
constexpr uint64_t kWaitNs = 1000000000ull;
constexpr int kMaxSplits = 32;

struct GemmParams {
  int M, N, tiles_n, units, splits, k_blocks;
  int turn_blocks;  // of k_blocks: past them the depth is walked again, with a's second piece
  bool a_mn, b_mn;
  bool y_tma, residual_tma;  // y, the residual start and step on 16 bytes (z always does)
  bool bias_vec;                 // so does the bias
  GemmEpilogue out;
  int32_t* status;
  uint32_t idesc;
};

template <typename T, int BN, int CG, bool PIECES>
struct Layout {
  static constexpr uint32_t A_BYTES = kBM * 128, B_BYTES = BN / CG * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr uint32_t STAGING = kEpilogueWarps * 2 * kBuffer;
  static constexpr int FIT = (227 * 1024 - 2048 - (int)STAGING) / (int)STAGE;
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static constexpr size_t off_staging = (size_t)STAGES * STAGE;
  static constexpr size_t off_bar = off_staging + STAGING;
  static constexpr size_t off_misc = off_bar + 8 * (2 * STAGES + 5 + 2 * kEpilogueWarps);
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

// Units of work: a tile and a share of the depth.
struct Unit {
  int m0, n0, kb0, kb1, split;
  __device__ __forceinline__ Unit(const GemmParams& p, uint32_t u, int BM, int BN) {
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

template <typename T, int BN, int CG, bool PIECES>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                const __grid_constant__ CUtensorMap ymap, const __grid_constant__ CUtensorMap zmap,
                const __grid_constant__ CUtensorMap rmap, const GemmParams p) {
  using L = Layout<T, BN, CG, PIECES>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + L::off_bar);
  uint64_t* empty = full + L::STAGES;
  uint64_t* acc_full = empty + L::STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2]
  uint64_t* drained = acc_empty + 2;
  uint64_t* res_full = drained + 1;        // [kEpilogueWarps][2]
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(base + L::off_misc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
  constexpr int BM = kBM * CG;
  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;

  // Pair: `full` and `acc_empty` are the leader's alone; the leader's products arrive on
  // `empty`, `acc_full` and `drained` of both.
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
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
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Unit w(p, u, BM, BN);
        const int am = w.m0 + (int)rank * kBM, bn = w.n0 + (int)rank * (BN / CG);
        for (int kb = w.kb0; kb < w.kb1 && !why; ++kb) {
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
      // after a wait that gave up, loads may be in flight that no product will wait for
      if (why && rank == 0)
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
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Unit w(p, u, BM, BN);
        for (int c0 = w.kb0; c0 < w.kb1 && !why; c0 += PIECES ? kChunk : w.kb1 - w.kb0) {
          const int c1 = PIECES ? min(c0 + kChunk, w.kb1) : w.kb1;
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
    unsigned char* bufs = base + L::off_staging + (size_t)warp * 2 * kBuffer;
    const GemmEpilogue& o = p.out;
    uint32_t acc = 0, acc_phase = 0, turn = 0, res_phase = 0;
    auto buffer = [&](uint32_t i) { return bufs + (i & 1) * kBuffer; };
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
    if constexpr (PIECES) {
      for (uint32_t u = first; u < (uint32_t)p.units && !why; u += step) {
        const Unit w(p, u, BM, BN);
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
        const Unit w(p, u, BM, BN);
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

// Adds the parts of a split depth and applies the epilogue: a thread takes 4 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) gemm_join_kernel(const float* partial, int splits, int64_t pitch, int64_t M,
                                                        int64_t N, GemmEpilogue o) {
  using Z = typename Kept<T>::type;
  pdl_wait();
  const int64_t groups = pitch / 4, total = M * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / groups, n = i % groups * 4;
    const int live = (int)min((int64_t)4, N - n);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float4 f = *reinterpret_cast<const float4*>(partial + ((int64_t)s * M + m) * pitch + n);
      v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
    }
    if (o.bias)
      for (int j = 0; j < live; ++j) v[j] += to_f32(static_cast<const T*>(o.bias)[n + j]);
    if (o.z)
      for (int j = 0; j < live; ++j)
        static_cast<Z*>(o.z)[m * o.z_stride + n + j] = from_f32<Z>(kept_z(o.act, v[j]));
    activate_all<T, 4>(o.act, v);
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

// Tile shape and depth shares: the least of an estimate over the shapes there are.  A
// unit's time is its stages of depth at the rate the shape can take them plus its
// accumulator's way out; units run in waves.
struct Shape {
  int bn, cg;
  // 64 of depth: the products' time, or the loads' at about 64 bytes a cycle an SM; of one
  // piece, and of three with their six products (0: no room for the stages or the sums)
  int cycles, cycles3;
};
constexpr Shape kShapes[] = {{256, 2, 560, 0}, {128, 2, 400, 1700}, {128, 1, 540, 0}, {64, 1, 400, 1300}};
constexpr int kMinShare = 4;  // stages of depth a share has at least
struct Plan {
  Shape shape;
  int tiles_n, tiles, splits, k_blocks;
};
Plan plan_of(int64_t M, int64_t N, int64_t K, int pieces, int turns) {
  Plan best{};
  double least = 0;
  for (const Shape& s : kShapes) {
    if (pieces > 1 && !s.cycles3) continue;
    Plan p{};
    p.shape = s;
    p.k_blocks = (int)((K + kBK - 1) / kBK) * turns;
    const int64_t tn = (N + s.bn - 1) / s.bn, tm = (M + kBM * s.cg - 1) / (kBM * s.cg);
    p.tiles_n = (int)tn;
    p.tiles = (int)(tn * tm);
    const int slots = kSms / s.cg;
    for (int splits = 1; splits <= kMaxSplits && (splits == 1 || p.k_blocks / splits >= kMinShare); ++splits) {
      if (splits > 1 && (int64_t)p.tiles * splits > 2 * slots) break;  // most shapes look at one split
      const int64_t waves = ((int64_t)p.tiles * splits + slots - 1) / slots;
      const int64_t deep = (p.k_blocks + splits - 1) / splits;
      // partials go through L2 twice, and joining them is a launch
      const double join = splits > 1 ? 4000 + 8.0 * splits * M * N / 4000 : 0;
      const double t = (double)waves * (deep * (pieces > 1 ? s.cycles3 : s.cycles) + 4 * s.bn) + join;
      if (best.splits == 0 || t < least) {
        least = t;
        best = p;
        best.splits = splits;
      }
    }
  }
  return best;
}
int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

template <typename T, int BN, int CG, bool PIECES>
int launch_tile(const GemmProblem& g, const GemmEpilogue& out, const Plan& plan, cudaStream_t stream) {
  using L = Layout<T, BN, CG, PIECES>;
  // encoding a tensor map is a driver call: it needs the device's context current in this thread,
  // which the runtime sees to at a launch, and this may be a thread's first (a backward's)
  int device = 0;
  if (cudaError_t e = cudaGetDevice(&device)) return (int)e;
  if (cudaError_t e = cudaSetDevice(device)) return (int)e;
  CUtensorMap amap, bmap, ymap{}, zmap{}, rmap{};
  if (!make_map(&amap, g.a, g.pieces * g.turns, g.op_dtype, kBM) ||
      !make_map(&bmap, g.b, g.pieces, g.op_dtype, BN / CG))
    return -1;
  GemmParams p{};
  p.M = (int)g.M;
  p.N = (int)g.N;
  p.tiles_n = plan.tiles_n;
  p.splits = plan.splits;
  p.units = plan.tiles * plan.splits;
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
  p.y_tma = on16(out.y, out.y_stride);
  // rows that overlap (a broadcast residual) are not a tensor map's
  p.residual_tma = out.residual && on16(out.residual, out.r_stride) && out.r_stride >= g.N;
  if (p.y_tma && !make_out_map<T>(&ymap, out.y, g.N, g.M, plan.splits, out.y_stride)) return -1;
  if (out.z && !make_out_map<T>(&zmap, out.z, g.N, g.M, 1, out.z_stride)) return -1;
  if (p.residual_tma && !make_out_map<T>(&rmap, out.residual, g.N, g.M, 1, out.r_stride)) return -1;
  p.bias_vec = reinterpret_cast<uintptr_t>(out.bias) % 16 == 0;
  auto kern = gemm_kernel<T, BN, CG, PIECES>;
  static std::atomic<uint64_t> allowed{0};  // devices whose limit has been raised for this kernel
  if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem))
      return (int)e;
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
  return (int)cudaLaunchKernelEx(&cfg, kern, amap, bmap, ymap, zmap, rmap, p);
}

template <typename T, bool PIECES>
int launch_shape(const GemmProblem& g, const GemmEpilogue& out, const Plan& plan, cudaStream_t stream) {
  const Shape& s = plan.shape;
  if constexpr (!PIECES) {
    if (s.bn == 256) return launch_tile<T, 256, 2, PIECES>(g, out, plan, stream);
    if (s.bn == 128 && s.cg == 1) return launch_tile<T, 128, 1, PIECES>(g, out, plan, stream);
  }
  if (s.cg == 2) return launch_tile<T, 128, 2, PIECES>(g, out, plan, stream);
  return launch_tile<T, 64, 1, PIECES>(g, out, plan, stream);
}

template <typename T>
int launch_type(const GemmProblem& g, cudaStream_t stream) {
  constexpr bool PIECES = std::is_same<T, float>::value;
  const Plan plan = plan_of(g.M, g.N, g.K, g.pieces, g.turns);
  if (plan.splits == 1) return launch_shape<T, PIECES>(g, g.out, plan, stream);
  GemmEpilogue parts{};
  parts.y = g.ws;
  parts.y_stride = round8(g.N);
  if (int rc = launch_shape<float, PIECES>(g, parts, plan, stream)) return rc;
  const int64_t work = (g.M * (parts.y_stride / 4) + 255) / 256;
  return (int)launch_pdl(gemm_join_kernel<T>, dim3((unsigned)std::min<int64_t>(work, 8 * kSms)), dim3(256), 0, stream,
                         static_cast<const float*>(g.ws), plan.splits, parts.y_stride, g.M, g.N, g.out);
}

}  // namespace

size_t gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, int pieces, int turns) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = plan_of(M, N, K, pieces, turns);
  return p.splits > 1 ? (size_t)p.splits * M * round8(N) * sizeof(float) : 0;
}

int launch_gemm(const GemmProblem& g, cudaStream_t stream) {
  if (g.M == 0 || g.N == 0) return 0;
  if (g.out_dtype == kBF16) return launch_type<__nv_bfloat16>(g, stream);
  if (g.out_dtype == kF16) return launch_type<__half>(g, stream);
  return launch_type<float>(g, stream);
}

}  // namespace wf

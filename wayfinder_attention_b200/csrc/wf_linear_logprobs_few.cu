// linear_token_logprobs' forward over up to 64 rows: the weight streams once, and a block of it is the
// product's tall operand.
//
// The tiled product pads the rows to 128 and multiplies them with 128 of the vocabulary: at 16 rows
// seven eighths of that is padding, which costs no bytes but power, and under a sustained load the
// power cap takes it out of the memory's rate.  4096 -> 131072 in fp16 without a bias, one pass after the other, there and
// here: 257 and 164 us for 1 row, 178 and 165 for 16, 199 and 182 for 64, where a copy's rate gives 164 (a warmer GPU
// takes up to 193 for 16 rows; with a bias of which a quarter is banned 179).  A weight that L2 holds most of: 1024 -> 50001 in bf16
// 42 and 33 us for 16 rows, but 35 and 41 for 64.  Here 128 rows of W are A, the given rows
// (padded to 16, 32 or 64) are B, and an accumulator's lanes are tokens of the vocabulary, its columns
// the rows.  A thread keeps the running maximum m, s = sum exp(z - m) and u = sum exp(z - m) (z - m) of
// its lane's tokens for each row, over all tiles of the block; lanes are joined once, at the end.
//
// Warp 0 streams 64-deep slices of W and x into a ring of stages, warp 1 issues the products into
// two accumulators in turn, the others take them: every kFewChunk stages they are added to fp32
// registers, as in the runs of the tiled product and for the same reason.
#include "wf_gemm_kernel.cuh"
#include "wf_linear_logprobs.cuh"

namespace wf {
namespace {

constexpr int kFewTile = 128;  // tokens of the vocabulary
// Stages of depth between additions to fp32 registers, half of kDeepChunk: log probabilities off by 1.5e-7
// of their size instead of 3e-7, in the time that the weight needs (16 rows, 4096 -> 131072 with 8, 4 and 2 stages:
// 174, 165 and 180 us; 64 rows 178, 182 and 203; 64 rows, 1024 -> 50001 40, 41 and 42).
constexpr int kFewChunk = 4;
template <int NT>
struct FewLayout {
  static constexpr int WARPS = 4 * (NT <= 32 ? 1 : NT / 32);  // of the epilogue: 32 rows at most each
  static constexpr int COLS = NT <= 32 ? NT : 32, THREADS = 32 * (2 + 2 + WARPS);
  static constexpr uint32_t W_BYTES = kFewTile * 128, X_BYTES = NT * 128, STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = (227 * 1024 - 2048) / (int)STAGE < 12 ? (227 * 1024 - 2048) / (int)STAGE : 12;
  static constexpr size_t off_bar = (size_t)STAGES * STAGE, off_misc = off_bar + 8 * (2 * STAGES + 5);
  static constexpr size_t smem = off_misc + 16 + 1024;
  static constexpr uint32_t TMEM_COLS = 2 * NT < 32 ? 32 : 2 * NT;
};
struct FewParams {
  const int64_t* tokens;
  const void* bias;    // [vocab] or null
  float* parts;        // [3][4 blocks][rows]
  float* token_logit;  // [rows]
  int rows, vocab, tiles, k_blocks;
  int32_t* status;
  uint32_t idesc;
};

template <typename T, int NT>
__global__ void __launch_bounds__(FewLayout<NT>::THREADS, 1)
    linear_logprobs_few_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                               const FewParams p) {
  using L = FewLayout<NT>;
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
      mbar_init(&acc_empty[i], L::WARPS);
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
  pdl_wait();
  const uint32_t tmem = *tmem_s;
  const int t0 = (int)((int64_t)p.tiles * blockIdx.x / gridDim.x), t1 = (int)((int64_t)p.tiles * (blockIdx.x + 1) / gridDim.x);
  uint32_t why = 0;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&wmap);
      prefetch_tmap(&xmap);
      Ring r;
      uint32_t issued = 0;
      for (int t = t0; t < t1 && !why; ++t)
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait_asleep(&empty[r.stage], r.phase ^ 1, kWaitNs)) { why = 4; break; }
          unsigned char* st = base + (size_t)r.stage * L::STAGE;
          mbar_arrive_expect_tx(&full[r.stage], L::STAGE);
          tma_load_3d(st, &wmap, &full[r.stage], kb * kBK, t * kFewTile, 0);
          tma_load_3d(st + L::W_BYTES, &xmap, &full[r.stage], kb * kBK, 0, 0);
          ++issued;
          r.next<L::STAGES>();
        }
      // where a wait gave up, here or in the products, loads may be in flight that no product will wait for
      for (uint32_t s = 0; s < (uint32_t)L::STAGES && s < issued; ++s)
        mbar_wait_asleep(&full[s], (issued - 1 - s) / L::STAGES & 1, kWaitNs);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      Ring r;
      uint32_t acc = 0, acc_phase = 0;
      for (int t = t0; t < t1 && !why; ++t)
        for (int c0 = 0; c0 < p.k_blocks && !why; c0 += kFewChunk) {
          const int c1 = min(c0 + kFewChunk, p.k_blocks);
          if (!mbar_wait_asleep(&acc_empty[acc], acc_phase ^ 1, kWaitNs)) { why = 8; break; }
          tc_fence_after();
          for (int kb = c0; kb < c1; ++kb) {
            if (!mbar_wait_asleep(&full[r.stage], r.phase, kWaitNs)) { why = 16; break; }
            tc_fence_after();
            const uint32_t ws = smem_u32(base + (size_t)r.stage * L::STAGE), xs = ws + L::W_BYTES;
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k)
              mma_f16(tmem + acc * NT, smem_desc_kmajor(ws + k * 32, 128), smem_desc_kmajor(xs + k * 32, 128), p.idesc,
                      kb > c0 || k > 0);
            mma_commit(&empty[r.stage]);
            r.next<L::STAGES>();
          }
          mma_commit(&acc_full[acc]);
          acc ^= 1;
          acc_phase ^= acc == 0;
        }
      mma_commit(drained);
    }
  } else if (warp >= 4) {
    // warp w reads lanes 32 (w % 4) .. + 31, columns from 32 ((w - 4) / 4) on
    constexpr int COLS = L::COLS;
    const int quadrant = warp & 3, first = (warp - 4) / 4 * COLS;
    const uint32_t lbase = tmem + ((uint32_t)(32 * quadrant) << 16) + first;
    uint32_t acc = 0, acc_phase = 0;
    float m[COLS], s[COLS], u[COLS];
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      m[j] = -INFINITY;
      s[j] = u[j] = 0.f;
    }
    // lane j has row first + j's token
    const int64_t token = first + lane < p.rows && lane < COLS ? p.tokens[first + lane] : -1;
    const int my_token = token >= 0 && token < p.vocab ? (int)token : -1;
    for (int t = t0; t < t1 && !why; ++t) {
      float z[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) z[j] = 0.f;
      const int v = t * kFewTile + 32 * quadrant + lane;
      const bool in = v < p.vocab;
      const float b = in && p.bias ? to_f32(static_cast<const T*>(p.bias)[v]) : 0.f;
      for (int c0 = 0; c0 < p.k_blocks; c0 += kFewChunk) {
        if (!__all_sync(0xffffffffu, mbar_wait_asleep(&acc_full[acc], acc_phase, kWaitNs))) {
          why = 32;
          break;
        }
        tc_fence_after();
        uint32_t r[COLS];
        tmem_ld(lbase + acc * NT, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < COLS; ++j) z[j] += __uint_as_float(r[j]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
        acc ^= 1;
        acc_phase ^= acc == 0;
      }
      if (why) break;
#pragma unroll
      for (int j = 0; j < COLS; ++j) {
        if (first + j >= p.rows) break;
        const float x = in ? z[j] + b : -INFINITY;
        if (v == __shfl_sync(0xffffffffu, my_token, j)) p.token_logit[first + j] = x;
        // one token against the sums so far: the smaller of the two maxima has an exponential
        const float top = max_keep_nan(m[j], x), d = fmaxf(m[j] - top, kNothing), dx = fmaxf(x - top, kNothing);
        const float a = exp2_approx(d * kLog2e), e = exp2_approx(dx * kLog2e);
        u[j] = fmaf(a, fmaf(s[j], d, u[j]), e * dx);
        s[j] = fmaf(a, s[j], top == -INFINITY ? 0.f : e);
        m[j] = top;
      }
    }
    // lanes are joined; lane j keeps row first + j
    float mine[3] = {};
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      if (first + j >= p.rows) break;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        join_sums(m[j], s[j], u[j], __shfl_xor_sync(0xffffffffu, m[j], o), __shfl_xor_sync(0xffffffffu, s[j], o),
                  __shfl_xor_sync(0xffffffffu, u[j], o));
      if (lane == j) {
        mine[0] = m[j];
        mine[1] = s[j];
        mine[2] = u[j];
      }
    }
    if (!why && lane < COLS && first + lane < p.rows) {
      float* to = p.parts + (int64_t)(4 * blockIdx.x + quadrant) * p.rows + first + lane;
      const int64_t stride = (int64_t)4 * gridDim.x * p.rows;
      to[0] = mine[0];
      to[stride] = mine[1];
      to[2 * stride] = mine[2];
    }
  }
  __syncwarp();
  if (why && p.status && lane == 0) atomicOr(p.status, 2 | (int)why);
  // TMEM is given back once no product writes to it
  if (warp == 0 && !__all_sync(0xffffffffu, mbar_wait_asleep(drained, 0, kWaitNs)) && p.status && lane == 0)
    atomicOr(p.status, 2 | 64);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
}

template <typename T, int NT>
int launch(const GemmOperand& x, const GemmOperand& w, FewParams p, int dtype, int blocks, cudaStream_t stream) {
  using L = FewLayout<NT>;
  int device = 0;  // as in launch_tile: encoding a tensor map needs the device's context current
  if (cudaError_t rc = cudaGetDevice(&device)) return (int)rc;
  if (cudaError_t rc = cudaSetDevice(device)) return (int)rc;
  CUtensorMap wmap, xmap;
  if (!make_map(&wmap, w, 1, dtype, kFewTile) || !make_map(&xmap, x, 1, dtype, NT)) return -1;
  p.idesc = idesc_f16(dtype == kBF16, kFewTile, NT);
  auto kern = linear_logprobs_few_kernel<T, NT>;
  static std::atomic<uint64_t> allowed{0};  // devices whose limit has been raised for this kernel
  if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
    if (cudaError_t rc = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem))
      return (int)rc;
    if (device < 64) allowed.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
  }
  return (int)launch_pdl(kern, dim3(blocks), dim3(L::THREADS), L::smem, stream, wmap, xmap, p);
}

template <typename T>
int launch_type(const GemmOperand& x, const GemmOperand& w, const LinearLogprobsParams& q, float* parts,
                float* token_logit, int dtype, cudaStream_t stream) {
  FewParams p{};
  p.tokens = q.tokens;
  p.bias = q.bias;
  p.parts = parts;
  p.token_logit = token_logit;
  p.rows = (int)q.rows;
  p.vocab = (int)q.vocab;
  p.tiles = (int)((q.vocab + kFewTile - 1) / kFewTile);
  p.k_blocks = (int)((q.d + kBK - 1) / kBK);
  p.status = q.status;
  const int blocks = linear_logprobs_few_parts(q.vocab) / 4;
  if (p.rows <= 16) return launch<T, 16>(x, w, p, dtype, blocks, stream);
  if (p.rows <= 32) return launch<T, 32>(x, w, p, dtype, blocks, stream);
  return launch<T, 64>(x, w, p, dtype, blocks, stream);
}

}  // namespace

int linear_logprobs_few_parts(int64_t vocab) {
  return 4 * (int)std::min<int64_t>(kSms, (vocab + kFewTile - 1) / kFewTile);
}

int launch_linear_logprobs_few(const GemmOperand& x, const GemmOperand& w, const LinearLogprobsParams& p, float* parts,
                               float* token_logit, int dtype, cudaStream_t stream) {
  return dtype == kBF16 ? launch_type<__nv_bfloat16>(x, w, p, parts, token_logit, dtype, stream)
                        : launch_type<__half>(x, w, p, parts, token_logit, dtype, stream);
}

}  // namespace wf

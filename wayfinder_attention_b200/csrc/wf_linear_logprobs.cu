// Log probabilities of given tokens and entropies from hidden rows and the head's weight,
// with their backward, in pieces of the vocabulary: the logits are never in memory.
//
//   z_j = x . w_j + b_j,  L = log sum_j exp z_j,  logprob = z_t - L,  H = L - sum_j p_j z_j
//   dz_j = gl (1[j = t] - p_j) - gh p_j (z_j - L + H),   p_j = exp(z_j - L)
//   dx = dz W,  dW = dz^T x,  db = sum_rows dz
//
// Forward: the tensor-core product (wf_gemm_kernel.cuh) whose epilogue keeps, for each row
// of its run of tiles, a base m, s = sum exp(z - m) and u = sum exp(z - m) (z - m), and
// picks the token's logit; a second kernel joins the runs' shares, and L = m + log s,
// H = log s - u / s.
//
// Backward: for a piece of the vocabulary at a time the same product again, whose epilogue
// makes dz of each logit and stores it in the operands' type; then dx += dz W over the piece
// (in fp32) and the piece's rows of dW.  Four products where three would do if the logits
// were kept: that is the price of not keeping them.
#include "wf_columns.cuh"
#include "wf_gemm_kernel.cuh"
#include "wf_linear_logprobs.cuh"
#include "wf_linear_logprobs_plan.h"
#include "wf_operand.cuh"
#include "wf_pair.cuh"

#include <cfloat>

namespace wf {
namespace {

constexpr int kShares = 4;  // epilogue warps that share a row of a tile, in every shape here

// ------------------------------------------------------------------ forward
// Running sums of a row over its run of tiles: s and u to a base m that is a logit of the row, though not
// always the largest.  A slice is taken with the base there is: three instructions and one exponential
// a logit.  Where its sum passes kBar, or it meets an infinity or NaN, and for the first slice,
// the base becomes the largest so far and the slice is done again.  -inf counts as nothing; a NaN or
// +inf stays in m (the sums may lose it); m is -inf while nothing has counted.
//
// The bar is for rows that are sure of a token.  z - m of such a token and log s cancel, so its base has to be
// that token: then z - m is 0, s is 1 or more and u 0 or less, and no log probability is above 0 and no
// entropy below.  With a base more than log(kBar) below it the slice is done again; with one that is nearer,
// the base itself keeps 1 - p above 1 / (1 + kBar).  (With 2^64 sure rows were off by 3e-6 in the log
// probability and 3e-5 in the entropy, with the sign as it fell.)  A slice of 32 logits below its base adds up to
// 32 at most; above that it is a matter of how many slices are done twice.  Over 32768 rows, 256 -> 50001, logits of a
// standard deviation of 2.5 take 731 to 772 us with 64, 256, 1024 and 2^64 alike, of 5: 847, 837, 802 and 789, of 10:
// 877, 859, 854 and 791.
constexpr float kBar = 256.f;
struct ScoreStats {
  static constexpr bool kRuns = true, kStores = false;
  static constexpr int kBuffers = 0;
  const int64_t* tokens;
  float* parts;        // [3][ranges * kShares][M]: m, s, u
  float* token_logit;  // [M]
  int64_t part_rows;   // ranges * kShares * M
  struct Row {
    float m, s, u;
    int token;
  };
  __device__ __forceinline__ void begin(Row& r, int row, int M, int N) const {
    r.m = -INFINITY;
    r.s = r.u = 0.f;
    const int64_t t = row < M ? tokens[row] : -1;
    r.token = t >= 0 && t < N ? (int)t : -1;
  }
  template <int SC>
  __device__ __forceinline__ void slice(Row& r, float* v, int row, int n, int N) const {
    if (n + SC > N) {
#pragma unroll
      for (int j = 0; j < SC; ++j)
        if (n + j >= N) v[j] = -INFINITY;
    }
    if ((uint32_t)(r.token - n) < (uint32_t)SC) {
      float z = v[0];
#pragma unroll
      for (int j = 1; j < SC; ++j)
        if (n + j == r.token) z = v[j];
      token_logit[row] = z;
    }
    float s0, s1, u0, u1;
    bool none = false;
#pragma unroll 1
    for (int again = 0;; ++again) {
      Pair s[2] = {Pair(0.f), Pair(0.f)}, u[2] = {Pair(0.f), Pair(0.f)};
      const Pair m(-r.m), log2e(kLog2e);
#pragma unroll
      for (int j = 0; j < SC; j += 2) {
        const Pair t = add2(Pair(v[j], v[j + 1]), m);
        float p0, p1;
        mul2(t, log2e).get(p0, p1);
        const Pair e(exp2_approx(p0), exp2_approx(p1));
        s[j / 2 % 2] = add2(s[j / 2 % 2], e);
        u[j / 2 % 2] = fma2(e, t, u[j / 2 % 2]);
      }
      add2(s[0], s[1]).get(s0, s1);
      add2(u[0], u[1]).get(u0, u1);
      s0 += s1;
      u0 += u1;
      if (again || __all_sync(0xffffffffu, s0 < kBar && u0 == u0)) break;
      float top = r.m;
#pragma unroll
      for (int j = 0; j < SC; j += 2) top = max_keep_nan(top, v[j], v[j + 1]);
      // far enough below the largest to have no weight, and near enough for the difference to be finite
      const float low = fmaxf(top - 0.5f * fabsf(top) - 1e5f, -FLT_MAX);
      const float d = fmaxf(r.m - top, kNothing), a = exp2_approx(d * kLog2e);
      r.u = a * fmaf(r.s, d, r.u);
      r.s *= a;
      r.m = top;
      none = top == -INFINITY;
      if (top == -FLT_MAX) {  // nothing finite is below it: a -inf will add its weight of 1, which comes off here
#pragma unroll
        for (int j = 0; j < SC; ++j) r.s -= v[j] == -INFINITY ? 1.f : 0.f;
      }
#pragma unroll
      for (int j = 0; j < SC; ++j) v[j] = fmaxf(v[j], low);
    }
    r.s += none ? 0.f : s0;
    r.u += none ? 0.f : u0;
  }
  __device__ __forceinline__ void end(const Row& r, int row, int M, int part) const {
    if (row >= M) return;
    float* to = parts + (int64_t)part * M + row;
    to[0] = r.m;
    to[part_rows] = r.s;
    to[2 * part_rows] = r.u;
  }
};

// Joins the parts of R rows a block: its threads share the parts, R neighbours a row each.
constexpr int kJoinThreads = 256;
template <int R>
__global__ void __launch_bounds__(kJoinThreads) linear_logprobs_join_kernel(const float* parts, int n_parts,
                                                                            const float* token_logit,
                                                                            LinearLogprobsParams p) {
  __shared__ float sm[kJoinThreads], ss[kJoinThreads], su[kJoinThreads];
  pdl_wait();
  const int64_t row = (int64_t)blockIdx.x * R + threadIdx.x % R, stride = (int64_t)n_parts * p.rows;
  float m = -INFINITY, s = 0.f, u = 0.f;
  if (row < p.rows)
#pragma unroll 4
    for (int i = threadIdx.x / R; i < n_parts; i += kJoinThreads / R) {
      const float* at = parts + (int64_t)i * p.rows + row;
      join_sums(m, s, u, at[0], at[stride], at[2 * stride]);
    }
  for (int half = kJoinThreads / 2; half >= R; half /= 2) {
    sm[threadIdx.x] = m;
    ss[threadIdx.x] = s;
    su[threadIdx.x] = u;
    __syncthreads();
    if ((int)threadIdx.x < half)
      join_sums(m, s, u, sm[threadIdx.x + half], ss[threadIdx.x + half], su[threadIdx.x + half]);
    __syncthreads();
  }
  if (threadIdx.x >= R || row >= p.rows) return;
  const bool none = m == -INFINITY;
  const bool bad = !(m < INFINITY);  // NaN or +inf
  const float log_s = none ? -INFINITY : logf(s);
  const int64_t tok = p.tokens[row];
  float lp;
  if (tok == p.ignore_index) {
    lp = 0.f;
  } else if (tok < 0 || tok >= p.vocab) {
    lp = NAN;
    if (p.status) atomicOr(p.status, 1);
  } else {
    lp = bad ? NAN : none ? -INFINITY : token_logit[row] - m - log_s;
  }
  p.logprob[row] = lp;
  p.entropy[row] = bad ? NAN : none ? 0.f : log_s - u / s;
  if (p.stats) {
    p.stats[row] = m;
    p.stats[p.rows + row] = log_s;
  }
}

// ------------------------------------------------------------------ backward
// A row's gradients, of its token's log probability (0 where that is not asked for) and its entropy.
struct RowInputs {
  const int64_t* tokens;
  const float* stats;  // [2][rows]
  const float* entropy;
  const float* dlogprob;  // or null
  const float* dentropy;  // or null
  int64_t rows, vocab, ignore_index;
  // The token in the vocabulary, or -1.  One outside of it that a gradient is asked for makes that NaN.
  __device__ __forceinline__ int gradients(int64_t row, float& gl, float& gh) const {
    gl = dlogprob ? dlogprob[row] : 0.f;
    gh = dentropy ? dentropy[row] : 0.f;
    const int64_t t = tokens[row];
    if (t != ignore_index && t >= 0 && t < vocab) return (int)t;
    gl = t == ignore_index || gl == 0.f ? 0.f : NAN;
    return -1;
  }
};

// fp16 has no room for p of a gradient that is small itself (a mean over many rows): there a row's
// gradient is multiplied by a power of two 2^h.  dx takes it off again by rows; for dW, x's rows are multiplied by
// 2^(least - h) and the product by 2^-least.
//
// e brings |gl| + 32 |gh|, which bounds |dz|, to 2^14 .. 2^15, and least is the smallest e, that of the largest
// gradient.  x's rows are normal fp16 numbers down to 2^-14 only, so h is not e but up to kSpare less: rows up to
// 2^10 below the largest leave x as it is, and those up to 2^24 below it still cost x no more than half its
// last bit at |x| = 1 (2^14 with h = e).  dz's smallest steps are then 2^-28 of the row's gradient instead of 2^-38: over
// 131072 tokens what they can lose is 2^-12 of the distribution.
constexpr int kSpare = 10;
constexpr int kNoRow = 1000;  // the exponent of a row without a gradient
__device__ __forceinline__ int held(int e, int least) { return max(e - kSpare, least); }
__global__ void __launch_bounds__(256) linear_logprobs_exponents_kernel(RowInputs in, int* exponent) {
  pdl_wait();
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int e = kNoRow;
  if (row < in.rows) {
    float gl, gh;
    in.gradients(row, gl, gh);
    const float size = fabsf(gl) + 32.f * fabsf(gh);
    if (in.stats[row] != -INFINITY && !(size == 0.f))
      e = size < INFINITY ? min(max(14 - ilogbf(size), -100), 100) : 0;
    exponent[row] = e;
  }
  const int least = __reduce_min_sync(0xffffffffu, e);
  if ((threadIdx.x & 31) == 0 && least != kNoRow) atomicMin(exponent + in.rows, least);
}
// 2^(least - h) and 2^-h of a row, and 2^-least: no row has a gradient where there is no least exponent.
__device__ __forceinline__ float down_by(int e, int least) {
  return least > 100 || e > 100 ? 0.f : ldexpf(1.f, least - held(e, least));
}
__device__ __forceinline__ float up_by(int e, int least) { return least > 100 || e > 100 ? 0.f : ldexpf(1.f, -held(e, least)); }
__device__ __forceinline__ float up_by(int least) { return least > 100 ? 0.f : ldexpf(1.f, -least); }

// Rounding dz to one piece of its type costs most where |dz| is large: at the row's token, where it is
// |gl| or a little less.  A value just above a power of two is rounded twice as coarsely for its size as one
// just below the next, and where all |gl| are alike (the mean of a loss) each row is off to the same
// side, by up to half a step of the type.  So dz is multiplied by 0.8125 / m (below 1: nothing overflows by it),
// m in [1, 2) the mean |gl|'s mantissa, which puts that mean at 1.625 of its binade, and the products by its reciprocal in fp32: equal |gl| then have no
// rounding of their own, and others are in the finer part of their binade: with |gl| of 1 +- 0.2 the
// gradients' error, of which their own rounding is 1, is 1.37 (1.26 to 1.43 over 96 to 1024 rows)
// where it was 1.45 (to 1.53).  3 us more a backward, and nothing in the products.
// The mean is over 4096 rows at most, evenly apart: any factor gives the same gradients to rounding.
constexpr int kFactorThreads = 1024, kFactorRows = 4096;
__global__ void __launch_bounds__(kFactorThreads) linear_logprobs_factor_kernel(RowInputs in, float* factor) {
  __shared__ float sums[32], counts[32];
  pdl_wait();
  const int64_t apart = (in.rows + kFactorRows - 1) / kFactorRows;
  float sum = 0.f, count = 0.f;
  for (int64_t row = threadIdx.x * apart; row < in.rows; row += kFactorThreads * apart) {
    float gl, gh;
    in.gradients(row, gl, gh);
    if (gl != 0.f && fabsf(gl) < INFINITY) {
      sum += fabsf(gl) * 0x1p-12f;  // 4096 of the largest are finite
      count += 1.f;
    }
  }
  auto over_warp = [](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  sum = over_warp(sum);
  count = over_warp(count);
  if ((threadIdx.x & 31) == 0) {
    sums[threadIdx.x / 32] = sum;
    counts[threadIdx.x / 32] = count;
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  sum = over_warp(sums[threadIdx.x]);
  count = over_warp(counts[threadIdx.x]);
  if (threadIdx.x) return;
  const float mean = sum / count;  // NaN where there are none
  const float c = mean > 0.f ? 0.8125f / scalbnf(mean, -ilogbf(mean)) : 1.f;
  factor[0] = c;
  factor[1] = 1.f / c;
}

// dz_j = p (a + b t) + g [j = token] with t = (z - m) log2 e - l2s and p = 2^t.
struct ScoreGrad {
  static constexpr bool kRuns = true, kStores = true;
  static constexpr int kBuffers = 1;
  int layers;
  int first;  // of the vocabulary's piece
  RowInputs in;
  const int* exponent;  // [rows], then the least; or null
  const float* factor;  // or null
  struct Row {
    float m, l2s, a, b, g;
    int token;
  };
  __device__ __forceinline__ void begin(Row& r, int row, int M, int) const {
    r = Row{0.f, INFINITY, 0.f, 0.f, 0.f, -1};  // no row, no distribution or no gradient: p is 0
    if (row >= M) return;
    float gl, gh;
    const int token = in.gradients(row, gl, gh);
    const float m = in.stats[row];
    if (m == -INFINITY || (gl == 0.f && gh == 0.f)) return;
    r.token = token - first;
    r.g = gl;
    if (!(m < INFINITY)) {  // a NaN or +inf among the row's logits
      r.l2s = 0.f;
      r.a = NAN;
      return;
    }
    r.m = m;
    r.l2s = in.stats[in.rows + row] * kLog2e;
    r.a = -fmaf(gh, in.entropy[row], gl);
    r.b = -gh * kLn2;
    if (exponent || factor) {
      const float up = (exponent ? ldexpf(1.f, held(exponent[row], exponent[in.rows])) : 1.f) * (factor ? *factor : 1.f);
      r.a *= up;
      r.b *= up;
      r.g *= up;
    }
  }
  template <int SC>
  __device__ __forceinline__ void slice(const Row& r, float* v, int, int n, int) const {
#pragma unroll
    for (int j = 0; j < SC; j += 2) {
      float t0, t1;
      fma2(add2(Pair(v[j], v[j + 1]), Pair(-r.m)), Pair(kLog2e), Pair(-r.l2s)).get(t0, t1);
      t0 = fmaxf(t0, kNothing);
      t1 = fmaxf(t1, kNothing);
      const Pair e(exp2_approx(t0), exp2_approx(t1));
      mul2(e, fma2(Pair(t0, t1), Pair(r.b), Pair(r.a))).get(v[j], v[j + 1]);
    }
    if ((uint32_t)(r.token - n) < (uint32_t)SC) {
#pragma unroll
      for (int j = 0; j < SC; ++j)
        if (n + j == r.token) v[j] += r.g;
    }
  }
  __device__ __forceinline__ void end(const Row&, int, int, int) const {}
};

// x's rows multiplied by 2^(least - h): the fp16 operand of dW.
__global__ void __launch_bounds__(256) scale_rows_kernel(const __half* x, int64_t stride, bool vec, int64_t rows,
                                                         int64_t cols, const int* exponent, __half* out) {
  pdl_wait();
  const int least = exponent[rows];
  const int64_t pitch = (cols + 7) / 8 * 8, groups = pitch / 8, total = rows * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / groups, c = i % groups * 8;
    Raw8<__half> raw;
    raw.load(x + r * stride, c, cols, vec);
    float f[8];
    raw.unpack(f);
    const float s = down_by(exponent[r], least);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= s;
    store_vec<__half, 8>(out + r * pitch + c, f);
  }
}

// fp32 rows to their type, with the power of two taken off where there is one (by rows, or the
// whole by the least exponent), and the factor.
template <typename T>
__global__ void __launch_bounds__(256) round_rows_kernel(const float* x, int64_t pitch, int64_t rows, int64_t cols,
                                                         const int* exponent, const int* least, const float* factor,
                                                         T* out) {
  pdl_wait();
  const int64_t groups = (cols + 3) / 4, total = rows * groups;
  const bool vec = cols % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const float down = factor ? factor[1] : 1.f, all = (least ? up_by(*least) : 1.f) * down;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / groups, c = i % groups * 4;
    const float4 f = *reinterpret_cast<const float4*>(x + r * pitch + c);
    const float s = exponent ? up_by(exponent[r], exponent[rows]) * down : all;
    const float v[4] = {f.x * s, f.y * s, f.z * s, f.w * s};
    T* to = out + r * cols + c;
    if (vec) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>(to) = make_uint2(pack2(T(), v[0], v[1]), pack2(T(), v[2], v[3]));
    } else {
      for (int j = 0; j < 4 && c + j < cols; ++j) to[j] = from_f32<T>(v[j]);
    }
  }
}

// Partial column sums of dz: a block takes 256 columns (8 a lane) of a share of the rows.
template <typename T>
__global__ void __launch_bounds__(256) dz_columns_kernel(const T* dz, int64_t pitch, int layers, int64_t M, int64_t N,
                                                         const int* exponent, const float* factor, float* partials) {
  __shared__ float red[8][32][9];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + lane) * 8;
  float s[8] = {};
  if (c < N)
    for (int64_t m = (int64_t)blockIdx.y * 8 + warp; m < M; m += (int64_t)gridDim.y * 8) {
      const float up = exponent ? up_by(exponent[m], exponent[M]) : 1.f;
      for (int layer = 0; layer < layers; ++layer) {
        Raw8<T> raw;
        raw.load(dz + (layer * M + m) * pitch, c, pitch, true);
        float f[8];
        raw.unpack(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = fmaf(f[j], up, s[j]);
      }
    }
#pragma unroll
  for (int j = 0; j < 8; ++j) red[warp][lane][j] = s[j];
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col < N) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += red[i][threadIdx.x / 8][threadIdx.x % 8];
    partials[(size_t)blockIdx.y * N + col] = factor ? v * factor[1] : v;
  }
}
// ------------------------------------------------------------------ plans
// Tile shape, runs and their order for the logits' product: the least of an estimate, as for other
// products (wf_gemm.cu), but a tile takes at least the 8 cycles a column that the exponentials of
// 128 rows need.
constexpr Shape kRunShapes[] = {{256, 2, 560, 0}, {128, 2, 400, 1700}, {128, 1, 540, 0}, {64, 1, 0, 1300}};
constexpr int kMaxRanges = 1024;
constexpr double kGroupBytes = 48e6;  // of A that a group's rows of tiles may have, to stay in L2
Plan run_plan(int64_t M, int64_t N, int64_t K, int pieces) {
  Plan best{};
  double least = 0;
  for (const Shape& s : kRunShapes) {
    const int cycles = pieces > 1 ? s.cycles3 : s.cycles;
    if (!cycles) continue;
    Plan p{};
    p.shape = s;
    p.splits = p.layers = 1;
    p.k_blocks = (int)((K + kBK - 1) / kBK);
    const int64_t tn = (N + s.bn - 1) / s.bn, tm = (M + kBM * s.cg - 1) / (kBM * s.cg);
    p.tiles_n = (int)tn;
    p.tiles_m = (int)tm;
    p.group = (int)std::max(1.0, std::min((double)tm, kGroupBytes / ((double)kBM * s.cg * K * 2 * pieces)));
    const int slots = kSms / s.cg;
    const double tile = std::max<double>((double)p.k_blocks * cycles, 8 * s.bn);
    // for each number of waves as many ranges as it holds, and one for each tile of columns
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>({tn, kMaxRanges, (1 << 30) / tm}));  // units in 32 bits
    for (int64_t n = 1, ranges = 0; ranges < most; ++n) {
      ranges = n > 64 ? most : std::min(most, std::max<int64_t>(ranges + 1, n * slots / tm));
      const double waves = (double)((tm * ranges + slots - 1) / slots), length = (double)((tn + ranges - 1) / ranges);
      // a wave ends with an epilogue that nothing covers; the parts are written and read once
      const double t = waves * (length * tile + 8 * s.bn) + 24.0 * kShares * ranges * M / 2000;
      if (best.ranges == 0 || t < least) {
        least = t;
        best = p;
        best.ranges = (int)ranges;
      }
    }
  }
  return best;
}

template <typename T, class E>
int launch_runs(const GemmProblem& g, const GemmEpilogue& out, const Plan& plan, const E& e, cudaStream_t stream) {
  constexpr bool PIECES = std::is_same<T, float>::value;
  const Shape& s = plan.shape;
  if constexpr (PIECES) {
    if (s.cg == 2) return launch_tile<T, 128, 2, true>(g, out, plan, e, stream);
    return launch_tile<T, 64, 1, true>(g, out, plan, e, stream);
  } else {
    if (s.bn == 256) return launch_tile<T, 256, 2, false>(g, out, plan, e, stream);
    if (s.cg == 2) return launch_tile<T, 128, 2, false>(g, out, plan, e, stream);
    return launch_tile<T, 128, 1, false>(g, out, plan, e, stream);
  }
}

bool few_rows(int64_t M, int dtype) { return M <= kFewLogprobRows && dtype != kF32; }
size_t parts_bytes(int parts, int64_t M) {
  return round256((size_t)3 * parts * M * sizeof(float)) + round256((size_t)M * sizeof(float));
}

template <typename T>
int launch_fwd(const LinearLogprobsParams& p, int dtype, cudaStream_t stream) {
  unsigned char* ws = static_cast<unsigned char*>(p.ws);
  GemmOperand o[2];
  if (int rc = operands<T>({{p.x, p.rows, p.d, p.x_stride}, {p.w, p.vocab, p.d, p.w_stride}}, dtype, &ws, o, stream))
    return rc;
  const bool few = few_rows(p.rows, dtype);
  const Plan plan = few ? Plan{} : run_plan(p.rows, p.vocab, p.d, kPieces<T>);
  const int n_parts = few ? linear_logprobs_few_parts(p.vocab) : plan.ranges * kShares;
  float* parts = reinterpret_cast<float*>(ws);
  float* token_logit = reinterpret_cast<float*>(ws + round256((size_t)3 * n_parts * p.rows * sizeof(float)));
  if (few) {
    if (int rc = launch_linear_logprobs_few(o[0], o[1], p, parts, token_logit, dtype, stream)) return rc;
  } else {
    GemmProblem g = problem<T>(o[0], o[1], p.rows, p.vocab, p.d, dtype, nullptr, p.status);
    GemmEpilogue out{};
    out.bias = p.bias;
    if (int rc = launch_runs<T>(g, out, plan, ScoreStats{p.tokens, parts, token_logit, n_parts * p.rows}, stream)) return rc;
  }
  auto join = [&](auto rows_a_block) {
    constexpr int R = decltype(rows_a_block)::value;
    return (int)launch_pdl(linear_logprobs_join_kernel<R>, dim3((unsigned)((p.rows + R - 1) / R)), dim3(kJoinThreads),
                           0, stream, static_cast<const float*>(parts), n_parts, static_cast<const float*>(token_logit), p);
  };
  // a sector's rows, or one row a block where they are few and their parts many
  if (p.rows <= kSms) return join(std::integral_constant<int, 1>());
  return p.rows <= 32 * kSms ? join(std::integral_constant<int, 8>()) : join(std::integral_constant<int, 32>());
}

// A call asks for its workspace's size and is then launched: 4 us of a plan's making, once.
BwdPlan bwd_plan(int64_t M, int64_t N, int64_t K, int dtype) {
  struct Last {
    int64_t M, N, K;
    int dtype;
    BwdPlan plan;
  };
  thread_local Last last{};
  if (last.M != M || last.N != N || last.K != K || last.dtype != dtype)
    last = Last{M, N, K, dtype, make_bwd_plan(M, N, K, dtype)};
  return last.plan;
}

template <typename T>
int launch_bwd(const LinearLogprobsBwdParams& p, int dtype, cudaStream_t stream) {
  const int64_t M = p.rows, N = p.vocab, K = p.d;
  if (M == 0) {  // sums over no rows
    for (auto [ptr, n] : {std::pair<void*, size_t>{p.dw, (size_t)N * K}, {p.db, (size_t)N}})
      if (ptr)
        if (cudaError_t e = cudaMemsetAsync(ptr, 0, n * sizeof(T), stream)) return (int)e;
    return 0;
  }
  const BwdPlan b = bwd_plan(M, N, K, dtype);
  unsigned char* ws = static_cast<unsigned char*>(p.ws);
  auto take = [&](size_t bytes) {
    unsigned char* at = ws;
    ws += bytes;
    return at;
  };
  int* exponents = reinterpret_cast<int*>(take(b.exponents));
  const int *exponent = b.scaled ? exponents : nullptr, *least = b.scaled ? exponents + M : nullptr;
  float* factor = b.factor ? reinterpret_cast<float*>(take(b.factor)) : nullptr;
  unsigned char* dz = take(b.dz);
  unsigned char* dz_operand = take(b.dz_operand);
  float* dx = reinterpret_cast<float*>(take(b.dx));
  float* dw = reinterpret_cast<float*>(take(b.dw));
  float* sums = reinterpret_cast<float*>(take(b.sums));
  unsigned char* scaled_x = take(b.scaled_x);
  unsigned char* gemm_ws = take(b.gemm);
  GemmOperand o[2];
  if (int rc = operands<T>({{p.x, M, K, p.x_stride}, {p.w, N, K, p.w_stride}}, dtype, &ws, o, stream)) return rc;
  const RowInputs in{p.tokens, p.stats, p.entropy, p.dlogprob, p.dentropy, M, N, p.ignore_index};
  if (b.scaled) {
    // a least exponent above every row's
    if (cudaError_t e = cudaMemsetAsync(exponents + M, 0x7f, sizeof(int), stream)) return (int)e;
    if (cudaError_t e = launch_pdl(linear_logprobs_exponents_kernel, dim3((unsigned)((M + 255) / 256)), dim3(256), 0,
                                   stream, in, exponents))
      return (int)e;
  }
  if (factor)
    if (cudaError_t e = launch_pdl(linear_logprobs_factor_kernel, dim3(1), dim3(kFactorThreads), 0, stream, in, factor))
      return (int)e;
  GemmOperand x_deep = o[0];  // of dW, whose depth are the rows
  if constexpr (std::is_same<T, __half>::value) {
    if (p.dw) {
      x_deep = blank_operand<T>(M, K, dtype, &scaled_x);
      const int64_t blocks = (M * (round8(K) / 8) + 255) / 256;
      if (cudaError_t e = launch_pdl(scale_rows_kernel, dim3((unsigned)std::min<int64_t>(blocks, 16 * kSms)), dim3(256),
                                     0, stream, static_cast<const __half*>(p.x), p.x_stride,
                                     on_16_bytes<T>(p.x, p.x_stride), M, K, exponent,
                                     static_cast<__half*>(const_cast<void*>(x_deep.ptr))))
        return (int)e;
    }
  }
  x_deep.mn_major = true;
  auto round_rows = [&](const float* from, int64_t n, const int* by_row, const int* all, const float* by, T* to) {
    const int64_t blocks = (n * ((K + 3) / 4) + 255) / 256;
    return launch_pdl(round_rows_kernel<T>, dim3((unsigned)std::min<int64_t>(blocks, 16 * kSms)), dim3(256), 0, stream,
                      from, round8(K), n, K, by_row, all, by, to);
  };
  for (int64_t first = 0; first < N; first += b.columns) {
    const int64_t n = std::min(b.columns, N - first), pitch = round8(n);
    GemmOperand w = o[1];
    w.ptr = static_cast<const unsigned char*>(w.ptr) + first * w.pitch * 2;
    w.rows = n;
    {
      GemmProblem g = problem<T>(o[0], w, M, n, K, dtype, nullptr, p.status);
      GemmEpilogue out{};
      out.bias = p.bias ? static_cast<const T*>(p.bias) + first : nullptr;
      out.y = dz;
      out.y_stride = pitch;
      Plan plan = run_plan(M, n, K, b.pieces);
      plan.layers = b.layers;
      if (int rc = launch_runs<T>(g, out, plan, ScoreGrad{b.layers, (int)first, in, exponent, factor}, stream)) return rc;
    }
    if (p.db) {
      const int shares = column_shares(M, n);
      if (cudaError_t e = launch_pdl(dz_columns_kernel<T>, dim3((unsigned)((n + 255) / 256), shares), dim3(256), 0,
                                     stream, reinterpret_cast<const T*>(dz), pitch, b.layers, M, n, exponent, factor, sums))
        return (int)e;
      if (cudaError_t e = join_columns<T>(sums, shares, n, n, static_cast<T*>(p.db) + first, nullptr, stream))
        return (int)e;
    }
    GemmOperand d{dz, M, n, pitch, M * pitch, false};
    if (dtype == kF32) {
      GemmOperand laid[2];
      unsigned char* at = dz_operand;
      if (int rc = operands<T>({{dz, M, n, pitch}, {nullptr, 0, 0, 0}}, dtype, &at, laid, stream)) return rc;
      d = laid[0];
    }
    if (p.dx) {
      w.mn_major = true;  // its columns are dx's, its rows the depth
      GemmProblem g = problem<T>(d, w, M, K, n, dtype, gemm_ws, p.status);
      g.turns = b.layers;
      const bool apart = b.dx_apart;
      g.out.y = apart ? static_cast<void*>(dx) : p.dx;
      g.out.y_stride = apart ? round8(K) : K;
      if (apart) g.out_dtype = kF32;
      else if (factor) g.out.factor = factor + 1;
      if (first) {
        g.out.residual = g.out.y;
        g.out.r_stride = g.out.y_stride;
      }
      if (int rc = launch_gemm(g, stream)) return rc;
    }
    if (p.dw) {
      d.mn_major = true;  // the rows of both are the depth
      GemmProblem g = problem<T>(d, x_deep, n, K, M, dtype, gemm_ws, p.status);
      g.turns = b.layers;
      T* to = static_cast<T*>(p.dw) + first * K;
      g.out.y = b.dw_apart ? static_cast<void*>(dw) : to;
      g.out.y_stride = b.dw_apart ? round8(K) : K;
      if (b.dw_apart) g.out_dtype = kF32;
      else if (factor) g.out.factor = factor + 1;
      if (int rc = launch_gemm(g, stream)) return rc;
      if (b.dw_apart)
        if (cudaError_t e = round_rows(dw, n, nullptr, least, factor, to)) return (int)e;
    }
  }
  if (p.dx && b.dx_apart)
    if (cudaError_t e = round_rows(dx, M, exponent, nullptr, factor, static_cast<T*>(p.dx))) return (int)e;
  return 0;
}

}  // namespace

size_t linear_logprobs_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, bool x_direct, bool w_direct) {
  const int pieces = dtype == kF32 ? 3 : 1;
  return (x_direct && pieces == 1 ? 0 : operand_bytes(M, K, dtype)) +
         (w_direct && pieces == 1 ? 0 : operand_bytes(N, K, dtype)) + parts_bytes(few_rows(M, dtype) ? linear_logprobs_few_parts(N) : run_plan(M, N, K, pieces).ranges * kShares, M);
}

size_t linear_logprobs_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, bool x_direct,
                                                bool w_direct) {
  const BwdPlan b = bwd_plan(M, N, K, dtype);
  return b.exponents + b.factor + b.dz + b.dz_operand + b.dx + b.dw + b.sums + b.scaled_x + b.gemm +
         (x_direct && b.pieces == 1 ? 0 : operand_bytes(M, K, dtype)) +
         (w_direct && b.pieces == 1 ? 0 : operand_bytes(N, K, dtype));
}

int launch_linear_logprobs(const LinearLogprobsParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_fwd<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_fwd<__half>(p, dtype, stream);
  return launch_fwd<float>(p, dtype, stream);
}

int launch_linear_logprobs_backward(const LinearLogprobsBwdParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_bwd<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_bwd<__half>(p, dtype, stream);
  return launch_bwd<float>(p, dtype, stream);
}

}  // namespace wf

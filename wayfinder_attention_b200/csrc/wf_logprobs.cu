// Log probabilities of given tokens, with the entropy and the top alternatives, and
// their backward.
//
//   L = log sum_j exp x_j,  logprob = x_t - L,  H = L - sum_j p_j x_j,  p_j = exp(x_j - L)
//   dx_j = gl (1[j = t] - p_j) - gh p_j (x_j - L + H)
//
// One pass over the logits.  Each thread keeps the running maximum m of what it has
// read, s = sum exp(x - m) and u = sum exp(x - m) (x - m); a larger maximum M rescales
// them by a = exp(m - M):  s' = a s,  u' = a (u + (m - M) s).  Threads, warps and the
// blocks of a cluster combine by the same rule, and L = m + log s, H = log s - u / s.
// Everything is fp32 (logits are widened exactly).
//
// The top n are kept while the logits stream by: a warp holds its n best as sorted
// 64-bit keys, one a lane (the logit's bits in an order-preserving form above the
// inverted index, so equal logits rank by the lower index), and a vector is looked at
// only if its maximum reaches the warp's n-th.  Lists merge like the sums do.
//
// -inf is a token that cannot be said: p = 0, nothing added to H.  A row of nothing
// else has no distribution: logprob -inf, H 0, gradient 0.  A NaN (or +inf) makes its
// row's logprob and H NaN; NaN ranks first among the alternatives.
//
// Bound by bytes: one read of the logits; the backward reads them again and writes dx.
#include "wf_kernels.h"
#include "wf_rowio.cuh"
#include "wf_sm100.cuh"

namespace wf {
namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;
constexpr unsigned kAll = 0xffffffffu;

// exp2_approx with results below 2^-126 kept: a gradient multiplies them by what it likes
__device__ __forceinline__ float exp2_small(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

struct Sums {
  float m, s, u;
  // Moves the sums to the maximum M >= m.  Nothing read yet (m = -inf) has s = u = 0.
  __device__ __forceinline__ void rebase(float M) {
    if (m != M && m != -INFINITY) {
      // a is 0 long before d = -200; the bound keeps 0 * inf out when m is the type's lowest value
      const float d = max_nan(m - M, -200.f), a = exp2_approx(d * kLog2e);
      u = a * fmaf(d, s, u);
      s *= a;
    }
    m = M;
  }
  __device__ __forceinline__ void join(Sums o) {
    const float M = max_nan(m, o.m);
    rebase(M);
    o.rebase(M);
    s += o.s;
    u += o.u;
  }
  template <int N>
  __device__ __forceinline__ void add(const float* x, float most) {
    if (!(most <= m)) rebase(max_nan(m, most));
    const float base = m == -INFINITY ? 0.f : m;  // -inf - -inf would be NaN
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = x[j] - base, e = exp2_approx(d * kLog2e);
      s += e;
      u = fmaf(e, fmaxf(d, -1e30f), u);  // e = 0 where d = -inf
    }
  }
};

__device__ __forceinline__ Sums warp_join(Sums a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(kAll, a.m, o);
    b.s = __shfl_xor_sync(kAll, a.s, o);
    b.u = __shfl_xor_sync(kAll, a.u, o);
    a.join(b);
  }
  return a;
}

__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  const uint32_t k = x != x ? 0xffffffffu : ordered_key(x);
  return (uint64_t)k << 32 | (uint32_t)~index;
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) { return __shfl_xor_sync(kAll, v, o); }

// A warp's best keys: lane i holds the i-th largest so far (0: none).
struct TopList {
  uint64_t mine;
  float bar;  // what a candidate has to reach: the n-th's logit or a lower bound of it; it only rises
  __device__ __forceinline__ void clear() {
    mine = 0;
    bar = -INFINITY;
  }
  __device__ __forceinline__ void set_bar(int n) {
    const uint64_t k = __shfl_sync(kAll, mine, n - 1);
    const uint32_t hi = (uint32_t)(k >> 32);
    // an empty slot admits everything; a NaN at the n-th leaves nothing but NaN to admit
    bar = fmaxf(bar, hi == 0 ? -INFINITY : hi == 0xffffffffu ? INFINITY : key_to_float(hi));
  }
  // `other`: one key a lane, sorted in descending order over the lanes.
  __device__ __forceinline__ void merge_sorted(uint64_t other, int lane) {
    const uint64_t r = __shfl_sync(kAll, other, 31 - lane);
    uint64_t v = mine > r ? mine : r;  // the 32 largest of both, in bitonic order
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t w = shfl_xor64(v, o);
      v = ((lane & o) == 0) == (v > w) ? v : w;
    }
    mine = v;
  }
  // Any keys, one a lane (0: none).
  __device__ __forceinline__ void merge(uint64_t v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int o = k >> 1; o > 0; o >>= 1) {
        const uint64_t w = shfl_xor64(v, o);
        const bool down = (lane & k) == 0;
        v = (((lane & o) == 0) == down) == (v > w) ? v : w;
      }
    merge_sorted(v, lane);
  }
  // Called by the whole warp; `live` lanes offer x at index.
  __device__ __forceinline__ void offer(float x, uint32_t index, bool live, int n, int lane) {
    unsigned want = __ballot_sync(kAll, live && !(x < bar));
    if (!want) return;
    const uint64_t key = live ? rank_key(x, index) : 0;
    if (__popc(want) > 6) {
      merge((want >> lane & 1) ? key : 0, lane);
    } else {
      while (want) {
        const int src = __ffs(want) - 1;
        want &= want - 1;
        const uint64_t k = __shfl_sync(kAll, key, src);
        const int at = __popc(__ballot_sync(kAll, mine > k));
        const uint64_t up = __shfl_up_sync(kAll, mine, 1);
        mine = lane < at ? mine : lane == at ? k : up;
      }
    }
    set_bar(n);
  }
};

// How a row [lo, hi) of x splits around 16-byte boundaries: single elements before
// `head` and from `tail`, vectors between.
template <typename T>
struct Span {
  static constexpr int V = Vec16<T>::N;
  int64_t head, tail;
  __device__ __forceinline__ Span(const T* x, int64_t lo, int64_t hi) {
    const int64_t off = (int64_t)((16 - (reinterpret_cast<uintptr_t>(x + lo) & 15)) & 15) / (int64_t)sizeof(T);
    head = min(lo + off, hi);
    tail = head + (hi - head) / V * V;
  }
};

constexpr int kWarps = 8;     // of a block
constexpr int kUnroll = 4;    // vectors a thread requests at once

// One row a warp (WIDE = false), or one row a cluster of 1 to 8 blocks (WIDE = true).
template <typename T, bool WIDE, bool TOP>
__global__ void __launch_bounds__(kWarps * 32) token_logprobs_kernel(LogprobParams p) {
  constexpr int V = Vec16<T>::N;
  constexpr int G = WIDE ? kWarps * 32 : 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t parts = WIDE ? p.cluster : 1, part = WIDE ? blockIdx.x % parts : 0;
  const int64_t row = WIDE ? blockIdx.x / parts : (int64_t)blockIdx.x * kWarps + warp;
  if (!WIDE && row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  int64_t lo = 0, hi = p.vocab;
  if (WIDE) {
    const int64_t share = ((p.vocab + parts - 1) / parts + V - 1) / V * V;
    lo = min((int64_t)part * share, p.vocab);
    hi = min(lo + share, p.vocab);
  }
  const Span<T> span(x, lo, hi);

  Sums a{-INFINITY, 0.f, 0.f};
  TopList top;
  if (TOP) top.clear();
  // A warp's lanes stay together (the list is the warp's): bounds are tested a vector.
  const int64_t first = span.head + (int64_t)(WIDE ? warp * 32 : 0) * V;
  for (int64_t c0 = first; c0 < span.tail; c0 += (int64_t)G * V * kUnroll) {
    RawVec<T, V> raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int64_t c = c0 + ((int64_t)i * G + lane) * V;
      if (c < span.tail) raw[i].load(x + c);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int64_t c = c0 + ((int64_t)i * G + lane) * V;
      const bool live = c < span.tail;
      float f[V];
      float most = -INFINITY;
      if (live) {
        raw[i].unpack(f);
        most = f[0];
#pragma unroll
        for (int j = 1; j < V; ++j) most = max_nan(most, f[j]);
        a.template add<V>(f, most);
      }
      if constexpr (TOP) {
        if (__any_sync(kAll, live && !(most < top.bar))) {
          if (top.bar == -INFINITY && c0 == first && i == 0) {
            // the n-th largest of the lanes' maxima is a first bar: n elements reach it
            TopList firsts;
            firsts.clear();
            firsts.merge(live ? rank_key(most, lane) : 0, lane);
            firsts.set_bar(p.top_n);
            top.bar = firsts.bar;
          }
#pragma unroll
          for (int j = 0; j < V; ++j) top.offer(live ? f[j] : 0.f, (uint32_t)(c + j), live, p.top_n, lane);
        }
      }
    }
  }
  // the ends: fewer than V elements each, offered by the first warp of the row
  if (!WIDE || warp == 0) {
    const int64_t n_head = span.head - lo, n_tail = hi - span.tail;
    const int64_t c = lane < n_head ? lo + lane : span.tail + (lane - n_head);
    const bool live = lane < n_head + n_tail;
    float f = 0.f;
    if (live) {
      f = to_f32(x[c]);
      a.template add<1>(&f, f);
    }
    if constexpr (TOP) top.offer(f, (uint32_t)c, live, p.top_n, lane);
  }
  a = warp_join(a);

  if constexpr (WIDE) {
    __shared__ Sums sums[8];  // of the cluster's blocks, in its first block
    __shared__ uint64_t keys[8][kMaxTopTokens];
    __shared__ uint64_t own[kWarps][kMaxTopTokens];
    __shared__ Sums own_sums[kWarps];
    if (lane == 0) own_sums[warp] = a;
    if (TOP) own[warp][lane] = top.mine;
    __syncthreads();
    if (warp == 0) {
      a = lane < kWarps ? own_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
      a = warp_join(a);
      if constexpr (TOP)
        for (int w = 1; w < kWarps; ++w) top.merge_sorted(own[w][lane], lane);
    }
    if (parts > 1) {
      if (warp == 0 && part > 0) {
        if (lane == 0) {
          const uint32_t d = map_peer(&sums[part], 0);
          st_peer_u32(d, __float_as_uint(a.m));
          st_peer_u32(d + 4, __float_as_uint(a.s));
          st_peer_u32(d + 8, __float_as_uint(a.u));
        }
        if (TOP) {
          const uint32_t d = map_peer(&keys[part][lane], 0);
          st_peer_u32(d, (uint32_t)top.mine);
          st_peer_u32(d + 4, (uint32_t)(top.mine >> 32));
        }
      }
      __syncwarp();
      cluster_sync();
      if (part > 0) return;
      if (warp == 0) {
        Sums b{-INFINITY, 0.f, 0.f};
        if (lane == 0) b = a;
        else if (lane < (int)parts) b = sums[lane];
        a = warp_join(b);
        if constexpr (TOP)
          for (uint32_t r = 1; r < parts; ++r) top.merge_sorted(keys[r][lane], lane);
      }
    }
    if (warp != 0) return;
  }

  const float log_s = logf(a.s);  // -inf for a row without a distribution
  const bool none = a.s == 0.f;
  if (lane == 0) {
    const int64_t tok = p.tokens[row];
    float lp;
    if (tok == p.ignore_index) {
      lp = 0.f;
    } else if (tok < 0 || tok >= p.vocab) {
      lp = NAN;
      if (p.status) atomicOr(p.status, 1);
    } else {
      lp = none ? -INFINITY : to_f32(x[tok]) - a.m - log_s;
    }
    p.logprob[row] = lp;
    p.entropy[row] = none ? 0.f : log_s - a.u / a.s;
    if (p.stats) {  // apart, so that p = exp((x - m) - log s) keeps its bits however large the logits are
      p.stats[row] = a.m;
      p.stats[p.rows + row] = log_s;
    }
  }
  if constexpr (TOP) {
    if (lane < p.top_n) {
      const uint32_t hi32 = (uint32_t)(top.mine >> 32), index = ~(uint32_t)top.mine;
      const float v = hi32 == 0xffffffffu ? NAN : key_to_float(hi32);
      p.top_logprobs[row * p.top_n + lane] = none ? -INFINITY : v - a.m - log_s;
      p.top_tokens[row * p.top_n + lane] = index;
    }
  }
}

// One row a warp (WIDE = false) or kSpan elements of a row a block (WIDE = true).
constexpr int64_t kBwdVectors = 4;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) token_logprobs_backward_kernel(LogprobBwdParams p, int64_t chunks) {
  constexpr int V = Vec16<T>::N;
  constexpr int G = WIDE ? kWarps * 32 : 32;
  const int t = WIDE ? (int)threadIdx.x : (int)(threadIdx.x & 31);
  const int64_t row = WIDE ? blockIdx.x / chunks : (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (!WIDE && row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  T* dx = static_cast<T*>(p.dx) + row * p.vocab;
  int64_t lo = 0, hi = p.vocab;
  if (WIDE) {
    const int64_t share = ((p.vocab + chunks - 1) / chunks + V - 1) / V * V;
    lo = min(blockIdx.x % chunks * share, p.vocab);
    hi = min(lo + share, p.vocab);
  }
  const int64_t tok = p.tokens[row];
  const float m = p.stats[row], log_s = p.stats[p.rows + row], h = p.entropy[row];
  const float gh = p.dentropy ? p.dentropy[row] : 0.f;
  float gl = p.dlogprob ? p.dlogprob[row] : 0.f;
  if (tok == p.ignore_index) gl = 0.f;
  else if (tok < 0 || tok >= p.vocab) gl = NAN;
  const bool none = m == -INFINITY;
  const float base = fmaf(gh, h, gl);
  auto grad = [&](float v, int64_t c) {
    const float lp = v - m - log_s, pr = exp2_small(lp * kLog2e);
    // p is 0 long before lp = -200; the bound keeps 0 * inf out
    float g = -pr * fmaf(gh, fmaxf(lp, -200.f), base);
    if (c == tok) g += gl;
    return none ? 0.f : g;
  };
  const Span<T> span(x, lo, hi);
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  for (int64_t c0 = span.head + (int64_t)t * V; c0 < span.tail; c0 += (int64_t)G * V * kBwdVectors) {
    RawVec<T, V> raw[kBwdVectors];
#pragma unroll
    for (int i = 0; i < kBwdVectors; ++i) {
      const int64_t c = c0 + (int64_t)i * G * V;
      if (c < span.tail) raw[i].load(x + c);
    }
#pragma unroll
    for (int i = 0; i < kBwdVectors; ++i) {
      const int64_t c = c0 + (int64_t)i * G * V;
      if (c < span.tail) {
        float f[V];
        raw[i].unpack(f);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = grad(f[j], c + j);
        if (same) {
          store_vec<T, V>(dx + c, f);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) dx[c + j] = from_f32<T>(f[j]);
        }
      }
    }
  }
  const int64_t n_head = span.head - lo, n_tail = hi - span.tail;
  if (t < n_head + n_tail) {
    const int64_t c = t < n_head ? lo + t : span.tail + (t - n_head);
    dx[c] = from_f32<T>(grad(to_f32(x[c]), c));
  }
}

// A warp takes a row of up to 1024 logits (4 KB at most); longer rows take a block, and
// a cluster of up to 8 when there are fewer rows than SMs to give them to.
constexpr int64_t kWarpRow = 1024;

template <typename T>
int launch_fwd(LogprobParams p, cudaStream_t stream) {
  if (p.vocab <= kWarpRow) {
    const unsigned grid = (unsigned)((p.rows + kWarps - 1) / kWarps);
    if (p.top_n) token_logprobs_kernel<T, false, true><<<grid, kWarps * 32, 0, stream>>>(p);
    else token_logprobs_kernel<T, false, false><<<grid, kWarps * 32, 0, stream>>>(p);
    return (int)cudaGetLastError();
  }
  int c = 1;
  while (c < 8 && p.rows * c <= kSms && p.vocab / c > 4 * kWarpRow) c *= 2;
  p.cluster = c;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * c));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)(p.top_n ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true, true>, p)
                       : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true, false>, p));
}

template <typename T>
int launch_bwd(const LogprobBwdParams& p, cudaStream_t stream) {
  if (p.vocab <= kWarpRow) {
    token_logprobs_backward_kernel<T, false>
        <<<(unsigned)((p.rows + kWarps - 1) / kWarps), kWarps * 32, 0, stream>>>(p, 1);
  } else {
    const int64_t span = (int64_t)kWarps * 32 * Vec16<T>::N * kBwdVectors;
    const int64_t chunks = (p.vocab + span - 1) / span;
    token_logprobs_backward_kernel<T, true><<<(unsigned)(p.rows * chunks), kWarps * 32, 0, stream>>>(p, chunks);
  }
  return (int)cudaGetLastError();
}

}  // namespace

int launch_token_logprobs(const LogprobParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_fwd<__nv_bfloat16>(p, stream);
  if (dtype == kF16) return launch_fwd<__half>(p, stream);
  return launch_fwd<float>(p, stream);
}

int launch_token_logprobs_backward(const LogprobBwdParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_bwd<__nv_bfloat16>(p, stream);
  if (dtype == kF16) return launch_bwd<__half>(p, stream);
  return launch_bwd<float>(p, stream);
}

}  // namespace wf

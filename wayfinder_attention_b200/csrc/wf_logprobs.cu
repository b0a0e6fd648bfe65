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
// Alternatives are ranked by 64-bit keys: the logit's bits in an order-preserving form above
// the inverted index, so that equal logits rank by the lower index and no two keys are
// equal.  Long rows: the n-th largest of the threads' maxima bounds the n-th logit from
// below; a second look at the row (in L2 by then) collects the few logits that reach it,
// and each finds its rank by counting the keys above its own.  Where too many reach it
// (ties, orders), and for short rows, each warp keeps its n best as it goes, one key a
// lane, and the lists are merged.
//
// -inf is a token that cannot be said: p = 0, nothing added to H.  A row of nothing
// else has no distribution: logprob -inf, H 0, gradient 0.  A NaN (or +inf) makes its
// row's logprob and H NaN; NaN ranks first among the alternatives.
//
// Bound by bytes: one read of the logits; the backward reads them again and writes dx.
#include "wf_kernels.h"
#include "wf_pair.cuh"
#include "wf_rowio.cuh"
#include "wf_sm100.cuh"

namespace wf {
namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.92596299e-8f;  // log2 e and what that leaves of it
constexpr unsigned kAll = 0xffffffffu;

// NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
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
  // N values (even, or 1) of which `most` is the largest.
  template <int N>
  __device__ __forceinline__ void add(const float* x, float most) {
    if (!(most <= m)) rebase(max_nan(m, most));
    const float base = m == -INFINITY ? 0.f : m;  // -inf - -inf would be NaN
    // e^d is 0 long before d = -200: the bound keeps 0 * inf out of u
    if constexpr (N == 1) {
      const float d = max_nan(x[0] - base, -200.f), e = exp2_approx(d * kLog2e);
      s += e;
      u = fmaf(e, d, u);
    } else {
      Pair ps(0.f), pu(0.f);
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float d0, d1, y0, y1;
        add2(Pair(x[j], x[j + 1]), Pair(-base)).get(d0, d1);
        const Pair d(max_nan(d0, -200.f), max_nan(d1, -200.f));
        mul2(d, Pair(kLog2e)).get(y0, y1);
        const Pair e(exp2_approx(y0), exp2_approx(y1));
        ps = add2(ps, e);
        pu = fma2(e, d, pu);
      }
      float a, b;
      ps.get(a, b);
      s += a + b;
      pu.get(a, b);
      u += a + b;
    }
  }
};

template <int N>
__device__ __forceinline__ float max_of(const float* x) {
  float m = x[0];
#pragma unroll
  for (int j = 1; j + 1 < N; j += 2) m = max3_nan(m, x[j], x[j + 1]);
  if constexpr (N % 2 == 0) m = max_nan(m, x[N - 1]);
  return m;
}

template <int LANES = 32>
__device__ __forceinline__ Sums warp_join(Sums a) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(kAll, a.m, o);
    b.s = __shfl_xor_sync(kAll, a.s, o);
    b.u = __shfl_xor_sync(kAll, a.u, o);
    a.join(b);
  }
  return a;
}

__device__ __forceinline__ uint32_t value_key(float x) { return x != x ? 0xffffffffu : ordered_key(x); }
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  return (uint64_t)value_key(x) << 32 | (uint32_t)~index;
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
constexpr int kThreads = 32 * kWarps;
constexpr int kUnroll = 4;    // vectors a thread requests at once

// What a row's sums say, written by one thread; `log_s` is -inf for a row without a
// distribution.
template <typename T>
__device__ __forceinline__ void write_row(const LogprobParams& p, int64_t row, const T* x, const Sums& a, float log_s) {
  const bool none = a.s == 0.f;
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
__device__ __forceinline__ void write_top(const LogprobParams& p, int64_t row, int rank, uint64_t key, const Sums& a,
                                          float log_s) {
  const uint32_t hi = (uint32_t)(key >> 32);
  const float v = hi == 0xffffffffu ? NAN : key_to_float(hi);
  p.top_logprobs[row * p.top_n + rank] = a.s == 0.f ? -INFINITY : v - a.m - log_s;
  p.top_tokens[row * p.top_n + rank] = (uint32_t)~(uint32_t)key;
}

// Short rows that start on 16 bytes, without alternatives: LANES lanes a row, which they hold
// in registers, so the maximum is known before the first exponential.
template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(kThreads) token_logprobs_short_kernel(LogprobParams p) {
  pdl_wait();
  constexpr int V = Vec16<T>::N;
  const int t = threadIdx.x % LANES;
  const int64_t row = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LANES;
  const bool live = row < p.rows;
  const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.x_stride;
  RawVec<T, V> raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + t) * V;
    if (c < p.vocab) raw[i].load(x + c);
  }
  float f[NV][V];
  Sums a{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * LANES + t) * V < p.vocab) {
      raw[i].unpack(f[i]);
      a.m = max_nan(a.m, max_of<V>(f[i]));
    }
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) a.m = max_nan(a.m, __shfl_xor_sync(kAll, a.m, o));
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * LANES + t) * V < p.vocab) a.template add<V>(f[i], a.m);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(kAll, a.s, o);
    a.u += __shfl_xor_sync(kAll, a.u, o);
  }
  if (t == 0 && live) write_row(p, row, x, a, logf(a.s));
}

// The streaming list of a warp over elements [lo, hi) of a row: `warp` of `warps` take vectors
// in turn, the first one the ends.
template <typename T>
__device__ void stream_top(TopList& top, const T* x, int64_t lo, int64_t hi, int warp, int warps, int lane, int n) {
  constexpr int V = Vec16<T>::N;
  const Span<T> span(x, lo, hi);
  bool first = true;
  for (int64_t c0 = span.head + (int64_t)warp * 32 * V; c0 < span.tail; c0 += (int64_t)warps * 32 * V) {
    const int64_t c = c0 + (int64_t)lane * V;
    const bool live = c < span.tail;
    float f[V], most = -INFINITY;
    if (live) {
      RawVec<T, V> raw;
      raw.load(x + c);
      raw.unpack(f);
      most = max_of<V>(f);
    }
    if (first) {
      // the n-th largest of the lanes' maxima is a first bar: n elements reach it
      TopList firsts;
      firsts.clear();
      firsts.merge(live ? rank_key(most, lane) : 0, lane);
      firsts.set_bar(n);
      top.bar = firsts.bar;
      first = false;
    }
    if (__any_sync(kAll, live && !(most < top.bar)))
#pragma unroll
      for (int j = 0; j < V; ++j) top.offer(live ? f[j] : 0.f, (uint32_t)(c + j), live, n, lane);
  }
  if (warp == 0) {
    const int64_t n_head = span.head - lo, n_tail = hi - span.tail;
    const int64_t c = lane < n_head ? lo + lane : span.tail + (lane - n_head);
    const bool live = lane < n_head + n_tail;
    top.offer(live ? to_f32(x[c]) : 0.f, (uint32_t)c, live, n, lane);
  }
}

// The sums of a thread over its share of [lo, hi): vectors t, t + threads, ... and, for the
// first threads, the ends.
template <typename T>
__device__ __forceinline__ Sums thread_sums(const T* x, int64_t lo, int64_t hi, int t, int threads) {
  constexpr int V = Vec16<T>::N;
  const Span<T> span(x, lo, hi);
  Sums a{-INFINITY, 0.f, 0.f};
  const int64_t stride = (int64_t)threads * V;
  int64_t c = span.head + (int64_t)t * V;
  for (; c + (kUnroll - 1) * stride < span.tail; c += kUnroll * stride) {
    RawVec<T, V> raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) raw[i].load(x + c + i * stride);
    float f[kUnroll * V];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) raw[i].unpack(f + i * V);
    a.template add<kUnroll * V>(f, max_of<kUnroll * V>(f));
  }
  for (; c < span.tail; c += stride) {
    RawVec<T, V> raw;
    raw.load(x + c);
    float f[V];
    raw.unpack(f);
    a.template add<V>(f, max_of<V>(f));
  }
  const int64_t n_head = span.head - lo, n_tail = hi - span.tail;
  if (t < n_head + n_tail) {
    const float f = to_f32(x[t < n_head ? lo + t : span.tail + (t - n_head)]);
    a.template add<1>(&f, f);
  }
  return a;
}

// Up to 32 N logits, with alternatives: a warp holds the row, an element a lane and turn, and
// sorts 32 keys a turn into its list.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) token_logprobs_sort_kernel(LogprobParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  float f[N];
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = lane + 32 * i < p.vocab ? to_f32(x[lane + 32 * i]) : -INFINITY;
  Sums a{-INFINITY, 0.f, 0.f};
  a.template add<N>(f, max_of<N>(f));
  a = warp_join(a);
  TopList top;
  top.clear();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (32 * i < p.vocab) top.merge(lane + 32 * i < p.vocab ? rank_key(f[i], lane + 32 * i) : 0, lane);
  const float log_s = logf(a.s);
  if (lane == 0) write_row(p, row, x, a, log_s);
  if (lane < p.top_n) write_top(p, row, lane, top.mine, a, log_s);
}

// Short rows of any start, or longer ones with alternatives: a warp a row.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_warp_kernel(LogprobParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const Sums a = warp_join(thread_sums(x, 0, p.vocab, lane, 32));
  const float log_s = logf(a.s);
  if (lane == 0) write_row(p, row, x, a, log_s);
  if constexpr (TOP) {
    TopList top;
    top.clear();
    stream_top(top, x, 0, p.vocab, 0, 1, lane, p.top_n);
    if (lane < p.top_n) write_top(p, row, lane, top.mine, a, log_s);
  }
}

constexpr int kCandidates = 256;  // keys that a block ranks at once

// Each thread's key finds its place among `count` of them in shared memory.
__device__ __forceinline__ int rank_of(uint64_t key, const uint64_t* keys, int count) {
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < count; ++i) above += keys[i] > key;
  return above;
}

// Long rows: one row a cluster of 1 to 8 blocks.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(LogprobParams p) {
  if (p.cluster > 1) cluster_arrive_started();
  pdl_wait();
  constexpr int V = Vec16<T>::N;
  __shared__ Sums warp_sums[kWarps];
  __shared__ Sums sums[8];  // of the cluster's blocks, in its first block
  __shared__ uint64_t found[kCandidates];             // keys of this block that reach its bar
  __shared__ uint64_t best[8][kMaxTopTokens];         // of the cluster's blocks, in its first block
  __shared__ uint64_t lists[kWarps][kMaxTopTokens];   // of the warps, and the block's own best
  __shared__ uint32_t maxima[kThreads];
  __shared__ uint32_t bar_key;
  __shared__ int n_found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t parts = p.cluster, part = blockIdx.x % parts;
  const int64_t row = blockIdx.x / parts;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const int64_t share = ((p.vocab + parts - 1) / parts + V - 1) / V * V;
  const int64_t lo = min((int64_t)part * share, p.vocab), hi = min(lo + share, p.vocab);

  Sums a = thread_sums(x, lo, hi, threadIdx.x, kThreads);
  if constexpr (TOP) {
    maxima[threadIdx.x] = value_key(a.m);
    if (threadIdx.x == 0) {
      n_found = 0;
      bar_key = 0;
    }
  }
  a = warp_join(a);
  if (lane == 0) warp_sums[warp] = a;
  __syncthreads();
  if constexpr (TOP) {
    // the n-th largest of the maxima, equal ones by thread
    const uint32_t mine = maxima[threadIdx.x];
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kThreads; ++i) {
      const uint32_t k = maxima[i];
      above += k > mine || (k == mine && i < (int)threadIdx.x);
    }
    if (above == p.top_n - 1) bar_key = mine;
    __syncthreads();
    const uint32_t bar = bar_key;
    // elements that reach it; beyond kCandidates only their number is kept
    auto look = [&](float f, int64_t c) {
      if (value_key(f) >= bar) {
        const int at = atomicAdd(&n_found, 1);
        if (at < kCandidates) found[at] = rank_key(f, (uint32_t)c);
      }
    };
    const Span<T> span(x, lo, hi);
    const float bar_value = bar == 0xffffffffu ? INFINITY : key_to_float(bar);
#pragma unroll 4
    for (int64_t c = span.head + (int64_t)threadIdx.x * V; c < span.tail; c += kThreads * V) {
      RawVec<T, V> raw;
      raw.load(x + c);
      float f[V];
      raw.unpack(f);
      if (!(max_of<V>(f) < bar_value))
#pragma unroll
        for (int j = 0; j < V; ++j) look(f[j], c + j);
    }
    const int64_t n_head = span.head - lo, n_tail = hi - span.tail;
    if ((int64_t)threadIdx.x < n_head + n_tail) {
      const int64_t c = threadIdx.x < n_head ? lo + threadIdx.x : span.tail + ((int64_t)threadIdx.x - n_head);
      look(to_f32(x[c]), c);
    }
    __syncthreads();
    const int count = n_found;
    if (count <= kCandidates) {
      if ((int)threadIdx.x < count) {
        const uint64_t key = found[threadIdx.x];
        const int rank = rank_of(key, found, count);
        if (rank < kMaxTopTokens) lists[0][rank] = key;
      }
      if ((int)threadIdx.x >= count && threadIdx.x < kMaxTopTokens) lists[0][threadIdx.x] = 0;
    } else {
      TopList top;
      top.clear();
      stream_top(top, x, lo, hi, warp, kWarps, lane, p.top_n);
      lists[warp][lane] = top.mine;
      __syncthreads();
      if (warp == 0) {
        for (int w = 1; w < kWarps; ++w) top.merge_sorted(lists[w][lane], lane);
        lists[0][lane] = top.mine;
      }
    }
    __syncthreads();
  }
  if (warp == 0) a = warp_join(lane < kWarps ? warp_sums[lane] : Sums{-INFINITY, 0.f, 0.f});
  if (parts > 1) {
    cluster_wait_started();  // the first block has started: its `sums` and `best` can be written
    if (warp == 0 && part > 0) {
      if (lane == 0) {
        const uint32_t d = map_peer(&sums[part], 0);
        st_peer_u32(d, __float_as_uint(a.m));
        st_peer_u32(d + 4, __float_as_uint(a.s));
        st_peer_u32(d + 8, __float_as_uint(a.u));
      }
      if (TOP) {
        const uint64_t key = lists[0][lane];
        const uint32_t d = map_peer(&best[part][lane], 0);
        st_peer_u32(d, (uint32_t)key);
        st_peer_u32(d + 4, (uint32_t)(key >> 32));
      }
    }
    if (warp == 0 && part == 0) {
      if (lane == 0) sums[0] = a;
      if (TOP) best[0][lane] = lists[0][lane];
    }
    __syncwarp();
    cluster_sync();
    if (part > 0) return;
    a = warp_join(lane < (int)parts ? sums[lane] : Sums{-INFINITY, 0.f, 0.f});  // every warp the same
    const float log_s = logf(a.s);
    if (threadIdx.x == 0) write_row(p, row, x, a, log_s);
    if constexpr (TOP) {
      // 32 keys a block at most 8 blocks: a thread each
      const int count = (int)parts * kMaxTopTokens;
      if ((int)threadIdx.x < count) {
        const uint64_t key = (&best[0][0])[threadIdx.x];
        const int rank = key ? rank_of(key, &best[0][0], count) : p.top_n;
        if (rank < p.top_n) write_top(p, row, rank, key, a, log_s);
      }
    }
    return;
  }
  if (warp != 0) return;
  const float log_s = logf(a.s);
  if (lane == 0) write_row(p, row, x, a, log_s);
  if constexpr (TOP)
    if (lane < p.top_n) write_top(p, row, lane, lists[0][lane], a, log_s);
}

// 2^(x log2 e - whole - part) 2^64 for two x, to fp32's bits: x log2 e is split into a whole number, which
// goes into the exponent with `whole`, and the rest to twice fp32's precision (a rounded product
// would carry 2^-24 of its whole part into the result).  |x| < 2^21; 0 below 2^-190.
__device__ __forceinline__ Pair exp_up64(Pair x, int whole, float part) {
  constexpr float kRound = 12582912.f;  // 1.5 2^23: a sum with it is rounded to a whole number
  const Pair t = fma2(x, Pair(kLog2e), Pair(kRound));
  const Pair rest = fma2(x, Pair(kLog2eLow), add2(fma2(x, Pair(kLog2e), fma2(t, Pair(-1.f), Pair(kRound))), Pair(-part)));
  float t0, t1, r0, r1;
  t.get(t0, t1);
  rest.get(r0, r1);
  const int bias = 64 + 127 - whole - (int)__float_as_uint(kRound);
  auto up = [&](float n) {
    const int e = (int)__float_as_uint(n) + bias;
    return __int_as_float(e > 0 ? e << 23 : 0);
  };
  return mul2(Pair(exp2_approx(r0), exp2_approx(r1)), Pair(up(t0), up(t1)));
}

// The gradient of a row's elements, for logits of type T.
template <typename T>
struct RowGrad {
  // 16-bit logits: p = exp((x - m) - log_s).  fp32: p = 2^(x' log2 e - whole - part) with x' = x - m; m is
  // 0 then, so that x' is exact, and the row's log sum exp is in whole + part to fp32's precision of
  // `part`; only rows with a maximum past 2^20 subtract it.
  static constexpr bool kSplit = sizeof(T) == 4;
  float m, log_s, gh, gl, base, lowest, part;
  int whole;
  bool none;
  int64_t tok;
  __device__ __forceinline__ RowGrad(const LogprobBwdParams& p, int64_t row)
      : m(p.stats[row]), log_s(p.stats[p.rows + row]), gh(p.dentropy ? p.dentropy[row] : 0.f),
        gl(p.dlogprob ? p.dlogprob[row] : 0.f), lowest(-200.f), tok(p.tokens[row]) {
    if (tok == p.ignore_index) gl = 0.f;
    else if (tok < 0 || tok >= p.vocab) gl = NAN;
    none = m == -INFINITY;
    base = fmaf(gh, p.entropy[row], gl);
    if constexpr (kSplit) {
      const bool far = !(fabsf(m) < 1048576.f);
      const float a = far ? 0.f : m, l = a + log_s, b = l - a;
      const float left = (a - (l - b)) + (log_s - b);  // a + log_s = l + left exactly
      const float power = l * kLog2e;
      whole = __float2int_rn(power);
      part = (power - (float)whole) + (fmaf(l, kLog2e, -power) + fmaf(l, kLog2eLow, left * kLog2e));
      lowest = far ? -200.f : m - 200.f;
      m = far ? m : 0.f;
      base = fmaf(gh, -l, base);
    }
  }
  // f[j] is x[c + j] and becomes dx[c + j].  p is computed 2^64 times too large, so that its
  // last bits survive where a gradient multiplies them up again; it is 0 long before
  // 200 below the maximum, which keeps 0 * inf out.  16-bit results take the exponential of a product
  // rounded with the 64 in it (2^-18 of p); fp32 ones exp_up64.
  template <int N>
  __device__ __forceinline__ void apply(float* f, int64_t c) const {
    constexpr float kDown = 5.421010862427522e-20f;  // 2^-64
    if constexpr (N == 1) {
      float lp, e, other;
      if constexpr (kSplit) {
        lp = max_nan(f[0] - m, lowest);
        exp_up64(Pair(lp, 0.f), whole, part).get(e, other);
      } else {
        lp = max_nan(f[0] - m - log_s, lowest);
        e = exp2_approx(fmaf(lp, kLog2e, 64.f));
      }
      f[0] = e * -fmaf(gh, lp, base) * kDown;
    } else {
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float l0, l1;
        Pair d = add2(Pair(f[j], f[j + 1]), Pair(-m)), e;
        if constexpr (!kSplit) d = add2(d, Pair(-log_s));
        d.get(l0, l1);
        const Pair lp(max_nan(l0, lowest), max_nan(l1, lowest));
        if constexpr (kSplit) {
          e = exp_up64(lp, whole, part);
        } else {
          float y0, y1;
          fma2(lp, Pair(kLog2e), Pair(64.f)).get(y0, y1);
          e = Pair(exp2_approx(y0), exp2_approx(y1));
        }
        const Pair q = fma2(lp, Pair(-gh), Pair(-base));
        mul2(mul2(e, q), Pair(kDown)).get(f[j], f[j + 1]);
      }
    }
    if (none) {
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = 0.f;
    } else if ((uint64_t)(tok - c) < (uint64_t)N) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j == tok) f[j] += gl;
    }
  }
};

// Short rows that start on 16 bytes, as in the forward.
template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(kThreads) token_logprobs_backward_short_kernel(LogprobBwdParams p) {
  pdl_wait();
  constexpr int V = Vec16<T>::N;
  const int t = threadIdx.x % LANES;
  const int64_t row = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LANES;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  T* dx = static_cast<T*>(p.dx) + row * p.vocab;
  RawVec<T, V> raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + t) * V;
    if (c < p.vocab) raw[i].load(x + c);
  }
  const RowGrad<T> g(p, row);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + t) * V;
    if (c < p.vocab) {
      float f[V];
      raw[i].unpack(f);
      g.template apply<V>(f, c);
      store_vec<T, V>(dx + c, f);
    }
  }
}

// Any rows: a warp a row (WIDE = false), or a block a share of one.
constexpr int64_t kBwdVectors = 4;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) token_logprobs_backward_kernel(LogprobBwdParams p, int64_t chunks) {
  pdl_wait();
  constexpr int V = Vec16<T>::N;
  constexpr int G = WIDE ? kThreads : 32;
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
  const RowGrad<T> g(p, row);
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
        g.template apply<V>(f, c);
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
    float f = to_f32(x[c]);
    g.template apply<1>(&f, c);
    dx[c] = from_f32<T>(f);
  }
}

// Whether rows of up to 1024 logits can be taken by whole vectors.
template <typename T>
bool short_vectors(const void* x, int64_t stride, const void* dx, int64_t vocab) {
  constexpr int V = Vec16<T>::N;
  return vocab <= 1024 && vocab % V == 0 && stride % V == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(dx) % 16 == 0;
}
// LAUNCH(LANES, NV): 8 lanes a row while 16 elements a lane hold it, else a warp.
#define WF_SHORT_ROWS(T, LAUNCH)                                           \
  constexpr int V = Vec16<T>::N;                                           \
  if (p.vocab <= 8 * V) LAUNCH(8, 1);                                      \
  else if (p.vocab <= 16 * V) LAUNCH(8, 2);                                \
  else if (V == 4 && p.vocab <= 32 * V) LAUNCH(8, 4);                      \
  else if (p.vocab <= 32 * V) LAUNCH(32, 1);                               \
  else if (p.vocab <= 64 * V) LAUNCH(32, 2);                               \
  else if (p.vocab <= 128 * V) LAUNCH(32, 4);                              \
  else LAUNCH(32, 8)

// A warp takes a row of up to 1024 logits (4 KB at most); longer rows take a block, and
// a cluster of up to 8 when there are fewer rows than SMs to give them to.
constexpr int64_t kWarpRow = 1024;

template <typename T>
int launch_fwd(LogprobParams p, cudaStream_t stream) {
  cudaError_t rc;
  auto launch = [&](void (*kern)(LogprobParams), int64_t blocks) {
    return launch_pdl(kern, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
  };
  if (p.top_n == 0 && short_vectors<T>(p.x, p.x_stride, nullptr, p.vocab)) {
#define WF_LAUNCH(LANES, NV) \
  rc = launch(token_logprobs_short_kernel<T, LANES, NV>, (p.rows * LANES + kThreads - 1) / kThreads)
    WF_SHORT_ROWS(T, WF_LAUNCH);
#undef WF_LAUNCH
    return (int)rc;
  }
  if (p.vocab <= kWarpRow) {
    const int64_t grid = (p.rows + kWarps - 1) / kWarps;
    if (p.top_n && p.vocab <= 64) rc = launch(token_logprobs_sort_kernel<T, 2>, grid);
    else if (p.top_n && p.vocab <= 256) rc = launch(token_logprobs_sort_kernel<T, 8>, grid);
    else if (p.top_n) rc = launch(token_logprobs_warp_kernel<T, true>, grid);
    else rc = launch(token_logprobs_warp_kernel<T, false>, grid);
    return (int)rc;
  }
  int c = 1;
  while (c < 8 && p.rows * c <= kSms && p.vocab / c > 4 * kWarpRow) c *= 2;
  p.cluster = c;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * c));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)(p.top_n ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, p)
                       : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, p));
}

template <typename T>
int launch_bwd(const LogprobBwdParams& p, cudaStream_t stream) {
  cudaError_t rc;
  auto launch = [&](void (*kern)(LogprobBwdParams), int64_t blocks) {
    return launch_pdl(kern, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
  };
  if (short_vectors<T>(p.x, p.x_stride, p.dx, p.vocab)) {
#define WF_LAUNCH(LANES, NV) \
  rc = launch(token_logprobs_backward_short_kernel<T, LANES, NV>, (p.rows * LANES + kThreads - 1) / kThreads)
    WF_SHORT_ROWS(T, WF_LAUNCH);
#undef WF_LAUNCH
  } else if (p.vocab <= kWarpRow) {
    rc = launch_pdl(token_logprobs_backward_kernel<T, false>, dim3((unsigned)((p.rows + kWarps - 1) / kWarps)),
                    dim3(kThreads), 0, stream, p, int64_t(1));
  } else {
    const int64_t span = (int64_t)kThreads * Vec16<T>::N * kBwdVectors;
    const int64_t chunks = (p.vocab + span - 1) / span;
    rc = launch_pdl(token_logprobs_backward_kernel<T, true>, dim3((unsigned)(p.rows * chunks)), dim3(kThreads), 0,
                    stream, p, chunks);
  }
  return (int)rc;
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

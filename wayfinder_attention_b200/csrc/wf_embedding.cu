// Token embedding with scaling and positions, and the gradients of its tables.
//
//   y_i = s W[t_i] + P[p_i], rounded once;   dW[v] = s sum of dy_i over t_i = v,  dP likewise
//
// The gradient sums rows of dy in a fixed order, with no atomics: the indices are sorted (stable
// radix sort, 8 or 9 bits a pass), and the sorted list is cut into chunks of equal length,
// whatever their rows: a group of threads walks a chunk with its columns' sum in registers
// and writes a table's row when the list moves on to the next.  A row whose list crosses the
// edge of a chunk leaves partial sums in fp32, which a second kernel adds.  Positions 0, 1, ...
// of each sequence need no sort: their sorted list is known.
//
// Bound by bytes: the forward reads and writes each row once; the backward reads dy once and
// writes the table, most of whose rows are zeros where the vocabulary is large.
#include "wf_common.cuh"
#include "wf_gemm.h"
#include "wf_kernels.h"
#include "wf_rowio.cuh"

#include <algorithm>

namespace wf {
namespace {

constexpr int kThreads = 256;

// Threads of a row: a power of two, at most a block's.
int group_of(int64_t vectors) {
  int g = 1;
  while (g < kThreads && g < vectors) g *= 2;
  return g;
}

// ------------------------------------------------------------------ forward
// G = 2^log_g threads a row, ROWS rows a group at once.
template <typename T, int VEC, int ROWS>
__global__ void __launch_bounds__(kThreads) embedding_kernel(EmbeddingParams p, int log_g) {
  pdl_wait();
  const int g = 1 << log_g, t = threadIdx.x & (g - 1);
  const int64_t per_block = (int64_t)(kThreads >> log_g) * ROWS;
  const int64_t row0 = (int64_t)blockIdx.x * per_block + (int64_t)(threadIdx.x >> log_g) * ROWS;
  const int64_t vectors = p.d / VEC;
  int64_t token[ROWS], place[ROWS];
  bool bad[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t row = row0 + r;
    token[r] = row < p.n ? p.tokens[row] : 0;
    place[r] = 0;
    if (p.position_weight && row < p.n) place[r] = p.positions ? p.positions[row] : (uint32_t)row % (uint32_t)p.seq;
    bad[r] = (uint64_t)token[r] >= (uint64_t)p.vocab || (p.position_weight && (uint64_t)place[r] >= (uint64_t)p.places);
    if (bad[r]) {
      token[r] = place[r] = 0;
      if (row < p.n && t == 0 && p.status) atomicOr(p.status, 1);
    }
  }
  const T* w = static_cast<const T*>(p.weight);
  const T* pw = static_cast<const T*>(p.position_weight);
  for (int64_t c = t; c < vectors; c += g) {
    RawVec<T, VEC> a[ROWS], b[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (row0 + r >= p.n) continue;
      a[r].load(w + token[r] * p.w_stride + c * VEC);
      if (pw) b[r].load(pw + place[r] * p.p_stride + c * VEC);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (row0 + r >= p.n) continue;
      float f[VEC], h[VEC];
      a[r].unpack(f);
      if (pw) b[r].unpack(h);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = bad[r] ? NAN : pw ? fmaf(f[j], p.scale, h[j]) : f[j] * p.scale;
      store_vec<T, VEC>(static_cast<T*>(p.y) + (row0 + r) * p.d + c * VEC, f);
    }
  }
}

// ------------------------------------------------------------------ sort
// The gradients of up to two tables are made side by side, a table's blocks in each launch.
struct Table {
  const int64_t* index;  // [n]; null: i % seq
  uint64_t* entries[2];  // sorted lists, by turns: index above, position below
  int* counts;           // [blocks][digits]; null where one block has all
  int* totals;           // [digits] where sort_scan_kernel has made the counts places within their digit, or null
  void* out;             // [rows][d]
  float* partials;       // [chunks][2][pitch]: a chunk's first row where it began before, its last where it goes on
  int64_t rows, skip;    // indices outside [0, rows), and `skip`, sort behind all others (as `rows`)
  int64_t fill0, fill1;  // bytes of out to be zeroed
  int passes, bits;
  float scale;
};
struct Tables {
  Table t[2];
  int64_t n, seq;
};

// Zeroes a share of a table: the sort's launches leave most of the GPU idle, and each does a part.
__device__ __forceinline__ void fill_share(const Table& t, int share, int shares, int64_t thread, int64_t threads) {
  const int64_t bytes = t.fill1 - t.fill0;
  unsigned char* out = static_cast<unsigned char*>(t.out);
  int64_t a = t.fill0 + bytes * share / shares, b = t.fill0 + bytes * (share + 1) / shares;
  const int64_t a16 = min((a + 15) / 16 * 16, b), b16 = max(b / 16 * 16, a16);
  if (thread < a16 - a) out[a + thread] = 0;
  if (thread < b - b16) out[b16 + thread] = 0;
  for (int64_t i = a16 + 16 * thread; i < b16; i += 16 * threads) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
}

// Stable radix sort of (index, position) pairs, 8 or 9 bits a pass.  A block's warps take kRounds
// times 32 of them each, and rank them 32 at a time, by ballots of the digit's bits, on top of
// their own count of each digit so far.  (A match instruction in place of the ballots: twice the
// time.)
constexpr int kRounds = 8, kMaxDigits = 512, kScanBlocks = 256;
constexpr int kSortWarps = 4, kAloneWarps = 16;  // of many blocks, and of one that has all
constexpr int kTile = 32 * kRounds * kSortWarps, kAlone = 32 * kRounds * kAloneWarps;

__device__ __forceinline__ uint64_t sort_entry(const Tables& p, const Table& t, int pass, int64_t i) {
  if (pass) return t.entries[(pass - 1) & 1][i];
  const int64_t v = t.index[i];
  const bool in = v >= 0 && v < t.rows && v != t.skip;
  return (uint64_t)(in ? v : t.rows) << 32 | (uint32_t)i;
}
__device__ __forceinline__ int digit_of(uint64_t e, int pass, int bits) {
  return (int)(e >> (32 + pass * bits)) & ((1 << bits) - 1);
}
// The lanes that hold this lane's digit (in-range lanes only).
__device__ __forceinline__ unsigned lanes_of(int digit, int bits, bool in) {
  unsigned same = __ballot_sync(0xffffffffu, in);
  for (int b = 0; b < bits; ++b) {
    const unsigned ones = __ballot_sync(0xffffffffu, digit >> b & 1);
    same &= digit >> b & 1 ? ones : ~ones;
  }
  return same;
}

__global__ void __launch_bounds__(32 * kSortWarps) sort_count_kernel(Tables p, int pass, int blocks, int share,
                                                                     int shares) {
  constexpr int THREADS = 32 * kSortWarps;
  __shared__ int count[kMaxDigits];
  pdl_wait();
  const Table& t = p.t[blockIdx.y];
  if ((int)blockIdx.x >= blocks) {
    fill_share(t, share, shares, (int64_t)(blockIdx.x - blocks) * THREADS + threadIdx.x, (int64_t)(gridDim.x - blocks) * THREADS);
    return;
  }
  if (pass >= t.passes) return;
  const int digits = 1 << t.bits;
  for (int d = threadIdx.x; d < digits; d += THREADS) count[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kTile + threadIdx.x;
  uint64_t entry[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) entry[k] = i0 + k * THREADS < p.n ? sort_entry(p, t, pass, i0 + k * THREADS) : 0;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool in = i0 + k * THREADS < p.n;
    const int d = digit_of(entry[k], pass, t.bits);
    const unsigned same = lanes_of(d, t.bits, in);
    if (in && (same & lanemask_lt()) == 0) atomicAdd(&count[d], __popc(same));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += THREADS) t.counts[(int64_t)blockIdx.x * digits + d] = count[d];
}

// Many blocks: their counts of a digit become each block's first place within it.  A block a digit.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(Tables p, int pass, int blocks) {
  __shared__ int warp_total[kThreads / 32];
  pdl_wait();
  const Table& t = p.t[blockIdx.y];
  const int digits = 1 << t.bits, d = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (pass >= t.passes || d >= digits) return;
  int so_far = 0;
  for (int b0 = 0; b0 < blocks; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const int c = b < blocks ? t.counts[(int64_t)b * digits + d] : 0;
    int scan = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += x;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    int place = so_far + scan - c;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) place += warp_total[w];
      so_far += warp_total[w];
    }
    if (b < blocks) t.counts[(int64_t)b * digits + d] = place;
    __syncthreads();
  }
  if (threadIdx.x == 0) t.totals[d] = so_far;
}

// Without counts the block's own are all there are.
template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) sort_place_kernel(Tables p, int pass, int blocks, int share, int shares) {
  constexpr int THREADS = 32 * WARPS, EACH = kMaxDigits / THREADS > 1 ? kMaxDigits / THREADS : 1;
  __shared__ int at[WARPS][kMaxDigits];  // counts, then places
  __shared__ int warp_total[WARPS];
  pdl_wait();
  const Table& t = p.t[blockIdx.y];
  if ((int)blockIdx.x >= blocks) {
    fill_share(t, share, shares, (int64_t)(blockIdx.x - blocks) * THREADS + threadIdx.x, (int64_t)(gridDim.x - blocks) * THREADS);
    return;
  }
  if (pass >= t.passes) return;
  const int digits = 1 << t.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int d = lane; d < digits; d += 32) at[warp][d] = 0;
  __syncwarp();
  const int64_t i0 = ((int64_t)blockIdx.x * WARPS + warp) * 32 * kRounds + lane;
  uint64_t entry[kRounds];
  int rank[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) entry[k] = i0 + 32 * k < p.n ? sort_entry(p, t, pass, i0 + 32 * k) : 0;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool in = i0 + 32 * k < p.n;
    const int d = digit_of(entry[k], pass, t.bits);
    const unsigned same = lanes_of(d, t.bits, in), before = same & lanemask_lt();
    const int so_far = at[warp][d];
    __syncwarp();
    if (in && !before) at[warp][d] = so_far + __popc(same);
    __syncwarp();
    rank[k] = so_far + __popc(before);
  }
  __syncthreads();
  // each digit's place: all of the smaller ones, and this one's in the blocks before.  A thread
  // takes EACH neighbours.
  int total[EACH], before[EACH], sum = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int d = threadIdx.x * EACH + e;
    total[e] = before[e] = 0;
    if (d < digits) {
      if (t.totals) {
        total[e] = t.totals[d];
        before[e] = t.counts[(int64_t)blockIdx.x * digits + d];
      } else if (t.counts) {
#pragma unroll 8
        for (int b = 0; b < blocks; ++b) {
          const int c = t.counts[(int64_t)b * digits + d];
          total[e] += c;
          if (b < (int)blockIdx.x) before[e] += c;
        }
      } else {
        for (int w = 0; w < WARPS; ++w) total[e] += at[w][d];
      }
    }
    sum += total[e];
  }
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += x;
  }
  if (lane == 31) warp_total[warp] = scan;
  __syncthreads();
  int first = scan - sum;
  for (int w = 0; w < warp; ++w) first += warp_total[w];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int d = threadIdx.x * EACH + e;
    if (d < digits) {
      int place = first + before[e];
      for (int w = 0; w < WARPS; ++w) {
        const int c = at[w][d];
        at[w][d] = place;
        place += c;
      }
    }
    first += total[e];
  }
  __syncthreads();
  uint64_t* to = t.entries[pass & 1];
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
    if (i0 + 32 * k < p.n) to[at[warp][digit_of(entry[k], pass, t.bits)] + rank[k]] = entry[k];
}

__global__ void __launch_bounds__(kThreads) fill_kernel(Tables p) {
  pdl_wait();
  fill_share(p.t[blockIdx.y], 0, 1, (int64_t)blockIdx.x * kThreads + threadIdx.x, (int64_t)gridDim.x * kThreads);
}

// ------------------------------------------------------------------ sums
// A table's sorted list: as sorted, or that of the positions 0 .. seq - 1 of n / seq sequences.
struct List {
  const uint64_t* entries;
  int64_t seq, batch;
  __device__ __forceinline__ List(const Tables& p, const Table& t)
      : entries(t.index ? t.entries[(t.passes - 1) & 1] : nullptr), seq(p.seq), batch(t.index ? 0 : p.n / p.seq) {}
  __device__ __forceinline__ void get(int64_t i, int& row, int& from) const {
    if (entries) {
      const uint64_t e = entries[i];
      row = (int)(e >> 32);
      from = (int)(uint32_t)e;
    } else {
      row = (int)((uint32_t)i / (uint32_t)batch);
      from = ((int)i - row * (int)batch) * (int)seq + row;
    }
  }
  __device__ __forceinline__ int row(int64_t i) const {
    int r, f;
    get(i, r, f);
    return r;
  }
};
struct Sum {
  const void* dy;
  int64_t stride, d, pitch;
  int chunk;  // 32 at most: a warp has a chunk's list in its lanes
};
constexpr int kAhead = 8;  // rows of dy on their way at once

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) embedding_sum_kernel(Tables tables, Sum p, int log_g) {
  pdl_wait();
  const Table& t = tables.t[blockIdx.z];
  const List list(tables, t);
  const int g = 1 << log_g, lane = threadIdx.x & 31;  // g is a warp at least
  const int64_t chunk = (int64_t)blockIdx.x * (kThreads >> log_g) + (threadIdx.x >> log_g);
  const int64_t c = ((int64_t)blockIdx.y * g + (threadIdx.x & (g - 1))) * VEC, i0 = chunk * p.chunk;
  const bool on = c < p.d;
  if (i0 >= tables.n) return;
  const int64_t i1 = min(i0 + p.chunk, tables.n);
  int my_row = (int)t.rows, my_from = 0;
  if (i0 + lane < i1) list.get(i0 + lane, my_row, my_from);
  const int outside = lane == 0 ? (i0 ? list.row(i0 - 1) : -1) : lane == 1 ? (i1 < tables.n ? list.row(i1) : -1) : 0;
  const int n = __popc(__ballot_sync(0xffffffffu, my_row < t.rows));  // those that count come first
  if (n == 0) return;
  const int before = __shfl_sync(0xffffffffu, outside, 0), after = __shfl_sync(0xffffffffu, outside, 1);
  const T* dy = static_cast<const T*>(p.dy) + c;
  float sum[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
  int row = __shfl_sync(0xffffffffu, my_row, 0);
  bool open = row == before;  // the row began in an earlier chunk
  auto flush = [&](bool goes_on) {
    if (!on) return;
    if (open || goes_on) {
      float* to = t.partials + (2 * chunk + (open ? 0 : 1)) * p.pitch + c;
      if constexpr (VEC == 1) {
        *to = sum[0];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
          *reinterpret_cast<float4*>(to + j) = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
      }
    } else {
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = sum[j] * t.scale;
      store_vec<T, VEC>(static_cast<T*>(t.out) + row * p.d + c, f);
    }
  };
  RawVec<T, VEC> v[kAhead];
  auto load = [&](int k, int i) {
    const int from = __shfl_sync(0xffffffffu, my_from, i & 31);
    if (i < n && on) v[k].load(dy + from * p.stride);
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k) load(k, k);
  for (int i = 0; i < n; i += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i + k >= n) break;
      const int next = __shfl_sync(0xffffffffu, my_row, i + k);
      if (next != row) {
        flush(false);
        row = next;
        open = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
      }
      float f[VEC];
      v[k].unpack(f);
      load(k, i + k + kAhead);
      if (on) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] += f[j];
      }
    }
  }
  flush(row == after);
}

// Rows that cross chunks: the chunk where one begins and goes on adds its parts, of the chunks up to
// the first that the row does not fill.  A block takes 128 columns; its warps share the parts.
constexpr int kJoinWarps = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) embedding_join_kernel(Tables tables, Sum p, int chunks) {
  __shared__ float4 part[kJoinWarps][32];
  pdl_wait();
  const Table& t = tables.t[blockIdx.z];
  const List list(tables, t);
  const int chunk = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i0 = (int64_t)chunk * p.chunk, i1 = i0 + p.chunk;
  if (i1 >= tables.n) return;
  const int row = list.row(i1 - 1), next = list.row(i1), first = list.row(i0), before = i0 ? list.row(i0 - 1) : -1;
  if (row >= t.rows || next != row) return;    // ends here
  if (first == row && before == row) return;   // began before
  int more = 0;  // chunks that the row fills
  for (int k = chunk + 1;;) {
    const int mine = k + threadIdx.x;
    const int64_t end = (int64_t)(mine + 1) * p.chunk;
    // filled, and going on in the next
    const bool filled = mine < chunks && end < tables.n && list.row(end) == row;
    const int n = __syncthreads_count(filled);
    more += n;
    k += n;
    if (n < 32 * kJoinWarps) break;
  }
  const int parts = more + 2;  // this chunk's, the filled ones', the last one's
  const int64_t c = (int64_t)blockIdx.y * 128 + lane * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < p.pitch)
#pragma unroll 4
    for (int k = warp; k < parts; k += kJoinWarps) {
      const float4 f =
          *reinterpret_cast<const float4*>(t.partials + (2 * (int64_t)(chunk + k) + (k ? 0 : 1)) * p.pitch + c);
      s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
    }
  part[warp][lane] = s;
  __syncthreads();
  if (warp) return;
  for (int w = 1; w < kJoinWarps; ++w) {
    const float4 f = part[w][lane];
    s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
  }
  const float v[4] = {s.x * t.scale, s.y * t.scale, s.z * t.scale, s.w * t.scale};
  T* to = static_cast<T*>(t.out) + row * p.d + c;
  for (int j = 0; j < 4 && c + j < p.d; ++j) to[j] = from_f32<T>(v[j]);
}

// ------------------------------------------------------------------ launches
int bits_of(int64_t most) {  // of the numbers 0 .. most
  int b = 1;
  while (most >> b) ++b;
  return b;
}
struct TablePlan {
  int passes, bits;
  size_t entries, counts, partials;
  size_t bytes() const { return 2 * entries + counts + partials; }
};
struct SumPlan {
  int blocks, chunk, log_g, columns;  // of the sort; of a list; threads a row; blocks over a row
  int64_t chunks;
};
SumPlan sum_plan(int64_t n, int64_t d, int vec) {
  SumPlan s{};
  s.blocks = n <= kAlone ? 1 : (int)((n + kTile - 1) / kTile);
  const int64_t vectors = (d + vec - 1) / vec;
  const int g = std::max(32, group_of(vectors));
  s.log_g = bits_of(g) - 1;
  s.columns = (int)((vectors + g - 1) / g);
  s.chunk = 32;
  while (s.chunk > 8 && (n + s.chunk - 1) / s.chunk * vectors < 512 * kSms) s.chunk /= 2;
  s.chunks = (n + s.chunk - 1) / s.chunk;
  return s;
}
TablePlan table_plan(const SumPlan& s, int64_t n, int64_t rows, int64_t d, bool sorted) {
  TablePlan t{};
  if (!sorted) {
    const int bits = bits_of(rows);
    t.passes = (bits + 8) / 9;
    t.bits = (bits + t.passes - 1) / t.passes;
    t.entries = round256((size_t)n * sizeof(uint64_t));
    t.counts = s.blocks > 1 ? round256((size_t)(s.blocks + 1) * (1 << t.bits) * sizeof(int)) : 0;
  }
  t.partials = round256((size_t)s.chunks * 2 * round8(d) * sizeof(float));
  return t;
}
int vec_of(int dtype, const void* a, int64_t stride_a, const void* b, int64_t stride_b, int64_t d) {
  const int64_t size = dtype == kF32 ? 4 : 2;
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | (uintptr_t)(stride_a * size) | reinterpret_cast<uintptr_t>(b) |
                        (uintptr_t)(stride_b * size) | (uintptr_t)(d * size);
  return all % 16 == 0 ? (int)(16 / size) : 1;
}

template <typename T, int VEC>
int launch_fwd(const EmbeddingParams& p, cudaStream_t stream) {
  const int64_t vectors = p.d / VEC;
  const int g = group_of(vectors), log_g = bits_of(g) - 1, per_block = kThreads / g;
  // four rows a group at once where that leaves work for all SMs
  if (p.n >= (int64_t)per_block * 4 * 4 * kSms)
    return (int)launch_pdl(embedding_kernel<T, VEC, 4>, dim3((unsigned)((p.n + 4 * per_block - 1) / (4 * per_block))),
                           dim3(kThreads), 0, stream, p, log_g);
  return (int)launch_pdl(embedding_kernel<T, VEC, 1>, dim3((unsigned)((p.n + per_block - 1) / per_block)),
                         dim3(kThreads), 0, stream, p, log_g);
}
template <typename T>
int launch_fwd_type(const EmbeddingParams& p, int dtype, cudaStream_t stream) {
  constexpr int V = Vec16<T>::N;
  const void* pw = p.position_weight;
  const bool vec = vec_of(dtype, p.weight, p.w_stride, p.y, p.d, p.d) == V && vec_of(dtype, pw, pw ? p.p_stride : 0, nullptr, 0, 0) == V;
  return vec ? launch_fwd<T, V>(p, stream) : launch_fwd<T, 1>(p, stream);
}

template <typename T, int VEC>
int launch_sums(const SumPlan& s, const Tables& tables, int count, const Sum& q, cudaStream_t stream) {
  const int per_block = kThreads >> s.log_g;
  if (cudaError_t e = launch_pdl(embedding_sum_kernel<T, VEC>,
                                 dim3((unsigned)((s.chunks + per_block - 1) / per_block), s.columns, count),
                                 dim3(kThreads), 0, stream, tables, q, s.log_g))
    return (int)e;
  if (s.chunks == 1) return 0;
  return (int)launch_pdl(embedding_join_kernel<T>, dim3((unsigned)s.chunks, (unsigned)((q.d + 127) / 128), count),
                         dim3(32 * kJoinWarps), 0, stream, tables, q, (int)s.chunks);
}

int launch_sort(const SumPlan& s, const Tables& tables, int count, cudaStream_t stream) {
  int passes = 0, digits = 0;
  int64_t fill = 0;
  bool scan = false;
  for (int i = 0; i < count; ++i) {
    const Table& t = tables.t[i];
    passes = std::max(passes, t.passes);
    digits = std::max(digits, t.passes ? 1 << t.bits : 0);
    fill = std::max(fill, t.fill1 - t.fill0);
    scan |= t.totals != nullptr;
  }
  // enough blocks to fill at full rate, 16 KB a block and launch at least
  const int shares = std::max(1, passes * (s.blocks > 1 ? 2 : 1));
  const int fillers = (int)std::min<int64_t>(((fill + shares - 1) / shares + 16383) / 16384, 8 * kSms);
  if (!passes) {
    if (!fill) return 0;
    return (int)launch_pdl(fill_kernel, dim3(fillers, count), dim3(kThreads), 0, stream, tables);
  }
  int share = 0;
  for (int pass = 0; pass < passes; ++pass) {
    cudaError_t e = cudaSuccess;
    if (s.blocks == 1) {
      e = launch_pdl(sort_place_kernel<kAloneWarps>, dim3(1 + fillers, count), dim3(32 * kAloneWarps), 0, stream, tables,
                     pass, 1, share++, shares);
    } else {
      e = launch_pdl(sort_count_kernel, dim3(s.blocks + fillers, count), dim3(32 * kSortWarps), 0, stream, tables, pass,
                     s.blocks, share++, shares);
      if (!e && scan) e = launch_pdl(sort_scan_kernel, dim3(digits, count), dim3(kThreads), 0, stream, tables, pass, s.blocks);
      if (!e)
        e = launch_pdl(sort_place_kernel<kSortWarps>, dim3(s.blocks + fillers, count), dim3(32 * kSortWarps), 0, stream,
                       tables, pass, s.blocks, share++, shares);
    }
    if (e) return (int)e;
  }
  return 0;
}

template <typename T>
int launch_bwd(const EmbeddingBwdParams& p, int dtype, cudaStream_t stream) {
  constexpr int V = Vec16<T>::N;
  struct Asked {
    void* out;
    const int64_t* index;
    int64_t rows, skip;
    float scale;
  } asked[2] = {{p.dweight, p.tokens, p.vocab, p.padding_index, p.scale}, {p.dposition_weight, p.positions, p.places, -1, 1.f}};
  if (p.n == 0) {
    for (const Asked& a : asked)
      if (a.out)
        if (cudaError_t e = cudaMemsetAsync(a.out, 0, (size_t)a.rows * p.d * sizeof(T), stream)) return (int)e;
    return 0;
  }
  int vec = vec_of(dtype, p.dy, p.dy_stride, nullptr, 0, p.d);
  for (const Asked& a : asked)
    if (a.out) vec = std::min(vec, vec_of(dtype, a.out, 0, nullptr, 0, p.d));
  const SumPlan s = sum_plan(p.n, p.d, vec);
  unsigned char* ws = static_cast<unsigned char*>(p.ws);
  Tables tables{};
  tables.n = p.n;
  tables.seq = p.seq;
  int count = 0;
  for (const Asked& a : asked) {
    if (!a.out) continue;
    const TablePlan q = table_plan(s, p.n, a.rows, p.d, !a.index);
    Table& t = tables.t[count++];
    t.index = a.index;
    t.out = a.out;
    t.rows = a.rows;
    t.skip = a.skip;
    t.scale = a.scale;
    t.passes = q.passes;
    t.bits = q.bits;
    // positions in order write the first seq rows themselves
    t.fill0 = a.index ? 0 : std::min(p.seq, a.rows) * p.d * (int64_t)sizeof(T);
    t.fill1 = a.rows * p.d * (int64_t)sizeof(T);
    t.entries[0] = reinterpret_cast<uint64_t*>(ws);
    t.entries[1] = reinterpret_cast<uint64_t*>(ws + q.entries);
    if (q.counts) {
      t.counts = reinterpret_cast<int*>(ws + 2 * q.entries);
      // every block adding up all blocks' counts is one launch less, but grows with their square
      if (s.blocks > kScanBlocks) t.totals = t.counts + ((size_t)s.blocks << q.bits);
    }
    t.partials = reinterpret_cast<float*>(ws + 2 * q.entries + q.counts);
    ws += q.bytes();
  }
  if (!count) return 0;
  if (int rc = launch_sort(s, tables, count, stream)) return rc;
  const Sum q{p.dy, p.dy_stride, p.d, round8(p.d), s.chunk};
  return vec == V ? launch_sums<T, V>(s, tables, count, q, stream) : launch_sums<T, 1>(s, tables, count, q, stream);
}

}  // namespace

size_t embedding_backward_workspace_bytes(int64_t n, int64_t vocab, int64_t places, int64_t d, int dtype, bool positions) {
  size_t most = 0;
  for (int vec : {1, dtype == kF32 ? 4 : 8}) {  // the plan goes by the alignment of dy: the larger of both
    const SumPlan s = sum_plan(n, d, vec);
    size_t bytes = 0;
    if (vocab) bytes += table_plan(s, n, vocab, d, false).bytes();
    if (places) bytes += table_plan(s, n, places, d, !positions).bytes();
    most = std::max(most, bytes);
  }
  return most;
}

int launch_embedding(const EmbeddingParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_fwd_type<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_fwd_type<__half>(p, dtype, stream);
  return launch_fwd_type<float>(p, dtype, stream);
}

int launch_embedding_backward(const EmbeddingBwdParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_bwd<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_bwd<__half>(p, dtype, stream);
  return launch_bwd<float>(p, dtype, stream);
}

}  // namespace wf

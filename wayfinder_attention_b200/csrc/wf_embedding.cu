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
    if (p.position_weight && row < p.n) place[r] = p.positions ? p.positions[row] : row % p.seq;
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
// Stable radix sort of (index, position) pairs.  A block takes kTile of them: a warp ranks 32 at
// a time by a match over its lanes, on top of its own count of each digit so far.
constexpr int kTile = 4096, kSortThreads = 512, kSortWarps = kSortThreads / 32, kPerWarp = kTile / kSortWarps;
constexpr int kMaxDigits = 512;
constexpr int kScanBlocks = 64;

struct SortParams {
  const int64_t* index;  // the first pass reads these; later ones `from`
  const uint64_t* from;  // index above, position below
  uint64_t* to;
  int* counts;           // [blocks][digits]; null where one block has all
  int* totals;           // [digits] where sort_scan_kernel has made the counts places within their digit, or null
  int64_t n;
  int64_t rows, skip;    // indices outside [0, rows), and `skip`, sort behind all others (as `rows`)
  int shift, bits;
};
__device__ __forceinline__ uint64_t sort_entry(const SortParams& p, int64_t i) {
  if (p.from) return p.from[i];
  const int64_t t = p.index[i];
  const bool in = t >= 0 && t < p.rows && t != p.skip;
  return (uint64_t)(in ? t : p.rows) << 32 | (uint32_t)i;
}
__device__ __forceinline__ int digit_of(const SortParams& p, uint64_t e) {
  return (int)(e >> (32 + p.shift)) & ((1 << p.bits) - 1);
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortParams p) {
  __shared__ int count[kMaxDigits];
  pdl_wait();
  const int digits = 1 << p.bits;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kTile;
#pragma unroll
  for (int k = 0; k < kTile / kSortThreads; ++k) {
    const int64_t i = i0 + k * kSortThreads + threadIdx.x;
    const int d = i < p.n ? digit_of(p, sort_entry(p, i)) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, d);
    if (d >= 0 && (same & lanemask_lt()) == 0) atomicAdd(&count[d], __popc(same));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) p.counts[(int64_t)blockIdx.x * digits + d] = count[d];
}

// Many blocks: their counts of a digit become each block's first place within it.  A block a digit.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(SortParams p, int blocks) {
  __shared__ int warp_total[kThreads / 32];
  pdl_wait();
  const int digits = 1 << p.bits, d = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int so_far = 0;
  for (int b0 = 0; b0 < blocks; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const int c = b < blocks ? p.counts[(int64_t)b * digits + d] : 0;
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
    if (b < blocks) p.counts[(int64_t)b * digits + d] = place;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.totals[d] = so_far;
}

// Without counts the block's own are all there are.
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortParams p) {
  __shared__ int at[kSortWarps][kMaxDigits];  // counts, then places
  __shared__ int warp_total[kSortWarps];
  pdl_wait();
  const int digits = 1 << p.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int d = lane; d < digits; d += 32) at[warp][d] = 0;
  __syncwarp();
  const int64_t i0 = (int64_t)blockIdx.x * kTile + warp * kPerWarp + lane;
  constexpr int kRounds = kPerWarp / 32;
  uint64_t entry[kRounds];
  int rank[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) entry[k] = i0 + 32 * k < p.n ? sort_entry(p, i0 + 32 * k) : 0;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int d = i0 + 32 * k < p.n ? digit_of(p, entry[k]) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, d), before = same & lanemask_lt();
    const int so_far = d >= 0 ? at[warp][d] : 0;
    __syncwarp();
    if (d >= 0 && !before) at[warp][d] = so_far + __popc(same);
    __syncwarp();
    rank[k] = so_far + __popc(before);
  }
  __syncthreads();
  // each digit's place: all of the smaller ones, and this one's in the blocks before
  int total = 0, before = 0;
  const int d = threadIdx.x;
  if (d < digits) {
    if (p.totals) {
      total = p.totals[d];
      before = p.counts[(int64_t)blockIdx.x * digits + d];
    } else if (p.counts) {
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const int c = p.counts[(int64_t)b * digits + d];
        total += c;
        if (b < (int)blockIdx.x) before += c;
      }
    } else {
      for (int w = 0; w < kSortWarps; ++w) total += at[w][d];
    }
  }
  int scan = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += x;
  }
  if (lane == 31) warp_total[warp] = scan;
  __syncthreads();
  if (d < digits) {
    int place = scan - total + before;
    for (int w = 0; w < warp; ++w) place += warp_total[w];
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = at[w][d];
      at[w][d] = place;
      place += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
    if (i0 + 32 * k < p.n) p.to[at[warp][digit_of(p, entry[k])] + rank[k]] = entry[k];
}

// ------------------------------------------------------------------ sums
// The sorted list: as sorted, or that of the positions 0 .. seq - 1 of n / seq sequences.
struct Sorted {
  const uint64_t* entries;
  int64_t n, seq, batch;
  __device__ __forceinline__ void get(int64_t i, int& row, int& from) const {
    if (entries) {
      const uint64_t e = entries[i];
      row = (int)(e >> 32);
      from = (int)(uint32_t)e;
    } else {
      row = (int)(i / batch);
      from = (int)(i - row * batch) * (int)seq + row;
    }
  }
  __device__ __forceinline__ int row(int64_t i) const {
    int r, f;
    get(i, r, f);
    return r;
  }
};
struct SumParams {
  Sorted list;
  const void* dy;
  void* out;        // [rows][d]
  float* partials;  // [chunks][2][pitch]: a chunk's first row where it began before, its last where it goes on
  int64_t stride, d, pitch, rows;
  int chunk;
  float scale;
};
constexpr int kAhead = 8;  // rows of dy on their way at once

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) embedding_sum_kernel(SumParams p, int log_g) {
  pdl_wait();
  const int g = 1 << log_g;
  const int64_t chunk = (int64_t)blockIdx.x * (kThreads >> log_g) + (threadIdx.x >> log_g);
  const int64_t c = ((int64_t)blockIdx.y * g + (threadIdx.x & (g - 1))) * VEC;
  const int64_t i0 = chunk * p.chunk;
  if (i0 >= p.list.n || c >= p.d) return;
  const int64_t i1 = min(i0 + p.chunk, p.list.n);
  const T* dy = static_cast<const T*>(p.dy) + c;
  float sum[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
  const int before = i0 ? p.list.row(i0 - 1) : -1, after = i1 < p.list.n ? p.list.row(i1) : -1;
  int row = p.list.row(i0);
  bool open = row == before;  // the row began in an earlier chunk
  if (row >= p.rows) return;
  auto flush = [&](bool goes_on) {
    if (open || goes_on) {
      float* to = p.partials + (2 * chunk + (open ? 0 : 1)) * p.pitch + c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) to[j] = sum[j];
    } else {
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = sum[j] * p.scale;
      store_vec<T, VEC>(static_cast<T*>(p.out) + row * p.d + c, f);
    }
  };
  for (int64_t i = i0; i < i1; i += kAhead) {
    int rows[kAhead], from[kAhead];
    RawVec<T, VEC> v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      rows[k] = (int)p.rows;
      if (i + k < i1) p.list.get(i + k, rows[k], from[k]);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (rows[k] < p.rows) v[k].load(dy + from[k] * p.stride);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (rows[k] >= p.rows) break;  // the end of the chunk, or of the indices that count
      if (rows[k] != row) {
        flush(false);
        row = rows[k];
        open = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
      }
      float f[VEC];
      v[k].unpack(f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] += f[j];
    }
  }
  flush(row == after);
}

// Rows that cross chunks: the chunk where one begins and goes on adds its parts, of the chunks up to
// the first that the row does not fill.  A block takes 128 columns; its warps share the parts.
constexpr int kJoinWarps = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) embedding_join_kernel(SumParams p, int chunks) {
  __shared__ float4 part[kJoinWarps][32];
  pdl_wait();
  const int chunk = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i0 = (int64_t)chunk * p.chunk, i1 = i0 + p.chunk;
  if (i1 >= p.list.n) return;
  const int row = p.list.row(i1 - 1);
  if (row >= p.rows || p.list.row(i1) != row) return;                            // ends here
  if (p.list.row(i0) == row && i0 && p.list.row(i0 - 1) == row) return;          // began before
  int more = 0;  // chunks that the row fills
  for (int k = chunk + 1;;) {
    const int mine = k + threadIdx.x;
    const int64_t end = (int64_t)(mine + 1) * p.chunk;
    // filled, and going on in the next
    const bool filled = mine < chunks && end < p.list.n && p.list.row(end) == row;
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
          *reinterpret_cast<const float4*>(p.partials + (2 * (int64_t)(chunk + k) + (k ? 0 : 1)) * p.pitch + c);
      s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
    }
  part[warp][lane] = s;
  __syncthreads();
  if (warp) return;
  for (int w = 1; w < kJoinWarps; ++w) {
    const float4 f = part[w][lane];
    s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
  }
  const float v[4] = {s.x * p.scale, s.y * p.scale, s.z * p.scale, s.w * p.scale};
  T* to = static_cast<T*>(p.out) + row * p.d + c;
  for (int j = 0; j < 4 && c + j < p.d; ++j) to[j] = from_f32<T>(v[j]);
}

// ------------------------------------------------------------------ launches
int bits_of(int64_t most) {  // of the numbers 0 .. most
  int b = 1;
  while (most >> b) ++b;
  return b;
}
struct SumPlan {
  int passes, bits, blocks, chunk, log_g, columns;  // columns: blocks over a row
  int64_t chunks;
  size_t entries, counts, partials;
  size_t bytes() const { return 2 * entries + counts + partials; }
};
SumPlan sum_plan(int64_t n, int64_t rows, int64_t d, bool sorted, int vec) {
  SumPlan s{};
  if (!sorted) {
    const int bits = bits_of(rows);
    s.passes = (bits + 8) / 9;
    s.bits = (bits + s.passes - 1) / s.passes;
    s.blocks = (int)((n + kTile - 1) / kTile);
    s.entries = round256((size_t)n * sizeof(uint64_t));
    s.counts = s.blocks > 1 ? round256((size_t)(s.blocks + 1) * (1 << s.bits) * sizeof(int)) : 0;
  }
  const int64_t vectors = (d + vec - 1) / vec;
  const int g = group_of(vectors);
  s.log_g = bits_of(g) - 1;
  s.columns = (int)((vectors + g - 1) / g);
  s.chunk = 32;
  while (s.chunk > 8 && (n + s.chunk - 1) / s.chunk * vectors < 512 * kSms) s.chunk /= 2;
  s.chunks = (n + s.chunk - 1) / s.chunk;
  s.partials = round256((size_t)s.chunks * 2 * ((d + 7) / 8 * 8) * sizeof(float));
  return s;
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
int launch_sum(const SumPlan& s, const SumParams& q, cudaStream_t stream) {
  const int per_block = kThreads >> s.log_g;
  if (cudaError_t e = launch_pdl(embedding_sum_kernel<T, VEC>,
                                 dim3((unsigned)((s.chunks + per_block - 1) / per_block), s.columns), dim3(kThreads), 0,
                                 stream, q, s.log_g))
    return (int)e;
  if (s.chunks == 1) return 0;
  return (int)launch_pdl(embedding_join_kernel<T>, dim3((unsigned)s.chunks, (unsigned)((q.d + 127) / 128)),
                         dim3(32 * kJoinWarps), 0, stream, q, (int)s.chunks);
}

template <typename T>
int launch_bwd(const EmbeddingBwdParams& p, int dtype, cudaStream_t stream) {
  if (cudaError_t e = cudaMemsetAsync(p.dweight, 0, (size_t)p.rows * p.d * sizeof(T), stream)) return (int)e;
  if (p.n == 0) return 0;
  constexpr int V = Vec16<T>::N;
  const int vec = vec_of(dtype, p.dy, p.dy_stride, p.dweight, 0, p.d);
  const SumPlan s = sum_plan(p.n, p.rows, p.d, !p.index, vec);
  unsigned char* ws = static_cast<unsigned char*>(p.ws);
  uint64_t* entries[2] = {reinterpret_cast<uint64_t*>(ws), reinterpret_cast<uint64_t*>(ws + s.entries)};
  SumParams q{};
  q.list = Sorted{nullptr, p.n, p.seq, p.index ? 0 : p.n / p.seq};
  if (p.index) {
    SortParams t{};
    t.index = p.index;
    t.counts = s.counts ? reinterpret_cast<int*>(ws + 2 * s.entries) : nullptr;
    // every block adding up all blocks' counts is one launch less (a pass of 32 blocks), but grows with their square
    if (s.blocks > kScanBlocks) t.totals = t.counts + ((size_t)s.blocks << s.bits);
    t.n = p.n;
    t.rows = p.rows;
    t.skip = p.padding_index;
    t.bits = s.bits;
    for (int pass = 0; pass < s.passes; ++pass) {
      t.shift = pass * s.bits;
      t.to = entries[pass & 1];
      if (t.counts)
        if (cudaError_t e = launch_pdl(sort_count_kernel, dim3(s.blocks), dim3(kSortThreads), 0, stream, t)) return (int)e;
      if (t.totals)
        if (cudaError_t e = launch_pdl(sort_scan_kernel, dim3(1 << s.bits), dim3(kThreads), 0, stream, t, s.blocks))
          return (int)e;
      if (cudaError_t e = launch_pdl(sort_place_kernel, dim3(s.blocks), dim3(kSortThreads), 0, stream, t)) return (int)e;
      t.from = t.to;
    }
    q.list.entries = t.from;
  }
  q.dy = p.dy;
  q.out = p.dweight;
  q.partials = reinterpret_cast<float*>(ws + 2 * s.entries + s.counts);
  q.stride = p.dy_stride;
  q.d = p.d;
  q.pitch = (p.d + 7) / 8 * 8;
  q.rows = p.rows;
  q.chunk = s.chunk;
  q.scale = p.scale;
  return vec == V ? launch_sum<T, V>(s, q, stream) : launch_sum<T, 1>(s, q, stream);
}

}  // namespace

size_t embedding_backward_workspace_bytes(int64_t n, int64_t rows, int64_t d, int dtype, bool sorted) {
  const int wide = dtype == kF32 ? 4 : 8;  // the plan goes by the alignment of dy: the larger of both
  return std::max(sum_plan(n, rows, d, sorted, 1).bytes(), sum_plan(n, rows, d, sorted, wide).bytes());
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

// Token embedding with scaling and positions, and the gradients of its tables.
//
//   y_i = s W[t_i] + P[p_i], rounded once;   dW[v] = s sum of dy_i over t_i = v,  dP likewise
//
// The gradient sums rows of dy in a fixed order, with no atomics on sums: the indices are sorted
// (stable radix sort, 8 or 9 bits a pass), and the sorted list is cut into chunks of equal length,
// whatever their rows: a group of threads walks a chunk with its columns' sum in registers
// and writes a table's row when the list moves on to the next.  A row whose list crosses the
// edge of a chunk leaves partial sums in fp32, which are added within the block, and across blocks
// by a second kernel.  The table is zeroed beside the sort, which leaves most of the GPU idle.
// Positions 0, 1, ... of each sequence need no sort: their sorted list is known.
//
// Bound by bytes: the forward reads and writes each row once; the backward reads dy once and
// writes the table, most of whose rows are zeros where the vocabulary is large.
#include "wf_common.cuh"
#include "wf_gemm.h"
#include "wf_kernels.h"
#include "wf_pair.cuh"
#include "wf_rowio.cuh"
#include "wf_sm100.cuh"

#include <algorithm>
#include <atomic>

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
// An index checked against its table: row 0 in place of one outside.
__device__ __forceinline__ bool checked(const EmbeddingParams& p, int64_t row, int64_t& token, int64_t& place) {
  token = p.tokens[row];
  place = !p.position_weight ? 0 : p.positions ? p.positions[row] : (uint32_t)row % (uint32_t)p.seq;
  const bool bad = (uint64_t)token >= (uint64_t)p.vocab || (p.position_weight && (uint64_t)place >= (uint64_t)p.places);
  if (bad) token = place = 0;
  return bad;
}
template <int VEC>
__device__ __forceinline__ void embed(float* f, const float* at, bool bad, float scale) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = bad ? NAN : at ? fmaf(f[j], scale, at[j]) : f[j] * scale;
}

// Few rows, or rows that do not start on 16 bytes: 2^log_g threads a row.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) embedding_kernel(EmbeddingParams p, int log_g) {
  pdl_wait();
  const int g = 1 << log_g, t = threadIdx.x & (g - 1);
  const int64_t row = (int64_t)blockIdx.x * (kThreads >> log_g) + (threadIdx.x >> log_g);
  if (row >= p.n) return;
  int64_t token, place;
  const bool bad = checked(p, row, token, place);
  if (bad && t == 0 && p.status) atomicOr(p.status, 1);
  const T* w = static_cast<const T*>(p.weight) + token * p.w_stride;
  const T* pw = p.position_weight ? static_cast<const T*>(p.position_weight) + place * p.p_stride : nullptr;
  T* y = static_cast<T*>(p.y) + row * p.d;
  for (int64_t c = (int64_t)t * VEC; c < p.d; c += g * VEC) {
    RawVec<T, VEC> a, b;
    a.load(w + c);
    if (pw) b.load(pw + c);
    float f[VEC], h[VEC];
    a.unpack(f);
    if (pw) b.unpack(h);
    embed<VEC>(f, pw ? h : nullptr, bad, p.scale);
    store_vec<T, VEC>(y + c, f);
  }
}

// Many rows: a warp walks up to 32 neighbours with its share of the columns, the next AHEAD rows on their
// way into its threads' own slots of shared memory.  Loads are then under way while others are
// stored, at no cost in registers: 60 us for 65536 rows of 2048 in fp16 (347 MB that have to move: 5.8 TB/s),
// where four rows loaded and then stored by each thread took 92.
template <typename T, bool POSITIONS>
__global__ void __launch_bounds__(kThreads) embedding_rows_kernel(EmbeddingParams p, int log_g, int chunk) {
  constexpr int VEC = Vec16<T>::N, AHEAD = POSITIONS ? 5 : 8;
  __shared__ uint4 ring[POSITIONS ? 2 : 1][AHEAD][kThreads];
  pdl_wait();
  const int g = 1 << log_g, lane = threadIdx.x & 31;  // g is a warp at least
  const int64_t i0 = ((int64_t)blockIdx.x * (kThreads >> log_g) + (threadIdx.x >> log_g)) * chunk;
  const int64_t c = ((int64_t)blockIdx.y * g + (threadIdx.x & (g - 1))) * VEC;
  const bool on = c < p.d;
  if (i0 >= p.n) return;
  const int n = (int)min((int64_t)chunk, p.n - i0);
  int64_t token = 0, place = 0;
  bool bad = false;
  if (lane < n) {
    bad = checked(p, i0 + lane, token, place);
    if (bad && p.status && blockIdx.y == 0 && (threadIdx.x & (g - 1)) < 32) atomicOr(p.status, 1);
  }
  const unsigned all_bad = __ballot_sync(0xffffffffu, bad);
  const T* w = static_cast<const T*>(p.weight) + c;
  const T* pw = static_cast<const T*>(p.position_weight) + c;
  T* y = static_cast<T*>(p.y) + i0 * p.d + c;
  const uint32_t slot = sm100::smem_u32(&ring[0][0][threadIdx.x]), apart = AHEAD * kThreads * 16;
  auto ask = [&](int i) {
    const int from = __shfl_sync(0xffffffffu, (int)token, i & 31), at = __shfl_sync(0xffffffffu, (int)place, i & 31);
    if (i < n && on) {
      copy_async<16>(slot + i % AHEAD * kThreads * 16, w + from * p.w_stride);
      if constexpr (POSITIONS) copy_async<16>(slot + apart + i % AHEAD * kThreads * 16, pw + at * p.p_stride);
    }
    copy_async_commit();
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) ask(i);
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    copy_async_wait<AHEAD - 1>();
    float f[VEC], h[VEC];
    Vec16<T>::unpack(sm100::ld_shared_16(slot + i % AHEAD * kThreads * 16), f);
    if constexpr (POSITIONS) Vec16<T>::unpack(sm100::ld_shared_16(slot + apart + i % AHEAD * kThreads * 16), h);
    ask(i + AHEAD);
    embed<VEC>(f, POSITIONS ? h : nullptr, all_bad >> i & 1, p.scale);
    if (on) store_vec<T, VEC>(y + i * p.d, f);
  }
  copy_async_wait<0>();
}

// ------------------------------------------------------------------ sort
// The gradients of up to two tables are made side by side, a table's blocks in each launch.
struct Table {
  const int64_t* index;  // [n]; null: i % seq
  uint64_t* entries[2];  // the sorted list, index above and position below, and what passes before the last leave
  int* counts;           // [blocks][digits], then each block's first place within the digit
  int* totals;           // [digits]
  void* out;             // [rows][d]
  float* partials;       // [blocks][2][pitch]: a block's first row where it began before, its last where it goes on
  int* crossings;        // how many rows begin in a block of chunks and go on in the next
  int2* crossing;        // those blocks and rows, in any order
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
// One thread a block issues bulk stores of zeros in shared memory (`bytes` of it, a multiple of 16);
// the share's ends that are not on 16 bytes are stored by bytes.
__device__ __forceinline__ void fill_share(const Table& t, int share, int shares, int block, int blocks, void* zeros,
                                           int bytes) {
  const int64_t all = t.fill1 - t.fill0;
  unsigned char* out = static_cast<unsigned char*>(t.out);
  const int64_t a = t.fill0 + all * share / shares, b = t.fill0 + all * (share + 1) / shares;
  const int64_t a16 = min((a + 15) / 16 * 16, b), b16 = max(b / 16 * 16, a16);
  if (block == 0) {
    if (threadIdx.x < a16 - a) out[a + threadIdx.x] = 0;
    if (threadIdx.x < b - b16) out[b16 + threadIdx.x] = 0;
  }
  for (int i = threadIdx.x; i < bytes / 16; i += blockDim.x) static_cast<uint4*>(zeros)[i] = make_uint4(0, 0, 0, 0);
  sm100::fence_async_shared();
  __syncthreads();
  if (threadIdx.x) return;  // nothing follows that all threads would have to reach
  for (int64_t i = a16 + (int64_t)block * bytes; i < b16; i += (int64_t)blocks * bytes) {
    const int n = (int)min((int64_t)bytes, b16 - i);
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(out + i),
                 "r"(sm100::smem_u32(zeros)), "r"(n)
                 : "memory");
  }
  sm100::bulk_commit();
  sm100::bulk_wait_all();
}

// Stable radix sort of (index, position) pairs, 8 or 9 bits a pass.  A warp takes 32 pairs at a time
// and ranks them by ballots of the digit's bits, on top of its own count of each digit so far.
// (A match instruction in place of the ballots took twice the time.)  Up to kAlone pairs are
// sorted by one cluster of blocks in one launch, which share their counts over distributed shared
// memory; more by three launches a pass.  The SMs without a part in it zero the table meanwhile.
constexpr int kMaxDigits = 512;
constexpr int kClusterWarps = 16, kMaxCluster = 8;
__host__ __device__ constexpr int cluster_tile(int rounds) { return 32 * kClusterWarps * rounds; }  // of a block
constexpr int kAlone = kMaxCluster * cluster_tile(16);
constexpr int kSortWarps = 8, kRounds = 8, kTile = 32 * kRounds * kSortWarps;

__device__ __forceinline__ uint64_t first_entry(const Table& t, int64_t i) {
  const int64_t v = t.index[i];
  const bool in = v >= 0 && v < t.rows && v != t.skip;
  return (uint64_t)(in ? v : t.rows) << 32 | (uint32_t)i;
}
__device__ __forceinline__ uint64_t sort_entry(const Table& t, int pass, int64_t i) {
  return pass ? t.entries[(t.passes - pass) & 1][i] : first_entry(t, i);  // the last pass ends in the first of the two
}
__device__ __forceinline__ int digit_of(uint64_t e, int pass, int bits) {
  return (int)(e >> (32 + pass * bits)) & ((1 << bits) - 1);
}
// The lanes that hold this lane's digit (in-range lanes only).
__device__ __forceinline__ unsigned lanes_of(int digit, bool in) {
  unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < 9; ++b) {
    const unsigned ones = __ballot_sync(0xffffffffu, digit >> b & 1);
    same &= digit >> b & 1 ? ones : ~ones;
  }
  return same;
}

// Ranks a warp's pairs, which are i0 + 32 k of the list (i0 has the lane in it): at[digit] counts them.
template <int ROUNDS>
__device__ __forceinline__ void rank_pairs(const Tables& p, const Table& t, int pass, int64_t i0, int* at,
                                           const uint64_t (&entry)[ROUNDS], int (&rank)[ROUNDS]) {
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) rank[k] = (int)lanes_of(digit_of(entry[k], pass, t.bits), i0 + 32 * k < p.n);
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const bool in = i0 + 32 * k < p.n;
    const int d = digit_of(entry[k], pass, t.bits);
    const unsigned same = rank[k], before = same & lanemask_lt();
    const int so_far = at[d];
    __syncwarp();
    if (in && !before) at[d] = so_far + __popc(same);
    __syncwarp();
    rank[k] = so_far + __popc(before);
  }
}
// Sum over the threads before this one.
template <int WARPS>
__device__ __forceinline__ int block_scan(int v, int* warp_total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int scan = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += x;
  }
  if (lane == 31) warp_total[warp] = scan;
  __syncthreads();
  int before = scan - v;
  for (int w = 0; w < warp; ++w) before += warp_total[w];
  return before;
}

// One cluster sorts a table's list, and the clusters behind those that sort (first, so that none waits for an SM)
// fill.  Between passes the list lies in the blocks' shared memory, a tile each.
template <int ROUNDS>
__global__ void __launch_bounds__(32 * kClusterWarps) sort_cluster_kernel(Tables p, int cluster, int count) {
  constexpr int THREADS = 32 * kClusterWarps, TILE = cluster_tile(ROUNDS);
  static_assert(THREADS == kMaxDigits, "a digit a thread");
  extern __shared__ __align__(16) unsigned char sort_smem[];
  uint64_t* list = reinterpret_cast<uint64_t*>(sort_smem);                            // [TILE]
  int* at = reinterpret_cast<int*>(list + TILE);                                      // [warps][digits]: counts, then places
  __shared__ int mine[kMaxDigits];  // this block's counts, which the others read
  __shared__ int warp_total[kClusterWarps];
  pdl_wait();
  const int behind = (int)blockIdx.x - cluster * count, block = blockIdx.x % cluster;
  if (behind >= 0) {
    for (int i = 0; i < count; ++i)
      fill_share(p.t[i], 0, 1, behind, gridDim.x - cluster * count, sort_smem, TILE * sizeof(uint64_t));
    return;
  }
  const Table& t = p.t[blockIdx.x / cluster];
  if (block == 0 && threadIdx.x == 0) *t.crossings = 0;
  const int digits = 1 << t.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = threadIdx.x;
  const int in_tile = warp * 32 * ROUNDS + lane;
  const int64_t i0 = (int64_t)block * TILE + in_tile;
  uint64_t entry[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) entry[k] = t.passes && i0 + 32 * k < p.n ? first_entry(t, i0 + 32 * k) : 0;
  for (int pass = 0; pass < t.passes; ++pass) {
    if (pass)
#pragma unroll
      for (int k = 0; k < ROUNDS; ++k) entry[k] = list[in_tile + 32 * k];
    int* counts = at + warp * kMaxDigits;
    for (int i = lane; i < digits; i += 32) counts[i] = 0;
    __syncwarp();
    int rank[ROUNDS];
    rank_pairs(p, t, pass, i0, counts, entry, rank);
    __syncthreads();
    if (d < digits) {
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) sum += at[w * kMaxDigits + d];
      mine[d] = sum;
    }
    sm100::cluster_sync();  // and all have their part of the list in registers
    int total = 0, before = 0, theirs[kMaxCluster];
    if (d < digits) {
#pragma unroll
      for (int b = 0; b < kMaxCluster; ++b)
        theirs[b] = b < cluster ? (int)sm100::ld_peer_u32(sm100::map_peer(&mine[d], b)) : 0;
#pragma unroll
      for (int b = 0; b < kMaxCluster; ++b) {
        total += theirs[b];
        if (b < block) before += theirs[b];
      }
    }
    int place = block_scan<kClusterWarps>(total, warp_total) + before;
    if (d < digits) {
      int count[kClusterWarps];
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) count[w] = at[w * kMaxDigits + d];
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) {
        at[w * kMaxDigits + d] = place;
        place += count[w];
      }
    }
    __syncthreads();
    const bool last = pass + 1 == t.passes;
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      if (i0 + 32 * k >= p.n) continue;
      const int to = counts[digit_of(entry[k], pass, t.bits)] + rank[k];
      if (last) t.entries[0][to] = entry[k];
      else sm100::st_peer_u64(sm100::map_peer(&list[to % TILE], to / TILE), entry[k]);
    }
    // the list is whole, and all have read this block's counts
    sm100::cluster_sync();
  }
}

__global__ void __launch_bounds__(32 * kSortWarps) sort_count_kernel(Tables p, int pass, int blocks, int share,
                                                                     int shares) {
  constexpr int THREADS = 32 * kSortWarps;
  __shared__ __align__(16) int count[kMaxDigits];
  pdl_wait();
  const Table& t = p.t[blockIdx.y];
  if ((int)blockIdx.x >= blocks) {
    fill_share(t, share, shares, blockIdx.x - blocks, gridDim.x - blocks, count, sizeof(count));
    return;
  }
  if (pass == 0 && blockIdx.x == 0 && threadIdx.x == 0) *t.crossings = 0;
  if (pass >= t.passes) return;
  const int digits = 1 << t.bits;
  for (int d = threadIdx.x; d < digits; d += THREADS) count[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kTile + threadIdx.x;
  uint64_t entry[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) entry[k] = i0 + k * THREADS < p.n ? sort_entry(t, pass, i0 + k * THREADS) : 0;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool in = i0 + k * THREADS < p.n;
    const int d = digit_of(entry[k], pass, t.bits);
    const unsigned same = lanes_of(d, in);
    if (in && (same & lanemask_lt()) == 0) atomicAdd(&count[d], __popc(same));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += THREADS) t.counts[(int64_t)blockIdx.x * digits + d] = count[d];
}

// The blocks' counts of a digit become each block's first place within it.  A block a digit.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(Tables p, int pass, int blocks) {
  __shared__ int warp_total[kThreads / 32];
  pdl_wait();
  const Table& t = p.t[blockIdx.y];
  const int digits = 1 << t.bits, d = blockIdx.x;
  if (pass >= t.passes || d >= digits) return;
  int so_far = 0;
  for (int b0 = 0; b0 < blocks; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const int c = b < blocks ? t.counts[(int64_t)b * digits + d] : 0;
    const int place = so_far + block_scan<kThreads / 32>(c, warp_total);
    for (int w = 0; w < kThreads / 32; ++w) so_far += warp_total[w];
    if (b < blocks) t.counts[(int64_t)b * digits + d] = place;
    __syncthreads();
  }
  if (threadIdx.x == 0) t.totals[d] = so_far;
}

__global__ void __launch_bounds__(32 * kSortWarps) sort_place_kernel(Tables p, int pass, int blocks, int share, int shares) {
  constexpr int THREADS = 32 * kSortWarps, EACH = kMaxDigits / THREADS;
  __shared__ __align__(16) int at[kSortWarps][kMaxDigits];  // counts, then places
  __shared__ int warp_total[kSortWarps];
  pdl_wait();
  const Table& t = p.t[blockIdx.y];
  if ((int)blockIdx.x >= blocks) {
    fill_share(t, share, shares, blockIdx.x - blocks, gridDim.x - blocks, at, sizeof(at));
    return;
  }
  if (pass >= t.passes) return;
  const int digits = 1 << t.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int d = lane; d < digits; d += 32) at[warp][d] = 0;
  __syncwarp();
  const int64_t i0 = ((int64_t)blockIdx.x * kSortWarps + warp) * 32 * kRounds + lane;
  uint64_t entry[kRounds];
  int rank[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) entry[k] = i0 + 32 * k < p.n ? sort_entry(t, pass, i0 + 32 * k) : 0;
  rank_pairs(p, t, pass, i0, at[warp], entry, rank);
  __syncthreads();
  // each digit's place: all of the smaller ones, and this one's in the blocks before.  A thread
  // takes EACH neighbours.
  int total[EACH], sum = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int d = threadIdx.x * EACH + e;
    total[e] = d < digits ? t.totals[d] : 0;
    sum += total[e];
  }
  int first = block_scan<kSortWarps>(sum, warp_total);
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int d = threadIdx.x * EACH + e;
    if (d < digits) {
      int place = first + t.counts[(int64_t)blockIdx.x * digits + d];
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = at[w][d];
        at[w][d] = place;
        place += c;
      }
    }
    first += total[e];
  }
  __syncthreads();
  uint64_t* to = t.entries[(t.passes - 1 - pass) & 1];
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
    if (i0 + 32 * k < p.n) to[at[warp][digit_of(entry[k], pass, t.bits)] + rank[k]] = entry[k];
}

// A table whose list is known needs no sort.
__global__ void __launch_bounds__(kThreads) fill_kernel(Tables p) {
  __shared__ uint4 zeros[1024];
  pdl_wait();
  const Table& t = p.t[blockIdx.y];
  if (blockIdx.x == 0 && threadIdx.x == 0) *t.crossings = 0;
  fill_share(t, 0, 1, blockIdx.x, gridDim.x, zeros, sizeof(zeros));
}

// ------------------------------------------------------------------ sums
// A table's sorted list: as sorted, or that of the positions 0 .. seq - 1 of n / seq sequences.
struct List {
  const uint64_t* entries;
  int64_t seq, batch;
  __device__ __forceinline__ List(const Tables& p, const Table& t)
      : entries(t.index ? t.entries[0] : nullptr), seq(p.seq), batch(t.index ? 0 : p.n / p.seq) {}
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


// VEC elements a vector (16 bytes, or one where rows do not start on them), W vectors a thread, 32 lanes apart.
template <typename T, int VEC, int W>
__global__ void __launch_bounds__(kThreads, 4) embedding_sum_kernel(Tables tables, Sum p, int log_g) {
  constexpr int N = VEC * W, kAhead = W > 1 ? 4 : 8;
  __shared__ uint4 ring[VEC > 1 ? kAhead * W * kThreads : 1];
  __shared__ float heads[(kThreads - 32) * N];  // of the block's chunks but the first: what belongs to a row that began before
  __shared__ bool fills[kThreads / 32];         // whether that is all of the chunk, and the row goes on
  pdl_wait();
  const Table& t = tables.t[blockIdx.z];
  const List list(tables, t);
  const int g = 1 << log_g, lane = threadIdx.x & 31;  // g is a warp at least
  const int group = threadIdx.x >> log_g, groups = kThreads >> log_g;
  const int64_t chunk = (int64_t)blockIdx.x * groups + group;
  // a warp's columns are next to each other: its w-th vectors start 32 VEC further each
  const int64_t c = (((int64_t)blockIdx.y * g + (threadIdx.x & (g - 32))) * W + lane) * VEC, i0 = chunk * p.chunk;
  const int64_t i1 = min(i0 + p.chunk, tables.n);
  int my_row = (int)t.rows, my_from = 0, outside = -1;
  if (i0 < tables.n) {
    if (i0 + lane < i1) list.get(i0 + lane, my_row, my_from);
    if (lane == 0 && i0) outside = list.row(i0 - 1);
    if (lane == 1 && i1 < tables.n) outside = list.row(i1);
  }
  const int n = __popc(__ballot_sync(0xffffffffu, my_row < t.rows));  // those that count come first
  const int before = __shfl_sync(0xffffffffu, outside, 0), after = __shfl_sync(0xffffffffu, outside, 1);
  const T* dy = static_cast<const T*>(p.dy) + c;
  const int64_t my_start = my_from * p.stride;  // of this lane's row in dy
  bool on[W];
#pragma unroll
  for (int w = 0; w < W; ++w) on[w] = c + 32 * VEC * w < p.d;
  float sum[N];
#pragma unroll
  for (int j = 0; j < N; ++j) sum[j] = 0.f;
  int row = __shfl_sync(0xffffffffu, my_row, 0);
  bool open = n && row == before;  // the row began in an earlier chunk
  auto write = [&](float* f) {
    T* out = static_cast<T*>(t.out) + row * p.d + c;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (!on[w]) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[w * VEC + j] *= t.scale;
      store_vec<T, VEC>(out + 32 * VEC * w, f + w * VEC);
    }
  };
  auto leave = [&](const float* f, int which) {
    float* to = t.partials + (2 * (int64_t)blockIdx.x + which) * p.pitch + c;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (!on[w]) continue;
      if constexpr (VEC == 1) {
        *to = f[0];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
          *reinterpret_cast<float4*>(to + 32 * VEC * w + j) =
              make_float4(f[w * VEC + j], f[w * VEC + j + 1], f[w * VEC + j + 2], f[w * VEC + j + 3]);
      }
    }
  };
  auto head = [&](int of, int j) -> float& { return heads[((of - 1) * N + j) * g + (threadIdx.x & (g - 1))]; };
  auto finish = [&] {  // of a row that ends in this chunk
    if (!open) {
      write(sum);
    } else if (group) {
#pragma unroll
      for (int j = 0; j < N; ++j) head(group, j) = sum[j];
    } else {
      leave(sum, 0);
    }
  };
  auto start = [&](int next) {
    finish();
    row = next;
    open = false;
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = 0.f;
  };
  auto start_of = [&](int i) {
    const uint32_t lo = __shfl_sync(0xffffffffu, (uint32_t)my_start, i & 31);
    return (int64_t)((uint64_t)__shfl_sync(0xffffffffu, (uint32_t)(my_start >> 32), i & 31) << 32 | lo);
  };
  // the next rows are on their way while one is added: in this thread's slots of shared memory, or
  // in registers where rows do not start on 16 bytes
  if constexpr (VEC > 1) {
    const uint32_t slot = sm100::smem_u32(&ring[threadIdx.x]);
    uint32_t asked = slot, read = slot;  // slots by turns
    constexpr uint32_t kTurn = W * kThreads * 16;
    auto turn = [&](uint32_t& at) { at = at == slot + (kAhead - 1) * kTurn ? slot : at + kTurn; };
    auto ask = [&](int i) {
      const T* from = dy + start_of(i);
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (i < n && on[w]) copy_async<16>(asked + w * kThreads * 16, from + 32 * VEC * w);
      copy_async_commit();
      turn(asked);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ask(i);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int next = __shfl_sync(0xffffffffu, my_row, i);
      if (next != row) start(next);
      copy_async_wait<kAhead - 1>();
      float f[N];
#pragma unroll
      for (int w = 0; w < W; ++w) Vec16<T>::unpack(sm100::ld_shared_16(read + w * kThreads * 16), f + w * VEC);
      turn(read);
      ask(i + kAhead);
#pragma unroll
      for (int j = 0; j < N; j += 2) add2(Pair(sum[j], sum[j + 1]), Pair(f[j], f[j + 1])).get(sum[j], sum[j + 1]);
    }
    copy_async_wait<0>();
  } else {
    static_assert(VEC > 1 || W == 1, "single elements");
    T v[kAhead];
    auto load = [&](int k, int i) {
      const int64_t from = start_of(i);
      if (i < n && on[0]) v[k] = dy[from];
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) load(k, k);
    for (int i = 0; i < n; i += kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (i + k >= n) break;
        const int next = __shfl_sync(0xffffffffu, my_row, i + k);
        if (next != row) start(next);
        const float f = to_f32(v[k]);
        load(k, i + k + kAhead);
        if (on[0]) sum[0] += f;
      }
    }
  }
  const bool goes_on = n && row == after, fills_chunk = open && goes_on;
  if (n && !goes_on) finish();
  if (fills_chunk && group) {
#pragma unroll
    for (int j = 0; j < N; ++j) head(group, j) = sum[j];
  }
  if ((threadIdx.x & (g - 1)) == 0) fills[group] = fills_chunk;
  __syncthreads();
  if (!goes_on || (open && group)) return;
  // this chunk's last row, or for the first chunk one that fills it, goes on in the next ones
  bool ends = false;
  for (int k = group + 1; k < groups && !ends; ++k) {
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] += head(k, j);
    ends = !fills[k];
  }
  if (open) {
    leave(sum, 0);
  } else if (ends) {
    write(sum);
  } else {  // and on in the next block: joined from here
    leave(sum, 1);
    if (blockIdx.y == 0 && (threadIdx.x & (g - 1)) == 0)
      t.crossing[atomicAdd(t.crossings, 1)] = make_int2((int)blockIdx.x, row);
  }
}

// Rows that cross blocks of chunks: the parts of the block where one begins and of the blocks up to the
// first that the row does not fill are added.  A thread block takes 512 columns of such a row; its warps
// share the parts.
constexpr int kJoinWarps = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) embedding_join_kernel(Tables tables, Sum p, int blocks, int64_t length) {
  __shared__ float4 part[kJoinWarps][128];
  pdl_wait();
  const Table& t = tables.t[blockIdx.z];
  const List list(tables, t);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = *t.crossings;
  int2 at = make_int2(0, 0);  // block and row
  if ((int)blockIdx.x < blocks) at = t.crossing[blockIdx.x];  // asked for before it is known whether there are as many
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    if (r != (int)blockIdx.x) at = t.crossing[r];
    const int block = at.x, row = at.y;
    int more = 0;  // blocks that the row fills
    for (int k = block + 1;;) {
      const int mine = k + threadIdx.x;
      const int64_t end = (mine + 1) * length;
      // filled, and going on in the next
      const bool filled = mine < blocks && end < tables.n && list.row(end) == row;
      const int n = __syncthreads_count(filled);
      more += n;
      k += n;
      if (n < 32 * kJoinWarps) break;
    }
    const int parts = more + 2;  // this block's, the filled ones', the last one's
    const int64_t c0 = (int64_t)blockIdx.y * 512;
    auto add = [&](float4& s, float4 f) { s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w; };
    float4 sum[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int k = warp; k < parts; k += kJoinWarps) {
      const float* from = t.partials + (2 * (int64_t)(block + k) + (k ? 0 : 1)) * p.pitch;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t c = c0 + 128 * i + 4 * lane;
        if (c < p.pitch) add(sum[i], *reinterpret_cast<const float4*>(from + c));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][32 * i + lane] = sum[i];
    __syncthreads();
    float4 s = part[0][threadIdx.x];
    for (int w = 1; w < kJoinWarps; ++w) add(s, part[w][threadIdx.x]);
    const float v[4] = {s.x * t.scale, s.y * t.scale, s.z * t.scale, s.w * t.scale};
    const int64_t c = c0 + 4 * threadIdx.x;
    T* to = static_cast<T*>(t.out) + row * p.d + c;
    for (int j = 0; j < 4 && c + j < p.d; ++j) to[j] = from_f32<T>(v[j]);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ launches
int bits_of(int64_t most) {  // of the numbers 0 .. most
  int b = 1;
  while (most >> b) ++b;
  return b;
}
// Vectors a thread, threads of a row, blocks over a row and rows of a warp's walk: long walks keep loads under way
// and leave few partial sums, short ones give all SMs work.
struct Walk {
  int chunk, wide, log_g, columns;
  int64_t chunks;
  int64_t sum_blocks() const { return (chunks + (kThreads >> log_g) - 1) / (kThreads >> log_g); }
};
Walk walk_of(int64_t n, int64_t d, int vec, int most_wide) {
  Walk s{};
  const int64_t vectors = (d + vec - 1) / vec;
  s.wide = vec > 1 && vectors >= 32 * most_wide ? most_wide : 1;
  const int64_t threads = (vectors + s.wide - 1) / s.wide;
  const int g = std::max(32, group_of(threads));
  s.log_g = bits_of(g) - 1;
  s.columns = (int)((threads + g - 1) / g);
  s.chunk = 32;
  while (s.chunk > 8 && (n + s.chunk - 1) / s.chunk * ((threads + 31) / 32) < 8 * kSms) s.chunk /= 2;
  s.chunks = (n + s.chunk - 1) / s.chunk;
  return s;
}
struct TablePlan {
  int passes, bits;
  size_t entries, counts, partials, crossing;
  size_t bytes() const { return 2 * entries + counts + partials + crossing; }
};
struct SumPlan : Walk {
  int cluster, blocks;  // of the sort: one cluster's, or (0) many blocks
};
SumPlan sum_plan(int64_t n, int64_t d, int vec) {
  SumPlan s{walk_of(n, d, vec, 2), 0, (int)((n + kTile - 1) / kTile)};
  if (n <= kAlone)
    for (s.cluster = 1; s.cluster < kMaxCluster && s.cluster * cluster_tile(8) < n;) s.cluster *= 2;
  return s;
}
TablePlan table_plan(const SumPlan& s, int64_t n, int64_t rows, int64_t d, bool sorted) {
  TablePlan t{};
  if (!sorted) {
    const int bits = bits_of(rows);
    t.passes = (bits + 8) / 9;
    t.bits = (bits + t.passes - 1) / t.passes;
    t.entries = round256((size_t)n * sizeof(uint64_t));
    t.counts = s.cluster ? 0 : round256((size_t)(s.blocks + 1) * (1 << t.bits) * sizeof(int));
  }
  t.partials = round256((size_t)s.sum_blocks() * 2 * round8(d) * sizeof(float));
  t.crossing = round256(sizeof(int)) + round256((size_t)s.sum_blocks() * sizeof(int2));
  return t;
}
int vec_of(int dtype, const void* a, int64_t stride_a, const void* b, int64_t stride_b, int64_t d) {
  const int64_t size = dtype == kF32 ? 4 : 2;
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | (uintptr_t)(stride_a * size) | reinterpret_cast<uintptr_t>(b) |
                        (uintptr_t)(stride_b * size) | (uintptr_t)(d * size);
  return all % 16 == 0 ? (int)(16 / size) : 1;
}

template <typename T>
int launch_fwd(const EmbeddingParams& p, int dtype, cudaStream_t stream) {
  constexpr int V = Vec16<T>::N;
  const void* pw = p.position_weight;
  const bool vec = vec_of(dtype, p.weight, p.w_stride, p.y, p.d, p.d) == V &&
                   vec_of(dtype, pw, pw ? p.p_stride : 0, nullptr, 0, 0) == V;
  const int64_t vectors = vec ? p.d / V : p.d;
  if (vec && p.n * vectors >= 64 * 8 * kSms) {  // rows for eight warps an SM to walk 16 and more
    const Walk s = walk_of(p.n, p.d, V, 1);
    const int per_block = kThreads >> s.log_g;
    const dim3 grid((unsigned)((s.chunks + per_block - 1) / per_block), s.columns);
    return (int)(pw ? launch_pdl(embedding_rows_kernel<T, true>, grid, dim3(kThreads), 0, stream, p, s.log_g, s.chunk)
                    : launch_pdl(embedding_rows_kernel<T, false>, grid, dim3(kThreads), 0, stream, p, s.log_g, s.chunk));
  }
  const int g = group_of(vectors), log_g = bits_of(g) - 1, per_block = kThreads / g;
  const dim3 grid((unsigned)((p.n + per_block - 1) / per_block));
  return (int)(vec ? launch_pdl(embedding_kernel<T, V>, grid, dim3(kThreads), 0, stream, p, log_g)
                   : launch_pdl(embedding_kernel<T, 1>, grid, dim3(kThreads), 0, stream, p, log_g));
}

template <typename T, int VEC, int W>
int launch_sums(const SumPlan& s, const Tables& tables, int count, const Sum& q, cudaStream_t stream) {
  const int blocks = (int)s.sum_blocks();
  if (cudaError_t e = launch_pdl(embedding_sum_kernel<T, VEC, W>, dim3(blocks, s.columns, count), dim3(kThreads), 0,
                                 stream, tables, q, s.log_g))
    return (int)e;
  if (blocks == 1) return 0;
  return (int)launch_pdl(embedding_join_kernel<T>,
                         dim3((unsigned)std::min(blocks, 8 * kSms), (unsigned)((q.d + 511) / 512), count),
                         dim3(32 * kJoinWarps), 0, stream, tables, q, blocks, (int64_t)q.chunk * (kThreads >> s.log_g));
}

template <int ROUNDS>
int launch_cluster_sort(const Tables& tables, int cluster, int count, int fillers, cudaStream_t stream) {
  constexpr size_t smem = cluster_tile(ROUNDS) * sizeof(uint64_t) + kClusterWarps * kMaxDigits * sizeof(int);
  int device = 0;
  if (cudaError_t e = cudaGetDevice(&device)) return (int)e;
  static std::atomic<uint64_t> allowed{0};  // devices whose limit has been raised for this kernel
  if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1)) {
    if (cudaError_t e = cudaFuncSetAttribute(sort_cluster_kernel<ROUNDS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem))
      return (int)e;
    if (device < 64) allowed.fetch_or(uint64_t(1) << device, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster * count + (fillers + cluster - 1) / cluster * cluster);
  cfg.blockDim = dim3(32 * kClusterWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, sort_cluster_kernel<ROUNDS>, tables, cluster, count);
}

int launch_sort(const SumPlan& s, const Tables& tables, int count, cudaStream_t stream) {
  int passes = 0, digits = 0;
  int64_t fill = 0;
  for (int i = 0; i < count; ++i) {
    const Table& t = tables.t[i];
    passes = std::max(passes, t.passes);
    digits = std::max(digits, t.passes ? 1 << t.bits : 0);
    fill = std::max(fill, t.fill1 - t.fill0);
  }
  // blocks that fill: two an SM at most, 16 KB each at least
  auto fillers = [&](int shares) {
    return (int)std::min<int64_t>(((fill + shares - 1) / shares + 16383) / 16384, 2 * kSms);
  };
  if (!passes) return (int)launch_pdl(fill_kernel, dim3(std::max(1, fillers(1)), count), dim3(kThreads), 0, stream, tables);
  if (s.cluster) {
    return s.cluster * cluster_tile(8) >= tables.n
               ? launch_cluster_sort<8>(tables, s.cluster, count, fillers(1), stream)
               : launch_cluster_sort<16>(tables, s.cluster, count, fillers(1), stream);
  }
  const int shares = 2 * passes, more = fillers(shares);
  int share = 0;
  for (int pass = 0; pass < passes; ++pass) {
    if (cudaError_t e = launch_pdl(sort_count_kernel, dim3(s.blocks + more, count), dim3(32 * kSortWarps), 0, stream,
                                   tables, pass, s.blocks, share++, shares))
      return (int)e;
    if (cudaError_t e = launch_pdl(sort_scan_kernel, dim3(digits, count), dim3(kThreads), 0, stream, tables, pass, s.blocks))
      return (int)e;
    if (cudaError_t e = launch_pdl(sort_place_kernel, dim3(s.blocks + more, count), dim3(32 * kSortWarps), 0, stream,
                                   tables, pass, s.blocks, share++, shares))
      return (int)e;
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
    t.counts = reinterpret_cast<int*>(ws + 2 * q.entries);
    t.totals = t.counts + ((size_t)s.blocks << q.bits);
    t.partials = reinterpret_cast<float*>(ws + 2 * q.entries + q.counts);
    t.crossings = reinterpret_cast<int*>(ws + 2 * q.entries + q.counts + q.partials);
    t.crossing = reinterpret_cast<int2*>(ws + 2 * q.entries + q.counts + q.partials + round256(sizeof(int)));
    ws += q.bytes();
  }
  if (!count) return 0;
  if (int rc = launch_sort(s, tables, count, stream)) return rc;
  const Sum q{p.dy, p.dy_stride, p.d, round8(p.d), s.chunk};
  if (vec != V) return launch_sums<T, 1, 1>(s, tables, count, q, stream);
  return s.wide == 2 ? launch_sums<T, V, 2>(s, tables, count, q, stream) : launch_sums<T, V, 1>(s, tables, count, q, stream);
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
  if (dtype == kBF16) return launch_fwd<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_fwd<__half>(p, dtype, stream);
  return launch_fwd<float>(p, dtype, stream);
}

int launch_embedding_backward(const EmbeddingBwdParams& p, int dtype, cudaStream_t stream) {
  if (dtype == kBF16) return launch_bwd<__nv_bfloat16>(p, dtype, stream);
  if (dtype == kF16) return launch_bwd<__half>(p, dtype, stream);
  return launch_bwd<float>(p, dtype, stream);
}

}  // namespace wf

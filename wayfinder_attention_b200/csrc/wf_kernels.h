// Host-side launch interface between the C ABI (wf_abi.cu) and the kernels.
// Not part of the public ABI: include/wayfinder.h is.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace wf {

constexpr int kSms = 148;  // of a B200

// Causal top-K over address vectors.
//   query rows:  q[b, l, :]  for local row l in [0, Tq); its sequence position
//                g(l) = ((l / rt) * rs + r0) * rt + l % rt   (identity when rs=1, r0=0, rt>=Tq)
//   keys:        k[b, j, :]  for j in [0, Tk); row g may retrieve j <= g only.
//   output:      idx[(b * Tq + l) * K + s], s = slot (descending score, ties -> lower index)
struct TopkParams {
  const void* q;
  const void* k;
  int64_t qsb, qst, qsr;
  int64_t ksb, kst, ksr;
  int B, Tq, Tk, R, K;
  int pad_mode;          // 0: reference pads (g + K + s + 1) % Tk; 1: -1 (masked)
  int rt, rs, r0;        // query row map
  int32_t* idx;
  int cap;               // candidate buffer capacity per row (multiple of 32)
  int32_t* status;       // nullable; bit 1 set if a bounded wait timed out
  void* ws;              // workspace of the tensor-core kernel (see topk_tc_workspace_bytes)
  size_t ws_bytes;
  // Optional [B][Tq] per-row key limits (replaces the row map): row l of batch b may
  // retrieve keys j < lim[b][l]; non-decreasing along the rows.  Null: causal row map.
  const int32_t* lim;
};

// Sparse attention over retrieved rows, indices shared across heads.
struct AttnParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* idx;
  void* out;
  int64_t qsb, qsh, qst;
  int64_t ksb, ksh, kst;
  int64_t vsb, vsh, vst;
  int64_t osb, osh, ost;
  int64_t isb, ist, iss;
  int B, H, Tq, Tk, D, K;
  float scale;
  int mask_negative;     // 1: negative index = masked slot; 0: wraps like torch indexing
  int out_vec_ok;        // output rows are 16-byte aligned (vector stores allowed)
  // Keys of a sequence sharded in cyclic row blocks and all-gathered rank-major:
  // key j lives in rank (j / kv_tile) % kv_world at local row
  // (j / kv_tile / kv_world) * kv_tile + j % kv_tile.  kv_world = 1: identity.
  int kv_tile, kv_world;
  int64_t k_rank_stride, v_rank_stride;
  // > 0: the gathered rows arrive in chunks of kv_chunk_rows local rows, stored
  // chunk-major: local row lr of rank r is row lr % kv_chunk_rows of block
  // (lr / kv_chunk_rows) * kv_world + r, blocks k/v_rank_stride apart.
  int kv_chunk_rows;
  int32_t* status;       // nullable; bit 0 set on an out-of-range index
  // Attention-probability dropout (training): rate in [0, 1), 0 = off.  Element
  // (b, h, t, k) is kept when dropout_uniform(seed, ((b*H + h)*Tq + t)*K + k) >= rate.
  float drop_rate;
  uint64_t drop_seed;
};

// Returns a cudaError_t; a negative value means "unsupported configuration"
// (the caller formats the message).
int launch_causal_topk(const TopkParams& p, int dtype, cudaStream_t stream);
int launch_sparse_attention(const AttnParams& p, int dtype, int out_dtype, cudaStream_t stream);

// Tensor-core (tcgen05) top-K: bf16/fp16 addresses, R in {16, 32, 64}, K <= 128,
// Tk <= 65536, unit address stride, 16-byte aligned rows.
bool topk_tc_supported(const TopkParams& p, int dtype);
int launch_causal_topk_tc(const TopkParams& p, int dtype, cudaStream_t stream);
// Test hook: the next tensor-core top-K launch withholds CTA 1's arrive of bisection
// exchange `round` (0..7; negative: off) and bounds those waits by wait_ns.
void topk_tc_test_withhold(int round, uint64_t wait_ns);
// Allocation-free retrieval: capacity of the library's built-in scratch array and
// its device address on the current device (first call per device looks it up).
size_t noalloc_scratch_capacity();
int noalloc_scratch(void** out);

// Workspace bytes the tensor-core path needs for B*Tq query rows (0 if K > 128).
size_t topk_tc_workspace_bytes(int64_t B, int64_t Tq, int64_t Tk, int R, int K, int dtype);

// Shared-memory bytes the top-K kernel needs for (R, K); 0 if unsupported.
size_t topk_smem_bytes(int R, int K);
int topk_max_k();
int attn_max_k();

// Fused address projection (wf_addr_proj.cu): out[m, :] = normalize_group(x[m] W^T + b).
int launch_address_projection(const void* x, int dtype, int64_t M, int K, int64_t x_stride, const void* w,
                              const void* bias, int N, int group, int normalize, void* out, int64_t out_stride,
                              int32_t* status, cudaStream_t stream);

// Top-K over the keys a (B, T) padding mask keeps (wf_keymask.cu).  `prep` holds
// topk_key_mask_prep_bytes; p.ws the top-K workspace for (B, T, T).
size_t topk_key_mask_prep_bytes(int64_t B, int64_t T, int R, int esz);
int launch_topk_key_mask(TopkParams p, int dtype, const uint8_t* mask, int64_t msb, int64_t mst, void* prep,
                         cudaStream_t stream);

// Backward of the sparse attention (wf_attn_bwd.cu).
struct AttnBwdParams {
  const void* q;
  const void* k;
  const void* v;
  const void* dout;
  const int32_t* idx;
  void* dq;
  void* dk;
  void* dv;
  int64_t qsb, qsh, qst, ksb, ksh, kst, vsb, vsh, vst, osb, osh, ost;
  int64_t dqsb, dqsh, dqst, dksb, dksh, dkst, dvsb, dvsh, dvst;
  int64_t isb, ist, iss;
  int B, H, Tq, Tk, D, K;
  float scale;
  int mask_negative;
  int dq_vec_ok, dk_vec_ok, dv_vec_ok;
  float drop_rate;       // the forward's dropout (see AttnParams); 0 = off
  uint64_t drop_seed;
  float* P;      // [B][Tq][K][H] softmax probabilities (workspace)
  float* DS;     // [B][Tq][K][H] scale * ds (workspace)
  int32_t* cnt;  // [B][Tk] per-key counts, then fill cursors (workspace)
  int32_t* off;  // [B][Tk + 1] list offsets (workspace)
  int32_t* list; // [B][Tq * K] (t * K + slot) entries grouped by key (workspace)
  int32_t* status;
};
size_t attn_bwd_workspace_bytes(int64_t B, int64_t H, int64_t Tq, int64_t Tk, int K);
int launch_sparse_attention_backward(AttnBwdParams p, void* ws, size_t ws_bytes, int dtype, int grad_dtype,
                                     cudaStream_t stream);

// Gather-rate ceiling (wf_bench.cu): K and V rows of row_bytes (<= 1024) at the
// indices idx[n_query][K], 16-byte loads, nothing computed; -1 for bad sizes.
int launch_gather_rows_bench(const void* k, const void* v, int64_t row_bytes, int64_t stride_bytes,
                             const int32_t* idx, int64_t n_query, int K, int64_t n_rows, uint32_t* sink,
                             cudaStream_t stream);
// The same 1 KB rows moved by cp.async.bulk into shared memory (read back or not).
int launch_gather_rows_bulk_bench(const void* k, const void* v, int64_t stride_bytes, const int32_t* idx,
                                  int64_t n_query, int K, int64_t n_rows, int read_back, uint32_t* sink,
                                  cudaStream_t stream);

// Layer norm over the last axis (wf_layer_norm.cu).  Rows are unit-strided; weight and
// bias may be null.
struct LayerNormParams {
  const void* x;
  void* y;
  const void* weight;
  const void* bias;
  float* mean;   // [rows], with rstd; both null when the backward will not run
  float* rstd;
  int64_t rows, x_stride, y_stride;
  int d;
  bool param_f32;  // weight and bias are fp32 (otherwise of x's type)
  float eps;
};
struct LayerNormBwdParams {
  const void* x;
  const void* dy;
  const void* weight;
  const float* mean;
  const float* rstd;
  void* dx;         // [rows][d] or null
  void* dweight;    // [d], null with dbias when neither is wanted
  void* dbias;
  float* partials;  // workspace; null when no parameter gradient is wanted
  int64_t rows, x_stride, dy_stride;
  int d;
  bool param_f32;
};
int launch_layer_norm(const LayerNormParams& p, int dtype, cudaStream_t stream);
size_t layer_norm_backward_workspace_bytes(int64_t rows, int64_t d, int dtype);
int launch_layer_norm_backward(const LayerNormBwdParams& p, int dtype, cudaStream_t stream);

// Log probabilities of given tokens (wf_logprobs.cu).
constexpr int kMaxTopTokens = 32;
struct LogprobParams {
  const void* x;          // [rows][vocab], unit stride on the vocabulary
  const int64_t* tokens;  // [rows]
  float* logprob;
  float* entropy;
  float* stats;           // [2][rows] for the backward, or null: the maximum m, and log sum exp(x - m)
  float* top_logprobs;    // [rows][top_n]
  int64_t* top_tokens;
  int64_t rows, x_stride, vocab, ignore_index;
  int top_n;
  int cluster;            // blocks a row (set by the launch)
  int32_t* status;        // nullable; bit 0 set on a token outside the vocabulary
};
struct LogprobBwdParams {
  const void* x;
  const int64_t* tokens;
  const float* stats;
  const float* entropy;
  const float* dlogprob;  // [rows] or null
  const float* dentropy;  // [rows] or null
  void* dx;               // [rows][vocab]
  int64_t rows, x_stride, vocab, ignore_index;
};
int launch_token_logprobs(const LogprobParams& p, int dtype, cudaStream_t stream);
int launch_token_logprobs_backward(const LogprobBwdParams& p, int dtype, cudaStream_t stream);

// Linear layer with bias, activation and residual (wf_linear.cu).  x (M, K) and
// w (N, K) are unit-strided on K; y and the gradients are contiguous.
enum Activation : int { kActNone = 0, kActGelu = 1, kActRelu = 2, kActSilu = 3 };
struct LinearParams {
  const void* x;
  const void* w;
  const void* bias;      // [N] or null
  const void* residual;  // (M, N) or null
  // pre-activations for the backward (fp16, or fp32 for fp32), M rows of N rounded up to 8; or null
  void* z;
  void* y;
  int64_t M, N, K, x_stride, w_stride, r_stride;
  int act;
  void* ws;
  int32_t* status;
};
struct LinearBwdParams {
  const void* x;
  const void* w;
  const void* z;
  const void* dy;
  void* dx;  // each of the three may be null
  void* dw;
  void* db;
  int64_t M, N, K, x_stride, w_stride, dy_stride;
  int act;
  void* ws;
  int32_t* status;
};
// *_direct: the matrix starts on 16 bytes and so does each of its rows.
size_t linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, bool x_direct, bool w_direct);
size_t linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int act, bool x_direct,
                                       bool w_direct, bool dy_direct);
int launch_linear(const LinearParams& p, int dtype, cudaStream_t stream);
int launch_linear_backward(const LinearBwdParams& p, int dtype, cudaStream_t stream);

}  // namespace wf

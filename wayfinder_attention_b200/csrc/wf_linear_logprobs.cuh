// Shared by the two forms of linear_token_logprobs' forward (wf_linear_logprobs.cu and
// wf_linear_logprobs_few.cu): running sums to a base, and how two of them become one.
#pragma once

#include "wf_activation.cuh"
#include "wf_gemm.h"
#include "wf_kernels.h"
#include "wf_rowio.cuh"

namespace wf {

// Up to kFewLogprobRows rows of a 16-bit type go by their own kernel, which leaves
// linear_logprobs_few_parts(vocab) parts of each row.
constexpr int kFewLogprobRows = 64;
int linear_logprobs_few_parts(int64_t vocab);
int launch_linear_logprobs_few(const GemmOperand& x, const GemmOperand& w, const LinearLogprobsParams& p, float* parts,
                               float* token_logit, int dtype, cudaStream_t stream);

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// e^d and 2^d are 0 below this: the bound keeps 0 * inf out where a logit is -inf
constexpr float kNothing = -200.f;

// s = sum exp(z - m) and u = sum exp(z - m) (z - m) of one part and of another, to the larger base.  m is
// -inf where nothing has counted, and a NaN or +inf among the logits stays in it.
__device__ __forceinline__ void join_sums(float& m, float& s, float& u, float m2, float s2, float u2) {
  const float top = max_keep_nan(m, m2);
  const float d = fmaxf(m - top, kNothing), d2 = fmaxf(m2 - top, kNothing);
  const float a = exp2_approx(d * kLog2e), a2 = exp2_approx(d2 * kLog2e);
  u = fmaf(a, fmaf(s, d, u), a2 * fmaf(s2, d2, u2));
  s = fmaf(a, s, a2 * s2);
  m = top;
}

}  // namespace
}  // namespace wf

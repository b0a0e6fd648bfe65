// The activations of wf_linear and their derivatives, in fp32.
#pragma once

#include "wf_rowio.cuh"
#include "wf_kernels.h"

namespace wf {

// Phi(-|z|) for 16-bit results: Abramowitz and Stegun 7.1.26 (erfc(x) = (a1 t + .. + a5 t^5)
// exp(-x^2), t = 1 / (1 + p x), off by at most 1.5e-7) at x = |z| / sqrt 2.  One reciprocal and
// one exponential where erff takes both of its branches in most warps: the gelu of a 128 x 256
// tile fell from 4 times its products' time (depth 256) to about theirs.  `e` gets exp(-z^2 / 2).
__device__ __forceinline__ float upper_tail(float az, float& e) {
  const float t = __fdividef(1.f, fmaf(0.3275911f * 0.70710678118654752f, az, 1.f));
  e = exp2_approx(az * az * (-0.5f * 1.4426950408889634f));
  float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  q = fmaf(t, q, 0.5f * 1.421413741f);
  q = fmaf(t, q, 0.5f * -0.284496736f);
  q = fmaf(t, q, 0.5f * 0.254829592f);
  return q * t * e;
}

// T: the type of the result.  fp32 takes CUDA's erff and expf and a true division.
template <int ACT, typename T>
__device__ __forceinline__ float activate(float z) {
  constexpr bool FAST = sizeof(T) == 2;
  if constexpr (ACT == kActGelu) {
    if constexpr (FAST) {
      // z Phi(z) = max(z, 0) - |z| Phi(-|z|); past 100 the tail is 0, and inf * 0 is kept out
      const float az = fminf(fabsf(z), 100.f);
      float e;
      return fmaf(-az, upper_tail(az, e), z < 0.f ? 0.f : z);
    } else {
      return z * 0.5f * (1.f + erff(z * 0.70710678118654752f));
    }
  } else if constexpr (ACT == kActRelu) {
    return z < 0.f ? 0.f : z;  // NaN stays
  } else if constexpr (ACT == kActSilu) {
    if constexpr (FAST) return z * __fdividef(1.f, 1.f + exp2_approx(-1.4426950408889634f * z));
    else return z / (1.f + expf(-z));
  } else {
    return z;
  }
}
template <int ACT, typename T>
__device__ __forceinline__ float activation_slope(float z) {
  constexpr bool FAST = sizeof(T) == 2;
  if constexpr (ACT == kActGelu) {
    if constexpr (FAST) {
      const float az = fminf(fabsf(z), 100.f);
      float e;
      const float h = upper_tail(az, e);
      const float s = fmaf(z < 0.f ? -az : az, 0.3989422804014327f * e, z < 0.f ? h : 1.f - h);
      return z != z ? z : s;
    } else {
      return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
    }
  } else if constexpr (ACT == kActRelu) {
    return z > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == kActSilu) {
    float s;
    if constexpr (FAST) s = __fdividef(1.f, 1.f + exp2_approx(-1.4426950408889634f * z));
    else s = 1.f / (1.f + expf(-z));
    return s * fmaf(z, 1.f - s, 1.f);
  } else {
    return 1.f;
  }
}

// One branch for N values instead of one for each.
template <typename T, int N>
__device__ __forceinline__ void activate_all(int act, float* v) {
  switch (act) {
    case kActGelu:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = activate<kActGelu, T>(v[j]);
      break;
    case kActRelu:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = activate<kActRelu, T>(v[j]);
      break;
    case kActSilu:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = activate<kActSilu, T>(v[j]);
      break;
    default: break;
  }
}

}  // namespace wf

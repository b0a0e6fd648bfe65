// The activations of wf_linear and their derivatives, in fp32.
#pragma once

#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

__device__ __forceinline__ float gelu_cdf(float z) { return 0.5f * (1.f + erff(z * 0.70710678118654752f)); }
__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == kActGelu) return z * gelu_cdf(z);
  else if constexpr (ACT == kActRelu) return z < 0.f ? 0.f : z;  // NaN stays
  else if constexpr (ACT == kActSilu) return z * sigmoid(z);
  else return z;
}
template <int ACT>
__device__ __forceinline__ float activation_slope(float z) {
  if constexpr (ACT == kActGelu) return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), gelu_cdf(z));
  else if constexpr (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  else if constexpr (ACT == kActSilu) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.f - s, 1.f);
  } else return 1.f;
}

// One branch for N values instead of one for each.
template <int N>
__device__ __forceinline__ void activate_all(int act, float* v) {
  switch (act) {
    case kActGelu:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = activate<kActGelu>(v[j]);
      break;
    case kActRelu:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = activate<kActRelu>(v[j]);
      break;
    case kActSilu:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = activate<kActSilu>(v[j]);
      break;
    default: break;
  }
}

}  // namespace wf

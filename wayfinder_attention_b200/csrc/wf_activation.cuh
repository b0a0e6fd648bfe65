// The activations of wf_linear and their derivatives, in fp32.
#pragma once

#include "wf_rowio.cuh"
#include "wf_kernels.h"

namespace wf {

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(-|z|) for 16-bit results: Abramowitz and Stegun 7.1.26 (erfc(x) = (a1 t + .. + a5 t^5)
// exp(-x^2), t = 1 / (1 + p x), off by at most 1.5e-7) at x = |z| / sqrt 2.  One reciprocal and
// one exponential, where erff takes both of its branches in most warps.
constexpr float kErfcP = 0.3275911f * 0.70710678118654752f;
constexpr float kErfc0 = 0.5f * 0.254829592f, kErfc1 = 0.5f * -0.284496736f, kErfc2 = 0.5f * 1.421413741f,
                kErfc3 = 0.5f * -1.453152027f, kErfc4 = 0.5f * 1.061405429f;
constexpr float kGaussExp2 = -0.5f * 1.4426950408889634f;  // exp(-z^2 / 2) = 2^(this z^2)
// `e` gets exp(-z^2 / 2).
__device__ __forceinline__ float upper_tail(float az, float& e) {
  const float t = rcp_approx(fmaf(kErfcP, az, 1.f));
  e = exp2_approx(az * az * kGaussExp2);
  float q = fmaf(t, kErfc4, kErfc3);
  q = fmaf(t, q, kErfc2);
  q = fmaf(t, q, kErfc1);
  q = fmaf(t, q, kErfc0);
  return q * t * e;
}

// Two fp32 values an instruction.
struct Pair {
  uint64_t v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float a, float b) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  }
  __device__ __forceinline__ explicit Pair(float a) : Pair(a, a) {}
  __device__ __forceinline__ void get(float& a, float& b) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ float max_keep_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// gelu(z) = max(z, 0) - |z| Phi(-|z|), two at a time with the polynomial in paired
// arithmetic.  Past 100 the tail is 0, and inf * 0 is kept out.
__device__ __forceinline__ void gelu2(float& a, float& b) {
  const Pair az(fminf(fabsf(a), 100.f), fminf(fabsf(b), 100.f));
  float d0, d1, x0, x1;
  fma2(az, Pair(kErfcP), Pair(1.f)).get(d0, d1);
  mul2(mul2(az, Pair(kGaussExp2)), az).get(x0, x1);
  const Pair t(rcp_approx(d0), rcp_approx(d1)), e(exp2_approx(x0), exp2_approx(x1));
  Pair q = fma2(t, Pair(-kErfc4), Pair(-kErfc3));
  q = fma2(t, q, Pair(-kErfc2));
  q = fma2(t, q, Pair(-kErfc1));
  q = fma2(t, q, Pair(-kErfc0));
  q = mul2(mul2(q, t), e);
  fma2(az, q, Pair(max_keep_nan(a, 0.f), max_keep_nan(b, 0.f))).get(a, b);
}

// T: the type of the result.  fp32 takes CUDA's erff and expf and a true division.
template <int ACT, typename T>
__device__ __forceinline__ float activate(float z) {
  constexpr bool FAST = sizeof(T) == 2;
  if constexpr (ACT == kActGelu) {
    static_assert(!FAST, "gelu2 is the 16-bit form");
    return z * 0.5f * (1.f + erff(z * 0.70710678118654752f));
  } else if constexpr (ACT == kActRelu) {
    return z < 0.f ? 0.f : z;  // NaN stays
  } else if constexpr (ACT == kActSilu) {
    if constexpr (FAST) return z * rcp_approx(1.f + exp2_approx(-1.4426950408889634f * z));
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
    if constexpr (FAST) s = rcp_approx(1.f + exp2_approx(-1.4426950408889634f * z));
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
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < N; j += 2) gelu2(v[j], v[j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = activate<kActGelu, T>(v[j]);
      }
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

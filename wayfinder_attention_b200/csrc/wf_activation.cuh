// The activations of wf_linear and their derivatives, in fp32.
#pragma once

#include "wf_rowio.cuh"
#include "wf_kernels.h"
#include "wf_pair.cuh"

namespace wf {

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max_keep_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float max_keep_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// gelu for 16-bit results, two values at a time with the polynomials in paired arithmetic
// (erff takes both of its branches in most warps).  Paired instructions take no immediates:
// the constants are made once, and hidden from the compiler so that it keeps them in registers
// instead of moving them there again for each pair.  B pairs go side by side: a pair alone is
// a chain of some hundred cycles.
__device__ __forceinline__ Pair kept_pair(float x) {
  Pair q(x);
  asm volatile("" : "+l"(q.v));
  return q;
}

// gelu(z) = max(z, 0) - |z| Phi(-|z|) with log2 Phi(-a) as a polynomial in a: one exponential a
// value and no reciprocal.  The logarithm is smooth where Phi itself falls by hundreds of
// binades, so a small error of it is a small RELATIVE error of the tail, which is all of the
// result where z < 0.  The coefficients are a weighted minimax fit (linear programming over 2300
// points of [0, 13.4]): a Phi(-a) is off by at most 2^-20 (1 + a), by 2^-14 of itself down to
// z = -5.8, where fp16 ends, and by 2^-10 beyond, where only bf16 is left.  Half of the
// logarithm is what is computed, and the exponential taken twice: 2^-126 is passed at a = 13 and
// bf16 ends at 13.6.  The bound on a keeps inf * 0 out.  (Abramowitz and Stegun 7.1.28, one
// reciprocal and four squarings, takes as long, 36 us at 32768 x 1024; it is off by 3e-7
// absolutely and so by 5% of the value at z = -5.  A ninth degree takes 1% longer.)
struct Gelu2 {
  Pair c8, c7, c6, c5, c4, c3, c2, c1, c0;  // of log2(Phi(-a)) / 2 in -a
  __device__ __forceinline__ Gelu2()
      : c8(kept_pair(2.07575042e-08f)), c7(kept_pair(1.22331039e-06f)), c6(kept_pair(3.09177485e-05f)),
        c5(kept_pair(0.000444811274f)), c4(kept_pair(0.00411469117f)), c3(kept_pair(0.0266025458f)),
        c2(kept_pair(-0.229678065f)), c1(kept_pair(0.575416028f)), c0(kept_pair(-0.500026405f)) {}
  template <int B>
  __device__ __forceinline__ void apply(float* v) const {
    Pair z[B], q[B];  // z: -|z|
#pragma unroll
    for (int i = 0; i < B; ++i) z[i] = Pair(fmaxf(-fabsf(v[2 * i]), -14.f), fmaxf(-fabsf(v[2 * i + 1]), -14.f));
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(z[i], c8, c7);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(z[i], q[i], c6);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(z[i], q[i], c5);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(z[i], q[i], c4);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(z[i], q[i], c3);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(z[i], q[i], c2);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(z[i], q[i], c1);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float l0, l1;
      fma2(z[i], q[i], c0).get(l0, l1);
      q[i] = Pair(exp2_approx(l0), exp2_approx(l1));
    }
#pragma unroll
    for (int i = 0; i < B; ++i)
      fma2(mul2(z[i], q[i]), q[i], Pair(max_keep_nan(v[2 * i], 0.f), max_keep_nan(v[2 * i + 1], 0.f)))
          .get(v[2 * i], v[2 * i + 1]);
  }
};

// gelu'(z) = Phi(z) + z phi(z).  phi's exponential is needed here, and Abramowitz and Stegun
// 7.1.26 shares it: erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + p x), off by at most
// 1.5e-7, and by 1e-4 of the slope down to z = -6 (z phi(z) is the larger part there).
struct GeluSlope2 {
  static constexpr float kP = 0.3275911f * 0.70710678118654752f, k1 = 0.5f * 0.254829592f, k2 = 0.5f * -0.284496736f,
                         k3 = 0.5f * 1.421413741f, k4 = 0.5f * -1.453152027f, k5 = 0.5f * 1.061405429f,
                         kGauss = -0.5f * 1.4426950408889634f;  // exp(-z^2 / 2) = 2^(this z^2)
  Pair p, g, c5, c4, c3, c2, c1, one;
  __device__ __forceinline__ GeluSlope2()
      : p(kept_pair(kP)), g(kept_pair(kGauss)), c5(kept_pair(-k5)), c4(kept_pair(-k4)), c3(kept_pair(-k3)),
        c2(kept_pair(-k2)), c1(kept_pair(-k1)), one(kept_pair(1.f)) {}
  template <int B>
  __device__ __forceinline__ void apply(float* v) const {
    Pair az[B], t[B], q[B], e[B];  // q: -Phi(-|z|), e: exp(-z^2 / 2)
#pragma unroll
    for (int i = 0; i < B; ++i) {
      az[i] = Pair(fminf(fabsf(v[2 * i]), 100.f), fminf(fabsf(v[2 * i + 1]), 100.f));
      float d0, d1;
      fma2(az[i], p, one).get(d0, d1);
      t[i] = Pair(rcp_approx(d0), rcp_approx(d1));
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float x0, x1;
      mul2(mul2(az[i], g), az[i]).get(x0, x1);
      e[i] = Pair(exp2_approx(x0), exp2_approx(x1));
    }
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(t[i], c5, c4);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(t[i], q[i], c3);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(t[i], q[i], c2);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = fma2(t[i], q[i], c1);
#pragma unroll
    for (int i = 0; i < B; ++i) q[i] = mul2(mul2(q[i], t[i]), e[i]);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float h0, h1, x0, x1, s0, s1;  // x: |z| phi(z)
      q[i].get(h0, h1);
      mul2(mul2(az[i], e[i]), Pair(0.3989422804014327f)).get(x0, x1);
      s0 = v[2 * i] < 0.f ? -(h0 + x0) : 1.f + (h0 + x0);
      s1 = v[2 * i + 1] < 0.f ? -(h1 + x1) : 1.f + (h1 + x1);
      v[2 * i] = v[2 * i] != v[2 * i] ? v[2 * i] : s0;
      v[2 * i + 1] = v[2 * i + 1] != v[2 * i + 1] ? v[2 * i + 1] : s1;
    }
  }
};

// T: the type of the result.  fp32 takes CUDA's erfcf and expf and a true division.
template <int ACT, typename T>
__device__ __forceinline__ float activate(float z) {
  constexpr bool FAST = sizeof(T) == 2;
  if constexpr (ACT == kActGelu) {
    static_assert(!FAST, "Gelu2 is the 16-bit form");
    return z * 0.5f * erfcf(z * -0.70710678118654752f);  // 1 + erff would cancel where z < 0
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
    static_assert(!FAST, "GeluSlope2 is the 16-bit form");
    return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), 0.5f * erfcf(z * -0.70710678118654752f));
  } else if constexpr (ACT == kActRelu) {
    return z > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == kActSilu) {
    float s;
    if constexpr (FAST) s = rcp_approx(1.f + exp2_approx(-1.4426950408889634f * z));
    else s = 1.f / (1.f + expf(-z));
    // z may have been kept as an infinity: 0 times that is the slope's limit, 0
    return s * fmaf(fabsf(z) > 200.f ? 0.f : z, 1.f - s, 1.f);
  } else {
    return 1.f;
  }
}

// How the forward keeps z for the backward: fp16 for both 16-bit types (a slope is flat where
// fp16 ends, and its eleven bits are worth more than bf16's range: with bf16's eight, the
// gradients' rounding errors grew by a half instead of by root two over one rounding).
template <typename T> struct Kept { using type = __half; };
template <> struct Kept<float> { using type = float; };
// What is kept of z; relu's slope asks for the sign only, which a rounding to 0 would lose.
__device__ __forceinline__ float kept_z(int act, float z) { return act == kActRelu && z > 0.f ? fmaxf(z, 6.2e-5f) : z; }

// g[j] *= act'(z[j]), z overwritten.
template <int ACT, typename T, int N>
__device__ __forceinline__ void times_slope(float* z, float* g) {
  if constexpr (ACT == kActNone) {
    return;
  } else if constexpr (ACT == kActGelu && sizeof(T) == 2) {
    const GeluSlope2 gelu;
    gelu.apply<N / 2>(z);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = activation_slope<ACT, T>(z[j]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) g[j] *= z[j];
}

// One branch for N values instead of one for each.
template <typename T, int N>
__device__ __forceinline__ void activate_all(int act, float* v) {
  switch (act) {
    case kActGelu:
      if constexpr (sizeof(T) == 2) {
        const Gelu2 gelu;
        constexpr int BATCH = N < 8 ? N / 2 : 4;
#pragma unroll
        for (int j = 0; j < N; j += 2 * BATCH) gelu.apply<BATCH>(v + j);
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

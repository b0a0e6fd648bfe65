// Row access shared by the row-wise kernels (layer norm, token log probabilities):
// 16-byte vectors where rows allow them, single elements otherwise, always widened
// to fp32 for arithmetic.
#pragma once

#include "wf_common.cuh"

namespace wf {

// 2^x by the hardware's approximation (2 units in the last place; results below 2^-126 are 0)
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// VEC consecutive elements as loaded: 16 bytes, two 16-bit elements, or one of any type.
template <typename T, int VEC> struct RawVec;
template <typename T> struct RawVec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void clear() { v = from_f32<T>(0.f); }
  __device__ __forceinline__ void unpack(float* f) const { f[0] = to_f32(v); }
};
template <typename T> struct RawVec<T, 2> {
  static_assert(sizeof(T) == 2, "four bytes");
  uint32_t v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ void clear() { v = 0; }
  __device__ __forceinline__ void unpack(float* f) const {
    const T* h = reinterpret_cast<const T*>(&v);
    f[0] = to_f32(h[0]);
    f[1] = to_f32(h[1]);
  }
};
template <typename T, int VEC> struct RawVec {
  static_assert(VEC == Vec16<T>::N, "vectors are 16 bytes");
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void unpack(float* f) const { Vec16<T>::unpack(v, f); }
};

__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Rounds VEC fp32 values once to T and stores them.
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(f[0]);
  } else if constexpr (VEC == 2) {
    *reinterpret_cast<uint32_t*>(p) = pack2(T(), f[0], f[1]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    uint4 r;
    r.x = pack2(T(), f[0], f[1]);
    r.y = pack2(T(), f[2], f[3]);
    r.z = pack2(T(), f[4], f[5]);
    r.w = pack2(T(), f[6], f[7]);
    *reinterpret_cast<uint4*>(p) = r;
  }
}

// BYTES (4 or 16) from global to this thread's slot in shared memory, without waiting; a
// group is what was asked for since the last commit, and wait<N> returns once all but the
// newest N groups of this thread have landed.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst_smem, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst_smem), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst_smem), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace wf

// Paired fp32 arithmetic: sm_100 computes two values an instruction (f32x2).
#pragma once

#include <stdint.h>

namespace wf {

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
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

}  // namespace wf

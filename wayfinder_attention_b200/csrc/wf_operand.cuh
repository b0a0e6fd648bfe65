// Matrices as the tensor-core product reads them.
//
// It takes 16-bit matrices whose rows start on 16 bytes.  Others are laid out in
// the workspace first: 16-bit rows of any width or offset are copied to such rows, and an
// fp32 matrix becomes three bf16 pieces, x = x0 + x1 + x2 to fp32's last bit.
#pragma once

#include "wf_gemm.h"
#include "wf_kernels.h"
#include "wf_rowio.cuh"

#include <algorithm>
#include <cstring>
#include <type_traits>

namespace wf {
namespace {

// x = p[0] + p[1] + p[2], each a rounding of what the ones before leave.  Infinities and
// NaN stay in p[0] alone; what would round to infinity is cut instead.
__device__ __forceinline__ void split3(float x, __nv_bfloat16* p) {
  p[0] = __float2bfloat16_rn(x);
  if (isinf(__bfloat162float(p[0])) && !isinf(x)) p[0] = __float2bfloat16_rz(x);
  float r = isfinite(x) ? x - __bfloat162float(p[0]) : 0.f;
  p[1] = __float2bfloat16_rn(r);
  p[2] = __float2bfloat16_rn(r - __bfloat162float(p[1]));
}

// 8 fp32 values to the operand at column c of a row: one 16-byte store a piece (the
// operand's rows are padded to whole vectors).
template <typename T>
__device__ __forceinline__ void store_operand(void* out, int64_t at, int64_t piece, const float* f) {
  if constexpr (std::is_same<T, float>::value) {
    __nv_bfloat16 p[8][3];
#pragma unroll
    for (int j = 0; j < 8; ++j) split3(f[j], p[j]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint4 v;
      uint32_t* u = &v.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __nv_bfloat162 h;
        h.x = p[2 * j][k];
        h.y = p[2 * j + 1][k];
        u[j] = *reinterpret_cast<uint32_t*>(&h);
      }
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + k * piece + at) = v;
    }
  } else {
    store_vec<T, 8>(static_cast<T*>(out) + at, f);
    if (piece) {  // what that rounding leaves, where the operand has a second piece
      float left[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float r = to_f32(from_f32<T>(f[j]));
        left[j] = isfinite(r) ? f[j] - r : 0.f;
      }
      store_vec<T, 8>(static_cast<T*>(out) + piece + at, left);
    }
  }
}

// 8 values of a row from column c (zeros past the end), by vectors where the row allows it.
template <typename T>
struct Raw8 {
  static constexpr int V = Vec16<T>::N;
  uint4 raw[8 / V];
  __device__ __forceinline__ void load(const T* row, int64_t c, int64_t cols, bool vec) {
    if (vec && c + 8 <= cols) {
#pragma unroll
      for (int j = 0; j < 8 / V; ++j) raw[j] = ldg16(row + c + j * V);
    } else {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = c + j < cols ? row[c + j] : from_f32<T>(0.f);
      memcpy(raw, e, sizeof(e));
    }
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) Vec16<T>::unpack(raw[j], f + j * V);
  }
};

// Lays matrices out as operands: the blocks are shared between up to two of them.
template <typename T>
struct LayOut {
  const T* x;
  void* out;
  int64_t rows, cols, stride, pitch, piece;
  int blocks;
  bool vec;
};
template <typename T>
__global__ void __launch_bounds__(256) lay_out_kernel(LayOut<T> first, LayOut<T> second) {
  pdl_wait();
  const bool one = (int)blockIdx.x < first.blocks;
  const LayOut<T>& j = one ? first : second;
  const int64_t block = one ? blockIdx.x : blockIdx.x - first.blocks;
  const int64_t groups = j.pitch / 8, total = j.rows * groups;
  for (int64_t i = block * 256 + threadIdx.x; i < total; i += (int64_t)j.blocks * 256) {
    const int64_t r = i / groups, c = i % groups * 8;
    Raw8<T> raw;
    raw.load(j.x + r * j.stride, c, j.cols, j.vec);
    float f[8];
    raw.unpack(f);
    store_operand<T>(j.out, r * j.pitch + c, j.piece, f);
  }
}

template <typename T>
constexpr int kPieces = std::is_same<T, float>::value ? 3 : 1;

template <typename T>
bool on_16_bytes(const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
}

// A (rows, cols) matrix as the product reads it: itself, or laid out at *ws, which moves on.
template <typename T>
GemmOperand blank_operand(int64_t rows, int64_t cols, int dtype, unsigned char** ws, int turns = 1) {
  GemmOperand o{};
  o.ptr = *ws;
  o.rows = rows;
  o.cols = cols;
  o.pitch = round8(cols);
  o.piece_stride = dtype == kF32 || turns > 1 ? rows * o.pitch : 0;
  *ws += operand_bytes(rows, cols, dtype, turns);
  return o;
}
// Two matrices as operands, either of which may be missing (no pointer); what has to be laid
// out goes in one launch.
struct Matrix {
  const void* ptr;
  int64_t rows, cols, stride;
};
template <typename T>
int operands(const Matrix (&m)[2], int dtype, unsigned char** ws, GemmOperand (&o)[2], cudaStream_t stream) {
  LayOut<T> jobs[2] = {};
  for (int i = 0; i < 2; ++i) {
    if (!m[i].ptr) continue;
    const bool vec = on_16_bytes<T>(m[i].ptr, m[i].stride);
    if (dtype != kF32 && vec) {
      o[i] = GemmOperand{m[i].ptr, m[i].rows, m[i].cols, m[i].stride, 0, false};
      continue;
    }
    o[i] = blank_operand<T>(m[i].rows, m[i].cols, dtype, ws);
    const int64_t blocks = (m[i].rows * (o[i].pitch / 8) + 255) / 256;
    jobs[i] = LayOut<T>{static_cast<const T*>(m[i].ptr), const_cast<void*>(o[i].ptr), m[i].rows, m[i].cols,
                        m[i].stride, o[i].pitch, o[i].piece_stride, (int)std::min<int64_t>(blocks, 16 * kSms), vec};
  }
  const int blocks = jobs[0].blocks + jobs[1].blocks;
  return blocks ? (int)launch_pdl(lay_out_kernel<T>, dim3(blocks), dim3(256), 0, stream, jobs[0], jobs[1]) : 0;
}

template <typename T>
GemmProblem problem(const GemmOperand& a, const GemmOperand& b, int64_t M, int64_t N, int64_t K, int dtype, void* ws,
                    int32_t* status) {
  GemmProblem g{};
  g.a = a;
  g.b = b;
  g.M = M;
  g.N = N;
  g.K = K;
  g.pieces = kPieces<T>;
  g.turns = 1;
  g.op_dtype = dtype == kF16 ? kF16 : kBF16;
  g.out_dtype = dtype;
  g.ws = ws;
  g.status = status;
  return g;
}

}  // namespace
}  // namespace wf

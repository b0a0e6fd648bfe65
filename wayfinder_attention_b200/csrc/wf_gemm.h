// Host interface of the tensor-core product (wf_gemm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "wf_kernels.h"

namespace wf {

inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }
inline int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// A row-major 16-bit matrix whose rows start on 16-byte boundaries.  K-major: rows are the
// product's rows and columns its depth; MN-major: the other way round.  An fp32 matrix is
// `pieces` = 3 of them, piece_stride elements apart.
struct GemmOperand {
  const void* ptr;
  int64_t rows, cols, pitch, piece_stride;
  bool mn_major;
};

// Bytes of a matrix laid out as an operand (wf_operand.cuh).
inline size_t operand_bytes(int64_t rows, int64_t cols, int dtype, int turns = 1) {
  return round256((size_t)rows * round8(cols) * 2 * (dtype == kF32 ? 3 : turns));
}

// C = act(factor A B^T + bias) + residual, or its parts.  Rows of bias/residual/z/y are unit-strided.
struct GemmEpilogue {
  const void* bias;
  const void* residual;
  void* z;
  void* y;
  int64_t r_stride, z_stride, y_stride;
  int act;
  const float* factor;  // one, on the device; null: 1.  Of a bf16 C only
};

struct GemmProblem {
  GemmOperand a, b;
  int64_t M, N, K;
  int pieces;       // 1, or 3 for fp32
  int turns;        // 2 where a 16-bit a is the sum of two pieces (then pieces is 1), else 1
  int op_dtype;     // kBF16 or kF16
  int out_dtype;    // of the epilogue's matrices (z apart): the operands' own, or fp32
  GemmEpilogue out;
  void* ws;         // gemm_workspace_bytes(M, N, K, pieces, turns)
  int32_t* status;
};

size_t gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, int pieces, int turns = 1);
int launch_gemm(const GemmProblem& p, cudaStream_t stream);

}  // namespace wf

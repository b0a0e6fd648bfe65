// The second half of a deterministic column sum: partial rows, added in a fixed order.
#pragma once

#include "wf_common.cuh"

namespace wf {

// partials[blocks][width] fp32 -> one row, rounded once to P: the first `split` columns
// to `a`, the others to `b` (either may be null).  A thread block takes 32 columns; its 32
// warps share the rows.
template <typename P>
__global__ void __launch_bounds__(1024) column_join_kernel(const float* partials, int blocks, int64_t width,
                                                           int64_t split, P* a, P* b) {
  __shared__ float red[32][33];
  pdl_wait();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < width) {
#pragma unroll 4
    for (int r = ty; r < blocks; r += 32) s += partials[(size_t)r * width + c];
  }
  red[ty][tx] = s;
  __syncthreads();
  s = warp_sum(red[tx][ty]);  // column ty of the 32
  const int64_t out = (int64_t)blockIdx.x * 32 + ty;
  if (tx == 0 && out < width) {
    if (out < split) {
      if (a) a[out] = from_f32<P>(s);
    } else if (b) {
      b[out - split] = from_f32<P>(s);
    }
  }
}

template <typename P>
inline cudaError_t join_columns(const float* partials, int blocks, int64_t width, int64_t split, void* a, void* b,
                                cudaStream_t stream) {
  return launch_pdl(column_join_kernel<P>, dim3((unsigned)((width + 31) / 32)), dim3(1024), 0, stream, partials, blocks,
                    width, split, static_cast<P*>(a), static_cast<P*>(b));
}

}  // namespace wf

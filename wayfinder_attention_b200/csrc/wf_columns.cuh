// The second half of a deterministic column sum: partial rows, added in a fixed order.
#pragma once

#include "wf_common.cuh"

namespace wf {

// partials[blocks][width] fp32 -> one row, rounded once to P: the first `split` columns
// to `a`, the others to `b` (either may be null).  32 columns x 8 shares of the blocks
// a thread block.
template <typename P>
__global__ void __launch_bounds__(256) column_join_kernel(const float* partials, int blocks, int64_t width,
                                                          int64_t split, P* a, P* b) {
  __shared__ float red[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < width)
    for (int r = ty; r < blocks; r += 8) s += partials[(size_t)r * width + c];
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][tx];
    if (c < split) {
      if (a) a[c] = from_f32<P>(s);
    } else if (b) {
      b[c - split] = from_f32<P>(s);
    }
  }
}

template <typename P>
inline cudaError_t join_columns(const float* partials, int blocks, int64_t width, int64_t split, void* a, void* b,
                                cudaStream_t stream) {
  column_join_kernel<P><<<(unsigned)((width + 31) / 32), 256, 0, stream>>>(partials, blocks, width, split,
                                                                          static_cast<P*>(a), static_cast<P*>(b));
  return cudaGetLastError();
}

}  // namespace wf

// Host interface of the linear layer over few rows (wf_linear_few.cu).
#pragma once

#include "wf_kernels.h"

namespace wf {

// Up to 16 rows of 16-bit elements on 16 bytes (in a depth of whole pieces), kFewRows otherwise.
constexpr int64_t kFewRows = 8;
bool linear_few_takes(const LinearParams& p, int dtype);
int launch_linear_few(const LinearParams& p, int dtype, cudaStream_t stream);

}  // namespace wf

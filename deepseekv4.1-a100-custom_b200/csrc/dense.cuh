// Internal interface shared by the dense operators (norm.cu, dense.cu).
#pragma once
#include <cuda_runtime.h>

namespace b200 {

// out[c] = sum over p of part[p][c] (fp32 [parts][dim]), in a fixed order; out in `dtype`
int column_sum(const float* part, int parts, int dim, int dtype, void* out, cudaStream_t stream);

}  // namespace b200

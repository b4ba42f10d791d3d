// Tree attention on the matrix instructions (tree_mma.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/iris_b200.h"

namespace iris {

// Head widths of whole 32-value steps; scale below 2^31 (a head of two values
// or more); a bound on the keys whose segments a grid holds (67 million); the row
// kernel takes the rest.
bool tree_mma_usable(const IrisTreeAttention& a);
uint64_t tree_mma_workspace(const IrisTreeAttention& a);
cudaError_t launch_tree_mma(const IrisTreeAttention& a, uint8_t* workspace, cudaStream_t stream);

}  // namespace iris

// Packed prompt attention on the matrix instructions (prompt_mma.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/iris_b200.h"

namespace iris {

// Head widths of whole 32-value steps; scale below 2^31 (a head of two values
// or more); the row kernel takes the rest.
bool prompt_mma_usable(const IrisPromptAttention& a);
uint64_t prompt_mma_workspace(const IrisPromptAttention& a);
cudaError_t launch_prompt_mma(const IrisPromptAttention& a, uint8_t* workspace, cudaStream_t stream);

}  // namespace iris

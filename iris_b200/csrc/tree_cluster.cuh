// Drafted trees of few rows in one launch (tree_cluster.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/iris_b200.h"

namespace iris {

// For calls that tree_mma_usable takes.
bool tree_cluster_usable(const IrisTreeAttention& a);
cudaError_t launch_tree_cluster(const IrisTreeAttention& a, cudaStream_t stream);

}  // namespace iris

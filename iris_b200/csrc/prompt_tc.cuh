// Packed prompt attention on the tcgen05 tensor cores (prompt_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/iris_b200.h"

namespace iris {

struct PromptTcScratch {
  uint8_t *qp, *kp, *vt;  // byte planes
  uint32_t* exp_bits;     // corrections of exp_term_floor
  uint32_t* wide;         // [flags], non-zero where a packing block met a value past 24 bits
  uint64_t tpitch;        // tokens a row of vt
  uint32_t pack_blocks, flags;
  // the item list and score scratch, shared with prompt_mma_kernel
  uint32_t *order, *tiles, *next;
  int32_t* scores;
  uint32_t pitch;
};

// Requests of at most 16,256 rows (the int32 diagonals, and the places on the near list).
bool prompt_tc_usable(const IrisPromptAttention& a);
size_t prompt_tc_carve(const IrisPromptAttention& a, uint8_t* base, PromptTcScratch* sc);
// Packs the operands and runs the attention unless a value is past 24 bits
// (the caller launches prompt_mma_kernel behind it for that).
cudaError_t launch_prompt_tc(const IrisPromptAttention& a, const PromptTcScratch& sc, uint32_t blocks,
                             cudaStream_t stream);

}  // namespace iris

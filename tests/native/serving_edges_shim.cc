// Pieces of the serving kernels as host code, for their edges
// (tests/test_serving_edges.py).
#include "../../iris_b200/csrc/detnum.cuh"

extern "C" {
// The kernels' score of each sum in halves, and the definition's.
void edge_scores(const int64_t* sum, uint64_t n, uint32_t scale, int32_t* got, int32_t* want) {
  for (uint64_t i = 0; i < n; ++i) {
    const int32_t hi = (int32_t)(uint32_t)((uint64_t)sum[i] >> 32);
    const uint32_t lo = (uint32_t)(uint64_t)sum[i];
    got[i] = scale ? iris::score_by<true, true>(hi, lo, scale) : iris::score_by<false, true>(hi, lo, scale);
    want[i] = scale ? iris::scaled_score_finish(sum[i], scale) : iris::requantize(sum[i]);
  }
}
uint32_t edge_place_within(uint32_t first, uint32_t count) { return iris::place_within(first, count); }
}

// The serving kernels' exponential (iris_b200/csrc/detnum.cuh) as host code.
#include "../../iris_b200/csrc/detnum.cuh"

extern "C" {
// term[d] = exp_term_near(d), estimate[d] = exp_term_estimate(d), doubt[d] what
// it says of itself, floor[d] = exp_term_floor(d) and want[d] = softmax_exp_term_act of a score d below the
// maximum, for 1 <= d < 2^20.
void serving_exp_terms(uint32_t* term, uint32_t* estimate, uint8_t* doubt, uint32_t* floor,
                       int64_t* want) {
  for (uint32_t d = 1; d < 1u << 20; ++d) {
    bool may_be_wrong;
    term[d] = iris::exp_term_near(d);
    estimate[d] = iris::exp_term_estimate(d, &may_be_wrong);
    doubt[d] = may_be_wrong;
    floor[d] = iris::exp_term_floor(d);
    want[d] = iris::softmax_exp_term_act(-(int32_t)d, 0);
  }
}
// The weights of n terms, by division and as the step (1 to 65536) that is reached and whose successor is not.
void serving_weights(const int64_t* term, const uint64_t* sum, uint64_t n, int32_t* want, uint8_t* agrees) {
  for (uint64_t i = 0; i < n; ++i) {
    const int32_t w = want[i] = iris::softmax_weight(term[i], sum[i]);
    agrees[i] = (w == 0 || iris::softmax_weight_reaches(term[i], sum[i], w)) &&
                (w == 65536 || !iris::softmax_weight_reaches(term[i], sum[i], w + 1));
  }
}
uint32_t serving_exact_below() { return iris::kExpExactBelow; }
}

// The chunked gated delta rule's kernels for bf16 rows (see delta_rule_chunk.hpp).
#include "delta_rule_chunk.hpp"

namespace ss {
template hipError_t dr_prep_launch<bf16_t>(const DrParams&, hipStream_t);
template hipError_t dr_walk_launch<bf16_t>(const DrParams&, bool, hipStream_t);
template hipError_t dr_grads_launch<bf16_t>(const DrParams&, hipStream_t);
}  // namespace ss

// The chunked gated delta rule's kernels for fp32 rows (see delta_rule_chunk.hpp).
#include "delta_rule_chunk.hpp"

namespace ss {
template hipError_t dr_prep_launch<float>(const DrParams&, hipStream_t);
template hipError_t dr_walk_launch<float>(const DrParams&, bool, hipStream_t);
template hipError_t dr_grads_launch<float>(const DrParams&, hipStream_t);
}  // namespace ss

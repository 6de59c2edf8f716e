// The chunked gated delta rule's kernels for fp16 rows (see delta_rule_chunk.hpp).
#include "delta_rule_chunk.hpp"

namespace ss {
template hipError_t dr_prep_launch<_Float16>(const DrParams&, hipStream_t);
template hipError_t dr_walk_launch<_Float16>(const DrParams&, bool, hipStream_t);
template hipError_t dr_grads_launch<_Float16>(const DrParams&, hipStream_t);
}  // namespace ss

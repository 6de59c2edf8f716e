// The chunked linear attention's kernels for bfloat16 rows (see linear_attn_chunk.hpp).
#include "linear_attn_chunk.hpp"

namespace ss {
template hipError_t la_local_launch<bf16_t>(const LaParams&, hipStream_t);
template hipError_t la_walk_launch<bf16_t>(const LaParams&, bool, hipStream_t);
}  // namespace ss

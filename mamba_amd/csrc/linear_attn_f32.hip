// The chunked linear attention's kernels for fp32 rows (see linear_attn_chunk.hpp).
#include "linear_attn_chunk.hpp"

namespace ss {
template hipError_t la_local_launch<float>(const LaParams&, hipStream_t);
template hipError_t la_walk_launch<float>(const LaParams&, bool, hipStream_t);
}  // namespace ss

// The chunked linear attention's kernels for fp16 rows (see linear_attn_chunk.hpp).
#include "linear_attn_chunk.hpp"

namespace ss {
template hipError_t la_local_launch<_Float16>(const LaParams&, hipStream_t);
template hipError_t la_walk_launch<_Float16>(const LaParams&, bool, hipStream_t);
}  // namespace ss

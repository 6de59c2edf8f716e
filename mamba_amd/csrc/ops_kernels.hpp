// Launcher declarations of the operators beside the scan (internal).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mamba_ss.h"

namespace ss {

// linear attention with a decay for each head (linear_attn.hip): tokens per
// segment, segments (at least 1), workspace bytes, launches
int64_t linear_attn_segment(const ss_linear_attn_args* a);
int64_t linear_attn_segs(const ss_linear_attn_args* a);
int64_t linear_attn_fwd_space(const ss_linear_attn_args* a);
int64_t linear_attn_bwd_space(const ss_linear_attn_bwd_args* g);
hipError_t linear_attn_fwd_launch(const ss_linear_attn_args* a, hipStream_t stream);
hipError_t linear_attn_bwd_launch(const ss_linear_attn_bwd_args* g, hipStream_t stream);
hipError_t linear_attn_update_launch(const ss_linear_attn_update_args* a, hipStream_t stream);
constexpr int64_t kLinearAttnMaxDim = 256, kLinearAttnMaxRows = int64_t(1) << 20;   // rows: batch * heads
// the norms around a block and the gated norm of each head (block_norm.hip)
int64_t block_norm_bwd_space(int64_t rows, int64_t dim);
int64_t gated_norm_bwd_space(int64_t rows, int64_t dim, int64_t groups);
hipError_t block_norm_fwd_launch(const ss_block_norm_args* a, hipStream_t stream);
hipError_t block_norm_bwd_launch(const ss_block_norm_bwd_args* g, hipStream_t stream);
hipError_t gated_norm_fwd_launch(const ss_gated_norm_args* a, hipStream_t stream);
hipError_t gated_norm_bwd_launch(const ss_gated_norm_bwd_args* g, hipStream_t stream);
constexpr int64_t kBlockNormMaxDim = 16384;      // a row lies in the registers of one workgroup
// the norm over many tensors (clip_grads.hip)
int64_t clip_grads_chunks(const ss_clip_grads_args* a);
hipError_t clip_grads_launch(const ss_clip_grads_args* a, hipStream_t stream);

}  // namespace ss

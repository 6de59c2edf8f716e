// The C ABI of the operators beside the scan: linear attention, the delta rule, the
// norms, gradient clipping.  One unit with ss_api.hip, whose checks and
// last error (per thread) it shares.
#include "ss_api.hip"

#include <new>

#include "ops_kernels.hpp"
#include "overlap.hpp"

extern "C" {

// Checks shared by the linear attention's calls.
static int check_linear_attn(const ss_linear_attn_args* a, bool bwd) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    const int64_t sizes[] = {a->batch, a->seqlen, a->heads, a->groups};
    for (int64_t n : sizes)
        if (n < 0)
            return fail(SS_ERR_INVALID, "negative size (batch=%lld seqlen=%lld heads=%lld groups=%lld)", (long long)a->batch,
                        (long long)a->seqlen, (long long)a->heads, (long long)a->groups);
    if (a->dtype != SS_F32 && a->dtype != SS_BF16 && a->dtype != SS_F16)
        return fail(SS_ERR_INVALID, "unknown dtype %d", a->dtype);
    if (a->d_key < 1 || a->d_key > ss::kLinearAttnMaxDim || a->d_value < 1 || a->d_value > ss::kLinearAttnMaxDim)
        return fail(SS_ERR_UNSUPPORTED, "d_key=%lld, d_value=%lld outside [1, %lld]", (long long)a->d_key,
                    (long long)a->d_value, (long long)ss::kLinearAttnMaxDim);
    if (a->heads > 0 && (a->groups < 1 || a->heads % a->groups != 0))
        return fail(SS_ERR_INVALID, "heads=%lld is not a multiple of groups=%lld", (long long)a->heads, (long long)a->groups);
    // (a launch holds at most batch x heads x 48 workgroups of 64 threads: three passes, 16 column tiles; and 2^32 threads)
    if (a->batch > 0 && a->heads > ss::kLinearAttnMaxRows / a->batch) return fail(SS_ERR_UNSUPPORTED, "batch * heads too large");
    if (a->seqlen > (int64_t(1) << 24)) return fail(SS_ERR_UNSUPPORTED, "seqlen=%lld above 2^24", (long long)a->seqlen);
    const int64_t st[] = {a->q_batch_stride, a->q_len_stride, a->q_head_stride, a->k_batch_stride, a->k_len_stride,
                          a->k_head_stride, a->v_batch_stride, a->v_len_stride, a->v_head_stride, a->g_batch_stride,
                          a->g_len_stride, a->g_head_stride};
    for (int64_t v : st)
        if (v < 0) return fail(SS_ERR_INVALID, "negative stride");
    if (a->batch == 0 || a->heads == 0) return ok();
    const size_t es = elem_size(a->dtype);
    if (a->seqlen > 0) {
        if (!a->q || !a->k || !a->v || !a->g) return fail(SS_ERR_INVALID, "q / k / v / g is NULL");
        if (!aligned(a->q, es) || !aligned(a->k, es) || !aligned(a->v, es) || !aligned(a->g, 4))
            return fail(SS_ERR_INVALID, "q / k / v / g is misaligned");
    }
    if (!aligned(a->initial_state, 4) || !aligned(a->lengths, 4) || !aligned(a->ends, 4))
        return fail(SS_ERR_INVALID, "initial_state / lengths / ends is misaligned");
    if (!bwd) {
        if (a->out_batch_stride < 0 || a->out_len_stride < 0 || a->out_head_stride < 0)
            return fail(SS_ERR_INVALID, "negative stride");
        if (a->seqlen > 0 && !a->out) return fail(SS_ERR_INVALID, "out is NULL");
        if (!aligned(a->out, es) || !aligned(a->last_state, 4))
            return fail(SS_ERR_INVALID, "out / last_state is misaligned");
    }
    return ok();
}

static int check_linear_attn_bwd(const ss_linear_attn_bwd_args* g) {
    const int rc = check_linear_attn(g ? &g->f : nullptr, true);
    if (rc != SS_OK || g->f.batch == 0 || g->f.heads == 0) return rc;
    if (g->dout_batch_stride < 0 || g->dout_len_stride < 0 || g->dout_head_stride < 0)
        return fail(SS_ERR_INVALID, "negative stride");
    if (!g->dg || (g->f.seqlen > 0 && (!g->dout || !g->dq || !g->dk || !g->dv)))
        return fail(SS_ERR_INVALID, "dout / dq / dk / dv / dg is NULL");
    if (!g->f.ends) return fail(SS_ERR_INVALID, "ends (the forward's states) is NULL");
    const size_t es = elem_size(g->f.dtype);
    if (!aligned(g->dout, es) || !aligned(g->dq, es) || !aligned(g->dk, es) || !aligned(g->dv, es) ||
        !aligned(g->dg, 4) || !aligned(g->dlast_state, 4) || !aligned(g->dinitial_state, 4))
        return fail(SS_ERR_INVALID, "a gradient is misaligned");
    return ok();
}

static int check_space(const void* workspace, int64_t bytes, int64_t need) {
    if (need > 0 && (!workspace || bytes < need))
        return fail(SS_ERR_INVALID, "workspace of %lld bytes needed (got %lld)", (long long)need,
                    (long long)(workspace ? bytes : 0));
    if (workspace && !aligned(workspace, 16)) return fail(SS_ERR_INVALID, "workspace must be 16-byte aligned");
    return SS_OK;
}

int64_t ss_linear_attn_segment(const ss_linear_attn_args* a) {
    return check_linear_attn(a, true) == SS_OK ? ss::linear_attn_segment(a) : -1;
}

int64_t ss_linear_attn_fwd_workspace_bytes(const ss_linear_attn_args* a) {
    return check_linear_attn(a, false) == SS_OK ? ss::linear_attn_fwd_space(a) : -1;
}

int64_t ss_linear_attn_bwd_workspace_bytes(const ss_linear_attn_bwd_args* g) {
    return check_linear_attn_bwd(g) == SS_OK ? ss::linear_attn_bwd_space(g) : -1;
}

int ss_linear_attn_fwd(const ss_linear_attn_args* a, void* stream) {
    int rc = check_linear_attn(a, false);
    if (rc != SS_OK || a->batch == 0 || a->heads == 0) return rc;
    rc = check_space(a->workspace, a->workspace_bytes, ss::linear_attn_fwd_space(a));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::linear_attn_fwd_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "linear attention forward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_linear_attn_bwd(const ss_linear_attn_bwd_args* g, void* stream) {
    int rc = check_linear_attn_bwd(g);
    if (rc != SS_OK || g->f.batch == 0 || g->f.heads == 0) return rc;
    rc = check_space(g->f.workspace, g->f.workspace_bytes, ss::linear_attn_bwd_space(g));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::linear_attn_bwd_launch(g, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "linear attention backward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_linear_attn_update(const ss_linear_attn_update_args* a, void* stream) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    if (a->batch < 0 || a->heads < 0 || a->groups < 0)
        return fail(SS_ERR_INVALID, "negative size (batch=%lld heads=%lld groups=%lld)", (long long)a->batch,
                    (long long)a->heads, (long long)a->groups);
    if (a->dtype != SS_F32 && a->dtype != SS_BF16 && a->dtype != SS_F16)
        return fail(SS_ERR_INVALID, "unknown dtype %d", a->dtype);
    if (a->d_key < 1 || a->d_key > ss::kLinearAttnMaxDim || a->d_value < 1 || a->d_value > ss::kLinearAttnMaxDim)
        return fail(SS_ERR_UNSUPPORTED, "d_key=%lld, d_value=%lld outside [1, %lld]", (long long)a->d_key,
                    (long long)a->d_value, (long long)ss::kLinearAttnMaxDim);
    if (a->heads > 0 && (a->groups < 1 || a->heads % a->groups != 0))
        return fail(SS_ERR_INVALID, "heads=%lld is not a multiple of groups=%lld", (long long)a->heads, (long long)a->groups);
    if (a->batch > 0 && a->heads > ss::kLinearAttnMaxRows / a->batch) return fail(SS_ERR_UNSUPPORTED, "batch * heads too large");
    const int64_t st[] = {a->state_batch_stride, a->state_head_stride, a->q_batch_stride, a->q_head_stride, a->k_batch_stride,
                          a->k_head_stride, a->v_batch_stride, a->v_head_stride, a->out_batch_stride, a->out_head_stride,
                          a->g_batch_stride, a->g_head_stride};
    for (int64_t v : st)
        if (v < 0) return fail(SS_ERR_INVALID, "negative stride");
    if (a->batch == 0 || a->heads == 0) return ok();
    if (!a->state || !a->q || !a->k || !a->v || !a->g || !a->out)
        return fail(SS_ERR_INVALID, "state / q / k / v / g / out is NULL");
    const size_t es = elem_size(a->dtype);
    if (!aligned(a->state, 4) || !aligned(a->g, 4) || !aligned(a->q, es) || !aligned(a->k, es) || !aligned(a->v, es) ||
        !aligned(a->out, es))
        return fail(SS_ERR_INVALID, "state / q / k / v / g / out is misaligned");
    if (ss::blocks_overlap(a->batch, a->state_batch_stride, a->heads, a->state_head_stride, a->d_key * a->d_value))
        return fail(SS_ERR_INVALID, "state's elements overlap (strides %lld, %lld): it is updated in place",
                    (long long)a->state_batch_stride, (long long)a->state_head_stride);
    if (ss::blocks_overlap(a->batch, a->out_batch_stride, a->heads, a->out_head_stride, a->d_value))
        return fail(SS_ERR_INVALID, "out's elements overlap (strides %lld, %lld)", (long long)a->out_batch_stride,
                    (long long)a->out_head_stride);
    const hipError_t e = ss::linear_attn_update_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "linear attention update launch failed: %s", hipGetErrorString(e));
    return ok();
}

// Checks shared by the delta rule's calls.
static int check_delta_rule(const ss_delta_rule_args* a, bool bwd) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    const int64_t sizes[] = {a->batch, a->seqlen, a->heads, a->groups};
    for (int64_t n : sizes)
        if (n < 0)
            return fail(SS_ERR_INVALID, "negative size (batch=%lld seqlen=%lld heads=%lld groups=%lld)", (long long)a->batch,
                        (long long)a->seqlen, (long long)a->heads, (long long)a->groups);
    if (a->dtype != SS_F32 && a->dtype != SS_BF16 && a->dtype != SS_F16)
        return fail(SS_ERR_INVALID, "unknown dtype %d", a->dtype);
    if (a->d_key < 1 || a->d_key > ss::kDeltaRuleMaxDim || a->d_value < 1 || a->d_value > ss::kDeltaRuleMaxDim)
        return fail(SS_ERR_UNSUPPORTED, "d_key=%lld, d_value=%lld outside [1, %lld]", (long long)a->d_key,
                    (long long)a->d_value, (long long)ss::kDeltaRuleMaxDim);
    if (a->heads > 0 && (a->groups < 1 || a->heads % a->groups != 0))
        return fail(SS_ERR_INVALID, "heads=%lld is not a multiple of groups=%lld", (long long)a->heads, (long long)a->groups);
    if (a->batch > 0 && a->heads > ss::kLinearAttnMaxRows / a->batch) return fail(SS_ERR_UNSUPPORTED, "batch * heads too large");
    if (a->seqlen > (int64_t(1) << 24)) return fail(SS_ERR_UNSUPPORTED, "seqlen=%lld above 2^24", (long long)a->seqlen);
    if (a->batch > 0 && a->heads > 0 && ss::delta_rule_chunks(a) > ss::kDeltaRuleMaxChunks)
        return fail(SS_ERR_UNSUPPORTED, "batch * heads * seqlen too large");
    const int64_t st[] = {a->q_batch_stride, a->q_len_stride, a->q_head_stride, a->k_batch_stride, a->k_len_stride,
                          a->k_head_stride, a->v_batch_stride, a->v_len_stride, a->v_head_stride, a->g_batch_stride,
                          a->g_len_stride, a->g_head_stride, a->beta_batch_stride, a->beta_len_stride, a->beta_head_stride};
    for (int64_t v : st)
        if (v < 0) return fail(SS_ERR_INVALID, "negative stride");
    if (a->batch == 0 || a->heads == 0) return ok();
    const size_t es = elem_size(a->dtype);
    if (a->seqlen > 0) {
        if (!a->q || !a->k || !a->v || !a->g || !a->beta) return fail(SS_ERR_INVALID, "q / k / v / g / beta is NULL");
        if (!aligned(a->q, es) || !aligned(a->k, es) || !aligned(a->v, es) || !aligned(a->g, 4) || !aligned(a->beta, 4))
            return fail(SS_ERR_INVALID, "q / k / v / g / beta is misaligned");
    }
    if (!aligned(a->initial_state, 4) || !aligned(a->lengths, 4)) return fail(SS_ERR_INVALID, "initial_state / lengths is misaligned");
    if (!bwd) {
        if (a->out_batch_stride < 0 || a->out_len_stride < 0 || a->out_head_stride < 0)
            return fail(SS_ERR_INVALID, "negative stride");
        if (a->seqlen > 0 && !a->out) return fail(SS_ERR_INVALID, "out is NULL");
        if (!aligned(a->out, es) || !aligned(a->last_state, 4))
            return fail(SS_ERR_INVALID, "out / last_state is misaligned");
    }
    return ok();
}

static int check_delta_rule_bwd(const ss_delta_rule_bwd_args* g) {
    const int rc = check_delta_rule(g ? &g->f : nullptr, true);
    if (rc != SS_OK || g->f.batch == 0 || g->f.heads == 0) return rc;
    if (g->dout_batch_stride < 0 || g->dout_len_stride < 0 || g->dout_head_stride < 0)
        return fail(SS_ERR_INVALID, "negative stride");
    if (g->f.seqlen > 0 && (!g->dout || !g->dq || !g->dk || !g->dv || !g->dg || !g->dbeta))
        return fail(SS_ERR_INVALID, "dout / dq / dk / dv / dg / dbeta is NULL");
    const size_t es = elem_size(g->f.dtype);
    if (!aligned(g->dout, es) || !aligned(g->dq, es) || !aligned(g->dk, es) || !aligned(g->dv, es) ||
        !aligned(g->dg, 4) || !aligned(g->dbeta, 4) || !aligned(g->dlast_state, 4) || !aligned(g->dinitial_state, 4))
        return fail(SS_ERR_INVALID, "a gradient is misaligned");
    return ok();
}

// what the forward keeps for the backward
static int check_saved(const ss_delta_rule_args* a, bool need) {
    const int64_t n = ss::delta_rule_saved_bytes(a);
    if ((need && n > 0 && !a->saved) || (a->saved && a->saved_bytes < n))
        return fail(SS_ERR_INVALID, "saved of %lld bytes needed (got %lld)", (long long)n, (long long)(a->saved ? a->saved_bytes : 0));
    if (!aligned(a->saved, 16)) return fail(SS_ERR_INVALID, "saved must be 16-byte aligned");
    return SS_OK;
}

int64_t ss_delta_rule_saved_bytes(const ss_delta_rule_args* a) {
    if (check_delta_rule(a, true) != SS_OK) return -1;
    return a->batch == 0 || a->heads == 0 ? 0 : ss::delta_rule_saved_bytes(a);
}

int64_t ss_delta_rule_fwd_workspace_bytes(const ss_delta_rule_args* a) {
    if (check_delta_rule(a, false) != SS_OK) return -1;
    return a->batch == 0 || a->heads == 0 ? 0 : ss::delta_rule_fwd_space(a);
}

int64_t ss_delta_rule_bwd_workspace_bytes(const ss_delta_rule_bwd_args* g) {
    if (check_delta_rule_bwd(g) != SS_OK) return -1;
    return g->f.batch == 0 || g->f.heads == 0 ? 0 : ss::delta_rule_bwd_space(g);
}

int ss_delta_rule_fwd(const ss_delta_rule_args* a, void* stream) {
    int rc = check_delta_rule(a, false);
    if (rc != SS_OK || a->batch == 0 || a->heads == 0) return rc;
    rc = check_saved(a, false);
    if (rc == SS_OK) rc = check_space(a->workspace, a->workspace_bytes, ss::delta_rule_fwd_space(a));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::delta_rule_fwd_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "delta rule forward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_delta_rule_bwd(const ss_delta_rule_bwd_args* g, void* stream) {
    int rc = check_delta_rule_bwd(g);
    if (rc != SS_OK || g->f.batch == 0 || g->f.heads == 0) return rc;
    rc = check_saved(&g->f, true);
    if (rc == SS_OK) rc = check_space(g->f.workspace, g->f.workspace_bytes, ss::delta_rule_bwd_space(g));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::delta_rule_bwd_launch(g, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "delta rule backward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_delta_rule_update(const ss_delta_rule_update_args* a, void* stream) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    if (a->batch < 0 || a->heads < 0 || a->groups < 0)
        return fail(SS_ERR_INVALID, "negative size (batch=%lld heads=%lld groups=%lld)", (long long)a->batch,
                    (long long)a->heads, (long long)a->groups);
    if (a->dtype != SS_F32 && a->dtype != SS_BF16 && a->dtype != SS_F16)
        return fail(SS_ERR_INVALID, "unknown dtype %d", a->dtype);
    if (a->d_key < 1 || a->d_key > ss::kDeltaRuleMaxDim || a->d_value < 1 || a->d_value > ss::kDeltaRuleMaxDim)
        return fail(SS_ERR_UNSUPPORTED, "d_key=%lld, d_value=%lld outside [1, %lld]", (long long)a->d_key,
                    (long long)a->d_value, (long long)ss::kDeltaRuleMaxDim);
    if (a->heads > 0 && (a->groups < 1 || a->heads % a->groups != 0))
        return fail(SS_ERR_INVALID, "heads=%lld is not a multiple of groups=%lld", (long long)a->heads, (long long)a->groups);
    if (a->batch > 0 && a->heads > ss::kLinearAttnMaxRows / a->batch) return fail(SS_ERR_UNSUPPORTED, "batch * heads too large");
    const int64_t st[] = {a->state_batch_stride, a->state_head_stride, a->q_batch_stride, a->q_head_stride, a->k_batch_stride,
                          a->k_head_stride, a->v_batch_stride, a->v_head_stride, a->out_batch_stride, a->out_head_stride,
                          a->g_batch_stride, a->g_head_stride, a->beta_batch_stride, a->beta_head_stride};
    for (int64_t v : st)
        if (v < 0) return fail(SS_ERR_INVALID, "negative stride");
    if (a->batch == 0 || a->heads == 0) return ok();
    if (!a->state || !a->q || !a->k || !a->v || !a->g || !a->beta || !a->out)
        return fail(SS_ERR_INVALID, "state / q / k / v / g / beta / out is NULL");
    const size_t es = elem_size(a->dtype);
    if (!aligned(a->state, 4) || !aligned(a->g, 4) || !aligned(a->beta, 4) || !aligned(a->q, es) || !aligned(a->k, es) ||
        !aligned(a->v, es) || !aligned(a->out, es))
        return fail(SS_ERR_INVALID, "state / q / k / v / g / beta / out is misaligned");
    if (ss::blocks_overlap(a->batch, a->state_batch_stride, a->heads, a->state_head_stride, a->d_key * a->d_value))
        return fail(SS_ERR_INVALID, "state's elements overlap (strides %lld, %lld): it is updated in place",
                    (long long)a->state_batch_stride, (long long)a->state_head_stride);
    if (ss::blocks_overlap(a->batch, a->out_batch_stride, a->heads, a->out_head_stride, a->d_value))
        return fail(SS_ERR_INVALID, "out's elements overlap (strides %lld, %lld)", (long long)a->out_batch_stride,
                    (long long)a->out_head_stride);
    const hipError_t e = ss::delta_rule_update_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "delta rule update launch failed: %s", hipGetErrorString(e));
    return ok();
}

static int check_block_norm(int64_t rows, int64_t dim, int dtype, int w_dtype) {
    if (rows < 0 || dim < 0)
        return fail(SS_ERR_INVALID, "negative size (rows=%lld dim=%lld)", (long long)rows, (long long)dim);
    if (dtype != SS_F32 && dtype != SS_BF16 && dtype != SS_F16) return fail(SS_ERR_INVALID, "unknown dtype %d", dtype);
    if (w_dtype != dtype && w_dtype != SS_F32)
        return fail(SS_ERR_UNSUPPORTED, "weight dtype %d must be the row dtype or fp32", w_dtype);
    if (dim > ss::kBlockNormMaxDim)
        return fail(SS_ERR_UNSUPPORTED, "dim=%lld above %lld", (long long)dim, (long long)ss::kBlockNormMaxDim);
    return SS_OK;
}

struct NormPtr { const void* p; int64_t stride; bool need; const char* name; };
// rows: present where needed, aligned to the element, strides not negative
static int check_norm_ptrs(std::initializer_list<NormPtr> rows, size_t es) {
    for (const NormPtr& r : rows) {
        if (!r.p) {
            if (r.need) return fail(SS_ERR_INVALID, "%s is NULL", r.name);
            continue;
        }
        if (!aligned(r.p, es)) return fail(SS_ERR_INVALID, "%s is misaligned", r.name);
        if (r.stride < 0) return fail(SS_ERR_INVALID, "negative row stride of %s", r.name);
    }
    return SS_OK;
}

int64_t ss_block_norm_bwd_workspace_bytes(int64_t rows, int64_t dim) {
    if (rows < 0 || dim < 0 || dim > ss::kBlockNormMaxDim) {
        fail(SS_ERR_INVALID, "rows=%lld, dim=%lld out of range", (long long)rows, (long long)dim);
        return -1;
    }
    return ss::block_norm_bwd_space(rows, dim);
}

int ss_block_norm_fwd(const ss_block_norm_args* a, void* stream) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    int rc = check_block_norm(a->rows, a->dim, a->dtype, a->w_dtype);
    if (rc != SS_OK) return rc;
    if (!(a->eps >= 0.f)) return fail(SS_ERR_INVALID, "eps must be >= 0");
    if (a->rows == 0 || a->dim == 0) return ok();
    rc = check_norm_ptrs({{a->x, a->x_row_stride, true, "x"}, {a->residual, a->residual_row_stride, true, "residual"},
                          {a->gate, a->gate_row_stride, false, "gate"}, {a->out, a->out_row_stride, true, "out"},
                          {a->residual_out, a->residual_out_row_stride, true, "residual_out"}}, elem_size(a->dtype));
    if (rc == SS_OK)
        rc = check_norm_ptrs({{a->post, 0, true, "post"}, {a->pre, 0, true, "pre"}, {a->scale_vec, 0, false, "scale_vec"}},
                             elem_size(a->w_dtype));
    if (rc == SS_OK) rc = check_norm_ptrs({{a->rstd, 0, false, "rstd"}}, 4);
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::block_norm_fwd_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "block norm forward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_block_norm_bwd(const ss_block_norm_bwd_args* g, void* stream) {
    if (!g) return fail(SS_ERR_INVALID, "null argument block");
    int rc = check_block_norm(g->rows, g->dim, g->dtype, g->w_dtype);
    if (rc != SS_OK) return rc;
    if (g->dim == 0) return ok();
    rc = check_norm_ptrs({{g->post, 0, true, "post"}, {g->pre, 0, true, "pre"}, {g->scale_vec, 0, false, "scale_vec"},
                          {g->dpost, 0, true, "dpost"}, {g->dpre, 0, true, "dpre"}, {g->dscale, 0, false, "dscale"}},
                         elem_size(g->w_dtype));
    if (rc == SS_OK && g->rows > 0) {
        rc = check_norm_ptrs({{g->x, g->x_row_stride, true, "x"}, {g->residual, g->residual_row_stride, true, "residual"},
                              {g->gate, g->gate_row_stride, false, "gate"}, {g->dout, g->dout_row_stride, false, "dout"},
                              {g->dresidual_out, g->dresidual_out_row_stride, false, "dresidual_out"},
                              {g->dx, 0, true, "dx"}, {g->dresidual, 0, false, "dresidual"},
                              {g->gate ? g->dgate : nullptr, 0, g->gate != nullptr, "dgate"}}, elem_size(g->dtype));
        if (rc == SS_OK) rc = check_norm_ptrs({{g->rstd, 0, true, "rstd"}}, 4);
    }
    if (rc == SS_OK) rc = check_space(g->workspace, g->workspace_bytes, ss::block_norm_bwd_space(g->rows, g->dim));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::block_norm_bwd_launch(g, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "block norm backward launch failed: %s", hipGetErrorString(e));
    return ok();
}

static int check_groups(int64_t dim, int64_t groups) {
    if (groups < 1 || dim % groups != 0)
        return fail(SS_ERR_INVALID, "dim=%lld is not a multiple of groups=%lld", (long long)dim, (long long)groups);
    return SS_OK;
}

int64_t ss_gated_norm_bwd_workspace_bytes(int64_t rows, int64_t dim, int64_t groups) {
    if (rows < 0 || dim < 0 || dim > ss::kBlockNormMaxDim) {
        fail(SS_ERR_INVALID, "rows=%lld, dim=%lld out of range", (long long)rows, (long long)dim);
        return -1;
    }
    if (check_groups(dim, groups) != SS_OK) return -1;
    return dim > 0 ? ss::gated_norm_bwd_space(rows, dim, groups) : 0;
}

int ss_gated_norm_fwd(const ss_gated_norm_args* a, void* stream) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    int rc = check_block_norm(a->rows, a->dim, a->dtype, a->w_dtype);
    if (rc == SS_OK) rc = check_groups(a->dim, a->groups);
    if (rc != SS_OK) return rc;
    if (!(a->eps >= 0.f)) return fail(SS_ERR_INVALID, "eps must be >= 0");
    if (a->rows == 0 || a->dim == 0) return ok();
    rc = check_norm_ptrs({{a->x, a->x_row_stride, true, "x"}, {a->gate, a->gate_row_stride, true, "gate"},
                          {a->out, a->out_row_stride, true, "out"}}, elem_size(a->dtype));
    if (rc == SS_OK) rc = check_norm_ptrs({{a->weight, 0, true, "weight"}}, elem_size(a->w_dtype));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::gated_norm_fwd_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "gated norm forward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_gated_norm_bwd(const ss_gated_norm_bwd_args* g, void* stream) {
    if (!g) return fail(SS_ERR_INVALID, "null argument block");
    int rc = check_block_norm(g->rows, g->dim, g->dtype, g->w_dtype);
    if (rc == SS_OK) rc = check_groups(g->dim, g->groups);
    if (rc != SS_OK) return rc;
    if (!(g->eps >= 0.f)) return fail(SS_ERR_INVALID, "eps must be >= 0");
    if (g->dim == 0) return ok();
    rc = check_norm_ptrs({{g->weight, 0, true, "weight"}, {g->dweight, 0, true, "dweight"}}, elem_size(g->w_dtype));
    if (rc == SS_OK && g->rows > 0)
        rc = check_norm_ptrs({{g->x, g->x_row_stride, true, "x"}, {g->gate, g->gate_row_stride, true, "gate"},
                              {g->dout, g->dout_row_stride, true, "dout"}, {g->dx, 0, true, "dx"},
                              {g->dgate, 0, true, "dgate"}}, elem_size(g->dtype));
    if (rc == SS_OK)
        rc = check_space(g->workspace, g->workspace_bytes, ss::gated_norm_bwd_space(g->rows, g->dim, g->groups));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::gated_norm_bwd_launch(g, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "gated norm backward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int64_t ss_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t dim) {
    if (rows < 0 || dim < 0 || dim > ss::kBlockNormMaxDim) {
        fail(SS_ERR_INVALID, "rows=%lld, dim=%lld out of range", (long long)rows, (long long)dim);
        return -1;
    }
    return ss::layer_norm_bwd_space(rows, dim);
}

int ss_layer_norm_fwd(const ss_layer_norm_args* a, void* stream) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    int rc = check_block_norm(a->rows, a->dim, a->dtype, a->w_dtype);
    if (rc != SS_OK) return rc;
    if (!(a->eps >= 0.f)) return fail(SS_ERR_INVALID, "eps must be >= 0");
    if (a->rows == 0 || a->dim == 0) return ok();
    rc = check_norm_ptrs({{a->x, a->x_row_stride, true, "x"}, {a->residual, a->residual_row_stride, false, "residual"},
                          {a->out, a->out_row_stride, true, "out"},
                          {a->residual_out, a->residual_out_row_stride, false, "residual_out"}}, elem_size(a->dtype));
    if (rc == SS_OK) rc = check_norm_ptrs({{a->weight, 0, true, "weight"}, {a->bias, 0, false, "bias"}}, elem_size(a->w_dtype));
    if (rc == SS_OK) rc = check_norm_ptrs({{a->stats, 0, false, "stats"}}, 4);
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::layer_norm_fwd_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "layer norm forward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_layer_norm_bwd(const ss_layer_norm_bwd_args* g, void* stream) {
    if (!g) return fail(SS_ERR_INVALID, "null argument block");
    int rc = check_block_norm(g->rows, g->dim, g->dtype, g->w_dtype);
    if (rc != SS_OK) return rc;
    if (g->dim == 0) return ok();
    rc = check_norm_ptrs({{g->weight, 0, true, "weight"}, {g->dweight, 0, true, "dweight"}, {g->dbias, 0, false, "dbias"}},
                         elem_size(g->w_dtype));
    if (rc == SS_OK && g->rows > 0) {
        rc = check_norm_ptrs({{g->s, g->s_row_stride, true, "s"}, {g->dout, g->dout_row_stride, false, "dout"},
                              {g->dresidual_out, g->dresidual_out_row_stride, false, "dresidual_out"},
                              {g->dx, 0, true, "dx"}}, elem_size(g->dtype));
        if (rc == SS_OK) rc = check_norm_ptrs({{g->stats, 0, true, "stats"}}, 4);
    }
    if (rc == SS_OK) rc = check_space(g->workspace, g->workspace_bytes, ss::layer_norm_bwd_space(g->rows, g->dim));
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::layer_norm_bwd_launch(g, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "layer norm backward launch failed: %s", hipGetErrorString(e));
    return ok();
}

int ss_unit_norm(const ss_unit_norm_args* a, void* stream) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    const int rc = check_block_norm(a->rows, a->dim, a->dtype, a->dtype);
    if (rc != SS_OK) return rc;
    if (a->heads < 0) return fail(SS_ERR_INVALID, "negative size (heads=%lld)", (long long)a->heads);
    if (!(a->eps >= 0.f)) return fail(SS_ERR_INVALID, "eps must be >= 0");
    if (a->rows == 0 || a->heads == 0 || a->dim == 0) return ok();
    if (a->rows > ((int64_t(1) << 32) - 1) / a->heads) return fail(SS_ERR_UNSUPPORTED, "rows * heads too large");
    const int rp = check_norm_ptrs({{a->x, a->x_row_stride, true, "x"}, {a->x, a->x_head_stride, true, "x"},
                                    {a->dout, a->dout_row_stride, false, "dout"}, {a->dout, a->dout_head_stride, false, "dout"},
                                    {a->out, 0, true, "out"}}, elem_size(a->dtype));
    if (rp != SS_OK) return rp;
    const hipError_t e = ss::unit_norm_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "unit norm launch failed: %s", hipGetErrorString(e));
    return ok();
}

static int check_clip_grads(const ss_clip_grads_args* a) {
    if (!a) return fail(SS_ERR_INVALID, "null argument block");
    if (a->count < 0) return fail(SS_ERR_INVALID, "negative count");
    if (a->count > 0 && (!a->grads || !a->outs || !a->numels || !a->dtypes))
        return fail(SS_ERR_INVALID, "grads / outs / numels / dtypes is NULL");
    int64_t total = 0;
    for (int64_t i = 0; i < a->count; ++i) {
        if (a->dtypes[i] != SS_F32 && a->dtypes[i] != SS_BF16 && a->dtypes[i] != SS_F16)
            return fail(SS_ERR_INVALID, "unknown dtype %d of tensor %lld", a->dtypes[i], (long long)i);
        if (a->numels[i] < 0) return fail(SS_ERR_INVALID, "negative size of tensor %lld", (long long)i);
        if (a->numels[i] > (int64_t(1) << 40) - total) return fail(SS_ERR_UNSUPPORTED, "more than 2^40 elements");
        total += a->numels[i];
        if (a->numels[i] == 0) continue;
        if (!a->grads[i] || !a->outs[i]) return fail(SS_ERR_INVALID, "tensor %lld is NULL", (long long)i);
        const size_t es = elem_size(a->dtypes[i]);
        if (!aligned(a->grads[i], es) || !aligned(a->outs[i], es))
            return fail(SS_ERR_INVALID, "tensor %lld is misaligned", (long long)i);
    }
    return ok();
}

// Two workgroups must not write, or write and read, one element.
static int check_clip_overlap(const ss_clip_grads_args* a) try {
    std::vector<ss::Span> ins, outs;
    outs.reserve(a->count);
    for (int64_t i = 0; i < a->count; ++i) {
        if (a->numels[i] == 0) continue;
        const uintptr_t bytes = uintptr_t(a->numels[i]) * elem_size(a->dtypes[i]);
        const uintptr_t in = reinterpret_cast<uintptr_t>(a->grads[i]), out = reinterpret_cast<uintptr_t>(a->outs[i]);
        outs.push_back({out, out + bytes, i});
        if (in != out) ins.push_back({in, in + bytes, i});
    }
    const int64_t at = ss::outputs_clash(ins, outs);
    if (at >= 0) return fail(SS_ERR_INVALID, "the output of tensor %lld lies over another tensor", (long long)at);
    return SS_OK;
} catch (const std::bad_alloc&) {
    return fail(SS_ERR_INVALID, "out of host memory");
}

int64_t ss_clip_grads_workspace_bytes(const ss_clip_grads_args* a) {
    return check_clip_grads(a) == SS_OK ? 16 + 8 * ss::clip_grads_chunks(a) : -1;
}

int ss_clip_grads(const ss_clip_grads_args* a, void* stream) {
    int rc = check_clip_grads(a);
    if (rc != SS_OK) return rc;
    if (!(a->max_norm >= 0.f) || !(a->eps >= 0.f)) return fail(SS_ERR_INVALID, "max_norm and eps must be >= 0");
    if (!a->norm || !aligned(a->norm, 4)) return fail(SS_ERR_INVALID, "norm is NULL or misaligned");
    rc = check_space(a->workspace, a->workspace_bytes, 16 + 8 * ss::clip_grads_chunks(a));
    if (rc == SS_OK) rc = check_clip_overlap(a);
    if (rc != SS_OK) return rc;
    const hipError_t e = ss::clip_grads_launch(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(SS_ERR_HIP, "gradient clipping launch failed: %s", hipGetErrorString(e));
    return ok();
}

}  // extern "C"

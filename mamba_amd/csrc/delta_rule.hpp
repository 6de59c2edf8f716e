// The gated delta rule: what its host and device sides share.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/mamba_ss.h"
#include "linear_attn.hpp"

namespace ss {

// Key columns of the kernels' tiles, and tokens a chunk.  terms: bf16 terms of a row's element (bf16 1, fp16 2, fp32 3).
// 64 tokens keep and read half the states of 32.  The tiles of fp16 keys above 128 do not fit the LDS at
// 64; fp32 rows are better off with two workgroups a compute unit at 32, at every size (us forward / with
// backward: 8 x 2048 tokens x 12 heads of 64 x 64 142 / 469 for 230 / 667, 1 x 16384 x 12 190 / 544 for 205 / 637, 2 x 500 x 6 41 / 100
// for 59 / 139); others are not: fp16 of 128 keys 258 / 883 for 263 / 805 (2 x 4096 x 16), bf16 of 256 316 / 1,162 for 300 / 1,108 (2 x 4096 x 8).
constexpr int dr_keys(int64_t k) { return k <= 64 ? 64 : k <= 128 ? 128 : 256; }
constexpr int dr_chunk(int64_t k, int terms) { return terms < 3 && dr_keys(k) * terms <= 256 ? 64 : 32; }
// Where two workgroups of a walk share a compute unit, each with half of its LDS.
constexpr int64_t kTwoTiles = 80 * 1024;
constexpr bool dr_two(int64_t k, int terms) { return dr_keys(k) * terms <= 128 || (dr_keys(k) <= 128 && terms == 3); }
constexpr int dr_round16(int64_t n) { return int((n + 15) / 16 * 16); }
constexpr int dr_round32(int64_t n) { return int((n + 31) / 32 * 32); }

// Rows of whole 16-byte vectors that do not overlap, a chunk's within 2^31 bytes: read and written through
// buffer resources, which end with the chunk's last row.  (8 x 2048 tokens x 24 heads of 64 x 64, bf16: a walk
// of 198 us with rows of any kind read behind branches, after each of which the compiler waits for all loads, was
// 170 without them; 157 by now.)
inline bool dr_whole(const LaRows& r, int64_t dim, int size) {
    return dim * size % 16 == 0 && r.l < (int64_t(1) << 22) && r.l >= dim;
}
// The rows of a tensor.  The token stride of a single token may be anything (0 or 1 of a permuted tensor, say): nothing
// is read or written by it, and the places past the row's only one lie past its end with a stride of the row's own width.
inline LaRows dr_rows(const void* p, int64_t b, int64_t l, int64_t h, int rep, int64_t dim, int64_t len) {
    return {p, b, len > 1 ? l : dim, h, rep};
}

// Per (batch, head) pair and chunk, what the kernels hand on (fp32):
//   plan    the chunk's gates and triangular inverse (delta_rule_chunk.hpp), dr_plan_bytes()
//   states  the state before the chunk, (Vp, Kp): a value column's keys side by side, in the order of state_key
//   err     the tokens' prediction errors, (Vp, chunk)
//   dstates the gradient of the state after the chunk;  derr: of the errors, as err
// Kp: keys rounded up to 32, Vp: value columns rounded up to 16, zero past the last.  Chunk n of pair bh is at n BH + bh,
// so that what the pairs' walks read and write at a time lies together, as the heads' rows of a token do (measured: no
// difference to a pair's chunks in a row).
constexpr int64_t dr_plan_bytes(int64_t chunk) { return chunk * 20 + 16 + chunk / 16 * (chunk / 16 + 1) / 2 * 1024; }
// Key at a place of a kept state: tile t of the walk's registers holds, in lane group g, keys 32 (t / 2) + 8 g + 4 (t % 2) ..
// (places 16 t + 4 g ..).
__host__ __device__ constexpr int state_key(int place) { return (place & ~31) + (place >> 2 & 3) * 8 + (place >> 4 & 1) * 4 + (place & 3); }

struct DrParams {
    int64_t B, L, H, BH;
    int K, V, Kp, Vp, rep, nch;               // rep: heads per group; nch: chunks of a row of L tokens
    float scale;
    int whole;                            // dr_whole of all rows (DrParams' q, k, v, o)
    LaRows q, k, v, o;                    // o: out, or the backward's dout
    const float* g; int64_t g_b, g_l, g_h;
    const float* beta; int64_t be_b, be_l, be_h;
    const int32_t* lens;
    const float* init; float* last;       // (B, H, K, V) before and after the walk (backward: dlast, dinitial), or null
    void* plan;
    float* states;                        // null: not kept
    float* err;
    float* dstates;
    float* derr;
    // a row's segments of seg_chunks chunks side by side (segs 1: the whole row)
    int segs, seg_chunks;
    int local;                            // the segments' own states from zero and what becomes of a state over one
    float* seg_add;                       // (B, H, segs, Vp, Kp): their states; then the states that they start from
    uint16_t* seg_mul;                    // (B, H, segs, 3, Kp, Kp): over a segment S becomes M S + its own; M in 3 bf16 terms, columns side by side
    // gradients
    void* dq; void* dk; void* dv;         // contiguous; dq and dk in fp32 per head with rep > 1
    float* dg; float* dbeta;              // (B, L, H)
};

// The chunks' triangular inverses; the walk over the chunks, forward or (rev) back; the gradients.
template <typename T> hipError_t dr_prep_launch(const DrParams& p, hipStream_t stream);
template <typename T> hipError_t dr_walk_launch(const DrParams& p, bool rev, hipStream_t stream);
template <typename T> hipError_t dr_grads_launch(const DrParams& p, hipStream_t stream);

}  // namespace ss

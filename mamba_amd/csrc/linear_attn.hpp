// Linear attention with a decay for each head: what its host and device
// sides share.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/mamba_ss.h"

namespace ss {

// rows of a (batch, len, head, dim) tensor: strides in elements, unit along dim
struct LaRows {
    const void* p;
    int64_t b, l, h;
    int rep;              // heads per row head (1, or LaParams' rep): head index is h / rep
};

// One pass of the recurrence
//   S_t = exp(g_t) S_{t-1} + k_t (vscale v_t)^T,   o_t = oscale q_t^T S_t
// in time order, or (rev) from the last token to the first with the decay
// after the token instead of before it:
//   R_t = C_t + k_t (vscale v_t)^T,  o_t = oscale q_t^T R_t,  C_{t-1} = exp(g_t) R_t.
// The forward is one pass; the backward is three, each a linear attention of
// its own:
//   dq = pass(q: dout, k: v, v: k), oscale scale, its state S^T
//   dk = rev (q: v, k: dout, v: q), vscale scale, its state dS^T
//   dv = rev (q: k, k: q, v: dout), vscale scale, its state dS
struct LaJob {
    LaRows q, k, v, o, x;             // x.p: rows for dot, or null
    int K, V;                         // dims of q, k and of v, o
    int rev, o_f32;                   // o in fp32 (partials of shared heads) instead of the rows' type
    float oscale, vscale;
    // states: fp32, element (i, j) of head (b, h) at ((b * H + h) * segs + s) * K * V + i * st_k + j * st_v
    int st_k, st_v;
    const float* in;                  // state before the first token of the walk (segs 1), or null: zero
    const float* carry;               // with it: state after each segment (in time order); the walk of segment s
                                      // starts from the one before it in walk order
    float* ends;                      // written: state after each segment in walk order, or null
    float* decays;                    // la_local: (B, H, segs) product of a segment's decays
    float* out_state;                 // written: state after the whole walk (segs 1), or null
    float* dot;                       // written: (V tiles, B, H, L) sums over the tile's columns of o * x, or null
};

struct LaParams {
    LaJob job[3];
    int njobs;
    int64_t B, L, H;
    const float* g;
    int64_t g_b, g_l, g_h;
    const int32_t* lens;
    int64_t seg_tokens;               // a multiple of 64: seg_chunks chunks of 32
    int segs, seg_chunks, rep;        // rep: heads per group
    int serial;                       // a workgroup walks a whole row (else a segment, from its carry)
    int tile, tiles;                  // value columns per workgroup, and tiles of the widest job
    int32_t* strong;                  // written by a backward's walk: (B, H, segs), whether the segment has a strong decay
};

// A log decay below it (2^-12) is a strong one: the decay's gradient is a sum that holds to
// about 2^-21 of terms without the decay's factor, which would leave it fewer than 9 bits.
constexpr float kLaStrong = -8.317766f;

// Most value columns a workgroup takes for q and k of up to k columns, in rows of
// so many bf16 terms (bf16 1, fp16 2, fp32 3): the state's share and the rows on their way about fill the
// 256 registers a lane that let two waves share a SIMD.  Spilled beyond them, of bf16 heads: 10
// registers by the 64 x 64 forward's walk (18 where tiles are not whole), 3 and 10 at 128 x 128, none and 6
// by the 64 x 64 backward's; of fp16 heads up to 19; fp32 rows of 128 take 512 registers and one wave.
constexpr int la_cols(int64_t k, int terms) { return k <= 64 ? (terms == 1 ? 64 : 32) : k <= 128 ? 32 : 16; }
// ... and those it takes of v columns: a multiple of 16, the shares even.
inline int la_tile(int64_t k, int64_t v, int terms) {
    const int64_t most = la_cols(k, terms) / 16, cols = (v + 15) / 16, n = (cols + most - 1) / most;
    return int((cols + n - 1) / n * 16);
}

// The segments' states from a zero start and their decays (job.ends,
// job.decays); and the walk itself (a backward's: what is computed in 3 terms
// for 16-bit rows too, and job.dot).
template <typename T> hipError_t la_local_launch(const LaParams& p, hipStream_t stream);
template <typename T> hipError_t la_walk_launch(const LaParams& p, bool backward, hipStream_t stream);

// dg of the tokens of one segment (see linear_attn.hip)
struct LaDgParams {
    int64_t B, L, H;
    const int32_t* lens;
    int64_t seg_tokens;
    int segs, qtiles, ktiles, K, V;
    const float* g;
    int64_t g_b, g_l, g_h;
    const float* dotq; const float* dotk;   // (tiles, B, H, L)
    const float* ends;                      // S after each segment (B, H, segs, K, V)
    const float* rends;                     // dS after each segment's walk (before it in time), same layout
    const float* dlast;                     // (B, H, K, V) or null
    float* dg;                              // (B, L, H), or null with part
    double* part;                           // (B, H, segs) sums over the segment's tokens, or null
    const int32_t* strong;                  // LaParams'
    // read only for those segments: the forward's rows, out's gradient, scale and the state before the first token
    LaRows q, k, v, dout;
    float scale;
    const float* first;                     // (B, H, K, V) or null
};

}  // namespace ss

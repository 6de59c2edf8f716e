// Linear attention with a decay for each head: the chunked form of LaJob's
// pass on the matrix cores (gfx950).
//
// A wave walks the chunks (32 tokens) of one segment, or of a whole row, for
// one (batch, head) and up to 16 NT value columns, and holds the state of its
// columns in registers.  Waves do not meet: a workgroup is one wave, and the 6 to
// 8 of a CU hide each other's loads.  (Four waves that shared a 64-token chunk and
// met at three barriers in it spent half their time waiting: 429 us for the
// training step below, 303 now.)
// With G the sum of the log2 decays from the chunk's start up to a token
// (itself included), the forward chunk is
//
//   P_ij = (q_i . k_j) 2^(G_i - G_j)  for j <= i, else 0
//   o_i  = P_i V + 2^G_i q_i S,    S <- 2^G_C S + sum_j 2^(G_C - G_j) k_j v_j^T
//
// and the reverse walk the same with G negated, j >= i, the factors
// 2^(G_C - G_i) at o and 2^G_j at k_j.  G is summed in 64 bits and kept as an
// integer I and a fraction F, so P's factor is 2^-F_j (a column), 2^F_i (a row)
// and an exact shift by I_i - I_j: however far the sums run, no factor loses
// bits, overflows by itself or needs an exponential for each pair.
//
// Products run on bf16 matrix instructions with 32-bit sums.  A row of type
// T is a sum of R bf16 terms, exactly: 1 (bf16), 2 (fp16, 11 bits) or 3
// (fp32); what is computed (P, S, the weighted rows of the state's update) is
// split into 2 or 3 terms (2^-18 off at most, or exact).  Of the products of terms
// those of the second with the third (2 terms: the second with the second) and beyond
// are left out: of 3 terms at most 2^-22 of a product, 2^-25 rms and of either sign,
// so a sum's share of them shrinks; of 2 terms 2^-16.  2 terms are enough where the
// result is rounded to 16 bits; states, and gradients that the decay's gradient is
// summed from, take 3.
//
// Layouts.  A 16x16x32 instruction takes 8 summands a lane (lane l: row or
// column l % 16, summands 8 (l / 16) ..) and returns 4 consecutive rows of a
// column.  Which summand a slot holds is free as long as both operands agree,
// and that keeps everything but k and v out of LDS:
//  - q and k come from global memory as operands, 8 elements of a row a lane;
//  - the state's rows are numbered so that the registers a lane holds are the 8
//    elements of q that it multiplies (state_row);
//  - P's registers are an operand as they are, in the token order of load_tokens;
//  - sums over tokens read k and v in that order through the transposing LDS
//    load, where 16 lanes read 4 rows of 16 elements and get a column of 4 each.
//
// Measured, 8 x 2048 tokens x 24 heads of 64 x 64, bf16 (the best and the median of ten
// launches): the forward's walk 56 and 61 us (225 MB: 4.0 TB/s, where plain reads of the
// same rows reach 6.5), the three passes of the backward together 159 and 173 us (about 1180 vector
// and 120 matrix instructions a chunk), a segment's states 27 and 29 us.  Vector instructions
// alone would take 19 of the forward's 56 us and 71 of the backward's 159.  With two
// waves a SIMD, the forward's waves issue for 37 % of their time, wait for their turn or an
// earlier instruction for 20 and for memory for 43; the backward's for 43, 31 and 26.  So it is bound by
// latency at that occupancy as much as by issue: splitting P, S and the weighted rows, and
// the decays.  With 2 terms in the backward as well it runs 5 % faster, and the decay's gradient is
// off by 7e-6 instead of 6e-7.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "bf16_terms.hpp"
#include "linear_attn.hpp"
#include "norm_rows.hpp"
#include "ss_device.hpp"

namespace ss {

namespace la {

constexpr float kDeepest = -300.f;        // log2 decays below it empty the state (fp32 ends at 2^-149)

// LDS of a wave: its accesses run in order; this keeps the compiler's order.
__device__ __forceinline__ void lds_in_order() { __asm__ volatile("" ::: "memory"); }

// The lane again, unknown to the compiler: what a rarely taken path derives from it
// is then computed there, and not once ahead of the loop and kept in registers.
__device__ __forceinline__ int late(int lane) {
    __asm__ volatile("" : "+v"(lane));
    return lane;
}

constexpr int C = 32;                     // tokens per chunk

// Column m of a wave's column tile n: as the state's rows, so that a lane's
// registers of two tiles are 8 neighbouring columns of the result (NT 1: 4).
template <int NT> constexpr __device__ __forceinline__ int value_col(int n, int m) {
    return NT == 1 ? m : 32 * (n >> 1) + 8 * (m >> 2) + 4 * (n & 1) + (m & 3);
}
// first column of the 4 that a lane reads of tile n for its group (load_tokens)
template <int NT> constexpr __device__ __forceinline__ int value_block(int n, int lane) {
    return NT == 1 ? 4 * (lane & 3) : 32 * (n >> 1) + 8 * (lane & 3) + 4 * (n & 1);
}
// whether the tile has columns below vdim
template <int NT> constexpr __device__ __forceinline__ bool tile_in(int n, int vdim) { return 32 * (n >> 1) < vdim; }

// 8-byte words at any element alignment; a lane's 4 or 8 columns of a result
typedef uint32_t words4_at2 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T, int W, bool WHOLE>
__device__ __forceinline__ void load_words(const char* p, uint2 (&w)[W], int cnt) {
    constexpr int COLS = 8 * W / int(sizeof(T));
    if (!WHOLE && cnt < COLS) {                             // (the first cnt elements, zero past them)
        uint32_t x[2 * W] = {};
#pragma unroll
        for (int e = 0; e < COLS - 1; ++e) {
            if (e < cnt) {
                if constexpr (sizeof(T) == 4) x[e] = *reinterpret_cast<const uint32_t*>(p + 4 * e);
                else x[e >> 1] |= uint32_t(*reinterpret_cast<const uint16_t*>(p + 2 * e)) << (16 * (e & 1));
            }
        }
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = make_uint2(x[2 * i], x[2 * i + 1]);
        return;
    }
    if constexpr (W == 1) {
        const half4_at2 x = *reinterpret_cast<const half4_at2*>(p);
        w[0] = make_uint2(x.x, x.y);
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 2) {
            const words4_at2 x = *reinterpret_cast<const words4_at2*>(p + 8 * i);
            w[i] = make_uint2(x.x, x.y);
            w[i + 1] = make_uint2(x.z, x.w);
        }
    }
}
template <typename T, int N, bool WHOLE>
__device__ __forceinline__ void store_cols(T* p, const float (&v)[N], int cnt) {
    using R = rowvec<T>;
    if constexpr (N < R::VE) {
        store4<T>(p, v, WHOLE ? 4 : cnt);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += R::VE) {
            float x[R::VE];
#pragma unroll
            for (int e = 0; e < R::VE; ++e) x[e] = v[i + e];
            R::store(p + i, x, WHOLE ? int(R::VE) : cnt - i);
        }
    }
}

// a vector of a row that may not exist, and (unless WHOLE) may end inside it
template <typename T, bool WHOLE>
__device__ __forceinline__ uint4 load_part(const T* p, bool in, int n) {
    if constexpr (WHOLE) {
        if (!in) return make_uint4(0u, 0u, 0u, 0u);
        const typename rowvec<T>::words w = *reinterpret_cast<const typename rowvec<T>::words*>(p);
        return make_uint4(w.x, w.y, w.z, w.w);
    } else {
        return rowvec<T>::load(p, in ? n : 0);
    }
}

// Whether kernels for other than whole tiles read and write rows of any width by
// vectors (load_any).  4 x 2048 tokens, 16 heads of 61 x 61, forward + backward: bf16 227 us
// with it and 284 without, fp16 257 and 306; but fp32 347 and 341, bf16 97 x 97 528 and 496.
template <typename T, int KP> constexpr bool kAny = sizeof(T) == 2 && KP <= 64;

// Elements col .. of a row of dim (at least a vector's) elements, zero past its end:
// the vector that ends with the row, shifted, where the one at col would cross it.
template <typename T>
__device__ __forceinline__ uint4 load_any(const char* row, int col, int dim) {
    using R = rowvec<T>;
    const int start = col < dim - R::VE ? col : dim - R::VE, cut = col - start;
    const typename R::words w = *reinterpret_cast<const typename R::words*>(row + start * int(sizeof(T)));
    uint32_t x[4] = {w.x, w.y, w.z, w.w};
    if (cut > 0) {
        const int half = int(sizeof(T)) == 2 ? 1 : 0, words = cut >> half;
        if (words & 2) { x[0] = x[2]; x[1] = x[3]; x[2] = x[3] = 0u; }
        if (words & 1) { x[0] = x[1]; x[1] = x[2]; x[2] = x[3]; x[3] = 0u; }
        if (half && (cut & 1)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (x[i] >> 16) | (i < 3 ? x[i < 3 ? i + 1 : 3] << 16 : 0u);
        }
        if (cut >= R::VE) x[0] = x[1] = x[2] = x[3] = 0u;
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// A chunk's rows of v on their way from global memory to LDS.
template <typename T, int WIDTH>
struct Stage {
    using R = rowvec<T>;
    static constexpr int PER_ROW = WIDTH / R::VE, N = C * PER_ROW / 64, STRIDE = WIDTH + 8, TERMS = kTerms<T>;
    static constexpr int TERM = C * STRIDE;                  // elements of one term's tile
    static constexpr int STEP = 64 / PER_ROW;                // rows between a lane's vectors
    uint4 v[N];

    // all rows of p (a row every `step` elements, near), whole
    __device__ __forceinline__ void load_all(const T* p, int64_t step, int lane) {
        const uint32_t off = (uint32_t(lane / PER_ROW) * uint32_t(step) + uint32_t(lane % PER_ROW * R::VE)) * uint32_t(sizeof(T));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const typename R::words w = *reinterpret_cast<const typename R::words*>(
                reinterpret_cast<const char*>(p + int64_t(i * STEP) * step) + off);
            v[i] = make_uint4(w.x, w.y, w.z, w.w);
        }
    }
    // all rows, of dim elements (at least a vector's)
    __device__ __forceinline__ void load_dim(const T* p, int64_t step, int dim, int lane) {
        const uint32_t off = uint32_t(lane / PER_ROW) * uint32_t(step) * uint32_t(sizeof(T));
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = load_any<T>(reinterpret_cast<const char*>(p + int64_t(i * STEP) * step) + off, lane % PER_ROW * R::VE, dim);
    }
    // the first `rows` rows of p, dim elements each; the others are zero
    template <bool WHOLE>
    __device__ __forceinline__ void load(const T* p, int64_t step, int rows, int dim, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = lane / PER_ROW + i * STEP, col = lane % PER_ROW * R::VE;
            v[i] = load_part<T, WHOLE>(p + int64_t(row) * step + col, row < rows, dim - col);
        }
    }
    // into the terms' tiles; CHECK: whether an element is infinite or NaN
    template <bool CHECK>
    __device__ __forceinline__ bool store(uint16_t* tile, int lane) const {
        typedef uint16_t h2 __attribute__((ext_vector_type(2)));
        h2 top = {0, 0};                                     // the largest exponents
        const auto look = [&](uint32_t w) {
            if constexpr (CHECK) top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, w & 0x7f807f80u));
        };
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint16_t* to = tile + (lane / PER_ROW + i * STEP) * STRIDE + lane % PER_ROW * R::VE;
            if constexpr (TERMS == 1) {
                look(v[i].x); look(v[i].y); look(v[i].z); look(v[i].w);
                *reinterpret_cast<uint4*>(to) = v[i];
            } else {
                float x[R::VE];
                R::unpack(v[i], x);
                uint32_t t[R::VE / 2][TERMS];
#pragma unroll
                for (int k = 0; k < R::VE / 2; ++k) {
                    split<TERMS>(x[2 * k], x[2 * k + 1], t[k]);
                    look(t[k][0]);
                }
#pragma unroll
                for (int n = 0; n < TERMS; ++n) {
                    if constexpr (R::VE == 8) *reinterpret_cast<uint4*>(to + n * TERM) = make_uint4(t[0][n], t[1][n], t[2][n], t[3][n]);
                    else *reinterpret_cast<uint2*>(to + n * TERM) = make_uint2(t[0][n], t[1][n]);
                }
            }
        }
        return top.x >= 0x7f80 || top.y >= 0x7f80;
    }
};
// whether a chunk of rows `step` elements apart lies within 32-bit byte offsets
__device__ __forceinline__ bool near(int64_t step) { return step < (int64_t(1) << 24); }

// A chunk's rows of q or k as operands: row 16 i + lane % 16, elements 32 kk + 8 (lane / 16) ..
template <typename T, int KP>
struct Rows {
    using R = rowvec<T>;
    static constexpr int W = int(sizeof(T)) / 2, STRIDE = KP + 8, TERMS = kTerms<T>, TERM = C * STRIDE;
    // Rows too wide to wait in registers (KP fp32 256: 128 a lane) are read where they
    // are used: only where they lie is kept.
    static constexpr bool STREAM = KP * int(sizeof(T)) > 512;
    uint4 v[2][STREAM ? 1 : KP / 32][W];
    const T* from;
    int64_t step;
    int rows, dim, lane;

    __device__ __forceinline__ void keep(const T* p, int64_t step_, int rows_, int dim_, int lane_) {
        from = p; step = step_; rows = rows_; dim = dim_; lane = lane_;
    }
    __device__ __forceinline__ void load_all(const T* p, int64_t step, int lane) {
        if constexpr (STREAM) return keep(p, step, C, KP, lane);
        const uint32_t off = (uint32_t(lane & 15) * uint32_t(step) + uint32_t(8 * (lane >> 4))) * uint32_t(sizeof(T));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int kk = 0; kk < (STREAM ? 0 : KP / 32); ++kk)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const typename R::words x = *reinterpret_cast<const typename R::words*>(
                        reinterpret_cast<const char*>(p + int64_t(16 * i) * step) + off + (32 * kk * int(sizeof(T)) + 16 * w));
                    v[i][kk][w] = make_uint4(x.x, x.y, x.z, x.w);
                }
    }
    __device__ __forceinline__ void load_dim(const T* p, int64_t step, int dim, int lane) {
        if constexpr (STREAM) return keep(p, step, C, dim, lane);
        const uint32_t off = uint32_t(lane & 15) * uint32_t(step) * uint32_t(sizeof(T));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int kk = 0; kk < (STREAM ? 0 : KP / 32); ++kk)
#pragma unroll
                for (int w = 0; w < W; ++w)
                    v[i][kk][w] = load_any<T>(reinterpret_cast<const char*>(p + int64_t(16 * i) * step) + off,
                                              32 * kk + 8 * (lane >> 4) + w * R::VE, dim);
    }
    template <bool WHOLE>
    __device__ __forceinline__ void load(const T* p, int64_t step, int rows, int dim, int lane) {
        if constexpr (STREAM) return keep(p, step, rows, dim, lane);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int kk = 0; kk < (STREAM ? 0 : KP / 32); ++kk)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const int row = 16 * i + (lane & 15), col = 32 * kk + 8 * (lane >> 4) + w * R::VE;
                    v[i][kk][w] = load_part<T, WHOLE>(p + int64_t(row) * step + col, row < rows, dim - col);
                }
    }
    __device__ __forceinline__ void terms(int i, int kk, u4 (&t)[TERMS]) const {
        uint4 x4[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if constexpr (STREAM) {
                const int row = 16 * i + (lane & 15), col = 32 * kk + 8 * (lane >> 4) + w * R::VE;
                x4[w] = R::load(from + int64_t(row) * step + col, row < rows ? dim - col : 0);
            } else {
                x4[w] = v[i][kk][w];
            }
        }
        if constexpr (TERMS == 1) {
            t[0] = u4{x4[0].x, x4[0].y, x4[0].z, x4[0].w};
        } else {
            float x[8];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                float y[R::VE];
                R::unpack(x4[w], y);
#pragma unroll
                for (int e = 0; e < R::VE; ++e) x[w * R::VE + e] = y[e];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t s[TERMS];
                split<TERMS>(x[2 * k], x[2 * k + 1], s);
#pragma unroll
                for (int n = 0; n < TERMS; ++n) t[n][k] = s[n];
            }
        }
    }
    __device__ __forceinline__ void store(uint16_t* tile, int lane) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int kk = 0; kk < KP / 32; ++kk) {
                u4 t[TERMS];
                terms(i, kk, t);
                if constexpr (STREAM) stage_end();
#pragma unroll
                for (int n = 0; n < TERMS; ++n)
                    *reinterpret_cast<u4*>(tile + n * TERM + (16 * i + (lane & 15)) * STRIDE + 32 * kk + 8 * (lane >> 4)) = t[n];
            }
    }
};

// The decays of two neighbouring chunks.  Lane t holds token t's log decay (0
// past the row's end).
struct __attribute__((aligned(16))) Decays {
    int I[64];             // integer part of H (G, or -G in reverse)
    float col[64];         // 2^-F, with the factor of v
    float row[64];         // 2^F, with the factor of o
    float in[64];          // the carried state's factor at a token, with the factor of o
    float upd[64];         // a token's factor in the state's update, with the factor of v
    float total[2];        // 2^G_C

    __device__ __forceinline__ static float exp2_of(double x) {
        const double i = floor(x);
        return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(float(x - i)), i < -2000.0 ? -2000 : i > 2000.0 ? 2000 : int(i));
    }
    __device__ __forceinline__ void fill(int lane, float g, bool rev, float vscale, float oscale) {
        double h = double(g) * 1.4426950408889634;
        h = h < kDeepest ? double(kDeepest) : h;          // (NaN stays)
        const int t = lane & 31;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            const double o = __shfl_up(h, m, 32);
            if (t >= m) h += o;
        }
        const double G = __shfl(h, 31, 32);
        const double H = rev ? -h : h, fl = floor(H);
        const float F = float(H - fl);
        I[lane] = int(fl);
        col[lane] = vscale * __builtin_amdgcn_exp2f(-F);
        row[lane] = oscale * __builtin_amdgcn_exp2f(F);
        in[lane] = oscale * exp2_of(rev ? H + G : H);
        upd[lane] = vscale * exp2_of(rev ? -H : G - H);
        if (t == 0) total[lane >> 5] = exp2_of(G);
    }
};

__device__ __forceinline__ int64_t tokens_of(const int32_t* lens, int64_t b, int64_t L) {
    if (!lens) return L;
    const int64_t n = lens[b];
    return n < 0 ? 0 : n < L ? n : L;
}

// S <- total S + sum over the chunk's tokens of k_t (w_t v_t)^T.  kt: k's tile;
// vf: v's columns; half: the chunk of the two in dec.
template <typename T, int KP, int NT, bool WHOLE>
__device__ __forceinline__ void update_state(f4 (&S)[KP / 16][NT], const uint16_t* kt, const u4 (&vf)[NT][kTerms<T>],
                                             const Decays& dec, int half, int kdim, int vdim, int lane) {
    constexpr int R = kTerms<T>;
    using SK = Rows<T, KP>;
    const float tot = dec.total[half];
    const f4 u0 = *reinterpret_cast<const f4*>(dec.upd + 32 * half + 4 * (lane >> 4));
    const f4 u1 = *reinterpret_cast<const f4*>(dec.upd + 32 * half + 16 + 4 * (lane >> 4));
    const float u[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
    for (int d = 0; d < KP / 16; ++d)
#pragma unroll
        for (int n = 0; n < NT; ++n) S[d][n] *= tot;
    // v's columns n, weighted, in 3 terms
    const auto weighted = [&](int n, u4 (&bv)[3]) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float x0 = lo_half(vf[n][R - 1][w]), x1 = hi_half(vf[n][R - 1][w]);
#pragma unroll
            for (int r = R - 2; r >= 0; --r) {                // small terms first: the sum is exact
                x0 += lo_half(vf[n][r][w]);
                x1 += hi_half(vf[n][r][w]);
            }
            uint32_t t[3];
            split<3, R == 1>(x0 * u[2 * w], x1 * u[2 * w + 1], t);
#pragma unroll
            for (int i = 0; i < 3; ++i) bv[i][w] = t[i];
        }
    };
    const auto rows = [&](int d, u4 (&kf)[R]) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            kf[r] = load_tokens<SK::STRIDE>(kt + r * SK::TERM, 32 * (d >> 1) + 8 * (lane & 3) + 4 * (d & 1), lane);
    };
    // (whichever of the two takes fewer registers is held)
    if constexpr (KP / 16 * R <= 3 * NT) {
        u4 kf[KP / 16][R];
#pragma unroll
        for (int d = 0; d < KP / 16; ++d) rows(d, kf[d]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (!WHOLE && !tile_in<NT>(n, vdim)) continue;
            u4 bv[3];
            weighted(n, bv);
            f4* to[KP / 16];
#pragma unroll
            for (int d = 0; d < KP / 16; ++d) to[d] = &S[d][n];
            mfma_terms<KP / 16, 1, 0, R, 3, 2>(kf, &bv, to);
            stage_end();
        }
    } else {
        u4 bv[NT][3];
#pragma unroll
        for (int n = 0; n < NT; ++n) weighted(n, bv[n]);
#pragma unroll
        for (int d = 0; d < KP / 16; ++d) {
            if (!WHOLE && 32 * (d >> 1) >= kdim) continue;
            u4 kf[R];
            rows(d, kf);
            f4* to[NT];                                       // (tiles past vdim: v's columns are zero)
#pragma unroll
            for (int n = 0; n < NT; ++n) to[n] = &S[d][n];
            mfma_terms<NT, 0, 1, R, 3, 2>(&kf, bv, to);
            stage_end();
        }
    }
}

// The launch's arguments where they lie: an index into their jobs is then a
// scalar load (an index into the by-value parameter copies it to scratch).
typedef __attribute__((address_space(4))) const LaParams Params;
typedef __attribute__((address_space(4))) const LaJob Job;
__device__ __forceinline__ Params& params() { return *(Params*)__builtin_amdgcn_kernarg_segment_ptr(); }

// Workgroup order: the jobs of a segment (they read the same rows), then its column
// tiles, side by side on one XCD.
// (32-bit divisions: a launch holds fewer than 2^26 workgroups of 64 threads, and the
// 64-bit ones cost a short walk a tenth of its time.)
struct Place { int job, tile, seg; uint32_t bh, b, h, shared; };      // (bh past the last one: nothing to do)
__device__ __forceinline__ Place place(Params& p, uint32_t segs) {
    uint32_t id = uint32_t(xcd_block_id());
    Place r;
    const uint32_t jobs = p.njobs, tiles = p.tiles, H = uint32_t(p.H);
    r.job = int(id % jobs);
    id /= jobs;
    r.tile = tiles > 1 ? int(id % tiles) : 0;
    if (tiles > 1) id /= tiles;
    r.h = id % H;
    id /= H;
    r.seg = int(id % segs);
    r.b = id / segs;
    r.bh = r.b * H + r.h;
    r.shared = p.rep > 1 ? r.h / uint32_t(p.rep) : r.h;      // the group whose q and k head h reads
    return r;
}
template <typename T, typename Row>
__device__ __forceinline__ const T* rows_of_head(Row& r, const Place& at) {
    return static_cast<const T*>(r.p) + int64_t(at.b) * r.b + int64_t(r.rep > 1 ? at.shared : at.h) * r.h;
}

// The tokens of a workgroup and what it reads of them, in the walk's order.
template <typename T, int KP, int NT, bool Q, bool WHOLE>
struct Walk {
    Params& p;
    Job& J;
    int64_t s0, s1, end;              // tokens: the span, and where the row's own end in it
    const T* qp; const T* kp; const T* vp; const float* gp;
    int chunks, vdim, lane;
    bool whole, rev;
    Rows<T, KP> q, k;
    Stage<T, 16 * NT> v;

    __device__ __forceinline__ Walk(Params& p_, Job& J_, const Place& at, int64_t span, int lane_) : p(p_), J(J_), lane(lane_) {
        s0 = at.seg * span;
        s1 = s0 + span < p.L ? s0 + span : p.L;
        const int64_t len = tokens_of(p.lens, at.b, p.L);
        end = len < s1 ? len : s1;
        chunks = int((s1 - s0 + C - 1) / C);
        const int n0 = at.tile * p.tile;
        vdim = J.V - n0 < p.tile ? J.V - n0 : p.tile;
        rev = J.rev;
        if (Q) qp = rows_of_head<T>(J.q, at);
        kp = rows_of_head<T>(J.k, at);
        vp = rows_of_head<T>(J.v, at) + n0;
        gp = p.g + int64_t(at.b) * p.g_b + int64_t(at.h) * p.g_h;
        whole = WHOLE || ((kAny<T, KP> ? J.K >= rowvec<T>::VE && vdim >= rowvec<T>::VE : J.K == KP && vdim == 16 * NT) && (!Q || near(J.q.l)) && near(J.k.l) && near(J.v.l));
    }
    __device__ __forceinline__ int chunk(int i) const { return rev ? chunks - 1 - i : i; }
    __device__ __forceinline__ void fetch(int i) {
        const int64_t t0 = s0 + int64_t(chunk(i)) * C;
        if ((WHOLE || (!kAny<T, KP> && whole)) && t0 + C <= end) {
            if (Q) q.load_all(qp + t0 * J.q.l, J.q.l, lane);
            k.load_all(kp + t0 * J.k.l, J.k.l, lane);
            v.load_all(vp + t0 * J.v.l, J.v.l, lane);
        } else if (!WHOLE && kAny<T, KP> && whole && t0 + C <= end) {
            if (Q) q.load_dim(qp + t0 * J.q.l, J.q.l, J.K, lane);
            k.load_dim(kp + t0 * J.k.l, J.k.l, J.K, lane);
            v.load_dim(vp + t0 * J.v.l, J.v.l, vdim, lane);
        } else {
            const int rows = t0 + C <= end ? C : t0 < end ? int(end - t0) : 0;
            const int l = late(lane);
            if (Q) q.template load<WHOLE>(qp + t0 * J.q.l, J.q.l, rows, J.K, l);
            k.template load<WHOLE>(kp + t0 * J.k.l, J.k.l, rows, J.K, l);
            v.template load<WHOLE>(vp + t0 * J.v.l, J.v.l, rows, vdim, l);
        }
    }
    // the log decays of the two chunks that `pair` names, a token a lane
    __device__ __forceinline__ float decay(int pair) const {
        const int64_t t = s0 + int64_t(pair) * 64 + lane;
        return t < end ? gp[t * p.g_l] : 0.f;
    }
};

// the element (register r of tile d, column tile n) of the state, and whether it exists
template <int KP, int NT, bool WHOLE, typename F>
__device__ __forceinline__ void each_state(f4 (&S)[KP / 16][NT], Job& J, int n0, int vdim, int lane, F&& f) {
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int col = value_col<NT>(n, c);
#pragma unroll
        for (int d = 0; d < KP / 16; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = state_row(d, g, r);
                S[d][n][r] = f(S[d][n][r], WHOLE || (row < J.K && col < vdim), uint32_t(row * J.st_k + (n0 + col) * J.st_v));
            }
    }
}
template <int KP, int NT, bool WHOLE>
__device__ __forceinline__ void write_state(f4 (&S)[KP / 16][NT], Job& J, int n0, int vdim, int lane, float* to) {
    each_state<KP, NT, WHOLE>(S, J, n0, vdim, late(lane), [&](float s, bool in, uint32_t i) __attribute__((always_inline)) {
        if (in) to[i] = s;
        return s;
    });
}

template <typename T, int KP, int NT>
struct Tiles {
    __attribute__((aligned(16))) uint16_t k[kTerms<T> * Rows<T, KP>::TERM];
    __attribute__((aligned(16))) uint16_t v[kTerms<T> * Stage<T, 16 * NT>::TERM];
    Decays dec;
};

// ------------------------------------------------------- state of a segment --
// Each segment's state from a zero start, and its decay.
template <typename T, int KP, int NT, bool WHOLE, bool rev>
__device__ __forceinline__ void local_rows(Params& p, Job& J, const Place& at, Tiles<T, KP, NT>& m) {
    constexpr int R = kTerms<T>;
    using SV = Stage<T, 16 * NT>;
    const int n0 = at.tile * p.tile, lane = int(threadIdx.x);
    const int64_t bh = at.bh;
    Walk<T, KP, NT, false, WHOLE> w(p, J, at, p.seg_tokens, lane);
    f4 S[KP / 16][NT];
    each_state<KP, NT, WHOLE>(S, J, n0, w.vdim, lane, [](float, bool, uint32_t) __attribute__((always_inline)) { return 0.f; });
    float decay = 1.f;
    int pair = -1;
    w.fetch(0);
    float g = w.decay(w.chunk(0) >> 1);
    for (int i = 0; i < w.chunks; ++i) {
        const int ch = w.chunk(i), half = ch & 1;
        lds_in_order();
        w.k.store(m.k, lane);
        (void)w.v.template store<false>(m.v, lane);
        if (i + 1 < w.chunks) w.fetch(i + 1);
        if (pair != ch >> 1) {
            pair = ch >> 1;
            m.dec.fill(lane, g, rev, J.vscale, 1.f);
            const int next = pair + (rev ? -1 : 1);
            if (next >= 0) g = w.decay(next);
            lds_in_order();
            decay *= m.dec.total[0] * m.dec.total[1];
        }
        lds_in_order();
        u4 vf[NT][R];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < R; ++r) vf[n][r] = load_tokens<SV::STRIDE>(m.v + r * SV::TERM, value_block<NT>(n, lane), lane);
        update_state<T, KP, NT, WHOLE>(S, m.k, vf, m.dec, half, J.K, w.vdim, lane);
    }
    write_state<KP, NT, WHOLE>(S, J, n0, w.vdim, lane, J.ends + (bh * p.segs + at.seg) * int64_t(J.K) * J.V);
    if (lane == 0 && at.tile == 0) J.decays[bh * p.segs + at.seg] = decay;
}

template <typename T, int KP, int NT, bool WHOLE>
__global__ __launch_bounds__(64, 2) void la_local(const LaParams) {
    Params& p = params();
    __shared__ Tiles<T, KP, NT> m;
    const Place at = place(p, p.segs);
    Job& J = p.job[at.job];
    if (at.tile * p.tile >= J.V || at.bh >= uint32_t(p.B * p.H)) return;
    if (J.rev) local_rows<T, KP, NT, WHOLE, true>(p, J, at, m);
    else local_rows<T, KP, NT, WHOLE, false>(p, J, at, m);
}

// ----------------------------------------------------------------- the walk --
// DOT: a pass of the backward (J.dot may be asked for)
template <typename T, int KP, int NT, int N, bool DOT, bool WHOLE>
__device__ __forceinline__ void walk_rows(Params& p, Job& J, const Place& at, Tiles<T, KP, NT>& m, int* bad_col, bool rev) {
    constexpr int R = kTerms<T>, kMax = N == 2 ? 1 : 2;
    using SV = Stage<T, 16 * NT>;
    const int n0 = at.tile * p.tile, lane = int(threadIdx.x), c = lane & 15, g = lane >> 4;
    const int64_t bh = at.bh, KV = int64_t(J.K) * J.V;
    Walk<T, KP, NT, true, WHOLE> w(p, J, at, p.serial ? p.L : p.seg_tokens, lane);
    const int vdim = w.vdim;
    const T* xp = DOT && J.dot ? rows_of_head<T>(J.x, at) + n0 : nullptr;
    const int64_t op = int64_t(at.b) * J.o.b + int64_t(at.h) * J.o.h + n0;
    const bool near_o = WHOLE || ((kAny<T, KP> || vdim == 16 * NT) && near(J.o.l) && near(J.x.l));

    // the state before the walk's first token
    const float* from = J.in ? J.in + bh * KV : nullptr;
    if (!p.serial) {
        const int before = rev ? at.seg + 1 : at.seg - 1;
        if (before >= 0 && before < p.segs) from = J.carry + (bh * p.segs + before) * KV;
    }
    f4 S[KP / 16][NT];
    if (from) each_state<KP, NT, WHOLE>(S, J, n0, vdim, lane, [&](float, bool in, uint32_t i) __attribute__((always_inline)) { return in ? from[i] : 0.f; });
    else each_state<KP, NT, WHOLE>(S, J, n0, vdim, lane, [](float, bool, uint32_t) __attribute__((always_inline)) { return 0.f; });

    int pair = -1;
    bool strong = false;                                     // (a lane's tokens, of the segment so far)
    float decay = 0.f;
    if (w.chunks > 0) {
        w.fetch(0);
        decay = w.decay(w.chunk(0) >> 1);
    }
    for (int ci = 0; ci < w.chunks; ++ci) {
        const int ch = w.chunk(ci), half = ch & 1;
        const int64_t t0 = w.s0 + int64_t(ch) * C;
        const bool last = ci + 1 == w.chunks;
        lds_in_order();
        w.k.store(m.k, lane);
        // A sum over tokens multiplies every v, by P's zeros too: infinities and
        // NaN of v are taken out of the tile here and put into the results from
        // their token on.
        const bool bad = __ballot(w.v.template store<true>(m.v, lane)) != 0;
        lds_in_order();
        if (bad && lane < 16 * NT) {
            int first = rev ? -1 : C;
            for (int i = 0; i < C; ++i) {
                const int row = rev ? i : C - 1 - i;
                if ((m.v[row * SV::STRIDE + lane] & 0x7f80u) == 0x7f80u) {
                    first = row;
                    for (int r = 0; r < R; ++r) m.v[r * SV::TERM + row * SV::STRIDE + lane] = 0;
                }
            }
            bad_col[lane] = first;
        }
        if (pair != ch >> 1) {
            pair = ch >> 1;
            m.dec.fill(lane, decay, rev, J.vscale, J.oscale);
            if (DOT) strong |= decay < kLaStrong;
            const int next = pair + (rev ? -1 : 1);
            if (next >= 0) decay = w.decay(next);
        }
        lds_in_order();
        const int d0 = 32 * half;

        // P^T's causal tiles (tokens j, rows i), and o^T = S^T q
        f4 o[2][NT], P[3];                                   // P: (0, 0), (0, 1) or in reverse (1, 0), (1, 1)
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
            for (int n = 0; n < NT; ++n) o[it][n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 3; ++i) P[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KP / 32; ++kk) {
            if (!WHOLE && 32 * kk >= J.K) continue;
            u4 qf[2][R], kf[2][R];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                w.q.terms(i, kk, qf[i]);
                w.k.terms(i, kk, kf[i]);
            }
            {
                f4* const diagonal[2] = {&P[0], &P[2]};
                f4* const beside[1] = {&P[1]};
                mfma_terms<2, 1, 1, R, R, 2>(kf, qf, diagonal);
                if (rev) mfma_terms<1, 0, 0, R, R, 2>(kf + 1, qf, beside);
                else mfma_terms<1, 0, 0, R, R, 2>(kf, qf + 1, beside);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (!WHOLE && !tile_in<NT>(n, vdim)) continue;
                u4 sf[N];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t t[N];
                    const f4& s = S[2 * kk + (x >> 1)][n];
                    split<N, R == 1>(s[2 * (x & 1)], s[2 * (x & 1) + 1], t);
#pragma unroll
                    for (int i = 0; i < N; ++i) sf[i][x] = t[i];
                }
                f4* const to[2] = {&o[0][n], &o[1][n]};
                mfma_terms<2, 0, 1, N, R, kMax>(&sf, qf, to);
            }
            stage_end();
        }
        // 8 columns (NT 1: 4) a lane: of the result, and of x for dot
        constexpr int COLS = NT == 1 ? 4 : 8, VECS = (16 * NT + 4 * COLS - 1) / (4 * COLS);
        constexpr int WORDS = COLS * int(sizeof(T)) / 8;       // 8-byte words of a row a vector
        uint2 xv[2][VECS][WORDS];
        const bool whole_o = near_o && t0 + C <= w.end && !bad;
        if (DOT && J.dot && whole_o) {
            const uint32_t off = (uint32_t(c) * uint32_t(J.x.l) + uint32_t(COLS * g)) * uint32_t(sizeof(T));
#pragma unroll
            for (int it = 0; it < 2; ++it)
#pragma unroll
                for (int n = 0; n < VECS; ++n)
                    load_words<T, WORDS, WHOLE || !kAny<T, KP>>(reinterpret_cast<const char*>(xp + (t0 + 16 * it) * J.x.l) + off + 4 * COLS * n * int(sizeof(T)), xv[it][n],
                                                vdim - COLS * (4 * n + g));
        }
        u4 vf[NT][R];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < R; ++r) vf[n][r] = load_tokens<SV::STRIDE>(m.v + r * SV::TERM, value_block<NT>(n, lane), lane);

        if (!DOT) stage_end();
        // P's decays and split, and o^T <- 2^G o^T + V^T P^T
        typedef int i4 __attribute__((ext_vector_type(4)));
        i4 Ij[2];
        f4 cj[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            Ij[j] = *reinterpret_cast<const i4*>(m.dec.I + d0 + 16 * j + 4 * g);
            cj[j] = *reinterpret_cast<const f4*>(m.dec.col + d0 + 16 * j + 4 * g);
        }
#pragma unroll
        for (int it = 0; it < 2; ++it) {
            const int Ii = m.dec.I[d0 + 16 * it + c];
            const float row = m.dec.row[d0 + 16 * it + c];
            u4 pf[N];
#pragma unroll
            for (int t = 0; t < N; ++t) pf[t] = u4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (it == j || (rev ? j > it : j < it)) {
                    f4 v = (it == j ? P[2 * it] : P[1]) * (cj[j] * row);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        v[r] = __builtin_amdgcn_ldexpf(v[r], Ii - Ij[j][r]);
                        if (it == j) v[r] = (rev ? 4 * g + r < c : 4 * g + r > c) ? 0.f : v[r];
                    }
                    uint32_t lo[N], hi[N];
                    split<N, R == 1>(v[0], v[1], lo);
                    split<N, R == 1>(v[2], v[3], hi);
#pragma unroll
                    for (int t = 0; t < N; ++t) {
                        pf[t][2 * j] = lo[t];
                        pf[t][2 * j + 1] = hi[t];
                    }
                }
            }
            const float carried = m.dec.in[d0 + 16 * it + c];
            f4* to[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                o[it][n] *= carried;
                to[n] = &o[it][n];
            }
            mfma_terms<NT, 1, 0, R, N, kMax>(vf, &pf, to);
        }

        float dot[2] = {0.f, 0.f};
        if (whole_o) {
            const uint32_t row = uint32_t(c) * uint32_t(J.o.l) + uint32_t(COLS * g);
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const int64_t first = op + (t0 + 16 * it) * J.o.l;
#pragma unroll
                for (int n = 0; n < VECS; ++n) {
                    float v[COLS];
#pragma unroll
                    for (int e = 0; e < COLS; ++e) v[e] = o[it][COLS / 4 * n + e / 4][e & 3];
                    const int cnt = vdim - COLS * (4 * n + g);
                    if (DOT && J.o_f32) store_cols<float, COLS, WHOLE || !kAny<T, KP>>(static_cast<float*>(const_cast<void*>(J.o.p)) + first + (row + 4 * COLS * n), v, cnt);
                    else store_cols<T, COLS, WHOLE || !kAny<T, KP>>(static_cast<T*>(const_cast<void*>(J.o.p)) + first + (row + 4 * COLS * n), v, cnt);
                    if (DOT && J.dot) {
#pragma unroll
                        for (int e = 0; e < COLS; e += 4) {
                            float x[4];
                            load4<T>(reinterpret_cast<const T*>(&xv[it][n][e * int(sizeof(T)) / 8]), x, 4);
#pragma unroll
                            for (int r = 0; r < 4; ++r) dot[it] = __builtin_fmaf(v[e + r], x[r], dot[it]);
                        }
                    }
                }
            }
        } else {
            const int l = late(lane), c = l & 15, g = l >> 4;
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const int i = 16 * it + c;
                const int64_t t = t0 + i;
                const bool live = t < w.end;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int col = value_col<NT>(n, 4 * g), cnt = t < w.s1 ? vdim - col : 0;
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        v[r] = live ? o[it][n][r] : 0.f;
                        if (bad && live && (rev ? i <= bad_col[col + r] : i >= bad_col[col + r])) v[r] = __builtin_nanf("");
                    }
                    if (cnt > 0) {
                        const int64_t to = op + t * J.o.l + col;
                        if (DOT && J.o_f32) store4<float>(static_cast<float*>(const_cast<void*>(J.o.p)) + to, v, cnt);
                        else store4<T>(static_cast<T*>(const_cast<void*>(J.o.p)) + to, v, cnt);
                        if (DOT && J.dot && live) {
                            float x[4];
                            load4<T>(xp + t * J.x.l + col, x, cnt);
#pragma unroll
                            for (int r = 0; r < 4; ++r) dot[it] = __builtin_fmaf(r < cnt ? v[r] : 0.f, x[r], dot[it]);
                        }
                    }
                }
            }
        }
        if (DOT && J.dot) {
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                // over the lanes of the token's other columns: g = 0 .. 3
                auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(dot[it]), __float_as_uint(dot[it]), false, false);
                float d = __uint_as_float(s[0]) + __uint_as_float(s[1]);
                s = __builtin_amdgcn_permlane16_swap(__float_as_uint(d), __float_as_uint(d), false, false);
                d = __uint_as_float(s[0]) + __uint_as_float(s[1]);
                const int64_t t = t0 + 16 * it + c;
                if (g == 0 && t < w.s1) J.dot[(int64_t(at.tile) * p.B * p.H + bh) * p.L + t] = d;
            }
        }
        // (the next rows are requested only here: in flight any earlier, they and
        // the results together would not fit the registers)
        if (!last) w.fetch(ci + 1);
        stage_end();
        if (!last || J.ends || J.out_state) update_state<T, KP, NT, WHOLE>(S, m.k, vf, m.dec, half, J.K, vdim, lane);
        if (bad) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int first = bad_col[value_col<NT>(n, c)];
                if (first >= 0 && first < C) {
#pragma unroll
                    for (int d = 0; d < KP / 16; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[d][n][r] = __builtin_nanf("");
                }
            }
        }
        // (a whole row's walk: the state at the end of each segment)
        const uint32_t seg = uint32_t(ch) / uint32_t(p.seg_chunks), next = uint32_t(rev ? ch - 1 : ch + 1) / uint32_t(p.seg_chunks);
        if (DOT && at.job == 0 && at.tile == 0 && (last || next != seg)) {
            const bool any = __ballot(strong) != 0;
            if (lane == 0) p.strong[bh * p.segs + (p.serial ? seg : uint32_t(at.seg))] = any;
            strong = false;
        }
        if (J.ends && (last || next != seg)) write_state<KP, NT, WHOLE>(S, J, n0, vdim, lane, J.ends + (bh * p.segs + seg) * KV);
    }
    if (w.chunks == 0 && J.ends) write_state<KP, NT, WHOLE>(S, J, n0, vdim, lane, J.ends + bh * p.segs * KV);
    if (J.out_state) write_state<KP, NT, WHOLE>(S, J, n0, vdim, lane, J.out_state + bh * KV);
}

template <typename T, int KP, int NT, int N, bool DOT, bool WHOLE>
__global__ __launch_bounds__(64, KP <= 128 ? 2 : 1) void la_walk(const LaParams) {
    Params& p = params();
    __shared__ Tiles<T, KP, NT> m;
    __shared__ int bad_col[16 * NT];
    const Place at = place(p, p.serial ? 1 : p.segs);
    Job& J = p.job[at.job];
    if (at.tile * p.tile >= J.V || at.bh >= uint32_t(p.B * p.H)) return;
    walk_rows<T, KP, NT, N, DOT, WHOLE>(p, J, at, m, bad_col, J.rev);
}

}  // namespace la

// f(KP, NT): the padded width of q and k, and the 16-column tiles of a wave
template <typename T, typename F>
hipError_t la_for_dims(const LaParams& p, F&& f) {
    int k = 0;
    for (int j = 0; j < p.njobs; ++j) k = p.job[j].K > k ? p.job[j].K : k;
    const auto with = [&](auto kp) {
        return f(kp, std::integral_constant<int, la_cols(decltype(kp)::value, la::kTerms<T>) / 16>{});
    };
    if (k <= 32) return with(std::integral_constant<int, 32>{});
    if (k <= 64) return with(std::integral_constant<int, 64>{});
    if (k <= 128) return with(std::integral_constant<int, 128>{});
    return with(std::integral_constant<int, 256>{});
}
// (a multiple of the XCDs, so that a segment's workgroups share one)
inline dim3 la_grid(const LaParams& p, int segs) {
    const int64_t n = p.B * p.H * segs * p.tiles * p.njobs;
    return dim3(unsigned((n + kXcds - 1) / kXcds * kXcds));
}

// every tile of every job is full, and rows are near
template <int KP, int NT>
bool la_whole(const LaParams& p) {
    const auto near = [](const LaRows& r) { return r.l < (int64_t(1) << 24); };
    for (int j = 0; j < p.njobs; ++j) {
        const LaJob& J = p.job[j];
        if (J.K != KP || p.tile != 16 * NT || J.V % p.tile != 0 || !near(J.q) || !near(J.k) || !near(J.v) || !near(J.o) || !near(J.x)) return false;
    }
    return true;
}
template <typename T>
hipError_t la_local_launch(const LaParams& p, hipStream_t stream) {
    return la_for_dims<T>(p, [&](auto kp, auto nt) {
        constexpr int KP = decltype(kp)::value, NT = decltype(nt)::value;
        const dim3 grid = la_grid(p, p.segs);
        if (la_whole<KP, NT>(p)) hipLaunchKernelGGL((la::la_local<T, KP, NT, true>), grid, dim3(64), 0, stream, p);
        else hipLaunchKernelGGL((la::la_local<T, KP, NT, false>), grid, dim3(64), 0, stream, p);
        return hipGetLastError();
    });
}
template <typename T>
hipError_t la_walk_launch(const LaParams& p, bool backward, hipStream_t stream) {
    return la_for_dims<T>(p, [&](auto kp, auto nt) {
        constexpr int KP = decltype(kp)::value, NT = decltype(nt)::value;
        const dim3 grid = la_grid(p, p.serial ? 1 : p.segs);
        const auto run = [&](auto n, auto dot) {
            constexpr int N = decltype(n)::value;
            constexpr bool DOT = decltype(dot)::value;
            if (la_whole<KP, NT>(p)) hipLaunchKernelGGL((la::la_walk<T, KP, NT, N, DOT, true>), grid, dim3(64), 0, stream, p);
            else hipLaunchKernelGGL((la::la_walk<T, KP, NT, N, DOT, false>), grid, dim3(64), 0, stream, p);
            return hipGetLastError();
        };
        constexpr int kForward = sizeof(T) == 2 ? 2 : 3;
        return backward ? run(std::integral_constant<int, 3>{}, std::true_type{}) : run(std::integral_constant<int, kForward>{}, std::false_type{});
    });
}

}  // namespace ss

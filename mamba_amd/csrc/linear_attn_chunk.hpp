// Linear attention with a decay for each head: the chunked form of LaJob's
// pass on the matrix cores (gfx950).
//
// A workgroup walks the chunks (C tokens) of one segment, or of a whole row,
// for one (batch, head) and 64 NT value columns; its 4 waves share the
// columns in tiles of 16 and hold the state of their tiles in registers.
// With G the sum of the log2 decays from the chunk's start up to a token
// (itself included), the forward chunk is
//
//   P_ij = (q_i . k_j) 2^(G_i - G_j)  for j <= i, else 0
//   o_i  = P_i V + 2^G_i q_i S,    S <- 2^G_C S + sum_j 2^(G_C - G_j) k_j v_j^T
//
// and the reverse walk the same with G negated, j >= i, the factors
// 2^(G_C - G_i) at o and 2^G_j at k_j.  G is summed in 64 bits and kept as an
// integer I and a fraction F, so P's factor is 2^-F_j (a column), 2^F_i (a row,
// applied to o at the end) and an exact shift by I_i - I_j: however far the sums
// run, no factor loses bits, overflows by itself or needs an exponential for
// each pair.
//
// Products run on bf16 matrix instructions with 32-bit sums.  A row of type
// T is a sum of R bf16 terms, exactly: 1 (bf16), 2 (fp16, 11 bits) or 3
// (fp32); what is computed (P, S, the weighted rows of the state's update) is
// split into 2 or 3 terms, and of the products of terms those below 2^-24
// (2 terms: 2^-16) are left out.  2 terms are enough where the result is rounded
// to 16 bits; states, and gradients that the decay's gradient is summed from,
// take 3.
//
// Layouts.  A 16x16x32 instruction takes 8 consecutive summands a lane (lane
// l: row or column l % 16, summands 8 (l / 16) ..) and returns 4 consecutive
// rows of a column.  q and k lie in LDS as rows, so q k^T reads both with
// 16-byte loads; sums over tokens (P V, the state's update) read v and k through
// the transposing LDS load; the state's registers are used as they are, with
// q read in the same order of summands.  P crosses LDS between the waves.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "linear_attn.hpp"
#include "norm_rows.hpp"
#include "ss_device.hpp"

namespace ss {

namespace la {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

constexpr float kDeepest = -300.f;        // log2 decays below it empty the state (fp32 ends at 2^-149)

template <typename T> constexpr int kTerms = sizeof(T) == 4 ? 3 : __is_same(T, bf16_t) ? 1 : 2;

__device__ __forceinline__ f4 mfma(const u4& a, const u4& b, const f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// x0, x1 as N bf16 terms each, packed (x0 low): the first N - 1 by cutting
// bits off, so what is left over is exact; the last of 2 rounded, of 3 exact
template <int N>
__device__ __forceinline__ void split(float x0, float x1, uint32_t (&t)[N]) {
    const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
    t[0] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    if constexpr (N > 1) {
        const float r0 = x0 - __uint_as_float(u0 & 0xffff0000u), r1 = x1 - __uint_as_float(u1 & 0xffff0000u);
        if constexpr (N == 2) {
            t[1] = io<bf16_t>::pack2(r0, r1);
        } else {
            const uint32_t m0 = __float_as_uint(r0), m1 = __float_as_uint(r1);
            t[1] = __builtin_amdgcn_perm(m1, m0, 0x07060302u);
            const float s0 = r0 - __uint_as_float(m0 & 0xffff0000u), s1 = r1 - __uint_as_float(m1 & 0xffff0000u);
            t[2] = __builtin_amdgcn_perm(__float_as_uint(s1), __float_as_uint(s0), 0x07060302u);
        }
    }
}

__device__ __forceinline__ float lo_half(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_half(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// c += sum of the products of a's NA and b's NB terms whose order is at most
// kMax (2: down to 2^-24; 1: to 2^-16), small ones first
template <int NA, int NB, int kMax>
__device__ __forceinline__ f4 mfma_terms(const u4 (&a)[NA], const u4 (&b)[NB], f4 c) {
#pragma unroll
    for (int o = kMax; o >= 0; --o) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = o - i;
            if (j >= 0 && j < NB) c = mfma(a[i], b[j], c);
        }
    }
    return c;
}

// 8 summands of column col0 + lane % 16 of rows row0 + 8 (lane / 16) .. of a
// row-major LDS tile, by two transposing loads (the 16 lanes of a group read
// 4 rows of 16 elements and get a column of 4 each)
template <int STRIDE>
__device__ __forceinline__ u4 load_cols(const uint16_t* tile, int row0, int col0, int lane) {
    const int g = lane >> 4, c = lane & 15;
    const uint16_t* p = tile + (row0 + 8 * g + (c >> 2)) * STRIDE + col0 + 4 * (c & 3);
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
    const u2 hi = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * STRIDE)));
    return u4{lo.x, lo.y, hi.x, hi.y};
}

// 4 consecutive elements, the first cnt of them
typedef uint32_t half4_at2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4], int cnt) {
    if (cnt >= 4) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<words_at4*>(p) = words_at4{__float_as_uint(v[0]), __float_as_uint(v[1]),
                                                                                   __float_as_uint(v[2]), __float_as_uint(v[3])};
        else if constexpr (__is_same(T, bf16_t)) *reinterpret_cast<half4_at2*>(p) = half4_at2{io<bf16_t>::pack2(v[0], v[1]), io<bf16_t>::pack2(v[2], v[3])};
        else {
            const auto h = [&](int i) { return uint32_t(__builtin_bit_cast(uint16_t, _Float16(v[i]))); };
            *reinterpret_cast<half4_at2*>(p) = half4_at2{h(0) | h(1) << 16, h(2) | h(3) << 16};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < cnt) io<T>::store(p + i, v[i]);
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4], int cnt) {
    if (cnt >= 4) {
        if constexpr (sizeof(T) == 4) {
            const words_at4 w = *reinterpret_cast<const words_at4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
        } else {
            const half4_at2 w = *reinterpret_cast<const half4_at2*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
                if constexpr (__is_same(T, bf16_t)) v[i] = __uint_as_float(u << 16);
                else v[i] = float(__builtin_bit_cast(_Float16, uint16_t(u)));
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < cnt ? io<T>::load(p + i) : 0.f;
}

template <typename T> constexpr int kChunk = sizeof(T) == 2 && kTerms<T> == 1 ? 64 : 32;   // tokens per chunk

// Rows of a tile on their way from global memory to LDS.
template <typename T, int C, int WIDTH>
struct Stage {
    using R = rowvec<T>;
    static constexpr int PER_ROW = WIDTH / R::VE, N = (C * PER_ROW + 255) / 256, STRIDE = WIDTH + 8, TERMS = kTerms<T>;
    static constexpr int TERM = C * STRIDE;                  // elements of one term's tile
    static constexpr int STEP = 256 / PER_ROW;               // rows between a thread's vectors
    static constexpr bool PARTIAL = C * PER_ROW % 256 != 0;  // threads without a row
    uint4 v[N];

    // whether a tile of rows `step` elements apart is within 32-bit byte offsets of its first
    static __device__ __forceinline__ bool near(int64_t step) { return step < (int64_t(1) << 24); }
    // all rows of p (a row every `step` elements, a tile that is near), whole
    __device__ __forceinline__ void load_all(const T* p, int64_t step) {
        const int row = int(threadIdx.x) / PER_ROW, col = int(threadIdx.x) % PER_ROW * R::VE;
        const uint32_t off = (uint32_t(row) * uint32_t(step) + uint32_t(col)) * uint32_t(sizeof(T));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (PARTIAL && row >= C) continue;
            const typename R::words w = *reinterpret_cast<const typename R::words*>(
                reinterpret_cast<const char*>(p + int64_t(i * STEP) * step) + off);
            v[i] = make_uint4(w.x, w.y, w.z, w.w);
        }
    }
    // rows t0 .. of p, dim elements each; rows from `end` on are zero
    __device__ __forceinline__ void load(const T* p, int64_t step, int64_t t0, int64_t end, int dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = int(threadIdx.x) + 256 * i, row = at / PER_ROW, col = at % PER_ROW * R::VE;
            const int64_t t = t0 + row;
            v[i] = R::load(p + t * step + col, row < C && t < end ? dim - col : 0);
        }
    }
    // into the terms' tiles; CHECK: whether an element is infinite or NaN
    template <bool CHECK>
    __device__ __forceinline__ bool store(uint16_t* tile) const {
        typedef uint16_t h2 __attribute__((ext_vector_type(2)));
        h2 top = {0, 0};                                     // the largest exponents
        const auto look = [&](uint32_t w) {
            if constexpr (CHECK) top = __builtin_elementwise_max(top, __builtin_bit_cast(h2, w & 0x7f807f80u));
        };
        const int row = int(threadIdx.x) / PER_ROW, col = int(threadIdx.x) % PER_ROW * R::VE;
        if (PARTIAL && row >= C) return false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint16_t* to = tile + row * STRIDE + col + i * STEP * STRIDE;
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

// The chunk's decays.  Lane t of one wave holds token t's log decay (0 past
// the row's end).
template <int C>
struct __attribute__((aligned(16))) Decays {
    int I[C];              // integer part of H (G, or -G in reverse)
    float col[C];          // 2^-F, with the factor of v
    float row[C];          // 2^F, with the factor of o
    float in[C];           // the carried state's factor at a token over `row`'s 2^F
    float upd[C];          // a token's factor in the state's update, with the factor of v
    float total;           // 2^G_C

    __device__ __forceinline__ static float exp2_of(double x) {
        const double i = floor(x);
        return ldexpf(__builtin_amdgcn_exp2f(float(x - i)), i < -2000.0 ? -2000 : i > 2000.0 ? 2000 : int(i));
    }
    __device__ __forceinline__ void fill(int t, float g, bool rev, float vscale, float oscale) {
        double h = double(g) * 1.4426950408889634;
        h = h < kDeepest ? double(kDeepest) : h;          // (NaN stays)
#pragma unroll
        for (int m = 1; m < C; m <<= 1) {
            const double o = __shfl_up(h, m, 64);
            if (t >= m) h += o;
        }
        const double G = __shfl(h, C - 1, 64);
        if (t >= C) return;
        const double H = rev ? -h : h, fl = floor(H);
        const float F = float(H - fl);
        I[t] = int(fl);
        col[t] = vscale * __builtin_amdgcn_exp2f(-F);
        row[t] = oscale * __builtin_amdgcn_exp2f(F);
        in[t] = exp2_of((rev ? H + G : H) - double(F));
        upd[t] = vscale * exp2_of(rev ? -H : G - H);
        if (t == 0) total = exp2_of(G);
    }
};

__device__ __forceinline__ int64_t tokens_of(const int32_t* lens, int64_t b, int64_t L) {
    if (!lens) return L;
    const int64_t n = lens[b];
    return n < 0 ? 0 : n < L ? n : L;
}

// S <- total S + sum over the chunk's tokens of k_t (w_t v_t)^T.  kt: k's tile; vf: v's
// columns of this wave, 8 tokens a lane and 32-token step.
template <typename T, int KP, int NT, int C, typename SK>
__device__ __forceinline__ void update_state(f4 (&S)[KP / 16][NT], const uint16_t* kt, const u4 (&vf)[C / 32][NT][kTerms<T>],
                                             const Decays<C>& dec, int dims, int lane) {
    constexpr int R = kTerms<T>;
    const float tot = dec.total;
#pragma unroll
    for (int d = 0; d < KP / 16; ++d)
#pragma unroll
        for (int n = 0; n < NT; ++n) S[d][n] *= tot;
#pragma unroll
    for (int ks = 0; ks < C / 32; ++ks) {
        const f4* up = reinterpret_cast<const f4*>(dec.upd + 32 * ks + 8 * (lane >> 4));
        const f4 u0 = up[0], u1 = up[1];
        const float u[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
        u4 bv[NT][3];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                float x0 = lo_half(vf[ks][n][R - 1][w]), x1 = hi_half(vf[ks][n][R - 1][w]);
#pragma unroll
                for (int r = R - 2; r >= 0; --r) {            // small terms first: the sum is exact
                    x0 += lo_half(vf[ks][n][r][w]);
                    x1 += hi_half(vf[ks][n][r][w]);
                }
                uint32_t t[3];
                split<3>(x0 * u[2 * w], x1 * u[2 * w + 1], t);
#pragma unroll
                for (int i = 0; i < 3; ++i) bv[n][i][w] = t[i];
            }
        }
#pragma unroll
        for (int d = 0; d < KP / 16; ++d) {
            if (16 * d < dims) {
                u4 kf[R];
#pragma unroll
                for (int r = 0; r < R; ++r) kf[r] = load_cols<SK::STRIDE>(kt + r * SK::TERM, 32 * ks, 16 * d, lane);
#pragma unroll
                for (int n = 0; n < NT; ++n) S[d][n] = mfma_terms<R, 3, 2>(kf, bv[n], S[d][n]);
            }
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
// (32-bit divisions: a launch holds fewer than 2^24 workgroups, and the 64-bit
// ones cost a short walk a tenth of its time.)
struct Place { int job, tile, seg; uint32_t bh, b, h, shared; };      // (bh past the last one: nothing to do)
__device__ __forceinline__ Place place(Params& p, uint32_t segs) {
    uint32_t id = uint32_t(xcd_block_id());
    Place r;
    const uint32_t jobs = p.njobs, tiles = p.tiles, H = uint32_t(p.H);
    r.job = int(id % jobs);
    id /= jobs;
    r.tile = tiles > 1 ? int(id % tiles) : 0;
    if (tiles > 1) id /= tiles;
    r.seg = int(id % segs);
    r.bh = id / segs;
    r.b = r.bh / H;
    r.h = r.bh - r.b * H;
    r.shared = p.rep > 1 ? r.h / uint32_t(p.rep) : r.h;      // the group whose q and k head h reads
    return r;
}
template <typename T, typename Row>
__device__ __forceinline__ const T* rows_of_head(Row& r, const Place& at) {
    return static_cast<const T*>(r.p) + int64_t(at.b) * r.b + int64_t(r.rep > 1 ? at.shared : at.h) * r.h;
}

// ------------------------------------------------------- state of a segment --
// Each segment's state from a zero start, and its decay.
template <typename T, int KP, int NT>
__global__ __launch_bounds__(256) void la_local(const LaParams) {
    Params& p = params();
    constexpr int C = kChunk<T>, R = kTerms<T>;
    using SK = Stage<T, C, KP>;
    using SV = Stage<T, C, 64 * NT>;
    __shared__ __attribute__((aligned(16))) uint16_t kt[R * SK::TERM], vt[R * SV::TERM];
    __shared__ Decays<C> dec;
    const Place at = place(p, p.segs);
    Job& J = p.job[at.job];
    const int n0 = at.tile * 64 * NT;
    if (n0 >= J.V || at.bh >= uint32_t(p.B * p.H)) return;
    const int64_t b = at.b, h = at.h, bh = at.bh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int64_t s0 = at.seg * p.seg_tokens, s1 = s0 + p.seg_tokens < p.L ? s0 + p.seg_tokens : p.L;
    const int64_t len = tokens_of(p.lens, b, p.L), end = len < s1 ? len : s1;
    const T* kp = rows_of_head<T>(J.k, at);
    const T* vp = rows_of_head<T>(J.v, at) + n0;
    const float* gp = p.g + b * p.g_b + h * p.g_h;
    const int chunks = int((s1 - s0 + C - 1) / C), vdim = J.V - n0;
    const bool whole = J.K == KP && vdim >= 64 * NT && SK::near(J.k.l) && SV::near(J.v.l);

    f4 S[KP / 16][NT];
#pragma unroll
    for (int d = 0; d < KP / 16; ++d)
#pragma unroll
        for (int n = 0; n < NT; ++n) S[d][n] = f4{0.f, 0.f, 0.f, 0.f};
    float decay = 1.f;
    SK sk;
    SV sv;
    float gv = 0.f;
    const auto fetch = [&](int i) __attribute__((always_inline)) {
        const int64_t t0 = s0 + int64_t(J.rev ? chunks - 1 - i : i) * C;
        if (whole && t0 + C <= end) {
            sk.load_all(kp + t0 * J.k.l, J.k.l);
            sv.load_all(vp + t0 * J.v.l, J.v.l);
        } else {
            sk.load(kp, J.k.l, t0, end, J.K);
            sv.load(vp, J.v.l, t0, end, vdim);
        }
        gv = 0.f;
        if (wave == 0 && lane < C && t0 + lane < end) gv = gp[(t0 + lane) * p.g_l];
    };
    fetch(0);
    for (int i = 0; i < chunks; ++i) {
        (void)sk.template store<false>(kt);
        (void)sv.template store<false>(vt);
        if (wave == 0) dec.fill(lane, gv, J.rev, J.vscale, 1.f);
        __syncthreads();
        if (i + 1 < chunks) fetch(i + 1);
        u4 vf[C / 32][NT][R];
#pragma unroll
        for (int ks = 0; ks < C / 32; ++ks)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < R; ++r) vf[ks][n][r] = load_cols<SV::STRIDE>(vt + r * SV::TERM, 32 * ks, 16 * (4 * n + wave), lane);
        decay *= dec.total;
        update_state<T, KP, NT, C, SK>(S, kt, vf, dec, J.K, lane);
        __syncthreads();
    }
    float* to = J.ends + (bh * p.segs + at.seg) * int64_t(J.K) * J.V;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int col = n0 + 16 * (4 * n + wave) + c;
#pragma unroll
        for (int d = 0; d < KP / 16; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * d + 4 * g + r;
                if (row < J.K && col < J.V) to[int64_t(row) * J.st_k + int64_t(col) * J.st_v] = S[d][n][r];
            }
    }
    if (threadIdx.x == 0 && at.tile == 0) J.decays[bh * p.segs + at.seg] = decay;
}

// ----------------------------------------------------------------- the walk --
// P's 32 x 32 blocks that hold causal tiles: rows' half + tokens' half is
// 0, 1 or 2, whichever way the walk goes.
template <int C, int N>
struct Causal {
    static constexpr int STRIDE = 40, BLOCK = 32 * STRIDE, BLOCKS = C / 16 - 1, TERM = BLOCKS * BLOCK;
    static __device__ __forceinline__ int at(int row, int token) {
        return ((row >> 5) + (token >> 5)) * BLOCK + (row & 31) * STRIDE + (token & 31);
    }
};

// Workgroups per CU that LDS has room for (160 KiB) set the registers a wave may
// take: up to 3 waves a SIMD, which hide each other's barriers and loads.
template <typename T, int KP, int NT, int N>
constexpr int walk_lds() {
    constexpr int C = kChunk<T>, R = kTerms<T>;
    return 2 * (2 * R * Stage<T, C, KP>::TERM + R * Stage<T, C, 64 * NT>::TERM + N * Causal<C, N>::TERM) + 2 * int(sizeof(Decays<C>)) +
           16 * C + 256 * NT + 16;
}
template <typename T, int KP, int NT, int N>
constexpr int kWalkWaves = KP <= 64 && NT == 1 && 3 * walk_lds<T, KP, NT, N>() <= 163840 ? 3 : KP <= 128 && 2 * walk_lds<T, KP, NT, N>() <= 163840 ? 2 : 1;

template <typename T, int KP, int NT, int N>
__global__ __launch_bounds__(256, (kWalkWaves<T, KP, NT, N>)) void la_walk(const LaParams) {
    Params& p = params();
    constexpr int C = kChunk<T>, R = kTerms<T>, IT = C / 16, TRI = IT * (IT + 1) / 2, kMax = N == 2 ? 1 : 2;
    using SK = Stage<T, C, KP>;
    using SV = Stage<T, C, 64 * NT>;
    using CP = Causal<C, N>;
    __shared__ __attribute__((aligned(16))) uint16_t qt[R * SK::TERM], kt[R * SK::TERM], vt[R * SV::TERM], pt[N * CP::TERM];
    __shared__ Decays<C> decs[2];
    __shared__ float dots[4][C];
    __shared__ int bad_any, bad_col[64 * NT];
    const int segs = p.serial ? 1 : p.segs;
    const Place at = place(p, segs);
    Job& J = p.job[at.job];
    const int n0 = at.tile * 64 * NT;
    if (n0 >= J.V || at.bh >= uint32_t(p.B * p.H)) return;
    const int64_t b = at.b, h = at.h, bh = at.bh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int64_t span = p.serial ? p.L : p.seg_tokens;
    const int64_t s0 = at.seg * span, s1 = s0 + span < p.L ? s0 + span : p.L;
    const int64_t len = tokens_of(p.lens, b, p.L), end = len < s1 ? len : s1;
    const T* qp = rows_of_head<T>(J.q, at);
    const T* kp = rows_of_head<T>(J.k, at);
    const T* vp = rows_of_head<T>(J.v, at) + n0;
    const T* xp = J.dot ? rows_of_head<T>(J.x, at) + n0 : nullptr;
    const int64_t op = b * J.o.b + h * J.o.h + n0;
    const float* gp = p.g + b * p.g_b + h * p.g_h;
    const int64_t KV = int64_t(J.K) * J.V;
    const int chunks = int((s1 - s0 + C - 1) / C), vdim = J.V - n0, rev = J.rev;
    const int64_t seg_mask = p.seg_tokens - 1;
    const bool whole_v = vdim >= 64 * NT;
    const bool whole = J.K == KP && whole_v && SK::near(J.q.l) && SK::near(J.k.l) && SV::near(J.v.l);
    const bool near_o = whole_v && SV::near(J.o.l) && SV::near(J.x.l);

    // the state before the walk's first token
    const float* from = J.in ? J.in + bh * KV : nullptr;
    if (!p.serial) {
        const int before = rev ? at.seg + 1 : at.seg - 1;
        if (before >= 0 && before < p.segs) from = J.carry + (bh * p.segs + before) * KV;
    }
    f4 S[KP / 16][NT];
    const auto each_state = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int col = n0 + 16 * (4 * n + wave) + c;
#pragma unroll
            for (int d = 0; d < KP / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * d + 4 * g + r;
                    S[d][n][r] = f(S[d][n][r], row < J.K && col < J.V, uint32_t(row * J.st_k + col * J.st_v));
                }
        }
    };
    if (from) each_state([&](float, bool in, uint32_t i) { return in ? from[i] : 0.f; });
    else each_state([](float, bool, uint32_t) { return 0.f; });
    const auto write_state = [&](float* to) __attribute__((always_inline)) {
        each_state([&](float s, bool in, uint32_t i) {
            if (in) to[i] = s;
            return s;
        });
    };

    SK sq, sk;
    SV sv;
    float gv = 0.f;                                   // (wave 3) the decays of the chunk after the staged one
    const auto start = [&](int i) { return s0 + int64_t(rev ? chunks - 1 - i : i) * C; };
    const auto fetch = [&](int i) __attribute__((always_inline)) {
        const int64_t t0 = start(i);
        if (whole && t0 + C <= end) {
            sq.load_all(qp + t0 * J.q.l, J.q.l);
            sk.load_all(kp + t0 * J.k.l, J.k.l);
            sv.load_all(vp + t0 * J.v.l, J.v.l);
        } else {
            sq.load(qp, J.q.l, t0, end, J.K);
            sk.load(kp, J.k.l, t0, end, J.K);
            sv.load(vp, J.v.l, t0, end, vdim);
        }
    };
    const auto fetch_decay = [&](int i) __attribute__((always_inline)) {
        gv = 0.f;
        if (wave == 3 && i < chunks) {
            const int64_t t = start(i) + lane;
            if (lane < C && t < end) gv = gp[t * p.g_l];
        }
    };
    // the tiles of P's blocks above (in reverse: below) the diagonal
    for (int i = threadIdx.x; i < N * (C / 32) * 64; i += 256) {
        const int e = i % 64, row = 32 * (i / 64 % (C / 32)) + (rev ? 16 : 0) + e / 4, token = 32 * (i / 64 % (C / 32)) + (rev ? 0 : 16) + 4 * (e % 4);
        *reinterpret_cast<u2*>(pt + i / (64 * (C / 32)) * CP::TERM + CP::at(row, token)) = u2{0u, 0u};
    }
    if (threadIdx.x == 0) bad_any = 0;
    if (chunks > 0) {
        fetch_decay(0);
        fetch(0);
        if (wave == 3) decs[0].fill(lane, gv, rev, J.vscale, J.oscale);
        fetch_decay(1);
    }
    __syncthreads();
    for (int ci = 0; ci < chunks; ++ci) {
        const int64_t t0 = start(ci);
        const Decays<C>& dec = decs[ci & 1];
        (void)sq.template store<false>(qt);
        (void)sk.template store<false>(kt);
        if (sv.template store<true>(vt)) bad_any = 1;
        __syncthreads();
        if (ci + 1 < chunks) fetch(ci + 1);
        // A sum over tokens multiplies every v, by P's zeros too: infinities and
        // NaN of v are taken out of the tile here and put into the results from
        // their token on.
        const bool bad = bad_any != 0;
        if (bad) {
            __syncthreads();
            if (threadIdx.x == 0) bad_any = 0;
            if (int(threadIdx.x) < 64 * NT) {
                int first = rev ? -1 : C;
                for (int i = 0; i < C; ++i) {
                    const int row = rev ? i : C - 1 - i;
                    if ((vt[row * SV::STRIDE + threadIdx.x] & 0x7f80u) == 0x7f80u) {
                        first = row;
                        for (int r = 0; r < R; ++r) vt[r * SV::TERM + row * SV::STRIDE + threadIdx.x] = 0;
                    }
                }
                bad_col[threadIdx.x] = first;
            }
            __syncthreads();
        }

        // P's causal tiles, dealt out to the waves
#pragma unroll
        for (int s = 0; s < (TRI + 3) / 4; ++s) {
            const int tile = 4 * s + wave;
            if (tile < TRI) {
                int it = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, jt = tile - it * (it + 1) / 2;
                if (rev) {
                    it = IT - 1 - it;
                    jt = IT - 1 - jt;
                }
                f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KP / 32; ++kk) {
                    if (32 * kk >= J.K) continue;
                    u4 kf[R], qf[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        kf[r] = *reinterpret_cast<const u4*>(kt + r * SK::TERM + (16 * jt + c) * SK::STRIDE + 32 * kk + 8 * g);
                        qf[r] = *reinterpret_cast<const u4*>(qt + r * SK::TERM + (16 * it + c) * SK::STRIDE + 32 * kk + 8 * g);
                    }
                    acc = mfma_terms<R, R, 2>(kf, qf, acc);
                }
                typedef int i4 __attribute__((ext_vector_type(4)));
                const i4 Ij = *reinterpret_cast<const i4*>(dec.I + 16 * jt + 4 * g);
                acc *= *reinterpret_cast<const f4*>(dec.col + 16 * jt + 4 * g);
                const int Ii = dec.I[16 * it + c];
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = __builtin_amdgcn_ldexpf(acc[r], Ii - Ij[r]);
                if (it == jt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = (rev ? 4 * g + r < c : 4 * g + r > c) ? 0.f : v[r];
                }
                uint32_t lo[N], hi[N];
                split<N>(v[0], v[1], lo);
                split<N>(v[2], v[3], hi);
#pragma unroll
                for (int t = 0; t < N; ++t)
                    *reinterpret_cast<u2*>(pt + t * CP::TERM + CP::at(16 * it + c, 16 * jt + 4 * g)) = u2{lo[t], hi[t]};
            }
        }
        // the next chunk's decays, by the wave with the fewest tiles
        if (wave == 3 && ci + 1 < chunks) decs[(ci + 1) & 1].fill(lane, gv, rev, J.vscale, J.oscale);
        fetch_decay(ci + 2);
        __syncthreads();

        // o^T: q S with the carried state's factor, then P V
        f4 o[IT][NT];
#pragma unroll
        for (int it = 0; it < IT; ++it)
#pragma unroll
            for (int n = 0; n < NT; ++n) o[it][n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KP / 32; ++kk) {
            if (32 * kk >= J.K) continue;
            u4 sf[NT][N];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t t[N];
                    const f4& s = S[2 * kk + (w >> 1)][n];
                    split<N>(s[2 * (w & 1)], s[2 * (w & 1) + 1], t);
#pragma unroll
                    for (int i = 0; i < N; ++i) sf[n][i][w] = t[i];
                }
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                u4 qf[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint16_t* q = qt + r * SK::TERM + (16 * it + c) * SK::STRIDE + 32 * kk + 4 * g;
                    const u2 a = *reinterpret_cast<const u2*>(q), d = *reinterpret_cast<const u2*>(q + 16);
                    qf[r] = u4{a.x, a.y, d.x, d.y};
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) o[it][n] = mfma_terms<N, R, kMax>(sf[n], qf, o[it][n]);
            }
        }
        u4 vf[C / 32][NT][R];
#pragma unroll
        for (int ks = 0; ks < C / 32; ++ks)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < R; ++r) vf[ks][n][r] = load_cols<SV::STRIDE>(vt + r * SV::TERM, 32 * ks, 16 * (4 * n + wave), lane);
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const float f = dec.in[16 * it + c];
#pragma unroll
            for (int n = 0; n < NT; ++n) o[it][n] *= f;
#pragma unroll
            for (int ks = 0; ks < C / 32; ++ks) {
                if (rev ? 32 * ks + 31 < 16 * it : 32 * ks > 16 * it + 15) continue;
                u4 pf[N];
#pragma unroll
                for (int t = 0; t < N; ++t) pf[t] = *reinterpret_cast<const u4*>(pt + t * CP::TERM + CP::at(16 * it + c, 32 * ks + 8 * g));
#pragma unroll
                for (int n = 0; n < NT; ++n) o[it][n] = mfma_terms<R, N, kMax>(vf[ks][n], pf, o[it][n]);
            }
            const float last = dec.row[16 * it + c];
#pragma unroll
            for (int n = 0; n < NT; ++n) o[it][n] *= last;
        }
        const bool last = ci + 1 == chunks;
        if (!last || J.ends || J.out_state) update_state<T, KP, NT, C, SK>(S, kt, vf, dec, J.K, lane);

        float dot[IT] = {};
        if (near_o && t0 + C <= end && !bad) {
            const int64_t first = op + t0 * J.o.l;
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                const uint32_t row = uint32_t(c) * uint32_t(J.o.l), xrow = uint32_t(c) * uint32_t(J.x.l);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t col = uint32_t(16 * (4 * n + wave) + 4 * g);
                    const float v[4] = {o[it][n][0], o[it][n][1], o[it][n][2], o[it][n][3]};
                    if (J.o_f32) store4<float>(static_cast<float*>(const_cast<void*>(J.o.p)) + (first + 16 * it * J.o.l) + (row + col), v, 4);
                    else store4<T>(static_cast<T*>(const_cast<void*>(J.o.p)) + (first + 16 * it * J.o.l) + (row + col), v, 4);
                    if (J.dot) {
                        float x[4];
                        load4<T>(xp + (t0 + 16 * it) * J.x.l + (xrow + col), x, 4);
#pragma unroll
                        for (int r = 0; r < 4; ++r) dot[it] = __builtin_fmaf(v[r], x[r], dot[it]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                const int i = 16 * it + c;
                const int64_t t = t0 + i;
                const bool live = t < len;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int col = 16 * (4 * n + wave) + 4 * g, cnt = t < s1 ? vdim - col : 0;
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        v[r] = live ? o[it][n][r] : 0.f;
                        if (bad && live && (rev ? i <= bad_col[col + r] : i >= bad_col[col + r])) v[r] = __builtin_nanf("");
                    }
                    if (cnt > 0) {
                        const int64_t to = op + t * J.o.l + col;
                        if (J.o_f32) store4<float>(static_cast<float*>(const_cast<void*>(J.o.p)) + to, v, cnt);
                        else store4<T>(static_cast<T*>(const_cast<void*>(J.o.p)) + to, v, cnt);
                        if (J.dot && live) {
                            float x[4];
                            load4<T>(xp + t * J.x.l + col, x, cnt);
#pragma unroll
                            for (int r = 0; r < 4; ++r) dot[it] = __builtin_fmaf(r < cnt ? v[r] : 0.f, x[r], dot[it]);
                        }
                    }
                }
            }
        }
        if (J.dot) {
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                // over the lanes of the token's other columns: g = 0 .. 3
                auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(dot[it]), __float_as_uint(dot[it]), false, false);
                float d = __uint_as_float(s[0]) + __uint_as_float(s[1]);
                s = __builtin_amdgcn_permlane16_swap(__float_as_uint(d), __float_as_uint(d), false, false);
                d = __uint_as_float(s[0]) + __uint_as_float(s[1]);
                if (g == 0) dots[wave][16 * it + c] = d;
            }
        }
        if (bad) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int first = bad_col[16 * (4 * n + wave) + c];
                if (first >= 0 && first < C) {
#pragma unroll
                    for (int d = 0; d < KP / 16; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[d][n][r] = __builtin_nanf("");
                }
            }
        }
        if (J.ends && ((rev ? t0 & seg_mask : (t0 + C) & seg_mask) == 0 || (!rev && last)))
            write_state(J.ends + (bh * p.segs + (t0 >> p.seg_shift)) * KV);
        __syncthreads();
        if (J.dot && int(threadIdx.x) < C && t0 + threadIdx.x < s1)
            J.dot[(int64_t(at.tile) * p.B * p.H + bh) * p.L + t0 + threadIdx.x] =
                (dots[0][threadIdx.x] + dots[1][threadIdx.x]) + (dots[2][threadIdx.x] + dots[3][threadIdx.x]);
    }
    if (chunks == 0 && J.ends) write_state(J.ends + bh * p.segs * KV);
    if (J.out_state) write_state(J.out_state + bh * KV);
}

}  // namespace la

// Launches over J.K <= KP, J.V in column tiles of 64 NT (see la_tile).
template <typename F>
hipError_t la_for_dims(const LaParams& p, F&& f) {
    using std::integral_constant;
    int k = 0;
    for (int j = 0; j < p.njobs; ++j) k = p.job[j].K > k ? p.job[j].K : k;
    const auto with = [&](auto kp) {
        return p.tile == 64 ? f(kp, integral_constant<int, 1>{}) : f(kp, integral_constant<int, 2>{});
    };
    if (k <= 32) return with(integral_constant<int, 32>{});
    if (k <= 64) return with(integral_constant<int, 64>{});
    if (k <= 128) return with(integral_constant<int, 128>{});
    return with(integral_constant<int, 256>{});
}
// (a multiple of the XCDs, so that a segment's workgroups share one)
inline dim3 la_grid(const LaParams& p, int segs) {
    const int64_t n = p.B * p.H * segs * p.tiles * p.njobs;
    return dim3(unsigned((n + kXcds - 1) / kXcds * kXcds));
}

template <typename T>
hipError_t la_local_launch(const LaParams& p, hipStream_t stream) {
    return la_for_dims(p, [&](auto kp, auto nt) {
        hipLaunchKernelGGL((la::la_local<T, decltype(kp)::value, decltype(nt)::value>), la_grid(p, p.segs), dim3(256), 0, stream, p);
        return hipGetLastError();
    });
}
template <typename T>
hipError_t la_walk_launch(const LaParams& p, bool fine, hipStream_t stream) {
    return la_for_dims(p, [&](auto kp, auto nt) {
        constexpr int KP = decltype(kp)::value, NT = decltype(nt)::value;
        const dim3 grid = la_grid(p, p.serial ? 1 : p.segs);
        if constexpr (sizeof(T) == 2) {
            if (!fine) {
                hipLaunchKernelGGL((la::la_walk<T, KP, NT, 2>), grid, dim3(256), 0, stream, p);
                return hipGetLastError();
            }
        }
        hipLaunchKernelGGL((la::la_walk<T, KP, NT, 3>), grid, dim3(256), 0, stream, p);
        return hipGetLastError();
    });
}

}  // namespace ss

// The gated delta rule in chunks on the matrix cores (gfx950).
//
// Per (batch, head), with a_t = exp(g_t) and the state S (d_key x d_value):
//
//   e_t = v_t - a_t S_{t-1}^T k_t,   S_t = a_t S_{t-1} + beta_t k_t e_t^T,   o_t = scale S_t^T q_t
//
// In a chunk, with S the state before it, G_i the sum of the log decays up to
// token i (itself included) and w_ij = exp(G_i - G_j):
//
//   E   = T (V - exp(G) K S),   T = (I + N)^-1,   N_ij = w_ij (k_i . k_j) beta_j  for j < i
//   O   = scale (exp(G) Q S + P U),   U = beta E,   P_ij = w_ij q_i . k_j  for j <= i
//   S'  = exp(G_end) S + sum_j exp(G_end - G_j) k_j u_j^T
//
// and back, from dS' (the gradient of S'):
//
//   dU = scale P^T dO + exp(G_end - G) K dS',   F = T^T (beta dU) = dV
//   dS = exp(G_end) dS' + scale sum_i exp(G_i) q_i dO_i^T - sum_i exp(G_i) k_i F_i^T
//
// with the gradients of q, k, g and beta from S, dS', E and F (dr_grads).
//
// Three kinds of launch.  T does not depend on the state, so the inverses of all
// chunks are formed side by side (dr_prep).  The walk (dr_walk) is what is
// serial: a workgroup holds the state's 64 value columns, 16 a wave, in registers and
// goes from chunk to chunk; value columns do not meet.  It keeps S and E (back: dS'
// and F) of each chunk, and from these all other gradients are formed chunk by
// chunk side by side (dr_grads).
//
// Products run on bf16 matrix instructions with 32-bit sums, over values split
// into bf16 terms (bf16_terms.hpp): rows as they are, what is computed in 3 terms
// (2^-24) on the way into a state or into a 32-bit gradient, in 2 (2^-17) where
// only a 16-bit result is formed from it.
//
// Layouts.  An instruction's result (4 rows of a column a lane) is an operand of the
// next one as it is: two 16-row tiles are 32 summands, slot i of lane group g
// being row 4 g + i of the first (i < 4) or of the second.  So the state, E, U
// and F never leave the registers of their wave on the way through the products; rows
// and triangles come from LDS in that order, or through the transposing load where
// sums run over their rows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "bf16_terms.hpp"
#include "delta_rule.hpp"
#include "norm_rows.hpp"
#include "ss_device.hpp"

namespace ss {

namespace dr {

using namespace la;

// log2 decays below it empty the state (fp32 ends at 2^-149) and leave 64-bit sums of
// a chunk's tokens 30 bits below the point
constexpr double kEmpty = -1e5;
// Where beta is zero (or smaller) the inverse takes this in its place, and so do F and M
// of the backward: then dbeta, the sum F . E over beta, keeps its value, and what else they
// enter changes by 2^-60 of E.
constexpr float kLeastBeta = 8.673617379884035e-19f;      // 2^-60
__device__ __forceinline__ float beta_or_least(float b) { return fabsf(b) < kLeastBeta ? kLeastBeta : b; }

template <typename T, int KP>
struct Dims {
    static constexpr int KT = kTerms<T>, C = dr_chunk(KP, KT), NR = C / 16, NP = C / 32, NK = KP / 32, NS = KP / 16;
    static constexpr int NT = NR * (NR + 1) / 2;             // lower tiles of a chunk's square
    static constexpr int KST = KP + 8, CST = C + 8;          // row strides in LDS, elements
    static constexpr int VST = 64 + 8;
    static constexpr int OT = sizeof(T) == 4 ? 3 : 2;        // terms of what only a result of type T is formed from
};

template <typename T, int KP> constexpr int kPrepThreads = 64 * Dims<T, KP>::NR;
template <typename T, int KP> constexpr int kGradThreads = 128 * Dims<T, KP>::NR;

template <int NA, int NB, int MAX>
__device__ __forceinline__ void mac(const u4 (&a)[NA], const u4 (&b)[NB], f4& c) {
#pragma unroll
    for (int o = MAX; o >= 0; --o)
#pragma unroll
        for (int x = 0; x < NA; ++x)
            if (o - x >= 0 && o - x < NB) c = mfma(a[x], b[o - x], c);
}
// 32 summands of two result tiles, in N terms
template <int N>
__device__ __forceinline__ void pack(const f4& lo, const f4& hi, u4 (&t)[N]) {
    uint32_t s[N];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const f4& x = h < 2 ? lo : hi;
        split<N>(x[2 * (h & 1)], x[2 * (h & 1) + 1], s);
#pragma unroll
        for (int n = 0; n < N; ++n) t[n][h] = s[n];
    }
}
// operands from N term tiles TERM elements apart: 8 neighbouring elements; 4 and the 4 that lie 16 further on
template <int N, int TERM>
__device__ __forceinline__ void frag8(const uint16_t* at, u4 (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = *reinterpret_cast<const u4*>(at + n * TERM);
}
template <int N, int TERM>
__device__ __forceinline__ void frag44(const uint16_t* at, u4 (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const u2 lo = *reinterpret_cast<const u2*>(at + n * TERM), hi = *reinterpret_cast<const u2*>(at + n * TERM + 16);
        t[n] = u4{lo.x, lo.y, hi.x, hi.y};
    }
}
// the same of a column: 32 rows of the tile from `at` on
template <int N, int TERM, int STRIDE>
__device__ __forceinline__ void frag_col(const uint16_t* at, int block, int lane, u4 (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = load_tokens<STRIDE>(at + n * TERM, block, lane);
}
// first of the 4 columns a lane reads for its group: of 16 neighbouring ones, and of the state's tile t
__device__ __forceinline__ int block16(int t, int lane) { return 16 * t + 4 * (lane & 3); }
__device__ __forceinline__ int state_block(int t, int lane) { return 32 * (t >> 1) + 8 * (lane & 3) + 4 * (t & 1); }

// A chunk's rows (C x KP of type T) from global memory into term tiles, by NTH threads.
template <typename T, int KP, int C, int NTH>
struct Tile {
    using R = rowvec<T>;
    static constexpr int PER = KP / R::VE, N = C * PER / NTH, KT = kTerms<T>, KST = KP + 8, TERM = C * KST;
    static_assert(C * PER % NTH == 0, "whole vectors a thread");
    uint4 v[N];
    __device__ __forceinline__ void load(const T* p, int64_t step, int rows, int dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = int(threadIdx.x) + i * NTH, row = at / PER, col = at % PER * R::VE;
            v[i] = R::load(p + int64_t(row) * step + col, row < rows ? dim - col : 0);
        }
    }
    __device__ __forceinline__ void store(uint16_t* tile) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = int(threadIdx.x) + i * NTH;
            uint16_t* to = tile + at / PER * KST + at % PER * R::VE;
            if constexpr (KT == 1) {
                *reinterpret_cast<uint4*>(to) = v[i];
            } else {
                float x[R::VE];
                R::unpack(v[i], x);
                uint32_t t[R::VE / 2][KT];
#pragma unroll
                for (int k = 0; k < R::VE / 2; ++k) split<KT>(x[2 * k], x[2 * k + 1], t[k]);
#pragma unroll
                for (int n = 0; n < KT; ++n) {
                    if constexpr (R::VE == 8) *reinterpret_cast<uint4*>(to + n * TERM) = make_uint4(t[0][n], t[1][n], t[2][n], t[3][n]);
                    else *reinterpret_cast<uint2*>(to + n * TERM) = make_uint2(t[0][n], t[1][n]);
                }
            }
        }
    }
};

// A chunk's decays and rates.  G: sums of log2 decays from the chunk's start, in 64
// bits, so that a difference of two keeps its bits however far they run.
template <int C>
struct Gates {
    double G[C];
    float gam[C], end[C], beta[C];         // exp(G), exp(G_end - G)
    float total, pad[3];                   // exp(G_end)
};
template <int C>
__device__ __forceinline__ void put_gates(Gates<C>& s, float g, float beta, int lane) {
    double x = double(g) * 1.4426950408889634;
    x = x < kEmpty ? kEmpty : x;
#pragma unroll
    for (int m = 1; m < C; m <<= 1) {
        const double y = __shfl_up(x, m, 64);
        x += lane >= m ? y : 0.0;
    }
    const double all = __shfl(x, C - 1, 64);
    if (lane < C) {
        s.G[lane] = x;
        s.gam[lane] = __builtin_amdgcn_exp2f(float(x));
        s.end[lane] = __builtin_amdgcn_exp2f(float(all - x));
        s.beta[lane] = beta;
    }
    if (lane == 0) s.total = __builtin_amdgcn_exp2f(float(all));
}
__device__ __forceinline__ float factor(double Gi, double Gj) { return __builtin_amdgcn_exp2f(float(Gi - Gj)); }

struct Head {
    int64_t bh, b, h, len;                 // len: the row's tokens
    __device__ __forceinline__ Head(const DrParams& p, int64_t bh_) : bh(bh_) {
        b = bh / p.H;
        h = bh % p.H;
        const int64_t n = p.lens ? p.lens[b] : p.L;
        len = n < 0 ? 0 : n < p.L ? n : p.L;
    }
    template <typename T> __device__ __forceinline__ const T* rows(const LaRows& r, int64_t t) const {
        return static_cast<const T*>(r.p) + b * r.b + t * r.l + (h / r.rep) * r.h;
    }
    __device__ __forceinline__ float g(const DrParams& p, int64_t t) const { return t < len ? p.g[b * p.g_b + t * p.g_l + h * p.g_h] : 0.f; }
    __device__ __forceinline__ float beta(const DrParams& p, int64_t t) const {
        return t < len ? p.beta[b * p.be_b + t * p.be_l + h * p.be_h] : 0.f;
    }
};

// ------------------------------------------------------------- inverses --
// T of a chunk.  Wave i forms N's row of tiles and the inverse of its diagonal tile by
// substitution (16 steps, every lane a column); then wave j the tiles below its
// diagonal one, T_ij = -T_ii sum_{j <= m < i} N_im T_mj, on fp32 matrix instructions.
// Substitution and these products keep the bits of a stable solve, which powers of N
// would not: for equal keys they reach binomial coefficients.
template <typename T, int KP>
__global__ __launch_bounds__((kPrepThreads<T, KP>)) void dr_prep(const DrParams p) {
    using D = Dims<T, KP>;
    constexpr int C = D::C, NR = D::NR, KT = D::KT, KST = D::KST, TERM = C * KST, NST = C + 4;
    __shared__ __attribute__((aligned(16))) uint16_t ks[KT * TERM];
    __shared__ __attribute__((aligned(16))) float ns[C * NST], ts[NR][16 * 20];
    __shared__ Gates<C> gates;
    const Head head(p, blockIdx.x / unsigned(p.nch));
    const int64_t n = blockIdx.x % unsigned(p.nch), t0 = n * C;
    if (t0 >= head.len) return;
    const int lane = int(threadIdx.x) & 63, w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), g = lane >> 4, c = lane & 15;
    const int cnt = head.len - t0 < C ? int(head.len - t0) : C;
    {
        Tile<T, KP, C, 64 * NR> k;
        k.load(head.rows<T>(p.k, t0), p.k.l, cnt, p.K);
        if (w == 0) {
            const bool in = lane < C;
            put_gates(gates, in ? head.g(p, t0 + lane) : 0.f, in ? head.beta(p, t0 + lane) : 0.f, lane);
        }
        k.store(ks);
    }
    __syncthreads();
    // N's row of tiles, transposed: rows j, column i
    const double Gi = gates.G[16 * w + c];
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        if (j > w) continue;
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < D::NK; ++kk) {
            u4 a[KT], b[KT];
            frag8<KT, TERM>(ks + (16 * j + c) * KST + 32 * kk + 8 * g, a);
            frag8<KT, TERM>(ks + (16 * w + c) * KST + 32 * kk + 8 * g, b);
            mac<KT, KT, 2>(a, b, acc);
        }
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * j + 4 * g + r;
            x[r] = row < 16 * w + c ? acc[r] * factor(Gi, gates.G[row]) * beta_or_least(gates.beta[row]) : 0.f;
        }
        *reinterpret_cast<float4*>(ns + (16 * w + c) * NST + 16 * j + 4 * g) = make_float4(x[0], x[1], x[2], x[3]);
    }
    __syncthreads();
    // the diagonal tile's inverse: column c, the rows of it
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float row[16];
#pragma unroll
        for (int j = 0; j < r; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(ns + (16 * w + r) * NST + 16 * w + j);
            row[j] = v.x; row[j + 1] = v.y; row[j + 2] = v.z; row[j + 3] = v.w;
        }
        float s0 = r == c ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < r; ++j) (j & 1 ? s1 : s0) = __builtin_fmaf(-row[j], x[j], j & 1 ? s1 : s0);
        x[r] = s0 + s1;
    }
    f4 t[NR];                                  // column w's tiles, from the diagonal one on
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float lo = g & 1 ? x[4 + r] : x[r], hi = g & 1 ? x[12 + r] : x[8 + r];
        t[0][r] = g & 2 ? hi : lo;
        ts[w][(4 * g + r) * 20 + c] = t[0][r];
    }
    __syncthreads();
    const auto mm = [&](const float* a, const f4& b, f4 acc) {       // a: 16 rows of this lane's, 4 summands from 4 g on
        const float4 v = *reinterpret_cast<const float4*>(a);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v.x, b[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v.y, b[1], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v.z, b[2], acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(v.w, b[3], acc, 0, 0, 0);
    };
    float* out = p.tri + (head.bh * p.nch + n) * (D::NT * 256);
#pragma unroll
    for (int d = 0; d < NR; ++d) {
        const int i = w + d;
        if (i >= NR) break;
        if (d > 0) {
            f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < d; ++m) acc = mm(ns + (16 * i + c) * NST + 16 * (w + m) + 4 * g, t[m], acc);
            f4 r = mm(&ts[i][c * 20 + 4 * g], acc, f4{0.f, 0.f, 0.f, 0.f});
            t[d] = -r;
        }
        float* to = out + (i * (i + 1) / 2 + w) * 256;
#pragma unroll
        for (int r = 0; r < 4; ++r) to[(4 * g + r) * 16 + c] = t[d][r];
    }
}

// ----------------------------------------------------------------- walk --
// A chunk's inverse on its way into LDS, in 3 terms (row-major, zero above the
// diagonal tiles: the caller clears the tiles (2 p, 2 p + 1) once)
template <int C, int NTH>
struct Tri {
    static constexpr int NR = C / 16, NT = NR * (NR + 1) / 2, N = (NT * 64 + NTH - 1) / NTH, CST = C + 8, TERM = C * CST;
    float4 v[N];
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = int(threadIdx.x) + i * NTH;
            if (at < NT * 64) v[i] = *reinterpret_cast<const float4*>(p + 4 * at);
        }
    }
    __device__ __forceinline__ void store(uint16_t* tile) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = int(threadIdx.x) + i * NTH;
            if (at >= NT * 64) continue;
            const int idx = at >> 6, row = idx < 1 ? 0 : idx < 3 ? 1 : idx < 6 ? 2 : 3, col = idx - row * (row + 1) / 2;
            uint16_t* to = tile + (16 * row + ((at >> 2) & 15)) * CST + 16 * col + 4 * (at & 3);
            uint32_t s0[3], s1[3];
            split<3>(v[i].x, v[i].y, s0);
            split<3>(v[i].z, v[i].w, s1);
#pragma unroll
            for (int n = 0; n < 3; ++n) *reinterpret_cast<uint2*>(to + n * TERM) = make_uint2(s0[n], s1[n]);
        }
    }
};

// The walk over the chunks of a segment (or of the whole row), forward (REV false) or back.
//
// Forward it writes out, the states and errors that a backward needs (unless null) and the
// last state; back, from dout, the states' and errors' gradients and the initial state's.
// LOCAL: the states only, from zero, and beside them what the segment makes of the
// columns of the identity (value tiles past the last: no values, the state starts as I).
template <typename T, int KP, bool REV, bool LOCAL>
__global__ __launch_bounds__(256) void dr_walk(const DrParams p) {
    using D = Dims<T, KP>;
    constexpr int C = D::C, NR = D::NR, NP = D::NP, NK = D::NK, NS = D::NS, KT = D::KT, KST = D::KST, CST = D::CST;
    constexpr int KTERM = C * KST, CTERM = C * CST;
    constexpr int PT = REV ? 3 : D::OT;                   // P's terms
    constexpr bool Q = REV || !LOCAL;                     // whether q is read
    __shared__ __attribute__((aligned(16))) uint16_t ks[KT * KTERM], qs[Q ? KT * KTERM : 8], tri[3 * CTERM], prob[Q ? PT * CTERM : 8];
    __shared__ Gates<C> gates[2];
    const int segs = p.segs, seg = int(blockIdx.x % unsigned(segs));
    const Head head(p, blockIdx.x / unsigned(segs));
    const int vt = int(blockIdx.y), vtiles = (p.V + 63) / 64;
    const int tid = int(threadIdx.x), lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const bool unit = LOCAL && vt >= vtiles;              // columns of the identity
    const int col0 = (unit ? vt - vtiles : vt) * 64 + 16 * w, col = col0 + c;
    const int cols = unit ? p.K : p.V, pitch = unit ? dr_round16(p.K) : p.Vp;
    const bool live = col0 < cols, mine = !unit && col < p.V;
    const int chunks = int((head.len + C - 1) / C);       // of the row
    const int n0 = seg * p.seg_chunks, n1 = n0 + p.seg_chunks < chunks ? n0 + p.seg_chunks : chunks;

    // the state: tile t, register r is row state_row(t, g, r), column col
    f4 S[NS];
    {
        const float* from = nullptr;
        int64_t step = 0;
        if (!LOCAL) {
            if (segs > 1) from = p.seg_add + (head.bh * segs + seg) * p.K * p.Vp + col, step = p.Vp;
            else if (p.init) from = p.init + head.bh * p.K * p.V + col, step = p.V;
        }
#pragma unroll
        for (int t = 0; t < NS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = state_row(t, g, r);
                S[t][r] = from && mine && key < p.K ? from[key * step] : unit && key == col && key < p.K ? 1.f : 0.f;
            }
    }
    const auto put_state = [&](float* to, int64_t step, bool in) {
#pragma unroll
        for (int t = 0; t < NS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = state_row(t, g, r);
                if (in && key < p.K) to[key * step] = S[t][r];
            }
    };

    Tile<T, KP, C, 256> kin, qin;
    Tri<C, 256> tin;
    float xin[NR][4], gin = 0.f, bin = 0.f;               // v (back: dout), rows 16 i + 4 g + r of column col
    const int step = REV ? -1 : 1, first = REV ? n1 - 1 : n0;
    const auto count = [&](int n) { return head.len - int64_t(n) * C < C ? int(head.len - int64_t(n) * C) : C; };
    const auto fetch_gates = [&](int n) {
        const bool in = n >= n0 && n < n1 && lane < C;
        gin = in ? head.g(p, int64_t(n) * C + lane) : 0.f;
        bin = in ? head.beta(p, int64_t(n) * C + lane) : 0.f;
    };
    const auto fetch = [&](int n) {
        if (n < n0 || n >= n1) return;
        const int64_t t0 = int64_t(n) * C;
        const int cnt = count(n);
        kin.load(head.rows<T>(p.k, t0), p.k.l, cnt, p.K);
        if constexpr (Q) qin.load(head.rows<T>(p.q, t0), p.q.l, cnt, p.K);
        tin.load(p.tri + (head.bh * p.nch + n) * (D::NT * 256));
        const LaRows& rows = REV ? p.o : p.v;
        const T* x = head.rows<T>(rows, t0) + col;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * i + 4 * g + r;
                xin[i][r] = mine && row < cnt ? io<T>::load(x + row * rows.l) : 0.f;
            }
    };
    // (tiles above the diagonal that pairs of tiles take in: zero for good)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        for (int e = tid; e < 16 * 16; e += 256) {
            const int at = (32 * i + (e >> 4)) * CST + 32 * i + 16 + (e & 15);
#pragma unroll
            for (int n = 0; n < 3; ++n) tri[n * CTERM + at] = 0;
            if constexpr (Q) {
#pragma unroll
                for (int n = 0; n < PT; ++n) prob[n * CTERM + at] = 0;
            }
        }
    }
    if (n0 < n1) {
        fetch_gates(first);
        fetch(first);
        if (w == 0) put_gates(gates[first & 1], gin, bin, lane);
        fetch_gates(first + step);
    }
    for (int n = first; n >= n0 && n < n1; n += step) {
        const int64_t at = head.bh * p.nch + n, t0 = int64_t(n) * C;
        const Gates<C>& G = gates[n & 1];
        __syncthreads();                                  // (the tiles of the chunk before are done with)
        kin.store(ks);
        if constexpr (Q) qin.store(qs);
        tin.store(tri);
        f4 x[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[i][r] = xin[i][r];
        __syncthreads();
        fetch(n + step);
        if (w == 0) {
            put_gates(gates[(n + 1) & 1], gin, bin, lane);
            fetch_gates(n + 2 * step);
        }
        if constexpr (Q) {                                // P, a share of its tiles a wave; formed transposed, rows j, column i
#pragma unroll
            for (int i = 0; i < NR; ++i) {
#pragma unroll
                for (int j = 0; j <= i; ++j) {
                    if (((i * (i + 1) / 2 + j) & 3) != w) continue;
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kk = 0; kk < NK; ++kk) {
                        u4 a[KT], b[KT];
                        frag8<KT, KTERM>(ks + (16 * j + c) * KST + 32 * kk + 8 * g, a);
                        frag8<KT, KTERM>(qs + (16 * i + c) * KST + 32 * kk + 8 * g, b);
                        mac<KT, KT, 2>(a, b, acc);
                    }
                    const double Gi = G.G[16 * i + c];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 16 * j + 4 * g + r;
                        acc[r] = row <= 16 * i + c ? acc[r] * factor(Gi, G.G[row]) : 0.f;
                    }
                    uint32_t s0[PT], s1[PT];
                    split<PT>(acc[0], acc[1], s0);
                    split<PT>(acc[2], acc[3], s1);
#pragma unroll
                    for (int m = 0; m < PT; ++m)
                        *reinterpret_cast<uint2*>(prob + m * CTERM + (16 * i + c) * CST + 16 * j + 4 * g) = make_uint2(s0[m], s1[m]);
                }
            }
        }
        if constexpr (!REV) {
            f4 O[NR];                                     // out, transposed: rows value columns, column token i
            u4 uf[NP][D::OT];
            if (live) {
                if (!LOCAL && p.states) put_state(p.states + at * p.K * p.Vp + col, p.Vp, true);
                f4 Y[NR];
#pragma unroll
                for (int i = 0; i < NR; ++i) Y[i] = O[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    u4 sf[3];
                    pack<3>(S[2 * kk], S[2 * kk + 1], sf);
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        u4 a[KT];
                        frag8<KT, KTERM>(ks + (16 * i + c) * KST + 32 * kk + 8 * g, a);
                        mac<KT, 3, 2>(a, sf, Y[i]);
                        if constexpr (!LOCAL) {
                            frag8<KT, KTERM>(qs + (16 * i + c) * KST + 32 * kk + 8 * g, a);
                            mac<3, KT, D::OT - 1>(sf, a, O[i]);
                        }
                    }
                }
                u4 yf[NP][3];
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const f4 gam = *reinterpret_cast<const f4*>(G.gam + 16 * i + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) Y[i][r] = __builtin_fmaf(-gam[r], Y[i][r], x[i][r]);
                }
#pragma unroll
                for (int q = 0; q < NP; ++q) pack<3>(Y[2 * q], Y[2 * q + 1], yf[q]);
                f4 U[NR];
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    f4 E = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int q = 0; q <= i / 2; ++q) {
                        u4 a[3];
                        frag44<3, CTERM>(tri + (16 * i + c) * CST + 32 * q + 4 * g, a);
                        mac<3, 3, 2>(a, yf[q], E);
                    }
                    if (!LOCAL && p.err) {
                        float* to = p.err + (at * C + 16 * i + 4 * g) * p.Vp + col;
#pragma unroll
                        for (int r = 0; r < 4; ++r) to[r * p.Vp] = E[r];
                    }
                    U[i] = E * *reinterpret_cast<const f4*>(G.beta + 16 * i + 4 * g);
                }
                if constexpr (!LOCAL) {
#pragma unroll
                    for (int q = 0; q < NP; ++q) pack<D::OT>(U[2 * q], U[2 * q + 1], uf[q]);
                }
                u4 wf[NP][3];
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    pack<3>(U[2 * q] * *reinterpret_cast<const f4*>(G.end + 32 * q + 4 * g),
                            U[2 * q + 1] * *reinterpret_cast<const f4*>(G.end + 32 * q + 16 + 4 * g), wf[q]);
                const float total = G.total;
#pragma unroll
                for (int t = 0; t < NS; ++t) {
                    S[t] *= total;
#pragma unroll
                    for (int q = 0; q < NP; ++q) {
                        u4 a[KT];
                        frag_col<KT, KTERM, KST>(ks + 32 * q * KST, state_block(t, lane), lane, a);
                        mac<KT, 3, 2>(a, wf[q], S[t]);
                    }
                }
            }
            if constexpr (!LOCAL) {
                __syncthreads();                          // P is there
                if (live) {
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        O[i] *= G.gam[16 * i + c];
#pragma unroll
                        for (int q = 0; q <= i / 2; ++q) {
                            u4 b[PT];
                            frag44<PT, CTERM>(prob + (16 * i + c) * CST + 32 * q + 4 * g, b);
                            mac<D::OT, PT, D::OT - 1>(uf[q], b, O[i]);
                        }
                        const int64_t t = t0 + 16 * i + c;
                        const float o[4] = {p.scale * O[i][0], p.scale * O[i][1], p.scale * O[i][2], p.scale * O[i][3]};
                        if (t < head.len)
                            store4<T>(const_cast<T*>(head.rows<T>(p.o, t)) + col0 + 4 * g, o, p.V - (col0 + 4 * g));
                    }
                }
            }
        } else {
            if (live && !LOCAL) put_state(p.dstates + at * p.K * p.Vp + col, p.Vp, true);
            __syncthreads();                              // P is there
            if (live) {
                f4 X[NR];
#pragma unroll
                for (int i = 0; i < NR; ++i) X[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    u4 sf[3];
                    pack<3>(S[2 * kk], S[2 * kk + 1], sf);
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        u4 a[KT];
                        frag8<KT, KTERM>(ks + (16 * i + c) * KST + 32 * kk + 8 * g, a);
                        mac<KT, 3, 2>(a, sf, X[i]);
                    }
                }
                u4 df[NP][KT];
#pragma unroll
                for (int q = 0; q < NP; ++q) pack<KT>(x[2 * q], x[2 * q + 1], df[q]);
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int q = j / 2; q < NP; ++q) {
                        u4 a[PT];
                        frag_col<PT, CTERM, CST>(prob + 32 * q * CST, block16(j, lane), lane, a);
                        mac<PT, KT, 2>(a, df[q], acc);
                    }
                    const f4 end = *reinterpret_cast<const f4*>(G.end + 16 * j + 4 * g), beta = *reinterpret_cast<const f4*>(G.beta + 16 * j + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) X[j][r] = beta_or_least(beta[r]) * __builtin_fmaf(end[r], X[j][r], p.scale * acc[r]);
                }
                u4 xf[NP][3];
#pragma unroll
                for (int q = 0; q < NP; ++q) pack<3>(X[2 * q], X[2 * q + 1], xf[q]);
                f4 F[NR];
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    F[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int q = j / 2; q < NP; ++q) {
                        u4 a[3];
                        frag_col<3, CTERM, CST>(tri + 32 * q * CST, block16(j, lane), lane, a);
                        mac<3, 3, 2>(a, xf[q], F[j]);
                    }
                    if (!LOCAL) {
                        float* to = p.derr + (at * C + 16 * j + 4 * g) * p.Vp + col;
#pragma unroll
                        for (int r = 0; r < 4; ++r) to[r * p.Vp] = F[j][r];
                    }
                }
                u4 gf[NP][3], ff[NP][3];
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const f4 lo = *reinterpret_cast<const f4*>(G.gam + 32 * q + 4 * g), hi = *reinterpret_cast<const f4*>(G.gam + 32 * q + 16 + 4 * g);
                    pack<3>(x[2 * q] * (p.scale * lo), x[2 * q + 1] * (p.scale * hi), gf[q]);
                    pack<3>(-(F[2 * q] * lo), -(F[2 * q + 1] * hi), ff[q]);
                }
                const float total = G.total;
#pragma unroll
                for (int t = 0; t < NS; ++t) {
                    S[t] *= total;
#pragma unroll
                    for (int q = 0; q < NP; ++q) {
                        u4 a[KT];
                        frag_col<KT, KTERM, KST>(qs + 32 * q * KST, state_block(t, lane), lane, a);
                        mac<KT, 3, 2>(a, gf[q], S[t]);
                        frag_col<KT, KTERM, KST>(ks + 32 * q * KST, state_block(t, lane), lane, a);
                        mac<KT, 3, 2>(a, ff[q], S[t]);
                    }
                }
            }
        }
    }
    if constexpr (LOCAL) {
        float* to = unit ? p.seg_mul : p.seg_add;
        if (live) put_state(to + (head.bh * segs + seg) * p.K * pitch + col, pitch, col < pitch);
    } else {
        // the segment that the walk ends with: forward the one with the row's last token
        const int end = REV || chunks == 0 ? 0 : (chunks - 1) / p.seg_chunks;
        if (p.last && seg == end) put_state(p.last + head.bh * p.K * p.V + col, p.V, mine);
        if (!REV) {                                       // zero out past the row's tokens
            const int64_t from = head.len > int64_t(n0) * C ? head.len : int64_t(n0) * C, all = int64_t(n0 + p.seg_chunks) * C;
            const int64_t to = all < p.L ? all : p.L;
            for (int64_t t = from + w; t < to; t += 4)
                if (vt * 64 + lane < p.V) io<T>::store(const_cast<T*>(head.rows<T>(p.o, t)) + vt * 64 + lane, 0.f);
        }
    }
}

// ------------------------------------------------------------ gradients --
// The gradients of a chunk's tokens from S (before it), dS' (after it), E and F:
// with M_ij = F_i . E_j, R_ij = scale beta_j dO_i . E_j,
//
//   dq_i = scale exp(G_i) S dO_i + sum_{j <= i} w_ij R_ij k_j
//   dk_i = -exp(G_i) S F_i - sum_{j < i} w_ij beta_j M_ij k_j                      (i reads the state)
//        + sum_{j > i} w_ji (R_ji q_j - beta_i M_ji k_j) + R_ii q_i + beta_i exp(G_end - G_i) dS' E_i     (i writes it)
//   dv_i = F_i,   dbeta_i = M_ii / beta_i
//   dg_t = sum_{j < t <= i} w_ij (R_ij q_i . k_j - beta_j M_ij k_i . k_j)
//        + sum_{i >= t} exp(G_i) (scale q_i . S dO_i - k_i . S F_i) + sum_{j < t} beta_j exp(G_end - G_j) k_j . dS' E_j
//        + exp(G_end) <S, dS'>
//
// Every term of dg_t has the factor exp(g_t): nothing cancels that does not in the
// formula, and dg_t is zero where the decay empties the state.
//
// Waves 0 .. NR - 1 take 16 tokens each as readers (columns i of the transposed
// tiles), waves NR .. 2 NR - 1 as writers (columns j); the writer's share of dk passes
// to the reader through LDS.
template <typename T, int KP>
__global__ __launch_bounds__((kGradThreads<T, KP>)) void dr_grads(const DrParams p) {
    using D = Dims<T, KP>;
    constexpr int C = D::C, NR = D::NR, NP = D::NP, NK = D::NK, NS = D::NS, KT = D::KT, KST = D::KST, VST = D::VST, NTH = kGradThreads<T, KP>;
    constexpr int KTERM = C * KST, VTERM = C * VST, XT = D::OT;
    struct Rows { uint16_t e[3 * VTERM], f[3 * VTERM], d[KT * VTERM]; };
    __shared__ __attribute__((aligned(16))) uint16_t ks[KT * KTERM], qs[KT * KTERM];
    __shared__ __attribute__((aligned(16))) Rows rows;
    __shared__ Gates<C> gates;
    __shared__ float across[NR][C], reads[C], writes[C], inner[NR], dbeta[C];
    constexpr int HALF = KP > 128 ? 128 : KP;             // keys of dk that pass through LDS at a time
    static_assert(sizeof(Rows) >= sizeof(float) * C * (HALF + 4), "dk's share over the rows' tiles");
    const Head head(p, blockIdx.x / unsigned(p.nch));
    const int n = int(blockIdx.x % unsigned(p.nch));
    const int64_t t0 = int64_t(n) * C, at = head.bh * p.nch + n;
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const bool reader = wave < NR;
    const int w = reader ? wave : wave - NR, own = 16 * w + c;
    const int cnt = head.len - t0 < C ? int(head.len > t0 ? head.len - t0 : 0) : C;
    const int toks = p.L - t0 < C ? int(p.L - t0) : C;    // to be written
    // element (t, h, 0) of a contiguous (B, L, heads, dim) tensor
    const auto row_of = [&](int64_t t, int64_t heads, int64_t h, int dim) { return ((head.b * p.L + t) * heads + h) * dim; };
    const bool part = p.rep > 1;
    // 4 neighbouring elements of dq or dk
    const auto put_keys = [&](void* to, int64_t t, int key, const float (&v)[4]) {
        if (key >= p.K) return;
        if (part) store4<float>(static_cast<float*>(to) + row_of(t, p.H, head.h, p.K) + key, v, p.K - key);
        else store4<T>(static_cast<T*>(to) + row_of(t, p.H, head.h, p.K) + key, v, p.K - key);
    };
    if (cnt == 0) {                                       // (no token: every gradient is zero)
        const float none[4] = {0.f, 0.f, 0.f, 0.f};
        for (int t = wave; t < toks; t += NTH / 64) {
            put_keys(p.dq, t0 + t, 4 * lane, none);
            put_keys(p.dk, t0 + t, 4 * lane, none);
            if (4 * lane < p.V) store4<T>(static_cast<T*>(p.dv) + row_of(t0 + t, p.H, head.h, p.V) + 4 * lane, none, p.V - 4 * lane);
            if (lane == 0) p.dg[row_of(t0 + t, p.H, head.h, 1)] = p.dbeta[row_of(t0 + t, p.H, head.h, 1)] = 0.f;
        }
        return;
    }
    {
        Tile<T, KP, C, NTH> in;
        in.load(head.rows<T>(p.k, t0), p.k.l, cnt, p.K);
        if (wave == 0) {
            const bool on = lane < C;
            put_gates(gates, on ? head.g(p, t0 + lane) : 0.f, on ? head.beta(p, t0 + lane) : 0.f, lane);
        }
        in.store(ks);
        in.load(head.rows<T>(p.q, t0), p.q.l, cnt, p.K);
        in.store(qs);
    }
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 M[NR], R[NR], dq[NS], dk[NS];                      // reader: M, R transposed (rows j); writer: rows i, and no dq
#pragma unroll
    for (int i = 0; i < NR; ++i) M[i] = R[i] = zero;
#pragma unroll
    for (int t = 0; t < NS; ++t) dq[t] = dk[t] = zero;
    float z = 0.f;
    for (int v0 = 0; v0 < p.V; v0 += 64) {
        __syncthreads();
        {
            Tile<T, 64, C, NTH> in;
            static_assert(Tile<T, 64, C, NTH>::KST == VST, "the same rows");
            in.load(head.rows<T>(p.o, t0) + v0, p.o.l, cnt, p.V - v0);
            in.store(rows.d);
            // E and F: 16 vectors of 4 a row
#pragma unroll
            for (int i = 0; i < C * 16 / NTH; ++i) {
                const int e = tid + i * NTH, row = e >> 4, col = 4 * (e & 15);
                const bool on = v0 + col < p.Vp;
                const int64_t from = (at * C + row) * p.Vp + v0 + col;
                const f4 ev = on ? *reinterpret_cast<const f4*>(p.err + from) : zero, fv = on ? *reinterpret_cast<const f4*>(p.derr + from) : zero;
                uint32_t a[3], b[3], x[3], y[3];
                split<3>(ev[0], ev[1], a);
                split<3>(ev[2], ev[3], b);
                split<3>(fv[0], fv[1], x);
                split<3>(fv[2], fv[3], y);
#pragma unroll
                for (int m = 0; m < 3; ++m) {
                    *reinterpret_cast<uint2*>(rows.e + m * VTERM + row * VST + col) = make_uint2(a[m], b[m]);
                    *reinterpret_cast<uint2*>(rows.f + m * VTERM + row * VST + col) = make_uint2(x[m], y[m]);
                }
                if (row < toks && v0 + col < p.V) {
                    const bool is = row < cnt && gates.beta[row] != 0.f;
                    const float o[4] = {is ? fv[0] : 0.f, is ? fv[1] : 0.f, is ? fv[2] : 0.f, is ? fv[3] : 0.f};
                    store4<T>(static_cast<T*>(p.dv) + row_of(t0 + row, p.H, head.h, p.V) + v0 + col, o, p.V - (v0 + col));
                }
            }
        }
        __syncthreads();
        const int vks = p.Vp - v0 > 32 ? 2 : 1;
        for (int kk = 0; kk < vks; ++kk) {
            const int vcol = 32 * kk + 8 * g;
            // operand rows of the state at `s`: row state_row's m = c of tile t, 8 value columns
            const auto state_at = [&](const float* s, int t, f4& lo, f4& hi) {
                const int key = 32 * (t >> 1) + 8 * (c >> 2) + 4 * (t & 1) + (c & 3);
                const bool on = key < p.K && v0 + vcol < p.Vp;
                const float* from = s + (at * p.K + key) * p.Vp + v0 + vcol;
                lo = on ? *reinterpret_cast<const f4*>(from) : zero;
                hi = on ? *reinterpret_cast<const f4*>(from + 4) : zero;
            };
            if (reader) {
                u4 df[KT], ff[3];
                frag8<KT, VTERM>(rows.d + own * VST + vcol, df);
                frag8<3, VTERM>(rows.f + own * VST + vcol, ff);
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    if (j > w) continue;
                    u4 a[3];
                    frag8<3, VTERM>(rows.e + (16 * j + c) * VST + vcol, a);
                    mac<3, KT, 2>(a, df, R[j]);
                    mac<3, 3, 2>(a, ff, M[j]);
                }
#pragma unroll
                for (int t = 0; t < NS; ++t) {
                    f4 lo, hi;
                    u4 a[3];
                    state_at(p.states, t, lo, hi);
                    pack<3>(lo, hi, a);
                    mac<3, KT, 2>(a, df, dq[t]);
                    mac<3, 3, 2>(a, ff, dk[t]);
                }
            } else {
                u4 ef[3];
                frag8<3, VTERM>(rows.e + own * VST + vcol, ef);
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    if (i < w) continue;
                    u4 a[3], d[KT];
                    frag8<3, VTERM>(rows.f + (16 * i + c) * VST + vcol, a);
                    frag8<KT, VTERM>(rows.d + (16 * i + c) * VST + vcol, d);
                    mac<3, 3, 2>(a, ef, M[i]);
                    mac<KT, 3, 2>(d, ef, R[i]);
                }
#pragma unroll
                for (int t = 0; t < NS; ++t) {
                    f4 lo, hi;
                    u4 a[3];
                    state_at(p.dstates, t, lo, hi);
                    pack<3>(lo, hi, a);
                    mac<3, 3, 2>(a, ef, dk[t]);
                    if (t % NR == w) {
                        f4 slo, shi;
                        state_at(p.states, t, slo, shi);
#pragma unroll
                        for (int r = 0; r < 4; ++r) z = __builtin_fmaf(lo[r], slo[r], __builtin_fmaf(hi[r], shi[r], z));
                    }
                }
            }
        }
    }
    // 8 keys 32 a + 8 g .. of the own token, of a row tile
    const auto keys8 = [&](const uint16_t* tile, int a, float (&v)[8]) {
        u4 t[KT];
        frag8<KT, KTERM>(tile + own * KST + 32 * a + 8 * g, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = 0.f;
#pragma unroll
            for (int m = KT - 1; m >= 0; --m) v[e] += e & 1 ? hi_half(t[m][e >> 1]) : lo_half(t[m][e >> 1]);
        }
    };
    const auto groups_sum = [](float v) {                 // over the 4 lane groups
        v += __shfl_xor(v, 16, 64);
        return v + __shfl_xor(v, 32, 64);
    };
    const double Gown = gates.G[own];
    const float bown = gates.beta[own];
    u4 qf[NK][KT], kf[NK][KT];                            // the own tokens' rows as operands
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
        frag8<KT, KTERM>(qs + own * KST + 32 * kk + 8 * g, qf[kk]);
        frag8<KT, KTERM>(ks + own * KST + 32 * kk + 8 * g, kf[kk]);
    }
    if (reader) {
        const float gam = gates.gam[own];
        float r = 0.f;
#pragma unroll
        for (int a = 0; a < NK; ++a) {
            float qv[8], kv[8];
            keys8(qs, a, qv);
            keys8(ks, a, kv);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = dq[2 * a + (e >> 2)][e & 3] * (p.scale * gam), y = dk[2 * a + (e >> 2)][e & 3] * -gam;
                dq[2 * a + (e >> 2)][e & 3] = x;
                dk[2 * a + (e >> 2)][e & 3] = y;
                r = __builtin_fmaf(qv[e], x, __builtin_fmaf(kv[e], y, r));
            }
        }
        r = groups_sum(r);
        if (g == 0) reads[own] = r;
        float before = 0.f;                               // sum of the column's terms in earlier tiles
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            if (j > w) continue;
            f4 kq = zero, kk2 = zero;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                u4 a[KT];
                frag8<KT, KTERM>(ks + (16 * j + c) * KST + 32 * kk + 8 * g, a);
                mac<KT, KT, 2>(a, qf[kk], kq);
                mac<KT, KT, 2>(a, kf[kk], kk2);
            }
            const f4 beta = *reinterpret_cast<const f4*>(gates.beta + 16 * j + 4 * g);
            float term[4], sum = 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 16 * j + 4 * g + q;
                const float f = row <= own ? factor(Gown, gates.G[row]) : 0.f;
                if (row == own) dbeta[own] = M[j][q] / beta_or_least(bown);
                R[j][q] = row <= own ? f * (p.scale * beta[q]) * R[j][q] : 0.f;
                M[j][q] = row < own ? -f * beta[q] * M[j][q] : 0.f;
                term[q] = __builtin_fmaf(R[j][q], kq[q], M[j][q] * kk2[q]);
                sum += term[q];
            }
            // dg of token t, tile j's rows: the terms of earlier rows, over the columns i >= t
            float lead = __shfl_up(sum, 16, 64);
            lead = g >= 1 ? lead : 0.f;
            float two = __shfl_up(lead + sum, 32, 64);    // (groups g - 2 and g - 3)
            float pre = before + lead + (g >= 2 ? two : 0.f);
            before += groups_sum(sum);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 16 * j + 4 * g + q;
                const float all = lanes_sum<16>(row <= own ? pre : 0.f);
                if (c == 0) across[w][row] = all;
                pre += term[q];
            }
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if (2 * q > w) continue;
            u4 rf[XT], mf[XT];
            pack<XT>(R[2 * q], R[2 * q + 1], rf);
            pack<XT>(M[2 * q], M[2 * q + 1], mf);
#pragma unroll
            for (int t = 0; t < NS; ++t) {
                u4 a[KT];
                frag_col<KT, KTERM, KST>(ks + 32 * q * KST, state_block(t, lane), lane, a);
                mac<KT, XT, XT - 1>(a, rf, dq[t]);
                mac<KT, XT, XT - 1>(a, mf, dk[t]);
            }
        }
    } else {
        const float by = gates.end[own] * bown;
        float r = 0.f;
#pragma unroll
        for (int a = 0; a < NK; ++a) {
            float kv[8];
            keys8(ks, a, kv);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = dk[2 * a + (e >> 2)][e & 3] * by;
                dk[2 * a + (e >> 2)][e & 3] = y;
                r = __builtin_fmaf(kv[e], y, r);
            }
        }
        r = groups_sum(r);
        if (g == 0) writes[own] = r;
        z = lanes_sum<64>(z);
        if (lane == 0) inner[w] = z;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (i < w) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 16 * i + 4 * g + q;
                const float f = row >= own ? factor(gates.G[row], Gown) : 0.f;
                R[i][q] = row >= own ? f * (p.scale * bown) * R[i][q] : 0.f;
                M[i][q] = row > own ? -f * bown * M[i][q] : 0.f;
            }
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if (2 * q + 1 < w) continue;
            u4 rf[XT], mf[XT];
            pack<XT>(R[2 * q], R[2 * q + 1], rf);
            pack<XT>(M[2 * q], M[2 * q + 1], mf);
#pragma unroll
            for (int t = 0; t < NS; ++t) {
                u4 a[KT];
                frag_col<KT, KTERM, KST>(qs + 32 * q * KST, state_block(t, lane), lane, a);
                mac<KT, XT, XT - 1>(a, rf, dk[t]);
                frag_col<KT, KTERM, KST>(ks + 32 * q * KST, state_block(t, lane), lane, a);
                mac<KT, XT, XT - 1>(a, mf, dk[t]);
            }
        }
    }
    float* share = reinterpret_cast<float*>(&rows);       // (C, HALF + 4)
    const bool on = own < cnt;
#pragma unroll
    for (int k0 = 0; k0 < KP; k0 += HALF) {
        __syncthreads();                                  // (the rows' tiles, or the half before, are done with)
        if (!reader) {
#pragma unroll
            for (int t = k0 / 16; t < (k0 + HALF) / 16; ++t)
                *reinterpret_cast<f4*>(share + own * (HALF + 4) + state_row(t, g, 0) - k0) = dk[t];
        }
        __syncthreads();
        if (reader && own < toks) {
#pragma unroll
            for (int t = k0 / 16; t < (k0 + HALF) / 16; ++t) {
                const int key = state_row(t, g, 0);
                const f4 sum = dk[t] + *reinterpret_cast<const f4*>(share + own * (HALF + 4) + key - k0);
                const float a[4] = {on ? dq[t][0] : 0.f, on ? dq[t][1] : 0.f, on ? dq[t][2] : 0.f, on ? dq[t][3] : 0.f};
                const float b[4] = {on ? sum[0] : 0.f, on ? sum[1] : 0.f, on ? sum[2] : 0.f, on ? sum[3] : 0.f};
                put_keys(p.dq, t0 + own, key, a);
                put_keys(p.dk, t0 + own, key, b);
            }
        }
    }
    if (wave == 0) {                                      // (after the barriers above)
        const bool in = lane < C;
        float suffix = in ? reads[lane] : 0.f, lead = in ? writes[lane] : 0.f, sum = 0.f;
#pragma unroll
        for (int m = 1; m < C; m <<= 1) {
            const float x = __shfl_down(suffix, m, 64), y = __shfl_up(lead, m, 64);
            suffix += lane + m < 64 ? x : 0.f;
            lead += lane >= m ? y : 0.f;
        }
        lead = __shfl_up(lead, 1, 64);
        lead = lane > 0 ? lead : 0.f;
        if (in) {
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                sum += 16 * i + 15 >= lane ? across[i][lane] : 0.f;
                z = i == 0 ? inner[0] : z + inner[i];
            }
            sum += suffix + lead + gates.total * z;
            if (lane < toks) {
                const int64_t to = row_of(t0 + lane, p.H, head.h, 1);
                p.dg[to] = lane < cnt ? sum : 0.f;
                p.dbeta[to] = lane < cnt ? dbeta[lane] : 0.f;
            }
        }
    }
}

}  // namespace dr

template <typename T, typename F>
hipError_t dr_by_keys(int K, F&& f) {
    if (K <= 64) return f(std::integral_constant<int, 64>{});
    if (K <= 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

template <typename T>
hipError_t dr_prep_launch(const DrParams& p, hipStream_t stream) {
    return dr_by_keys<T>(p.K, [&](auto kp) {
        constexpr int KP = decltype(kp)::value;
        hipLaunchKernelGGL((dr::dr_prep<T, KP>), dim3(unsigned(p.B * p.H * p.nch)), dim3(dr::kPrepThreads<T, KP>), 0, stream, p);
        return hipGetLastError();
    });
}

template <typename T>
hipError_t dr_walk_launch(const DrParams& p, bool rev, hipStream_t stream) {
    const unsigned tiles = unsigned(p.V + 63) / 64, units = p.local && !rev ? unsigned(p.K + 63) / 64 : 0;
    const dim3 grid(unsigned(p.B * p.H * p.segs), tiles + units);
    return dr_by_keys<T>(p.K, [&](auto kp) {
        constexpr int KP = decltype(kp)::value;
        if (rev && p.local) hipLaunchKernelGGL((dr::dr_walk<T, KP, true, true>), grid, dim3(256), 0, stream, p);
        else if (rev) hipLaunchKernelGGL((dr::dr_walk<T, KP, true, false>), grid, dim3(256), 0, stream, p);
        else if (p.local) hipLaunchKernelGGL((dr::dr_walk<T, KP, false, true>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((dr::dr_walk<T, KP, false, false>), grid, dim3(256), 0, stream, p);
        return hipGetLastError();
    });
}

template <typename T>
hipError_t dr_grads_launch(const DrParams& p, hipStream_t stream) {
    return dr_by_keys<T>(p.K, [&](auto kp) {
        constexpr int KP = decltype(kp)::value;
        hipLaunchKernelGGL((dr::dr_grads<T, KP>), dim3(unsigned(p.B * p.H * p.nch)), dim3(dr::kGradThreads<T, KP>), 0, stream, p);
        return hipGetLastError();
    });
}

}  // namespace ss

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
// of the backward: then dbeta, the sum F . E over beta, keeps its value.  The token's own dv and
// dk, which have the factor beta, are scaled back (least_to_beta); what else F and M enter changes by 2^-60 of E.
constexpr float kLeastBeta = 8.673617379884035e-19f;      // 2^-60
__device__ __forceinline__ float beta_or_least(float b) { return fabsf(b) < kLeastBeta ? kLeastBeta : b; }
__device__ __forceinline__ float least_to_beta(float b) { return fabsf(b) < kLeastBeta ? b * (1.f / kLeastBeta) : 1.f; }

template <typename T, int KP>
struct Dims {
    static constexpr int KT = kTerms<T>, C = dr_chunk(KP, KT), NR = C / 16, NP = C / 32, NK = KP / 32, NS = KP / 16;
    static constexpr int NT = NR * (NR + 1) / 2;             // lower tiles of a chunk's square
    static constexpr int KST = KP + 8;                       // row stride of q and k in LDS, elements
    static constexpr int VST = sizeof(T) == 4 ? 68 : 72;     // of 64 value columns as they are
    // of out's rows on their way to memory (fp16: with 72, 272 bytes too many for two walks of 64 keys on a compute unit;
    // prompts of 24 heads of 64 x 64, 1 x 32768 tokens 543 us with one, 497 with two, 16 x 2048 390 and 304)
    static constexpr int OST = KT == 2 && KP == 64 ? 68 : VST;
    static constexpr int OT = sizeof(T) == 4 ? 3 : 2;        // terms of what only a result of type T is formed from
    // dr_grads: value columns and keys of the states that it takes at a time (tiles of q, k and these fill the LDS)
    static constexpr int VW = 32, KW = KP <= 128 ? KP : KT == 3 ? 64 : 128;
};
template <typename T, int KP> constexpr int kPrepThreads = 64 * Dims<T, KP>::NR;
// A walk's workgroup: 4 waves, 64 value columns; of the segments' own states 8, 4 of them the identity's columns.
// Waves a SIMD that it is compiled for: with 2 its results stay out of the accumulation registers, where
// vector instructions do not reach them, and two workgroups share a compute unit (dr_two: up to 64 keys, bf16 and fp32 up to 128;
// 1 x 32768 tokens x 24 heads of 64 x 64, bf16: 223 us to 170).  Wider tiles leave room for one.
template <bool REV, bool LOCAL> constexpr int kWalkThreads = LOCAL && !REV ? 512 : 256;
template <typename T, int KP> constexpr int kWalkWaves = dr_two(KP, kTerms<T>) ? 2 : 1;
// dr_grads: a wave takes its tokens in both roles where two such workgroups fit a compute unit's LDS (80 KB each:
// one is at its products while the other waits for its loads; 317 us to 218 with what came along)
template <typename T, int KP> constexpr bool kGradBoth = sizeof(T) == 2 && kTerms<T> == 1 && KP == 64;
template <typename T, int KP> constexpr int kGradThreads = (kGradBoth<T, KP> ? 64 : 128) * Dims<T, KP>::NR;

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
// 4 neighbouring elements in N term tiles TERM elements apart
template <int N, int TERM>
__device__ __forceinline__ void put4(uint16_t* to, const f4& x) {
    uint32_t a[N], b[N];
    split<N>(x[0], x[1], a);
    split<N>(x[2], x[3], b);
#pragma unroll
    for (int n = 0; n < N; ++n) *reinterpret_cast<uint2*>(to + n * TERM) = make_uint2(a[n], b[n]);
}

// Operands from N term tiles.  Of a row: 8 neighbouring elements.
template <int N, int TERM>
__device__ __forceinline__ void frag8(const uint16_t* at, u4 (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = *reinterpret_cast<const u4*>(at + n * TERM);
}
// Of a column (the transposing load): rows 4 g .. and 16 + 4 g .. of `at`, the order of two result tiles; or
// 8 neighbouring rows, 8 g ..
template <int N, int TERM, int STRIDE>
__device__ __forceinline__ void frag_col(const uint16_t* at, int block, int lane, u4 (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = load_tokens<STRIDE>(at + n * TERM, block, lane);
}
typedef __attribute__((address_space(3))) s4 lds_s4;
__device__ __forceinline__ u2 load_tr(const uint16_t* p) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
}
template <int N, int TERM, int STRIDE>
__device__ __forceinline__ void frag_col8(const uint16_t* at, int block, int lane, u4 (&t)[N]) {
    const uint16_t* p = at + (8 * (lane >> 4) + ((lane & 15) >> 2)) * STRIDE + block;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const u2 lo = load_tr(p + n * TERM), hi = load_tr(p + n * TERM + 4 * STRIDE);
        t[n] = u4{lo.x, lo.y, hi.x, hi.y};
    }
}
// Of two 16 x 16 tiles that lie as 256 elements each (a wave's reads of one are the whole of it, in
// order): a row of both, or with TR a column.  A tile below 0 is zero.
template <int N, int TERM, bool TR>
__device__ __forceinline__ void frag_tiles(const uint16_t* at, int lo, int hi, int lane, u4 (&t)[N]) {
    const int g = lane >> 4, c = lane & 15;
    const uint16_t* p = at + (TR ? 16 * (4 * g + (c >> 2)) + 4 * (c & 3) : 16 * c + 4 * g);
    const auto get = [&](int tile, int n) {
        if (tile < 0) return u2{0u, 0u};
        if constexpr (TR) return load_tr(p + n * TERM + tile * 256);
        else return *reinterpret_cast<const u2*>(p + n * TERM + tile * 256);
    };
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const u2 a = get(lo, n), b = get(hi, n);
        t[n] = u4{a.x, a.y, b.x, b.y};
    }
}
// f(integral_constant<0>), f(integral_constant<1>): the pairs of tiles of a chunk
template <int N, typename F>
__device__ __forceinline__ void each_pair(F&& f) {
    f(std::integral_constant<int, 0>{});
    if constexpr (N > 1) f(std::integral_constant<int, 1>{});
}
// place of the lower tile (i, j); none above the diagonal
constexpr __device__ __forceinline__ int tile_at(int i, int j) { return j <= i ? i * (i + 1) / 2 + j : -1; }
// first of the 4 columns a lane reads for its group: of 16 neighbouring ones, and of the state's tile t
__device__ __forceinline__ int block16(int t, int lane) { return 16 * t + 4 * (lane & 3); }
__device__ __forceinline__ int state_block(int t, int lane) { return 32 * (t >> 1) + 8 * (lane & 3) + 4 * (t & 1); }

// A chunk's rows (C x W of type T) from global memory by NTH threads: into term tiles, or as they are.
// WHOLE (dr_whole): rows of whole vectors, read through a buffer resource that ends with the last
// one: no branch, so nothing waits for the loads before they are stored.
template <typename T, int W, int C, int NTH, bool WHOLE>
struct Tile {
    using R = rowvec<T>;
    static constexpr int PER = W / R::VE, ALL = C * PER, N = (ALL + NTH - 1) / NTH, KT = kTerms<T>;
    uint4 v[N];
    // the first `rows` rows and `dim` columns; zero past them
    __device__ __forceinline__ void load(const T* p, int64_t step, int rows, int dim) {
        const int row = int(threadIdx.x) / PER, col = int(threadIdx.x) % PER * R::VE;
        if constexpr (WHOLE) {
            constexpr uint32_t es = sizeof(T), none = 0x80000000u;
            const rsrc_t r = make_rsrc_n(p, rows > 0 && dim > 0 ? int((uint32_t(rows - 1) * uint32_t(step) + uint32_t(dim)) * es) : 0);
            const uint32_t off = col < dim ? (uint32_t(row) * uint32_t(step) + uint32_t(col)) * es : none;
#pragma unroll
            for (int i = 0; i < N; ++i)
                v[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, int(off + uint32_t(i * (NTH / PER)) * uint32_t(step) * es), 0, 0));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row + i * (NTH / PER);
                v[i] = R::load(p + int64_t(r) * step + col, r < rows ? dim - col : 0);
            }
        }
    }
    template <int STRIDE>
    __device__ __forceinline__ void store(uint16_t* tile) const {
        static_assert(NTH % PER == 0, "rows of whole threads");
        uint16_t* to = tile + int(threadIdx.x) / PER * STRIDE + int(threadIdx.x) % PER * R::VE;
#pragma unroll
        for (int i = 0; i < N; ++i, to += NTH / PER * STRIDE) {
            if (ALL % NTH != 0 && int(threadIdx.x) + i * NTH >= ALL) continue;
            if constexpr (KT == 1) {
                *reinterpret_cast<uint4*>(to) = v[i];
            } else {
                float x[R::VE];
                R::unpack(v[i], x);
#pragma unroll
                for (int h = 0; h < R::VE; h += 4) put4<KT, C * STRIDE>(to + h, f4{x[h], x[h + 1], x[h + 2], x[h + 3]});
            }
        }
    }
    // a vector of a raw tile whose rows are STRIDE elements, whole vectors or halves of them
    template <int STRIDE>
    static __device__ __forceinline__ u4 read16(const T* at) {
        if constexpr (STRIDE * sizeof(T) % 16 == 0) return *reinterpret_cast<const u4*>(at);
        const u2 lo = reinterpret_cast<const u2*>(at)[0], hi = reinterpret_cast<const u2*>(at)[1];
        return u4{lo.x, lo.y, hi.x, hi.y};
    }
    // the first `rows` rows and `dim` columns of a raw tile to global memory
    template <int STRIDE>
    static __device__ __forceinline__ void put(T* p, int64_t step, const T* tile, int rows, int dim) {
        const int row = int(threadIdx.x) / PER, col = int(threadIdx.x) % PER * R::VE;
        const T* from = tile + row * STRIDE + col;
        if constexpr (WHOLE) {
            constexpr uint32_t es = sizeof(T), none = 0x80000000u;
            const rsrc_t r = make_rsrc_n(p, rows > 0 && dim > 0 ? int((uint32_t(rows - 1) * uint32_t(step) + uint32_t(dim)) * es) : 0);
            const uint32_t off = col < dim ? (uint32_t(row) * uint32_t(step) + uint32_t(col)) * es : none;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const u4 w = read16<STRIDE>(from + i * (NTH / PER) * STRIDE);
                __builtin_amdgcn_raw_buffer_store_b128(w, r, int(off + uint32_t(i * (NTH / PER)) * uint32_t(step) * es), 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float x[R::VE];
                R::unpack(__builtin_bit_cast(uint4, read16<STRIDE>(from + i * (NTH / PER) * STRIDE)), x);
                const int r = row + i * (NTH / PER);
                R::store(p + int64_t(r) * step + col, x, r < rows ? dim - col : 0);
            }
        }
    }
    template <int STRIDE>
    __device__ __forceinline__ void store_raw(T* tile) const {
        T* to = tile + int(threadIdx.x) / PER * STRIDE + int(threadIdx.x) % PER * R::VE;
#pragma unroll
        for (int i = 0; i < N; ++i, to += NTH / PER * STRIDE) {
            if (ALL % NTH != 0 && int(threadIdx.x) + i * NTH >= ALL) continue;
            *reinterpret_cast<uint4*>(to) = v[i];
        }
    }
};
// 32 rows of column `block16(t)` + c of a raw tile, in the order of two result tiles; and as an operand
template <typename T, int STRIDE>
__device__ __forceinline__ void raw_col(const T* at, int t, int lane, f4& lo, f4& hi, u4 (&f)[kTerms<T>]) {
    if constexpr (sizeof(T) == 2) {
        const u4 w = load_tokens<STRIDE>(reinterpret_cast<const uint16_t*>(at), block16(t, lane), lane);
        float x[8];
        rowvec<T>::unpack(make_uint4(w.x, w.y, w.z, w.w), x);
        lo = f4{x[0], x[1], x[2], x[3]};
        hi = f4{x[4], x[5], x[6], x[7]};
        if constexpr (kTerms<T> == 1) f[0] = w;
        else pack<kTerms<T>>(lo, hi, f);
    } else {
        const T* p = at + 4 * (lane >> 4) * STRIDE + 16 * t + (lane & 15);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            lo[r] = p[r * STRIDE];
            hi[r] = p[(16 + r) * STRIDE];
        }
        pack<kTerms<T>>(lo, hi, f);
    }
}

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
// factors of one token with 4 neighbouring ones: of it over them, or with OVER false of them over it
// (read before any of them is chosen: no branch per element)
template <bool OVER>
__device__ __forceinline__ f4 factors(double own, const double* four) {
    typedef double d2 __attribute__((ext_vector_type(2)));
    const d2 a = reinterpret_cast<const d2*>(four)[0], b = reinterpret_cast<const d2*>(four)[1];
    return OVER ? f4{factor(own, a[0]), factor(own, a[1]), factor(own, b[0]), factor(own, b[1])}
                : f4{factor(a[0], own), factor(a[1], own), factor(b[0], own), factor(b[1], own)};
}

// What dr_prep leaves of a chunk: its gates, and T's lower tiles in fp32, each transposed
// (element (row, column) of tile n at n * 256 + column * 16 + row).
template <typename T, int KP> struct Plan {
    Gates<Dims<T, KP>::C> gates;
    float tri[Dims<T, KP>::NT * 256];
};
template <typename T, int KP>
__device__ __forceinline__ Plan<T, KP>* plan_at(const DrParams& p, int64_t chunk) { return static_cast<Plan<T, KP>*>(p.plan) + chunk; }

struct Head {
    int64_t bh, b, h, group, len;          // len: the row's tokens
    __device__ __forceinline__ Head(const DrParams& p, uint32_t bh_) : bh(bh_) {
        const uint32_t heads = uint32_t(p.H), row = bh_ / heads, head = bh_ - row * heads;
        b = row;
        h = head;
        group = head / uint32_t(p.rep);
        const int64_t n = p.lens ? p.lens[b] : p.L;
        len = n < 0 ? 0 : n < p.L ? n : p.L;
    }
    // the head's (rep above 1: its group's) first row
    template <typename T> __device__ __forceinline__ const T* rows(const LaRows& r) const {
        return static_cast<const T*>(r.p) + b * r.b + (r.rep > 1 ? group : h) * r.h;
    }
};

// ------------------------------------------------------------- inverses --
// T of a chunk.  Wave i forms N's row of tiles and the inverse of its diagonal tile by
// substitution (16 steps, every lane a column); then wave j the tiles below its
// diagonal one, T_ij = -T_ii sum_{j <= m < i} N_im T_mj, on fp32 matrix instructions.
// Substitution and these products keep the bits of a stable solve, which powers of N
// would not: for equal keys they reach binomial coefficients.  12,288 chunks of 64 keys, bf16: 61 us, 240 MB
// at 3.9 TB/s (33 KB of LDS a workgroup in place of 14 and a branch for each factor: 115).
template <typename T, int KP, bool WHOLE>
__global__ __launch_bounds__((kPrepThreads<T, KP>)) void dr_prep(const DrParams p) {
    using D = Dims<T, KP>;
    constexpr int C = D::C, NR = D::NR, KT = D::KT, KST = D::KST, TERM = C * KST, NST = 20, NTH = kPrepThreads<T, KP>;
    // k, and over it N's lower tiles (rows of 16 + 4), the diagonal ones then their inverses
    union Lds { uint16_t k[KT * TERM]; float n[D::NT * 16 * NST]; };
    __shared__ __attribute__((aligned(16))) Lds lds;
    __shared__ __attribute__((aligned(16))) Gates<C> gates;
    uint16_t* const ks = lds.k;
    const auto tile = [&](int i, int j) { return lds.n + tile_at(i, j) * (16 * NST); };
    const Head head(p, blockIdx.x % uint32_t(p.BH));
    const int64_t n = blockIdx.x / uint32_t(p.BH), t0 = n * C;
    if (t0 >= head.len) return;
    const int lane = int(threadIdx.x) & 63, w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), g = lane >> 4, c = lane & 15;
    const int cnt = head.len - t0 < C ? int(head.len - t0) : C;
    Plan<T, KP>* plan = plan_at<T, KP>(p, blockIdx.x);
    {
        Tile<T, KP, C, NTH, WHOLE> k;
        k.load(head.rows<T>(p.k) + t0 * p.k.l, p.k.l, cnt, p.K);
        if (w == 0) {
            const bool in = lane < cnt;
            const float gv = in ? p.g[head.b * p.g_b + (t0 + lane) * p.g_l + head.h * p.g_h] : 0.f;
            put_gates(gates, gv, in ? p.beta[head.b * p.be_b + (t0 + lane) * p.be_l + head.h * p.be_h] : 0.f, lane);
        }
        k.template store<KST>(ks);
    }
    __syncthreads();
    for (int i = int(threadIdx.x); i < int(sizeof(Gates<C>) / 16); i += NTH)
        reinterpret_cast<uint4*>(&plan->gates)[i] = reinterpret_cast<const uint4*>(&gates)[i];
    // N's row of tiles, transposed: rows j, column i
    const double Gi = gates.G[16 * w + c];
    f4 x[NR];
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
        const f4 f = factors<true>(Gi, gates.G + 16 * j + 4 * g), beta = *reinterpret_cast<const f4*>(gates.beta + 16 * j + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = acc[r] * f[r] * beta_or_least(beta[r]);
            x[j][r] = 16 * j + 4 * g + r < 16 * w + c ? v : 0.f;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NR; ++j)
        if (j <= w) *reinterpret_cast<f4*>(tile(w, j) + c * NST + 4 * g) = x[j];
    __syncthreads();
    // the diagonal tile's inverse: column c, the rows of it
    float y[16];
    float* const own = tile(w, w);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float row[16];
#pragma unroll
        for (int j = 0; j < r; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(own + r * NST + j);
            row[j] = v.x; row[j + 1] = v.y; row[j + 2] = v.z; row[j + 3] = v.w;
        }
        float s0 = r == c ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < r; ++j) (j & 1 ? s1 : s0) = __builtin_fmaf(-row[j], y[j], j & 1 ? s1 : s0);
        y[r] = s0 + s1;
    }
    f4 t[NR];                                  // column w's tiles, from the diagonal one on
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float y0 = y[r], y1 = y[4 + r], y2 = y[8 + r], y3 = y[12 + r];
        const float lo = g & 1 ? y1 : y0, hi = g & 1 ? y3 : y2;
        t[0][r] = g & 2 ? hi : lo;
        own[(4 * g + r) * NST + c] = t[0][r];     // (of this wave's tile, which it has read)
    }
    __syncthreads();
    const auto mm = [&](const float* a, const f4& b, f4 acc) {       // a: 16 rows of this lane's, 4 summands from 4 g on
        const float4 v = *reinterpret_cast<const float4*>(a);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v.x, b[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v.y, b[1], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v.z, b[2], acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(v.w, b[3], acc, 0, 0, 0);
    };
#pragma unroll
    for (int d = 0; d < NR; ++d) {
        const int i = w + d;
        if (i >= NR) break;
        if (d > 0) {
            f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < d; ++m) acc = mm(tile(i, w + m) + c * NST + 4 * g, t[m], acc);
            t[d] = -mm(tile(i, i) + c * NST + 4 * g, acc, f4{0.f, 0.f, 0.f, 0.f});
        }
        *reinterpret_cast<f4*>(plan->tri + tile_at(i, w) * 256 + 16 * c + 4 * g) = t[d];
    }
}

// ----------------------------------------------------------------- walk --
// A chunk's plan on its way into LDS: the gates as they are, T in 3 terms.
template <typename T, int KP, int NTH>
struct PlanIn {
    using D = Dims<T, KP>;
    static constexpr int NG = sizeof(Gates<D::C>) / 16, N = (D::NT * 64 + NTH - 1) / NTH;
    static_assert(NG <= NTH && sizeof(Gates<D::C>) % 16 == 0, "a vector of the gates a thread");
    uint4 gates;
    f4 v[N];
    __device__ __forceinline__ void load(const Plan<T, KP>* p) {
        const int tid = int(threadIdx.x);
        // (a thread past the last vector reads it too)
        gates = reinterpret_cast<const uint4*>(&p->gates)[tid < NG ? tid : NG - 1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = tid + i * NTH;
            v[i] = *reinterpret_cast<const f4*>(p->tri + 4 * (at < D::NT * 64 ? at : D::NT * 64 - 1));
        }
    }
    __device__ __forceinline__ void store(Gates<D::C>& g, uint16_t* tri) const {
        const int tid = int(threadIdx.x);
        if (tid < NG) reinterpret_cast<uint4*>(&g)[tid] = gates;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (D::NT * 64 % NTH == 0 || i + 1 < N || tid + i * NTH < D::NT * 64) put4<3, D::NT * 256>(tri + 4 * (tid + i * NTH), v[i]);
    }
};

// The walk over the chunks of a segment (or of the whole row), forward (REV false) or back.
//
// Forward it writes out, the states and errors that a backward needs (unless null) and the
// last state; back, from dout, the states' and errors' gradients and the initial state's.
// LOCAL: the states only, from zero, and (forward) in 4 waves more what the segment makes of
// the columns of the identity: no values, the state starts as I.
//
// Bound by latency and issue.  8 x 2048 tokens x 24 heads of 64 x 64, bf16: 157 us forward, 166 back, 32 chunks of
// 4.9 us on 192 of the 256 compute units; a chunk is 1,105 instructions a wave, 124 of them matrix
// products, in sums that wait for each other (S to K S to E to U to S'); its bytes at the copy rate are 3.0 us.
// The next chunk's loads are issued as soon as this one's tiles are in LDS, barriers wait for LDS only,
// and stores of 64 bytes a lane group lie around the loads, never between them and their wait.  Two waves
// a column tile (half the rows each, joined through LDS) took 187 us for 172 then, fp16 of 128 keys 216 for 157, fp32 51
// for 62; one design was kept.
template <typename T, int KP, bool REV, bool LOCAL, bool WHOLE>
__global__ __launch_bounds__((kWalkThreads<REV, LOCAL>), (kWalkWaves<T, KP>)) void dr_walk(const DrParams p) {
    using D = Dims<T, KP>;
    constexpr int NTH = kWalkThreads<REV, LOCAL>;
    constexpr int C = D::C, NR = D::NR, NP = D::NP, NK = D::NK, NS = D::NS, KT = D::KT, KST = D::KST, NT = D::NT, VST = D::VST, OST = D::OST;
    constexpr int KTERM = C * KST, CTERM = NT * 256;
    constexpr int PT = REV ? 3 : D::OT;                   // P's terms
    constexpr bool Q = REV || !LOCAL;                     // whether q is read
    __shared__ __attribute__((aligned(16))) uint16_t ks[KT * KTERM], qs[Q ? KT * KTERM : 8], tri[3 * CTERM], prob[Q ? PT * CTERM : 8];
    __shared__ __attribute__((aligned(16))) T vs[C * VST], os[!REV && !LOCAL ? C * OST : 4];
    __shared__ __attribute__((aligned(16))) Gates<C> G;
    static_assert(!dr_two(KP, KT) || sizeof(ks) + sizeof(qs) + sizeof(tri) + sizeof(prob) + sizeof(vs) + sizeof(os) + sizeof(G) <= kTwoTiles,
                  "two workgroups' tiles in a compute unit's LDS");
    const int segs = p.segs, seg = int(blockIdx.x % unsigned(segs));
    // (nothing starts from the last segment's own state; a backward takes its M)
    if (LOCAL && seg == (REV ? 0 : segs - 1) && (REV || !p.states)) return;
    const Head head(p, blockIdx.x / uint32_t(segs));
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave & 3, g = lane >> 4, c = lane & 15;
    const bool unit = wave >= 4;                          // columns of the identity
    const int v0 = 64 * int(blockIdx.y), col0 = v0 + 16 * w, col = col0 + c;
    const bool live = col0 < (unit ? p.Kp : p.V), mine = !unit && col < p.V;
    const int chunks = int((head.len + C - 1) / C);       // of the row
    const int n0 = seg * p.seg_chunks, n1 = n0 + p.seg_chunks < chunks ? n0 + p.seg_chunks : chunks;
    const f4 zero = {0.f, 0.f, 0.f, 0.f};

    // the state: tile t, register r is row state_row(t, g, r), column col; 8 neighbouring rows a pair of tiles
    f4 S[NS];
#pragma unroll
    for (int t = 0; t < NS; ++t) S[t] = zero;
    if (unit) {
#pragma unroll
        for (int t = 0; t < NS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] = state_row(t, g, r) == col && col < p.K ? 1.f : 0.f;
    } else if (!LOCAL && segs > 1) {
        if (live) {
#pragma unroll
            for (int t = 0; t < NS; ++t)
                if (32 * (t >> 1) < p.Kp)
                    S[t] = *reinterpret_cast<const f4*>(p.seg_add + ((head.bh * segs + seg) * p.Vp + col) * p.Kp + 16 * t + 4 * g);
        }
    } else if (!LOCAL && p.init) {
#pragma unroll
        for (int t = 0; t < NS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = state_row(t, g, r);
                if (mine && key < p.K) S[t][r] = p.init[(head.bh * p.K + key) * p.V + col];
            }
    }
    // kept states: a column's rows side by side in the order of the tiles, so that a store covers 64 bytes of each
    const auto keep_state = [&](float* to) {
        float* at = to + col * p.Kp + 4 * g;
        if (KP == p.Kp) {
#pragma unroll
            for (int t = 0; t < NS; ++t) *reinterpret_cast<f4*>(at + 16 * t) = S[t];
            return;
        }
#pragma unroll
        for (int t = 0; t < NS; ++t)
            if (32 * (t >> 1) < p.Kp) *reinterpret_cast<f4*>(at + 16 * t) = S[t];
    };

    Tile<T, KP, C, NTH, WHOLE> kin, qin;
    Tile<T, 64, C, NTH, WHOLE> vin;                       // v (back: dout)
    PlanIn<T, KP, NTH> plan;
    const int step = REV ? -1 : 1, first = REV ? n1 - 1 : n0;
    T* const op = const_cast<T*>(head.rows<T>(p.o)) + v0;  // out (back: not written)
    const auto count = [&](int n) { return head.len - int64_t(n) * C < C ? int(head.len - int64_t(n) * C) : C; };
    const int64_t vstep = REV ? p.o.l : p.v.l;
    // the next chunk to fetch, and where its rows and plan are
    int next = first;
    const T* kp = head.rows<T>(p.k) + int64_t(first) * C * p.k.l;
    const T* qp = head.rows<T>(p.q) + int64_t(first) * C * p.q.l;
    const T* vp = head.rows<T>(REV ? p.o : p.v) + v0 + int64_t(first) * C * vstep;
    const Plan<T, KP>* pp = plan_at<T, KP>(p, first * p.BH + head.bh);
    const int64_t kstep = int64_t(step) * C * p.k.l, qstep = int64_t(step) * C * p.q.l, rstep = int64_t(step) * C * vstep;
    const auto fetch = [&] {
        const int cnt = count(next);
        plan.load(pp);
        kin.load(kp, p.k.l, cnt, p.K);
        if constexpr (Q) qin.load(qp, p.q.l, cnt, p.K);
        vin.load(vp, vstep, cnt, p.V - v0);
        if (next + step >= n0 && next + step < n1) {      // (past the last chunk: that one again)
            next += step;
            kp += kstep;
            qp += qstep;
            vp += rstep;
            pp += step * p.BH;
        }
    };
    // S += sum over 32 tokens of a tile's rows by the columns f, 4 tiles at a time
    const auto add_rows = [&](const uint16_t* rows, const u4 (&f)[1][3]) {
#pragma unroll
        for (int t = 0; t < NS; t += 4) {
            u4 a[4][KT];
            f4* to[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                frag_col<KT, KTERM, KST>(rows, state_block(t + i, lane), lane, a[i]);
                to[i] = &S[t + i];
            }
            mfma_terms<4, 1, 0, KT, 3, 2>(a, f, to);
        }
    };
    const auto stage = [&] {
        kin.template store<KST>(ks);
        if constexpr (Q) qin.template store<KST>(qs);
        vin.template store_raw<VST>(vs);
        plan.store(G, tri);
    };
    if (n0 < n1) {
        fetch();
        stage();
        lds_barrier();
    }
    for (int n = first; n >= n0 && n < n1; n += step) {
        const int64_t at = n * p.BH + head.bh, t0 = int64_t(n) * C;
        // Stores first and last: the loads of the next chunk then wait for no younger store.
        if (!LOCAL && live && (REV || p.states)) keep_state((REV ? p.dstates : p.states) + at * p.Vp * p.Kp);
        f4 kept[NR];                                      // E (back: F), column col
        fetch();
        if constexpr (Q) {                                // P, a share of its tiles a wave; formed transposed, rows j, column i
            // As many tiles side by side as their operands have registers for: all is read ahead of
            // the first product, else each product waits for its own reads.
            constexpr int TILES = (NT + 3) / 4, SIDE = NK * KT <= 2 ? TILES : 1;
#pragma unroll
            for (int e0 = 0; e0 < TILES; e0 += SIDE) {
                u4 a[SIDE][NK][KT], b[SIDE][NK][KT];
                double Gi[SIDE], Gj[SIDE][4];
                int tile[SIDE], row[SIDE], col_[SIDE];
#pragma unroll
                for (int e = 0; e < SIDE; ++e) {
                    // (past the last: that one again, the same values to the same place)
                    const int at_tile = w + 4 * (e0 + e);
                    tile[e] = at_tile < NT ? at_tile : NT - 1;
                    const int i = tile[e] < 1 ? 0 : tile[e] < 3 ? 1 : tile[e] < 6 ? 2 : 3, j = tile[e] - i * (i + 1) / 2;
                    row[e] = 16 * j + 4 * g;
                    col_[e] = 16 * i + c;
#pragma unroll
                    for (int kk = 0; kk < NK; ++kk) {
                        frag8<KT, KTERM>(ks + (16 * j + c) * KST + 32 * kk + 8 * g, a[e][kk]);
                        frag8<KT, KTERM>(qs + col_[e] * KST + 32 * kk + 8 * g, b[e][kk]);
                    }
                    Gi[e] = G.G[col_[e]];
#pragma unroll
                    for (int r = 0; r < 4; ++r) Gj[e][r] = G.G[row[e] + r];
                }
                if constexpr (SIDE > 1) stage_end();
                f4 acc[SIDE];
#pragma unroll
                for (int e = 0; e < SIDE; ++e) acc[e] = zero;
#pragma unroll
                for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                    for (int e = 0; e < SIDE; ++e) mac<KT, KT, 2>(a[e][kk], b[e][kk], acc[e]);
#pragma unroll
                for (int e = 0; e < SIDE; ++e) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float f = factor(Gi[e], Gj[e][r]);
                        acc[e][r] = row[e] + r <= col_[e] ? acc[e][r] * f : 0.f;
                    }
                    put4<PT, CTERM>(prob + tile[e] * 256 + 16 * c + 4 * g, acc[e]);
                }
            }
        }
        if constexpr (!REV) {
            f4 O[NR];                                     // out, transposed: rows value columns, column token i
            u4 uf[NP][D::OT];
            if (live) {
                f4 Y[NR];
#pragma unroll
                for (int i = 0; i < NR; ++i) Y[i] = O[i] = zero;
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    u4 sf[1][3], a[NR][KT];
                    pack<3>(S[2 * kk], S[2 * kk + 1], sf[0]);
                    f4* to[NR];
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        frag8<KT, KTERM>(ks + (16 * i + c) * KST + 32 * kk + 8 * g, a[i]);
                        to[i] = &Y[i];
                    }
                    mfma_terms<NR, 1, 0, KT, 3, 2>(a, sf, to);
                    if constexpr (!LOCAL) {
#pragma unroll
                        for (int i = 0; i < NR; ++i) {
                            frag8<KT, KTERM>(qs + (16 * i + c) * KST + 32 * kk + 8 * g, a[i]);
                            to[i] = &O[i];
                        }
                        mfma_terms<NR, 0, 1, 3, KT, D::OT - 1>(sf, a, to);
                    }
                }
                u4 yf[NP][3];
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    f4 lo, hi;
                    u4 raw[KT];
                    raw_col<T, VST>(vs + 32 * q * VST, w, lane, lo, hi, raw);
                    if (LOCAL && unit) lo = hi = zero;
                    const f4 glo = *reinterpret_cast<const f4*>(G.gam + 32 * q + 4 * g), ghi = *reinterpret_cast<const f4*>(G.gam + 32 * q + 16 + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        lo[r] = __builtin_fmaf(-glo[r], Y[2 * q][r], lo[r]);
                        hi[r] = __builtin_fmaf(-ghi[r], Y[2 * q + 1][r], hi[r]);
                    }
                    pack<3>(lo, hi, yf[q]);
                }
                f4 U[NR];
#pragma unroll
                for (int i = 0; i < NR; ++i) U[i] = zero;
                // (independent sums in turn: a product need not wait for the one before it)
                each_pair<NP>([&](auto qc) {
                    constexpr int q = decltype(qc)::value, I = NR - 2 * q;
                    u4 a[I][3];
                    f4* to[I];
#pragma unroll
                    for (int i = 0; i < I; ++i) {
                        frag_tiles<3, CTERM, true>(tri, tile_at(2 * q + i, 2 * q), tile_at(2 * q + i, 2 * q + 1), lane, a[i]);
                        to[i] = &U[2 * q + i];
                    }
                    mfma_terms<I, 1, 0, 3, 3, 2>(a, &yf[q], to);
                });
#pragma unroll
                for (int i = 0; i < NR; ++i) kept[i] = U[i];
#pragma unroll
                for (int i = 0; i < NR; ++i) U[i] *= *reinterpret_cast<const f4*>(G.beta + 16 * i + 4 * g);
                if constexpr (!LOCAL) {
#pragma unroll
                    for (int q = 0; q < NP; ++q) pack<D::OT>(U[2 * q], U[2 * q + 1], uf[q]);
                }
                const float total = G.total;
#pragma unroll
                for (int t = 0; t < NS; ++t) S[t] *= total;
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    u4 wf[1][3];
                    pack<3>(U[2 * q] * *reinterpret_cast<const f4*>(G.end + 32 * q + 4 * g),
                            U[2 * q + 1] * *reinterpret_cast<const f4*>(G.end + 32 * q + 16 + 4 * g), wf[0]);
                    add_rows(ks + 32 * q * KST, wf);
                }
            }
            if constexpr (!LOCAL) {
                lds_barrier();                            // P is there
                if (live) {
#pragma unroll
                    for (int i = 0; i < NR; ++i) O[i] *= G.gam[16 * i + c];
                    each_pair<NP>([&](auto qc) {
                        constexpr int q = decltype(qc)::value, I = NR - 2 * q;
                        u4 b[I][PT];
                        f4* to[I];
#pragma unroll
                        for (int i = 0; i < I; ++i) {
                            frag_tiles<PT, CTERM, false>(prob, tile_at(2 * q + i, 2 * q), tile_at(2 * q + i, 2 * q + 1), lane, b[i]);
                            to[i] = &O[2 * q + i];
                        }
                        mfma_terms<I, 0, 1, D::OT, PT, D::OT - 1>(&uf[q], b, to);
                    });
                }
                if (live) {                               // out's rows meet in LDS, to be stored whole
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        const float o[4] = {p.scale * O[i][0], p.scale * O[i][1], p.scale * O[i][2], p.scale * O[i][3]};
                        store4<T>(os + (16 * i + c) * OST + 16 * w + 4 * g, o, 4);
                    }
                }
                lds_barrier();                            // (the chunk's tiles are done with)
                stage();
                Tile<T, 64, C, NTH, WHOLE>::template put<OST>(op + t0 * p.o.l, p.o.l, os, count(n), p.V - v0);
            }
        } else {
            f4 X[NR];
            if (live) {
#pragma unroll
                for (int i = 0; i < NR; ++i) X[i] = zero;
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    u4 sf[1][3], a[NR][KT];
                    pack<3>(S[2 * kk], S[2 * kk + 1], sf[0]);
                    f4* to[NR];
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        frag8<KT, KTERM>(ks + (16 * i + c) * KST + 32 * kk + 8 * g, a[i]);
                        to[i] = &X[i];
                    }
                    mfma_terms<NR, 1, 0, KT, 3, 2>(a, sf, to);
                }
            }
            lds_barrier();                                // P is there
            if (live) {
                f4 x[NR];
                u4 df[NP][KT];
#pragma unroll
                for (int q = 0; q < NP; ++q) raw_col<T, VST>(vs + 32 * q * VST, w, lane, x[2 * q], x[2 * q + 1], df[q]);
                f4 acc[NR];
#pragma unroll
                for (int j = 0; j < NR; ++j) acc[j] = zero;
                each_pair<NP>([&](auto qc) {
                    constexpr int q = decltype(qc)::value, I = 2 * q + 2;
                    u4 a[I][PT];
                    f4* to[I];
#pragma unroll
                    for (int j = 0; j < I; ++j) {
                        frag_tiles<PT, CTERM, true>(prob, tile_at(2 * q, j), tile_at(2 * q + 1, j), lane, a[j]);
                        to[j] = &acc[j];
                    }
                    mfma_terms<I, 1, 0, PT, KT, 2>(a, &df[q], to);
                });
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    const f4 end = *reinterpret_cast<const f4*>(G.end + 16 * j + 4 * g), beta = *reinterpret_cast<const f4*>(G.beta + 16 * j + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) X[j][r] = beta_or_least(beta[r]) * __builtin_fmaf(end[r], X[j][r], p.scale * acc[j][r]);
                }
                u4 xf[NP][3];
#pragma unroll
                for (int q = 0; q < NP; ++q) pack<3>(X[2 * q], X[2 * q + 1], xf[q]);
                f4 F[NR];
#pragma unroll
                for (int j = 0; j < NR; ++j) F[j] = zero;
                each_pair<NP>([&](auto qc) {
                    constexpr int q = decltype(qc)::value, I = 2 * q + 2;
                    u4 a[I][3];
                    f4* to[I];
#pragma unroll
                    for (int j = 0; j < I; ++j) {
                        frag_tiles<3, CTERM, false>(tri, tile_at(2 * q, j), tile_at(2 * q + 1, j), lane, a[j]);
                        to[j] = &F[j];
                    }
                    mfma_terms<I, 1, 0, 3, 3, 2>(a, &xf[q], to);
                });
#pragma unroll
                for (int j = 0; j < NR; ++j) kept[j] = F[j];
                const float total = G.total;
#pragma unroll
                for (int t = 0; t < NS; ++t) S[t] *= total;
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const f4 lo = *reinterpret_cast<const f4*>(G.gam + 32 * q + 4 * g), hi = *reinterpret_cast<const f4*>(G.gam + 32 * q + 16 + 4 * g);
                    u4 gf[1][3], ff[1][3];
                    pack<3>(x[2 * q] * (p.scale * lo), x[2 * q + 1] * (p.scale * hi), gf[0]);
                    add_rows(qs + 32 * q * KST, gf);
                    pack<3>(-(F[2 * q] * lo), -(F[2 * q + 1] * hi), ff[0]);
                    add_rows(ks + 32 * q * KST, ff);
                }
            }
        }
        if constexpr (REV || LOCAL) {
            lds_barrier();                                // (the chunk's tiles are done with)
            stage();
        }
        float* const err = REV ? p.derr : p.err;
        if (!LOCAL && live && err) {                      // (value column, token)
            float* to = err + (at * p.Vp + col) * C + 4 * g;
#pragma unroll
            for (int i = 0; i < NR; ++i) *reinterpret_cast<f4*>(to + 16 * i) = kept[i];
        }
        lds_barrier();
    }
    if constexpr (LOCAL) {
        if (live && unit) {                               // in the terms and the order that dr_join takes it in
            uint16_t* to = p.seg_mul + ((head.bh * segs + seg) * 3 * p.Kp + col) * p.Kp + 8 * g;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                if (32 * k >= p.Kp) continue;
                u4 t[3];
                pack<3>(S[2 * k], S[2 * k + 1], t);
#pragma unroll
                for (int i = 0; i < 3; ++i) *reinterpret_cast<u4*>(to + int64_t(i) * p.Kp * p.Kp + 32 * k) = t[i];
            }
        } else if (live) keep_state(p.seg_add + (head.bh * segs + seg) * p.Vp * p.Kp);
    } else {
        // the segment that the walk ends with: forward the one with the row's last token
        const int end = REV || chunks == 0 ? 0 : (chunks - 1) / p.seg_chunks;
        if (p.last && seg == end && mine) {
#pragma unroll
            for (int t = 0; t < NS; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = state_row(t, g, r);
                    if (key < p.K) p.last[(head.bh * p.K + key) * p.V + col] = S[t][r];
                }
        }
        if (!REV) {                                       // zero out past the row's tokens
            const int64_t from = head.len > int64_t(n0) * C ? head.len : int64_t(n0) * C, all = int64_t(n0 + p.seg_chunks) * C;
            const int64_t to = all < p.L ? all : p.L;
            for (int64_t t = from + w; t < to; t += 4)
                if (v0 + lane < p.V) io<T>::store(op + t * p.o.l + lane, 0.f);
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
// Waves 0 .. NR - 1 take 16 tokens each as readers (columns i of the transposed tiles: w + 1 tiles
// of M and R) and waves NR .. 2 NR - 1 as writers (columns j: the other NR - w), whose share of dk
// passes to the reader through LDS; or (kGradBoth) a wave is both for its tokens.  Value columns
// pass 32 at a time, those of the next step on their way meanwhile.
//
// 8 x 2048 tokens x 24 heads of 64 x 64, bf16 (6,144 chunks): 198 us, 690 MB at 3.5 TB/s; 2 x 4096 x 16 heads of 128 x 128,
// fp16 (2,048): 234 us, 590 MB at 2.5.  Both at two waves a SIMD; workgroups that go from chunk to chunk, the next one's
// loads in registers, took 279 and 245: what the loop shares spills.
template <typename T, int KP, bool WHOLE>
__global__ __launch_bounds__((kGradThreads<T, KP>), (kGradThreads<T, KP> > 256 || kGradBoth<T, KP> ? 2 : 1)) void dr_grads(const DrParams p) {
    using D = Dims<T, KP>;
    constexpr int C = D::C, NR = D::NR, NP = D::NP, NK = D::NK, NS = D::NS, KT = D::KT, KST = D::KST, NTH = kGradThreads<T, KP>, NW = NTH / 64;
    constexpr bool BOTH = kGradBoth<T, KP>;
    constexpr int VW = D::VW, KW = D::KW, SST = KW + 8, EST = C + 8, DST = VW + 8, XT = D::OT;
    constexpr int KTERM = C * KST, STERM = VW * SST, ETERM = VW * EST, DTERM = C * DST;
    // S, dS' (rows value columns, columns keys), E, F (columns tokens), dout (rows tokens)
    struct Stage { uint16_t s[3 * STERM], t[3 * STERM], e[3 * ETERM], f[3 * ETERM], d[KT * DTERM]; };
    __shared__ __attribute__((aligned(16))) uint16_t ks[KT * KTERM], qs[KT * KTERM];
    __shared__ __attribute__((aligned(16))) Stage st;
    __shared__ __attribute__((aligned(16))) Gates<C> gates;
    __shared__ __attribute__((aligned(16))) float across[NR][C], reads[C], writes[C], inner[NW];
    constexpr int HALF = KP > 128 ? 128 : KP;             // keys of dk that pass through LDS at a time
    static_assert(sizeof(Stage) >= sizeof(float) * C * (HALF + 4), "dk's share over the tiles");
    const int tid = int(threadIdx.x);
    const bool part = p.rep > 1;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const bool reader = BOTH || wave < NR, writer = BOTH || wave >= NR;
    const int w = wave < NR ? wave : wave - NR, own = 16 * w + c;
    const Head head(p, blockIdx.x % uint32_t(p.BH));
    const int64_t n = blockIdx.x / uint32_t(p.BH), t0 = n * C, at = blockIdx.x;
    const int cnt = head.len - t0 < C ? int(head.len > t0 ? head.len - t0 : 0) : C;
    const int toks = p.L - t0 < C ? int(p.L - t0) : C;    // to be written
    // token t's row of a contiguous (B, L, heads, dim) tensor
    const auto row_of = [&](int t, int dim) { return ((head.b * p.L + t0 + t) * p.H + head.h) * dim; };
    // 8 neighbouring elements of a row of type O, those below dim
    const auto put8 = [&](auto* row, int from, int dim, const f4& lo, const f4& hi) {
        using O = std::remove_pointer_t<decltype(row)>;
        using R = rowvec<O>;
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
        for (int h = 0; h < 8; h += R::VE) {
            float x[R::VE];
#pragma unroll
            for (int e = 0; e < R::VE; ++e) x[e] = v[h + e];
            if (!WHOLE) R::store(row + from + h, x, dim - (from + h));
            else if (from + h < dim) R::store(row + from + h, x, R::VE);
        }
    };
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    // a step: VW value columns of E, F and dout (with the first of its states' keys), KW keys of S and dS'
    constexpr int NSV = VW * KW / 4 / NTH, NEV = VW * C / 4 / NTH;
    static_assert(VW * KW / 4 % NTH == 0 && VW * C / 4 % NTH == 0, "whole vectors a thread");
    f4 si[NSV], ti[NSV], ei[NEV], fi[NEV];
    Tile<T, VW, C, NTH, WHOLE> di;
    const auto fetch = [&](int v0, int k0) {
#pragma unroll
        for (int i = 0; i < NSV; ++i) {
            const int x = tid + i * NTH, v = v0 + x / (KW / 4), place = k0 + x % (KW / 4) * 4;
            const bool in = v < p.Vp && place < p.Kp;
            const int64_t from = (at * p.Vp + v) * p.Kp + place;
            si[i] = in ? *reinterpret_cast<const f4*>(p.states + from) : zero;
            ti[i] = in ? *reinterpret_cast<const f4*>(p.dstates + from) : zero;
        }
        if (k0 > 0) return;
#pragma unroll
        for (int i = 0; i < NEV; ++i) {
            const int x = tid + i * NTH, v = v0 + x / (C / 4);
            const int64_t from = (at * p.Vp + v) * C + x % (C / 4) * 4;
            ei[i] = v < p.Vp ? *reinterpret_cast<const f4*>(p.err + from) : zero;
            fi[i] = v < p.Vp ? *reinterpret_cast<const f4*>(p.derr + from) : zero;
        }
        di.load(head.rows<T>(p.o) + t0 * p.o.l + v0, p.o.l, cnt, p.V - v0);
    };
    T* const dq_rows = static_cast<T*>(p.dq) + row_of(0, p.K);
    T* const dk_rows = static_cast<T*>(p.dk) + row_of(0, p.K);
    T* const dv_rows = static_cast<T*>(p.dv) + row_of(0, p.V);
    if (cnt == 0) {                                       // (no token: every gradient is zero)
        for (int t = wave; t < toks; t += NTH / 64) {
            if (8 * lane < p.K) {
                if (part) {
                    put8(static_cast<float*>(p.dq) + row_of(t, p.K), 8 * lane, p.K, zero, zero);
                    put8(static_cast<float*>(p.dk) + row_of(t, p.K), 8 * lane, p.K, zero, zero);
                } else {
                    put8(static_cast<T*>(p.dq) + row_of(t, p.K), 8 * lane, p.K, zero, zero);
                    put8(static_cast<T*>(p.dk) + row_of(t, p.K), 8 * lane, p.K, zero, zero);
                }
            }
            if (8 * lane < p.V) put8(static_cast<T*>(p.dv) + row_of(t, p.V), 8 * lane, p.V, zero, zero);
            if (lane == 0) p.dg[row_of(t, 1)] = p.dbeta[row_of(t, 1)] = 0.f;
        }
        return;
    }
    // its q, k, gates and first step
    fetch(0, 0);
    {
        Tile<T, KP, C, NTH, WHOLE> kin, qin;
        kin.load(head.rows<T>(p.k) + t0 * p.k.l, p.k.l, cnt, p.K);
        qin.load(head.rows<T>(p.q) + t0 * p.q.l, p.q.l, cnt, p.K);
        if (tid < int(sizeof(Gates<C>) / 16))
            reinterpret_cast<uint4*>(&gates)[tid] = reinterpret_cast<const uint4*>(&plan_at<T, KP>(p, at)->gates)[tid];
        kin.template store<KST>(ks);
        qin.template store<KST>(qs);
    }
    // reader: M, R transposed (rows j); writer: rows i, and no dq
    f4 Ms[1 + BOTH][NR], Rs[1 + BOTH][NR], dq[NS], dks[1 + BOTH][NS];
#pragma unroll
    for (int b = 0; b <= BOTH; ++b) {
#pragma unroll
        for (int i = 0; i < NR; ++i) Ms[b][i] = Rs[b][i] = zero;
#pragma unroll
        for (int t = 0; t < NS; ++t) dq[t] = dks[b][t] = zero;
    }
    float z = 0.f;
    for (int v0 = 0; v0 < p.V; v0 += VW) {
#pragma unroll
        for (int k0 = 0; k0 < KP; k0 += KW) {
            lds_barrier();
#pragma unroll
            for (int i = 0; i < NSV; ++i) {
                const int x = tid + i * NTH, to = x / (KW / 4) * SST + state_key(x % (KW / 4) * 4);
                put4<3, STERM>(st.s + to, si[i]);
                put4<3, STERM>(st.t + to, ti[i]);
#pragma unroll
                for (int r = 0; r < 4; ++r) z = __builtin_fmaf(si[i][r], ti[i][r], z);
            }
            if (k0 == 0) {
#pragma unroll
                for (int i = 0; i < NEV; ++i) {
                    const int x = tid + i * NTH, to = x / (C / 4) * EST + x % (C / 4) * 4;
                    put4<3, ETERM>(st.e + to, ei[i]);
                    put4<3, ETERM>(st.f + to, fi[i]);
                }
                di.template store<DST>(st.d);
            }
            lds_barrier();
            if (k0 + KW < KP) fetch(v0, k0 + KW);
            else if (v0 + VW < p.V) fetch(v0 + VW, 0);
            if (reader) {
                f4 (&M)[NR] = Ms[0], (&R)[NR] = Rs[0], (&dk)[NS] = dks[0];
                u4 df[KT], ff[3];
                frag8<KT, DTERM>(st.d + own * DST + 8 * g, df);
                frag_col8<3, ETERM, EST>(st.f, block16(w, lane), lane, ff);
                if (k0 == 0) {
#pragma unroll
                    for (int j = 0; j < NR; j += 2) {     // (two tiles side by side: the one past w is masked below)
                        if (j > w) continue;
                        u4 a[2][3];
                        f4* const r2[2] = {&R[j], &R[j + 1]};
                        f4* const m2[2] = {&M[j], &M[j + 1]};
                        frag_col8<3, ETERM, EST>(st.e, block16(j, lane), lane, a[0]);
                        frag_col8<3, ETERM, EST>(st.e, block16(j + 1, lane), lane, a[1]);
                        mfma_terms<2, 1, 0, 3, KT, 2>(a, &df, r2);
                        mfma_terms<2, 1, 0, 3, 3, 2>(a, &ff, m2);
                    }
                    if (own < toks && v0 + 8 * g < p.V) { // dv: F of the own token
                        const uint32_t is = own < cnt && gates.beta[own] != 0.f ? ~0u : 0u;
                        const float to_beta = least_to_beta(gates.beta[own]);
                        f4 x[2];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const auto half = [&](const u4& t) { return e & 1 ? hi_half(t[e >> 1]) : lo_half(t[e >> 1]); };
                            x[e >> 2][e & 3] = __builtin_bit_cast(float, is & __builtin_bit_cast(uint32_t, to_beta * (half(ff[0]) + (half(ff[1]) + half(ff[2])))));
                        }
                        put8(dv_rows + int64_t(own) * p.H * p.V, v0 + 8 * g, p.V, x[0], x[1]);
                    }
                }
#pragma unroll
                for (int t = k0 / 16; t < (k0 + KW) / 16; t += 2) {
                    u4 a[2][3];
                    f4* const q2[2] = {&dq[t], &dq[t + 1]};
                    f4* const k2[2] = {&dk[t], &dk[t + 1]};
                    frag_col8<3, STERM, SST>(st.s - k0, state_block(t, lane), lane, a[0]);
                    frag_col8<3, STERM, SST>(st.s - k0, state_block(t + 1, lane), lane, a[1]);
                    mfma_terms<2, 1, 0, 3, KT, 2>(a, &df, q2);
                    mfma_terms<2, 1, 0, 3, 3, 2>(a, &ff, k2);
                }
            }
            if (writer) {
                f4 (&M)[NR] = Ms[BOTH], (&R)[NR] = Rs[BOTH], (&dk)[NS] = dks[BOTH];
                u4 ef[3];
                frag_col8<3, ETERM, EST>(st.e, block16(w, lane), lane, ef);
                if (k0 == 0) {
#pragma unroll
                    for (int i = 0; i < NR; i += 2) {
                        if (i + 1 < w) continue;
                        u4 a[2][3], d[2][KT];
                        f4* const r2[2] = {&R[i], &R[i + 1]};
                        f4* const m2[2] = {&M[i], &M[i + 1]};
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            frag_col8<3, ETERM, EST>(st.f, block16(i + e, lane), lane, a[e]);
                            frag8<KT, DTERM>(st.d + (16 * (i + e) + c) * DST + 8 * g, d[e]);
                        }
                        mfma_terms<2, 1, 0, 3, 3, 2>(a, &ef, m2);
                        mfma_terms<2, 1, 0, KT, 3, 2>(d, &ef, r2);
                    }
                }
#pragma unroll
                for (int t = k0 / 16; t < (k0 + KW) / 16; t += 2) {
                    u4 a[2][3];
                    f4* const k2[2] = {&dk[t], &dk[t + 1]};
                    frag_col8<3, STERM, SST>(st.t - k0, state_block(t, lane), lane, a[0]);
                    frag_col8<3, STERM, SST>(st.t - k0, state_block(t + 1, lane), lane, a[1]);
                    mfma_terms<2, 1, 0, 3, 3, 2>(a, &ef, k2);
                }
            }
        }
    }
    z = lanes_sum<64>(z);
    if (lane == 0) inner[wave] = z;
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
    if (reader) {
        f4 (&M)[NR] = Ms[0], (&R)[NR] = Rs[0], (&dk)[NS] = dks[0];
        const float gam = gates.gam[own], to_beta = least_to_beta(bown);
        float r = 0.f;
#pragma unroll
        for (int a = 0; a < NK; ++a) {
            float qv[8], kv[8];
            keys8(qs, a, qv);
            keys8(ks, a, kv);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = dq[2 * a + (e >> 2)][e & 3] * (p.scale * gam), y = dk[2 * a + (e >> 2)][e & 3] * (-gam * to_beta);
                dq[2 * a + (e >> 2)][e & 3] = x;
                dk[2 * a + (e >> 2)][e & 3] = y;
                r = __builtin_fmaf(qv[e], x, __builtin_fmaf(kv[e], y, r));
            }
        }
        r = groups_sum(r);
        if (g == 0) reads[own] = r;
        float before = 0.f, diag = 0.f;                   // sum of the column's terms in earlier tiles; M_ii
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            if (j > w) {
                R[j] = M[j] = zero;
                continue;
            }
            f4 kq = zero, kk2 = zero;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                u4 a[1][KT], b[2][KT];
                f4* const to[2] = {&kq, &kk2};
                frag8<KT, KTERM>(ks + (16 * j + c) * KST + 32 * kk + 8 * g, a[0]);
                frag8<KT, KTERM>(qs + own * KST + 32 * kk + 8 * g, b[0]);
                frag8<KT, KTERM>(ks + own * KST + 32 * kk + 8 * g, b[1]);
                mfma_terms<2, 0, 1, KT, KT, 2>(a, b, to);
            }
            const f4 beta = *reinterpret_cast<const f4*>(gates.beta + 16 * j + 4 * g);
            const f4 fs = factors<true>(Gown, gates.G + 16 * j + 4 * g);
            float term[4], sum = 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 16 * j + 4 * g + q;
                diag = row == own ? M[j][q] : diag;
                const float rv = fs[q] * (p.scale * beta[q]) * R[j][q], mv = -fs[q] * (to_beta * beta[q]) * M[j][q];
                R[j][q] = row <= own ? rv : 0.f;
                M[j][q] = row < own ? mv : 0.f;
                term[q] = __builtin_fmaf(R[j][q], kq[q], M[j][q] * kk2[q]);
                sum += term[q];
            }
            // dg of token t, tile j's rows: the terms of earlier rows, over the columns i >= t
            float lead = __shfl_up(sum, 16, 64);
            lead = g >= 1 ? lead : 0.f;
            const float two = __shfl_up(lead + sum, 32, 64);    // (groups g - 2 and g - 3)
            float pre = before + lead + (g >= 2 ? two : 0.f);
            before += groups_sum(sum);
            f4 all;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                all[q] = lanes_sum<16>(16 * j + 4 * g + q <= own ? pre : 0.f);
                pre += term[q];
            }
            if (c == 0) *reinterpret_cast<f4*>(&across[w][16 * j + 4 * g]) = all;
        }
        if (c >> 2 == g && own < toks) p.dbeta[row_of(own, 1)] = own < cnt ? diag / beta_or_least(bown) : 0.f;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if (2 * q > w) continue;
            u4 rf[XT], mf[XT];
            pack<XT>(R[2 * q], R[2 * q + 1], rf);
            pack<XT>(M[2 * q], M[2 * q + 1], mf);
#pragma unroll
            for (int t = 0; t < NS; ++t) {
                u4 a[1][KT], b[2][XT];
                f4* const to[2] = {&dq[t], &dk[t]};
                frag_col<KT, KTERM, KST>(ks + 32 * q * KST, state_block(t, lane), lane, a[0]);
#pragma unroll
                for (int n = 0; n < XT; ++n) b[0][n] = rf[n], b[1][n] = mf[n];
                mfma_terms<2, 0, 1, KT, XT, XT - 1>(a, b, to);
            }
        }
    }
    if (writer) {
        f4 (&M)[NR] = Ms[BOTH], (&R)[NR] = Rs[BOTH], (&dk)[NS] = dks[BOTH];
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
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (i < w) {
                R[i] = M[i] = zero;
                continue;
            }
            const f4 fs = factors<false>(Gown, gates.G + 16 * i + 4 * g);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 16 * i + 4 * g + q;
                const float rv = fs[q] * (p.scale * bown) * R[i][q], mv = -fs[q] * bown * M[i][q];
                R[i][q] = row >= own ? rv : 0.f;
                M[i][q] = row > own ? mv : 0.f;
            }
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            if (2 * q + 1 < w) continue;
            u4 rf[XT], mf[XT];
            pack<XT>(R[2 * q], R[2 * q + 1], rf);
            pack<XT>(M[2 * q], M[2 * q + 1], mf);
#pragma unroll
            for (int t = 0; t < NS; t += 2) {
                u4 a[2][KT], b[2][KT];
                f4* const to[2] = {&dk[t], &dk[t + 1]};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    frag_col<KT, KTERM, KST>(qs + 32 * q * KST, state_block(t + e, lane), lane, a[e]);
                    frag_col<KT, KTERM, KST>(ks + 32 * q * KST, state_block(t + e, lane), lane, b[e]);
                }
                mfma_terms<2, 1, 0, KT, XT, XT - 1>(a, &rf, to);
                mfma_terms<2, 1, 0, KT, XT, XT - 1>(b, &mf, to);
            }
        }
    }
    float* share = reinterpret_cast<float*>(&st);         // (C, HALF + 4)
    T* const q_out = reinterpret_cast<T*>(qs);            // dq and dk in the rows' type, over q and k
    T* const k_out = reinterpret_cast<T*>(ks);
    const bool on = own < cnt;
#pragma unroll
    for (int k0 = 0; k0 < KP; k0 += HALF) {
        lds_barrier();                                    // (the tiles, or the half before, are done with)
        if constexpr (!BOTH) {
            if (writer) {
#pragma unroll
                for (int t = k0 / 16; t < (k0 + HALF) / 16; ++t)
                    *reinterpret_cast<f4*>(share + own * (HALF + 4) + state_row(t, g, 0) - k0) = dks[0][t];
            }
            lds_barrier();
        }
        if (reader) {
#pragma unroll
            for (int t = k0 / 16; t < (k0 + HALF) / 16; t += 2) {
                const int key = state_row(t, g, 0);
                f4 lo = dks[0][t], hi = dks[0][t + 1];
                if constexpr (BOTH) {
                    lo += dks[BOTH][t];
                    hi += dks[BOTH][t + 1];
                } else {
                    const float* with = share + own * (HALF + 4) + key - k0;
                    lo += *reinterpret_cast<const f4*>(with);
                    hi += *reinterpret_cast<const f4*>(with + 4);
                }
                if (!on) lo = hi = dq[t] = dq[t + 1] = zero;
                if (!part) {
                    put8(q_out + own * KST, key, KP, dq[t], dq[t + 1]);
                    put8(k_out + own * KST, key, KP, lo, hi);
                } else if (own < toks && key < p.K) {
                    put8(static_cast<float*>(p.dq) + row_of(own, p.K), key, p.K, dq[t], dq[t + 1]);
                    put8(static_cast<float*>(p.dk) + row_of(own, p.K), key, p.K, lo, hi);
                }
            }
        }
    }
    if (!part) {
        lds_barrier();
        Tile<T, KP, C, NTH, WHOLE>::template put<KST>(dq_rows, p.H * p.K, q_out, toks, p.K);
        Tile<T, KP, C, NTH, WHOLE>::template put<KST>(dk_rows, p.H * p.K, k_out, toks, p.K);
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
            z = 0.f;
#pragma unroll
            for (int i = 0; i < NR; ++i) sum += 16 * i + 15 >= lane ? across[i][lane] : 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) z += inner[i];
            sum += suffix + lead + gates.total * z;
            if (lane < toks) p.dg[row_of(lane, 1)] = lane < cnt ? sum : 0.f;
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
        const dim3 grid(unsigned(p.B * p.H * p.nch)), block(dr::kPrepThreads<T, KP>);
        if (p.whole) hipLaunchKernelGGL((dr::dr_prep<T, KP, true>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((dr::dr_prep<T, KP, false>), grid, block, 0, stream, p);
        return hipGetLastError();
    });
}

template <typename T>
hipError_t dr_walk_launch(const DrParams& p, bool rev, hipStream_t stream) {
    const int64_t widest = p.local && !rev && p.Kp > p.V ? p.Kp : p.V;
    const dim3 grid(unsigned(p.B * p.H * p.segs), unsigned(widest + 63) / 64);
    return dr_by_keys<T>(p.K, [&](auto kp) {
        constexpr int KP = decltype(kp)::value;
        const auto go = [&](auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            if (rev && p.local) hipLaunchKernelGGL((dr::dr_walk<T, KP, true, true, WHOLE>), grid, dim3(256), 0, stream, p);
            else if (rev) hipLaunchKernelGGL((dr::dr_walk<T, KP, true, false, WHOLE>), grid, dim3(256), 0, stream, p);
            else if (p.local) hipLaunchKernelGGL((dr::dr_walk<T, KP, false, true, WHOLE>), grid, dim3(512), 0, stream, p);
            else hipLaunchKernelGGL((dr::dr_walk<T, KP, false, false, WHOLE>), grid, dim3(256), 0, stream, p);
        };
        if (p.whole) go(std::true_type{});
        else go(std::false_type{});
        return hipGetLastError();
    });
}

template <typename T>
hipError_t dr_grads_launch(const DrParams& p, hipStream_t stream) {
    return dr_by_keys<T>(p.K, [&](auto kp) {
        constexpr int KP = decltype(kp)::value;
        const int64_t all = p.BH * p.nch;
        const dim3 grid(unsigned(all), 1), block(dr::kGradThreads<T, KP>);
        if (p.whole) hipLaunchKernelGGL((dr::dr_grads<T, KP, true>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((dr::dr_grads<T, KP, false>), grid, block, 0, stream, p);
        return hipGetLastError();
    });
}

}  // namespace ss

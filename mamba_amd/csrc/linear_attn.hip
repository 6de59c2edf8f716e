// Linear attention with a decay for each head, on gfx950: the launches of a
// prompt or a training step, the kernels that finish the backward, and the
// recurrence for one token.
//
// A pass (LaJob) is the recurrence of linear_attn.hpp, run in chunks
// (linear_attn_chunk.hpp).  With few rows a pass takes three launches: each
// segment's state from a zero start, the states joined along the row, and the
// segments walked side by side, each from its carry.  The backward is three
// passes, then the decay's gradient.  With D_s = q_s . dq_s - k_s . dk_s
// and M_ij the share of token j in the output at i (times its gradient),
// D_s is row s of M less column s, and
//   dg_t = sum of M_ij over i >= t > j
//        = <S_e, dS_e> + sum of D_s over t <= s < e
// for any e >= t: S_e the state before token e, dS_e the gradient arriving at
// it from token e on.  e is the end of t's segment, so the sum, which cancels,
// runs over one segment and not the whole row.  Its terms lack the factor exp(g_t)
// that dg_t has, so where that is small dg_t is formed without it
// (la_decay_grad_strong), and e of the tokens before is that token.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "linear_attn.hpp"
#include "norm_rows.hpp"
#include "ops_kernels.hpp"
#include "ss_device.hpp"

namespace ss {

namespace {

__device__ __forceinline__ int64_t row_len(const int32_t* lens, int64_t b, int64_t L) {
    if (!lens) return L;
    const int64_t n = lens[b];
    return n < 0 ? 0 : n < L ? n : L;
}

// The segments' states in walk order, each from the one before it: ends[s] <-
// ends[s] + decays[s] ends[before s].  A thread an element of the state, 8 segments
// requested at a time; bound by their bytes (25 MB in and out in 12 us: 4.3 TB/s).
__global__ __launch_bounds__(256) void la_carry(const LaParams p) {
    const LaJob& J = p.job[blockIdx.z];
    const int64_t bh = blockIdx.y, KV = int64_t(J.K) * J.V, i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= KV) return;
    float s = J.in ? J.in[bh * KV + i] : 0.f;
    float* ends = J.ends + bh * p.segs * KV + i;
    const float* decays = J.decays + bh * p.segs;
    const int step = J.rev ? -1 : 1;
    int at = J.rev ? p.segs - 1 : 0;
    constexpr int kAhead = 8;
    for (int n = 0; n < p.segs; n += kAhead) {
        const int cnt = p.segs - n < kAhead ? p.segs - n : kAhead;
        float own[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) own[k] = k < cnt ? ends[int64_t(at + step * k) * KV] : 0.f;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (k < cnt) {
                s = __builtin_fmaf(decays[at + step * k], s, own[k]);
                ends[int64_t(at + step * k) * KV] = s;
            }
        }
        at += step * cnt;
    }
    if (J.out_state) J.out_state[bh * KV + i] = s;
}

// Sum over the 4 waves of a workgroup, in every thread.
__device__ __forceinline__ double sum_all(double v, double (&red)[4]) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// dg of one segment: the inner product of the two states at its end, and the
// sums of D from its last token down.  256 threads, up to 4 tokens each.  15 us for
// 1536 segments of 256 tokens: the states' 50 MB, and dg's stores of 4 bytes a row.
constexpr int kDgTok = 4, kDgSegMax = 256 * kDgTok;

// A segment's tokens and, token top - i a thread's i-th, dg by the sums of D
struct DgSeg {
    int64_t bh, b, h, s0, s1;
    int seg, n, top;                                    // n: the row's own tokens in it
    const float* dS;                                    // what arrives at its end, or null
    double d[kDgTok];                                   // dg
    __device__ __forceinline__ DgSeg(const LaDgParams& p, int64_t bh_, int seg_, double (&red)[4]) : bh(bh_), seg(seg_) {
        const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
        const int64_t KV = int64_t(p.K) * p.V;
        b = bh / p.H;
        h = bh % p.H;
        s0 = seg * p.seg_tokens;
        s1 = s0 + p.seg_tokens < p.L ? s0 + p.seg_tokens : p.L;
        const int64_t len = row_len(p.lens, b, p.L);
        n = int((len < s1 ? len : s1) - s0);
        top = int(s1 - s0) - 1 - tid * kDgTok;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kDgTok; ++i) {
            const int64_t t = s0 + (top - i);
            double v = 0.0;
            if (t >= s0 && t < len) {
                for (int q = 0; q < p.qtiles; ++q) v += p.dotq[(int64_t(q) * p.B * p.H + bh) * p.L + t];
                for (int k = 0; k < p.ktiles; ++k) v -= p.dotk[(int64_t(k) * p.B * p.H + bh) * p.L + t];
            }
            d[i] = v;
        }
        double f = 0.0;
        dS = seg + 1 < p.segs ? p.rends + (bh * p.segs + seg + 1) * KV : p.dlast ? p.dlast + bh * KV : nullptr;
        if (dS) {
            const float* S = p.ends + (bh * p.segs + seg) * KV;
#pragma unroll 4
            for (int i = 4 * tid; i < KV; i += 1024) {
                float x[4], y[4];
                rowvec<float>::unpack(rowvec<float>::load(S + i, int(KV) - i), x);
                rowvec<float>::unpack(rowvec<float>::load(dS + i, int(KV) - i), y);
#pragma unroll
                for (int e = 0; e < 4; ++e) f += double(x[e]) * double(y[e]);
            }
        }
        const double F = sum_all(f, red);
#pragma unroll
        for (int i = 0; i < kDgTok; ++i) {
            sum += d[i];
            d[i] = sum;
        }
        double upto = sum;                              // sums over the threads up to this one
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const double o = __shfl_up(upto, m, 64);
            if (lane >= m) upto += o;
        }
        __syncthreads();
        if (lane == 63) red[wave] = upto;
        __syncthreads();
        double base = F + (upto - sum);
        for (int w = 0; w < wave; ++w) base += red[w];
#pragma unroll
        for (int i = 0; i < kDgTok; ++i) d[i] += base;
    }
    __device__ __forceinline__ void store(const LaDgParams& p, double (&red)[4]) const {
        double mine = 0.0;
#pragma unroll
        for (int i = 0; i < kDgTok; ++i) {
            const int t = top - i;
            if (t >= 0) {
                const double v = t < n ? d[i] : 0.0;
                if (p.dg) p.dg[(b * p.L + s0 + t) * p.H + h] = float(v);
                mine += v;
            }
        }
        if (!p.part) return;
        mine = sum_all(mine, red);
        if (threadIdx.x == 0) p.part[bh * p.segs + seg] = mine;
    }
};

__global__ __launch_bounds__(256) void la_decay_grad(const LaDgParams p) {
    __shared__ double red[4];
    const DgSeg s(p, blockIdx.x, int(blockIdx.y), red);
    s.store(p, red);
}

// The segments with strong decays once more: dg of those is formed by itself, and the
// sums of D start at the next one.  With a chunk of 32 tokens c0 .. c1-1 around token t, S the
// state before c0, R the gradient arriving at c1 and M_ij = scale (q_i . k_j) (dout_i . v_j),
// each times the decays on its way,
//   dg_t = R . S + sum over i >= t of scale q_i^T S dout_i + sum over j < t of k_j^T R v_j
//          + sum over i >= t > j of M_ij        (i, j in the chunk)
// has the factor exp(g_t) in every term.  S is walked once from the segment's start; R is
// summed for each chunk that has a strong decay, over the tokens after it as far as
// their factors matter.  256 threads hold 4 x 4 elements each of a 64 x 64 part of both.
// The rows get their factors on the way into LDS, so a token costs S and R 16 products each.
// Bound by the latency of its rows and barriers at two workgroups a CU and by its vector instructions.  Forward +
// backward of 8 x 2048 tokens x 24 heads of 64 x 64, bf16: 340 us without a strong decay (5
// of them this launch's), 700 with one token in 256 strong, 950 with one in 32 or with all.
constexpr float kVanished = 0x1p-60f;
constexpr int kStrongBlocks = 512;                     // (two a CU, by their LDS)
constexpr int kDgChunk = 32, kDgPart = 64;

struct StrongShared {
    // a chunk's rows, a part of their columns, with their factors: (q, dout, k, v); [2] holds M afterwards
    __attribute__((aligned(16))) float rows[4][kDgChunk][kDgPart + 4];
    double red[4], alone[kDgSegMax], across[kDgSegMax / kDgChunk];      // across: <S, R> of a chunk
    float upto[kDgSegMax], after[kDgSegMax];               // the decays from a token's chunk's start to it, and after it to the end
    float A[kDgSegMax], B[kDgSegMax], sums[4][kDgChunk];   // the tokens' sums over S and over R
    uint32_t flags[kDgSegMax / kDgChunk], live[kDgSegMax / kDgChunk];     // a bit a token: strong; and with a factor above 0
    uint64_t found[4];
};

template <typename T>
__device__ __forceinline__ void strong_segment(const LaDgParams& p, int64_t id, StrongShared& m) {
    constexpr int C = kDgChunk, W = kDgPart;
    const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6, ti = 4 * (tid >> 4), tj = 4 * (tid & 15);
    DgSeg s(p, id / p.segs, int(id % p.segs), m.red);
    const int n = s.n;
    float g[kDgTok];
    if (tid < kDgSegMax / C) {
        m.flags[tid] = m.live[tid] = 0u;
        m.across[tid] = 0.0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kDgTok; ++i) {
        const int t = s.top - i;
        g[i] = 0.f;
        if (t < 0 || t >= n) continue;
        g[i] = p.g[s.b * p.g_b + (s.s0 + t) * p.g_l + s.h * p.g_h];
        m.A[t] = m.B[t] = 0.f;
        m.alone[t] = 0.0;
        if (!(g[i] < kLaStrong)) continue;
        atomicOr(&m.flags[t / C], 1u << (t % C));
        if (expf(g[i]) > 0.f) atomicOr(&m.live[t / C], 1u << (t % C));
    }
    // log2 of the decays from the chunk's start to a token, a chunk 32 lanes (a reset far below any other)
    const auto logs = [&](int t) __attribute__((always_inline)) {
        double G = 0.0;
        if (t < n) {
            const float gt = p.g[s.b * p.g_b + (s.s0 + t) * p.g_l + s.h * p.g_h];
            G = gt < -1e6f ? -1e6 : double(gt) * 1.4426950408889634;
        }
#pragma unroll
        for (int x = 1; x < C; x <<= 1) {
            const double o = __shfl_up(G, x, C);
            if ((lane & (C - 1)) >= x) G += o;
        }
        return G;
    };
    const auto factor = [](double x) {                      // 2^x
        const double w = floor(x);
        return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(float(x - w)), w < -2000.0 ? -2000 : w > 2000.0 ? 2000 : int(w));
    };
    for (int t = tid; t < (n + C - 1) / C * C; t += 256) {
        const double G = logs(t);
        m.upto[t] = factor(G);
        m.after[t] = factor(__shfl(G, C - 1, C) - G);
    }
    __syncthreads();
    int last = -1;
    for (int c = 0; c * C < n; ++c)
        if (m.live[c]) last = c;

    const int64_t KV = int64_t(p.K) * p.V;
    const auto head = [&](const LaRows& r) { return static_cast<const T*>(r.p) + s.b * r.b + s.s0 * r.l + s.h / r.rep * r.h; };
    const T *q = head(p.q), *k = head(p.k), *v = head(p.v), *dout = head(p.dout);
    // columns from `col` on of the tokens from c0 on (zero past both ends), times f and the tokens' factors
    const auto stage = [&](int to, const T* rows, int64_t step, int dim, int col, int c0, const float* factors = nullptr, float f = 1.f)
                           __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = (tid >> 4) + 16 * h;
            float x[4];
            load4<T>(rows + int64_t(c0 + r) * step + col + tj, x, c0 + r < n ? dim - col - tj : 0);
            const float w = factors ? f * factors[c0 + r] : f;
            *reinterpret_cast<float4*>(&m.rows[to][r][tj]) = make_float4(w * x[0], w * x[1], w * x[2], w * x[3]);
        }
    };
    const auto quad = [&](int from, int r, int at, float (&x)[4]) __attribute__((always_inline)) {
        const float4 w = *reinterpret_cast<const float4*>(&m.rows[from][r][at]);
        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    };
    // a <- a + x y^T summed over the rows of xs and ys (those past cnt are zero), and the wave's sums of x^T a y for each
    const auto add = [&](float (&a)[4][4], int xs, int ys, int cnt) __attribute__((always_inline)) {
        for (int t = 0; t < cnt; t += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float x[4], y[4];
                quad(xs, t + u, ti, x);
                quad(ys, t + u, tj, y);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[i][j] = __builtin_fmaf(x[i], y[j], a[i][j]);
            }
        }
    };
    const auto products = [&](const float (&a)[4][4], int xs, int ys, int cnt) __attribute__((always_inline)) {
        for (int t = 0; t < cnt; t += 4) {
            float f[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float x[4], y[4];
                quad(xs, t + u, ti, x);
                quad(ys, t + u, tj, y);
                f[u] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float r = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) r = __builtin_fmaf(a[i][j], y[j], r);
                    f[u] = __builtin_fmaf(x[i], r, f[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) f[u] = lanes_sum<64>(f[u]);
            if (lane == 0) {
#pragma unroll
                for (int u = 0; u < 4; ++u) m.sums[wave][t + u] = f[u];
            }
        }
    };
    const auto gather = [&](float* to, int cnt) __attribute__((always_inline)) {        // the 4 waves' sums
        __syncthreads();
        if (tid < cnt) to[tid] += (m.sums[0][tid] + m.sums[1][tid]) + (m.sums[2][tid] + m.sums[3][tid]);
    };
    const float* S0 = s.seg > 0 ? p.ends + (s.bh * p.segs + s.seg - 1) * KV : p.first ? p.first + s.bh * KV : nullptr;
    for (int k0 = 0; k0 < p.K; k0 += W) {
        for (int v0 = 0; v0 < p.V; v0 += W) {
            const auto state = [&](const float* from, int i, int j) {
                return from && k0 + ti + i < p.K && v0 + tj + j < p.V ? from[(k0 + ti + i) * p.V + v0 + tj + j] : 0.f;
            };
            float S[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) S[i][j] = state(S0, i, j);
            for (int c = 0; c <= last; ++c) {
                const int c0 = c * C, c1 = c0 + C < n ? c0 + C : n;
                const bool here = m.live[c] != 0u;
                float R[4][4] = {};
                if (here) {
                    float w = 1.f;                          // the decays from c1 to the chunk at t
                    int t = c1;
                    for (; t < n && !(w < kVanished); t += C) {
                        const int cnt = t + C < n ? C : n - t;
                        __syncthreads();
                        stage(0, q, p.q.l, p.K, k0, t, m.upto, w * p.scale);
                        stage(1, dout, p.dout.l, p.V, v0, t);
                        __syncthreads();
                        add(R, 0, 1, cnt);
                        w *= m.upto[t + cnt - 1];
                    }
                    double f = 0.0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (t >= n) R[i][j] = __builtin_fmaf(w, state(s.dS, i, j), R[i][j]);
                            f = __builtin_fma(double(S[i][j]), double(R[i][j]), f);
                        }
                    f = sum_all(f, m.red);
                    if (tid == 0) m.across[c] += f;
                }
                __syncthreads();
                if (here) {
                    stage(0, q, p.q.l, p.K, k0, c0, m.upto, p.scale);
                    stage(1, dout, p.dout.l, p.V, v0, c0);
                }
                stage(2, k, p.k.l, p.K, k0, c0, m.after);
                stage(3, v, p.v.l, p.V, v0, c0);
                __syncthreads();
                if (here) {
                    products(S, 0, 1, c1 - c0);
                    gather(m.A + c0, c1 - c0);
                    __syncthreads();
                    products(R, 2, 3, c1 - c0);
                    gather(m.B + c0, c1 - c0);
                }
                const float total = m.upto[c1 - 1];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) S[i][j] *= total;
                add(S, 2, 3, c1 - c0);
            }
        }
    }
    // the chunks' own pairs, and the sums
    for (int c = 0; c <= last; ++c) {
        if (!m.live[c]) continue;
        const int c0 = c * C, c1 = c0 + C < n ? c0 + C : n, cnt = c1 - c0;
        // 4 pairs a thread: row i, and j, j + 8 ..
        const int i = tid >> 3, j0 = tid & 7;
        const auto pairs = [&](const T* xs, int64_t xl, const T* ys, int64_t yl, int dim, float (&o)[4]) __attribute__((always_inline)) {
            for (int col = 0; col < dim; col += W) {
                __syncthreads();
                stage(0, xs, xl, dim, col, c0);
                stage(1, ys, yl, dim, col, c0);
                __syncthreads();
#pragma unroll 4
                for (int e = 0; e < W; e += 4) {
                    float x[4], y[4];
                    quad(0, i, e, x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        quad(1, j0 + 8 * j, e, y);
#pragma unroll
                        for (int a = 0; a < 4; ++a) o[j] = __builtin_fmaf(x[a], y[a], o[j]);
                    }
                }
            }
        };
        float qk[4] = {}, dv[4] = {};
        pairs(q, p.q.l, k, p.k.l, p.K, qk);
        pairs(dout, p.dout.l, v, p.v.l, p.V, dv);
        const double G = logs(c0 + (lane & (C - 1))), Gi = __shfl(G, i, C);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double Gj = __shfl(G, j0 + 8 * j, C);
            if (i < cnt && j0 + 8 * j < i) m.rows[2][i][j0 + 8 * j] = p.scale * factor(Gi - Gj) * qk[j] * dv[j];
        }
        __syncthreads();
        const int t = i, l = j0;                            // 8 lanes a token
        const bool mine = m.live[c] >> t & 1;
        double f = 0.0;
        if (mine) {
            for (int r = t + l; r < cnt; r += 8) {
                f += m.A[c0 + r];
#pragma unroll 8
                for (int j = 0; j < t; ++j) f += m.rows[2][r][j];
            }
            for (int j = l; j < t; j += 8) f += m.B[c0 + j];
            if (l == 0) f += double(m.upto[c1 - 1]) * m.across[c];
        }
#pragma unroll
        for (int x = 4; x >= 1; x >>= 1) f += __shfl_xor(f, x, 64);
        if (l == 0 && mine) m.alone[c0 + t] = f;
    }
    __syncthreads();
    // the tokens before a strong decay start at it: alone <- what it is more than the sum was
    double own[kDgTok];
#pragma unroll
    for (int i = 0; i < kDgTok; ++i) {
        own[i] = 0.0;
        if (!(g[i] < kLaStrong)) continue;
        own[i] = m.alone[s.top - i];
        m.alone[s.top - i] -= s.d[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kDgTok; ++i) {
        const int t = s.top - i;
        if (t < 0 || t >= n) continue;
        int word = t / C;
        uint32_t next = m.flags[word] & (~0u << (t % C));
        while (!next && ++word < kDgSegMax / C) next = m.flags[word];
        if (g[i] < kLaStrong) s.d[i] = own[i];
        else if (next) s.d[i] += m.alone[C * word + __builtin_ctz(next)];
    }
    s.store(p, m.red);
}

template <typename T>
__global__ __launch_bounds__(256) void la_decay_grad_strong(const LaDgParams p) {
    __shared__ StrongShared m;
    const int tid = int(threadIdx.x);
    // this workgroup's segments, a thread looks at one
    const int64_t all = p.B * p.H * p.segs, step = gridDim.x;
    for (int64_t first = blockIdx.x; first < all; first += 256 * step) {
        const int64_t mine = first + tid * step;
        const uint64_t found = __ballot(mine < all && p.strong[mine]);
        __syncthreads();
        if ((tid & 63) == 0) m.found[tid >> 6] = found;
        __syncthreads();
        for (int w = 0; w < 4; ++w) {
            for (uint64_t left = m.found[w]; left; left &= left - 1) {
                strong_segment<T>(p, first + (64 * w + __builtin_ctzll(left)) * step, m);
                __syncthreads();
            }
        }
    }
}

// dg of a head with one decay: the sum over batch rows and segments
__global__ __launch_bounds__(256) void la_decay_grad_heads(const double* part, float* dg, int64_t B, int64_t H, int segs) {
    const int64_t h = blockIdx.x;
    __shared__ double red[256];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < B * segs; i += 256) s += part[((i / segs) * H + h) * segs + i % segs];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int m = 128; m >= 1; m >>= 1) {
        if (int(threadIdx.x) < m) red[threadIdx.x] += red[threadIdx.x + m];
        __syncthreads();
    }
    if (threadIdx.x == 0) dg[h] = float(red[0]);
}

// The heads of a group share q and k: out[r, j, :] = sum over i of part[r, j * rep + i, :]
template <typename T>
__global__ __launch_bounds__(256) void la_group_sum(const float* part0, T* out0, const float* part1, T* out1, int64_t n,
                                                    int rep, int dim) {
    const float* part = blockIdx.y ? part1 : part0;
    T* out = blockIdx.y ? out1 : out0;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
        const int64_t g = i / dim, c = i % dim;
        float s = 0.f;
        for (int r = 0; r < rep; ++r) s += part[(g * rep + r) * dim + c];
        io<T>::store(out + i, s);
    }
}

// Workgroups that fill the GPU: with fewer rows (batch x heads x tiles) than
// that a row's segments run side by side, about kSegsWanted of them in all: a
// wave a segment, 8 a CU.  Fewer leave SIMDs idle, more cost the states' bytes (64
// KB a segment of 64 x 64): a prompt of 32768 tokens, 24 heads of 64 x 64, takes 193,
// 181 and 219 us with 1024, 1536 and 2112 of them, a training step of 8 x 2048
// tokens 311, 304 and 315.
constexpr int64_t kFull = 1024, kSegsWanted = 1536, kSegTokMin = 64, kSegTokMax = kDgSegMax;

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

int terms(const ss_linear_attn_args& a) { return a.dtype == SS_F32 ? 3 : a.dtype == SS_BF16 ? 1 : 2; }
int64_t tile_count(int64_t dim, int tile) { return (dim + tile - 1) / tile; }
// the backward's passes share a launch: the tile of the widest
int bwd_tile(const ss_linear_attn_args& a) {
    const int64_t d = a.d_key > a.d_value ? a.d_key : a.d_value;
    return la_tile(d, d, terms(a));
}

struct BwdSpace { int64_t dotq, dotk, rends, decays, part, strong, dq, dk, bytes; };
BwdSpace bwd_space(const ss_linear_attn_bwd_args* g) {
    const ss_linear_attn_args& a = g->f;
    const int64_t bh = a.batch * a.heads, segs = linear_attn_segs(&a);
    BwdSpace s{};
    int64_t at = 0;
    const auto take = [&](int64_t bytes) { const int64_t r = at; at += round16(bytes); return r; };
    const int64_t tiles = tile_count(a.d_key, bwd_tile(a));
    s.dotq = take(tiles * bh * a.seqlen * 4);
    s.dotk = take(tiles * bh * a.seqlen * 4);
    s.rends = take(bh * segs * a.d_key * a.d_value * 4);
    s.decays = take(bh * segs * 4);
    s.part = take(g->g_per_head ? bh * segs * 8 : 0);
    s.strong = take(bh * segs * 4);
    const int64_t shared = a.heads > a.groups ? a.batch * a.seqlen * a.heads * a.d_key * 4 : 0;
    s.dq = take(shared);
    s.dk = take(shared);
    s.bytes = at;
    return s;
}

// The segments' states where the caller keeps none, and their decays.
bool serial(const ss_linear_attn_args& a, int64_t tiles) {
    return linear_attn_segs(&a) == 1 || a.batch * a.heads * tiles >= kFull;
}
struct FwdSpace { int64_t ends, decays, bytes; };
FwdSpace fwd_space(const ss_linear_attn_args& a) {
    FwdSpace s{};
    if (serial(a, tile_count(a.d_value, la_tile(a.d_key, a.d_value, terms(a))))) return s;
    const int64_t n = a.batch * a.heads * linear_attn_segs(&a);
    s.decays = a.ends ? 0 : round16(n * a.d_key * a.d_value * 4);
    s.bytes = s.decays + round16(n * 4);
    return s;
}

LaParams common(const ss_linear_attn_args& a) {
    LaParams p{};
    p.B = a.batch; p.L = a.seqlen; p.H = a.heads;
    p.g = a.g; p.g_b = a.g_batch_stride; p.g_l = a.g_len_stride; p.g_h = a.g_head_stride;
    p.lens = a.lengths;
    p.seg_tokens = linear_attn_segment(&a);
    p.seg_chunks = int(p.seg_tokens / 32);
    p.segs = int(linear_attn_segs(&a));
    p.rep = int(a.heads / a.groups);
    return p;
}

template <typename F>
hipError_t for_type(int dtype, F&& f) {
    switch (dtype) {
        case SS_F32: return f(float{});
        case SS_BF16: return f(bf16_t{});
        default: return f(_Float16{});
    }
}

// p's jobs over whole rows or, where segments run side by side, over the
// segments: `local` (each job its own states) then gives their carries.
hipError_t carries(int dtype, const LaParams& local, hipStream_t stream) {
    const hipError_t e = for_type(dtype, [&](auto t) { return la_local_launch<decltype(t)>(local, stream); });
    if (e != hipSuccess) return e;
    const int64_t KV = int64_t(local.job[0].K) * local.job[0].V, bh = local.B * local.H;
    hipLaunchKernelGGL(la_carry, dim3(unsigned((KV + 255) / 256), unsigned(bh), unsigned(local.njobs)), dim3(256), 0, stream, local);
    return hipGetLastError();
}
hipError_t walk(int dtype, const LaParams& p, bool backward, hipStream_t stream) {
    return for_type(dtype, [&](auto t) { return la_walk_launch<decltype(t)>(p, backward, stream); });
}

}  // namespace

int64_t linear_attn_segment(const ss_linear_attn_args* a) {
    const int64_t bh = a->batch * a->heads;
    const int64_t segs = bh > 0 && bh < kSegsWanted ? kSegsWanted / bh : 1;
    const int64_t n = ((a->seqlen + segs - 1) / segs + 63) / 64 * 64;
    return n < kSegTokMin ? kSegTokMin : n > kSegTokMax ? kSegTokMax : n;
}
int64_t linear_attn_segs(const ss_linear_attn_args* a) {
    const int64_t n = linear_attn_segment(a);
    return a->seqlen <= n ? 1 : (a->seqlen + n - 1) / n;
}

int64_t linear_attn_fwd_space(const ss_linear_attn_args* a) { return fwd_space(*a).bytes; }
int64_t linear_attn_bwd_space(const ss_linear_attn_bwd_args* g) { return bwd_space(g).bytes; }

hipError_t linear_attn_fwd_launch(const ss_linear_attn_args* a, hipStream_t stream) {
    LaParams p = common(*a);
    const int rep = int(a->heads / a->groups);
    p.njobs = 1;
    p.tile = la_tile(a->d_key, a->d_value, terms(*a));
    p.tiles = int(tile_count(a->d_value, p.tile));
    p.serial = serial(*a, p.tiles);
    LaJob& j = p.job[0];
    j.q = {a->q, a->q_batch_stride, a->q_len_stride, a->q_head_stride, rep};
    j.k = {a->k, a->k_batch_stride, a->k_len_stride, a->k_head_stride, rep};
    j.v = {a->v, a->v_batch_stride, a->v_len_stride, a->v_head_stride, 1};
    j.o = {a->out, a->out_batch_stride, a->out_len_stride, a->out_head_stride, 1};
    j.K = int(a->d_key); j.V = int(a->d_value);
    j.oscale = a->scale; j.vscale = 1.f;
    j.st_k = j.V; j.st_v = 1;
    j.in = a->initial_state; j.ends = a->ends; j.out_state = a->last_state;
    if (!p.serial) {
        const FwdSpace sp = fwd_space(*a);
        char* ws = static_cast<char*>(a->workspace);
        if (!j.ends) j.ends = reinterpret_cast<float*>(ws + sp.ends);
        j.decays = reinterpret_cast<float*>(ws + sp.decays);
        const hipError_t e = carries(a->dtype, p, stream);
        if (e != hipSuccess) return e;
        j.carry = j.ends;
        j.ends = j.out_state = nullptr;
    }
    return walk(a->dtype, p, false, stream);
}

hipError_t linear_attn_bwd_launch(const ss_linear_attn_bwd_args* g, hipStream_t stream) {
    const ss_linear_attn_args& a = g->f;
    const BwdSpace sp = bwd_space(g);
    char* ws = static_cast<char*>(a.workspace);
    const int rep = int(a.heads / a.groups), K = int(a.d_key), V = int(a.d_value);
    LaParams p = common(a);
    const LaRows q{a.q, a.q_batch_stride, a.q_len_stride, a.q_head_stride, rep};
    const LaRows k{a.k, a.k_batch_stride, a.k_len_stride, a.k_head_stride, rep};
    const LaRows v{a.v, a.v_batch_stride, a.v_len_stride, a.v_head_stride, 1};
    const LaRows dout{g->dout, g->dout_batch_stride, g->dout_len_stride, g->dout_head_stride, 1};
    const auto grad = [&](void* p, int dim) {           // contiguous (batch, seqlen, heads, dim)
        return LaRows{p, a.seqlen * a.heads * dim, a.heads * dim, dim, 1};
    };
    const bool part = rep > 1;
    float* rends = reinterpret_cast<float*>(ws + sp.rends);
    p.njobs = 3;
    p.tile = bwd_tile(a);
    p.tiles = int(tile_count(K > V ? K : V, p.tile));
    p.serial = serial(a, p.tiles);
    p.strong = reinterpret_cast<int32_t*>(ws + sp.strong);
    LaJob& jq = p.job[0];
    jq.q = dout; jq.k = v; jq.v = k; jq.x = q;
    jq.o = grad(part ? ws + sp.dq : g->dq, K);
    jq.o_f32 = part;
    jq.K = V; jq.V = K;
    jq.oscale = a.scale; jq.vscale = 1.f;
    jq.st_k = 1; jq.st_v = V;
    jq.in = a.initial_state;
    jq.dot = reinterpret_cast<float*>(ws + sp.dotq);
    LaJob& jk = p.job[1];
    jk.q = v; jk.k = dout; jk.v = q; jk.x = k;
    jk.o = grad(part ? ws + sp.dk : g->dk, K);
    jk.o_f32 = part;
    jk.K = V; jk.V = K; jk.rev = 1;
    jk.oscale = 1.f; jk.vscale = a.scale;
    jk.st_k = 1; jk.st_v = V;
    jk.in = g->dlast_state;
    jk.dot = reinterpret_cast<float*>(ws + sp.dotk);
    LaJob& jv = p.job[2];
    jv.q = k; jv.k = q; jv.v = dout;
    jv.o = grad(g->dv, V);
    jv.K = K; jv.V = V; jv.rev = 1;
    jv.oscale = 1.f; jv.vscale = a.scale;
    jv.st_k = V; jv.st_v = 1;
    jv.in = g->dlast_state; jv.ends = rends; jv.out_state = g->dinitial_state;
    hipError_t e = hipSuccess;
    if (!p.serial) {
        LaParams own = p;                               // dS of the segments: jv's states
        own.njobs = 1;
        own.job[0] = jv;
        own.job[0].decays = reinterpret_cast<float*>(ws + sp.decays);
        e = carries(a.dtype, own, stream);
        if (e != hipSuccess) return e;
        jq.carry = a.ends;
        jk.carry = jv.carry = rends;
        jv.ends = jv.out_state = nullptr;
    }
    e = walk(a.dtype, p, true, stream);
    if (e != hipSuccess) return e;

    LaDgParams d{};
    d.B = a.batch; d.L = a.seqlen; d.H = a.heads;
    d.lens = a.lengths; d.seg_tokens = p.seg_tokens; d.segs = p.segs;
    d.qtiles = d.ktiles = int(tile_count(K, p.tile));
    d.K = K; d.V = V;
    d.g = p.g; d.g_b = p.g_b; d.g_l = p.g_l; d.g_h = p.g_h;
    d.strong = p.strong;
    d.q = q; d.k = k; d.v = v; d.dout = dout;
    d.scale = a.scale; d.first = a.initial_state;
    d.dotq = jq.dot; d.dotk = jk.dot; d.ends = a.ends; d.rends = rends; d.dlast = g->dlast_state;
    d.dg = g->g_per_head ? nullptr : g->dg;
    d.part = g->g_per_head ? reinterpret_cast<double*>(ws + sp.part) : nullptr;
    hipLaunchKernelGGL(la_decay_grad, dim3(unsigned(a.batch * a.heads), unsigned(p.segs)), dim3(256), 0, stream, d);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    e = for_type(a.dtype, [&](auto t) {
        const int64_t n = a.batch * a.heads * p.segs;
        hipLaunchKernelGGL((la_decay_grad_strong<decltype(t)>), dim3(unsigned(n < kStrongBlocks ? n : kStrongBlocks)), dim3(256), 0, stream, d);
        return hipGetLastError();
    });
    if (e != hipSuccess) return e;
    if (g->g_per_head) {
        hipLaunchKernelGGL(la_decay_grad_heads, dim3(unsigned(a.heads)), dim3(256), 0, stream, d.part, g->dg, a.batch,
                           a.heads, p.segs);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (part && a.seqlen > 0) {
        const int64_t n = a.batch * a.seqlen * a.groups * K;
        const int64_t want = (n + 255) / 256;
        const dim3 grid(unsigned(want < 65536 ? want : 65536), 2);
        const float* pq = reinterpret_cast<const float*>(ws + sp.dq);
        const float* pk = reinterpret_cast<const float*>(ws + sp.dk);
        const auto sum = [&](auto* dq, auto* dk) {
            using T = std::remove_pointer_t<decltype(dq)>;
            hipLaunchKernelGGL((la_group_sum<T>), grid, dim3(256), 0, stream, pq, dq, pk, dk, n, rep, K);
        };
        if (a.dtype == SS_F32) sum(static_cast<float*>(g->dq), static_cast<float*>(g->dk));
        else if (a.dtype == SS_BF16) sum(static_cast<bf16_t*>(g->dq), static_cast<bf16_t*>(g->dk));
        else sum(static_cast<_Float16*>(g->dq), static_cast<_Float16*>(g->dk));
        e = hipGetLastError();
    }
    return e;
}

namespace {

// One token.  Bound by the state's bytes: 64 x 16 heads of 128 x 128, 134 MB in and
// out, take 22 us (6.0 TB/s); one row of 24 heads 6 us, a launch.  A workgroup owns
// COLS value columns of one (batch, head):
// thread (i, c) holds 4 neighbouring columns of rows i, i + rows ... and reads
// and writes them as 16-byte vectors (element by element where the rows are
// not 16-byte aligned); the outputs' sums over the rows meet in LDS.
template <typename T, int COLS, bool VEC>
__global__ __launch_bounds__(256) void la_update(const ss_linear_attn_update_args a) {
    constexpr int C = VEC ? COLS / 4 : COLS, RG = 256 / C, W = VEC ? 4 : 1;
    const int64_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads, j = h / (a.heads / a.groups);
    const int c = int(threadIdx.x) % C, rg = int(threadIdx.x) / C;
    const int n = int(blockIdx.y) * COLS + c * W;
    const int K = int(a.d_key), V = int(a.d_value);
    __shared__ float qs[256], ks[256], red[RG][COLS];
    if (int(threadIdx.x) < K) {
        qs[threadIdx.x] = a.scale * io<T>::load(static_cast<const T*>(a.q) + b * a.q_batch_stride + j * a.q_head_stride + threadIdx.x);
        ks[threadIdx.x] = io<T>::load(static_cast<const T*>(a.k) + b * a.k_batch_stride + j * a.k_head_stride + threadIdx.x);
    }
    const float dec = expf(a.g[b * a.g_batch_stride + h * a.g_head_stride]);
    float v[W], o[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        v[w] = n + w < V ? io<T>::load(static_cast<const T*>(a.v) + b * a.v_batch_stride + h * a.v_head_stride + n + w) : 0.f;
        o[w] = 0.f;
    }
    __syncthreads();
    float* S = a.state + b * a.state_batch_stride + h * a.state_head_stride;
    if (n < V) {
        for (int d = rg; d < K; d += RG) {
            float* at = S + int64_t(d) * V + n;
            float s[W];
            if constexpr (VEC) {
                const float4 t = *reinterpret_cast<const float4*>(at);
                s[0] = t.x; s[1] = t.y; s[2] = t.z; s[3] = t.w;
            } else {
                s[0] = *at;
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                s[w] = __builtin_fmaf(ks[d], v[w], dec * s[w]);
                o[w] = __builtin_fmaf(qs[d], s[w], o[w]);
            }
            if constexpr (VEC) *reinterpret_cast<float4*>(at) = make_float4(s[0], s[1], s[2], s[3]);
            else *at = s[0];
        }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) red[rg][c * W + w] = o[w];
    __syncthreads();
    if (int(threadIdx.x) < COLS) {
        const int m = int(blockIdx.y) * COLS + int(threadIdx.x);
        float t = 0.f;
        for (int i = 0; i < RG; ++i) t += red[i][threadIdx.x];
        if (m < V) io<T>::store(static_cast<T*>(a.out) + b * a.out_batch_stride + h * a.out_head_stride + m, t);
    }
}

template <typename T>
hipError_t update_t(const ss_linear_attn_update_args* a, hipStream_t stream) {
    const bool vec = a->d_value % 4 == 0 && a->state_batch_stride % 4 == 0 && a->state_head_stride % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(a->state) & 15) == 0;
    const unsigned bh = unsigned(a->batch * a->heads), V = unsigned(a->d_value);
    if (vec) hipLaunchKernelGGL((la_update<T, 64, true>), dim3(bh, (V + 63) / 64), dim3(256), 0, stream, *a);
    else hipLaunchKernelGGL((la_update<T, 64, false>), dim3(bh, (V + 63) / 64), dim3(256), 0, stream, *a);
    return hipGetLastError();
}

}  // namespace

hipError_t linear_attn_update_launch(const ss_linear_attn_update_args* a, hipStream_t stream) {
    switch (a->dtype) {
        case SS_F32: return update_t<float>(a, stream);
        case SS_BF16: return update_t<bf16_t>(a, stream);
        default: return update_t<_Float16>(a, stream);
    }
}

}  // namespace ss

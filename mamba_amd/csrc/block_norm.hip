// The norms around a block, and the gated norm of each head inside one, on
// gfx950, forward and backward.
//
// Border (block_norm): with rms(v) = v (mean(v^2) + eps)^-1/2,
//
//   t   = rms(x) (1 + post) [* silu(gate)]
//   s   = residual + scale t                 (stored in the rows' type)
//   out = rms(s) (1 + pre)                   (of the unrounded s)
//
// Backward, with n1, n2 the two reciprocal roots (kept by the forward),
// c = scale silu(gate) (1 + post) n1 x (so s = residual + c) and
// h = ds + n2 dout (1 + pre):
//
//   a2 = n2 mean(n2 dout (1 + pre) s),   dr = h - a2 n2 s = dresidual
//   dx = n1 dr scale silu(gate) (1 + post) - n1 x a1,   a1 = n1 mean(dr c)
//   dgate = dr scale x n1 (1 + post) silu'(gate)
//   dpost, dpre, dscale: sums over rows of dr scale silu(gate) x n1,
//                        dout s n2, dr x n1 (1 + post) silu(gate)
//
// mean(dr c) = mean(h c) - a2 n2 mean(s c), so a row needs one reduction (of
// three sums) and is read once.  No product holds a root's square alone: rows of
// 1e-15 or 1e15 keep their gradients.
//
// Heads (gated_norm), each row in groups of n elements with a norm of its own:
//
//   out = rms_group(x) (1 + weight) silu(gate)
//   with g = dout silu(gate):  dx = r g (1 + weight) - x r (r mean(r g (1 + weight) x)),
//   dgate = dout x r (1 + weight) silu'(gate),  dweight = sum over rows of g x r
//
// (r recomputed in the backward: its sum rides with the other one.)
//
// A row (a group) lies in the registers of a team of lanes, 8 or 16 elements
// a lane, between its one load and its one store: the kernels are bound by
// HBM.  16384 x 768 bf16 with gate and scale: forward 26 us (126 MB, 4.8 TB/s),
// backward 56 us (201 MB, 3.6 TB/s: 246 registers leave two waves a SIMD; with the
// weights as fp32 there was one, 80 us).  16384 x 24 heads of 64: forward 27 us
// (5.6 TB/s), backward 51 us (4.9 TB/s).  Weights and column sums stay in the team's registers over its rows.
// The column sums leave as one fp32 row per workgroup, summed by a second
// kernel in a fixed order: the same bits on every run.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/mamba_ss.h"
#include "norm_rows.hpp"
#include "norm_teams.hpp"
#include "ops_kernels.hpp"
#include "ss_device.hpp"

namespace ss {

namespace {

constexpr int kMaxParts = 512;                // workgroups (rows of column sums) of a border's backward (1024: 83 us for 76)
constexpr int kHeadParts = 1024, kHeadBlocks = 4096;   // workgroups of the heads' backward (512: 60 us for 51) and forward (38 for 27)

struct BorderParams {
    int64_t rows, x_rs, res_rs, gate_rs, out_rs, s_rs;
    int dim;
    float eps, scale;
    const void* x; const void* res; const void* gate;
    const void* post; const void* pre; const void* wscale;   // wscale null: scale
    void* out; void* s; float* rstd;                         // rstd (rows, 2), forward: written unless null
    // backward: out_rs / s_rs are dout's and ds's
    const void* dout; const void* ds;                        // null: zero
    void* dx; void* dres; void* dgate;                       // contiguous
    float* part;                                             // (workgroups, 3, dim): dpost, dpre, dscale
};

struct GatedParams {
    int64_t rows, x_rs, gate_rs, out_rs;                     // out_rs: dout's in the backward
    int dim, groups, n;                                      // n = dim / groups
    int gpw, rpw;                                            // groups and rows at a time per workgroup
    float eps;
    const void* x; const void* gate; const void* w;
    void* out;
    const void* dout; void* dx; void* dgate;
    float* part;                                             // (row blocks, dim)
};

template <typename T, typename TW, int WPR, int EPT>
__global__ __launch_bounds__(kBlock<WPR>) void block_norm_fwd(const BorderParams p) {
    using R = rowvec<T>;
    constexpr int VE = R::VE, NV = EPT / VE, TEAM = 64 * WPR, ROWS = kBlock<WPR> / TEAM;
    __shared__ float red[2][WPR][1];
    const int u = int(threadIdx.x) % TEAM, wave = u >> 6;
    int col[NV], cnt[NV];
    float wpost[NV][VE], wpre[NV][VE], wsc[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        col[k] = (k * TEAM + u) * VE;
        cnt[k] = p.dim - col[k];
        R::template weights<TW>(static_cast<const TW*>(p.post) + col[k], cnt[k], wpost[k]);
        R::template weights<TW>(static_cast<const TW*>(p.pre) + col[k], cnt[k], wpre[k]);
        if (p.wscale) R::template weights<TW>(static_cast<const TW*>(p.wscale) + col[k], cnt[k], wsc[k]);
        else {
#pragma unroll
            for (int e = 0; e < VE; ++e) wsc[k][e] = p.scale;
        }
    }
    const float inv = 1.f / float(p.dim);
    for (int64_t row = int64_t(blockIdx.x) * ROWS + threadIdx.x / TEAM; row < p.rows; row += int64_t(gridDim.x) * ROWS) {
        uint4 cx[NV], cr[NV], cz[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            cx[k] = R::load(static_cast<const T*>(p.x) + row * p.x_rs + col[k], cnt[k]);
            cr[k] = R::load(static_cast<const T*>(p.res) + row * p.res_rs + col[k], cnt[k]);
            if (p.gate) cz[k] = R::load(static_cast<const T*>(p.gate) + row * p.gate_rs + col[k], cnt[k]);
        }
        float sum[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float x[VE];
            R::unpack(cx[k], x);
#pragma unroll
            for (int e = 0; e < VE; ++e) sum[0] = __builtin_fmaf(x[e], x[e], sum[0]);
        }
        team_sum<WPR>(sum, red[0], wave);
        const float n1 = rsqrtf(sum[0] * inv + p.eps);
        float s[NV][VE];
        sum[0] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float x[VE], z[VE];
            R::unpack(cx[k], x);
            R::unpack(cr[k], s[k]);
            if (p.gate) R::unpack(cz[k], z);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                float t = x[e] * n1 * (1.f + wpost[k][e]);
                if (p.gate) t *= z[e] * sigmoid(z[e]);
                s[k][e] = __builtin_fmaf(wsc[k][e], t, s[k][e]);
                sum[0] = e < cnt[k] ? __builtin_fmaf(s[k][e], s[k][e], sum[0]) : sum[0];
            }
            R::store(static_cast<T*>(p.s) + row * p.s_rs + col[k], s[k], cnt[k]);
        }
        team_sum<WPR>(sum, red[1], wave);
        const float n2 = rsqrtf(sum[0] * inv + p.eps);
        if (p.rstd && u == 0) {
            p.rstd[2 * row] = n1;
            p.rstd[2 * row + 1] = n2;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float o[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) o[e] = s[k][e] * n2 * (1.f + wpre[k][e]);
            R::store(static_cast<T*>(p.out) + row * p.out_rs + col[k], o, cnt[k]);
        }
    }
}

template <typename T, typename TW, int WPR, int EPT>
__global__ __launch_bounds__(kBlock<WPR>, kBlock<WPR> / 256 > 2 ? kBlock<WPR> / 256 : 2) void block_norm_bwd(const BorderParams p) {
    using R = rowvec<T>;
    constexpr int VE = R::VE, NV = EPT / VE, TEAM = 64 * WPR, ROWS = kBlock<WPR> / TEAM;
    __shared__ float red[2][WPR][3];
    __shared__ float cols[ROWS > 1 ? 3 * TEAM * EPT : 1];
    const int u = int(threadIdx.x) % TEAM, wave = u >> 6;
    int col[NV], cnt[NV];
    // (weights stay in their own type: as fp32 they and the sums would leave room for one wave a SIMD)
    PackedWeights<T, TW, EPT * sizeof(TW) <= 32> kpost[NV], kpre[NV], ksc[NV];
    float apost[NV][VE], apre[NV][VE], asc[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        col[k] = (k * TEAM + u) * VE;
        cnt[k] = p.dim - col[k];
        kpost[k].load(static_cast<const TW*>(p.post) + col[k], cnt[k]);
        kpre[k].load(static_cast<const TW*>(p.pre) + col[k], cnt[k]);
        ksc[k].load(static_cast<const TW*>(p.wscale) + col[k], p.wscale ? cnt[k] : 0);
#pragma unroll
        for (int e = 0; e < VE; ++e) apost[k][e] = apre[k][e] = asc[k][e] = 0.f;
    }
    const float inv = 1.f / float(p.dim);
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    int turn = 0;
    for (int64_t row = int64_t(blockIdx.x) * ROWS + threadIdx.x / TEAM; row < p.rows; row += int64_t(gridDim.x) * ROWS) {
        uint4 cx[NV], cr[NV], cz[NV], co[NV], cs[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            cx[k] = R::load(static_cast<const T*>(p.x) + row * p.x_rs + col[k], cnt[k]);
            cr[k] = R::load(static_cast<const T*>(p.res) + row * p.res_rs + col[k], cnt[k]);
            cz[k] = p.gate ? R::load(static_cast<const T*>(p.gate) + row * p.gate_rs + col[k], cnt[k]) : none;
            co[k] = p.dout ? R::load(static_cast<const T*>(p.dout) + row * p.out_rs + col[k], cnt[k]) : none;
            cs[k] = p.ds ? R::load(static_cast<const T*>(p.ds) + row * p.s_rs + col[k], cnt[k]) : none;
        }
        const float n1 = p.rstd[2 * row], n2 = p.rstd[2 * row + 1];
        float sig[NV][VE], sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float x[VE], r[VE], z[VE], o[VE], d[VE], wpost[VE], wpre[VE], wsc[VE];
            kpost[k].get(wpost);
            kpre[k].get(wpre);
            ksc[k].get(wsc);
            R::unpack(cx[k], x);
            R::unpack(cr[k], r);
            R::unpack(cz[k], z);
            R::unpack(co[k], o);
            R::unpack(cs[k], d);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                if (!p.wscale) wsc[e] = p.scale;
                float sil = 1.f;
                if (p.gate) {
                    sig[k][e] = sigmoid(z[e]);
                    sil = z[e] * sig[k][e];
                }
                const float c = wsc[e] * sil * (1.f + wpost[e]) * (x[e] * n1), s = r[e] + c;
                const float ow = o[e] * (1.f + wpre[e]), h = __builtin_fmaf(n2, ow, d[e]);
                sum[0] = __builtin_fmaf(ow, s, sum[0]);
                sum[1] = __builtin_fmaf(h, c, sum[1]);
                sum[2] = __builtin_fmaf(s, c, sum[2]);
            }
        }
        team_sum<WPR>(sum, red[turn], wave);
        turn ^= 1;
        const float a2 = n2 * (n2 * sum[0] * inv);
        const float a1 = n1 * ((sum[1] - a2 * (n2 * sum[2])) * inv);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float x[VE], r[VE], z[VE], o[VE], d[VE], gz[VE], wpost[VE], wpre[VE], wsc[VE];
            kpost[k].get(wpost);
            kpre[k].get(wpre);
            ksc[k].get(wsc);
            R::unpack(cx[k], x);
            R::unpack(cr[k], r);
            R::unpack(cz[k], z);
            R::unpack(co[k], o);
            R::unpack(cs[k], d);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                if (!p.wscale) wsc[e] = p.scale;
                const float w1 = 1.f + wpost[e], sil = p.gate ? z[e] * sig[k][e] : 1.f, xn = x[e] * n1;
                const float c = wsc[e] * sil * w1 * xn, sn = (r[e] + c) * n2;
                const float ow = o[e] * (1.f + wpre[e]);
                const float dr = __builtin_fmaf(n2, ow, d[e]) - a2 * sn;
                const float dt = dr * wsc[e];
                apre[k][e] = __builtin_fmaf(o[e], sn, apre[k][e]);
                apost[k][e] = __builtin_fmaf(dt * sil, xn, apost[k][e]);
                asc[k][e] = __builtin_fmaf(dr, xn * w1 * sil, asc[k][e]);
                gz[e] = p.gate ? dt * (xn * w1) * sig[k][e] * __builtin_fmaf(z[e], 1.f - sig[k][e], 1.f) : 0.f;
                d[e] = dr;
                x[e] = n1 * (dt * sil * w1) - xn * a1;
            }
            if (p.gate) R::store(static_cast<T*>(p.dgate) + row * p.dim + col[k], gz, cnt[k]);
            if (p.dres) R::store(static_cast<T*>(p.dres) + row * p.dim + col[k], d, cnt[k]);
            R::store(static_cast<T*>(p.dx) + row * p.dim + col[k], x, cnt[k]);
        }
    }
    // the workgroup's column sums, its rows' teams in order
    float* part = p.part + int64_t(blockIdx.x) * 3 * p.dim;
    for (int w = 0; w < ROWS; ++w) {
        if (int(threadIdx.x) / TEAM == w) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    float v[3] = {apost[k][e], apre[k][e], asc[k][e]};
                    const int c = col[k] + e;
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        if constexpr (ROWS > 1) {
                            if (w > 0) v[i] += cols[i * TEAM * EPT + c];
                            if (w + 1 < ROWS) cols[i * TEAM * EPT + c] = v[i];
                        }
                        if (w + 1 == ROWS && e < cnt[k]) part[i * p.dim + c] = v[i];
                    }
                }
            }
        }
        if constexpr (ROWS > 1) __syncthreads();
    }
}

// ------------------------------------------------------ norms of the heads --
// L lanes hold a group's n elements, EPT a lane (8 as long as a wave's 64 lanes hold
// the group, so that neighbouring lanes read neighbouring vectors); a workgroup's teams of L
// lanes hold gpw neighbouring groups of rpw rows and walk down the rows, so a
// team's group, its weights and column sums do not change.  L above 64: a
// workgroup a group.
template <int L> constexpr int kHeadBlock = L > 256 ? L : 256;

template <typename T, typename TW, int L, int EPT, bool BWD>
__global__ __launch_bounds__(kHeadBlock<L>) void gated_norm(const GatedParams p) {
    using R = rowvec<T>;
    constexpr int VE = R::VE, NV = (EPT + VE - 1) / VE, WPR = L > 64 ? L / 64 : 1;
    __shared__ float red[2][WPR][2];
    __shared__ float cols[BWD && L <= 64 ? kHeadBlock<L> * NV * VE : 1];
    const int sub = int(threadIdx.x) / L, u = int(threadIdx.x) % L, wave = u >> 6;
    const int g = int(blockIdx.x) * p.gpw + sub % p.gpw, r0 = sub / p.gpw;
    const bool on = g < p.groups && r0 < p.rpw;
    int col[NV], cnt[NV];
    float w[NV][VE], acc[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int at = (k * L + u) * VE;
        col[k] = g * p.n + at;
        cnt[k] = on ? p.n - at : 0;
        R::template weights<TW>(static_cast<const TW*>(p.w) + col[k], cnt[k], w[k]);
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[k][e] = 0.f;
    }
    const float inv = 1.f / float(p.n);
    int turn = 0;
    // (every team of the workgroup walks as often: rows past the end load and store nothing)
    for (int64_t base = int64_t(blockIdx.y) * p.rpw; base < p.rows; base += int64_t(gridDim.y) * p.rpw) {
        const int64_t row = base + r0;
        const bool live = on && row < p.rows;
        uint4 cx[NV], cz[NV], co[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int n = live ? cnt[k] : 0;
            cx[k] = R::load(static_cast<const T*>(p.x) + row * p.x_rs + col[k], n);
            cz[k] = R::load(static_cast<const T*>(p.gate) + row * p.gate_rs + col[k], n);
            if constexpr (BWD) co[k] = R::load(static_cast<const T*>(p.dout) + row * p.out_rs + col[k], n);
        }
        float sig[NV][VE], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float x[VE], z[VE], o[VE];
            R::unpack(cx[k], x);
            R::unpack(cz[k], z);
            if constexpr (BWD) R::unpack(co[k], o);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                sig[k][e] = sigmoid(z[e]);
                sum[0] = __builtin_fmaf(x[e], x[e], sum[0]);
                if constexpr (BWD) sum[1] = __builtin_fmaf(o[e] * (z[e] * sig[k][e]) * (1.f + w[k][e]), x[e], sum[1]);
            }
        }
        if constexpr (L > 64) {
            team_sum<WPR>(sum, red[turn], wave);
            turn ^= 1;
        } else {
            sum[0] = lanes_sum<L>(sum[0]);
            if constexpr (BWD) sum[1] = lanes_sum<L>(sum[1]);
        }
        const float r = rsqrtf(sum[0] * inv + p.eps);
        const float a = r * (r * sum[1] * inv);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int n = live ? cnt[k] : 0;
            float x[VE], z[VE], o[VE], gz[VE];
            R::unpack(cx[k], x);
            R::unpack(cz[k], z);
            if constexpr (BWD) R::unpack(co[k], o);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float w1 = 1.f + w[k][e], sil = z[e] * sig[k][e], xr = x[e] * r;
                if constexpr (BWD) {
                    const float gr = o[e] * sil;
                    acc[k][e] = __builtin_fmaf(gr, xr, acc[k][e]);
                    gz[e] = o[e] * (xr * w1) * sig[k][e] * __builtin_fmaf(z[e], 1.f - sig[k][e], 1.f);
                    x[e] = r * (gr * w1) - xr * a;
                } else {
                    x[e] = xr * w1 * sil;
                }
            }
            if constexpr (BWD) {
                R::store(static_cast<T*>(p.dx) + row * p.dim + col[k], x, n);
                R::store(static_cast<T*>(p.dgate) + row * p.dim + col[k], gz, n);
            } else {
                R::store(static_cast<T*>(p.out) + row * p.out_rs + col[k], x, n);
            }
        }
    }
    if constexpr (BWD) {
        // the row block's column sums: the teams of the same groups in order
        float* part = p.part + int64_t(blockIdx.y) * p.dim;
        if constexpr (L > 64) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    if (e < cnt[k]) part[col[k] + e] = acc[k][e];
                }
            }
        } else {
            const int mine = (sub % p.gpw) * L + u;             // this lane's place among its row's
            for (int q = 0; q < p.rpw; ++q) {
                if (on && r0 == q) {
#pragma unroll
                    for (int k = 0; k < NV; ++k) {
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            float v = acc[k][e];
                            float& at = cols[(k * VE + e) * kHeadBlock<L> + mine];
                            if (q > 0) v += at;
                            if (q + 1 < p.rpw) at = v;
                            else if (e < cnt[k]) part[col[k] + e] = v;
                        }
                    }
                }
                __syncthreads();
            }
        }
    }
}

int border_rows_at_once(int64_t dim) { return dim <= 1024 ? 4 : 1; }

template <typename F>
hipError_t for_group(int64_t n, F&& f) {
    using std::integral_constant;
    const integral_constant<int, 8> e8{};
    const integral_constant<int, 16> e16{};
    if (n <= 16) return f(integral_constant<int, 2>{}, e8);
    if (n <= 32) return f(integral_constant<int, 4>{}, e8);
    if (n <= 64) return f(integral_constant<int, 8>{}, e8);
    if (n <= 128) return f(integral_constant<int, 16>{}, e8);
    if (n <= 256) return f(integral_constant<int, 32>{}, e8);
    if (n <= 512) return f(integral_constant<int, 64>{}, e8);
    if (n <= 1024) return f(integral_constant<int, 64>{}, e16);
    if (n <= 4096) return f(integral_constant<int, 256>{}, e16);
    return f(integral_constant<int, 1024>{}, e16);
}

int64_t border_parts(int64_t rows, int64_t dim) {
    const int at = border_rows_at_once(dim);
    const int64_t n = (rows + at - 1) / at;
    return n < kMaxParts ? n : kMaxParts;
}

// the teams' places in a workgroup, and the row blocks of a launch
struct HeadGrid { int gpw, rpw, threads; int64_t sets, blocks; };
HeadGrid head_grid(int64_t rows, int64_t groups, int64_t n, bool bwd) {
    HeadGrid h{};
    int L = 2;
    (void)for_group(n, [&](auto l, auto) { L = decltype(l)::value; return hipSuccess; });
    const int teams = L > 64 ? 1 : 256 / L;
    h.gpw = int(groups < teams ? groups : teams);
    h.rpw = teams / h.gpw;
    if (h.rpw > rows && rows > 0) h.rpw = int(rows);
    h.threads = (h.gpw * h.rpw * L + 63) / 64 * 64;
    h.sets = (groups + h.gpw - 1) / h.gpw;
    // (the backward's row blocks are rows of column sums: fewer of them)
    const int64_t want = (rows + h.rpw - 1) / h.rpw, all = bwd ? kHeadParts : kHeadBlocks, most = (all + h.sets - 1) / h.sets;
    h.blocks = want < most ? want : most;
    return h;
}

template <bool BWD>
hipError_t gated_launch(GatedParams p, int dtype, int w_dtype, void* dweight, hipStream_t stream) {
    const HeadGrid h = head_grid(p.rows, p.groups, p.n, BWD);
    p.gpw = h.gpw; p.rpw = h.rpw;
    return for_types(dtype, w_dtype, [&](auto t, auto tw) {
        using T = decltype(t);
        using TW = decltype(tw);
        if (p.rows > 0) {
            const hipError_t e = for_group(p.n, [&](auto l, auto ept) {
                hipLaunchKernelGGL((gated_norm<T, TW, decltype(l)::value, decltype(ept)::value, BWD>),
                                   dim3(unsigned(h.sets), unsigned(h.blocks)), dim3(unsigned(h.threads)), 0, stream, p);
                return hipGetLastError();
            });
            if (e != hipSuccess) return e;
        }
        if constexpr (BWD) {
            const ColSums c{p.part, p.rows > 0 ? h.blocks : 0, p.dim, p.dim, {dweight, nullptr, nullptr}};
            hipLaunchKernelGGL((norm_col_sums<TW>), dim3(unsigned((p.dim + 63) / 64), 1), dim3(64 * kSumWaves), 0, stream, c);
        }
        return hipGetLastError();
    });
}

}  // namespace

int64_t block_norm_bwd_space(int64_t rows, int64_t dim) { return border_parts(rows, dim) * 3 * dim * 4; }
int64_t gated_norm_bwd_space(int64_t rows, int64_t dim, int64_t groups) {
    return groups > 0 && rows > 0 ? head_grid(rows, groups, dim / groups, true).blocks * dim * 4 : 0;
}

hipError_t block_norm_fwd_launch(const ss_block_norm_args* a, hipStream_t stream) {
    BorderParams p{};
    p.rows = a->rows; p.dim = int(a->dim); p.eps = a->eps; p.scale = a->scale;
    p.x_rs = a->x_row_stride; p.res_rs = a->residual_row_stride; p.gate_rs = a->gate_row_stride;
    p.out_rs = a->out_row_stride; p.s_rs = a->residual_out_row_stride;
    p.x = a->x; p.res = a->residual; p.gate = a->gate; p.post = a->post; p.pre = a->pre; p.wscale = a->scale_vec;
    p.out = a->out; p.s = a->residual_out; p.rstd = a->rstd;
    const int at = border_rows_at_once(a->dim);
    const int64_t want = (a->rows + at - 1) / at;
    return for_types(a->dtype, a->w_dtype, [&](auto t, auto tw) {
        return for_row(a->dim, [&](auto wpr, auto ept) {
            hipLaunchKernelGGL((block_norm_fwd<decltype(t), decltype(tw), decltype(wpr)::value, decltype(ept)::value>),
                               dim3(unsigned(want < 2048 ? want : 2048)), dim3(kBlock<decltype(wpr)::value>), 0, stream, p);
            return hipGetLastError();
        });
    });
}

hipError_t block_norm_bwd_launch(const ss_block_norm_bwd_args* g, hipStream_t stream) {
    BorderParams p{};
    p.rows = g->rows; p.dim = int(g->dim); p.scale = g->scale;
    p.x_rs = g->x_row_stride; p.res_rs = g->residual_row_stride; p.gate_rs = g->gate_row_stride;
    p.out_rs = g->dout_row_stride; p.s_rs = g->dresidual_out_row_stride;
    p.x = g->x; p.res = g->residual; p.gate = g->gate; p.post = g->post; p.pre = g->pre; p.wscale = g->scale_vec;
    p.rstd = const_cast<float*>(g->rstd);
    p.dout = g->dout; p.ds = g->dresidual_out; p.dx = g->dx; p.dres = g->dresidual; p.dgate = g->dgate;
    p.part = static_cast<float*>(g->workspace);
    const int64_t parts = border_parts(g->rows, g->dim);
    return for_types(g->dtype, g->w_dtype, [&](auto t, auto tw) {
        if (p.rows > 0) {
            const hipError_t e = for_row(g->dim, [&](auto wpr, auto ept) {
                hipLaunchKernelGGL((block_norm_bwd<decltype(t), decltype(tw), decltype(wpr)::value, decltype(ept)::value>),
                                   dim3(unsigned(parts)), dim3(kBlock<decltype(wpr)::value>), 0, stream, p);
                return hipGetLastError();
            });
            if (e != hipSuccess) return e;
        }
        const ColSums c{p.part, parts, 3 * int64_t(p.dim), p.dim, {g->dpost, g->dpre, g->dscale}};
        hipLaunchKernelGGL((norm_col_sums<decltype(tw)>), dim3(unsigned((p.dim + 63) / 64), 3), dim3(64 * kSumWaves), 0,
                           stream, c);
        return hipGetLastError();
    });
}

hipError_t gated_norm_fwd_launch(const ss_gated_norm_args* a, hipStream_t stream) {
    GatedParams p{};
    p.rows = a->rows; p.dim = int(a->dim); p.groups = int(a->groups); p.n = int(a->dim / a->groups); p.eps = a->eps;
    p.x_rs = a->x_row_stride; p.gate_rs = a->gate_row_stride; p.out_rs = a->out_row_stride;
    p.x = a->x; p.gate = a->gate; p.w = a->weight; p.out = a->out;
    return gated_launch<false>(p, a->dtype, a->w_dtype, nullptr, stream);
}

hipError_t gated_norm_bwd_launch(const ss_gated_norm_bwd_args* g, hipStream_t stream) {
    GatedParams p{};
    p.rows = g->rows; p.dim = int(g->dim); p.groups = int(g->groups); p.n = int(g->dim / g->groups); p.eps = g->eps;
    p.x_rs = g->x_row_stride; p.gate_rs = g->gate_row_stride; p.out_rs = g->dout_row_stride;
    p.x = g->x; p.gate = g->gate; p.w = g->weight; p.dout = g->dout; p.dx = g->dx; p.dgate = g->dgate;
    p.part = static_cast<float*>(g->workspace);
    return gated_launch<true>(p, g->dtype, g->w_dtype, g->dweight, stream);
}

}  // namespace ss

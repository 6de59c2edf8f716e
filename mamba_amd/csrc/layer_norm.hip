// Layer norm with the residual add in front of it, on gfx950, forward and backward.
//
//   s   = x + residual                       (rounded to the rows' type; s = x without residual)
//   out = (s - m) r w + b,   m = mean(s),  r = (mean((s - m)^2) + eps)^-1/2
//
// and back, with h = (s - m) r and o = dout w:
//
//   dx = dresidual = r (o - mean(o) - h mean(o h)) + ds,   dw = sum over rows of dout h,   db = sum of dout
//
// A row lies in the registers of a team of lanes between its one load and its one
// store, so the mean is known before the squares are summed: rows far from zero keep
// the bits of their spread.  Backward, the two means take one reduction; weights and column
// sums stay in the team's registers over its rows, and the sums leave as one fp32 row a
// workgroup, summed by a second kernel in a fixed order.
//
// Bound by HBM and the last-level cache: 16384 x 768, bf16, with residual, forward 17.8 us (101 MB at 5.7 TB/s), backward
// 23.3 (101 MB at 4.3) and 3.8 for the column sums; 2047 x 1001, fp16 (rows off 16 bytes), 6.6, 10.1 and 3.3.
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

constexpr int kParts = 512;                   // workgroups (rows of column sums) of the backward

struct LayerParams {
    int64_t rows, x_rs, res_rs, out_rs, s_rs;          // backward: s's, ds's, dout's
    int dim;
    float eps;
    const void* x; const void* res;                    // backward: s, ds (null: zero)
    const void* w; const void* b;                      // b null: none
    void* out; void* s; float* stats;                  // s, stats (rows, 2): null, not written
    const void* dout; void* dx; float* part;           // part: (workgroups, 2, dim)
};

template <typename T> __device__ __forceinline__ float rounded(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (__is_same(T, bf16_t)) return __uint_as_float(uint32_t(io<bf16_t>::round(v)) << 16);
    else return float(_Float16(v));
}

template <typename T, typename TW, int WPR, int EPT>
__global__ __launch_bounds__(kBlock<WPR>) void layer_norm_fwd(const LayerParams p) {
    using R = rowvec<T>;
    constexpr int VE = R::VE, NV = EPT / VE, TEAM = 64 * WPR, ROWS = kBlock<WPR> / TEAM;
    __shared__ float red[2][WPR][1];
    const int u = int(threadIdx.x) % TEAM, wave = u >> 6;
    int col[NV], cnt[NV];
    float w[NV][VE], b[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        col[k] = (k * TEAM + u) * VE;
        cnt[k] = p.dim - col[k];
        R::template weights<TW>(static_cast<const TW*>(p.w) + col[k], cnt[k], w[k]);
        R::template weights<TW>(static_cast<const TW*>(p.b) + col[k], p.b ? cnt[k] : 0, b[k]);
    }
    const float n = float(p.dim), inv = 1.f / n;
    for (int64_t row = int64_t(blockIdx.x) * ROWS + threadIdx.x / TEAM; row < p.rows; row += int64_t(gridDim.x) * ROWS) {
        uint4 cx[NV], cr[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            cx[k] = R::load(static_cast<const T*>(p.x) + row * p.x_rs + col[k], cnt[k]);
            if (p.res) cr[k] = R::load(static_cast<const T*>(p.res) + row * p.res_rs + col[k], cnt[k]);
        }
        float s[NV][VE], sum[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            R::unpack(cx[k], s[k]);
            if (p.res) {
                float r[VE];
                R::unpack(cr[k], r);
#pragma unroll
                for (int e = 0; e < VE; ++e) s[k][e] = rounded<T>(s[k][e] + r[e]);
                if (p.s) R::store(static_cast<T*>(p.s) + row * p.s_rs + col[k], s[k], cnt[k]);
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) sum[0] += s[k][e];
        }
        team_sum<WPR>(sum, red[0], wave);
        const float m = sum[0] / n;                // (divided: a row of one value has exactly that mean where its sum is exact)
        sum[0] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                s[k][e] -= m;
                sum[0] = e < cnt[k] ? __builtin_fmaf(s[k][e], s[k][e], sum[0]) : sum[0];
            }
        team_sum<WPR>(sum, red[1], wave);
        const float r = rsqrtf(sum[0] * inv + p.eps);
        if (p.stats && u == 0) {
            p.stats[2 * row] = m;
            p.stats[2 * row + 1] = r;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float o[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) o[e] = __builtin_fmaf(s[k][e] * r, w[k][e], b[k][e]);
            R::store(static_cast<T*>(p.out) + row * p.out_rs + col[k], o, cnt[k]);
        }
    }
}

template <typename T, typename TW, int WPR, int EPT>
__global__ __launch_bounds__(kBlock<WPR>) void layer_norm_bwd(const LayerParams p) {
    using R = rowvec<T>;
    constexpr int VE = R::VE, NV = EPT / VE, TEAM = 64 * WPR, ROWS = kBlock<WPR> / TEAM;
    __shared__ float red[2][WPR][2];
    __shared__ float cols[ROWS > 1 ? 2 * TEAM * EPT : 1];
    const int u = int(threadIdx.x) % TEAM, wave = u >> 6;
    int col[NV], cnt[NV];
    PackedWeights<T, TW, EPT * sizeof(TW) <= 32> kw[NV];
    float aw[NV][VE], ab[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        col[k] = (k * TEAM + u) * VE;
        cnt[k] = p.dim - col[k];
        kw[k].load(static_cast<const TW*>(p.w) + col[k], cnt[k]);
#pragma unroll
        for (int e = 0; e < VE; ++e) aw[k][e] = ab[k][e] = 0.f;
    }
    const float inv = 1.f / float(p.dim);
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    int turn = 0;
    for (int64_t row = int64_t(blockIdx.x) * ROWS + threadIdx.x / TEAM; row < p.rows; row += int64_t(gridDim.x) * ROWS) {
        uint4 cs[NV], cd[NV], co[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            cs[k] = R::load(static_cast<const T*>(p.x) + row * p.x_rs + col[k], cnt[k]);
            co[k] = p.dout ? R::load(static_cast<const T*>(p.dout) + row * p.out_rs + col[k], cnt[k]) : none;
            cd[k] = p.res ? R::load(static_cast<const T*>(p.res) + row * p.res_rs + col[k], cnt[k]) : none;
        }
        const float m = p.stats[2 * row], r = p.stats[2 * row + 1];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float s[VE], o[VE], w[VE];
            kw[k].get(w);
            R::unpack(cs[k], s);
            R::unpack(co[k], o);
#pragma unroll
            for (int e = 0; e < VE; ++e) {                 // (past the row's end o is zero)
                const float ow = o[e] * w[e];
                sum[0] += ow;
                sum[1] = __builtin_fmaf(ow, (s[e] - m) * r, sum[1]);
            }
        }
        team_sum<WPR>(sum, red[turn], wave);
        turn ^= 1;
        const float m0 = sum[0] * inv, m1 = sum[1] * inv;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float s[VE], o[VE], d[VE], w[VE];
            kw[k].get(w);
            R::unpack(cs[k], s);
            R::unpack(co[k], o);
            R::unpack(cd[k], d);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float h = (s[e] - m) * r;
                aw[k][e] = __builtin_fmaf(o[e], h, aw[k][e]);
                ab[k][e] += o[e];
                d[e] = __builtin_fmaf(r, (o[e] * w[e] - m0) - h * m1, d[e]);
            }
            R::store(static_cast<T*>(p.dx) + row * p.dim + col[k], d, cnt[k]);
        }
    }
    // the workgroup's column sums, its rows' teams in order
    float* part = p.part + int64_t(blockIdx.x) * 2 * p.dim;
    for (int t = 0; t < ROWS; ++t) {
        if (int(threadIdx.x) / TEAM == t) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    float v[2] = {aw[k][e], ab[k][e]};
                    const int c = col[k] + e;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if constexpr (ROWS > 1) {
                            if (t > 0) v[i] += cols[i * TEAM * EPT + c];
                            if (t + 1 < ROWS) cols[i * TEAM * EPT + c] = v[i];
                        }
                        if (t + 1 == ROWS && e < cnt[k]) part[i * p.dim + c] = v[i];
                    }
                }
            }
        }
        if constexpr (ROWS > 1) __syncthreads();
    }
}

int rows_at_once(int64_t dim) { return dim <= 1024 ? 4 : 1; }
int64_t parts_of(int64_t rows, int64_t dim) {
    const int at = rows_at_once(dim);
    const int64_t n = (rows + at - 1) / at;
    return n < kParts ? n : kParts;
}

}  // namespace

int64_t layer_norm_bwd_space(int64_t rows, int64_t dim) { return parts_of(rows, dim) * 2 * dim * 4; }

hipError_t layer_norm_fwd_launch(const ss_layer_norm_args* a, hipStream_t stream) {
    LayerParams p{};
    p.rows = a->rows; p.dim = int(a->dim); p.eps = a->eps;
    p.x_rs = a->x_row_stride; p.res_rs = a->residual_row_stride; p.out_rs = a->out_row_stride; p.s_rs = a->residual_out_row_stride;
    p.x = a->x; p.res = a->residual; p.w = a->weight; p.b = a->bias;
    p.out = a->out; p.s = a->residual_out; p.stats = a->stats;
    const int at = rows_at_once(a->dim);
    const int64_t want = (a->rows + at - 1) / at;
    return for_types(a->dtype, a->w_dtype, [&](auto t, auto tw) {
        return for_row(a->dim, [&](auto wpr, auto ept) {
            hipLaunchKernelGGL((layer_norm_fwd<decltype(t), decltype(tw), decltype(wpr)::value, decltype(ept)::value>),
                               dim3(unsigned(want < 2048 ? want : 2048)), dim3(kBlock<decltype(wpr)::value>), 0, stream, p);
            return hipGetLastError();
        });
    });
}

hipError_t layer_norm_bwd_launch(const ss_layer_norm_bwd_args* g, hipStream_t stream) {
    LayerParams p{};
    p.rows = g->rows; p.dim = int(g->dim);
    p.x_rs = g->s_row_stride; p.out_rs = g->dout_row_stride; p.res_rs = g->dresidual_out_row_stride;
    p.x = g->s; p.w = g->weight; p.stats = const_cast<float*>(g->stats);
    p.dout = g->dout; p.res = g->dresidual_out; p.dx = g->dx;
    p.part = static_cast<float*>(g->workspace);
    const int64_t parts = parts_of(g->rows, g->dim);
    return for_types(g->dtype, g->w_dtype, [&](auto t, auto tw) {
        if (p.rows > 0) {
            const hipError_t e = for_row(g->dim, [&](auto wpr, auto ept) {
                hipLaunchKernelGGL((layer_norm_bwd<decltype(t), decltype(tw), decltype(wpr)::value, decltype(ept)::value>),
                                   dim3(unsigned(parts)), dim3(kBlock<decltype(wpr)::value>), 0, stream, p);
                return hipGetLastError();
            });
            if (e != hipSuccess) return e;
        }
        const ColSums c{p.part, p.rows > 0 ? parts : 0, 2 * int64_t(p.dim), p.dim, {g->dweight, g->dbias, nullptr}};
        hipLaunchKernelGGL((norm_col_sums<decltype(tw)>), dim3(unsigned((p.dim + 63) / 64), 2), dim3(64 * kSumWaves), 0, stream, c);
        return hipGetLastError();
    });
}

}  // namespace ss

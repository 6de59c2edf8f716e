// Teams of lanes that hold a row each, their sums, and the column sums over rows
// that the norms' backward passes leave in parts (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/mamba_ss.h"
#include "norm_rows.hpp"
#include "ss_device.hpp"

namespace ss {

namespace {

constexpr int kSumWaves = 16;                 // column sums: waves per workgroup

// a lane's weights in their own type; HOLD: in registers, else read at each use
// (from the caches: 16 fp32 weights a lane of three vectors would spill)
template <typename T, typename TW, bool HOLD>
struct PackedWeights {
    static constexpr int VE = rowvec<T>::VE, PER = rowvec<TW>::VE, N = VE / PER;
    uint4 v[HOLD ? N : 1];
    const TW* at;
    int n;
    __device__ __forceinline__ void load(const TW* p, int n_) {
        at = p;
        n = n_;
        if constexpr (HOLD) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = rowvec<TW>::load(p + i * PER, n - i * PER);
        }
    }
    // (unpacked at each use: the compiler would do it once, ahead of the rows)
    __device__ __forceinline__ void get(float (&o)[VE]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t[PER];
            uint4 w;
            if constexpr (HOLD) w = v[i];
            else w = rowvec<TW>::load(at + i * PER, n - i * PER);
            __asm__ volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
            rowvec<TW>::unpack(w, t);
#pragma unroll
            for (int e = 0; e < PER; ++e) o[i * PER + e] = t[e];
        }
    }
};

// sums over the waves of a row's team; red: two buffers, used in turn, so one
// barrier a sum is enough
template <int WPR, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (*red)[N], int wave) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<64>(v[i]);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) red[wave][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) t += red[w][i];
            v[i] = t;
        }
    }
}

// WPR waves hold a row, EPT elements a lane (WPR * 64 * EPT >= dim); a
// workgroup of at least 4 waves.
template <int WPR> constexpr int kBlock = 64 * (WPR > 4 ? WPR : 4);

// out[c] = sum over the parts of part[i * stride + blockIdx.y * dim + c], in a
// fixed order: wave i takes rows i, i + kSumWaves, ...
struct ColSums { const float* part; int64_t parts, stride; int dim; void* out[3]; };

template <typename TW>
__global__ __launch_bounds__(64 * kSumWaves) void norm_col_sums(const ColSums p) {
    if (!p.out[blockIdx.y]) return;
    __shared__ float red[kSumWaves][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = int(blockIdx.x) * 64 + lane;
    float acc = 0.f;
    if (c < p.dim) {
        const float* at = p.part + int64_t(blockIdx.y) * p.dim + c;
#pragma unroll 8
        for (int64_t i = wv; i < p.parts; i += kSumWaves) acc += at[i * p.stride];
    }
    red[wv][lane] = acc;
    __syncthreads();
    if (wv == 0 && c < p.dim) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kSumWaves; ++i) t += red[i][lane];
        io<TW>::store(static_cast<TW*>(p.out[blockIdx.y]) + c, t);
    }
}

// f(integral_constant<WPR>, integral_constant<EPT>) for a row of dim elements
template <typename F>
hipError_t for_row(int64_t dim, F&& f) {
    const auto I = [](auto v) { return v; };
    using std::integral_constant;
    if (dim <= 512) return f(I(integral_constant<int, 1>{}), I(integral_constant<int, 8>{}));
    if (dim <= 1024) return f(I(integral_constant<int, 1>{}), I(integral_constant<int, 16>{}));
    if (dim <= 2048) return f(I(integral_constant<int, 4>{}), I(integral_constant<int, 8>{}));
    if (dim <= 4096) return f(I(integral_constant<int, 4>{}), I(integral_constant<int, 16>{}));
    if (dim <= 8192) return f(I(integral_constant<int, 8>{}), I(integral_constant<int, 16>{}));
    return f(I(integral_constant<int, 16>{}), I(integral_constant<int, 16>{}));
}
template <typename F>
hipError_t for_types(int dtype, int w_dtype, F&& f) {
    switch (dtype) {
        case SS_F32: return f(float{}, float{});
        case SS_BF16: return w_dtype == SS_F32 ? f(bf16_t{}, float{}) : f(bf16_t{}, bf16_t{});
        default: return w_dtype == SS_F32 ? f(_Float16{}, float{}) : f(_Float16{}, _Float16{});
    }
}

}  // namespace

}  // namespace ss

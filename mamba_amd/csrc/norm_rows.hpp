// Rows read and written by the norm kernels: 16-byte vectors at any element
// alignment, and sums over aligned sets of lanes (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "ss_device.hpp"

namespace ss {

// Global memory takes 16-byte accesses at any element address (a misaligned
// one costs the extra cache line it touches), so rows of odd widths use the
// same vectors; only a row's last, partial vector goes element by element.
typedef uint32_t words_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t words_at4 __attribute__((ext_vector_type(4), aligned(4)));

template <typename T>
struct rowvec {
    static constexpr int VE = 16 / int(sizeof(T));
    using words = std::conditional_t<sizeof(T) == 2, words_at2, words_at4>;

    // elements [0, n) of p (n at most VE; 0 or less: none), zero past them
    static __device__ __forceinline__ uint4 load(const T* p, int n) {
        if (n >= VE) {
            const words w = *reinterpret_cast<const words*>(p);
            return make_uint4(w.x, w.y, w.z, w.w);
        }
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < VE - 1; ++e) {
            if (e < n) {
                if constexpr (sizeof(T) == 4) w[e] = *reinterpret_cast<const uint32_t*>(p + e);
                else w[e >> 1] |= uint32_t(*reinterpret_cast<const uint16_t*>(p + e)) << (16 * (e & 1));
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&o)[VE]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = __uint_as_float(w[k]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (__is_same(T, bf16_t)) {
                    o[2 * k] = __uint_as_float(w[k] << 16);
                    o[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
                } else {
                    o[2 * k] = float(__builtin_bit_cast(_Float16, uint16_t(w[k] & 0xffffu)));
                    o[2 * k + 1] = float(__builtin_bit_cast(_Float16, uint16_t(w[k] >> 16)));
                }
            }
        }
    }
    static __device__ __forceinline__ void store(T* p, const float (&v)[VE], int n) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
            else if constexpr (__is_same(T, bf16_t)) w[k] = io<bf16_t>::pack2(v[2 * k], v[2 * k + 1]);
            else w[k] = uint32_t(__builtin_bit_cast(uint16_t, _Float16(v[2 * k]))) |
                        (uint32_t(__builtin_bit_cast(uint16_t, _Float16(v[2 * k + 1]))) << 16);
        }
        if (n >= VE) {
            *reinterpret_cast<words*>(p) = words{w[0], w[1], w[2], w[3]};
            return;
        }
#pragma unroll
        for (int e = 0; e < VE - 1; ++e) {
            if (e < n) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p + e) = w[e];
                else *reinterpret_cast<uint16_t*>(p + e) = uint16_t(w[e >> 1] >> (16 * (e & 1)));
            }
        }
    }
    // VE elements of a weight vector of type TW as float
    template <typename TW>
    static __device__ __forceinline__ void weights(const TW* p, int n, float (&o)[VE]) {
        if constexpr (sizeof(TW) == sizeof(T)) {
            unpack(load(reinterpret_cast<const T*>(p), n), o);
        } else {
#pragma unroll
            for (int h = 0; h < VE; h += 4) {
                float t[4];
                rowvec<float>::unpack(rowvec<float>::load(reinterpret_cast<const float*>(p) + h, n - h), t);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[h + e] = t[e];
            }
        }
    }
};

// 4 consecutive elements at any element alignment, the first cnt of them and zero past them
typedef uint32_t half4_at2 __attribute__((ext_vector_type(2), aligned(2)));
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

// Sum over each aligned set of N lanes (N a power of two up to 64), in every
// lane of it.  Within 16 lanes by DPP: once quads agree, a half-row mirror
// brings the other quad of 8 lanes, and a rotation by 8 the other half row.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
    const auto dpp = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (N >= 2) v += dpp(v, std::integral_constant<int, 0xB1>{});    // quad_perm [1,0,3,2]
    if constexpr (N >= 4) v += dpp(v, std::integral_constant<int, 0x4E>{});    // quad_perm [2,3,0,1]
    if constexpr (N >= 8) v += dpp(v, std::integral_constant<int, 0x141>{});   // row_half_mirror
    if constexpr (N >= 16) v += dpp(v, std::integral_constant<int, 0x128>{});  // row_ror:8
    if constexpr (N >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if constexpr (N >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}

// 1 / (1 + e^-z); 0 and 1 far out
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + expf(-z)); }

}  // namespace ss

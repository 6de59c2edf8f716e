// Products of bf16 terms on the matrix cores (gfx950): fp32 values as sums of bf16
// terms, and operands read from LDS tiles.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "norm_rows.hpp"
#include "ss_device.hpp"

namespace ss {

namespace la {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

template <typename T> constexpr int kTerms = sizeof(T) == 4 ? 3 : __is_same(T, bf16_t) ? 1 : 2;

__device__ __forceinline__ f4 mfma(const u4& a, const u4& b, const f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float lo_half(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_half(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// x0, x1 as N bf16 terms each, packed (x0 low).  2 terms: both rounded, 2^-18 off
// at most.  3 terms, exact: the first cut (so that none of a finite value is
// infinite), 16 bits left over; the second rounded, so that the third, what is left, has either
// sign.  CUT: the second cut as well, where no product of terms is left out.
template <int N, bool CUT = false>
__device__ __forceinline__ void split(float x0, float x1, uint32_t (&t)[N]) {
    if constexpr (N <= 2) {
        t[0] = io<bf16_t>::pack2(x0, x1);
        if constexpr (N == 2) t[1] = io<bf16_t>::pack2(x0 - lo_half(t[0]), x1 - hi_half(t[0]));
    } else {
        const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
        t[0] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        const float r0 = x0 - __uint_as_float(u0 & 0xffff0000u), r1 = x1 - __uint_as_float(u1 & 0xffff0000u);
        if constexpr (CUT) t[1] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), 0x07060302u);
        else t[1] = io<bf16_t>::pack2(r0, r1);
        const float s0 = r0 - lo_half(t[1]), s1 = r1 - hi_half(t[1]);
        t[2] = __builtin_amdgcn_perm(__float_as_uint(s1), __float_as_uint(s0), 0x07060302u);
    }
}

// No instruction moves across: without it the scheduler raises the loads and
// splits of all steps to the front and runs out of registers.
__device__ __forceinline__ void stage_end() { __builtin_amdgcn_sched_barrier(0); }

// c[i] += sum of the products of a[i]'s NA and b[i]'s NB terms whose order is at
// most kMax (left out: with 2 up to 2^-22 of a product, with 1 2^-16), small ones first.  I independent sums
// at once: a product then need not wait for the one before it.  ai, bi: which operand
// the sums take (a stride of 0 shares one).
template <int I, int SA, int SB, int NA, int NB, int kMax>
__device__ __forceinline__ void mfma_terms(const u4 (*a)[NA], const u4 (*b)[NB], f4* const (&c)[I]) {
#pragma unroll
    for (int o = kMax; o >= 0; --o) {
#pragma unroll
        for (int x = 0; x < NA; ++x) {
            const int y = o - x;
            if (y < 0 || y >= NB) continue;
#pragma unroll
            for (int i = 0; i < I; ++i) *c[i] = mfma(a[SA * i][x], b[SB * i][y], *c[i]);
        }
    }
}

// Slot i of lane group g holds token 4 g + i (i < 4) or 16 + 4 g + i - 4.
// The 8 tokens of a column of a row-major LDS tile; block: first column of the 4
// that this lane reads for its 16-lane group.
template <int STRIDE>
__device__ __forceinline__ u4 load_tokens(const uint16_t* tile, int block, int lane) {
    const int g = lane >> 4, c = lane & 15;
    const uint16_t* p = tile + (4 * g + (c >> 2)) * STRIDE + block;
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
    const u2 hi = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 16 * STRIDE)));
    return u4{lo.x, lo.y, hi.x, hi.y};
}

// The state's tile t (16 rows), register r of lane group g: row of the state
__device__ __forceinline__ int state_row(int t, int g, int r) { return 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r; }

// 4 consecutive elements, the first cnt of them
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
}  // namespace la

}  // namespace ss

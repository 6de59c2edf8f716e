// The norm over all gradients of a model, and the gradients clipped to it, on
// gfx950:
//
//   norm = sqrt(sum over tensors and elements of g^2),  out = g min(1, max_norm / (norm + eps))
//
// Two passes over the gradients in chunks of kChunk elements, any number of
// tensors to a launch's table (up to kTable, passed by value with the launch,
// so a captured graph holds it): sums of squares, one per chunk; then one
// workgroup joins them, in a fixed order; then the products.  Squares are
// summed in 64 bits: gradients of 1e-30 or 1e30 neither vanish nor overflow
// (their squares do in 32 bits), and HBM, not the adder, bounds the pass.
// The second pass takes the last table first and each table's chunks from the last one
// down, as what the first pass read last may still be in the last-level cache (256 MB);
// the other tables follow in order (all of them downwards: 173.0 us for 171.5).  The 129 M bf16
// gradients of a 24-layer 768-wide model (218 tensors, three tables): 171 us, 777 MB
// at 4.5 TB/s, 66 of them the sums, 93 the products and 5 the join.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/mamba_ss.h"
#include "norm_rows.hpp"
#include "ops_kernels.hpp"
#include "ss_device.hpp"

namespace ss {

namespace {

constexpr int kTable = 96;              // tensors per launch: the table stays below 4 KiB of arguments
constexpr int kChunk = 16384;           // elements per workgroup
constexpr int kJoin = 1024;             // threads that join the chunks' sums

struct ClipTable {
    const void* in[kTable];
    void* out[kTable];
    int64_t n[kTable];
    uint32_t first[kTable + 1];         // first chunk of each tensor
    uint8_t dtype[kTable];
    int count;
};

// the tensor that a chunk belongs to: the last one whose first chunk is at or before it
__device__ __forceinline__ int tensor_of(const ClipTable& t, uint32_t chunk) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// f(element offset, elements) for this thread's vectors of a chunk
template <typename T, typename F>
__device__ __forceinline__ void vectors(int64_t n, int64_t at, F&& f) {
    constexpr int VE = rowvec<T>::VE;
    const int cnt = int(n - at < kChunk ? n - at : kChunk);
#pragma unroll 4
    for (int i = int(threadIdx.x) * VE; i < cnt; i += 256 * VE) f(at + i, cnt - i);
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int64_t n, int64_t at) {
    using R = rowvec<T>;
    double s = 0.0;
    vectors<T>(n, at, [&](int64_t i, int k) {
        float v[R::VE];
        R::unpack(R::load(p + i, k), v);
#pragma unroll
        for (int e = 0; e < R::VE; ++e) s = __builtin_fma(double(v[e]), double(v[e]), s);
    });
    return s;
}

__global__ __launch_bounds__(256) void clip_squares(const ClipTable t, double* sums) {
    const int i = tensor_of(t, blockIdx.x);
    const int64_t at = int64_t(blockIdx.x - t.first[i]) * kChunk, n = t.n[i];
    double s;
    if (t.dtype[i] == SS_F32) s = chunk_squares(static_cast<const float*>(t.in[i]), n, at);
    else if (t.dtype[i] == SS_BF16) s = chunk_squares(static_cast<const bf16_t*>(t.in[i]), n, at);
    else s = chunk_squares(static_cast<const _Float16*>(t.in[i]), n, at);
    __shared__ double red[256];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int m = 128; m >= 1; m >>= 1) {
        if (int(threadIdx.x) < m) red[threadIdx.x] += red[threadIdx.x + m];
        __syncthreads();
    }
    if (threadIdx.x == 0) sums[blockIdx.x] = red[0];
}

__global__ __launch_bounds__(kJoin) void clip_join(const double* sums, int64_t n, float max_norm, float eps, float* norm,
                                                   float* coef) {
    __shared__ double red[kJoin];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kJoin) s += sums[i];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int m = kJoin / 2; m >= 1; m >>= 1) {
        if (int(threadIdx.x) < m) red[threadIdx.x] += red[threadIdx.x + m];
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    const float v = float(sqrt(red[0])), c = max_norm / (v + eps);
    *norm = v;
    *coef = c > 1.f ? 1.f : c;              // (NaN stays)
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* p, T* o, int64_t n, int64_t at, float c) {
    using R = rowvec<T>;
    if (p == o && c == 1.f) return;
    vectors<T>(n, at, [&](int64_t i, int k) {
        float v[R::VE];
        R::unpack(R::load(p + i, k), v);
#pragma unroll
        for (int e = 0; e < R::VE; ++e) v[e] *= c;
        R::store(o + i, v, k);
    });
}

__global__ __launch_bounds__(256) void clip_scale(const ClipTable t, const float* coef) {
    const uint32_t chunk = gridDim.x - 1 - blockIdx.x;
    const int i = tensor_of(t, chunk);
    const int64_t at = int64_t(chunk - t.first[i]) * kChunk, n = t.n[i];
    const float c = *coef;
    if (t.dtype[i] == SS_F32) chunk_scale(static_cast<const float*>(t.in[i]), static_cast<float*>(t.out[i]), n, at, c);
    else if (t.dtype[i] == SS_BF16) chunk_scale(static_cast<const bf16_t*>(t.in[i]), static_cast<bf16_t*>(t.out[i]), n, at, c);
    else chunk_scale(static_cast<const _Float16*>(t.in[i]), static_cast<_Float16*>(t.out[i]), n, at, c);
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// The next table from tensor i on (empty tensors left out, at most 2^30
// chunks); returns the tensor after its last one.
int64_t fill(ClipTable& t, const ss_clip_grads_args* a, int64_t i) {
    t.count = 0;
    t.first[0] = 0;
    for (; i < a->count && t.count < kTable; ++i) {
        if (a->numels[i] == 0) continue;
        const int64_t end = t.first[t.count] + chunks_of(a->numels[i]);
        if (end > (int64_t(1) << 30)) break;
        t.in[t.count] = a->grads[i];
        t.out[t.count] = a->outs[i];
        t.n[t.count] = a->numels[i];
        t.dtype[t.count] = uint8_t(a->dtypes[i]);
        t.first[++t.count] = uint32_t(end);
    }
    return i;
}

}  // namespace

int64_t clip_grads_chunks(const ss_clip_grads_args* a) {
    int64_t n = 0;
    for (int64_t i = 0; i < a->count; ++i) n += chunks_of(a->numels[i]);
    return n;
}

hipError_t clip_grads_launch(const ss_clip_grads_args* a, hipStream_t stream) {
    // workspace: the factor (16 bytes), then a sum for each chunk
    float* coef = static_cast<float*>(a->workspace);
    double* sums = reinterpret_cast<double*>(static_cast<char*>(a->workspace) + 16);
    int64_t done = 0;
    ClipTable t, last;
    int tables = 0;
    for (int64_t i = 0; i < a->count;) {
        i = fill(t, a, i);
        if (t.count == 0) break;
        last = t;
        ++tables;
        hipLaunchKernelGGL(clip_squares, dim3(t.first[t.count]), dim3(256), 0, stream, t, sums + done);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        done += t.first[t.count];
    }
    hipLaunchKernelGGL(clip_join, dim3(1), dim3(kJoin), 0, stream, sums, done, a->max_norm, a->eps, a->norm, coef);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (tables == 0) return hipSuccess;
    const auto scale = [&](const ClipTable& tab) {
        hipLaunchKernelGGL(clip_scale, dim3(tab.first[tab.count]), dim3(256), 0, stream, tab, coef);
        return hipGetLastError();
    };
    e = scale(last);                        // the last table first
    if (e != hipSuccess) return e;
    for (int64_t i = 0; tables > 1; --tables) {
        i = fill(t, a, i);
        e = scale(t);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ss

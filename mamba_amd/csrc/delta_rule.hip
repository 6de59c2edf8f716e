// The gated delta rule on gfx950: the launches of a prompt or a training step
// (kernels in delta_rule_chunk.hpp), and the recurrence for one token.
//
// A pass is two launches, the chunks' inverses and the walk over the chunks; the
// backward is the walk back and the gradients of all chunks side by side.  A walk is
// serial along a row, so with few rows it is cut into segments that run side by side:
// over a segment a state S becomes M S + N, with M and N the same walk's result from the
// identity and from zero; they are joined along the row (dr_join), and each
// segment is then walked from the state it starts with.  Back, dS becomes M^T dS + N'.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "bf16_terms.hpp"
#include "delta_rule.hpp"
#include "norm_rows.hpp"
#include "ops_kernels.hpp"
#include "ss_device.hpp"

namespace ss {

namespace {

using namespace la;

// The states that the segments start from, in place of their own: S <- M S + N along the
// row (REV: M^T, from the last segment on).  Value columns do not meet: two waves have 16 (every second pair
// of tiles each; S's terms through LDS).  M comes through LDS in 3 terms, as the walk left it, CW columns at a time,
// the next slices and the next N on their way meanwhile.
// Serial along the row, a latency a segment: 24 rows of 20 steps at 64 keys 30 us, 32 rows of 3 steps at 128 20 (56 and 34 with
// loads behind branches, one step ahead, and one wave a column tile), 4 rows of 15 steps at 256 187 (319 with one wave).
template <int KP> constexpr int kJoinTiles = KP <= 128 ? 4 : 2;           // column tiles of a workgroup, two waves each
template <int KP, bool REV>
__global__ __launch_bounds__(128 * kJoinTiles<KP>) void dr_join(const DrParams p) {
    constexpr int CT = kJoinTiles<KP>, WAVES = 2, NTH = 64 * CT * WAVES;
    constexpr int NK = KP / 32, NP = NK / WAVES, CW = 64, MST = KP + 8, TERM = CW * MST, PER = KP / 8, N = 3 * CW * PER / NTH;
    constexpr int SL = KP / CW, AHEAD = KP <= 128 ? 2 : 1, STEPS = SL < AHEAD ? 2 : 1;    // slices of an M, those on their way, segments the loop takes at a time
    __shared__ __attribute__((aligned(16))) uint16_t ms[3 * TERM];       // CW columns of M, a row each
    __shared__ __attribute__((aligned(16))) u4 parts[CT][NK][3][64];
    const int tid = int(threadIdx.x), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), ct = wave % CT, own_pair = wave / CT;    // pairs own_pair, + WAVES ...
    const int64_t bh = blockIdx.x;
    const int col = int(blockIdx.y) * 16 * CT + 16 * ct + c, steps = p.segs - 1;
    const bool live = col - c < p.V;
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 S[2 * NP], own[2 * NP];                            // tiles 2 (own_pair + WAVES j) + e at 2 j + e
    u4 sf[NK][3];                                         // S before the step, all keys
    u4 in[AHEAD][N];
    const auto tile = [&](int t) { return 2 * ((t >> 1) * WAVES + own_pair) + (t & 1); };
#pragma unroll
    for (int t = 0; t < 2 * NP; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = state_row(tile(t), g, r);
            S[t][r] = p.init && key < p.K && col < p.V ? p.init[(bh * p.K + key) * p.V + col] : 0.f;
        }
    const auto seg_of = [&](int i) { return bh * p.segs + (REV ? p.segs - 1 - i : i); };
    // (what is past the tensors reads as zero and is not stored: no branch waits for the loads)
    constexpr int none = int(0x80000000u);
    const auto place = [&](int t) { return 32 * (tile(t) >> 1) < p.Kp ? (c * p.Kp + 16 * tile(t) + 4 * g) * 4 : none; };
    const auto add_of = [&](int i) {
        return make_rsrc_n(p.seg_add + (seg_of(i) * p.Vp + (live ? col - c : 0)) * p.Kp, live ? 16 * p.Kp * 4 : 0);
    };
    const auto fetch = [&](int slice, u4 (&to)[N]) {
        const int i = slice / SL, c0 = slice % SL * CW;
        const rsrc_t from = make_rsrc_n(p.seg_mul + seg_of(i < steps ? i : 0) * 3 * p.Kp * p.Kp, i < steps ? p.Kp * p.Kp * 6 : 0);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int x = tid + k * NTH, at = c0 + x / PER % CW, key = x % PER * 8;
            const int off = ((x / (CW * PER) * p.Kp + at) * p.Kp + key) * 2;
            to[k] = __builtin_amdgcn_raw_buffer_load_b128(from, at < p.Kp && key < p.Kp ? off : none, 0, 0);
        }
    };
    const auto fetch_own = [&](int i) {
        const rsrc_t from = add_of(i < steps ? i : 0);
#pragma unroll
        for (int t = 0; t < 2 * NP; ++t)
            own[t] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(from, place(t), 0, 0));
    };
    const auto keep = [&](int i) {
        const rsrc_t to = add_of(i);
#pragma unroll
        for (int t = 0; t < 2 * NP; ++t) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, S[t]), to, place(t), 0, 0);
    };
    fetch_own(0);
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) fetch(x, in[x]);
    for (int i0 = 0; i0 < steps; i0 += STEPS) {
#pragma unroll
        for (int x = 0; x < SL * STEPS; ++x) {
            const int i = i0 + x / SL, c0 = x % SL * CW;
            if (i >= steps) break;
            if (x % SL == 0) {
                keep(i);
#pragma unroll
                for (int k = 0; k < NP; ++k) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const f4& from = S[2 * k + (h >> 1)];
                        uint32_t t[3];
                        split<3>(from[2 * (h & 1)], from[2 * (h & 1) + 1], t);
#pragma unroll
                        for (int n = 0; n < 3; ++n) sf[k][n][h] = t[n];
                    }
                }
#pragma unroll
                for (int t = 0; t < 2 * NP; ++t) S[t] = own[t];
                fetch_own(i + 1);
            }
            lds_barrier();
            if (x % SL == 0) {
#pragma unroll
                for (int k = 0; k < NP; ++k)
#pragma unroll
                    for (int n = 0; n < 3; ++n) parts[ct][k * WAVES + own_pair][n][lane] = sf[k][n];
            }
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int at = tid + k * NTH;
                *reinterpret_cast<u4*>(ms + at / (CW * PER) * TERM + at / PER % CW * MST + at % PER * 8) = in[x % AHEAD][k];
            }
            lds_barrier();
            fetch(i0 * SL + x + AHEAD, in[x % AHEAD]);
            stage_end();                                  // (the compiler would issue them after the products)
            if (x % SL == 0) {
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int n = 0; n < 3; ++n) sf[k][n] = parts[ct][k][n][lane];
            }
            if constexpr (REV) {                          // rows of M^T: these columns, all keys
#pragma unroll
                for (int j = c0 / 32 / WAVES; j < (c0 + CW) / 32 / WAVES; ++j) {
                    f4* const to[2] = {&S[2 * j], &S[2 * j + 1]};
#pragma unroll
                    for (int k = 0; k < NK; ++k) {
                        u4 a[2][3];
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int n = 0; n < 3; ++n)
                                a[e][n] = *reinterpret_cast<const u4*>(ms + n * TERM + (16 * tile(2 * j) + 8 * (c >> 2) + 4 * e + (c & 3) - c0) * MST + 8 * g + 32 * k);
                        mfma_terms<2, 1, 0, 3, 3, 2>(a, &sf[k], to);
                    }
                }
            } else {                                      // all rows of M, these columns
                typedef __attribute__((address_space(3))) s4 lds_s4;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    f4* const to[2] = {&S[2 * j], &S[2 * j + 1]};
#pragma unroll
                    for (int k = c0 / 32; k < (c0 + CW) / 32; ++k) {
                        u4 a[2][3];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint16_t* at = ms + (32 * k - c0 + 8 * g + (c >> 2)) * MST + 16 * tile(2 * j) + 8 * (c & 3) + 4 * e;
#pragma unroll
                            for (int n = 0; n < 3; ++n) {
                                const u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + n * TERM)));
                                const u2 hi = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + n * TERM + 4 * MST)));
                                a[e][n] = u4{lo.x, lo.y, hi.x, hi.y};
                            }
                        }
                        mfma_terms<2, 1, 0, 3, 3, 2>(a, &sf[k], to);
                    }
                }
            }
        }
    }
    keep(steps);
}

// The heads of a group share q and k: out[r, j, :] = sum over i of part[r, j * rep + i, :], heads in order.
// W neighbouring elements a thread (4 where dim is a multiple of 4).  16384 rows of 4 groups of 6 heads of 64 keys, bf16: 36 us
// for both, 218 MB (64 with one element a thread and 64-bit divisions).
template <typename T, int W>
__global__ __launch_bounds__(256) void dr_group_sum(const float* dq, T* outq, const float* dk, T* outk, int64_t rows, int rep, int dim) {
    const float* part = blockIdx.y ? dk : dq;
    T* out = blockIdx.y ? outk : outq;
    const uint32_t per = uint32_t(dim / W);
    const int64_t step = int64_t(gridDim.x) * 256, n = rows * per;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) {
        const int64_t row = n <= 0xffffffffll ? int64_t(uint32_t(i) / per) : i / per;
        const int c = int(i - row * per) * W;
        const float* from = part + row * rep * dim + c;
        if constexpr (W == 4) {
            f4 s = *reinterpret_cast<const f4*>(from);
            for (int r = 1; r < rep; ++r) s += *reinterpret_cast<const f4*>(from + int64_t(r) * dim);
            const float v[4] = {s[0], s[1], s[2], s[3]};
            store4<T>(out + row * dim + c, v, 4);
        } else {
            float s = from[0];
            for (int r = 1; r < rep; ++r) s += from[int64_t(r) * dim];
            io<T>::store(out + row * dim + c, s);
        }
    }
}

template <typename F>
hipError_t for_type(int32_t dtype, F&& f) {
    switch (dtype) {
        case SS_F32: return f(float{});
        case SS_BF16: return f(bf16_t{});
        default: return f(_Float16{});
    }
}

int terms(int32_t dtype) { return dtype == SS_F32 ? 3 : dtype == SS_BF16 ? 1 : 2; }

// Compute units.  Rows are cut into segments, enough for one workgroup each, or for the two that fit
// where tiles and registers are small (1 x 32768 tokens x 24 heads of 64 x 64: walk 223 us with 10 segments, 170 with 21).
// With wider keys only the walk back gains from the second one (bf16, 1 x 32768 tokens x 16 heads of 128 x 128:
// forward and backward 2,422 us to 2,246, forward alone 710 to 729, as its join takes twice the steps), so a prompt has one.
// The segments' own states cost about what their walk does, so two are not worth it: 8 x 2048 tokens
// x 24 heads of 64 x 64, bf16, 88 us for the states and 113 for the walk, 157 in one.  A segment keeps at least 4 chunks (2 x 515 tokens x 6 heads of 96 x 80, fp32:
// 104 us in two of 9 chunks, 76 in four).
constexpr int64_t kUnits = 256, kSegChunksMin = 4, kSegsMin = 3;

struct Plan {
    int64_t bh, nch, plan, state, rows, mul;     // (batch, head) pairs, chunks; floats of a chunk's plan, a state, a chunk's rows, an M
    int segs, seg_chunks, chunk;
};
// train: of a forward whose states are kept, and of its backward
Plan plan_of(const ss_delta_rule_args& a, bool train) {
    Plan p{};
    p.chunk = dr_chunk(a.d_key, terms(a.dtype));
    p.bh = a.batch * a.heads;
    p.nch = (a.seqlen + p.chunk - 1) / p.chunk;
    const int64_t kp = dr_round32(a.d_key), vp = dr_round16(a.d_value);
    p.plan = dr_plan_bytes(p.chunk) / 4;
    p.state = kp * vp;
    p.rows = p.chunk * vp;
    p.mul = kp * kp * 3 / 2;
    const int64_t walks = p.bh * ((a.d_value + 63) / 64);
    const bool two = train ? dr_two(a.d_key, terms(a.dtype)) : a.d_key <= 64;
    int64_t segs = walks > 0 ? (two ? 2 : 1) * kUnits / walks : 1;
    if (segs > p.nch / kSegChunksMin) segs = p.nch / kSegChunksMin;
    if (segs < kSegsMin) segs = 1;
    const int64_t per = p.nch > 0 ? (p.nch + segs - 1) / segs : 1;
    p.segs = p.nch > 0 ? int((p.nch + per - 1) / per) : 1;
    p.seg_chunks = int(per);
    return p;
}

// floats at offsets of one buffer, each part 16-byte aligned
struct Parts {
    int64_t bytes = 0;
    int64_t take(int64_t floats) {
        const int64_t at = bytes;
        bytes += (floats * 4 + 15) / 16 * 16;
        return at;
    }
};
struct Saved { int64_t plan, states, err, mul, bytes; };
Saved saved_of(const Plan& p) {
    Saved s{};
    Parts parts;
    s.plan = parts.take(p.bh * p.nch * p.plan);
    s.states = parts.take(p.bh * p.nch * p.state);
    s.err = parts.take(p.bh * p.nch * p.rows);
    s.mul = p.segs > 1 ? parts.take(p.bh * p.segs * p.mul) : 0;
    s.bytes = parts.bytes;
    return s;
}
struct FwdSpace { int64_t add, plan, mul, bytes; };
FwdSpace fwd_space(const ss_delta_rule_args& a, const Plan& p) {
    FwdSpace s{};
    Parts parts;
    if (p.segs > 1) s.add = parts.take(p.bh * p.segs * p.state);
    if (!a.saved) {
        s.plan = parts.take(p.bh * p.nch * p.plan);
        if (p.segs > 1) s.mul = parts.take(p.bh * p.segs * p.mul);
    }
    s.bytes = parts.bytes;
    return s;
}
struct BwdSpace { int64_t dstates, derr, add, dq, dk, bytes; };
BwdSpace bwd_space(const ss_delta_rule_args& a, const Plan& p) {
    BwdSpace s{};
    Parts parts;
    s.dstates = parts.take(p.bh * p.nch * p.state);
    s.derr = parts.take(p.bh * p.nch * p.rows);
    if (p.segs > 1) s.add = parts.take(p.bh * p.segs * p.state);
    if (a.groups != a.heads) {
        s.dq = parts.take(p.bh * a.seqlen * a.d_key);
        s.dk = parts.take(p.bh * a.seqlen * a.d_key);
    }
    s.bytes = parts.bytes;
    return s;
}

DrParams params_of(const ss_delta_rule_args& a, const Plan& plan) {
    DrParams p{};
    p.B = a.batch; p.L = a.seqlen; p.H = a.heads; p.BH = a.batch * a.heads;
    p.K = int(a.d_key); p.V = int(a.d_value); p.Kp = dr_round32(a.d_key); p.Vp = dr_round16(a.d_value);
    p.rep = int(a.heads / a.groups); p.nch = int(plan.nch);
    p.scale = a.scale;
    p.q = dr_rows(a.q, a.q_batch_stride, a.q_len_stride, a.q_head_stride, p.rep, p.K, p.L);
    p.k = dr_rows(a.k, a.k_batch_stride, a.k_len_stride, a.k_head_stride, p.rep, p.K, p.L);
    p.v = dr_rows(a.v, a.v_batch_stride, a.v_len_stride, a.v_head_stride, 1, p.V, p.L);
    p.g = a.g; p.g_b = a.g_batch_stride; p.g_l = a.g_len_stride; p.g_h = a.g_head_stride;
    p.beta = a.beta; p.be_b = a.beta_batch_stride; p.be_l = a.beta_len_stride; p.be_h = a.beta_head_stride;
    p.lens = a.lengths;
    p.segs = plan.segs; p.seg_chunks = plan.seg_chunks;
    return p;
}

// (p.o is set by then: out, or the backward's dout)
void set_whole(DrParams& p, int32_t dtype) {
    const int size = dtype == SS_F32 ? 4 : 2;
    p.whole = dr_whole(p.q, p.K, size) && dr_whole(p.k, p.K, size) && dr_whole(p.v, p.V, size) && dr_whole(p.o, p.V, size) &&
              p.H * (p.K > p.V ? p.K : p.V) < (int64_t(1) << 22);
}

float* at(void* base, int64_t bytes) { return reinterpret_cast<float*>(static_cast<char*>(base) + bytes); }

// the walk, of segments side by side after what they start from
hipError_t walk(int32_t dtype, DrParams p, bool rev, hipStream_t stream) {
    const auto launch = [&](const DrParams& q) {
        return for_type(dtype, [&](auto t) { return dr_walk_launch<decltype(t)>(q, rev, stream); });
    };
    if (p.segs > 1) {
        DrParams own = p;
        own.local = 1;
        hipError_t e = launch(own);
        if (e != hipSuccess) return e;
        const auto join = [&](auto kp) {
            constexpr int KP = decltype(kp)::value, CT = kJoinTiles<KP>;
            const dim3 grid(unsigned(p.B * p.H), unsigned(p.V + 16 * CT - 1) / (16 * CT)), block(128 * CT);
            if (rev) hipLaunchKernelGGL((dr_join<KP, true>), grid, block, 0, stream, p);
            else hipLaunchKernelGGL((dr_join<KP, false>), grid, block, 0, stream, p);
            return hipGetLastError();
        };
        const int64_t kp = dr_keys(p.K);
        e = kp == 64 ? join(std::integral_constant<int, 64>{}) : kp == 128 ? join(std::integral_constant<int, 128>{})
                                                                          : join(std::integral_constant<int, 256>{});
        if (e != hipSuccess) return e;
    }
    return launch(p);
}

}  // namespace

int64_t delta_rule_chunks(const ss_delta_rule_args* a) {
    const Plan p = plan_of(*a, false);
    return p.bh * p.nch;
}
int64_t delta_rule_saved_bytes(const ss_delta_rule_args* a) { return saved_of(plan_of(*a, true)).bytes; }
int64_t delta_rule_fwd_space(const ss_delta_rule_args* a) { return fwd_space(*a, plan_of(*a, a->saved)).bytes; }
int64_t delta_rule_bwd_space(const ss_delta_rule_bwd_args* g) { return bwd_space(g->f, plan_of(g->f, true)).bytes; }

hipError_t delta_rule_fwd_launch(const ss_delta_rule_args* a, hipStream_t stream) {
    const Plan plan = plan_of(*a, a->saved);
    const FwdSpace sp = fwd_space(*a, plan);
    const Saved sv = saved_of(plan);
    DrParams p = params_of(*a, plan);
    p.o = dr_rows(a->out, a->out_batch_stride, a->out_len_stride, a->out_head_stride, 1, p.V, p.L);
    set_whole(p, a->dtype);
    p.init = a->initial_state; p.last = a->last_state;
    p.seg_add = at(a->workspace, sp.add);
    if (a->saved) {
        p.plan = at(a->saved, sv.plan); p.states = at(a->saved, sv.states); p.err = at(a->saved, sv.err);
        p.seg_mul = reinterpret_cast<uint16_t*>(at(a->saved, sv.mul));
    } else {
        p.plan = at(a->workspace, sp.plan);
        p.seg_mul = reinterpret_cast<uint16_t*>(at(a->workspace, sp.mul));
    }
    if (plan.nch > 0) {
        const hipError_t e = for_type(a->dtype, [&](auto t) { return dr_prep_launch<decltype(t)>(p, stream); });
        if (e != hipSuccess) return e;
    }
    return walk(a->dtype, p, false, stream);
}

hipError_t delta_rule_bwd_launch(const ss_delta_rule_bwd_args* g, hipStream_t stream) {
    const ss_delta_rule_args& a = g->f;
    const Plan plan = plan_of(a, true);
    const BwdSpace sp = bwd_space(a, plan);
    const Saved sv = saved_of(plan);
    DrParams p = params_of(a, plan);
    p.o = dr_rows(g->dout, g->dout_batch_stride, g->dout_len_stride, g->dout_head_stride, 1, p.V, p.L);
    set_whole(p, a.dtype);
    p.init = g->dlast_state; p.last = g->dinitial_state;
    p.plan = at(a.saved, sv.plan); p.states = at(a.saved, sv.states); p.err = at(a.saved, sv.err); p.seg_mul = reinterpret_cast<uint16_t*>(at(a.saved, sv.mul));
    p.dstates = at(a.workspace, sp.dstates); p.derr = at(a.workspace, sp.derr); p.seg_add = at(a.workspace, sp.add);
    hipError_t e = walk(a.dtype, p, true, stream);
    if (e != hipSuccess || plan.nch == 0) return e;
    const bool part = p.rep > 1;
    p.dq = part ? at(a.workspace, sp.dq) : g->dq; p.dk = part ? at(a.workspace, sp.dk) : g->dk; p.dv = g->dv;
    p.dg = g->dg; p.dbeta = g->dbeta;
    e = for_type(a.dtype, [&](auto t) { return dr_grads_launch<decltype(t)>(p, stream); });
    if (e != hipSuccess || !part) return e;
    return for_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t rows = a.batch * a.seqlen * a.groups;
        const auto go = [&](auto w) {
            constexpr int W = decltype(w)::value;
            const int64_t want = (rows * (p.K / W) + 255) / 256;
            hipLaunchKernelGGL((dr_group_sum<T, W>), dim3(unsigned(want < 65536 ? want : 65536), 2), dim3(256), 0, stream,
                               static_cast<const float*>(p.dq), static_cast<T*>(g->dq), static_cast<const float*>(p.dk),
                               static_cast<T*>(g->dk), rows, p.rep, p.K);
        };
        if (p.K % 4 == 0) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 1>{});
        return hipGetLastError();
    });
}

namespace {

// One token.  With the state S before it, u = beta (v - a S^T k) and
// q^T (a S + k u^T) = a S^T q + (q . k) u, so both sums over the state's rows are taken
// together and the state is read once: bound by its bytes (64 rows x 16 heads of 128 x 128, bf16: 134 MB in 25.9 us,
// 5.2 TB/s with what the last-level cache holds; 24 heads of 64 x 64: 4.2 us, a launch).  A workgroup owns 64 value
// columns of one (batch, head); thread (i, c) holds 4 neighbouring columns (1 where rows are not
// 16-byte aligned) of up to RPT rows i, i + RG ... in registers.
template <typename T, int RPT, bool VEC>
__global__ __launch_bounds__(256) void dr_update(const ss_delta_rule_update_args a) {
    constexpr int W = VEC ? 4 : 1, CT = 64 / W, RG = 256 / CT;
    const int64_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads, j = h / (a.heads / a.groups);
    const int tid = int(threadIdx.x), c = tid % CT, rg = tid / CT, n = int(blockIdx.y) * 64 + c * W;
    const int K = int(a.d_key), V = int(a.d_value);
    __shared__ float qs[256], ks[256];
    __shared__ __attribute__((aligned(16))) float redk[4][64], redq[4][64], redqk[4];
    float* S = a.state + b * a.state_batch_stride + h * a.state_head_stride;
    float s[RPT][W];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int d = rg + i * RG;
        const bool in = d < K && n < V;
        if constexpr (VEC) {
            const float4 t = in ? *reinterpret_cast<const float4*>(S + int64_t(d) * V + n) : make_float4(0.f, 0.f, 0.f, 0.f);
            s[i][0] = t.x; s[i][1] = t.y; s[i][2] = t.z; s[i][3] = t.w;
        } else {
            s[i][0] = in ? S[int64_t(d) * V + n] : 0.f;
        }
    }
    qs[tid] = tid < K ? io<T>::load(static_cast<const T*>(a.q) + b * a.q_batch_stride + j * a.q_head_stride + tid) : 0.f;
    ks[tid] = tid < K ? io<T>::load(static_cast<const T*>(a.k) + b * a.k_batch_stride + j * a.k_head_stride + tid) : 0.f;
    const float dec = expf(a.g[b * a.g_batch_stride + h * a.g_head_stride]), beta = a.beta[b * a.beta_batch_stride + h * a.beta_head_stride];
    float v[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
        v[w] = n + w < V ? io<T>::load(static_cast<const T*>(a.v) + b * a.v_batch_stride + h * a.v_head_stride + n + w) : 0.f;
    __syncthreads();
    // a wave's 64 lanes: CT columns (or all 64) by 64 / CT rows
    float kS[W] = {}, qS[W] = {};
    const float qk = lanes_sum<64>(qs[tid] * ks[tid]);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int d = rg + i * RG;
        const float kd = d < K ? ks[d] : 0.f, qd = d < K ? qs[d] : 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            s[i][w] *= dec;
            kS[w] = __builtin_fmaf(kd, s[i][w], kS[w]);
            qS[w] = __builtin_fmaf(qd, s[i][w], qS[w]);
        }
    }
    const int wave = tid >> 6, lane = tid & 63;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if constexpr (VEC) {
            kS[w] += __shfl_xor(kS[w], 16, 64); kS[w] += __shfl_xor(kS[w], 32, 64);
            qS[w] += __shfl_xor(qS[w], 16, 64); qS[w] += __shfl_xor(qS[w], 32, 64);
        }
        if (!VEC || lane < 16) {
            redk[wave][c * W + w] = kS[w];
            redq[wave][c * W + w] = qS[w];
        }
    }
    if (lane == 0) redqk[wave] = qk;
    __syncthreads();
    const float dot = (redqk[0] + redqk[1]) + (redqk[2] + redqk[3]);
    float u[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int m = c * W + w;
        const float kx = (redk[0][m] + redk[1][m]) + (redk[2][m] + redk[3][m]), qx = (redq[0][m] + redq[1][m]) + (redq[2][m] + redq[3][m]);
        u[w] = beta * (v[w] - kx);
        if (rg == 0 && n + w < V)
            io<T>::store(static_cast<T*>(a.out) + b * a.out_batch_stride + h * a.out_head_stride + n + w, a.scale * __builtin_fmaf(dot, u[w], qx));
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int d = rg + i * RG;
        if (d >= K || n >= V) continue;
        const float kd = ks[d];
#pragma unroll
        for (int w = 0; w < W; ++w) s[i][w] = __builtin_fmaf(kd, u[w], s[i][w]);
        if constexpr (VEC) *reinterpret_cast<float4*>(S + int64_t(d) * V + n) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        else S[int64_t(d) * V + n] = s[i][0];
    }
}

template <typename T>
hipError_t update_t(const ss_delta_rule_update_args* a, hipStream_t stream) {
    const bool vec = a->d_value % 4 == 0 && a->state_batch_stride % 4 == 0 && a->state_head_stride % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(a->state) & 15) == 0;
    const dim3 grid(unsigned(a->batch * a->heads), unsigned(a->d_value + 63) / 64);
    if (vec && a->d_key <= 64) hipLaunchKernelGGL((dr_update<T, 4, true>), grid, dim3(256), 0, stream, *a);
    else if (vec && a->d_key <= 128) hipLaunchKernelGGL((dr_update<T, 8, true>), grid, dim3(256), 0, stream, *a);
    else if (vec) hipLaunchKernelGGL((dr_update<T, 16, true>), grid, dim3(256), 0, stream, *a);
    else if (a->d_key <= 128) hipLaunchKernelGGL((dr_update<T, 32, false>), grid, dim3(256), 0, stream, *a);
    else hipLaunchKernelGGL((dr_update<T, 64, false>), grid, dim3(256), 0, stream, *a);
    return hipGetLastError();
}

}  // namespace

hipError_t delta_rule_update_launch(const ss_delta_rule_update_args* a, hipStream_t stream) {
    return for_type(a->dtype, [&](auto t) { return update_t<decltype(t)>(a, stream); });
}

}  // namespace ss

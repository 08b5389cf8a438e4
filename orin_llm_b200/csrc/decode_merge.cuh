// The merge of partial attention results (m, l, O) shared by the decode kernels: the running log-sum-exp merge, the
// hand-over between the CTAs of one kv head, and what the CTA that holds the merged result does with it.
#pragma once

#include "attn_internal.h"

namespace oattn {

namespace {

constexpr int kMergeThreads = 128;     // threads of a CTA that hold pieces of the block, unless said otherwise

// ---- how the threads of a CTA share one kv head's [G][HD] block of fp32 values ------------------------------------
// The block is cut into float4 pieces; thread `tid` < THREADS owns pieces tid, tid + THREADS, ... (piece -> row = head in the group,
// col4 = which four dims).  With HD = 128 a warp owns whole rows (rows warp, warp + 4, ...), a lane four dims.
template <int HD, bool WIDE, int THREADS = kMergeThreads>
struct Slots {
    static constexpr int F4_PER_ROW = HD / 4;
    static constexpr int ROWS = WIDE ? 16 : 8;
    static constexpr int N = ROWS * F4_PER_ROW / THREADS;
    static_assert(N >= 1, "at least one piece per thread");
    __device__ static __forceinline__ int row(int tid, int k) { return (tid + k * THREADS) / F4_PER_ROW; }
    __device__ static __forceinline__ int col4(int tid, int k) { return (tid + k * THREADS) % F4_PER_ROW; }
};

// Running log-sum-exp merge of one piece: acc = sum_i e^(m_i - M) O_i, L = sum_i e^(m_i - M) l_i, M = max m_i.
struct RunState {
    float M, L;
    float4 acc;
};
__device__ __forceinline__ RunState run_empty() { return RunState{-CUDART_INF_F, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)}; }

// Adds n <= 8 parts; c turns a difference of m values into a base-2 exponent.
__device__ __forceinline__ void run_add(RunState& s, const float (&m)[8], const float (&l)[8], const float4 (&o)[8], int n, float c) {
    float mx = s.M;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) mx = fmaxf(mx, m[i]);
    if (mx == -CUDART_INF_F) return;           // only empty parts so far
    const float a = (s.M == -CUDART_INF_F) ? 0.f : fast_exp2((s.M - mx) * c);
    s.L *= a;
    s.acc.x *= a; s.acc.y *= a; s.acc.z *= a; s.acc.w *= a;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i < n) {
            const float w = (m[i] == -CUDART_INF_F) ? 0.f : fast_exp2((m[i] - mx) * c);
            s.L = fmaf(w, l[i], s.L);
            s.acc.x = fmaf(w, o[i].x, s.acc.x);
            s.acc.y = fmaf(w, o[i].y, s.acc.y);
            s.acc.z = fmaf(w, o[i].z, s.acc.z);
            s.acc.w = fmaf(w, o[i].w, s.acc.w);
        }
    }
    s.M = mx;
}

// Merges parts 0..n-1 of one kv head, stored [part][G][HD] and [part][G][2], in index order.  The parts were written by
// other SMs a moment ago: read them from L2 (ld.cg), never through this SM's L1.  This runs on the critical path of the
// launch as a chain of L2 round trips, so a pass issues every load it needs before it uses any of them: the lanes that
// share a row (HD/4 of them) each fetch the (m, l) of one part and exchange the weights by shuffle, and every lane keeps
// its O pieces of up to 16 parts in flight.  Called by all THREADS threads.
template <int HD, bool WIDE, int THREADS = kMergeThreads>
__device__ __forceinline__ void merge_parts(const float* o_base, const float* ml_base, int n, int G, float c,
                                            RunState (&st)[Slots<HD, WIDE, THREADS>::N]) {
    using S = Slots<HD, WIDE, THREADS>;
    constexpr int LPR = S::F4_PER_ROW;            // lanes per row: 32 or 16
    constexpr int PASS = 16;                      // parts per pass
    constexpr int KB = S::N < 2 ? S::N : 2;       // pieces per thread handled together
    const int tid = threadIdx.x;
    const int j = tid % LPR;
#pragma unroll
    for (int k = 0; k < S::N; ++k) st[k] = run_empty();
    for (int i0 = 0; i0 < n; i0 += PASS) {
        const int nn = min(PASS, n - i0);
#pragma unroll
        for (int k0 = 0; k0 < S::N; k0 += KB) {
            float2 ml[KB];
            float4 o[KB][PASS];
#pragma unroll
            for (int kk = 0; kk < KB; ++kk) {
                const int row = S::row(tid, k0 + kk), c4 = S::col4(tid, k0 + kk);
                const bool valid = row < G;
                ml[kk] = make_float2(-CUDART_INF_F, 0.f);
                if (valid && j < nn) ml[kk] = __ldcg(reinterpret_cast<const float2*>(ml_base + ((size_t)(i0 + j) * G + row) * 2));
#pragma unroll
                for (int i = 0; i < PASS; ++i) {
                    o[kk][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (valid && i < nn) o[kk][i] = __ldcg(reinterpret_cast<const float4*>(o_base + ((size_t)(i0 + i) * G + row) * HD + c4 * 4));
                }
            }
#pragma unroll
            for (int kk = 0; kk < KB; ++kk) {
                RunState& r = st[k0 + kk];
                float mx = ml[kk].x;          // (over all lanes of the row: those past the parts hold -inf and need it just as well)
#pragma unroll
                for (int off = LPR / 2; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off, LPR));
                const float m_new = fmaxf(r.M, mx);
                const bool empty = m_new == -CUDART_INF_F;
                const float a = (empty || r.M == -CUDART_INF_F) ? 0.f : fast_exp2((r.M - m_new) * c);
                const float w = (empty || ml[kk].x == -CUDART_INF_F) ? 0.f : fast_exp2((ml[kk].x - m_new) * c);
                r.L *= a;
                r.acc.x *= a; r.acc.y *= a; r.acc.z *= a; r.acc.w *= a;
#pragma unroll
                for (int i = 0; i < PASS; ++i) {
                    // parts are added in index order; lanes >= nn hold w = 0 and o = 0
                    const float wi = __shfl_sync(0xffffffffu, w, i, LPR);
                    const float li = __shfl_sync(0xffffffffu, ml[kk].y, i, LPR);
                    r.L = fmaf(wi, li, r.L);
                    r.acc.x = fmaf(wi, o[kk][i].x, r.acc.x);
                    r.acc.y = fmaf(wi, o[kk][i].y, r.acc.y);
                    r.acc.z = fmaf(wi, o[kk][i].z, r.acc.z);
                    r.acc.w = fmaf(wi, o[kk][i].w, r.acc.w);
                }
                r.M = m_new;
            }
        }
    }
}

template <int HD, bool WIDE, int THREADS = kMergeThreads>
__device__ __forceinline__ void store_part(float* o_base, float* ml_base, int G, const RunState (&st)[Slots<HD, WIDE, THREADS>::N]) {
    using S = Slots<HD, WIDE, THREADS>;
    const int tid = threadIdx.x;
#pragma unroll
    for (int k = 0; k < S::N; ++k) {
        const int row = S::row(tid, k), c4 = S::col4(tid, k);
        if (row < G) {
            *reinterpret_cast<float4*>(o_base + (size_t)row * HD + c4 * 4) = st[k].acc;
            if (c4 == 0) *reinterpret_cast<float2*>(ml_base + (size_t)row * 2) = make_float2(st[k].M, st[k].L);
        }
    }
}

// All threads of the CTA store their share of a partial, then one ticket is drawn from `counter`, which counts
// 0..n-1 and wraps to zero.  Returns true in every thread of the CTA that drew the last ticket.  Its later reads of
// the other arrivals' partials go to L2 (ld.cg), where those stores were made visible before their tickets were drawn,
// and cannot start before the ticket is known (barrier + branch).
__device__ __forceinline__ bool arrive_last(unsigned* counter, int n) {
    __shared__ unsigned s_ticket;
    if (n <= 1) return true;
    __syncthreads();                 // every thread's stores precede thread 0's fence (the fence is cumulative)
    if (threadIdx.x == 0) {
        __threadfence();
        s_ticket = atomicInc(counter, (unsigned)(n - 1));
    }
    __syncthreads();
    return s_ticket == (unsigned)(n - 1);
}

// q8_1 form of four consecutive output values per lane (see store_q8_group): a group of 32 values sits in 8 neighbouring
// lanes.  Called by all 32 lanes; `valid` only guards the stores.
__device__ __forceinline__ void store_q8_group4(float4 x, bool valid, size_t flat, int8_t* qs, float* scales) {
    float amax = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
    for (int off = 4; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const float d = __fdiv_rn(amax, 127.0f);
    if (!valid) return;
    char4 q = make_char4(0, 0, 0, 0);
    if (amax != 0.0f) {
        q.x = (signed char)roundf(__fdiv_rn(x.x, d));
        q.y = (signed char)roundf(__fdiv_rn(x.y, d));
        q.z = (signed char)roundf(__fdiv_rn(x.z, d));
        q.w = (signed char)roundf(__fdiv_rn(x.w, d));
    }
    *reinterpret_cast<char4*>(qs + flat) = q;
    if ((flat & 31) == 0) scales[flat >> 5] = d;
}

__device__ __forceinline__ float4 normalised(const RunState& s) {
    if (!(s.L > 0.f)) return make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(s.acc.x / s.L, s.acc.y / s.L, s.acc.z / s.L, s.acc.w / s.L);
}

// What the CTA that holds the merged (M, L, O) of the G heads from head0 on does with it.  Called by all THREADS
// threads.
template <int HD, bool WIDE, int THREADS = kMergeThreads, typename Args>
__device__ __forceinline__ void emit_final(const Args& p, int head0, int G, const RunState (&st)[Slots<HD, WIDE, THREADS>::N]) {
    using S = Slots<HD, WIDE, THREADS>;
    const int tid = threadIdx.x;
    if (!p.emit_partial) {
#pragma unroll
        for (int k = 0; k < S::N; ++k) {
            const int row = S::row(tid, k), c4 = S::col4(tid, k);
            const bool valid = row < G;
            const size_t flat = (size_t)(head0 + row) * HD + c4 * 4;
            const float4 v = valid ? normalised(st[k]) : make_float4(0.f, 0.f, 0.f, 0.f);
            if (valid && p.out) *reinterpret_cast<float4*>(p.out + flat) = v;
            if (p.out_qs) store_q8_group4(v, valid, flat, p.out_qs, p.out_scales);
        }
        return;
    }
    // per-rank record {O, m, l, 0, 0}, m in natural-log units of the scaled score
#pragma unroll
    for (int k = 0; k < S::N; ++k) {
        const int row = S::row(tid, k), c4 = S::col4(tid, k);
        if (row < G) {
            float* rec = p.out + (size_t)(head0 + row) * (HD + PART_PAD);
            *reinterpret_cast<float4*>(rec + c4 * 4) = st[k].acc;
            if (c4 == 0) *reinterpret_cast<float4*>(rec + HD) = make_float4(st[k].M * p.scale, st[k].L, 0.f, 0.f);
        }
    }
}

} // namespace

} // namespace oattn

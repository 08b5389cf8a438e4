// Writing, reading back and rolling the 4-bit KV cache, and the prologue of the prefill call that uses it.
#include <math.h>

#include <mutex>

#include "kv_q4.cuh"

namespace oattn {

namespace {

template <int HD>
__device__ __forceinline__ void load_row(const float* src, int lane, float (&x)[Q4<HD>::EPL]) {
#pragma unroll
    for (int e = 0; e < Q4<HD>::EPL; ++e) x[e] = src[Q4<HD>::EPL * lane + e];
}

// ---- store: one warp per (token, head, K or V) row --------------------------------------------------------------
constexpr int kStoreWarps = 8;

template <int HD>
__global__ void __launch_bounds__(32 * kStoreWarps) kv_store_q4_kernel(uint8_t* cache, const float* k, const float* v, int heads,
                                                                       int n_ctx, int pos_base, int batch, const int* d_pos) {
    const int lane = threadIdx.x & 31;
    const long long job = (long long)blockIdx.x * kStoreWarps + (threadIdx.x >> 5);
    const long long row = job >> 1;                       // token * heads + head
    if (row >= (long long)batch * heads) return;
    const int head = (int)(row % heads), b = (int)(row / heads);
    const int pos = d_pos ? *d_pos : pos_base + b;
    if (pos < 0 || pos >= n_ctx) return;
    uint8_t* blk = cache + ((size_t)head * q4_blocks(n_ctx) + (pos >> 4)) * Q4<HD>::BLOCK;
    float x[Q4<HD>::EPL];
    load_row<HD>(((job & 1) ? v : k) + (size_t)row * HD, lane, x);
    const Q4Scale s = q4_scale<HD>(x, lane);
    const uint32_t codes = q4_codes<HD>(x, s);
    if (job & 1) q4_store_row<HD, true>(blk, pos & 15, codes, s, lane);
    else         q4_store_row<HD, false>(blk, pos & 15, codes, s, lane);
}

// ---- read back: a warp turns one row into fp16 ------------------------------------------------------------------
// (row `pos` of `blk`; dst = K and V rows of HD fp16 values)
template <int HD>
__device__ __forceinline__ void q4_load_row(const uint8_t* blk, int s, uint16_t* dk, uint16_t* dv, int lane) {
    using F = Q4<HD>;
    const int D = F::EPL * lane, g = D / 64;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const uint32_t sw = *reinterpret_cast<const uint32_t*>(blk + (which ? F::VS_OFF : F::KS_OFF) + s * F::SROWB + 4 * g);
        const float d = __half2float(__ushort_as_half((uint16_t)sw)), m = __half2float(__ushort_as_half((uint16_t)(sw >> 16)));
        uint16_t* dst = which ? dv : dk;
#pragma unroll
        for (int e = 0; e < F::EPL; e += 2) {
            const uint32_t c = blk[which ? q4_v_byte<HD>(s, D + e) : q4_k_byte<HD>(s, D + e)];
            *reinterpret_cast<uint32_t*>(dst + D + e) = pack_half2(q4_value(c & 15u, d, m), q4_value(c >> 4, d, m));
        }
    }
}

constexpr int kLoadWarps = 8;

template <int HD>
__global__ void __launch_bounds__(32 * kLoadWarps) kv_load_q4_kernel(const uint8_t* cache, uint16_t* kc, uint16_t* vc, int heads,
                                                                     int n_ctx, int row_base, int rows, int dst_ctx, int dst_base) {
    const long long job = (long long)blockIdx.x * kLoadWarps + (threadIdx.x >> 5);
    if (job >= (long long)heads * rows) return;
    const int head = (int)(job / rows), i = (int)(job % rows);
    const int pos = row_base + i;
    const uint8_t* blk = cache + ((size_t)head * q4_blocks(n_ctx) + (pos >> 4)) * Q4<HD>::BLOCK;
    const size_t dst = ((size_t)head * dst_ctx + dst_base + i) * HD;
    q4_load_row<HD>(blk, pos & 15, kc + dst, vc + dst, threadIdx.x & 31);
}

// ---- roll: one CTA per (layer, kv head) -------------------------------------------------------------------------
// Row r becomes row r + shift for n_keep <= r < n_ctx - shift, the last `shift` rows become zero.  A step composes
// kShiftBlocks blocks in shared memory from the rows `shift` further on and then writes them; what later steps read lies
// behind everything written so far, so one CTA can work in place.
constexpr int kShiftThreads = 256;
constexpr int kShiftBlocks = 8;

template <int HD>
__global__ void __launch_bounds__(kShiftThreads) kv_shift_q4_kernel(uint8_t* cache, int n_ctx, int n_keep, int shift) {
    using F = Q4<HD>;
    extern __shared__ __align__(16) uint8_t smem[];       // kShiftBlocks composed blocks
    const int nblk = q4_blocks(n_ctx);
    uint8_t* base = cache + (size_t)blockIdx.x * nblk * F::BLOCK;
    for (int b0 = n_keep >> 4; b0 < nblk; b0 += kShiftBlocks) {
        const int nb = min(kShiftBlocks, nblk - b0);
        // one warp per row
        for (int i = threadIdx.x >> 5; i < nb * 16; i += kShiftThreads / 32) {
            const int lane = threadIdx.x & 31;
            const int row = b0 * 16 + i;
            int src = row < n_keep || row >= n_ctx ? row : row + shift;
            const bool zero = row < n_ctx && src >= n_ctx;
            if (zero) src = row;
            const uint8_t* sb = base + (size_t)(src >> 4) * F::BLOCK;
            uint8_t* db = smem + (size_t)(i >> 4) * F::BLOCK;
            const int ss = src & 15, ds = i & 15;
            for (int D = 2 * lane; D < HD; D += 64) {
                db[q4_k_byte<HD>(ds, D)] = zero ? (uint8_t)0 : sb[q4_k_byte<HD>(ss, D)];
                db[q4_v_byte<HD>(ds, D)] = zero ? (uint8_t)0 : sb[q4_v_byte<HD>(ss, D)];
            }
            if (lane < 2 * F::NG) {
                const int off = (lane >= F::NG ? F::VS_OFF : F::KS_OFF), g = lane % F::NG;
                *reinterpret_cast<uint32_t*>(db + off + ds * F::SROWB + 4 * g) =
                    zero ? 0u : *reinterpret_cast<const uint32_t*>(sb + off + ss * F::SROWB + 4 * g);
            }
        }
        __syncthreads();
        uint4* dst = reinterpret_cast<uint4*>(base + (size_t)b0 * F::BLOCK);
        const uint4* from = reinterpret_cast<const uint4*>(smem);
        for (int i = threadIdx.x; i < nb * F::BLOCK / 16; i += kShiftThreads) dst[i] = from[i];
        __syncthreads();
    }
}

// ---- prefill prologue -------------------------------------------------------------------------------------------
// The chunk's tokens, one CTA each: q -> [bias, norm, RoPE] -> * scale*log2(e) -> fp16 (what the attention kernels read),
// k -> [bias, norm, RoPE] -> 4-bit row, v -> [bias] -> 4-bit row; the rows' fp16 values also go to the copies the attention
// reads.  The CTAs behind them turn the cache rows in front of the chunk into fp16.
constexpr int kPrologueThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kPrologueThreads) prefill_q4_prologue_kernel(const __grid_constant__ KvQ4PrologueArgs p) {
    using F = Q4<HD>;
    const PrefillArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.n_past + a.batch;
    const int nblk = q4_blocks(p.cache_ctx);
    const bool rope_q = (a.fuse & 1) != 0, rope_k = (a.fuse & 2) != 0, append = (a.fuse & 4) != 0;
    pdl_trigger();
    if ((int)blockIdx.x >= a.batch) {
        pdl_wait();
        const int expand = append ? a.n_past : rows;
        const long long job = (long long)(blockIdx.x - a.batch) * (kPrologueThreads / 32) + warp;
        if (job >= (long long)a.n_kv * expand) return;
        const int head = (int)(job / expand), pos = (int)(job % expand);
        const uint8_t* blk = p.cache + ((size_t)head * nblk + (pos >> 4)) * F::BLOCK;
        const size_t dst = ((size_t)head * rows + pos) * HD;
        q4_load_row<HD>(blk, pos & 15, reinterpret_cast<uint16_t*>(p.k16) + dst, reinterpret_cast<uint16_t*>(p.v16) + dst, lane);
        return;
    }
    // cos and sin in double: a key's code is a decision at a border, so the rotated key is rounded to fp32 once
    __shared__ double s_cos[HD / 2], s_sin[HD / 2];
    __shared__ float s_row[kPrologueThreads / 32][HD];
    const int b = blockIdx.x, pos = a.n_past + b;
    if (rope_q || rope_k) {
        for (int i = tid; i < a.rope.n_rot / 2; i += kPrologueThreads) {
            float f = p.freq[i];
            if (a.rope.freq_factors) f = __fdiv_rn(f, a.rope.freq_factors[i]);
            sincos((double)__fmul_rn((float)pos, f), &s_sin[i], &s_cos[i]);
        }
    }
    pdl_wait();
    __syncthreads();
    if (b == 0 && tid == 0 && a.status) *a.status = 0;
    const float qs = a.scale * LOG2E;
    const int jobs = a.n_head + (append ? 2 * a.n_kv : 0);
    float* row = s_row[warp];
    for (int job = warp; job < jobs; job += kPrologueThreads / 32) {
        const int kind = job < a.n_head ? 0 : (job < a.n_head + a.n_kv ? 1 : 2);
        const int head = kind == 0 ? job : (kind == 1 ? job - a.n_head : job - a.n_head - a.n_kv);
        const int heads = kind == 0 ? a.n_head : a.n_kv;
        const float* src = (kind == 0 ? a.q : (kind == 1 ? a.k_new : a.v_new)) + ((size_t)b * heads + head) * HD;
        const float* bias0 = kind == 0 ? a.pre.bias_q : (kind == 1 ? a.pre.bias_k : a.pre.bias_v);
        const float* bias = bias0 ? bias0 + (size_t)head * HD : nullptr;
        const float* nw = kind == 0 ? a.pre.norm_q : (kind == 1 ? a.pre.norm_k : nullptr);
        const float rn = nw ? warp_row_rnorm(src, bias, HD, a.pre.eps, lane) : 1.f;
        for (int e = lane; e < HD; e += 32) row[e] = pre_value(src, bias, nw, rn, e);
        __syncwarp();
        if (kind == 0 ? rope_q : (kind == 1 && rope_k)) {
            for (int pp = lane; pp < a.rope.n_rot / 2; pp += 32) {
                int i0, i1;
                rope_pair_index(a.rope.rope_type, pp, a.rope.n_rot, i0, i1);
                const double u = row[i0], w = row[i1], c = s_cos[pp], s = s_sin[pp];
                row[i0] = (float)(u * c - w * s);
                row[i1] = (float)(u * s + w * c);
            }
            __syncwarp();
        }
        float x[F::EPL];
#pragma unroll
        for (int e = 0; e < F::EPL; ++e) x[e] = row[F::EPL * lane + e];
        __syncwarp();
        if (kind == 0) {
            __half* dst = a.q16 + ((size_t)b * a.n_head + head) * HD + F::EPL * lane;
#pragma unroll
            for (int e = 0; e < F::EPL; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_half2(x[e] * qs, x[e + 1] * qs);
        } else {
            const Q4Scale s = q4_scale<HD>(x, lane);
            const uint32_t codes = q4_codes<HD>(x, s);
            uint8_t* blk = p.cache + ((size_t)head * nblk + (pos >> 4)) * F::BLOCK;
            if (kind == 2) q4_store_row<HD, true>(blk, pos & 15, codes, s, lane);
            else           q4_store_row<HD, false>(blk, pos & 15, codes, s, lane);
            __half* dst = (kind == 1 ? p.k16 : p.v16) + ((size_t)head * rows + pos) * HD + F::EPL * lane;
            const float d = __half2float(s.d), m = __half2float(s.m);
#pragma unroll
            for (int e = 0; e < F::EPL; e += 2)
                *reinterpret_cast<uint32_t*>(dst + e) = pack_half2(q4_value((codes >> (4 * e)) & 15u, d, m), q4_value((codes >> (4 * e + 4)) & 15u, d, m));
        }
    }
}

} // namespace

void rope_freq_table(const RopeArgs& r, float (&freq)[64]) {
    // a model has one (theta, n_rot); the last few are kept
    struct Entry { int n_rot = 0; float theta = 0.f; float freq[64]; };
    static Entry kept[4];
    static int next = 0;
    static std::mutex mutex;
    std::lock_guard<std::mutex> lock(mutex);
    Entry* e = nullptr;
    for (Entry& k : kept)
        if (k.n_rot == r.n_rot && k.theta == r.theta) e = &k;
    if (!e) {
        e = &kept[next];
        next = (next + 1) % 4;
        e->n_rot = r.n_rot;
        e->theta = r.theta;
        for (int i = 0; i < 64; ++i) {
            const float x = r.n_rot > 0 ? (-2.0f * (float)i) / (float)r.n_rot : 0.f;
            e->freq[i] = (float)exp2((double)x * log2((double)r.theta));
        }
    }
    for (int i = 0; i < 64; ++i) freq[i] = e->freq[i];
}

cudaError_t launch_kv_store_q4(uint8_t* cache, const float* k, const float* v, int heads, int head_dim, int n_ctx, int pos_base,
                               int batch, const int* d_pos, cudaStream_t stream, unsigned long long* launches) {
    const long long jobs = 2LL * batch * heads;
    const dim3 grid((unsigned)((jobs + kStoreWarps - 1) / kStoreWarps));
    if (head_dim == 128) kv_store_q4_kernel<128><<<grid, 32 * kStoreWarps, 0, stream>>>(cache, k, v, heads, n_ctx, pos_base, batch, d_pos);
    else                 kv_store_q4_kernel<64><<<grid, 32 * kStoreWarps, 0, stream>>>(cache, k, v, heads, n_ctx, pos_base, batch, d_pos);
    if (launches) *launches += 1;
    return cudaGetLastError();
}

cudaError_t launch_kv_load_q4(const uint8_t* cache, uint16_t* kc, uint16_t* vc, int heads, int head_dim, int n_ctx, int row_base,
                              int rows, int dst_ctx, int dst_base, cudaStream_t stream, unsigned long long* launches) {
    const long long jobs = (long long)heads * rows;
    const dim3 grid((unsigned)((jobs + kLoadWarps - 1) / kLoadWarps));
    if (head_dim == 128) kv_load_q4_kernel<128><<<grid, 32 * kLoadWarps, 0, stream>>>(cache, kc, vc, heads, n_ctx, row_base, rows, dst_ctx, dst_base);
    else                 kv_load_q4_kernel<64><<<grid, 32 * kLoadWarps, 0, stream>>>(cache, kc, vc, heads, n_ctx, row_base, rows, dst_ctx, dst_base);
    if (launches) *launches += 1;
    return cudaGetLastError();
}

cudaError_t launch_kv_shift_q4(uint8_t* cache, int n_layer, int n_kv, int head_dim, int n_ctx, int n_keep, int shift,
                               cudaStream_t stream, unsigned long long* launches) {
    const int grid = n_layer * n_kv;
    if (head_dim == 128) kv_shift_q4_kernel<128><<<grid, kShiftThreads, kShiftBlocks * Q4<128>::BLOCK, stream>>>(cache, n_ctx, n_keep, shift);
    else                 kv_shift_q4_kernel<64><<<grid, kShiftThreads, kShiftBlocks * Q4<64>::BLOCK, stream>>>(cache, n_ctx, n_keep, shift);
    if (launches) *launches += 1;
    return cudaGetLastError();
}

cudaError_t launch_prefill_q4_prologue(const KvQ4PrologueArgs& p, cudaStream_t stream, unsigned long long* launches) {
    const PrefillArgs& a = p.a;
    const long long jobs = (long long)a.n_kv * ((a.fuse & 4) ? a.n_past : a.n_past + a.batch);
    constexpr int W = kPrologueThreads / 32;
    const dim3 grid((unsigned)(a.batch + (jobs + W - 1) / W));
    const cudaError_t e = a.head_dim == 128 ? launch_dependent(prefill_q4_prologue_kernel<128>, grid, kPrologueThreads, 0, stream, 1, p)
                                            : launch_dependent(prefill_q4_prologue_kernel<64>, grid, kPrologueThreads, 0, stream, 1, p);
    if (launches) *launches += 1;
    return e;
}

} // namespace oattn

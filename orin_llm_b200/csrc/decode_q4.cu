// Single-token decode attention over the 4-bit KV cache (format: kv_q4.cuh), split over the sequence, in ONE launch.
//
// The sequence of every kv head is cut into slices, one CTA of eight warps each (grid = slices x kv heads, two CTAs per SM);
// a warp takes every eighth 16-position block of the slice and brings it to shared memory with cp.async, one contiguous
// piece, four blocks deep, for itself alone: no barrier across warps until the end.  The grid never depends on the
// position, so the launch replays from a CUDA graph.  The slices are merged as in decode.cu (decode_merge.cuh).
//
// The codes are never turned into values.  With x = m + d * code per row and 64-dim group g,
//     q . k  = sum_g d_g (q_g . code_g) + m_g sum(q_g)            P V = sum_k (P_k d_gk) code_k + sum_k P_k m_gk
// so the matrix instructions (m16n8k16, fp16 in, fp32 out) take the codes as they are: a masked nibble is an fp16
// subnormal, exactly code * 2^-24 or code * 2^-20, and the powers of two go into q and the final scale.  The left operands q and
// P d are fp32; a decode step has at most eight heads per CTA, so the other eight rows of the tile hold what the rounding of the
// first eight to fp16 left over (x = hi + lo, 22 bits together): the result keeps fp32 accuracy and the instruction count is
// the same.  q is scaled by a power of two per head, P d by a power of two that is lowered when a step of 2 or more is met,
// so that neither half leaves the fp16 range.
#include "decode_merge.cuh"
#include "kv_q4.cuh"

namespace oattn {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 4;                 // blocks in flight per warp

template <int HD>
struct Q4Smem {
    static constexpr int BLOCK = Q4<HD>::BLOCK;
    static constexpr int RING = kWarps * kStages * BLOCK;
    static constexpr int QF_OFF = RING;                                // q fragments [HD/16 steps][32 lanes][4 words]
    static constexpr int QF_BYTES = HD / 16 * 512;
    static constexpr int IN_OFF = QF_OFF + QF_BYTES;                   // fp32 rows: q [8], k_new, v_new
    static constexpr int CS_OFF = IN_OFF + 10 * HD * 4;                // cos, sin of q's angles [2][HD/2] fp32
    static constexpr int CD_OFF = CS_OFF + HD * 4;                     // the same for k_new in double
    static constexpr int NEW_OFF = CD_OFF + HD * 8;                    // codes of the new row per lane: [2][32] u32, scales [2][2] u32
    static constexpr int QS_OFF = NEW_OFF + 2 * 32 * 4 + 32;           // per head: group sums of q [8][2], unit [8]
    static constexpr int TOTAL = QS_OFF + 8 * 2 * 4 + 8 * 4;
    // merge buffers over the ring once it has drained: [warps][8 rows][HD + 8] fp32, then (m, l) [warps][8][2]
    static constexpr int MSTRIDE = HD + 8;
    static constexpr int ML_OFF = kWarps * 8 * MSTRIDE * 4;
    static_assert(ML_OFF + kWarps * 8 * 2 * 4 <= RING, "the merge area lies in the ring");
};

struct Q4Plan {
    int blocks, per_split, active;       // 16-row blocks in all, of one slice, slices that have any
};
__device__ __forceinline__ Q4Plan q4_plan(int npos, int n_splits) {
    Q4Plan s;
    s.blocks = (npos + 15) >> 4;
    const int units = (s.blocks + kWarps - 1) / kWarps;                // a unit: one block for each warp
    const int per = max(1, (units + n_splits - 1) / n_splits);
    s.per_split = per * kWarps;
    s.active = (units + per - 1) / per;
    return s;
}

__device__ __forceinline__ float2 half2_word(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }

// hi = fp16(x), lo = fp16(x - hi), for a pair
__device__ __forceinline__ void split_half2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    hi = pack_half2(x0, x1);
    const float2 h = half2_word(hi);
    lo = pack_half2(x0 - h.x, x1 - h.y);
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 2) decode_q4_kernel(const DecodeQ4Args p) {
    using F = Q4<HD>;
    using L = Q4Smem<HD>;
    using S = Slots<HD, false>;
    constexpr int NG = F::NG, NW = HD / 32;      // groups of a row, code words of a lane per K row
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = lane >> 2, t = lane & 3;
    const int hb = blockIdx.x % p.head_blocks, split = blockIdx.x / p.head_blocks, kvh = blockIdx.y;
    const int GA = p.n_head / p.n_kv;                        // heads of the kv head, and of this CTA
    const int head0 = kvh * GA + hb * p.heads_per_cta;
    const int G = min(p.heads_per_cta, GA - hb * p.heads_per_cta);

    pdl_trigger();
    if (p.overlap != 2) pdl_wait();
    const int npos = max(0, min(*p.d_pos + 1, p.n_ctx));
    const Q4Plan plan = q4_plan(npos, p.n_splits);
    if (split >= max(plan.active, 1)) return;
    const int vh = kvh * p.head_blocks + hb;                 // place of this CTA's heads in the scratch block
    const int GP = p.heads_per_cta;                          // rows kept there per slice
    if (plan.active == 0) {
        if (p.overlap == 2) pdl_wait();
        if (tid < kMergeThreads) {
            RunState st[S::N];
#pragma unroll
            for (int k = 0; k < S::N; ++k) st[k] = run_empty();
            emit_final<HD, false>(p, head0, G, st);
        }
        return;
    }
    const int blk0 = split * plan.per_split, blk1 = min(blk0 + plan.per_split, plan.blocks);
    const bool append = (p.fuse & 4) != 0;
    const bool last_slice = split == plan.active - 1;
    const bool owner = append && last_slice;
    const int new_pos = npos - 1;
    uint8_t* cache = p.cache + (size_t)kvh * q4_blocks(p.n_ctx) * F::BLOCK;
    uint8_t* ring = smem + warp * kStages * F::BLOCK;

    // block `b` of the sequence -> stage; 16-byte pieces, consecutive lanes
    auto load_block = [&](int b, int stage) {
        const uint8_t* src = cache + (size_t)b * F::BLOCK;
        const uint32_t dst = smem_u32(ring + stage * F::BLOCK);
#pragma unroll
        for (int i = 0; i < (F::BLOCK / 16 + 31) / 32; ++i) {
            const int c = lane + 32 * i;
            if (c < F::BLOCK / 16) cp_async_16(dst + 16 * c, src + 16 * c, 16);
        }
    };
    const int nb = blk1 - blk0 > warp ? (blk1 - blk0 - warp + kWarps - 1) / kWarps : 0;      // blocks of this warp
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
        if (s < nb) load_block(blk0 + warp + s * kWarps, s);
        cp_async_commit();
    }

    // ---- prologue -----------------------------------------------------------------------------------------------
    float* s_cos = reinterpret_cast<float*>(smem + L::CS_OFF);
    float* s_sin = s_cos + HD / 2;
    double* s_cd = reinterpret_cast<double*>(smem + L::CD_OFF);
    double* s_sd = s_cd + HD / 2;
    const bool rope_q = (p.fuse & 1) != 0, rope_k = (p.fuse & 2) != 0;
    if (rope_q || (rope_k && owner)) {
        const int half = p.rope.n_rot / 2;
        for (int i = tid; i < 2 * HD / 2; i += kThreads) {
            const int pair = i & (HD / 2 - 1);
            if (pair >= half) continue;
            const float f = rope_freq(pair, p.rope.n_rot, p.rope.theta, p.rope.freq_factors);
            if (i < HD / 2) rope_cs(new_pos, f, s_cos[pair], s_sin[pair]);
            else if (rope_k && owner) sincos((double)__fmul_rn((float)new_pos, f), &s_sd[pair], &s_cd[pair]);
        }
    }
    if (p.overlap == 2) pdl_wait();
    float* s_in = reinterpret_cast<float*>(smem + L::IN_OFF);
    float* s_qsum = reinterpret_cast<float*>(smem + L::QS_OFF);
    float* s_unit = s_qsum + 16;
    uint32_t* s_new = reinterpret_cast<uint32_t*>(smem + L::NEW_OFF);
    const int in_rows = G + (owner ? 2 : 0);
    for (int idx = tid; idx < in_rows * (HD / 4); idx += kThreads) {
        const int row = idx / (HD / 4), c4 = idx % (HD / 4);
        const float* src = row < G ? p.q + (size_t)(head0 + row) * HD : (row == G ? p.k_new : p.v_new) + (size_t)kvh * HD;
        const float* bias = row < G ? (p.pre.bias_q ? p.pre.bias_q + (size_t)(head0 + row) * HD : nullptr)
                                    : (row == G ? p.pre.bias_k : p.pre.bias_v);
        if (row >= G && bias) bias += (size_t)kvh * HD;
        float4 v = *reinterpret_cast<const float4*>(src + c4 * 4);
        if (bias) {
            const float4 bv = *reinterpret_cast<const float4*>(bias + c4 * 4);
            v.x += bv.x; v.y += bv.y; v.z += bv.z; v.w += bv.w;
        }
        *reinterpret_cast<float4*>(s_in + (row < G ? row : 8 + row - G) * HD + c4 * 4) = v;
    }
    __syncthreads();
    // Warp h: head h.  Norm, rotation, then the power of two that brings the largest |q| to [2^13, 2^14), and the group sums.
    if (warp < G) {
        float* row = s_in + warp * HD;
        if (p.pre.norm_q) {
            const float rn = warp_row_rnorm(row, nullptr, HD, p.pre.eps, lane);
            __syncwarp();
            for (int e = lane; e < HD; e += 32) row[e] = row[e] * rn * p.pre.norm_q[e];
            __syncwarp();
        }
        if (rope_q) {
            for (int pp = lane; pp < p.rope.n_rot / 2; pp += 32) {
                int i0, i1;
                rope_pair_index(p.rope.rope_type, pp, p.rope.n_rot, i0, i1);
                const float a = row[i0], b = row[i1], c = s_cos[pp], s = s_sin[pp];
                row[i0] = a * c - b * s;
                row[i1] = a * s + b * c;
            }
            __syncwarp();
        }
        float amax = 0.f;
        for (int e = lane; e < HD; e += 32) amax = fmaxf(amax, fabsf(row[e]));
#pragma unroll
        for (int off = 16; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        int k = 13 - ((int)(__float_as_uint(amax) >> 23) - 127);
        k = amax == 0.f ? 0 : max(-100, min(100, k));
        const float up = __uint_as_float((uint32_t)(127 + k) << 23);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            const float v = row[lane + 32 * i] * up;
            row[lane + 32 * i] = v;
            sum[i >> 1] += v;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
            for (int off = 16; off; off >>= 1) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], off);
            if (lane == 0) s_qsum[warp * 2 + g] = sum[g] * 5.9604644775390625e-8f;           // 2^-24
        }
        if (lane == 0) s_unit[warp] = __uint_as_float((uint32_t)(127 + 24 - k) << 23);         // back to q . k
    } else {
        for (int e = lane; e < HD; e += 32) s_in[warp * HD + e] = 0.f;
        if (lane < 2) s_qsum[warp * 2 + lane] = 0.f;
        if (lane == 0) s_unit[warp] = 1.f;
    }
    // the new row of K (warp 0) and V (warp 1): codes, into the cache and into s_new for this CTA's copy of the block
    if (owner && warp < 2) {
        float* row = s_in + (8 + warp) * HD;
        if (warp == 0 && p.pre.norm_k) {
            const float rn = warp_row_rnorm(row, nullptr, HD, p.pre.eps, lane);
            __syncwarp();
            for (int e = lane; e < HD; e += 32) row[e] = row[e] * rn * p.pre.norm_k[e];
            __syncwarp();
        }
        if (warp == 0 && rope_k) {
            for (int pp = lane; pp < p.rope.n_rot / 2; pp += 32) {
                int i0, i1;
                rope_pair_index(p.rope.rope_type, pp, p.rope.n_rot, i0, i1);
                const double a = row[i0], b = row[i1], c = s_cd[pp], s = s_sd[pp];
                row[i0] = (float)(a * c - b * s);
                row[i1] = (float)(a * s + b * c);
            }
            __syncwarp();
        }
        float x[F::EPL];
#pragma unroll
        for (int e = 0; e < F::EPL; ++e) x[e] = row[F::EPL * lane + e];
        const Q4Scale sc = q4_scale<HD>(x, lane);
        const uint32_t codes = q4_codes<HD>(x, sc);
        s_new[warp * 32 + lane] = codes;
        if (F::EPL * lane % 64 == 0) s_new[64 + warp * 2 + F::EPL * lane / 64] = q4_scale_word(sc);
        if (hb == 0) {
            uint8_t* blk = cache + (size_t)(new_pos >> 4) * F::BLOCK;
            if (warp == 0) q4_store_row<HD, false>(blk, new_pos & 15, codes, sc, lane);
            else           q4_store_row<HD, true>(blk, new_pos & 15, codes, sc, lane);
        }
    }
    __syncthreads();
    // q fragments: step 2i + o of word i takes the nibbles 0, 4 | 2, 6 (o = 0) or 1, 5 | 3, 7 (o = 1, whose codes read 16 times as
    // large); words: row r hi, row r lo (as row r + 8), and the same for k + 8
    for (int idx = tid; idx < HD / 16 * 32; idx += kThreads) {
        const int step = idx >> 5, ln = idx & 31, o = step & 1;
        const float* row = s_in + (ln >> 2) * HD + 32 * (step >> 1) + 8 * (ln & 3) + o;
        const float f = o ? 0.0625f : 1.f;
        uint4 w;
        split_half2(row[0] * f, row[4] * f, w.x, w.y);
        split_half2(row[2] * f, row[6] * f, w.z, w.w);
        *reinterpret_cast<uint4*>(smem + L::QF_OFF + idx * 16) = w;
    }
    __syncthreads();

    float qsum[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) qsum[g] = s_qsum[r * 2 + g];
    const float unit = s_unit[r];
    const float c = p.scale * LOG2E * unit;
    const uint4* qf = reinterpret_cast<const uint4*>(smem + L::QF_OFF) + lane;

    float o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f; }
    float om[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) om[g] = 0.f;
    float m_run = -CUDART_INF_F, l_run = 0.f;
    float pscale = 8192.f;                                   // P d is carried times this; 2^-2 once a step of 2 or more was met

    for (int it = 0; it < nb; ++it) {
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const int b = blk0 + warp + it * kWarps;
        uint8_t* blk = ring + (it % kStages) * F::BLOCK;
        const int nrow = npos - b * 16;                      // valid rows, where fewer than 16
        if (b == plan.blocks - 1) {
            if (owner) {
                // the new row, which is not (or not safely) in what was copied
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t codes = s_new[w * 32 + lane];
                    if (w == 0) {
                        if (F::EPL == 4) *reinterpret_cast<uint16_t*>(blk + q4_k_byte<HD>(new_pos & 15, F::EPL * lane)) = (uint16_t)codes;
                        else             blk[q4_k_byte<HD>(new_pos & 15, F::EPL * lane)] = (uint8_t)codes;
                    } else {
#pragma unroll
                        for (int e = 0; e < F::EPL; e += 2) blk[q4_v_byte<HD>(new_pos & 15, F::EPL * lane + e)] = (uint8_t)(codes >> (4 * e));
                    }
                }
                if (lane < 2 * NG) {
                    const int w = lane / NG, g = lane % NG;
                    *reinterpret_cast<uint32_t*>(blk + (w ? F::VS_OFF : F::KS_OFF) + (new_pos & 15) * F::SROWB + 4 * g) = s_new[64 + w * 2 + g];
                }
            } else if (!append && p.overlap == 2) {
                // copied ahead of the dependency wait: the newest row may have been written since
                const uint4* src = reinterpret_cast<const uint4*>(cache + (size_t)b * F::BLOCK);
                for (int i = lane; i < F::BLOCK / 16; i += 32) reinterpret_cast<uint4*>(blk)[i] = __ldcg(src + i);
            }
            __syncwarp();
            // rows past the end: whatever the memory held, their steps and offsets count as zero
            for (int i = lane; i < 2 * 16 * NG; i += 32) {
                const int row = (i % (16 * NG)) / NG;
                if (row >= nrow) reinterpret_cast<uint32_t*>(blk + F::KS_OFF)[i] = 0u;
            }
            __syncwarp();
        }

        // ---- S = q . K for two tiles of eight rows --------------------------------------------------------------
        float s[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t w[NW];
            if constexpr (NW == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(blk + (8 * j + r) * F::ROWB + t * 16);
                w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(blk + (8 * j + r) * F::ROWB + t * 8);
                w[0] = v.x; w[1] = v.y;
            }
            s[j][0] = s[j][1] = 0.f;
            const uint32_t* sc = reinterpret_cast<const uint32_t*>(blk + F::KS_OFF + (8 * j + 2 * t) * F::SROWB);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 2 * g; i < 2 * g + 2; ++i) {
                    const uint32_t w8 = w[i] >> 8;
                    const uint4 a0 = qf[(2 * i) * 32], a1 = qf[(2 * i + 1) * 32];
                    mma_16816(acc, a0.x, a0.y, a0.z, a0.w, w[i] & 0x000F000Fu, w8 & 0x000F000Fu);
                    mma_16816(acc, a1.x, a1.y, a1.z, a1.w, w[i] & 0x00F000F0u, w8 & 0x00F000F0u);
                }
                const float2 s0 = half2_word(sc[g]), s1 = half2_word(sc[NG + g]);
                s[j][0] = fmaf(s0.x, acc[0] + acc[2], fmaf(s0.y, qsum[g], s[j][0]));
                s[j][1] = fmaf(s1.x, acc[1] + acc[3], fmaf(s1.y, qsum[g], s[j][1]));
            }
        }
        if (nrow < 16) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (8 * j + 2 * t + e >= nrow) s[j][e] = -CUDART_INF_F;
        }

        // ---- online softmax -------------------------------------------------------------------------------------
        float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run, mx);
        const float m_safe = m_new == -CUDART_INF_F ? 0.f : m_new;
        const float alpha = fast_exp2((m_run - m_safe) * c);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[j][e] = fast_exp2((s[j][e] - m_safe) * c);
        l_run = fmaf(l_run, alpha, (s[0][0] + s[0][1]) + (s[1][0] + s[1][1]));
        m_run = m_new;
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) { o[j][0] *= alpha; o[j][1] *= alpha; o[j][2] *= alpha; o[j][3] *= alpha; }
#pragma unroll
            for (int g = 0; g < NG; ++g) om[g] *= alpha;
        }

        // ---- O += (P d) codes, and P m --------------------------------------------------------------------------
        uint32_t vs[2][2][NG];                               // scales of rows 8j + 2t + e
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t* sc = reinterpret_cast<const uint32_t*>(blk + F::VS_OFF + (8 * j + 2 * t) * F::SROWB);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int g = 0; g < NG; ++g) vs[j][e][g] = sc[e * NG + g];
        }
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int g = 0; g < NG; ++g) big |= vs[j][0][g] | vs[j][1][g];
        if (pscale > 1.f && __any_sync(0xffffffffu, (big & 0x4000u) != 0)) {     // a step of 2 or more
            pscale = 0.25f;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] *= 3.0517578125e-5f;         // 2^-15
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float pd[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 dm = half2_word(vs[j][e][g]);
                    om[g] = fmaf(s[j][e], dm.y, om[g]);
                    pd[j][e] = s[j][e] * pscale * dm.x;
                }
            uint32_t a0, a1, a2, a3;
            split_half2(pd[0][0], pd[0][1], a0, a1);
            split_half2(pd[1][0], pd[1][1], a2, a3);
            const uint4 v = *reinterpret_cast<const uint4*>(blk + F::V_OFF + g * 512 + lane * 16);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 4 * g + i;
                const uint32_t w8 = w[i] >> 8;
                mma_16816(o[2 * j], a0, a1, a2, a3, w[i] & 0x000F000Fu, w8 & 0x000F000Fu);
                mma_16816(o[2 * j + 1], a0, a1, a2, a3, w[i] & 0x00F000F0u, w8 & 0x00F000F0u);
            }
        }
        __syncwarp();                                        // every lane has read the stage
        const int nxt = it + kStages;
        if (nxt < nb) load_block(blk0 + warp + nxt * kWarps, it % kStages);
        cp_async_commit();
    }

    // ---- merge the warps: O of a warp scaled by e^(m_w - M), sums in warp order ----------------------------------
    cp_async_wait<0>();
    __syncthreads();
    float* mO = reinterpret_cast<float*>(smem);
    float* mML = reinterpret_cast<float*>(smem + L::ML_OFF);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        om[g] += __shfl_xor_sync(0xffffffffu, om[g], 1);
        om[g] += __shfl_xor_sync(0xffffffffu, om[g], 2);
    }
    const float m_raw = m_run * unit;                        // q . k, the unit the CTAs share
    if (t == 0) *reinterpret_cast<float2*>(&mML[(warp * 8 + r) * 2]) = make_float2(m_raw, l_run);
    __syncthreads();
    const float c_raw = p.scale * LOG2E;
    {
        float M = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, mML[(w * 8 + r) * 2]);
        const float wgt = m_raw == -CUDART_INF_F ? 0.f : fast_exp2((m_raw - M) * c_raw);
        const float lo = 16777216.f / pscale * wgt, hi = 1048576.f / pscale * wgt;     // 2^24, 2^20: the scale of the codes
        float* dst = mO + (size_t)(warp * 8 + r) * L::MSTRIDE + 4 * t;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
            const float a = om[j / 4] * wgt;
            const float* e = o[2 * j];
            const float* f = o[2 * j + 1];
            *reinterpret_cast<float4*>(dst + 16 * j) = make_float4(fmaf(e[0] + e[2], lo, a), fmaf(f[0] + f[2], hi, a),
                                                                   fmaf(e[1] + e[3], lo, a), fmaf(f[1] + f[3], hi, a));
        }
    }
    __syncthreads();
    RunState st[S::N];
    if (tid < kMergeThreads) {
#pragma unroll
        for (int k = 0; k < S::N; ++k) {
            const int row = S::row(tid, k), c4 = S::col4(tid, k);
            st[k] = run_empty();
            if (row < G) {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) st[k].M = fmaxf(st[k].M, mML[(w * 8 + row) * 2]);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float2 ml = *reinterpret_cast<const float2*>(&mML[(w * 8 + row) * 2]);
                    const float wgt = ml.x == -CUDART_INF_F ? 0.f : fast_exp2((ml.x - st[k].M) * c_raw);
                    st[k].L = fmaf(wgt, ml.y, st[k].L);
                    const float4 v = *reinterpret_cast<const float4*>(mO + (size_t)(w * 8 + row) * L::MSTRIDE + c4 * 4);
                    st[k].acc.x += v.x; st[k].acc.y += v.y; st[k].acc.z += v.z; st[k].acc.w += v.w;
                }
            }
        }
    }

    // ---- merge across the CTAs of these heads (one or two levels, see decode.cu) -----------------------------------
    if (plan.active > 1) {
        const size_t blk = (size_t)GP * HD;
        if (tid < kMergeThreads) {
            const size_t part = (size_t)vh * p.n_splits + split;
            store_part<HD, false>(p.ws_o + part * blk, p.ws_ml + part * GP * 2, G, st);
        }
        const int group = plan.active <= 16 ? plan.active : p.group;
        const int grp = split / group;
        const int grp_n = min(group, plan.active - grp * group);
        if (!arrive_last(p.tickets + vh * p.n_groups + grp, grp_n)) return;
        if (tid < kMergeThreads) {
            const size_t part0 = (size_t)vh * p.n_splits + (size_t)grp * group;
            merge_parts<HD, false>(p.ws_o + part0 * blk, p.ws_ml + part0 * GP * 2, grp_n, GP, c_raw, st);
        }
        const int n_grp = (plan.active + group - 1) / group;
        if (n_grp > 1) {
            if (tid < kMergeThreads) {
                const size_t gpart = (size_t)vh * p.n_groups + grp;
                store_part<HD, false>(p.grp_o + gpart * blk, p.grp_ml + gpart * GP * 2, G, st);
            }
            if (!arrive_last(p.tickets + p.n_kv * p.head_blocks * p.n_groups + vh, n_grp)) return;
            if (tid < kMergeThreads) {
                const size_t g0 = (size_t)vh * p.n_groups;
                merge_parts<HD, false>(p.grp_o + g0 * blk, p.grp_ml + g0 * GP * 2, n_grp, GP, c_raw, st);
            }
        }
    }
    if (tid < kMergeThreads) {
        // a NaN among the scores or values shows in the output
#pragma unroll
        for (int k = 0; k < S::N; ++k)
            if (st[k].L != st[k].L) { st[k].acc = make_float4(st[k].L, st[k].L, st[k].L, st[k].L); st[k].L = 1.f; }
        emit_final<HD, false>(p, head0, G, st);
    }
}

} // namespace

int decode_q4_num_splits(int n_kv, int sm_count) { return decode_num_splits(n_kv, sm_count); }

cudaError_t decode_q4_set_attributes() {
    cudaError_t e = cudaFuncSetAttribute(decode_q4_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4Smem<128>::TOTAL);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(decode_q4_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4Smem<64>::TOTAL);
}

cudaError_t launch_decode_q4(const DecodeQ4Args& a, int head_dim, cudaStream_t stream, unsigned long long* launches) {
    const dim3 grid(a.n_splits * a.head_blocks, a.n_kv);
    const cudaError_t e = head_dim == 128 ? launch_dependent(decode_q4_kernel<128>, grid, kThreads, Q4Smem<128>::TOTAL, stream, a.overlap, a)
                                          : launch_dependent(decode_q4_kernel<64>, grid, kThreads, Q4Smem<64>::TOTAL, stream, a.overlap, a);
    if (launches) *launches += 1;
    return e;
}

} // namespace oattn

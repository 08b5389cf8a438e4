// Single-token decode attention over the 4-bit KV cache (format: kv_q4.cuh), split over the sequence, in ONE launch.
//
// The sequence of every kv head is cut into slices, one CTA of eight warps each (grid = slices x kv heads, two CTAs per SM);
// a warp takes every eighth pair of 16-position blocks of the slice and brings it to shared memory with cp.async, one contiguous
// piece, two pairs deep, for itself alone: no barrier across warps until the end.  The grid never depends on the
// position, so the launch replays from a CUDA graph.  The slices are merged as in decode.cu (decode_merge.cuh).
//
// The codes are never turned into values.  With x = m + d * code per row and 64-dim group g,
//     q . k  = sum_g d_g (q_g . code_g) + m_g sum(q_g)            P V = sum_k (P_k d_gk) code_k + sum_k P_k m_gk
// so the matrix instructions (m16n8k16, fp16 in, fp32 out) take the codes as they are: a masked nibble in bits 4..7
// is an fp16 subnormal, exactly code * 2^-20, and the powers of two go into q and the final scale.  The left operands q and
// P d are fp32; a decode step has at most eight heads per CTA, so the other eight rows of the tile hold what the rounding of the
// first eight to fp16 left over (x = hi + lo, 22 bits together): the result keeps fp32 accuracy and the instruction count is
// the same.  q is scaled by a power of two per head, P d by one that goes by the largest step d so far and is lowered when a larger
// one comes, as a running maximum is, with the sums so far: so neither half leaves the fp16 range, and what the rounding of
// P d loses is at most 2^-22 of it or 2^-38 of the largest step.
//
// What bounds it: the warp-level matrix instruction takes its scheduler 8.1 cycles and lets nothing else issue beside it (measured:
// with 8 fp32 multiply-adds per product 16.0 cycles, with 4 logic operations 13.2).  A 16-position block is 32 products, 259 cycles,
// and about 340 other instructions (counted by ncu), 600 cycles of a scheduler; every further block takes one 0.33 us, which is about
// that at the clocks seen, and at the measured copy bandwidth its bytes would arrive in 0.21.  One million rows of 16/2 heads: 86 to
// 87 us, 3.5 TB/s of cache, 0.53 of the copy bandwidth (the fp16 cache: 158 us).  8, 12 and 16 warps per SM took 90.8, 87.5 and 88.9
// us at the time, so latency is not the limit.  The 8-bit float form of the instruction is emulated (21 cycles); the 8-bit integer
// form takes the same 8.1 for twice the depth, but q needs three digits, so nothing is won.
// At a few thousand rows a call is a chain of dependent round trips: 5.3 us from launch to output in one CTA, 2.3 more for a merge.
#include <type_traits>

#include "decode_merge.cuh"
#include "f32x2.cuh"
#include "kv_q4.cuh"

namespace oattn {

namespace {

constexpr int kWarps = 8;
constexpr int kCtas = 2;                   // per SM
constexpr int kThreads = 32 * kWarps;
constexpr int kTurns = 2;                  // pairs of blocks in the ring of a warp

template <int HD>
struct Q4Smem {
    static constexpr int BLOCK = Q4<HD>::BLOCK;
    static constexpr int RING = kWarps * kTurns * 2 * BLOCK;
    static constexpr int QF_OFF = RING;                                // q fragments [HD/16 steps][32 lanes][4 words]
    static constexpr int QF_BYTES = HD / 16 * 512;
    static constexpr int IN_OFF = QF_OFF + QF_BYTES;                   // an fp32 row per warp
    static constexpr int NEW_OFF = IN_OFF + kWarps * HD * 4;           // codes of the new row per lane: [2][32] u32, scales [2][2] u32
    static constexpr int QS_OFF = NEW_OFF + 2 * 32 * 4 + 32;           // per head: group sums of q [8][2], unit [8]
    static constexpr int TOTAL = QS_OFF + 8 * 2 * 4 + 8 * 4;
    // merge buffers over the ring once it has drained: [warps][8 rows][HD + 8] fp32, then (m, l) [warps][8][2]
    static constexpr int MSTRIDE = HD + 8;
    static constexpr int ML_OFF = kWarps * 8 * MSTRIDE * 4;
    static_assert(ML_OFF + kWarps * 8 * 2 * 4 <= RING, "the merge area lies in the ring");
};

struct Q4Plan {
    int blocks, per_split, active, step; // 16-row blocks in all, of one slice, slices that have any; blocks a warp takes at a time
};
// A warp works on pairs of blocks (half the softmax bookkeeping) where there are enough of them.  A merge across CTAs costs about
// 2.3 us and a second level 1.5, one turn of a CTA's eight warps 0.7 (one block each) or 1.4 (two), so up to 512 rows stay in one
// CTA (28/4 heads, 256 rows: 6.6 us against 7.8 from two CTAs), up to 4096 in 16, which merge in one level (4096 rows: 10.3
// us against 10.7 from 32); behind that the blocks are spread evenly over all slices.
__device__ __forceinline__ Q4Plan q4_plan(int npos, int n_splits) {
    Q4Plan s;
    s.blocks = (npos + 15) >> 4;
    const int even = 2 * (((s.blocks + 1) / 2 + n_splits - 1) / n_splits);           // no slice may be left without a CTA
    s.step = 2;
    s.per_split = even;
    if (s.blocks <= 32) {
        s.step = s.blocks <= kWarps ? 1 : 2;
        s.per_split = 32;
    } else if (s.blocks <= 16 * kWarps && s.blocks <= n_splits * kWarps) {
        s.step = 1;
        s.per_split = kWarps;
    } else if (s.blocks <= 32 * kWarps) {
        s.per_split = max(2 * kWarps, even);
    } else if (s.blocks <= n_splits * kWarps) {
        s.step = 1;
        s.per_split = kWarps;
    }
    s.active = (s.blocks + s.per_split - 1) / s.per_split;
    return s;
}

__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)w)); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)(w >> 16))); }

// hi = fp16(x), lo = fp16(x - hi), for a pair
__device__ __forceinline__ void split_half2(F2 x, uint32_t& hi, uint32_t& lo) {
    hi = pack_half2(x.x(), x.y());
    const F2 rest = fma2(F2(half_lo(hi), half_hi(hi)), F2(-1.f, -1.f), x);
    lo = pack_half2(rest.x(), rest.y());
}

// Scale words (d, m) of two neighbouring rows, [row][group], in one load.
template <int NG>
__device__ __forceinline__ void load_scales(const uint8_t* at, uint32_t (&w)[2][NG]) {
    if constexpr (NG == 2) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        w[0][0] = v.x; w[0][1] = v.y; w[1][0] = v.z; w[1][1] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        w[0][0] = v.x; w[1][0] = v.y;
    }
}

// Nibbles i and i + 4 of a code word as a pair of fp16 subnormals, code * 2^-20 (bits 4..7 of each half).  Two of the four
// pairs would need no shift at all as code * 2^-24, but the matrix unit aligns products by the operands' exponent fields: the
// more leading zeros a subnormal has, the more low bits of every partial sum are cut off (measured: the error of a step over
// 1K rows is 4e-6 of the output with codes at bits 0..3, against 1e-7 with these).
struct Nibbles {
    uint32_t x[4];
    __device__ __forceinline__ explicit Nibbles(uint32_t w) {
        const uint32_t w8 = w >> 8;
        x[0] = (w << 4) & 0x00F000F0u;
        x[1] = w & 0x00F000F0u;
        x[2] = (w8 << 4) & 0x00F000F0u;
        x[3] = w8 & 0x00F000F0u;
    }
};

__device__ __forceinline__ F2 shfl_xor(F2 v, int mask) { return F2(__shfl_xor_sync(0xffffffffu, v.x(), mask), __shfl_xor_sync(0xffffffffu, v.y(), mask)); }

// Transposes an 8 x 8 matrix of 16-bit values held as one row per quad of lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}

// TURNED (at most four heads): the codes are the 16-row operand of both products -- 16 positions by 16 dims, 16 dims by 16
// positions, the same words in the same lanes -- and the heads with their low halves its eight columns, so there are half as
// many products.  A lane then has two heads' scores of positions r and r + 8 instead of one head's of four, and P has to be
// transposed between the products.  32/8 heads of 128, 131072 rows: 43.8 us against 47.4; 32/8 heads of 64, 32001 rows: 12.4
// against 12.7; below a few thousand rows no difference.
//
// CHUNK: a few tokens behind a long context.  The tile's eight rows are (token, head) pairs, each with the positions up to its own
// token; everything else is as for one token.  32/8 heads behind 8192 rows: 16 us with its prologue for one token, 22 for eight.
template <int HD, bool TURNED, bool CHUNK>
__global__ void __launch_bounds__(kThreads, kCtas) decode_q4_kernel(const __grid_constant__ DecodeQ4Args p) {
    static_assert(!(TURNED && CHUNK), "a chunk fills the tile");
    using F = Q4<HD>;
    using L = Q4Smem<HD>;
    constexpr int MT = HD == 128 && kThreads >= 256 ? 256 : 128;    // threads that hold pieces of the merged block
    using S = Slots<HD, false, MT>;
    constexpr int NG = F::NG, NW = HD / 32;      // groups of a row, code words of a lane per K row
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = lane >> 2, t = lane & 3;
    const int hb = blockIdx.x % p.head_blocks, split = blockIdx.x / p.head_blocks, kvh = blockIdx.y;
    const int GA = p.n_head / p.n_kv;                        // heads of the kv head, and of this CTA
    const int head0 = kvh * GA + hb * p.heads_per_cta;
    const int row0 = hb * p.heads_per_cta;                   // CHUNK: first (token, head) pair
    const int G = min(p.heads_per_cta, (CHUNK ? p.batch * GA : GA) - row0);
    // head row `i` of this CTA in q and in the output, in units of HD
    auto head_row = [&](int i) { return CHUNK ? (size_t)((row0 + i) / GA) * p.n_head + kvh * GA + (row0 + i) % GA : (size_t)head0 + i; };

    // Inputs of the step: warp h has the row of head h, the last two warps the new rows of V and K as well, a lane EPL
    // consecutive dims.  All are issued together and, where the order against preceding kernels allows it, along with the
    // position word; from there to the barrier in front of the loop a warp waits for nobody.
    static_assert(kWarps == 8, "one warp per head");
    constexpr int E = F::EPL, kWarpK = kWarps - 1, kWarpV = kWarps - 2;
    const bool append = !CHUNK && (p.fuse & 4) != 0;
    float in_q[E], in_kv[E];
    auto load_lane = [&](float (&x)[E], const float* src, const float* bias, size_t row) {
        const size_t at = row * HD + E * lane;
        if constexpr (E == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + at);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2*>(src + at);
            x[0] = v.x; x[1] = v.y;
        }
        if (bias) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] += bias[at + e];
        }
    };
    auto load_inputs = [&]() {
        if (warp < G) load_lane(in_q, p.q, CHUNK ? nullptr : p.pre.bias_q, head_row(warp));
        if (append && warp >= kWarpV) load_lane(in_kv, warp == kWarpK ? p.k_new : p.v_new, warp == kWarpK ? p.pre.bias_k : p.pre.bias_v, (size_t)kvh);
    };

    pdl_trigger();
    if (p.overlap != 2) {
        pdl_wait();
        load_inputs();
    }
    const int npos = CHUNK ? p.n_past + (row0 + G - 1) / GA + 1 : max(0, min(*p.d_pos, p.n_ctx - 1) + 1);
    // CHUNK: positions that this lane's row sees, and that every row of the CTA sees
    const int lim = CHUNK ? p.n_past + (row0 + min(r, G - 1)) / GA + 1 : npos, lim_all = CHUNK ? p.n_past + row0 / GA + 1 : npos;
    const Q4Plan plan = q4_plan(npos, p.n_splits);
    if (split >= max(plan.active, 1)) return;
    const int vh = kvh * p.head_blocks + hb;                 // place of this CTA's heads in the scratch block
    const int GP = p.heads_per_cta;                          // rows kept there per slice
    if (plan.active == 0) {
        if (p.overlap == 2) pdl_wait();
        if (tid < MT) {
            RunState st[S::N];
#pragma unroll
            for (int k = 0; k < S::N; ++k) st[k] = run_empty();
            emit_final<HD, false, MT>(p, head0, G, st);
        }
        return;
    }
    const int blk0 = split * plan.per_split, blk1 = min(blk0 + plan.per_split, plan.blocks);
    const bool owner = append && split == plan.active - 1;
    const int new_pos = npos - 1;
    uint8_t* cache = p.cache + (size_t)kvh * q4_blocks(p.n_ctx) * F::BLOCK;
    uint8_t* ring = smem + warp * kTurns * 2 * F::BLOCK;

    // This warp's it-th turn: blocks b, b + 1 (one with step 1, or at the end), b = first(it); ring slots 2 (it % kTurns), + 1.
    auto first = [&](int it) { return blk0 + plan.step * (warp + kWarps * it); };
    const int turns = first(0) < blk1 ? (blk1 - first(0) + plan.step * kWarps - 1) / (plan.step * kWarps) : 0;
    auto load_turn = [&](int it) {
        const int b = first(it);
        const uint8_t* src = cache + (size_t)b * F::BLOCK + 16 * lane;
        const uint32_t dst = smem_u32(ring + (it % kTurns) * 2 * F::BLOCK + 16 * lane);
        const int n16 = (plan.step == 2 && b + 1 < blk1 ? 2 : 1) * (F::BLOCK / 16) - lane;
        constexpr int ALL = (2 * F::BLOCK / 16 + 31) / 32;
        if (2 * F::BLOCK % 512 == 0 && n16 > F::BLOCK / 16) {
#pragma unroll
            for (int i = 0; i < ALL; ++i) cp_async_16(dst + 512 * i, src + 512 * i, 16);
        } else {
#pragma unroll
            for (int i = 0; i < ALL; ++i)
                if (32 * i < n16) cp_async_16(dst + 512 * i, src + 512 * i, 16);
        }
    };
#pragma unroll
    for (int s = 0; s < kTurns; ++s) {
        if (s < turns) load_turn(s);
        cp_async_commit();
    }

    // ---- prologue -----------------------------------------------------------------------------------------------
    const bool rope_q = !CHUNK && (p.fuse & 1) != 0, rope_k = !CHUNK && (p.fuse & 2) != 0;
    float* s_row = reinterpret_cast<float*>(smem + L::IN_OFF) + warp * HD;       // this warp's row on its way
    float* s_qsum = reinterpret_cast<float*>(smem + L::QS_OFF);
    float* s_unit = s_qsum + 16;
    uint32_t* s_new = reinterpret_cast<uint32_t*>(smem + L::NEW_OFF);
    // angles of pairs lane, lane + 32: the fp32 product of position and frequency
    float angle[HD / 64];
    if (rope_q || rope_k) {
#pragma unroll
        for (int u = 0; u < HD / 64; ++u) {
            const int pp = lane + 32 * u;
            float f = pp < p.rope.n_rot / 2 ? p.freq[pp] : 0.f;
            if (p.rope.freq_factors && pp < p.rope.n_rot / 2) f = __fdiv_rn(f, p.rope.freq_factors[pp]);
            angle[u] = __fmul_rn((float)new_pos, f);
        }
    }
    if (p.overlap == 2) {
        pdl_wait();
        load_inputs();
    }
    auto norm_lane = [&](float (&x)[E], const float* w) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        const float rn = 1.0f / sqrtf(ss / (float)HD + p.pre.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * rn * w[E * lane + e];
    };
    // rotates the row through shared memory: a pair's elements may lie in any two lanes
    auto rotate_lane = [&](float (&x)[E], bool precise) {
#pragma unroll
        for (int e = 0; e < E; ++e) s_row[E * lane + e] = x[e];
        __syncwarp();
#pragma unroll
        for (int u = 0; u < HD / 64; ++u) {
            const int pp = lane + 32 * u;
            if (pp < p.rope.n_rot / 2) {
                int i0, i1;
                rope_pair_index(p.rope.rope_type, pp, p.rope.n_rot, i0, i1);
                if (precise) {
                    double sn, cs;
                    sincos((double)angle[u], &sn, &cs);
                    const double a = s_row[i0], b = s_row[i1];
                    s_row[i0] = (float)(a * cs - b * sn);
                    s_row[i1] = (float)(a * sn + b * cs);
                } else {
                    float sn, cs;
                    sincosf(angle[u], &sn, &cs);
                    const float a = s_row[i0], b = s_row[i1];
                    s_row[i0] = a * cs - b * sn;
                    s_row[i1] = a * sn + b * cs;
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = s_row[E * lane + e];
        __syncwarp();
    };
    uint4* s_frag = reinterpret_cast<uint4*>(smem + L::QF_OFF);
    if (warp < G) {
        if (!CHUNK && p.pre.norm_q) norm_lane(in_q, p.pre.norm_q);
        if (rope_q) rotate_lane(in_q, false);
        // the power of two that brings the largest |q| to [2^13, 2^14), and the group sums
        float amax = fabsf(in_q[0]);
#pragma unroll
        for (int e = 1; e < E; ++e) amax = fmaxf(amax, fabsf(in_q[e]));
#pragma unroll
        for (int off = 16; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        int k = 13 - ((int)(__float_as_uint(amax) >> 23) - 127);
        k = amax == 0.f ? 0 : max(-100, min(100, k));
        const float up = __uint_as_float((uint32_t)(127 + k) << 23);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            in_q[e] *= up;
            sum += in_q[e];
            s_row[E * lane + e] = in_q[e];
        }
#pragma unroll
        for (int off = 16 / NG; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane % (32 / NG) == 0) s_qsum[warp * 2 + lane / (32 / NG)] = sum * 9.5367431640625e-7f;              // 2^-20
        if (lane == 0) s_unit[warp] = __uint_as_float((uint32_t)(127 + 20 - k) << 23);     // back to q . k
        __syncwarp();
        // Fragments of this head: step 2i + o of word i takes the nibbles 0, 4 | 2, 6 (o = 0) or 1, 5 | 3, 7 (o = 1); words: row r
        // hi, row r lo (as row r + 8), and the same for k + 8
        if (lane < HD / 16 * 4) {
            const int step = lane >> 2;
            const float* row = s_row + 32 * (step >> 1) + 8 * t + (step & 1);
            uint4 w;
            split_half2(F2(row[0], row[4]), w.x, w.y);
            split_half2(F2(row[2], row[6]), w.z, w.w);
            if (TURNED) {                                    // columns: head, and head + 4 for what its rounding left
                reinterpret_cast<uint2*>(s_frag)[step * 32 + 4 * warp + t] = make_uint2(w.x, w.z);
                reinterpret_cast<uint2*>(s_frag)[step * 32 + 4 * (warp + 4) + t] = make_uint2(w.y, w.w);
            } else {
                s_frag[step * 32 + 4 * warp + t] = w;
            }
        }
        __syncwarp();
    } else {
        if (lane < HD / 16 * 4) {
            if (!TURNED) {
                s_frag[(lane >> 2) * 32 + 4 * warp + t] = make_uint4(0u, 0u, 0u, 0u);
            } else if (warp < 4) {
                reinterpret_cast<uint2*>(s_frag)[(lane >> 2) * 32 + 4 * warp + t] = make_uint2(0u, 0u);
                reinterpret_cast<uint2*>(s_frag)[(lane >> 2) * 32 + 4 * (warp + 4) + t] = make_uint2(0u, 0u);
            }
        }
        if (lane < 2) s_qsum[warp * 2 + lane] = 0.f;
        if (lane == 0) s_unit[warp] = 1.f;
    }
    // the new row of K or V: codes, into the cache and into s_new for this CTA's copy of the block
    if (owner && warp >= kWarpV) {
        const bool is_v = warp == kWarpV;
        if (!is_v) {
            if (p.pre.norm_k) norm_lane(in_kv, p.pre.norm_k);
            if (rope_k) rotate_lane(in_kv, true);
        }
        const Q4Scale sc = q4_scale<HD>(in_kv, lane);
        const uint32_t codes = q4_codes<HD>(in_kv, sc);
        s_new[is_v * 32 + lane] = codes;
        if (E * lane % 64 == 0) s_new[64 + is_v * 2 + E * lane / 64] = q4_scale_word(sc);
        if (hb == 0) {
            uint8_t* blk = cache + (size_t)(new_pos >> 4) * F::BLOCK;
            if (is_v) q4_store_row<HD, true>(blk, new_pos & 15, codes, sc, lane);
            else      q4_store_row<HD, false>(blk, new_pos & 15, codes, sc, lane);
        }
    }
    __syncthreads();

    // a lane's head, or its two heads
    const int hA = TURNED ? 2 * (t & 1) : r, hB = TURNED ? hA + 1 : r;
    F2 qsum[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) qsum[g] = F2(s_qsum[hA * 2 + g], s_qsum[hB * 2 + g]);
    const F2 unit(s_unit[hA], s_unit[hB]);
    const float c_raw = p.scale * LOG2E;
    const F2 c = unit * F2(c_raw, c_raw);
    const uint4* qf = reinterpret_cast<const uint4*>(smem + L::QF_OFF) + lane;
    const uint2* qt = reinterpret_cast<const uint2*>(smem + L::QF_OFF) + lane;

    // O in the scale of the codes: of head r, dims 16 j + 4 t + {0, 2} (o[2j]) and {1, 3} (o[2j+1]); TURNED: of the two heads (their
    // low halves in lanes t >= 2), dim 16 j + 2 r (o[2j]) and the next (o[2j+1])
    F2 o[HD / 8], om[NG];
    F2 m_run, l_run;                                         // per head (the same twice, and the two keys' shares, where a lane has one)
    // P d is carried times `pscale`; d_lim = 2^16 / pscale, the first step that would leave fp16 (P is at most 1).  The same in all lanes,
    // but for a chunk's last blocks, where a row goes by the positions it sees.
    float pscale = 137438953472.f, d_lim = 4.76837158203125e-7f;       // 2^37: the smallest step, 2^-24, comes to 2^13
    auto lower = [&](float d_max) {                          // brings d_max to [2^13, 2^14): steps up to four times as large fit after it
        if (!(d_max >= d_lim)) return;
        const uint32_t e = __float_as_uint(d_max) >> 23, next = (267 - e) << 23;      // exponent fields
        const float by = __uint_as_float(next - __float_as_uint(pscale) + (127u << 23));
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) o[j] = o[j] * F2(by, by);
        pscale = __uint_as_float(next);
        d_lim = __uint_as_float((e + 3) << 23);
    };
    auto finite = [](float d) { return d <= 65504.f ? d : 0.f; };
    // ... before P d of the NB blocks at `blk`, all of whose rows count: a lane looks at one row, or at the same as another lane
    auto fit = [&](int nb, const uint8_t* blk) {
        const uint8_t* at = blk + (nb == 2 ? lane >> 4 : 0) * F::BLOCK + F::VS_OFF + (lane & 15) * F::SROWB;
        float d0, d1 = 0.f;
        if constexpr (NG == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(at);
            d0 = half_lo(w.x);
            d1 = half_lo(w.y);
        } else {
            d0 = half_lo(*reinterpret_cast<const uint32_t*>(at));
        }
        if (!__any_sync(0xffffffffu, fmaxf(d0, d1) >= d_lim)) return;
        // (a step that is not finite shows in the output at any scale; positive numbers are in the order of their bits)
        lower(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(finite(d0), finite(d1))))));
    };

    // One turn over NB blocks that lie next to each other in the ring.
    auto turn = [&](auto nb_c, const uint8_t* blk, int nrow, int nrow_all) {
        constexpr int NB = decltype(nb_c)::value, NT = 2 * NB;         // tiles of eight rows
        // ---- S = q . K ------------------------------------------------------------------------------------------
        F2 s[NT];                                            // rows 8j + 2t, + 1
        {
            uint32_t w[NT][NW], ks[NT][2][NG];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint8_t* row = blk + (j >> 1) * F::BLOCK + (8 * (j & 1) + r) * F::ROWB + t * (F::ROWB / 4);
                if constexpr (NW == 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(row);
                    w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(row);
                    w[j][0] = v.x; w[j][1] = v.y;
                }
                load_scales<NG>(blk + (j >> 1) * F::BLOCK + F::KS_OFF + (8 * (j & 1) + 2 * t) * F::SROWB, ks[j]);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float acc[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
                for (int i = 2 * g; i < 2 * g + 2; ++i) {
                    const uint4 a0 = qf[(2 * i) * 32], a1 = qf[(2 * i + 1) * 32];
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const Nibbles n(w[j][i]);
                        mma_16816(acc[j], a0.x, a0.y, a0.z, a0.w, n.x[0], n.x[2]);
                        mma_16816(acc[j], a1.x, a1.y, a1.z, a1.w, n.x[1], n.x[3]);
                    }
                }
                const F2 qs = qsum[g];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const F2 m(half_hi(ks[j][0][g]), half_hi(ks[j][1][g])), d(half_lo(ks[j][0][g]), half_lo(ks[j][1][g]));
                    const F2 mq = g == 0 ? m * qs : fma2(m, qs, s[j]);
                    s[j] = fma2(d, F2(acc[j][0], acc[j][1]) + F2(acc[j][2], acc[j][3]), mq);
                }
            }
        }
        if (nrow_all < 16 * NB) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
                s[j] = F2(8 * j + 2 * t >= nrow ? -CUDART_INF_F : s[j].x(), 8 * j + 2 * t + 1 >= nrow ? -CUDART_INF_F : s[j].y());
        }

        // ---- online softmax -------------------------------------------------------------------------------------
        float mx = m_run.x();
#pragma unroll
        for (int j = 0; j < NT; ++j) mx = fmaxf(mx, fmaxf(s[j].x(), s[j].y()));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_safe = mx == -CUDART_INF_F ? 0.f : mx;
        const float alpha = fast_exp2((m_run.x() - m_safe) * c.x());
        const F2 alpha2(alpha, alpha);
        m_run = F2(mx, mx);
        F2 sum(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const F2 x = (s[j] + F2(-m_safe, -m_safe)) * c;
            s[j] = F2(fast_exp2(x.x()), fast_exp2(x.y()));
            sum = j == 0 ? s[j] : sum + s[j];
        }
        l_run = fma2(l_run, alpha2, sum);

        // ---- O = alpha O + (P d) codes, and P m -----------------------------------------------------------------
        uint32_t vs[NT][2][NG];
#pragma unroll
        for (int j = 0; j < NT; ++j) load_scales<NG>(blk + (j >> 1) * F::BLOCK + F::VS_OFF + (8 * (j & 1) + 2 * t) * F::SROWB, vs[j]);
        if (CHUNK && nrow_all < 16 * NB) {                   // a later token's row may hold anything: 0 * NaN would show
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (8 * j + 2 * t >= nrow) vs[j][0][g] = 0u;
                    if (8 * j + 2 * t + 1 >= nrow) vs[j][1][g] = 0u;
                }
            float d_max = 0.f;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int g = 0; g < NG; ++g) d_max = fmaxf(d_max, fmaxf(finite(half_lo(vs[j][0][g])), finite(half_lo(vs[j][1][g]))));
            d_max = fmaxf(d_max, __shfl_xor_sync(0xffffffffu, d_max, 1));
            lower(fmaxf(d_max, __shfl_xor_sync(0xffffffffu, d_max, 2)));
        } else {
            fit(NB, blk);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint32_t a[NB][4];
            om[g] = om[g] * alpha2;
#pragma unroll
            for (int h = 0; h < NB; ++h) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int j = 2 * h + e;
                    om[g] = fma2(s[j], F2(half_hi(vs[j][0][g]), half_hi(vs[j][1][g])), om[g]);
                    const F2 d(half_lo(vs[j][0][g]), half_lo(vs[j][1][g]));
                    split_half2(s[j] * F2(pscale, pscale) * d, a[h][2 * e], a[h][2 * e + 1]);
                }
            }
            uint32_t w[NB][4];
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                const uint4 v = *reinterpret_cast<const uint4*>(blk + h * F::BLOCK + F::V_OFF + g * 512 + lane * 16);
                w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < NB; ++h) {
                    const Nibbles n(w[h][i]);
                    mma_16816(x, a[h][0], a[h][1], a[h][2], a[h][3], n.x[0], n.x[2]);
                    mma_16816(y, a[h][0], a[h][1], a[h][2], a[h][3], n.x[1], n.x[3]);
                }
                F2& ox = o[2 * (4 * g + i)];
                F2& oy = o[2 * (4 * g + i) + 1];
                ox = fma2(ox, alpha2, F2(x[0], x[1]) + F2(x[2], x[3]));
                oy = fma2(oy, alpha2, F2(y[0], y[1]) + F2(y[2], y[3]));
            }
        }
    };

    // The same with the operands turned around.
    auto turn_turned = [&](auto nb_c, const uint8_t* blk, int nrow) {
        constexpr int NB = decltype(nb_c)::value, NT = 2 * NB;         // tiles of eight positions; a lane has position r of each
        F2 s[NT];
        {
            uint32_t w[NT][NW], ks[NT][NG];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint8_t* b = blk + (j >> 1) * F::BLOCK;
                const int row = 8 * (j & 1) + r;
                if constexpr (NW == 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(b + row * F::ROWB + t * 16);
                    w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
                    const uint2 k = *reinterpret_cast<const uint2*>(b + F::KS_OFF + row * F::SROWB);
                    ks[j][0] = k.x; ks[j][NG - 1] = k.y;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(b + row * F::ROWB + t * 8);
                    w[j][0] = v.x; w[j][1] = v.y;
                    ks[j][0] = *reinterpret_cast<const uint32_t*>(b + F::KS_OFF + row * F::SROWB);
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float acc[NB][4];
#pragma unroll
                for (int h = 0; h < NB; ++h) acc[h][0] = acc[h][1] = acc[h][2] = acc[h][3] = 0.f;
#pragma unroll
                for (int i = 2 * g; i < 2 * g + 2; ++i) {
                    const uint2 b0 = qt[(2 * i) * 32], b1 = qt[(2 * i + 1) * 32];
#pragma unroll
                    for (int h = 0; h < NB; ++h) {
                        const Nibbles n(w[2 * h][i]), u(w[2 * h + 1][i]);
                        mma_16816(acc[h], n.x[0], u.x[0], n.x[2], u.x[2], b0.x, b0.y);
                        mma_16816(acc[h], n.x[1], u.x[1], n.x[3], u.x[3], b1.x, b1.y);
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float d = half_lo(ks[j][g]);
                    const F2 x(acc[j >> 1][2 * (j & 1)], acc[j >> 1][2 * (j & 1) + 1]);
                    s[j] = g == 0 ? F2(d, d) * x : fma2(F2(d, d), x, s[j]);
                }
            }
            // what the rounding of q left over comes from the lane two places on
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                s[j] = s[j] + shfl_xor(s[j], 2);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float m = half_hi(ks[j][g]);
                    s[j] = fma2(F2(m, m), qsum[g], s[j]);
                }
            }
        }
        if (nrow < 16 * NB) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (8 * j + r >= nrow) s[j] = F2(-CUDART_INF_F, -CUDART_INF_F);
        }

        float mx = m_run.x(), my = m_run.y();
#pragma unroll
        for (int j = 0; j < NT; ++j) { mx = fmaxf(mx, s[j].x()); my = fmaxf(my, s[j].y()); }
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, off));
        }
        const F2 neg(mx == -CUDART_INF_F ? 0.f : -mx, my == -CUDART_INF_F ? 0.f : -my);
        const F2 xa = (m_run + neg) * c;
        const F2 alpha(fast_exp2(xa.x()), fast_exp2(xa.y()));
        m_run = F2(mx, my);
        F2 sum(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const F2 x = (s[j] + neg) * c;
            s[j] = F2(fast_exp2(x.x()), fast_exp2(x.y()));
            sum = j == 0 ? s[j] : sum + s[j];
        }
        l_run = fma2(l_run, alpha, sum);

        fit(NB, blk);
        uint32_t vs[NT][NG];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint8_t* at = blk + (j >> 1) * F::BLOCK + F::VS_OFF + (8 * (j & 1) + r) * F::SROWB;
            if constexpr (NG == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(at);
                vs[j][0] = v.x; vs[j][NG - 1] = v.y;
            } else {
                vs[j][0] = *reinterpret_cast<const uint32_t*>(at);
            }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint32_t b[NT];
            om[g] = om[g] * alpha;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float m = half_hi(vs[j][g]), d = half_lo(vs[j][g]) * pscale;
                om[g] = fma2(s[j], F2(m, m), om[g]);
                uint32_t hi, lo;
                split_half2(s[j] * F2(d, d), hi, lo);
                b[j] = transpose8(t < 2 ? hi : lo);          // position r, heads in pairs -> column r, positions 2t, 2t + 1
            }
            uint32_t w[NB][4];
#pragma unroll
            for (int h = 0; h < NB; ++h) {
                const uint4 v = *reinterpret_cast<const uint4*>(blk + h * F::BLOCK + F::V_OFF + g * 512 + lane * 16);
                w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < NB; ++h) {
                    const Nibbles n(w[h][i]);
                    mma_16816(x, n.x[0], n.x[1], n.x[2], n.x[3], b[2 * h], b[2 * h + 1]);
                }
                F2& oe = o[2 * (4 * g + i)];
                F2& od = o[2 * (4 * g + i) + 1];
                oe = fma2(oe, alpha, F2(x[0], x[1]));
                od = fma2(od, alpha, F2(x[2], x[3]));
            }
        }
    };

#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j] = F2(0.f, 0.f);
#pragma unroll
    for (int g = 0; g < NG; ++g) om[g] = F2(0.f, 0.f);
    m_run = F2(-CUDART_INF_F, -CUDART_INF_F);
    l_run = F2(0.f, 0.f);
    for (int it = 0; it < turns; ++it) {
        cp_async_wait<kTurns - 1>();
        __syncwarp();
        const int b = first(it);
        const bool two = plan.step == 2 && b + 1 < blk1;
        uint8_t* blk = ring + (it % kTurns) * 2 * F::BLOCK;
        const int nrow = npos - b * 16;                      // valid rows from the first block on
        if (b + (two ? 1 : 0) == plan.blocks - 1) {
            // the block of the newest row
            uint8_t* last = blk + (two ? F::BLOCK : 0);
            if (owner) {
                // ... which is not (or not safely) in what was copied
                const int slot = new_pos & 15, D = F::EPL * lane;
                const uint32_t kcode = s_new[lane], vcode = s_new[32 + lane];
                if (F::EPL == 4) *reinterpret_cast<uint16_t*>(last + q4_k_byte<HD>(slot, D)) = (uint16_t)kcode;
                else             last[q4_k_byte<HD>(slot, D)] = (uint8_t)kcode;
#pragma unroll
                for (int e = 0; e < F::EPL; e += 2) last[q4_v_byte<HD>(slot, D + e)] = (uint8_t)(vcode >> (4 * e));
                if (lane < 2 * NG) {
                    const int w = lane / NG, g = lane % NG;
                    *reinterpret_cast<uint32_t*>(last + (w ? F::VS_OFF : F::KS_OFF) + slot * F::SROWB + 4 * g) = s_new[64 + w * 2 + g];
                }
            } else if (!append && p.overlap == 2) {
                // copied ahead of the dependency wait: the newest row may have been written since
                const uint4* src = reinterpret_cast<const uint4*>(cache + (size_t)(plan.blocks - 1) * F::BLOCK);
                for (int i = lane; i < F::BLOCK / 16; i += 32) reinterpret_cast<uint4*>(last)[i] = __ldcg(src + i);
            }
            __syncwarp();
            // rows past the end: whatever the memory held, their steps and offsets count as zero
            for (int i = lane; i < 2 * 16 * NG; i += 32) {
                const int row = (i % (16 * NG)) / NG;
                if (row > (new_pos & 15)) reinterpret_cast<uint32_t*>(last + F::KS_OFF)[i] = 0u;
            }
            __syncwarp();
        }
        if constexpr (TURNED) {
            if (two) turn_turned(std::integral_constant<int, 2>{}, blk, nrow);
            else     turn_turned(std::integral_constant<int, 1>{}, blk, nrow);
        } else {
            if (two) turn(std::integral_constant<int, 2>{}, blk, lim - b * 16, lim_all - b * 16);
            else     turn(std::integral_constant<int, 1>{}, blk, lim - b * 16, lim_all - b * 16);
        }
        __syncwarp();                                        // every lane has read the ring slots
        if (it + kTurns < turns) load_turn(it + kTurns);
        cp_async_commit();
    }
    cp_async_wait<0>();

    // ---- merge the warps: O of a warp scaled by e^(m_w - M), sums in warp order ----------------------------------
    __syncthreads();
    float* mO = reinterpret_cast<float*>(smem);
    float* mML = reinterpret_cast<float*>(smem + L::ML_OFF);
    // a head's sums lie in the four lanes of a quad, or (TURNED) in the eight of one place t
    F2 total[NG + 1];
#pragma unroll
    for (int g = 0; g <= NG; ++g) {
        F2 v = g < NG ? om[g < NG ? g : 0] : l_run;
        if constexpr (TURNED) {
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) v = v + shfl_xor(v, off);
        } else {
            float x = v.x() + v.y();
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            v = F2(x, x);
        }
        total[g] = v;
    }
    const F2 m_raw = m_run * unit;                           // q . k, the unit the CTAs share
    if (TURNED ? (r == 0 && t < 2) : t == 0) {
        *reinterpret_cast<float2*>(&mML[(warp * 8 + hA) * 2]) = make_float2(m_raw.x(), total[NG].x());
        if (TURNED) *reinterpret_cast<float2*>(&mML[(warp * 8 + hB) * 2]) = make_float2(m_raw.y(), total[NG].y());
    }
    __syncthreads();
    {
        float M[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            M[0] = fmaxf(M[0], mML[(w * 8 + hA) * 2]);
            if (TURNED) M[1] = fmaxf(M[1], mML[(w * 8 + hB) * 2]);
        }
        const float wx = m_raw.x() == -CUDART_INF_F ? 0.f : fast_exp2((m_raw.x() - M[0]) * c_raw);
        const float f = 1048576.f / pscale;                  // 2^20: the scale of the codes
        if constexpr (TURNED) {
            const float wy = m_raw.y() == -CUDART_INF_F ? 0.f : fast_exp2((m_raw.y() - M[1]) * c_raw);
            const F2 wgt(wx, wy), fw = F2(f, f) * wgt;
            float* dst = mO + (size_t)(warp * 8 + hA) * L::MSTRIDE + 2 * r;
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                const F2 a = total[j / 4] * wgt;
                const F2 e = fma2(o[2 * j] + shfl_xor(o[2 * j], 2), fw, a), d = fma2(o[2 * j + 1] + shfl_xor(o[2 * j + 1], 2), fw, a);
                if (t < 2) {
                    *reinterpret_cast<float2*>(dst + 16 * j) = make_float2(e.x(), d.x());
                    *reinterpret_cast<float2*>(dst + L::MSTRIDE + 16 * j) = make_float2(e.y(), d.y());
                }
            }
        } else {
            const float fw = f * wx;
            float* dst = mO + (size_t)(warp * 8 + r) * L::MSTRIDE + 4 * t;
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                const float a = total[j / 4].x() * wx;
                *reinterpret_cast<float4*>(dst + 16 * j) = make_float4(fmaf(o[2 * j].x(), fw, a), fmaf(o[2 * j + 1].x(), fw, a),
                                                                       fmaf(o[2 * j].y(), fw, a), fmaf(o[2 * j + 1].y(), fw, a));
            }
        }
    }
    __syncthreads();
    RunState st[S::N];
    if (tid < MT) {
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
        if (tid < MT) {
            const size_t part = (size_t)vh * p.n_splits + split;
            store_part<HD, false, MT>(p.ws_o + part * blk, p.ws_ml + part * GP * 2, G, st);
        }
        const int group = plan.active <= 16 ? plan.active : p.group;
        const int grp = split / group;
        const int grp_n = min(group, plan.active - grp * group);
        if (!arrive_last(p.tickets + vh * p.n_groups + grp, grp_n)) return;
        if (tid < MT) {
            const size_t part0 = (size_t)vh * p.n_splits + (size_t)grp * group;
            merge_parts<HD, false, MT>(p.ws_o + part0 * blk, p.ws_ml + part0 * GP * 2, grp_n, GP, c_raw, st);
        }
        const int n_grp = (plan.active + group - 1) / group;
        if (n_grp > 1) {
            if (tid < MT) {
                const size_t gpart = (size_t)vh * p.n_groups + grp;
                store_part<HD, false, MT>(p.grp_o + gpart * blk, p.grp_ml + gpart * GP * 2, G, st);
            }
            if (!arrive_last(p.tickets + p.n_kv * p.head_blocks * p.n_groups + vh, n_grp)) return;
            if (tid < MT) {
                const size_t g0 = (size_t)vh * p.n_groups;
                merge_parts<HD, false, MT>(p.grp_o + g0 * blk, p.grp_ml + g0 * GP * 2, n_grp, GP, c_raw, st);
            }
        }
    }
    if (tid < MT) {
        // a NaN among the scores or values shows in the output
#pragma unroll
        for (int k = 0; k < S::N; ++k)
            if (st[k].L != st[k].L) { st[k].acc = make_float4(st[k].L, st[k].L, st[k].L, st[k].L); st[k].L = 1.f; }
        if constexpr (CHUNK) {
#pragma unroll
            for (int k = 0; k < S::N; ++k) {
                const int row = S::row(tid, k), c4 = S::col4(tid, k);
                if (row >= G) continue;
                const float4 v = normalised(st[k]);
                const size_t at = head_row(row) * HD + c4 * 4;
                if (p.out16) *reinterpret_cast<uint2*>(p.out16 + at) = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
                else         *reinterpret_cast<float4*>(p.out + at) = v;
            }
        } else {
            emit_final<HD, false, MT>(p, head0, G, st);
        }
    }
}

} // namespace

// One wave: kCtas per SM over the kv heads, or over their halves where a kv head's query heads take two CTAs (32/2 heads, 32768
// rows: 14.8 us against 21.5 from two waves).
int decode_q4_num_splits(int head_blocks, int sm_count) { return max(1, min(DECODE_MAX_SPLITS, kCtas * sm_count / head_blocks)); }

namespace {
template <int HD, bool TURNED, bool CHUNK>
cudaError_t set_attributes() {
    return cudaFuncSetAttribute(decode_q4_kernel<HD, TURNED, CHUNK>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4Smem<HD>::TOTAL);
}
template <int HD, bool TURNED, bool CHUNK>
cudaError_t launch(const DecodeQ4Args& a, cudaStream_t stream) {
    return launch_dependent(decode_q4_kernel<HD, TURNED, CHUNK>, dim3(a.n_splits * a.head_blocks, a.n_kv), kThreads, Q4Smem<HD>::TOTAL, stream, 1, a);
}
template <int HD>
cudaError_t set_attributes_hd() {
    cudaError_t e;
    if ((e = set_attributes<HD, false, false>()) != cudaSuccess || (e = set_attributes<HD, true, false>()) != cudaSuccess) return e;
    return set_attributes<HD, false, true>();
}
template <int HD>
cudaError_t launch_hd(const DecodeQ4Args& a, cudaStream_t stream) {
    if (a.batch > 0) return launch<HD, false, true>(a, stream);
    return a.heads_per_cta <= 4 ? launch<HD, true, false>(a, stream) : launch<HD, false, false>(a, stream);
}
} // namespace

cudaError_t decode_q4_set_attributes() {
    const cudaError_t e = set_attributes_hd<128>();
    return e != cudaSuccess ? e : set_attributes_hd<64>();
}

cudaError_t launch_decode_q4(const DecodeQ4Args& a, int head_dim, cudaStream_t stream, unsigned long long* launches) {
    const cudaError_t e = head_dim == 128 ? launch_hd<128>(a, stream) : launch_hd<64>(a, stream);
    if (launches) *launches += 1;
    return e;
}

} // namespace oattn

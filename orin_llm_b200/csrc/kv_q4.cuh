// The 4-bit KV cache: block format, quantiser and addresses shared by its kernels (kv_q4.cu, decode_q4.cu).
//
// One layer is [n_kv][ceil(n_ctx / 16)][block]; a block is 16 consecutive positions of one kv head, K and V together, so
// that a reader fetches one contiguous piece (2304 bytes for head_dim 128, 4.5 bits a value against 16).  A head row is cut
// into groups of 64 dims; a group keeps an fp16 offset m and an fp16 step d, a value is m + d * code, code 0..15:
//     m = fp16(min x)    d = fp16(max(0, (max x - m) / 15))    code = clamp(round((x - m) / d), 0, 15), 0 where d = 0
// Each right-hand side is evaluated exactly and rounded once (ties to even), so the bytes depend on the row alone, not on
// the launch that wrote them.  A group that holds a NaN, an infinity or a minimum beyond fp16 gets d = m = NaN.
//
// The code order is the one the decode kernel's m16n8k16 products read without moving anything between lanes:
//   K: row s at word s * HD/8; word t * HD/32 + i (t < 4: the lane's place in its quad) holds dims 32 i + 8 t + e, dim e in
//      bits 4e..4e+3.  Nibbles i and i + 4 of a word, shifted to bits 4..7 of its halves, are a B register: a pair of fp16
//      subnormals code * 2^-20, exactly; the four pairs make two k-steps.
//   V: a byte holds dims 2p (low half) and 2p + 1 of one row; the four bytes of a word belong to rows 2t, 2t+8, 2t+1, 2t+9 of
//      the block, so that the same pairs are rows (2t, 2t+1) and (2t+8, 2t+9) of an even and an odd dim.  With p = 8 j + r the word sits at
//      (j/4) * 512 + (4 r + t) * 16 + (j%4) * 4: lane 4r + t reads 16 bytes.  One byte belongs to one row, so appending a
//      row never reads what its neighbours hold.
//   scales: fp16 [16 rows][HD/64][d, m] for K, then for V.
#pragma once

#include "attn_internal.h"

namespace oattn {

template <int HD>
struct Q4 {
    static constexpr int NG = HD / 64;                    // groups of a row
    static constexpr int ROWB = HD / 2;                   // code bytes of a row
    static constexpr int V_OFF = 16 * ROWB;
    static constexpr int KS_OFF = 32 * ROWB;
    static constexpr int SROWB = 4 * NG;                  // scale bytes of a row
    static constexpr int VS_OFF = KS_OFF + 16 * SROWB;
    static constexpr int BLOCK = VS_OFF + 16 * SROWB;
    static constexpr int EPL = HD / 32;                   // dims of a row that one lane of a warp handles: EPL*lane ...
};
static_assert(Q4<128>::BLOCK == 2304 && Q4<64>::BLOCK == 1152, "block bytes");

__host__ __device__ inline size_t q4_block_bytes(int head_dim) { return (size_t)head_dim * 18; }
__host__ __device__ inline int q4_blocks(int n_ctx) { return (n_ctx + 15) / 16; }

// Byte of the codes of dims D, D+1 (D even) of K row s inside a block, and the same for V.
template <int HD>
__device__ __forceinline__ int q4_k_byte(int s, int D) {
    return s * Q4<HD>::ROWB + (((D & 31) >> 3) * (HD / 32) + (D >> 5)) * 4 + ((D & 7) >> 1);
}
template <int HD>
__device__ __forceinline__ int q4_v_byte(int s, int D) {
    const int p = D >> 1, j = p >> 3, r = p & 7, t = (s & 7) >> 1;
    return Q4<HD>::V_OFF + (j >> 2) * 512 + (4 * r + t) * 16 + (j & 3) * 4 + 2 * (s & 1) + (s >> 3);
}

struct Q4Scale { __half d, m; };

// fp16((max - m) / 15) in one rounding, out of line: next to the midpoint of two fp16 numbers, and among the subnormal ones.
static __device__ __noinline__ __half q4_step_exact(float mx, float m) { return __double2half(((double)mx - (double)m) / 15.0); }

// (d, m) of a group with this minimum and maximum (NaN or infinite where the group has such a value).  The fp32 quotient is off
// by at most two of its last places, so its rounding to fp16 (13 places fewer) is the exact quotient's unless it lies within
// four of a midpoint.  Without that case one group in about 4000 would get a step that is off by an fp16 place.
__device__ __forceinline__ Q4Scale q4_scale_of(float mn, float mx) {
    Q4Scale s;
    s.m = __float2half_rn(mn);
    const float m = __half2float(s.m);
    if (!(fabsf(mx) <= 3.402823466e38f) || !(fabsf(m) <= 65504.f)) {
        s.d = s.m = __ushort_as_half(0x7fff);
        return s;
    }
    const float step = __fmul_rn(__fsub_rn(mx, m), 1.0f / 15.0f);
    s.d = __float2half_rn(fmaxf(step, 0.f));
    if (((__float_as_uint(step) - 0xffcu) & 0x1fffu) <= 8u || (step > 0.f && step < 6.2e-5f)) s.d = step > 0.f ? q4_step_exact(mx, m) : __ushort_as_half(0);
    return s;
}

// (d, m) of the group whose EPL-value shares lie in the lanes of `x`: lanes of the same half warp (HD = 128) or of the whole
// warp (HD = 64) hold one group.  Called by full warps.
template <int HD>
__device__ __forceinline__ Q4Scale q4_scale(const float (&x)[Q4<HD>::EPL], int lane) {
    constexpr int W = 32 / Q4<HD>::NG;                    // lanes of a group
    float mn = x[0], mx = x[0];
    bool bad = !(fabsf(x[0]) <= 3.402823466e38f);
#pragma unroll
    for (int e = 1; e < Q4<HD>::EPL; ++e) {
        mn = fminf(mn, x[e]);
        mx = fmaxf(mx, x[e]);
        bad |= !(fabsf(x[e]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int off = W / 2; off; off >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    }
    const unsigned mask = __ballot_sync(0xffffffffu, bad) & (W == 32 ? 0xffffffffu : (0xffffu << (lane & 16)));
    return q4_scale_of(mask ? CUDART_NAN_F : mn, mx);
}

static __device__ __noinline__ float q4_code_at_border(float x, float m, float d) { return (float)rint(((double)x - (double)m) / (double)d); }

// code of x.  The fp32 quotient is off by less than 4e-6 where it is below 16; only next to a border between two codes
// does that matter, and there the quotient is formed in double (an fp32 value minus an fp16 one and the border times d are
// both exact in double, or far apart).
__device__ __forceinline__ uint32_t q4_code(float x, float m, float d, float inv) {
    if (!(d > 0.f)) return 0u;
    const float y = (x - m) * inv;
    float q = rintf(y);
    if (fabsf(fabsf(y - q) - 0.5f) < 1e-5f) q = q4_code_at_border(x, m, d);
    return (uint32_t)fminf(fmaxf(q, 0.f), 15.f);
}

// The codes of a lane's EPL values, dim e in bits 4e.
template <int HD>
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[Q4<HD>::EPL], Q4Scale s) {
    const float m = __half2float(s.m), d = __half2float(s.d), inv = __frcp_rn(d);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < Q4<HD>::EPL; ++e) w |= q4_code(x[e], m, d, inv) << (4 * e);
    return w;
}

__device__ __forceinline__ uint32_t q4_scale_word(Q4Scale s) {
    return (uint32_t)__half_as_ushort(s.d) | ((uint32_t)__half_as_ushort(s.m) << 16);
}

// A warp stores the codes and scales of one row of K (V = false) or V into a block at `blk` (shared or global memory).
template <int HD, bool V>
__device__ __forceinline__ void q4_store_row(uint8_t* blk, int s, uint32_t codes, Q4Scale sc, int lane) {
    using F = Q4<HD>;
    const int D = F::EPL * lane;
    if (V) {
#pragma unroll
        for (int e = 0; e < F::EPL; e += 2) blk[q4_v_byte<HD>(s, D + e)] = (uint8_t)(codes >> (4 * e));
    } else if (F::EPL == 4) {
        *reinterpret_cast<uint16_t*>(blk + q4_k_byte<HD>(s, D)) = (uint16_t)codes;
    } else {
        blk[q4_k_byte<HD>(s, D)] = (uint8_t)codes;
    }
    if (D % 64 == 0)
        *reinterpret_cast<uint32_t*>(blk + (V ? F::VS_OFF : F::KS_OFF) + s * F::SROWB + 4 * (D / 64)) = q4_scale_word(sc);
}

// fp16 value of a code: m + d * code, exact in fp32 but for far apart m and d, rounded to fp16 once.
__device__ __forceinline__ float q4_value(uint32_t code, float d, float m) { return fmaf((float)code, d, m); }

// The frequencies rope_freq() computes, before the factors, once on the host: in the kernels every CTA would spend two double
// transcendentals per pair on them, on the path in front of its first product.
void rope_freq_table(const RopeArgs& r, float (&freq)[64]);

struct KvQ4PrologueArgs {
    PrefillArgs a;             // kc, vc, out are those of the attention launch behind it and not used here
    uint8_t* cache;
    __half* k16;               // fp16 copies of the cache rows [n_kv][n_past + batch][hd]
    __half* v16;
    float* q32;                // or nullptr; the queries as fp32, rotated and not scaled, instead of a.q16, and no copies
    unsigned* tickets;         // arrival counters of the launch behind this one, set to zero
    int n_tickets;
    int cache_ctx;             // positions of the 4-bit cache
    float freq[64];            // see rope_freq_table
};

cudaError_t kv_q4_set_attributes();
cudaError_t launch_kv_store_q4(uint8_t* cache, const float* k, const float* v, int heads, int head_dim, int n_ctx, int pos_base,
                               int batch, const int* d_pos, cudaStream_t stream, unsigned long long* launches);
cudaError_t launch_kv_load_q4(const uint8_t* cache, uint16_t* kc, uint16_t* vc, int heads, int head_dim, int n_ctx, int row_base,
                              int rows, int dst_ctx, int dst_base, cudaStream_t stream, unsigned long long* launches);
cudaError_t launch_kv_shift_q4(uint8_t* cache, int n_layer, int n_kv, int head_dim, int n_ctx, int n_keep, int shift,
                               cudaStream_t stream, unsigned long long* launches);
cudaError_t launch_prefill_q4_prologue(const KvQ4PrologueArgs& a, cudaStream_t stream, unsigned long long* launches);

// Decode over the 4-bit cache.  The heads of a kv head are taken eight at a time (a kv head with more is read by two CTAs).
struct DecodeQ4Args {
    const float* q;
    const float* k_new;
    const float* v_new;
    uint8_t* cache;
    float* out;
    float* ws_o;
    float* ws_ml;
    float* grp_o;
    float* grp_ml;
    unsigned* tickets;
    const int* d_pos;
    int n_head, n_kv, n_ctx, n_splits, group, n_groups;
    int heads_per_cta, head_blocks;     // heads of one CTA, CTAs that share a kv head's slice
    float scale;
    int fuse, overlap;
    RopeArgs rope;
    PreArgs pre;
    float freq[64];                     // RoPE frequencies before the optional factors, theta^(-2i/n_rot) rounded to fp32
    // A chunk of `batch` tokens behind n_past rows instead of one token at *d_pos (batch 0): the rows of a kv head are its
    // (token, head) pairs, heads_per_cta = 8 of them per CTA, q is rotated already and the chunk's rows are in the cache.
    int n_past = 0, batch = 0;
    __half* out16 = nullptr;            // fp16 output of a chunk, instead of `out`
    static constexpr int emit_partial = 0;       // always the normalised output (emit_final)
    int8_t* out_qs = nullptr;
    float* out_scales = nullptr;
};
int decode_q4_num_splits(int head_blocks, int sm_count);
cudaError_t decode_q4_set_attributes();
cudaError_t launch_decode_q4(const DecodeQ4Args& a, int head_dim, cudaStream_t stream, unsigned long long* launches);

} // namespace oattn

// Writing, reading back and rolling the 4-bit KV cache, and the prologue of the prefill call that uses it.
#include <math.h>

#include <mutex>

#include "f32x2.cuh"
#include "kv_q4.cuh"

namespace oattn {

namespace {

// The careful form of a lane's 16 codes, out of line and from the row itself: hardly ever taken.
__device__ __noinline__ uint2 q4_codes16(const float* src, float m, float d, float inv) {
    uint2 w = make_uint2(0u, 0u);
    for (int i = 0; i < 8; ++i) {
        w.x |= q4_code(src[i], m, d, inv) << (4 * i);
        w.y |= q4_code(src[32 + i], m, d, inv) << (4 * i);
    }
    return w;
}

// of three, NaN where any of them is
__device__ __forceinline__ float min_nan(float a, float b, float c) { float r; asm("min.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float max_nan(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// ---- store --------------------------------------------------------------------------------------------------------
// One CTA per (block of 16 positions, kv head): warps 0..3 four rows of K each, warps 4..7 four rows of V.  Eight lanes (HD 128)
// or four (HD 64) share a row, four lanes a 64-dim group, a lane 16 dims: the 8 of word t, i and the 8 of word t, i + 1, so that
// it owns two neighbouring code words of K, and the minimum and maximum of a group cost two shuffles.  The block is put
// together in shared memory and leaves in 16-byte pieces; of a block at either end of the range only the stored rows' bytes do.
// Bound by the fp32 rows it reads, 1024 bytes per position and head against 144 written: 16384 positions of 8 heads take 33.4 us
// on a cold cache (4.6 TB/s, 0.70 of the measured copy bandwidth), with the issue slots 62 % busy and 5.4 cycles per issue
// spent on loads -- neither alone is the limit.  A warp per row, four or two values a lane, needs five shuffles twice per
// row and a double division per row instead of per four: 49 us against 21 for 8192 positions.  The heads of a block are
// neighbours in the grid because they are neighbours in the rows.
constexpr int kStoreThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kStoreThreads, 5) kv_store_q4_kernel(uint8_t* cache, const float* k, const float* v, int heads,
                                                                    int n_ctx, int pos_base, int batch, const int* d_pos) {
    using F = Q4<HD>;
    constexpr int LPR = 4 * F::NG;                        // lanes of a row
    __shared__ __align__(16) uint8_t s_blk[F::BLOCK];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();                                           // no early trigger: with it a read-back behind this call took 4 us longer
    const int head = blockIdx.x;                          // the heads of a token lie next to each other in k and v
    int first = pos_base;
    if (d_pos) {
        first = *d_pos;
        if (first < 0 || first >= n_ctx) return;
    }
    const int b = (first >> 4) + blockIdx.y + 65535 * blockIdx.z;      // block of the sequence
    const int row0 = max(first - 16 * b, 0), row1 = min(first + batch - 16 * b, 16);     // its rows that are stored
    if (row1 <= 0) return;                                // the grid's last plane is not full
    const bool is_v = warp >= 4;
    const int s = (warp & 3) * 4 + lane / 8, t = lane & 3, g = (lane % 8) / 4;           // HD 64: lanes with g = 1 idle
    const bool on = g < F::NG && s >= row0 && s < row1;
    const float* src = (is_v ? v : k) + ((long long)(16 * b + s - first) * heads + head) * HD + 64 * g + 8 * t;
    float x[16];
    if (on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 q = *reinterpret_cast<const float4*>(src + 32 * (i >> 1) + 4 * (i & 1));
            x[4 * i] = q.x; x[4 * i + 1] = q.y; x[4 * i + 2] = q.z; x[4 * i + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.f;
    }
    float mn = x[0], mx = x[0];
#pragma unroll
    for (int i = 0; i < 16; i += 2) { mn = min_nan(mn, x[i], x[i + 1]); mx = max_nan(mx, x[i], x[i + 1]); }
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, mn, off), w = __shfl_xor_sync(0xffffffffu, mx, off);
        mn = min_nan(mn, u, u);
        mx = max_nan(mx, w, w);
    }
    const Q4Scale sc = q4_scale_of(mn, mx);
    const float m = __half2float(sc.m), d = __half2float(sc.d), inv = __frcp_rn(d);
    uint32_t w[2] = {0u, 0u};
    // code = round((x - m) / d): adding 1.5 * 2^23 rounds to an integer, ties to even.  `far`: how close any of the 16 came to a
    // border between two codes.  Four codes are put together in fp32, 16 bits of an integer.
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const F2 lo(x[i], x[i + 1]), hi(x[i + 2], x[i + 3]), mm(-m, -m), ii(inv, inv), up(12582912.f, 12582912.f), down(-12582912.f, -12582912.f);
        const F2 y0 = (lo + mm) * ii, y1 = (hi + mm) * ii;
        const F2 c0 = (y0 + up) + down, c1 = (y1 + up) + down;
        const F2 e0 = fma2(c0, F2(-1.f, -1.f), y0), e1 = fma2(c1, F2(-1.f, -1.f), y1);
        far = fmaxf(far, fmaxf(fmaxf(fabsf(e0.x()), fabsf(e0.y())), fmaxf(fabsf(e1.x()), fabsf(e1.y()))));
        const float four = fmaf(fmaf(fmaf(c1.y(), 16.f, c1.x()), 16.f, c0.y()), 16.f, c0.x());
        w[i >> 3] |= (__float_as_uint(four + 8388608.f) & 0xffffu) << (4 * (i & 4));
    }
    if (!(d > 0.f)) {
        w[0] = w[1] = 0u;
    } else if (on && (far > 0.5f - 1e-5f || (mn - m) * inv < -0.25f || (mx - m) * inv > 15.25f)) {
        // next to a border, or a group whose offset is coarse against its step, so that codes have to be clamped
        const uint2 c = q4_codes16(src, m, d, inv);
        w[0] = c.x;
        w[1] = c.y;
    }
    if (on) {
        if (!is_v) {
            *reinterpret_cast<uint2*>(s_blk + s * F::ROWB + (t * (HD / 32) + 2 * g) * 4) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                s_blk[q4_v_byte<HD>(s, 64 * g + 32 * (i >> 2) + 8 * t + 2 * (i & 3))] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
        }
        if (t == 0) *reinterpret_cast<uint32_t*>(s_blk + (is_v ? F::VS_OFF : F::KS_OFF) + s * F::SROWB + 4 * g) = q4_scale_word(sc);
    }
    static_assert(LPR <= 8, "eight lanes per row");
    __syncthreads();
    uint8_t* blk = cache + ((size_t)head * q4_blocks(n_ctx) + b) * F::BLOCK;
    if (row0 == 0 && row1 == 16) {
        if (tid < F::BLOCK / 16) *reinterpret_cast<uint4*>(blk + 16 * tid) = *reinterpret_cast<const uint4*>(s_blk + 16 * tid);
        return;
    }
    // some rows: K words and the scales word by word, V byte by byte
    for (int i = tid; i < 4 * F::ROWB; i += kStoreThreads)
        if (i / (F::ROWB / 4) >= row0 && i / (F::ROWB / 4) < row1) reinterpret_cast<uint32_t*>(blk)[i] = reinterpret_cast<const uint32_t*>(s_blk)[i];
    for (int i = tid; i < 16 * F::ROWB; i += kStoreThreads) {
        const int row = 8 * (i & 1) + 2 * ((i >> 4) & 3) + ((i >> 1) & 1);
        if (row >= row0 && row < row1) blk[F::V_OFF + i] = s_blk[F::V_OFF + i];
    }
    if (tid < 2 * 16 * F::NG) {
        const int row = tid % (16 * F::NG) / F::NG;
        if (row >= row0 && row < row1) reinterpret_cast<uint32_t*>(blk + F::KS_OFF)[tid] = reinterpret_cast<const uint32_t*>(s_blk + F::KS_OFF)[tid];
    }
}

// ---- read back ----------------------------------------------------------------------------------------------------
// One warp turns rows [row0, row1) of a block into fp16; dk, dv: where row 0 of the block would go.  K: a lane takes the four
// (two) code words of place t of a row, 16 bytes, and writes 16-byte pieces, four lanes 64 bytes.  V: a word holds a pair of
// dims of four rows, so the block passes through shared memory (`s_v`, kVStride bytes a row: the lanes' 4-byte stores
// then fall into 32 different banks).  FIT: for products, where a group with a value beyond fp16 is NaN (see q4_fit).  32768 positions of 8 heads: 28.8 us for 172 MB, 0.91 of the measured copy bandwidth; a warp
// per row with byte loads took 61.5 us.
template <int HD>
constexpr int kVStride = HD * 2 + 16;

template <int HD>
__device__ __forceinline__ uint4 q4_eight(uint32_t w, float d, float m) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = q4_value((w >> (4 * e)) & 15u, d, m);
    return make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
}

// The step of a group whose values become operands in fp16.  One that holds a larger value counts as NaN: as an infinity it would
// give a score of minus infinity where the query is negative, and the row would vanish from a softmax that it belongs to.
__device__ __forceinline__ float q4_fit(float d, float m) { return fmaf(15.f, d, m) >= 65520.f ? CUDART_NAN_F : d; }

template <int HD, bool FIT>
__device__ __forceinline__ void q4_load_block(const uint8_t* blk, __half* dk, __half* dv, int row0, int row1, uint8_t* s_v, int lane) {
    using F = Q4<HD>;
    constexpr int NW = HD / 32, NG = F::NG;
    const int r = lane >> 2, t = lane & 3;
    uint32_t kw[2][NW], vw[NG][4], ks[2][NG], vs[4][NG];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint8_t* at = blk + (8 * j + r) * F::ROWB + t * (F::ROWB / 4);
        if constexpr (NW == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            kw[j][0] = v.x; kw[j][1] = v.y; kw[j][2] = v.z; kw[j][3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            kw[j][0] = v.x; kw[j][1] = v.y;
        }
    }
#pragma unroll
    for (int q = 0; q < NG; ++q) {
        const uint4 v = *reinterpret_cast<const uint4*>(blk + F::V_OFF + 512 * q + 16 * lane);
        vw[q][0] = v.x; vw[q][1] = v.y; vw[q][2] = v.z; vw[q][3] = v.w;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int j = 0; j < 2; ++j) ks[j][g] = *reinterpret_cast<const uint32_t*>(blk + F::KS_OFF + (8 * j + r) * F::SROWB + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i)      // byte i of a word: row 2t, 2t + 8, 2t + 1, 2t + 9
            vs[i][g] = *reinterpret_cast<const uint32_t*>(blk + F::VS_OFF + (2 * t + 8 * (i & 1) + (i >> 1)) * F::SROWB + 4 * g);
    }
    auto dm = [](uint32_t w, float& d, float& m) {
        d = __half2float(__ushort_as_half((uint16_t)w));
        m = __half2float(__ushort_as_half((uint16_t)(w >> 16)));
        if (FIT) d = q4_fit(d, m);
    };
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = 8 * j + r;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            float d, m;
            dm(ks[j][i >> 1], d, m);
            const uint4 v = q4_eight<HD>(kw[j][i], d, m);
            if (row >= row0 && row < row1) *reinterpret_cast<uint4*>(dk + (size_t)row * HD + 32 * i + 8 * t) = v;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + 8 * (i & 1) + (i >> 1);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float d, m;
            dm(vs[i][g], d, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t c = vw[g][j] >> (8 * i);
                *reinterpret_cast<uint32_t*>(s_v + row * kVStride<HD> + 32 * (4 * g + j) + 4 * r) =
                    pack_half2(q4_value(c & 15u, d, m), q4_value((c >> 4) & 15u, d, m));
            }
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
        const int c = lane + 32 * i, row = c / (HD / 8), col = c % (HD / 8);
        const uint4 v = *reinterpret_cast<const uint4*>(s_v + row * kVStride<HD> + 16 * col);
        if (row >= row0 && row < row1) *reinterpret_cast<uint4*>(dv + (size_t)row * HD + 8 * col) = v;
    }
    __syncwarp();
}

constexpr int kLoadWarps = 8;

template <int HD>
__global__ void __launch_bounds__(32 * kLoadWarps) kv_load_q4_kernel(const uint8_t* cache, uint16_t* kc, uint16_t* vc, int heads,
                                                                     int n_ctx, int row_base, int rows, int dst_ctx, int dst_base) {
    __shared__ __align__(16) uint8_t s_v[kLoadWarps][16 * kVStride<HD>];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    pdl_wait();
    const int b0 = row_base >> 4, nb = ((row_base + rows - 1) >> 4) - b0 + 1;
    const long long job = (long long)blockIdx.x * kLoadWarps + warp;
    if (job >= (long long)heads * nb) return;
    const int head = (int)(job / nb), b = b0 + (int)(job % nb);
    const uint8_t* blk = cache + ((size_t)head * q4_blocks(n_ctx) + b) * Q4<HD>::BLOCK;
    // row 0 of the block; may lie in front of the destination, whose rows outside [row0, row1) are not touched
    const long long at = ((long long)head * dst_ctx + dst_base + 16 * b - row_base) * HD;
    q4_load_block<HD, false>(blk, reinterpret_cast<__half*>(kc) + at, reinterpret_cast<__half*>(vc) + at, max(row_base - 16 * b, 0),
                      min(row_base + rows - 16 * b, 16), s_v[warp], lane);
}

// ---- roll -----------------------------------------------------------------------------------------------------------
// Row r becomes row r + shift for n_keep <= r < n_ctx - shift, the last `shift` rows become zero.  One CTA per (layer, kv head),
// tensor and 64 dims' worth of its bytes: 32 bytes of every K row, or 512 consecutive bytes of V codes, and one group's
// scales.  It walks the blocks in order; a step brings the blocks that hold the source rows of kShiftBlocks blocks to
// shared memory and writes those blocks from there.  Sources lie at or behind the place they go to, and those of later
// steps behind everything a step writes, so the copies of the next steps run while this one writes.
constexpr int kShiftThreads = 512;
constexpr int kShiftBlocks = 32;
constexpr int kShiftWindows = 4;           // steps in flight, this one among them

template <int HD>
struct ShiftWindow {
    static constexpr int CODES = 512, SCALES = 16 * Q4<HD>::SROWB, PART = CODES + SCALES;
    static constexpr int BYTES = (kShiftBlocks + 1) * PART;
};

constexpr int shift_smem(int head_dim) { return kShiftWindows * (head_dim == 128 ? ShiftWindow<128>::BYTES : ShiftWindow<64>::BYTES); }

template <int HD>
__global__ void __launch_bounds__(kShiftThreads) kv_shift_q4_kernel(uint8_t* cache, int n_ctx, int n_keep, int shift) {
    using F = Q4<HD>;
    using W = ShiftWindow<HD>;
    extern __shared__ __align__(16) uint8_t smem[];       // kShiftWindows windows
    pdl_wait();
    const bool is_v = blockIdx.x >= F::NG;
    const int h = blockIdx.x % F::NG;                      // which 32 bytes of a K row, which 512 of V; group of the scales
    const int warp = threadIdx.x >> 5, c = threadIdx.x & 31;
    const int nblk = q4_blocks(n_ctx);
    uint8_t* base = cache + (size_t)blockIdx.y * nblk * F::BLOCK;
    const int first = n_keep >> 4;
    const int last = n_ctx - shift;                       // first row that becomes zero
    const int skip = shift & 15;                          // row i of a step lies at row i + skip of its window
    // A warp takes a block, lane c the 16-byte piece c of its codes (two pieces per K row) and row c's scale word
    const int piece = is_v ? F::V_OFF + 512 * h + 16 * c : (c >> 1) * F::ROWB + 32 * h + 16 * (c & 1);
    const int s_off = is_v ? F::VS_OFF : F::KS_OFF;

    auto load = [&](int step) {
        const int b0 = first + step * kShiftBlocks + (shift >> 4);
        const uint32_t dst = smem_u32(smem + (step % kShiftWindows) * W::BYTES) + 16 * c;
        for (int i = warp; i < kShiftBlocks + 1; i += kShiftThreads / 32) {
            if (b0 + i >= nblk) break;
            const uint8_t* blk = base + (size_t)(b0 + i) * F::BLOCK;
            cp_async_16(dst + i * W::PART, blk + piece, 16);
            if (c < W::SCALES / 16) cp_async_16(dst + i * W::PART + W::CODES, blk + s_off + 16 * c, 16);
        }
        cp_async_commit();
    };
    // Where the lane's bytes come from, relative to the window's block: K one piece, V the words of place t of the four source
    // rows 2t, 2t + 8, 2t + 1, 2t + 9 (t = c % 4) and which byte of them; the scale word.
    int from[4];
    uint32_t sel[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = 2 * (c & 3) + 8 * (e & 1) + (e >> 1) + skip, ss = i & 15;
        from[e] = (i >> 4) * W::PART + ((c & ~3) + ((ss & 7) >> 1)) * 16;
        sel[e] = (uint32_t)(4 + 2 * (ss & 1) + (ss >> 3)) << (4 * e) | (0x3210u & ~(0xfu << (4 * e)));
    }
    const int k_from = (((c >> 1) + skip) >> 4) * W::PART + (((c >> 1) + skip) & 15) * 32 + 16 * (c & 1);
    const int sc_from = (((c & 15) + skip) >> 4) * W::PART + W::CODES + (((c & 15) + skip) & 15) * F::SROWB + 4 * h;

    const int steps = (nblk - first + kShiftBlocks - 1) / kShiftBlocks;
#pragma unroll
    for (int step = 0; step < kShiftWindows - 1; ++step) {
        if (step < steps) load(step); else cp_async_commit();
    }
    for (int step = 0; step < steps; ++step) {
        cp_async_wait<kShiftWindows - 2>();
        __syncthreads();                                  // this step's window has landed, the one before is free
        if (step + kShiftWindows - 1 < steps) load(step + kShiftWindows - 1); else cp_async_commit();
        const int b0 = first + step * kShiftBlocks, nb = min(kShiftBlocks, nblk - b0);
        for (int bl = warp; bl < nb; bl += kShiftThreads / 32) {
            const uint8_t* win = smem + (step % kShiftWindows) * W::BYTES + bl * W::PART;
            uint8_t* blk = base + (size_t)(b0 + bl) * F::BLOCK;
            const int row_b = (b0 + bl) * 16;             // first row of the block
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            uint32_t sw = 0u;
            // rows from `end` on become zero: their source words may lie outside what was loaded, and are cleared below
            const int end = last - row_b;
            if (end > 0) {
                if (is_v) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint4 u = *reinterpret_cast<const uint4*>(win + from[e]);
                        v.x = __byte_perm(v.x, u.x, sel[e]);
                        v.y = __byte_perm(v.y, u.y, sel[e]);
                        v.z = __byte_perm(v.z, u.z, sel[e]);
                        v.w = __byte_perm(v.w, u.w, sel[e]);
                    }
                    if (end < 16) {
                        uint32_t keep = 0u;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (2 * (c & 3) + 8 * (e & 1) + (e >> 1) < end) keep |= 255u << (8 * e);
                        v.x &= keep; v.y &= keep; v.z &= keep; v.w &= keep;
                    }
                } else if ((c >> 1) < end) {
                    v = *reinterpret_cast<const uint4*>(win + k_from);
                }
                if ((c & 15) < end) sw = *reinterpret_cast<const uint32_t*>(win + sc_from);
            }
            uint8_t* dst = blk + piece;
            if (row_b >= n_keep && row_b + 16 <= n_ctx) {
                *reinterpret_cast<uint4*>(dst) = v;
                if (c < 16) *reinterpret_cast<uint32_t*>(blk + s_off + c * F::SROWB + 4 * h) = sw;
                continue;
            }
            // a block at either end: only the rows that move
            auto moves = [&](int i) { return row_b + i >= n_keep && row_b + i < n_ctx; };
            if (is_v) {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (moves(2 * (c & 3) + 8 * (e & 1) + (e >> 1)))
#pragma unroll
                        for (int k = 0; k < 4; ++k) dst[4 * k + e] = (uint8_t)(w[k] >> (8 * e));
            } else if (moves(c >> 1)) {
                *reinterpret_cast<uint4*>(dst) = v;
            }
            if (c < 16 && moves(c)) *reinterpret_cast<uint32_t*>(blk + s_off + c * F::SROWB + 4 * h) = sw;
        }
    }
}

// ---- prefill prologue -------------------------------------------------------------------------------------------
// The chunk's tokens, one CTA each: q -> [bias, norm, RoPE] -> * scale*log2(e) -> fp16 (what the attention kernels read),
// k -> [bias, norm, RoPE] -> 4-bit row, v -> [bias] -> 4-bit row; the rows' fp16 values also go to the copies the attention
// reads.  The other CTAs turn the cache rows in front of the chunk into fp16, once for all query tiles: expanding them inside
// the attention kernel would repeat that for each of its tiles (16 for 512 tokens of a 4-head group), on the warps that bound it.
// 512 tokens of 32/8 heads behind 8192 rows: 19 us on a cold cache, 13 for the tokens alone (instruction issue, 0.6 of the slots:
// a warp takes a row at a time) and 9.6 for the rows alone (43 MB); the attention behind it takes 72.  Queries rotated in registers instead
// of through shared memory: 1.1 us less, included.
// For a short chunk (see DecodeQ4Args) the queries stay fp32 and nothing is copied: the decode kernel reads the 4-bit rows.
constexpr int kPrologueThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kPrologueThreads, 4) prefill_q4_prologue_kernel(const __grid_constant__ KvQ4PrologueArgs p) {
    using F = Q4<HD>;
    const PrefillArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.n_past + a.batch;
    const int nblk = q4_blocks(p.cache_ctx);
    const bool rope_q = (a.fuse & 1) != 0, rope_k = (a.fuse & 2) != 0, append = (a.fuse & 4) != 0;
    pdl_trigger();
    __shared__ __align__(16) uint8_t s_v[kPrologueThreads / 32][16 * kVStride<HD>];
    // the two kinds of CTAs alternate, so that an SM has copies to run while its tokens wait for their rows
    const int n_copy = (int)gridDim.x - a.batch, both = 2 * min(a.batch, n_copy);
    const int bid = blockIdx.x;
    const bool copies = bid < both ? (bid & 1) != 0 : n_copy > a.batch;
    const int idx = bid < both ? bid >> 1 : bid - both / 2;
    if (copies) {
        pdl_wait();
        const int expand = append ? a.n_past : rows, nb = q4_blocks(expand);
        const long long job = (long long)idx * (kPrologueThreads / 32) + warp;
        if (job >= (long long)a.n_kv * nb) return;
        const int head = (int)(job / nb), b = (int)(job % nb);
        const size_t dst = ((size_t)head * rows + 16 * b) * HD;
        q4_load_block<HD, true>(p.cache + ((size_t)head * nblk + b) * F::BLOCK, p.k16 + dst, p.v16 + dst, 0, min(expand - 16 * b, 16), s_v[warp], lane);
        return;
    }
    const int b = idx, pos = a.n_past + b;
    const float qs = a.scale * LOG2E;
    const int jobs = a.n_head + (append ? 2 * a.n_kv : 0);
    // A warp has eight head rows in flight (48 rows over 8 warps is the usual case), in shared memory rather than in registers: the loop
    // over them is not unrolled, because the instruction cache is what a launch of a few microseconds waits for.
    constexpr int W = kPrologueThreads / 32, RB = 8;
    static_assert(RB * HD * 4 <= 16 * kVStride<HD>, "the rows fit in the warp's part of s_v");
    float* rows_s = reinterpret_cast<float*>(s_v[warp]);
    struct Row { int kind, head; };                       // q, k or v
    auto describe = [&](int job) {
        Row r;
        r.kind = job < a.n_head ? 0 : (job < a.n_head + a.n_kv ? 1 : 2);
        r.head = r.kind == 0 ? job : (r.kind == 1 ? job - a.n_head : job - a.n_head - a.n_kv);
        return r;
    };
    auto load_rows = [&](int j0) {
        for (int u = 0; u < RB && j0 + u * W < jobs; ++u) {
            const Row r = describe(j0 + u * W);
            const float* src = (r.kind == 0 ? a.q : (r.kind == 1 ? a.k_new : a.v_new)) + ((size_t)b * (r.kind == 0 ? a.n_head : a.n_kv) + r.head) * HD;
            if (4 * lane < HD) cp_async_16(smem_u32(rows_s + u * HD + 4 * lane), src + 4 * lane, 16);
        }
        cp_async_commit();
    };
    pdl_wait();
    load_rows(warp);
    // cos and sin in double: a key's code is a decision at a border, so the rotated key is rounded to fp32 once
    __shared__ double s_cos[HD / 2], s_sin[HD / 2];
    __shared__ float2 s_cs[HD / 2];                       // rounded, for the queries
    if (rope_q || rope_k) {
        for (int i = tid; i < a.rope.n_rot / 2; i += kPrologueThreads) {
            float f = p.freq[i];
            if (a.rope.freq_factors) f = __fdiv_rn(f, a.rope.freq_factors[i]);
            double sn, cs;
            sincos((double)__fmul_rn((float)pos, f), &sn, &cs);
            s_sin[i] = sn; s_cos[i] = cs;
            s_cs[i] = make_float2((float)cs, (float)sn);
        }
    }
    __syncthreads();
    if (b == 0) {
        if (tid == 0 && a.status) *a.status = 0;
        for (int i = tid; i < p.n_tickets; i += kPrologueThreads) p.tickets[i] = 0;
    }
    for (int j0 = warp; j0 < jobs; j0 += W * RB) {
        if (j0 != warp) load_rows(j0);
        cp_async_wait<0>();
        __syncwarp();
#pragma unroll 1
        for (int u = 0; u < RB && j0 + u * W < jobs; ++u) {
            const Row r = describe(j0 + u * W);
            float* row = rows_s + u * HD;
            float x[F::EPL];
#pragma unroll
            for (int e = 0; e < F::EPL; ++e) x[e] = row[F::EPL * lane + e];
            const float* bias = r.kind == 0 ? a.pre.bias_q : (r.kind == 1 ? a.pre.bias_k : a.pre.bias_v);
            if (bias) {
#pragma unroll
                for (int e = 0; e < F::EPL; ++e) x[e] += bias[(size_t)r.head * HD + F::EPL * lane + e];
            }
            const float* nw = r.kind == 0 ? a.pre.norm_q : (r.kind == 1 ? a.pre.norm_k : nullptr);
            if (nw) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < F::EPL; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
                for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
                const float rn = 1.0f / sqrtf(ss / (float)HD + a.pre.eps);
#pragma unroll
                for (int e = 0; e < F::EPL; ++e) x[e] = x[e] * rn * nw[F::EPL * lane + e];
            }
            if (r.kind == 0 && rope_q && a.rope.n_rot == HD) {
                // a pair's two elements are in this lane or 16 lanes away
                if (a.rope.rope_type != 1) {
#pragma unroll
                    for (int e = 0; e < F::EPL; e += 2) {
                        const float2 cs = s_cs[(F::EPL * lane + e) / 2];
                        const float v0 = x[e], v1 = x[e + 1];
                        x[e] = v0 * cs.x - v1 * cs.y;
                        x[e + 1] = v0 * cs.y + v1 * cs.x;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < F::EPL; ++e) {
                        const float2 cs = s_cs[F::EPL * (lane & 15) + e];
                        const float y = __shfl_xor_sync(0xffffffffu, x[e], 16);
                        x[e] = fmaf(lane < 16 ? -y : y, cs.y, x[e] * cs.x);
                    }
                }
            } else if (r.kind == 0 ? rope_q : (r.kind == 1 && rope_k)) {
                // the row passes through shared memory: a pair's two elements may lie in any two lanes
#pragma unroll
                for (int e = 0; e < F::EPL; ++e) row[F::EPL * lane + e] = x[e];
                __syncwarp();
                for (int pp = lane; pp < a.rope.n_rot / 2; pp += 32) {
                    int i0, i1;
                    rope_pair_index(a.rope.rope_type, pp, a.rope.n_rot, i0, i1);
                    if (r.kind == 0) {
                        const float v0 = row[i0], v1 = row[i1], c = s_cs[pp].x, s = s_cs[pp].y;
                        row[i0] = v0 * c - v1 * s;
                        row[i1] = v0 * s + v1 * c;
                    } else {
                        const double v0 = row[i0], v1 = row[i1], c = s_cos[pp], s = s_sin[pp];
                        row[i0] = (float)(v0 * c - v1 * s);
                        row[i1] = (float)(v0 * s + v1 * c);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < F::EPL; ++e) x[e] = row[F::EPL * lane + e];
            }
            if (r.kind == 0 && p.q32) {
                float* dst = p.q32 + ((size_t)b * a.n_head + r.head) * HD + F::EPL * lane;
#pragma unroll
                for (int e = 0; e < F::EPL; ++e) dst[e] = x[e];
                continue;
            }
            if (r.kind == 0) {
                __half* dst = a.q16 + ((size_t)b * a.n_head + r.head) * HD + F::EPL * lane;
#pragma unroll
                for (int e = 0; e < F::EPL; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_half2(x[e] * qs, x[e + 1] * qs);
                continue;
            }
            const Q4Scale s = q4_scale<HD>(x, lane);
            const uint32_t codes = q4_codes<HD>(x, s);
            uint8_t* blk = p.cache + ((size_t)r.head * nblk + (pos >> 4)) * F::BLOCK;
            if (r.kind == 2) q4_store_row<HD, true>(blk, pos & 15, codes, s, lane);
            else             q4_store_row<HD, false>(blk, pos & 15, codes, s, lane);
            if (p.q32) continue;
            __half* dst = (r.kind == 1 ? p.k16 : p.v16) + ((size_t)r.head * rows + pos) * HD + F::EPL * lane;
            const float m = __half2float(s.m), d = q4_fit(__half2float(s.d), m);
#pragma unroll
            for (int e = 0; e < F::EPL; e += 2)
                *reinterpret_cast<uint32_t*>(dst + e) = pack_half2(q4_value((codes >> (4 * e)) & 15u, d, m), q4_value((codes >> (4 * e + 4)) & 15u, d, m));
        }
        __syncwarp();                                     // every lane is done with the rows
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

cudaError_t kv_q4_set_attributes() {
    cudaError_t e = cudaFuncSetAttribute(kv_shift_q4_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, shift_smem(128));
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(kv_shift_q4_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, shift_smem(64));
}

cudaError_t launch_kv_store_q4(uint8_t* cache, const float* k, const float* v, int heads, int head_dim, int n_ctx, int pos_base,
                               int batch, const int* d_pos, cudaStream_t stream, unsigned long long* launches) {
    const int blocks = d_pos ? 1 : ((pos_base + batch - 1) >> 4) - (pos_base >> 4) + 1;
    const dim3 grid(heads, min(blocks, 65535), (blocks + 65534) / 65535);
    const cudaError_t e = head_dim == 128 ? launch_dependent(kv_store_q4_kernel<128>, grid, kStoreThreads, 0, stream, 1, cache, k, v, heads, n_ctx, pos_base, batch, d_pos)
                                          : launch_dependent(kv_store_q4_kernel<64>, grid, kStoreThreads, 0, stream, 1, cache, k, v, heads, n_ctx, pos_base, batch, d_pos);
    if (launches) *launches += 1;
    return e;
}

cudaError_t launch_kv_load_q4(const uint8_t* cache, uint16_t* kc, uint16_t* vc, int heads, int head_dim, int n_ctx, int row_base,
                              int rows, int dst_ctx, int dst_base, cudaStream_t stream, unsigned long long* launches) {
    const long long jobs = (long long)heads * (((row_base + rows - 1) >> 4) - (row_base >> 4) + 1);
    const dim3 grid((unsigned)((jobs + kLoadWarps - 1) / kLoadWarps));
    const cudaError_t e = head_dim == 128 ? launch_dependent(kv_load_q4_kernel<128>, grid, 32 * kLoadWarps, 0, stream, 1, cache, kc, vc, heads, n_ctx, row_base, rows, dst_ctx, dst_base)
                                          : launch_dependent(kv_load_q4_kernel<64>, grid, 32 * kLoadWarps, 0, stream, 1, cache, kc, vc, heads, n_ctx, row_base, rows, dst_ctx, dst_base);
    if (launches) *launches += 1;
    return e;
}

cudaError_t launch_kv_shift_q4(uint8_t* cache, int n_layer, int n_kv, int head_dim, int n_ctx, int n_keep, int shift,
                               cudaStream_t stream, unsigned long long* launches) {
    const dim3 grid(2 * head_dim / 64, n_layer * n_kv);
    const cudaError_t e = head_dim == 128 ? launch_dependent(kv_shift_q4_kernel<128>, grid, kShiftThreads, shift_smem(128), stream, 1, cache, n_ctx, n_keep, shift)
                                          : launch_dependent(kv_shift_q4_kernel<64>, grid, kShiftThreads, shift_smem(64), stream, 1, cache, n_ctx, n_keep, shift);
    if (launches) *launches += 1;
    return e;
}

cudaError_t launch_prefill_q4_prologue(const KvQ4PrologueArgs& p, cudaStream_t stream, unsigned long long* launches) {
    const PrefillArgs& a = p.a;
    const long long jobs = p.q32 ? 0 : (long long)a.n_kv * q4_blocks((a.fuse & 4) ? a.n_past : a.n_past + a.batch);
    constexpr int W = kPrologueThreads / 32;
    const dim3 grid((unsigned)(a.batch + (jobs + W - 1) / W));
    const cudaError_t e = a.head_dim == 128 ? launch_dependent(prefill_q4_prologue_kernel<128>, grid, kPrologueThreads, 0, stream, 1, p)
                                            : launch_dependent(prefill_q4_prologue_kernel<64>, grid, kPrologueThreads, 0, stream, 1, p);
    if (launches) *launches += 1;
    return e;
}

} // namespace oattn

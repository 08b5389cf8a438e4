// Chunked-prefill causal GQA attention, warp-level mma.sync version.
//
// Same contract as flash_attention_prefill_mma_k (src/kernels.cu:1351-1568): query token t of
// the chunk sees cache rows 0..n_past+t.  This kernel is the in-library cross-check and the
// fall-back shape coverage for the tcgen05 kernel (prefill_tc.cu); it shares that kernel's
// prologue (q already rotated, scaled by scale*log2(e) and converted to fp16 in q16).
//
// One CTA = 4 warps = 64 query rows of ONE kv head, a row being a (token, head-in-group) pair:
// row R -> token t0 + R/G, head kvh*G + R%G, so one pass over the K/V rows of the kv head serves
// all G heads of floor(64/G) tokens.  K/V tiles of 64 rows are staged with cp.async (2 stages in
// flight); each warp computes S (16 x 64), the causal mask, online softmax and O += P V for its
// 16 rows.
#include "attn_internal.h"

namespace oattn {

namespace {

constexpr int kThreads = 128;
constexpr int kTile = 64;
constexpr int kStages = 3;

template <int HD>
struct PrefillSmem {
    static constexpr int ROWB = HD * 2;
    static constexpr int CHUNKS = ROWB / 16;
    static constexpr int TILE_BYTES = kTile * ROWB;
    static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
    static constexpr int Q_OFF = kStages * STAGE_BYTES;
    static constexpr int TOTAL = Q_OFF + 64 * ROWB;
};

// SPLIT (see PrefillArgs): a CTA walks one of n_split slices of its rows and leaves the unscaled output.
template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2) prefill_mma_kernel(const PrefillArgs p) {
    using L = PrefillSmem<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = lane >> 2, t = lane & 3;
    const int G = p.n_head / p.n_kv;
    const int TB = 64 / G;                       // tokens per CTA
    const int kvh = blockIdx.y;
    // heaviest blocks (latest tokens) first
    const int tb = gridDim.x - 1 - blockIdx.x;
    const int t0 = tb * TB;
    const int ntok = min(TB, p.batch - t0);
    const int kv_end = p.n_past + t0 + ntok;     // rows any query of this CTA may see
    const int nt_all = (kv_end + kTile - 1) / kTile;
    const int split = SPLIT ? blockIdx.z : 0;
    const int tile0 = SPLIT ? (int)((long long)nt_all * split / p.n_split) : 0;
    const int nt = SPLIT ? (int)((long long)nt_all * (split + 1) / p.n_split) - tile0 : nt_all;

    const __half* Kg = reinterpret_cast<const __half*>(p.kc) + (size_t)kvh * p.n_ctx * HD;
    const __half* Vg = reinterpret_cast<const __half*>(p.vc) + (size_t)kvh * p.n_ctx * HD;
    const uint32_t smem_base = smem_u32(smem);

    auto load_tile = [&](int tile, int stage) {
        const int row0 = (tile0 + tile) * kTile;
        const uint32_t sb = smem_base + stage * L::STAGE_BYTES;
        constexpr int PER_MAT = kTile * L::CHUNKS;
#pragma unroll
        for (int i = 0; i < 2 * PER_MAT / kThreads; ++i) {
            const int idx = tid + i * kThreads;
            const int which = idx / PER_MAT;
            const int rem = idx % PER_MAT;
            const int row = rem / L::CHUNKS, chunk = rem % L::CHUNKS;
            const int grow = row0 + row;
            const bool ok = grow < kv_end;
            const __half* src = (which ? Vg : Kg) + (size_t)(ok ? grow : 0) * HD + chunk * 8;
            cp_async_16(sb + which * L::TILE_BYTES + swz<L::ROWB>(row, chunk), src, ok ? 16 : 0);
        }
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        if (s < nt) load_tile(s, s);
        cp_async_commit();
    }

    // Q rows -> shared (zero for rows that map to no token)
    for (int i = tid; i < 64 * L::CHUNKS; i += kThreads) {
        const int R = i / L::CHUNKS, chunk = i % L::CHUNKS;
        const int tok = R / G, hg = R % G;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (tok < ntok) v = *reinterpret_cast<const uint4*>(p.q16 + ((size_t)(t0 + tok) * p.n_head + kvh * G + hg) * HD + chunk * 8);
        *reinterpret_cast<uint4*>(smem + L::Q_OFF + swz<L::ROWB>(R, chunk)) = v;
    }
    __syncthreads();
    uint32_t qa[HD / 16][4];
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
        const int row = warp * 16 + (lane & 7) + 8 * ((lane >> 3) & 1);
        ldmatrix_x4(smem_base + L::Q_OFF + swz<L::ROWB>(row, 2 * kk + (lane >> 4)), qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3]);
    }

    // last visible cache row of this thread's two query rows
    int vis[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        const int R = warp * 16 + r + 8 * hh;
        const int tok = R / G;
        vis[hh] = (tok < ntok) ? p.n_past + t0 + tok : -1;
    }

    float o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f; }
    float m_run[2] = {-CUDART_INF_F, -CUDART_INF_F};
    float l_run[2] = {0.f, 0.f};

    for (int it = 0; it < nt; ++it) {
        cp_async_wait<kStages - 2>();
        __syncthreads();
        {
            const int nxt = it + kStages - 1;
            if (nxt < nt) load_tile(nxt, nxt % kStages);
            cp_async_commit();
        }
        const int stage = it % kStages;
        const int row0 = (tile0 + it) * kTile;
        const uint32_t sK = smem_base + stage * L::STAGE_BYTES;
        const uint32_t sV = sK + L::TILE_BYTES;

        float s[kTile / 8][4];
#pragma unroll
        for (int j = 0; j < kTile / 8; ++j) { s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f; }
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
#pragma unroll
            for (int jp = 0; jp < kTile / 16; ++jp) {
                uint32_t b0, b1, b2, b3;
                const int row = 16 * jp + 8 * (lane >> 4) + (lane & 7);
                ldmatrix_x4(sK + swz<L::ROWB>(row, 2 * kk + ((lane >> 3) & 1)), b0, b1, b2, b3);
                mma_16816(s[2 * jp], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b0, b1);
                mma_16816(s[2 * jp + 1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b2, b3);
            }
        }
        // causal mask (also hides zero-filled rows >= kv_end, which are > vis for every row)
        if (row0 + kTile - 1 > p.n_past + t0) {
#pragma unroll
            for (int j = 0; j < kTile / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row0 + 8 * j + 2 * t + (e & 1) > vis[e >> 1]) s[j][e] = -CUDART_INF_F;
        }
        float alpha[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            float mx = -CUDART_INF_F;
#pragma unroll
            for (int j = 0; j < kTile / 8; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * hh], s[j][2 * hh + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run[hh], mx);
            const float m_safe = (m_new == -CUDART_INF_F) ? 0.f : m_new;
            alpha[hh] = fast_exp2(m_run[hh] - m_safe);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < kTile / 8; ++j) {
                s[j][2 * hh] = fast_exp2(s[j][2 * hh] - m_safe);
                s[j][2 * hh + 1] = fast_exp2(s[j][2 * hh + 1] - m_safe);
                sum += s[j][2 * hh] + s[j][2 * hh + 1];
            }
            l_run[hh] = l_run[hh] * alpha[hh] + sum;
            m_run[hh] = m_new;
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) {
                o[j][0] *= alpha[0]; o[j][1] *= alpha[0];
                o[j][2] *= alpha[1]; o[j][3] *= alpha[1];
            }
        }
#pragma unroll
        for (int ks = 0; ks < kTile / 16; ++ks) {
            const uint32_t pa0 = pack_half2(s[2 * ks][0], s[2 * ks][1]);
            const uint32_t pa1 = pack_half2(s[2 * ks][2], s[2 * ks][3]);
            const uint32_t pa2 = pack_half2(s[2 * ks + 1][0], s[2 * ks + 1][1]);
            const uint32_t pa3 = pack_half2(s[2 * ks + 1][2], s[2 * ks + 1][3]);
#pragma unroll
            for (int jp = 0; jp < HD / 16; ++jp) {
                uint32_t b0, b1, b2, b3;
                const int row = 16 * ks + (lane & 7) + 8 * ((lane >> 3) & 1);
                ldmatrix_x4_trans(sV + swz<L::ROWB>(row, 2 * jp + (lane >> 4)), b0, b1, b2, b3);
                mma_16816(o[2 * jp], pa0, pa1, pa2, pa3, b0, b1);
                mma_16816(o[2 * jp + 1], pa0, pa1, pa2, pa3, b2, b3);
            }
        }
    }
    cp_async_wait<0>();

#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        float l = l_run[hh];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int R = warp * 16 + r + 8 * hh;
        const int tok = R / G, hg = R % G;
        if (tok < ntok) {
            if constexpr (SPLIT) {
                const size_t row = ((size_t)split * (gridDim.x * TB) + t0 + tok) * p.n_head + kvh * G + hg;
                if (t == 0) reinterpret_cast<float2*>(p.part_ml)[row] = make_float2(m_run[hh], l);
#pragma unroll
                for (int j = 0; j < HD / 8; ++j)
                    *reinterpret_cast<float2*>(p.part_o + row * HD + 8 * j + 2 * t) = make_float2(o[j][2 * hh], o[j][2 * hh + 1]);
                continue;
            }
            const float inv = 1.f / l;
            if (p.out16) {
                __half* dst16 = p.out16 + ((size_t)(t0 + tok) * p.n_head + kvh * G + hg) * HD;
#pragma unroll
                for (int j = 0; j < HD / 8; ++j)
                    *reinterpret_cast<uint32_t*>(dst16 + 8 * j + 2 * t) = pack_half2(o[j][2 * hh] * inv, o[j][2 * hh + 1] * inv);
                continue;
            }
            float* dst = p.out + ((size_t)(t0 + tok) * p.n_head + kvh * G + hg) * HD;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j)
                *reinterpret_cast<float2*>(dst + 8 * j + 2 * t) = make_float2(o[j][2 * hh] * inv, o[j][2 * hh + 1] * inv);
        }
    }
}

// Joins the slices of a split call: a row's HD/4 threads take 4 dims each.  Bound by reading the slices, from L2: 64 tokens of 32
// heads in eight slices are 8 MB.
template <int HD>
__global__ void __launch_bounds__(256) prefill_merge_kernel(const PrefillArgs p, int tokens) {
    pdl_trigger();
    pdl_wait();
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = at / (HD / 4);                     // (token, head)
    const int c4 = (int)(at % (HD / 4));
    if (row >= (long long)p.batch * p.n_head) return;
    const size_t step = (size_t)tokens * p.n_head;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row;
    const float4* o = reinterpret_cast<const float4*>(p.part_o) + row * (HD / 4) + c4;
    float M = -CUDART_INF_F;
#pragma unroll 4
    for (int s = 0; s < p.n_split; ++s) M = fmaxf(M, ml[s * step].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f;
#pragma unroll 4
    for (int s = 0; s < p.n_split; ++s) {
        const float2 x = ml[s * step];
        const float4 v = o[s * step * (HD / 4)];
        const float w = x.x == -CUDART_INF_F ? 0.f : fast_exp2(x.x - M);       // a slice that the mask hides from this row
        L += w * x.y;
        acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
    }
    const float inv = 1.f / L;
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    if (p.out16) reinterpret_cast<uint2*>(p.out16)[at] = make_uint2(pack_half2(acc.x, acc.y), pack_half2(acc.z, acc.w));
    else         reinterpret_cast<float4*>(p.out)[at] = acc;
}

template <int HD>
cudaError_t set_attributes() {
    const cudaError_t e = cudaFuncSetAttribute(prefill_mma_kernel<HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PrefillSmem<HD>::TOTAL);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(prefill_mma_kernel<HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PrefillSmem<HD>::TOTAL);
}

} // namespace

cudaError_t prefill_mma_set_attributes() {
    const cudaError_t e = set_attributes<128>();
    return e != cudaSuccess ? e : set_attributes<64>();
}

cudaError_t launch_prefill_merge(const PrefillArgs& a, int tokens, cudaStream_t stream, unsigned long long* launches) {
    const long long threads = (long long)a.batch * a.n_head * (a.head_dim / 4);
    const dim3 grid((unsigned)((threads + 255) / 256));
    const cudaError_t e = a.head_dim == 128 ? launch_dependent(prefill_merge_kernel<128>, grid, 256, 0, stream, 1, a, tokens)
                                            : launch_dependent(prefill_merge_kernel<64>, grid, 256, 0, stream, 1, a, tokens);
    if (launches) *launches += 1;
    return e;
}

// Two CTAs per SM; a 64-row tile takes one about 0.9 us.  64 tokens of 32/8 heads behind 8192 rows (32 CTAs, 9 slices) 32 us
// against 114, behind 1024 rows (2 slices) 21.5 against 23.
int prefill_mma_splits(int n_head, int n_kv, int n_past, int batch, int sm_count) {
    const int TB = 64 / (n_head / n_kv);
    const long long ctas = (long long)n_kv * ((batch + TB - 1) / TB);
    const int blocks = (n_past + min(batch, TB) + 127) / 128;            // of the shortest tile
    return (int)min(min(2ll * min(sm_count, kSplitCtas) / ctas, (long long)blocks / kSplitMinBlocks), (long long)kMaxPrefillSplits);
}

cudaError_t launch_prefill_mma(const PrefillArgs& a, cudaStream_t stream, unsigned long long* launches) {
    const int G = a.n_head / a.n_kv;
    const int TB = 64 / G;
    const dim3 grid((a.batch + TB - 1) / TB, a.n_kv, a.n_split);
    if (a.n_split > 1) {
        if (a.head_dim == 128) prefill_mma_kernel<128, true><<<grid, kThreads, PrefillSmem<128>::TOTAL, stream>>>(a);
        else                   prefill_mma_kernel<64, true><<<grid, kThreads, PrefillSmem<64>::TOTAL, stream>>>(a);
    } else {
        if (a.head_dim == 128) prefill_mma_kernel<128, false><<<grid, kThreads, PrefillSmem<128>::TOTAL, stream>>>(a);
        else                   prefill_mma_kernel<64, false><<<grid, kThreads, PrefillSmem<64>::TOTAL, stream>>>(a);
    }
    if (launches) *launches += 1;
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess || a.n_split == 1 ? e : launch_prefill_merge(a, (int)grid.x * TB, stream, launches);
}

} // namespace oattn

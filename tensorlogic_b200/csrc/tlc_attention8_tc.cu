// Attention of a long prompt over the 8-bit KV cache, on tcgen05 + TMEM.
//
// kv8_widen has written the sequence's blocks as f16 rows of whole-number codes, with the factors s_k, s_v of each block
// of 64 keys; a block is a tile here.  One CTA owns up to 128 (query, head) rows that share a KV head -- the G heads of
// the group times 128 / G positions -- and walks the tiles; two CTAs share an SM, so that one's matrix products run
// under the other's softmax.
//   S = Q.C_k^T   Q and codes in shared memory (TMA, 128-byte swizzle), f32 in tensor memory
//   softmax       one row per thread: x = S s_k scale log2(e) + log2(s_v), P = 2^(x - m + 8) in f16, where m follows the
//                 row's largest x only when that has risen by more than 2^7 (P stays below 2^15): the block's
//                 factor of V is part of P, its sum is divided by it again.  The sum is of P before it is rounded: a block
//                 of small values has little of P, which f16 may cut off, but all its part of the sum.  (f16 because the
//                 product's operands are: against 64 bits the output is off by 2.6e-4 to 2.7e-4, by 2.1e-4 from its own
//                 rounding alone.)  The open block's values are their own codes, factor 1, however small they are: it
//                 comes last, so that what it lifts m by is taken from sums in f32, not from P of a later block.
//   O += P.C_v    P from tensor memory, over the scores it was made from; codes of V as [key][d], the N-major operand
//
// Warps:  0  Q, K and V by TMA      1  tensor memory and MMA issue      2-5  softmax, rescale, output
//
// Bound by the tiles' way out of the L2: 2048 queries, 32 heads of 128 move 285 MB there in 41 us (7 TB/s; tensor pipe
// 45 %, as a product of 64 keys takes as long as one of 128), behind 11 us for the image: 54 us a call.  One CTA with twice
// the rows moves half of it and took 55 to 61 us a call, its softmax in turn with its own products.
//
// All waits are bounded; one that runs out sets the status word and lets the CTA drain, free its tensor memory and
// return.
#include <cuda.h>

#include "tlc_gemm_kernel.cuh"
#include "tlc_kv8.h"

using namespace tlc_gemm;

namespace {

constexpr int kRows = 128, kKeys = kKv8Block, kThreads = 192;
constexpr int kHalf = kKeys * 128;  // bytes of 64 keys x 64 values
template <int D> constexpr int kv_bytes() { return kHalf * (D / 64); }
// K and V tiles in flight: what two CTAs an SM leave room for
template <int D> constexpr int stages() { return D == 128 ? 2 : 3; }
template <int D> constexpr int smem_bytes_tc() { return 1024 + 1024 + kRows * D * 2 + 2 * stages<D>() * kv_bytes<D>(); }
constexpr int kTmemCols = 256;  // scores: two tiles of 64 columns; O: D
constexpr int kColO = 128;
constexpr float kBase = 8.f, kRise = 7.f;  // P = 2^(x - m + kBase), x <= m + kRise

struct Params {
    __half *out;
    const float4 *factors;  // [kv head][block]
    const int *lengths;     // [kv head][K, V]
    int I, H, G, RQ;
    int q_tiles, n_blocks, n_kv_heads;
    int pos0;
    float scale;  // times log2(e)
    tlc_dev_status *status;
    uint64_t wait_ns;
};

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tma_load_3d_el(uint32_t dst, const void *map, int x, int y, int z, uint32_t bar, uint32_t el) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"
        " @q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n}\n" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(el)
        : "memory");
}
// An average of what the cache holds lies within f16.  Its sum of P is of the values before they were rounded, so that
// values next to 65504 could come out up to 2^-11 above it, an infinity.  (NaN stays.)
__device__ __forceinline__ __half2 in_range(__half2 v) { return __hmax2_nan(__hmin2_nan(v, __float2half2_rn(65504.f)), __float2half2_rn(-65504.f)); }
// Columns of this thread's lane.  The load is waited for by tmem_ld_wait, which the registers pass through: nothing
// that uses them can be moved in front of it.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&a)[32], uint32_t (&b)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 32; e++) asm volatile("" : "+r"(a[e]), "+r"(b[e]));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}


template <int D>
__global__ void __launch_bounds__(kThreads, 2)
    attention8_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap q_map,
                         const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    constexpr int HALVES = D / 64, ST = stages<D>(), KV = kv_bytes<D>();
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *k_full = reinterpret_cast<uint64_t *>(base), *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST;
    uint64_t *s_full = v_empty + ST, *p_full = s_full + 2, *pv_done = p_full + 2, *q_full = pv_done + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(q_full + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    uint8_t *qs = base + 1024, *ks = qs + kRows * D * 2, *vs = ks + ST * KV;

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(q_full, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // (Dependents are let in when this CTA has its tensor memory: theirs must not be asked for first.)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // The last queries see the most keys: their tiles go first.
    const int hk = blockIdx.x % p.n_kv_heads, qt = p.q_tiles - 1 - blockIdx.x / p.n_kv_heads;
    const int G = p.G, RQ = p.RQ;
    const int keys = min(p.lengths[2 * hk], p.pos0 + p.I);  // (fewer than the queries' own: said below)
    const int k_end = min(keys, p.pos0 + min(p.I, (qt + 1) * RQ));
    const int n = (k_end + kKeys - 1) / kKeys;
    if (tid == 0 && qt == 0 && keys < p.pos0 + p.I && atomicCAS(&p.status->code, 0, TLC_DEV_INDEX) == 0) p.status->where = 400;

    if (warp == 0) {
        // ------------------------------ Q, K, V ------------------------------
        const uint32_t el = elect_one();
        const uint32_t bar_q = smem_u32(q_full);
        if (n > 0) mbar_arrive_expect_tx_el(q_full, G * RQ * D * 2, el);
#pragma unroll
        for (int h = 0; h < HALVES; h++)
            if (n > 0) tma_load_3d_el(smem_u32(qs + h * kRows * 128), &q_map, 64 * h, hk * G, qt * RQ, bar_q, el);
        bool ok = true;
        int sk = 0, sv = 0;
        uint32_t pk = 1, pv = 1;
        for (int j = 0; ok && n > 0 && j <= n; j++) {  // K of tile j, V of tile j - 1: the order in which they are used
            if (j < n) {
                ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[sk], pk, abort_flag, p.status, 61, p.wait_ns));
                if (!ok) break;
                const uint32_t bar = smem_u32(&k_full[sk]);
                mbar_arrive_expect_tx_el(&k_full[sk], KV, el);
#pragma unroll
                for (int h = 0; h < HALVES; h++) tma_load_3d_el(smem_u32(ks + sk * KV + h * kHalf), &k_map, 64 * h, j * kKeys, hk, bar, el);
                if (++sk == ST) sk = 0, pk ^= 1u;
            }
            if (j > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[sv], pv, abort_flag, p.status, 62, p.wait_ns));
                if (!ok) break;
                const uint32_t bar = smem_u32(&v_full[sv]);
                mbar_arrive_expect_tx_el(&v_full[sv], KV, el);
#pragma unroll
                for (int h = 0; h < HALVES; h++)
                    tma_load_3d_el(smem_u32(vs + sv * KV + h * kHalf), &v_map, 64 * h, (j - 1) * kKeys, hk, bar, el);
                if (++sv == ST) sv = 0, pv ^= 1u;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------ MMA ------------------------------
        const uint32_t el = elect_one();
        const uint32_t idesc_s = idesc_for(kKeys), idesc_o = idesc_for(D) | 1u << 16;  // (V: N-major)
        constexpr uint32_t MN = (uint32_t)(kHalf >> 4) << 16;  // the next 64 values of d: the next box
        const uint32_t q0 = (smem_u32(qs) & 0x3FFFF) >> 4, k0 = (smem_u32(ks) & 0x3FFFF) >> 4, v0 = (smem_u32(vs) & 0x3FFFF) >> 4;
        bool ok = n > 0 && mbar_wait(q_full, 0, abort_flag, p.status, 63, p.wait_ns);
        int sk = 0, sv = 0;
        uint32_t pk = 0, pv = 0;
        auto scores = [&](int j) {  // S of tile j
            ok = mbar_wait(&k_full[sk], pk, abort_flag, p.status, 64, p.wait_ns) && ok;
            // its columns hold P of tile j - 2
            if (j >= 2) ok = mbar_wait(&pv_done[j & 1], (uint32_t)((j - 2) >> 1) & 1u, abort_flag, p.status, 65, p.wait_ns) && ok;
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            if (ok) {
                const uint32_t at = tmem + (j & 1) * kKeys, kd = k0 + sk * (KV >> 4);
#pragma unroll
                for (int k16 = 0; k16 < D / 16; k16++)
                    umma_f16(at, desc_at(q0 + (k16 >> 2) * (kRows * 128 >> 4) + (k16 & 3) * 2),
                             desc_at(kd + (k16 >> 2) * (kHalf >> 4) + (k16 & 3) * 2), idesc_s, k16 > 0, el);
            }
            umma_commit(&k_empty[sk], el);
            umma_commit(&s_full[j & 1], el);
            if (++sk == ST) sk = 0, pk ^= 1u;
        };
        if (n > 0) scores(0);
        for (int j = 0; j < n; j++) {
            if (j + 1 < n) scores(j + 1);
            ok = mbar_wait(&v_full[sv], pv, abort_flag, p.status, 66, p.wait_ns) && ok;
            ok = mbar_wait(&p_full[j & 1], (uint32_t)(j >> 1) & 1u, abort_flag, p.status, 67, p.wait_ns) && ok;
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            if (ok) {
                const uint32_t at = tmem + (j & 1) * kKeys, vd = v0 + sv * (KV >> 4);
#pragma unroll
                for (int k16 = 0; k16 < kKeys / 16; k16++)
                    umma_f16_ts(tmem + kColO, at + k16 * 8, (desc_at(vd + k16 * 128) & ~(uint64_t)(1u << 16)) | MN, idesc_o,
                                (j > 0 || k16 > 0) ? 1u : 0u, el);
            }
            umma_commit(&v_empty[sv], el);
            umma_commit(&pv_done[j & 1], el);
            if (++sv == ST) sv = 0, pv ^= 1u;
        }
        __syncwarp();
    } else {
        // ------------------------------ softmax ------------------------------
        const int quarter = warp & 3, r = 32 * quarter + lane;
        const uint32_t tl = tmem + ((uint32_t)(32 * quarter) << 16);
        const int qi = qt * RQ + r / G, head = hk * G + r % G;
        const bool there = r < G * RQ && qi < p.I;
        const int last = min(p.pos0 + qi, k_end - 1);         // last key this row sees
        const int warp_first = p.pos0 + qt * RQ + 32 * quarter / G;
        const bool negative = p.scale < 0.f;
        const float scale = fabsf(p.scale);
        const float4 *factors = p.factors + (size_t)hk * p.n_blocks;
        float m_run = -INFINITY, l_run = 0.f;
        float4 next = n > 0 ? factors[0] : make_float4(0.f, 0.f, 0.f, 0.f);
        for (int j = 0; j < n; j++) {
            const int j0 = j * kKeys;
            const float4 fac = next;
            if (j + 1 < n) next = factors[j + 1];
            const uint32_t ts = tl + (j & 1) * kKeys;
            // (a factor of zero would make NaN of a masked score)
            const float f = fmaxf(fac.x * scale, 1e-30f), lw = fac.y;
            mbar_wait(&s_full[j & 1], (uint32_t)(j >> 1) & 1u, abort_flag, p.status, 68, p.wait_ns);
            __syncwarp();
            tc_fence_after();
            uint32_t s[2][32];
            tmem_ld32_issue(ts, s[0]);
            tmem_ld32_issue(ts + 32, s[1]);
            tmem_ld_wait(s[0], s[1]);
            if (negative) {
#pragma unroll
                for (int e = 0; e < 64; e++) s[e >> 5][e & 31] ^= 0x80000000u;
            }
            if (j0 + kKeys - 1 > warp_first || j0 + kKeys > k_end) {
#pragma unroll
                for (int e = 0; e < 64; e++)
                    if (e > last - j0) s[e >> 5][e & 31] = 0xFF800000u;
            }
            float mx[4];
#pragma unroll
            for (int e = 0; e < 4; e++) mx[e] = __uint_as_float(s[0][e]);
#pragma unroll
            for (int e = 4; e < 64; e += 2) mx[(e >> 1) & 3] = fmaxf(mx[(e >> 1) & 3], fmaxf(__uint_as_float(s[e >> 5][e & 31]), __uint_as_float(s[e >> 5][(e & 31) + 1])));
            const float xm = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), f, lw);
            const bool moved = xm > m_run + kRise;  // (the first finite one always: m_run is -inf)
            const float m_new = moved ? xm : m_run;
            const float corr = moved ? exp2_of(m_run - m_new) : 1.f;
            m_run = m_new;
            const float c = lw + kBase - (m_run == -INFINITY ? 0.f : m_run);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t pk[32];
#pragma unroll
            for (int e = 0; e < 32; e++) {
                const float a = exp2_of(fmaf(__uint_as_float(s[e >> 4][2 * (e & 15)]), f, c));
                const float d = exp2_of(fmaf(__uint_as_float(s[e >> 4][2 * (e & 15) + 1]), f, c));
                sum[e & 3] += a;
                sum[e & 3] += d;
                const __half2 h = __floats2half2_rn(a, d);
                pk[e] = *reinterpret_cast<const uint32_t *>(&h);
            }
            l_run = l_run * corr + ((sum[0] + sum[1]) + (sum[2] + sum[3])) * fac.z;
            if (j > 0 && __any_sync(0xffffffffu, moved)) {
                mbar_wait(&pv_done[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u, abort_flag, p.status, 69, p.wait_ns);
                __syncwarp();
                tc_fence_after();
#pragma unroll
                for (int d = 0; d < D; d += 32) {
                    uint32_t o[32];
                    tmem_ld32(tl + kColO + d, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                    tmem_st32(tl + kColO + d, o);
                }
            }
            tmem_st32(ts, pk);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[j & 1]);
        }
        const bool ok = n == 0 || mbar_wait(&pv_done[(n - 1) & 1], (uint32_t)((n - 1) >> 1) & 1u, abort_flag, p.status, 70, p.wait_ns);
        __syncwarp();
        tc_fence_after();
        const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;  // (no keys: zeros; NaN stays)
        __half *out = p.out + ((size_t)qi * p.H + head) * D;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            if (n > 0) tmem_ld32(tl + kColO + c, o);
            else
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = 0u;
            if (ok && there) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    __align__(16) __half2 h[4];
#pragma unroll
                    for (int i = 0; i < 8; i += 2)
                        h[i / 2] = in_range(__floats2half2_rn(__uint_as_float(o[e + i]) * inv, __uint_as_float(o[e + i + 1]) * inv));
                    *reinterpret_cast<uint4 *>(out + c + e) = *reinterpret_cast<const uint4 *>(h);
                }
            }
            __syncwarp();
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemCols) : "memory");
    }
}

template <int D>
int32_t launch(tlc_ctx *ctx, const Params &p, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v) {
    static bool configured[64] = {};
    if (!configured[ctx->device & 63]) {
        TLC_CUDA(cudaFuncSetAttribute(attention8_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes_tc<D>()));
        TLC_CUDA(cudaFuncSetAttribute(attention8_tc_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                      cudaSharedmemCarveoutMaxShared));
        configured[ctx->device & 63] = true;
    }
    const cudaError_t le = tlc_launch_pdl(ctx, attention8_tc_kernel<D>, dim3((unsigned)(p.q_tiles * p.n_kv_heads)), dim3(kThreads),
                                          smem_bytes_tc<D>(), p, q, k, v);
    if (le != cudaSuccess) {
        cudaGetLastError();
        return tlc_fail(TLC_ERR_CUDA, "attention8 launch failed: %s", cudaGetErrorString(le));
    }
    TLC_CHECK_LAUNCH(ctx);
    return TLC_OK;
}

}  // namespace

int32_t kv8_attention_tc(tlc_ctx *ctx, tlc_kvcache8 *cache, int layer, int sequence, const __half *q, __half *out, int I, int H,
                         int pos0, float scale) {
    const uint64_t D = cache->head_dim, Hkv = cache->n_kv_heads, rows = (uint64_t)cache->n_blocks * kKv8Block;
    Params p{};
    p.out = out;
    p.factors = cache->factors;
    p.lengths = kv8_view(cache, layer, sequence).lengths;
    p.I = I;
    p.H = H;
    p.G = H / (int)Hkv;
    p.RQ = kRows / p.G;
    p.q_tiles = (I + p.RQ - 1) / p.RQ;
    p.n_blocks = cache->n_blocks;
    p.n_kv_heads = (int)Hkv;
    p.pos0 = pos0;
    p.scale = scale * 1.4426950408889634f;
    p.status = ctx->dev_status;
    p.wait_ns = ctx->wait_ns;
    const uint64_t qd[3] = {D, (uint64_t)H, (uint64_t)I}, qst[2] = {D * 2, (uint64_t)H * D * 2};
    const uint32_t qb[3] = {64, (uint32_t)p.G, (uint32_t)p.RQ};
    const uint64_t kd[3] = {D, rows, Hkv}, kst[2] = {D * 2, rows * D * 2};
    const uint32_t kb[3] = {64, kKeys, 1};
    CUtensorMap qm, km, vm;
    if (!encode_map_nd(&qm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, q, 3, qd, qst, qb) ||
        !encode_map_nd(&km, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, cache->wide, 3, kd, kst, kb) ||
        !encode_map_nd(&vm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, cache->wide + Hkv * rows * D, 3, kd, kst, kb))
        return tlc_fail(TLC_ERR_CUDA, "attention8: tensor maps");
    if (int32_t rc = kv8_widen(ctx, cache, layer, sequence, (pos0 + I + kKv8Block - 1) / kKv8Block)) return rc;
    return D == 64 ? launch<64>(ctx, p, qm, km, vm) : launch<128>(ctx, p, qm, km, vm);
}

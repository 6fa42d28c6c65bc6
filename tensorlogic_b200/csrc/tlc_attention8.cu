// Grouped-query attention over the 8-bit KV cache (tlc_kv8.h).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale q_r.k_j - m_r),   j = 0 .. position of row r
//
// On sealed blocks k_j = s_k c_j and v_j = s_v c_j with integer codes c and one scale per block, so the tensor cores
// multiply the codes as they are (exact in f16) and s_k multiplies a score, s_v a block's product.
//
// attention8_kernel: an item is 8 * NT (query, head) rows that share a KV head, queries in the order (position, head of
// the group).  One, two or four warps of a CTA, or those of several CTAs, share its blocks; a warp takes one at a time,
// alone:
//   S^T = K.Q^T  16 keys x 8 rows a product, codes as the 16-row operand (PRMT makes it, tlc_kv8.h)
//   P            f32 maximum and sums over the keys of a row, P rounded to f16, times 2^12 so that small
//                probabilities keep their bits; the sum is of the rounded values.  (The product's operands are f16, and
//                P in two of them would be the product twice over: against 64 bits the output is off by 2.4e-4 to
//                3e-4, by 2.1e-4 from its own rounding alone.  The codes are off by up to 2^-8 of their block's largest.)
//   O^T += V^T.P P turned over by movmatrix, f32 accumulators of the block, scaled by s_v when they join O
// A warp's blocks arrive by cp.async in a ring of its own; a lane copies the very bytes it will use, so a warp needs no
// barrier and no other lane until the results of an item's warps are merged in shared memory.  CTAs that share its keys
// form clusters of up to eight: between two cluster barriers each takes some of the rows and pulls the others' results
// (distributed shared memory); of several clusters the last one (a ticket for each share of the rows) joins what all have
// left in the cache's workspace.
//
// Many sequences: bound by HBM while all warps have blocks (32 sequences of about 600 keys, 32 heads of 128: 33 us, 157 MB
// at 0.72 of the copy's rate; the tensor pipe is 15 % busy).  One sequence: by latency, 1.0 us a block and warp, and the
// merge (65000 keys, 4 KV heads of 64: 13.5 us, 12.3 where the L2 holds them; 512 keys 5.5, of which a call's launch is 3.6).
#include <cuda_fp16.h>

#include <algorithm>

#include "tlc_kv8.h"

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr float kShift = 12.f;        // P is held times 2^12
constexpr float kUp = 16777216.f;     // the codes' 2^24
constexpr float kLog2e = 1.4426950408889634f;
// CTAs an SM.  Rows of 64 values, up to eight rows an item: four, at 128 registers and half the ring, as a block is more
// latency than bytes (65000 keys, 4 KV heads: 13.7 -> 12.4 us; 64 sequences of 1500: 11.1 -> 10.4).
constexpr int places(int D, int nt) { return D == 64 && nt == 1 ? 4 : 2; }
template <int D, int NT> constexpr int stages() { return D == 64 && NT == 2 ? 6 : 3; }  // of 64 * D bytes (K or V of a block) per warp

struct Params {
    const __half *q;  // [batch * I, H, D]
    __half *out;
    Kv8View c;
    int I, H, G;
    int pos0;              // position of query 0 (positions == null)
    const int *positions;  // device int32[batch]: position of each sequence's query; negative: none
    int key_limit;         // keys the launch was sized for
    float scale;
    int items, row_tiles;
    int warps, nsplit;  // warps of a CTA per item (1, 2, 4), CTAs per item (more than one: of four warps)
    int cluster;        // CTAs of a cluster: nsplit if that is 1, 2, 4 or 8, else 8
    float *partial;  // of several clusters: [item][cluster][row][2], then [item][cluster][row][D]
    int *tickets;
    tlc_dev_status *status;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t low2(uint32_t w) { return __byte_perm(w, 0, 0x4140); }
__device__ __forceinline__ uint32_t high2(uint32_t w) { return __byte_perm(w, 0, 0x4342); }

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, places(D, NT)) attention8_kernel(const Params p) {
    constexpr int ROWS = 8 * NT, STAGE = kKv8Block * D, ST = stages<D, NT>(), LOADS = STAGE / 512, PITCH = D + 4;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float sm_m[kWarps][ROWS], sm_l[kWarps][ROWS];  // in a cluster: of the CTA in [0], for its peers
    __shared__ int sm_last;
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int warps = p.warps, sub = warp % warps, gtid = sub * 32 + lane, threads = 32 * warps;
    // (neighbours in different CTAs: a batch in the order of its lengths leaves no SM the longest ones)
    const int item = p.nsplit > 1 ? blockIdx.x / p.nsplit : blockIdx.x + warp / warps * gridDim.x;
    if (item >= p.items) return;
    const int split = p.nsplit > 1 ? blockIdx.x % p.nsplit : 0;
    const int rt = item % p.row_tiles, hk = item / p.row_tiles % p.c.n_kv_heads, b = item / p.row_tiles / p.c.n_kv_heads;
    auto barrier = [&]() {  // of the item's warps of this CTA
        if (warps == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / warps), "r"(threads) : "memory");
    };
    const int rows = p.I * p.G, r0 = rt * ROWS;
    const size_t head = (size_t)b * p.c.n_kv_heads + hk;
    auto row_of = [&](int r) { return ((size_t)b * p.I + r / p.G) * p.H + hk * p.G + r % p.G; };

    const int at0 = p.positions ? p.positions[b] : p.pos0, held = p.c.lengths[head * 2];
    const int keys = min(held, p.key_limit);  // what a row may see at most
    if (at0 >= 0 && at0 > keys - p.I && gtid == 0 && split == 0 && atomicCAS(&p.status->code, 0, TLC_DEV_INDEX) == 0)
        p.status->where = 400 + b;  // a query in front of its key: it sees what there is, and that is said
    const int pos0 = min(at0, keys);
    const int last = min(rows, r0 + ROWS) - 1;  // last row of the tile
    const int seen = pos0 < 0 ? 0 : min(keys, pos0 + last / p.G + 1);
    if (seen <= 0) {  // an idle slot, or nothing in the cache
        if (split == 0)
            for (int i = gtid; i < (last - r0 + 1) * (D / 8); i += threads)
                *reinterpret_cast<uint4 *>(p.out + row_of(r0 + i / (D / 8)) * D + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
        return;
    }
    const int units = (seen + kKv8Block - 1) / kKv8Block, sealed = held / kKv8Block;
    const int stride = p.nsplit * warps, u0 = split * warps + sub;
    const uint8_t *codes = p.c.codes + head * p.c.n_blocks * (2 * STAGE);
    const float2 *scales = reinterpret_cast<const float2 *>(p.c.scales) + head * p.c.n_blocks;

    // The ring: K and V of a block in turn.  Rows of 128 values: at the end the open block's, where this warp's turn comes
    // to it, f16, two stages of 32 keys each, and only the 16-key groups that anyone sees (32 sequences of about 600 keys,
    // 32 heads: 35.8 us with all of them read straight from memory behind the ring, 32.9 so).  Rows of 64: all of the open
    // block's loads at once, behind the ring (a token behind 512, 32 heads: 5.6 us so, 5.9 through the ring).
    constexpr bool kOpenInRing = D == 128;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (uint32_t)(warp * ST * STAGE + lane * 16);
    const int n_sealed = min(units, sealed), steps = u0 < n_sealed ? 2 * ((n_sealed - u0 + stride - 1) / stride) : 0;
    const bool has_open = kOpenInRing && units > sealed && u0 + (steps >> 1) * stride == sealed;
    const int groups = has_open ? (seen - sealed * kKv8Block + 15) / 16 : 0;
    const uint8_t *open = reinterpret_cast<const uint8_t *>(p.c.open + head * (2 * STAGE));
    auto fetch = [&](int n) {
        if constexpr (kOpenInRing) {
            const int part = n - steps, have = part < 0 ? 2 : part < 4 ? groups - 2 * (part & 1) : 0;  // halves of a stage
            const uint8_t *src = (part < 0 ? codes + ((size_t)(u0 + (n >> 1) * stride) * 2 + (n & 1)) * STAGE : open + part * STAGE) + lane * 16;
            const uint32_t dst = ring + (uint32_t)(n % ST * STAGE);
            if (have > 0) {
#pragma unroll
                for (int i = 0; i < LOADS / 2; i++) copy16(dst + i * 512, src + i * 512);
            }
            if (have > 1) {
#pragma unroll
                for (int i = LOADS / 2; i < LOADS; i++) copy16(dst + i * 512, src + i * 512);
            }
        } else if (n < steps) {
            const uint8_t *src = codes + ((size_t)(u0 + (n >> 1) * stride) * 2 + (n & 1)) * STAGE + lane * 16;
            const uint32_t dst = ring + (uint32_t)(n % ST * STAGE);
#pragma unroll
            for (int i = 0; i < LOADS; i++) copy16(dst + i * 512, src + i * 512);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");  // (empty ones keep the count)
    };
    const float2 first = u0 < n_sealed ? scales[u0] : make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < ST - 1; i++) fetch(i);

    // Queries: row r0 + 8 nt + g as the 8-column operand, and -128 sum q for rows 2t and 2t + 1
    uint32_t qf[NT][D / 16][2];
    float start[NT][2];
    int end[NT][2];  // keys that rows 2t and 2t + 1 see
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = r0 + 8 * nt + g;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < rows) v = *reinterpret_cast<const uint4 *>(p.q + row_of(r) * D + c * 32 + t * 8);
            qf[nt][2 * c][0] = v.x;
            qf[nt][2 * c][1] = v.y;
            qf[nt][2 * c + 1][0] = v.z;
            qf[nt][2 * c + 1][1] = v.w;
            const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
            for (int e = 0; e < 4; e++) sum += __low2float(h[e]) + __high2float(h[e]);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            start[nt][e] = __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4) * (-128.f / kUp);
            end[nt][e] = min(keys, pos0 + min(r0 + 8 * nt + 2 * t + e, rows - 1) / p.G + 1);
        }
    }
    const int all_see = min(keys, pos0 + r0 / p.G + 1);  // keys that every row sees

    float m_run[NT][2], l_run[NT][2], o[NT][D / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m_run[nt][0] = m_run[nt][1] = -INFINITY;
        l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }

    // Softmax of a block's scores s[kg][nt][..] (keys 16 kg + kv8_key(g), .. + kv8_key(g + 8) of rows 2t, 2t + 1): P as
    // the second product's operand, this lane's part of its sums, and what the rows' O has to be multiplied with.
    auto softmax = [&](int u, float (&s)[4][NT][4], float factor, uint32_t (&pf)[4][NT][2], float (&psum)[NT][2], float (&corr)[NT][2]) {
        const bool masked = (u + 1) * kKv8Block > all_see;
        float shift[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float mx[2][4];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[kg][nt][e] *= factor;
                    if (masked && u * kKv8Block + 16 * kg + 4 * (g >> 1) + (g & 1) + 2 * (e >> 1) >= end[nt][e & 1]) s[kg][nt][e] = -INFINITY;
                }
                mx[0][kg] = fmaxf(s[kg][nt][0], s[kg][nt][2]);
                mx[1][kg] = fmaxf(s[kg][nt][1], s[kg][nt][3]);
            }
#pragma unroll
            for (int e = 0; e < 2; e++) shift[nt][e] = fmaxf(fmaxf(mx[e][0], mx[e][1]), fmaxf(mx[e][2], mx[e][3]));
        }
#pragma unroll
        for (int d = 4; d < 32; d *= 2)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) shift[nt][e] = fmaxf(shift[nt][e], __shfl_xor_sync(0xffffffffu, shift[nt][e], d));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float m_new = fmaxf(m_run[nt][e], shift[nt][e]), m_safe = m_new == -INFINITY ? 0.f : m_new;
                corr[nt][e] = exp2_of(m_run[nt][e] - m_safe);
                m_run[nt][e] = m_new;
                shift[nt][e] = kShift - m_safe;
                psum[nt][e] = 0.f;
            }
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const __half2 v = __floats2half2_rn(exp2_of(s[kg][nt][2 * h] + shift[nt][0]), exp2_of(s[kg][nt][2 * h + 1] + shift[nt][1]));
                    psum[nt][0] += __low2float(v);
                    psum[nt][1] += __high2float(v);
                    pf[kg][nt][h] = turned(*reinterpret_cast<const uint32_t *>(&v));
                }
        }
    };
    // The rows' sums of P over the lanes, while the second product runs.
    auto reduce = [&](float (&psum)[NT][2], const float (&corr)[NT][2]) {
#pragma unroll
        for (int d = 4; d < 32; d *= 2)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++) psum[nt][e] += __shfl_xor_sync(0xffffffffu, psum[nt][e], d);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) l_run[nt][e] = l_run[nt][e] * corr[nt][e] + psum[nt][e];
    };
    // O of 16 values of d (index dt): times corr, plus the block's product less 128 times the sum of P where V is codes
    auto join = [&](int dt, int nt, const float (&acc)[4], float factor, const float (&less)[NT][2], const float (&corr)[NT][2]) {
#pragma unroll
        for (int e = 0; e < 4; e++) o[nt][dt][e] = fmaf(o[nt][dt][e], corr[nt][e & 1], (acc[e] - less[nt][e & 1]) * factor);
    };

    // (Products that follow each other belong to different sums: a warp issues in order, and a sum is a chain.)
    constexpr int WIDE = NT == 1 ? 2 : 1;  // pairs of 16 values of d whose second products run side by side
    int step = 0;
    float2 factor = first;
    for (int u = u0; u < n_sealed; u += stride) {
        const float sk = factor.x, sv = factor.y;
        if (u + stride < n_sealed) factor = scales[u + stride];  // the next block's, a trip to memory ahead
        float s[4][NT][4], psum[NT][2], corr[NT][2], less[NT][2];
        uint32_t pf[4][NT][2];
        fetch(step + ST - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        uint32_t at = ring + (uint32_t)(step % ST * STAGE);
#pragma unroll
        for (int kg = 0; kg < 4; kg++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                s[kg][nt][0] = s[kg][nt][2] = start[nt][0];
                s[kg][nt][1] = s[kg][nt][3] = start[nt][1];
            }
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            uint4 w[4];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) w[kg] = lds128(at + (uint32_t)((kg * (D / 32) + c) * 512));
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    mma(s[kg][nt], low2(w[kg].x), low2(w[kg].z), high2(w[kg].x), high2(w[kg].z), qf[nt][2 * c][0], qf[nt][2 * c][1]);
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    mma(s[kg][nt], low2(w[kg].y), low2(w[kg].w), high2(w[kg].y), high2(w[kg].w), qf[nt][2 * c + 1][0], qf[nt][2 * c + 1][1]);
        }
        step++;
        softmax(u, s, kUp * sk * p.scale * kLog2e, pf, psum, corr);
        fetch(step + ST - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        at = ring + (uint32_t)(step % ST * STAGE);
#pragma unroll
        for (int c0 = 0; c0 < D / 32; c0 += WIDE) {
            float acc[WIDE][2][NT][4];
#pragma unroll
            for (int c = 0; c < WIDE; c++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[c][0][nt][e] = acc[c][1][nt][e] = 0.f;
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
#pragma unroll
                for (int c = 0; c < WIDE; c++) {
                    const uint4 w = lds128(at + (uint32_t)((kg * (D / 32) + c0 + c) * 512));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        mma(acc[c][0][nt], low2(w.x), low2(w.y), high2(w.x), high2(w.y), pf[kg][nt][0], pf[kg][nt][1]);
                        mma(acc[c][1][nt], low2(w.z), low2(w.w), high2(w.z), high2(w.w), pf[kg][nt][0], pf[kg][nt][1]);
                    }
                }
            }
            if (c0 == 0) {
                reduce(psum, corr);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) less[nt][e] = psum[nt][e] * (128.f / kUp);
            }
#pragma unroll
            for (int c = 0; c < WIDE; c++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    join(2 * (c0 + c), nt, acc[c][0][nt], kUp * sv, less, corr);
                    join(2 * (c0 + c) + 1, nt, acc[c][1][nt], kUp * sv, less, corr);
                }
        }
        step++;
    }
    // The open block
    if (kOpenInRing && has_open) {
        float s[4][NT][4], psum[NT][2], corr[NT][2];
        const float none[NT][2] = {};
        uint32_t pf[4][NT][2];
#pragma unroll
        for (int kg = 0; kg < 4; kg++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[kg][nt][0] = s[kg][nt][1] = s[kg][nt][2] = s[kg][nt][3] = 0.f;
        // (What a group that was not copied leaves of its scores is masked; of V it counts as zeros.)
        auto at = [&](int half) { return ring + (uint32_t)((step + half) % ST * STAGE); };
        fetch(step + ST - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
#pragma unroll
        for (int k16 = 0; k16 < D / 16; k16++) {
            uint4 w[4];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) w[kg] = lds128(at(kg >> 1) + (uint32_t)(((kg & 1) * (D / 16) + k16) * 512));
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma(s[kg][nt], w[kg].x, w[kg].z, w[kg].y, w[kg].w, qf[nt][k16][0], qf[nt][k16][1]);
        }
        step += 2;
        fetch(step + ST - 2);
        fetch(step + ST - 1);
        softmax(sealed, s, p.scale * kLog2e, pf, psum, corr);
        reduce(psum, corr);
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) {
            float acc[NT][4];
            uint4 w[4];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
                w[kg] = lds128(at(kg >> 1) + (uint32_t)(((kg & 1) * (D / 16) + dt) * 512));
                if (kg >= groups) w[kg] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma(acc[nt], w[kg].x, w[kg].z, w[kg].y, w[kg].w, pf[kg][nt][0], pf[kg][nt][1]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) join(dt, nt, acc[nt], 1.f, none, corr);
        }
    }
    if (!kOpenInRing && units > sealed && sealed % stride == u0) {
        const uint4 *kt = reinterpret_cast<const uint4 *>(p.c.open + head * (2 * STAGE)) + lane, *vt = kt + STAGE / 8;
        float s[4][NT][4], psum[NT][2], corr[NT][2];
        const float none[NT][2] = {};
        uint32_t pf[4][NT][2];
#pragma unroll
        for (int kg = 0; kg < 4; kg++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[kg][nt][0] = s[kg][nt][1] = s[kg][nt][2] = s[kg][nt][3] = 0.f;
#pragma unroll
        for (int k16 = 0; k16 < D / 16; k16++) {
            uint4 w[4];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) w[kg] = kt[(kg * (D / 16) + k16) * 32];
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma(s[kg][nt], w[kg].x, w[kg].z, w[kg].y, w[kg].w, qf[nt][k16][0], qf[nt][k16][1]);
        }
        softmax(sealed, s, p.scale * kLog2e, pf, psum, corr);
        reduce(psum, corr);
#pragma unroll
        for (int dt = 0; dt < D / 16; dt++) {
            float acc[NT][4];
            uint4 w[4];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) w[kg] = vt[(kg * (D / 16) + dt) * 32];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma(acc[nt], w[kg].x, w[kg].z, w[kg].y, w[kg].w, pf[kg][nt][0], pf[kg][nt][1]);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) join(dt, nt, acc[nt], 1.f, none, corr);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (warps == 1 && p.nsplit == 1) {
        // Nobody to merge with: O of rows 2t, 2t + 1 by their sums, turned over, two values of d a lane of row g.
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const float inv[2] = {1.0f / l_run[nt][0], 1.0f / l_run[nt][1]};
            const int r = r0 + 8 * nt + g;
            __half *to = p.out + row_of(min(r, rows - 1)) * D + 2 * t;
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const __half2 v = __floats2half2_rn(o[nt][i][2 * h] * inv[0], o[nt][i][2 * h + 1] * inv[1]);
                    const uint32_t w = turned(*reinterpret_cast<const uint32_t *>(&v));
                    if (r < rows) *reinterpret_cast<uint32_t *>(to + 16 * i + 8 * h) = w;
                }
        }
        return;
    }
    // A warp's O takes its ring's place: [row][D], rows PITCH apart.
    static_assert(ROWS * PITCH * 4 <= ST * STAGE, "O in the place of the ring");
    auto o_of = [&](int w) { return reinterpret_cast<float *>(smem + w * ST * STAGE); };
    __syncwarp();
    float *so = o_of(warp);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        if (g == 0) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                sm_m[warp][8 * nt + 2 * t + e] = m_run[nt][e];
                sm_l[warp][8 * nt + 2 * t + e] = l_run[nt][e];
            }
        }
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) so[(8 * nt + 2 * t + (e & 1)) * PITCH + 16 * i + g + 8 * (e >> 1)] = o[nt][i][e];
    }
    barrier();

    auto weight = [](float m, float l, float M) { return m == -INFINITY && l == 0.f ? 0.f : exp2_of(m - (M == -INFINITY ? 0.f : M)); };
    auto add = [](float4 &acc, const float4 &v, float w) {
        acc.x = fmaf(v.x, w, acc.x), acc.y = fmaf(v.y, w, acc.y), acc.z = fmaf(v.z, w, acc.z), acc.w = fmaf(v.w, w, acc.w);
    };
    auto store = [&](int r, int q, const float4 &acc, float l) {
        if (r0 + r >= rows) return;
        const float inv = 1.0f / l;  // (the largest p is 2^12; a row whose scores are NaN stays NaN)
        __align__(8) __half2 h[2] = {__floats2half2_rn(acc.x * inv, acc.y * inv), __floats2half2_rn(acc.z * inv, acc.w * inv)};
        *reinterpret_cast<uint2 *>(p.out + row_of(r0 + r) * D + 4 * q) = *reinterpret_cast<const uint2 *>(h);
    };
    // The warps of this CTA, four values a thread at a time
    constexpr int Q = D / 4;
    const int w0 = warp - sub;
    float M, L;
    float4 acc;
    auto of_warps = [&](int i) {
        const int r = i / Q;
        M = -INFINITY, L = 0.f, acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < warps; w++) M = fmaxf(M, sm_m[w0 + w][r]);
        for (int w = 0; w < warps; w++) {
            const float wgt = weight(sm_m[w0 + w][r], sm_l[w0 + w][r], M);
            L += sm_l[w0 + w][r] * wgt;
            add(acc, *reinterpret_cast<const float4 *>(o_of(w0 + w) + r * PITCH + 4 * (i % Q)), wgt);
        }
    };
    if (p.nsplit == 1) {
        for (int i = gtid; i < ROWS * Q; i += threads) {
            of_warps(i);
            store(i / Q, i % Q, acc, L);
        }
        return;
    }
    // (all four warps of the CTA are this item's from here on)
    {
        constexpr int MINE = ROWS * Q / kThreads;
        float4 mine[MINE];
        float M_of[MINE], L_of[MINE];
#pragma unroll
        for (int k = 0; k < MINE; k++) {
            of_warps(tid + k * kThreads);
            mine[k] = acc, M_of[k] = M, L_of[k] = L;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < MINE; k++) {
            const int i = tid + k * kThreads, r = i / Q;
            *reinterpret_cast<float4 *>(o_of(0) + r * PITCH + 4 * (i % Q)) = mine[k];
            if (i % Q == 0) sm_m[0][r] = M_of[k], sm_l[0][r] = L_of[k];
        }
    }
    const int rank = split % p.cluster, per = ROWS / p.cluster;  // this CTA's rows: per * rank ..
    auto cluster_barrier = [&]() {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    };
    auto peer = [](const void *at, int of) {
        uint32_t a;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(of));
        return a;
    };
    cluster_barrier();
    const int n_clusters = p.nsplit / p.cluster;
    const size_t slot = (size_t)item * n_clusters + split / p.cluster;
    float *part_ml = p.partial, *part_o = p.partial + (size_t)kKv8MaxParts * kKv8MaxRows * 2;
    for (int i = tid; i < per * Q; i += kThreads) {
        const int r = per * rank + i / Q, q = i % Q;
        float m[8], l[8];
        float4 v[8];
#pragma unroll
        for (int c = 0; c < 8; c++) {
            m[c] = -INFINITY, l[c] = 0.f, v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c >= p.cluster) continue;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(m[c]) : "r"(peer(&sm_m[0][r], c)));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(l[c]) : "r"(peer(&sm_l[0][r], c)));
            asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                         : "=f"(v[c].x), "=f"(v[c].y), "=f"(v[c].z), "=f"(v[c].w)
                         : "r"(peer(o_of(0) + r * PITCH + 4 * q, c)));
        }
        M = -INFINITY, L = 0.f, acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 8; c++) M = fmaxf(M, m[c]);
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const float wgt = weight(m[c], l[c], M);
            L += l[c] * wgt;
            add(acc, v[c], wgt);
        }
        if (n_clusters == 1) {
            store(r, q, acc, L);
        } else {
            if (q == 0) *reinterpret_cast<float2 *>(part_ml + (slot * ROWS + r) * 2) = make_float2(M, L);
            *reinterpret_cast<float4 *>(part_o + (slot * ROWS + r) * D + 4 * q) = acc;
        }
    }
    __syncwarp();
    cluster_barrier();  // a CTA leaves when its peers have pulled
    if (n_clusters == 1) return;
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        int *ticket = p.tickets + item * p.cluster + rank;
        sm_last = atomicAdd(ticket, 1) == n_clusters - 1;
        if (sm_last) *ticket = 0;
    }
    __syncthreads();
    if (!sm_last) return;
    __threadfence();
    // The last cluster, in the clusters' order: eight results in flight (one after the other, 74 of them took 16 us).
    for (int i = tid; i < per * Q; i += kThreads) {
        const int r = per * rank + i / Q, q = i % Q;
        M = -INFINITY, L = 0.f, acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c0 = 0; c0 < n_clusters; c0 += 8) {
            float2 ml[8];
            float4 v[8];
#pragma unroll
            for (int c = 0; c < 8; c++) {
                ml[c] = make_float2(-INFINITY, 0.f), v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c0 + c >= n_clusters) continue;
                const size_t at = ((size_t)item * n_clusters + c0 + c) * ROWS + r;
                ml[c] = __ldcg(reinterpret_cast<const float2 *>(part_ml + at * 2));
                v[c] = __ldcg(reinterpret_cast<const float4 *>(part_o + at * D + 4 * q));
            }
            float M_new = M;
#pragma unroll
            for (int c = 0; c < 8; c++) M_new = fmaxf(M_new, ml[c].x);
            const float old = weight(M, L, M_new);
            L *= old;
            acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
            M = M_new;
#pragma unroll
            for (int c = 0; c < 8; c++) {
                const float wgt = weight(ml[c].x, ml[c].y, M);
                L += ml[c].y * wgt;
                add(acc, v[c], wgt);
            }
        }
        store(r, q, acc, L);
    }
}

template <int D, int NT>
int32_t launch(tlc_ctx *ctx, const Params &p) {
    constexpr size_t smem = (size_t)kWarps * stages<D, NT>() * kKv8Block * D;
    int ctas = p.items * p.nsplit;
    if (p.nsplit == 1) {  // all places of every SM, as far as items go
        const int groups = kWarps / p.warps, least = (p.items + groups - 1) / groups;
        ctas = std::min(p.items, places(D, NT) * ctx->sm_count);
        if (ctas < least) ctas = least;
    }
    const dim3 grid((unsigned)ctas);
    static bool configured[64] = {};
    if (!configured[ctx->device & 63]) {
        TLC_CUDA(cudaFuncSetAttribute(attention8_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        TLC_CUDA(cudaFuncSetAttribute(attention8_kernel<D, NT>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                      cudaSharedmemCarveoutMaxShared));
        configured[ctx->device & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (p.cluster > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = (unsigned)p.cluster;
        attr[na].val.clusterDim.y = 1;
        attr[na++].val.clusterDim.z = 1;
    }
    if (ctx->use_pdl && ctx->pdl_small) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    const cudaError_t le = cudaLaunchKernelEx(&cfg, attention8_kernel<D, NT>, p);
    if (le != cudaSuccess) {
        cudaGetLastError();
        return tlc_fail(TLC_ERR_CUDA, "attention8 launch failed: %s", cudaGetErrorString(le));
    }
    TLC_CHECK_LAUNCH(ctx);
    return TLC_OK;
}

// Warps that share an item of `units` blocks -- 1, 2, 4, or four in each of 2, 4, 8 or a multiple of eight CTAs: the
// fewest microseconds of
//   blocks of a warp x (the larger of a block's latency and its share of the SM, 44 KB/us for its warps), and the merge
//   -- in shared memory, in a cluster, or of clusters --
// as often as the SM's warps have to be filled.  (Clusters of eight lie in one part of the chip: beyond two for nine SMs they
// leave some SMs with more CTAs than others.)
// 2048 queries, 32 heads of 128, fill them several times over: one warp an item takes 187 us, two (the rule's) 207, four 228,
// eight 369, 32 1204.
// One query, 32 heads on four of 64, behind 40000 positions takes 14.2 us with 64 warps to a KV head, 11.7 with 128, 10.9
// with 256, 16.2 with 576; behind 130000 32, 23, 19 and 23.
// Sixteen queries behind 1000 positions, 32 heads of 128: one warp 29.9 us, two 21.0, four 13.7, sixteen 11.3; 192
// queries: 49.5, 31.9, 35.9, 68.
double share_out(const tlc_ctx *ctx, int D, int nt, int units, Params &p) {
    const double latency = D == 64 ? nt == 1 ? 0.85 : 1.05 : nt == 1 ? 1.2 : 1.6, share = kKv8Block * D * 2 / 44e3;
    const int warps = kWarps * places(D, nt);  // of an SM
    double best = 1e30;
    for (int w = 1; w <= 4 * kKv8MaxCtas; w = w < 32 ? 2 * w : w + 32) {
        const int nsplit = w <= kWarps ? 1 : w / kWarps, cluster = nsplit < 8 ? nsplit : 8;
        if (w > 1 && w >= 2 * units) break;  // (fewer would do)
        if (nsplit > 8 && ((long long)p.items * nsplit > kKv8MaxCtas || p.items * 8 > kKv8Tickets)) break;
        const long long clusters = (long long)p.items * (nsplit / 8), layer = ctx->sm_count / 9 > 0 ? ctx->sm_count / 9 : 1;
        const long long per_sm = nsplit > 8 && clusters > 2 * layer ? kWarps * ((clusters + layer - 1) / layer)
                                                                    : ((long long)p.items * w + ctx->sm_count - 1) / ctx->sm_count;
        const long long rounds = (per_sm + warps - 1) / warps;
        const double at_once = (double)(per_sm < warps ? per_sm : warps), block = latency > at_once * share ? latency : at_once * share;
        const double merge = w == 1 ? 0.0 : w <= kWarps ? 0.7 : nsplit <= 8 ? 1.5 : 3.0 + 0.12 * (nsplit / 8);
        const double t = (double)rounds * ((units + w - 1) / w * block + merge);
        if (t < best) {
            best = t;
            p.warps = w < kWarps ? w : kWarps;
            p.nsplit = nsplit;
            p.cluster = cluster;
        }
    }
    return best;
}
// Microseconds that the tcgen05 form takes more than a launch of the other one: another launch and the longer start of its
// CTAs, the image of the blocks (three bytes moved a value), and its tiles of 128 rows x 64 keys, by the longest CTA or by
// what an SM gets through.  32 heads of 128: 192 queries 12.3 us here, 8.8 there, behind 1000 positions 31.6 and 22.7;
// 64 behind 1000 15.2 and 24.7.  2048 queries 207 and 48.
double tcgen05_us(const tlc_ctx *ctx, int D, int Hkv, int G, int I, int pos0) {
    const int rq = 128 / G, tiles = (I + rq - 1) / rq, units = (pos0 + I + kKv8Block - 1) / kKv8Block;
    const double image = (double)units * Hkv * kKv8Block * D * 6 / 5e6, longest = units * (D == 64 ? 0.45 : 0.55);
    const double all = (double)tiles * Hkv * (pos0 + 0.5 * I + kKv8Block) / kKv8Block / ctx->sm_count * (D == 64 ? 0.45 : 0.7);
    return 2.0 + image + (longest > all ? longest : all);
}

}  // namespace

extern "C" int32_t tlc_attention8(tlc_ctx *ctx, tlc_kvcache8 *cache, int32_t layer, const void *q_dev, void *out_dev,
                                  int32_t batch, int32_t n_queries, int32_t n_heads, int32_t sequence, int32_t q_pos0,
                                  const int32_t *positions_dev, int32_t max_keys, float scale) {
    if (int32_t rc = tlc_enter(ctx)) return rc;
    tlc_perf_scope perf(ctx, "attention8(batch=%d, queries=%d, heads=%d)", batch, n_queries, n_heads);
    TLC_REQUIRE(q_dev && out_dev, TLC_ERR_INVALID_OPERATION, "attention8: null pointer");
    TLC_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) == 0, TLC_ERR_INVALID_OPERATION,
                "attention8: queries and output must be 16-byte aligned");
    TLC_REQUIRE(batch >= 1, TLC_ERR_SHAPE_MISMATCH, "attention8: batch %d", batch);
    if (int32_t rc = kv8_check(ctx, cache, "attention8", layer, sequence, batch)) return rc;
    const int D = cache->head_dim, Hkv = cache->n_kv_heads;
    TLC_REQUIRE(n_heads >= 1 && n_heads % Hkv == 0, TLC_ERR_SHAPE_MISMATCH, "attention8: %d query heads over %d KV heads",
                n_heads, Hkv);
    TLC_REQUIRE(n_queries >= 1 && (!positions_dev || n_queries == 1), TLC_ERR_INVALID_OPERATION,
                "attention8: per-sequence positions need one query per sequence");
    TLC_REQUIRE(positions_dev || (q_pos0 >= 0 && q_pos0 <= cache->max_seq), TLC_ERR_INDEX,
                "Index out of bounds: index %d, size %d", q_pos0, cache->max_seq);
    const long long T = positions_dev ? max_keys : (long long)q_pos0 + n_queries;
    TLC_REQUIRE(T >= 1 && T <= cache->max_seq, TLC_ERR_INDEX, "Index out of bounds: index %lld, size %d", T, cache->max_seq);
    const int G = n_heads / Hkv;
    TLC_REQUIRE(batch <= 65535 && (long long)n_queries * G <= INT_MAX / 64, TLC_ERR_INVALID_DIMENSION,
                "attention8: %d sequences of %d queries", batch, n_queries);
    Params p{};
    p.q = static_cast<const __half *>(q_dev);
    p.out = static_cast<__half *>(out_dev);
    p.c = kv8_view(cache, layer, sequence);
    p.I = n_queries;
    p.H = n_heads;
    p.G = G;
    p.pos0 = q_pos0;
    p.positions = positions_dev;
    p.key_limit = (int)T;
    p.scale = scale;
    p.partial = cache->partial;
    p.tickets = cache->tickets;
    p.status = ctx->dev_status;
    const int nt = n_queries * G > 8 ? 2 : 1;
    p.row_tiles = (n_queries * G + 8 * nt - 1) / (8 * nt);
    const long long items = (long long)batch * Hkv * p.row_tiles;
    TLC_REQUIRE(items <= INT_MAX, TLC_ERR_INVALID_DIMENSION, "attention8: %d sequences of %d queries", batch, n_queries);
    p.items = (int)items;
    const double t = share_out(ctx, D, nt, (int)((T + kKv8Block - 1) / kKv8Block), p);
    if (n_queries > 1 && G <= 128 && (ctx->attn8_tc == 0 ? batch * tcgen05_us(ctx, D, Hkv, G, n_queries, q_pos0) < t : ctx->attn8_tc == 1)) {
        for (int b = 0; b < batch; b++) {  // through one image, a sequence at a time
            const size_t at = (size_t)b * n_queries * n_heads * D;
            if (int32_t rc = kv8_attention_tc(ctx, cache, layer, sequence + b, static_cast<const __half *>(q_dev) + at,
                                              static_cast<__half *>(out_dev) + at, n_queries, n_heads, q_pos0, scale))
                return rc;
        }
        return TLC_OK;
    }
    if (D == 64) return nt == 1 ? launch<64, 1>(ctx, p) : launch<64, 2>(ctx, p);
    return nt == 1 ? launch<128, 1>(ctx, p) : launch<128, 2>(ctx, p);
}

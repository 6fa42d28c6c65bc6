// The 8-bit KV cache (tlc_kv8.h): creation, append, read-back.
#include <cuda_fp16.h>

#include <new>

#include "tlc_kv8.h"

namespace {

constexpr int kThreads = 128;

// The orders of tlc_kv8.h take every value of a block to a place of its own.
template <int D>
constexpr bool places_are_distinct() {
    bool seen[4][kKv8Block * D] = {};
    for (int j = 0; j < kKv8Block; j++)
        for (int d = 0; d < D; d++) {
            const int at[4] = {kv8_k_code<D>(j, d), kv8_v_code<D>(j, d), kv8_k_open<D>(j, d), kv8_v_open<D>(j, d)};
            for (int i = 0; i < 4; i++) {
                if (at[i] < 0 || at[i] >= kKv8Block * D || seen[i][at[i]]) return false;
                seen[i][at[i]] = true;
            }
        }
    return true;
}
static_assert(places_are_distinct<64>(), "64 values a row");
static_assert(kv8_row(kv8_key(5)) == 5 && kv8_row(kv8_key(14)) == 14, "a row's key is in that row");

struct AppendParams {
    const __half *k, *v;   // [m][kv heads][D]
    Kv8View c;
    int m;                 // rows of one sequence, or sequences with a row each
    int pos;               // position of row 0 (positions == null)
    const int *positions;  // device int32[m]; negative: no row for this sequence
    tlc_dev_status *status;
};

__device__ __forceinline__ uint32_t u32(const __half2 &h) { return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); }
// What the cache holds is finite: NaN as zero, infinities as the largest f16.
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
    const __half2 x = h2(w & __heq2_mask(h2(w), h2(w)));
    return u32(__hmin2(__hmax2(x, h2(0xFBFFFBFFu)), h2(0x7BFF7BFFu)));
}
__device__ __forceinline__ uint4 finite8(uint4 v) { return make_uint4(finite2(v.x), finite2(v.y), finite2(v.z), finite2(v.w)); }

// Codes rint(127 x / a) of sixteen values as bytes code + 128; r = 127 / a.  x r in one fused multiply-add that rounds to
// whole numbers is off by less than 1e-5, so that only next to a border is the quotient itself needed.  (Correctly
// rounded it decides every border rightly: 127 x / a of two f16 is k + 1/2 exactly or at least 2^-20 of the power
// of two below it away, and f32 resolves 2^-24 of that.)
__device__ __forceinline__ uint4 encode16(const uint32_t (&x)[8], float a, float r) {
    constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: the sum's low byte is the code
    uint32_t out[4];
    float edge = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 lo = __half22float2(h2(x[2 * i])), hi = __half22float2(h2(x[2 * i + 1]));
        const float v[4] = {lo.x, lo.y, hi.x, hi.y};
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float w = fmaf(v[e], r, kWhole);
            edge = fmaxf(edge, fabsf(fmaf(v[e], r, kWhole - w)));
            y[e] = __float_as_uint(w);
        }
        out[i] = __byte_perm(__byte_perm(y[0], y[1], 0x0040), __byte_perm(y[2], y[3], 0x0040), 0x5410) ^ 0x80808080u;
    }
    if (edge > 0.4999f) {
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t pair = i == 0 ? x[e / 2] : i == 1 ? x[2 + e / 2] : i == 2 ? x[4 + e / 2] : x[6 + e / 2];
                const float v = e & 1 ? __high2float(h2(pair)) : __low2float(h2(pair));
                w |= (uint32_t)((int)rintf(__fdiv_rn(127.f * v, a)) + 128) << (8 * e);
            }
            if (i == 0) out[0] = w;
            else if (i == 1) out[1] = w;
            else if (i == 2) out[2] = w;
            else out[3] = w;
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}
// What sixteen codes stand for, in f16.
__device__ __forceinline__ void decode16(const uint4 &q, float s, uint32_t (&x)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int p = 0; p < 2; p++) {
            // 1024 + code + 128, minus 1152: exact
            const float2 c = __half22float2(__hsub2(h2(__byte_perm(w[i], 0x64646464u, p ? 0x4342 : 0x4140)), __float2half2_rn(1152.f)));
            x[2 * i + p] = u32(__floats2half2_rn(s * c.x, s * c.y));
        }
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void stsm4_trans(void *p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"((uint32_t)__cvta_generic_to_shared(p)), "r"(a),
                 "r"(b), "r"(c), "r"(d)
                 : "memory");
}
// Where a lane's row of the four 8 x 8 matrices lies that turn rows [key][32 values] into V's order and back: matrices
// {keys 4i, 4i+1}, {4i+2, 4i+3} of eight values of d, and of the next eight.
__device__ __forceinline__ int turn_key(int lane) { return 4 * ((lane & 7) >> 1) + (lane & 1) + 2 * ((lane >> 3) & 1); }
__device__ __forceinline__ int turn_d(int lane) { return 8 * (lane >> 4); }

// Rows of K or V (blockIdx.z) of one KV head (blockIdx.y).  A row for each sequence: blockIdx.x is the sequence.  Rows of
// one sequence: they fall into blocks first .. last, and CTA i takes block first + i, all of whose rows are new if i > 0.
// Where the first block has rows already and the last one stays open, CTA 0 takes that too, behind the first: both may
// live in the open block's place.  CTA 0 writes the length.
//
// A block that is sealed stays in registers: warp w holds its keys 16 w .. 16 w + 15 in the order in which the codes lie,
// so that old rows (16 bytes a lane) and codes (512 a warp) are read and written as they are.  K's order takes eight
// neighbouring values of a row, which is how new rows come too; V's takes four keys of a value, and new rows are turned
// by ldmatrix.  Rows of an open block go the same way, 16 keys a warp; fewer than four, or behind older ones, one by one.
// Bound by the rows' bytes and, for few of them, by the launch: 2048 rows of 32 heads of 128 take 15.4 us (3.3 TB/s; 14.0
// where the L2 holds the rows already), 300 of them 6.7, 60 3.2 (8.2 and 5.0 with the open block one by one behind the first;
// the launch alone is 3.1), and 2048 with their read-back 25.0 against 53 for a form that went through shared memory value
// by value.
template <int D>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendParams p) {
    constexpr int PITCH = D + 8, PIECES = D / 8, C = D / 32;
    __shared__ __align__(16) __half xs[kKv8Block * PITCH];
    __shared__ float warp_max[kThreads / 32];
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, hk = blockIdx.y, kv = blockIdx.z;
    const bool batched = p.positions != nullptr;
    const int seq = batched ? blockIdx.x : 0;
    const int pos = batched ? p.positions[seq] : p.pos, m = batched ? 1 : p.m;
    if (batched && pos < 0) return;
    const size_t head = (size_t)seq * p.c.n_kv_heads + hk;
    int *length = p.c.lengths + head * 2 + kv;
    // (CTAs of the same call that read the new length here decide the same: it is at least pos.)
    const int held = *length;
    if (pos > held || pos > p.c.max_seq - m) {  // a gap in front of the rows, or no room: skipped, and said so
        if (tid == 0 && atomicCAS(&p.status->code, 0, TLC_DEV_INDEX) == 0) p.status->where = 300 + seq;
        return;
    }
    const __half *src = (kv ? p.v : p.k) + ((size_t)(batched ? seq : 0) * p.c.n_kv_heads + hk) * D;
    const size_t row = (size_t)p.c.n_kv_heads * D;
    uint8_t *codes = p.c.codes + (head * p.c.n_blocks * 2 + kv) * (size_t)(kKv8Block * D);
    float *scales = p.c.scales + head * p.c.n_blocks * 2 + kv;
    __half *open = p.c.open + (head * 2 + kv) * (size_t)(kKv8Block * D);
    const int first = pos / kKv8Block, last = (pos + m - 1) / kKv8Block;

    // Rows 64 b + [j0, 64) are new, and fill the block.
    auto seal = [&](int b, int j0) {
        uint32_t x[C][8];  // K: rows g and g + 8, eight values each; V: keys 4t .. 4t + 3 of values g, 8 + g, 16 + g, 24 + g
        const bool old = 16 * warp < j0, sealed = b < held / kKv8Block;
        uint8_t *to = codes + (size_t)b * (2 * kKv8Block * D) + (warp * C * 32 + lane) * 16;
        if (old) {
            if (sealed) {  // a rewind: what the codes stand for
                const float s = scales[2 * b];
#pragma unroll
                for (int c = 0; c < C; c++) decode16(*reinterpret_cast<const uint4 *>(to + c * 512), s, x[c]);
            } else {
                const uint4 *from = reinterpret_cast<const uint4 *>(open) + warp * C * 64 + lane;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const uint4 u = from[c * 64], v = from[c * 64 + 32];
                    if (kv == 0) {
                        x[c][0] = u.x, x[c][1] = u.y, x[c][2] = v.x, x[c][3] = v.y;
                        x[c][4] = u.z, x[c][5] = u.w, x[c][6] = v.z, x[c][7] = v.w;
                    } else {
                        x[c][0] = u.x, x[c][1] = u.y, x[c][2] = u.z, x[c][3] = u.w;
                        x[c][4] = v.x, x[c][5] = v.y, x[c][6] = v.z, x[c][7] = v.w;
                    }
                }
            }
        }
        {
            const int key[2] = {16 * warp + kv8_key(g), 16 * warp + kv8_key(g + 8)};
            uint4 v[C][2];
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (key[h] >= j0) v[c][h] = *reinterpret_cast<const uint4 *>(src + (size_t)(b * kKv8Block + key[h] - pos) * row + c * 32 + t * 8);
            if (kv == 0) {
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (key[h] >= j0) {
                            const uint4 f = finite8(v[c][h]);
                            x[c][4 * h] = f.x, x[c][4 * h + 1] = f.y, x[c][4 * h + 2] = f.z, x[c][4 * h + 3] = f.w;
                        }
            } else {
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (key[h] >= j0) *reinterpret_cast<uint4 *>(xs + key[h] * PITCH + c * 32 + t * 8) = finite8(v[c][h]);
                __syncwarp();
                // which of keys 4t .. 4t + 3 are new
                const int n = 16 * warp + 4 * t;
                const uint32_t m0 = (n >= j0 ? 0xFFFFu : 0u) | (n + 1 >= j0 ? 0xFFFF0000u : 0u);
                const uint32_t m1 = (n + 2 >= j0 ? 0xFFFFu : 0u) | (n + 3 >= j0 ? 0xFFFF0000u : 0u);
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        uint32_t r[4];
                        ldsm4_trans(r, xs + (16 * warp + turn_key(lane)) * PITCH + c * 32 + s * 16 + turn_d(lane));
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t mask = e & 1 ? m1 : m0;
                            x[c][4 * s + e] = old ? (r[e] & mask) | (x[c][4 * s + e] & ~mask) : r[e];
                        }
                    }
            }
        }
        __half2 mx = __float2half2_rn(0.f);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) mx = __hmax2(mx, __habs2(h2(x[c][e])));
        float a = fmaxf(__low2float(mx), __high2float(mx));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (lane == 0) warp_max[warp] = a;
        __syncthreads();
        a = fmaxf(fmaxf(warp_max[0], warp_max[1]), fmaxf(warp_max[2], warp_max[3]));
        const float r = a > 0.f ? __fdiv_rn(127.f, a) : 0.f;
        if (tid == 0) scales[2 * b] = __fdiv_rn(a, 127.f);
#pragma unroll
        for (int c = 0; c < C; c++) *reinterpret_cast<uint4 *>(to + c * 512) = encode16(x[c], a, r);
    };
    // Rows 64 b + [j0, j1) are new, and the block stays open.
    auto keep = [&](int b, int j0, int j1) {
        if (j0 > 0 && b < held / kKv8Block) {  // a rewind: the rows in front of the new ones, as the codes stand for
            const uint8_t *old = codes + (size_t)b * (2 * kKv8Block * D);
            const float s = scales[2 * b];
            for (int i = tid; i < j0 * D; i += kThreads) {
                const int j = i / D, d = i % D;
                open[kv ? kv8_v_open<D>(j, d) : kv8_k_open<D>(j, d)] =
                    __float2half_rn(s * (float)((int)old[kv ? kv8_v_code<D>(j, d) : kv8_k_code<D>(j, d)] - 128));
            }
        }
        // this warp's 16 keys: by registers where all of them are new and several come (zeros behind them), else one by one
        const int n0 = j0 > 16 * warp ? j0 : 16 * warp, n1 = j1 < 16 * warp + 16 ? j1 : 16 * warp + 16;
        if (n0 == 16 * warp && n1 - n0 >= 4) {
            const int key[2] = {n0 + kv8_key(g), n0 + kv8_key(g + 8)};
            uint4 *to = reinterpret_cast<uint4 *>(open) + warp * C * 64 + lane;
            uint4 f[C][2];
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    f[c][h] = make_uint4(0, 0, 0, 0);
                    if (key[h] < n1) f[c][h] = *reinterpret_cast<const uint4 *>(src + (size_t)(b * kKv8Block + key[h] - pos) * row + c * 32 + t * 8);
                }
#pragma unroll
            for (int c = 0; c < C; c++) {
                f[c][0] = finite8(f[c][0]), f[c][1] = finite8(f[c][1]);
                if (kv == 0) {
                    to[c * 64] = make_uint4(f[c][0].x, f[c][0].y, f[c][1].x, f[c][1].y);
                    to[c * 64 + 32] = make_uint4(f[c][0].z, f[c][0].w, f[c][1].z, f[c][1].w);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) *reinterpret_cast<uint4 *>(xs + key[h] * PITCH + c * 32 + t * 8) = f[c][h];
                }
            }
            if (kv == 0) return;
            __syncwarp();
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    uint32_t r[4];
                    ldsm4_trans(r, xs + (16 * warp + turn_key(lane)) * PITCH + c * 32 + s * 16 + turn_d(lane));
                    to[c * 64 + s * 32] = make_uint4(r[0], r[1], r[2], r[3]);
                }
            return;
        }
        for (int i = n0 * PIECES + lane; i < n1 * PIECES; i += 32) {
            const int j = i / PIECES, d = i % PIECES * 8;
            const uint4 f = finite8(*reinterpret_cast<const uint4 *>(src + (size_t)(b * kKv8Block + j - pos) * row + d));
            if (kv == 0) {
                *reinterpret_cast<uint2 *>(open + kv8_k_open<D>(j, d)) = make_uint2(f.x, f.y);
                *reinterpret_cast<uint2 *>(open + kv8_k_open<D>(j, d + 4)) = make_uint2(f.z, f.w);
            } else {
                const __half *h = reinterpret_cast<const __half *>(&f);
#pragma unroll
                for (int e = 0; e < 8; e++) open[kv8_v_open<D>(j, d + e)] = h[e];
            }
        }
    };
    const int j0 = pos - first * kKv8Block, j1 = pos + m - last * kKv8Block;
    const int b = first + (batched ? 0 : blockIdx.x);
    if (b > first && (b < last || j1 == kKv8Block)) {
        seal(b, 0);
        return;
    }
    if (b == first) {
        if (last > first || j1 == kKv8Block) seal(first, j0);
        else __syncthreads();  // (every warp has read the length)
        if (tid == 0) *length = pos + m;
        if (j1 == kKv8Block || (last > first && gridDim.x > last - first)) return;  // nothing is open, or another CTA's
        if (last > first) __syncthreads();                                          // (the open block has been read)
    }
    keep(last, last > first ? 0 : j0, j1);
}

// Block b of a head (K or V), whose cache holds `have` of its rows: the codes (times s) or the open rows of this warp's
// keys, in the order of the codes.
template <int D>
__device__ __forceinline__ void load_block(const Kv8View &c8, size_t head, int b, int kv, int have, float s, uint32_t (&x)[D / 32][8]) {
    constexpr int C = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (have >= kKv8Block) {
        const uint4 *from = reinterpret_cast<const uint4 *>(c8.codes + ((head * c8.n_blocks + b) * 2 + kv) * (size_t)(kKv8Block * D)) +
                            warp * C * 32 + lane;
        uint4 q[C];
#pragma unroll
        for (int c = 0; c < C; c++) q[c] = from[c * 32];
#pragma unroll
        for (int c = 0; c < C; c++) decode16(q[c], s, x[c]);
        return;
    }
    const uint4 *from = reinterpret_cast<const uint4 *>(c8.open + (head * 2 + kv) * (size_t)(kKv8Block * D)) + warp * C * 64 + lane;
#pragma unroll
    for (int c = 0; c < C; c++) {
        uint4 u = make_uint4(0, 0, 0, 0), v = u;
        if (have > 16 * warp) {
            u = from[c * 64];
            v = from[c * 64 + 32];
        }
        if (kv == 0) {
            x[c][0] = u.x, x[c][1] = u.y, x[c][2] = v.x, x[c][3] = v.y;
            x[c][4] = u.z, x[c][5] = u.w, x[c][6] = v.z, x[c][7] = v.w;
        } else {
            x[c][0] = u.x, x[c][1] = u.y, x[c][2] = u.z, x[c][3] = u.w;
            x[c][4] = v.x, x[c][5] = v.y, x[c][6] = v.z, x[c][7] = v.w;
        }
    }
}

// What the cache holds of rows [first, first + n) of the view's sequences, in f16; zeros past a sequence's rows.
// A CTA for a block of one head, K or V; warp w has its keys 16 w .. 16 w + 15, as above.  Bound by the bytes written.
struct RowsParams {
    Kv8View c;
    __half *k, *v;  // [sequence][n][kv heads][D]
    int first, n;
};
template <int D>
__global__ void __launch_bounds__(kThreads) kv8_rows_kernel(const RowsParams p) {
    constexpr int PITCH = D + 8, C = D / 32;
    __shared__ __align__(16) __half xs[kKv8Block * PITCH];
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int per = (p.n + p.first % kKv8Block + kKv8Block - 1) / kKv8Block;
    const int seq = blockIdx.x / per, b = p.first / kKv8Block + blockIdx.x % per, hk = blockIdx.y, kv = blockIdx.z;
    const size_t head = (size_t)seq * p.c.n_kv_heads + hk;
    const int have = p.c.lengths[head * 2 + kv] - b * kKv8Block;  // rows of this block
    __half *out = (kv ? p.v : p.k) + ((size_t)seq * p.n * p.c.n_kv_heads + hk) * D + t * 8;
    const size_t row = (size_t)p.c.n_kv_heads * D;
    uint32_t x[C][8];
    load_block<D>(p.c, head, b, kv, have, have >= kKv8Block ? p.c.scales[(head * p.c.n_blocks + b) * 2 + kv] : 0.f, x);
    if (kv == 1) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int s = 0; s < 2; s++)
                stsm4_trans(xs + (16 * warp + turn_key(lane)) * PITCH + c * 32 + s * 16 + turn_d(lane), x[c][4 * s], x[c][4 * s + 1],
                            x[c][4 * s + 2], x[c][4 * s + 3]);
        __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int j = 16 * warp + kv8_key(g + 8 * h), at = b * kKv8Block + j - p.first;
        if (at < 0 || at >= p.n) continue;
#pragma unroll
        for (int c = 0; c < C; c++) {
            uint4 v = make_uint4(x[c][4 * h], x[c][4 * h + 1], x[c][4 * h + 2], x[c][4 * h + 3]);
            if (kv == 1) v = *reinterpret_cast<const uint4 *>(xs + j * PITCH + c * 32 + t * 8);
            if (j >= have) v = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(out + (size_t)at * row + c * 32) = v;
        }
    }
}

// The blocks of one sequence as f16 rows [K, V][kv head][position][D] for the tensor-memory attention: codes as they are,
// the open block's values.  factors[kv head][block]: what K's count in scores, log2 of what V's count, and one over that.
struct WidenParams {
    Kv8View c;
    __half *wide;
    float4 *factors;
    int rows;  // of a head in `wide`
};
template <int D>
__global__ void __launch_bounds__(kThreads) kv8_widen_kernel(const WidenParams p) {
    constexpr int PITCH = D + 8, C = D / 32;
    __shared__ __align__(16) __half xs[kKv8Block * PITCH];
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int b = blockIdx.x, hk = blockIdx.y, kv = blockIdx.z, have = p.c.lengths[hk * 2 + kv] - b * kKv8Block;
    uint32_t x[C][8];
    load_block<D>(p.c, hk, b, kv, have, 1.f, x);
    const float s = have >= kKv8Block ? p.c.scales[((size_t)hk * p.c.n_blocks + b) * 2 + kv] : 1.f;
    if (have < kKv8Block) {  // rows it does not have: zeros
        const int n = 16 * warp + (kv ? 4 * t : 0), jk[2] = {n + kv8_key(g), n + kv8_key(g + 8)};
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int j = n + 2 * (e & 1);
                if (kv == 0) x[c][e] = jk[e >> 2] < have ? x[c][e] : 0u;
                else x[c][e] &= (j < have ? 0xFFFFu : 0u) | (j + 1 < have ? 0xFFFF0000u : 0u);
            }
    }
    if (tid == 0) {
        float *to = reinterpret_cast<float *>(p.factors + (size_t)hk * p.c.n_blocks + b);
        // A block of zeros counts for nothing in P.V, so what it is given must not lift the running maximum, which log2 of
        // the factor is part of, over other blocks: 2^-31, below the smallest scale there is (2^-24 / 127).
        const float w = s > 0.f ? s : 0x1p-31f;
        if (kv == 0) to[0] = s;
        else to[1] = log2f(w), to[2] = 1.f / w;
    }
    if (kv == 1) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int q = 0; q < 2; q++)
                stsm4_trans(xs + (16 * warp + turn_key(lane)) * PITCH + c * 32 + q * 16 + turn_d(lane), x[c][4 * q], x[c][4 * q + 1],
                            x[c][4 * q + 2], x[c][4 * q + 3]);
        __syncwarp();
    }
    __half *out = p.wide + (((size_t)kv * p.c.n_kv_heads + hk) * p.rows + b * kKv8Block) * D + t * 8;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int j = 16 * warp + kv8_key(g + 8 * h);
#pragma unroll
        for (int c = 0; c < C; c++)
            *reinterpret_cast<uint4 *>(out + j * D + c * 32) =
                kv ? *reinterpret_cast<const uint4 *>(xs + j * PITCH + c * 32 + t * 8)
                   : make_uint4(x[c][4 * h], x[c][4 * h + 1], x[c][4 * h + 2], x[c][4 * h + 3]);
    }
}

int32_t launched(tlc_ctx *ctx, const char *what, cudaError_t e) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        return tlc_fail(TLC_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    }
    TLC_CHECK_LAUNCH(ctx);
    return TLC_OK;
}

}  // namespace

int32_t kv8_check(tlc_ctx *ctx, const tlc_kvcache8 *cache, const char *what, int layer, int first, int sequences) {
    TLC_REQUIRE(cache, TLC_ERR_INVALID_OPERATION, "%s: null pointer", what);
    // (its workspace serves one stream)
    TLC_REQUIRE(cache->ctx == ctx, TLC_ERR_DEVICE, "%s: the cache belongs to another context", what);
    TLC_REQUIRE(layer >= 0 && layer < cache->n_layers, TLC_ERR_INDEX, "Index out of bounds: index %d, size %d", layer,
                cache->n_layers);
    TLC_REQUIRE(first >= 0 && sequences >= 0 && sequences <= cache->max_batch - first, TLC_ERR_SHAPE_MISMATCH,
                "%s: sequences %d .. %lld exceed the cache's %d", what, first, (long long)first + sequences - 1, cache->max_batch);
    return TLC_OK;
}

int32_t kv8_widen(tlc_ctx *ctx, tlc_kvcache8 *cache, int layer, int sequence, int blocks) {
    WidenParams p{};
    p.c = kv8_view(cache, layer, sequence);
    p.wide = cache->wide;
    p.factors = cache->factors;
    p.rows = cache->n_blocks * kKv8Block;
    const dim3 grid(blocks, cache->n_kv_heads, 2);
    return launched(ctx, "kvcache8 image",
                    cache->head_dim == 64 ? tlc_launch_pdl(ctx, kv8_widen_kernel<64>, grid, dim3(kThreads), 0, p)
                                          : tlc_launch_pdl(ctx, kv8_widen_kernel<128>, grid, dim3(kThreads), 0, p));
}

extern "C" int32_t tlc_kvcache8_create(tlc_ctx *ctx, int32_t n_layers, int32_t max_batch, int32_t max_seq,
                                       int32_t n_kv_heads, int32_t head_dim, tlc_kvcache8 **out) {
    if (int32_t rc = tlc_enter(ctx)) return rc;
    TLC_REQUIRE(out, TLC_ERR_INVALID_OPERATION, "kvcache8_create: null out pointer");
    *out = nullptr;
    TLC_REQUIRE(n_layers > 0 && max_batch > 0 && max_seq > 0 && n_kv_heads > 0 && max_seq <= INT_MAX - kKv8Block &&
                    n_kv_heads <= 65535,
                TLC_ERR_INVALID_DIMENSION, "kvcache8_create: bad shape");
    TLC_REQUIRE(head_dim == 64 || head_dim == 128, TLC_ERR_INVALID_OPERATION,
                "kvcache8_create: head_dim %d unsupported (64, 128)", head_dim);
    const size_t blocks = (size_t)(max_seq + kKv8Block - 1) / kKv8Block, block = (size_t)kKv8Block * head_dim;
    size_t heads = 0, codes = 0;  // all layers
    TLC_REQUIRE(!__builtin_mul_overflow((size_t)n_layers * max_batch, (size_t)n_kv_heads, &heads) &&
                    !__builtin_mul_overflow(heads, blocks * 2 * block, &codes) && codes < (size_t)1 << 62,
                TLC_ERR_INVALID_DIMENSION, "kvcache8_create: bad shape");
    tlc_kvcache8 *c = new (std::nothrow) tlc_kvcache8();
    TLC_REQUIRE(c, TLC_ERR_ALLOCATION, "kvcache8_create: out of host memory");
    c->ctx = ctx;
    c->n_layers = n_layers;
    c->max_batch = max_batch;
    c->max_seq = max_seq;
    c->n_kv_heads = n_kv_heads;
    c->head_dim = head_dim;
    c->n_blocks = (int)blocks;
    const size_t blocks_of_one = (size_t)n_kv_heads * blocks, wide = blocks_of_one * 2 * block * sizeof(__half);  // a sequence and layer
    const size_t open = heads * 2 * block * sizeof(__half), lengths = heads * 2 * sizeof(int), tickets = kKv8Tickets * sizeof(int);
    cudaError_t e = cudaMalloc(&c->codes, codes);
    if (e == cudaSuccess) e = cudaMalloc(&c->scales, heads * blocks * 2 * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&c->open, open);
    if (e == cudaSuccess) e = cudaMalloc(&c->lengths, lengths);
    if (e == cudaSuccess) e = cudaMalloc(&c->tickets, tickets);
    if (e == cudaSuccess) e = cudaMalloc(&c->partial, (size_t)kKv8MaxParts * kKv8MaxRows * (head_dim + 2) * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&c->wide, wide);
    if (e == cudaSuccess) e = cudaMalloc(&c->factors, blocks_of_one * sizeof(float4));
    // Codes and scales are read only after they have been written; rows of an open block past its length are
    // multiplied by zero, and have to be finite for that.
    if (e == cudaSuccess) e = cudaMemsetAsync(c->open, 0, open, ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->lengths, 0, lengths, ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->tickets, 0, tickets, ctx->stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        tlc_kvcache8_destroy(c);
        return tlc_fail(TLC_ERR_ALLOCATION, "8-bit KV cache allocation of %zu bytes failed: %s", codes + open + wide, cudaGetErrorString(e));
    }
    *out = c;
    return TLC_OK;
}

extern "C" int32_t tlc_kvcache8_destroy(tlc_kvcache8 *cache) {
    if (!cache) return TLC_OK;
    cudaSetDevice(cache->ctx->device);
    cudaFree(cache->codes);
    cudaFree(cache->scales);
    cudaFree(cache->open);
    cudaFree(cache->lengths);
    cudaFree(cache->tickets);
    cudaFree(cache->partial);
    cudaFree(cache->wide);
    cudaFree(cache->factors);
    delete cache;
    return TLC_OK;
}

extern "C" int32_t tlc_kvcache8_append(tlc_ctx *ctx, tlc_kvcache8 *cache, int32_t layer, const void *k_dev,
                                       const void *v_dev, int32_t m, int32_t sequence, int32_t pos_offset,
                                       const int32_t *positions_dev) {
    if (int32_t rc = tlc_enter(ctx)) return rc;
    tlc_perf_scope perf(ctx, "kvcache8_append(rows=%d)", m);
    TLC_REQUIRE(k_dev && v_dev, TLC_ERR_INVALID_OPERATION, "kvcache8_append: null pointer");
    TLC_REQUIRE((((uintptr_t)k_dev | (uintptr_t)v_dev) & 15) == 0, TLC_ERR_INVALID_OPERATION,
                "kvcache8_append: rows must be 16-byte aligned");
    TLC_REQUIRE(m >= 0, TLC_ERR_INVALID_DIMENSION, "kvcache8_append: %d rows", m);
    const bool batched = positions_dev != nullptr;
    if (int32_t rc = kv8_check(ctx, cache, "kvcache8_append", layer, sequence, batched ? m : 1)) return rc;
    if (!batched)
        TLC_REQUIRE(pos_offset >= 0 && pos_offset <= cache->max_seq && m <= cache->max_seq - pos_offset, TLC_ERR_INDEX,
                    "Index out of bounds: index %lld, size %d", (long long)pos_offset + m, cache->max_seq);
    if (m == 0) return TLC_OK;
    AppendParams p{};
    p.k = static_cast<const __half *>(k_dev);
    p.v = static_cast<const __half *>(v_dev);
    p.c = kv8_view(cache, layer, sequence);
    p.m = m;
    p.pos = pos_offset;
    p.positions = positions_dev;
    p.status = ctx->dev_status;
    const int blocks = (pos_offset + m - 1) / kKv8Block - pos_offset / kKv8Block + 1;  // (a row for each sequence: not used)
    const int both = blocks > 1 && pos_offset % kKv8Block > 0 && (pos_offset + m) % kKv8Block > 0;  // first and last, one CTA
    const dim3 grid(batched ? m : blocks - both, cache->n_kv_heads, 2);
    return launched(ctx, "kvcache8_append",
                    cache->head_dim == 64 ? tlc_launch_pdl(ctx, kv8_append_kernel<64>, grid, dim3(kThreads), 0, p)
                                          : tlc_launch_pdl(ctx, kv8_append_kernel<128>, grid, dim3(kThreads), 0, p));
}

extern "C" int32_t tlc_kvcache8_rows(tlc_ctx *ctx, tlc_kvcache8 *cache, int32_t layer, int32_t sequence,
                                     int32_t n_sequences, int32_t first, int32_t n, void *k_out_dev, void *v_out_dev) {
    if (int32_t rc = tlc_enter(ctx)) return rc;
    tlc_perf_scope perf(ctx, "kvcache8_rows(sequences=%d, rows=%d)", n_sequences, n);
    TLC_REQUIRE(k_out_dev && v_out_dev, TLC_ERR_INVALID_OPERATION, "kvcache8_rows: null pointer");
    TLC_REQUIRE((((uintptr_t)k_out_dev | (uintptr_t)v_out_dev) & 15) == 0, TLC_ERR_INVALID_OPERATION,
                "kvcache8_rows: rows must be 16-byte aligned");
    if (int32_t rc = kv8_check(ctx, cache, "kvcache8_rows", layer, sequence, n_sequences)) return rc;
    TLC_REQUIRE(first >= 0 && n >= 0 && first <= cache->max_seq && n <= cache->max_seq - first, TLC_ERR_INDEX,
                "Index out of bounds: index %lld, size %d", (long long)first + n, cache->max_seq);
    if (n == 0 || n_sequences == 0) return TLC_OK;
    RowsParams p{};
    p.c = kv8_view(cache, layer, sequence);
    p.k = static_cast<__half *>(k_out_dev);
    p.v = static_cast<__half *>(v_out_dev);
    p.first = first;
    p.n = n;
    const size_t ctas = (size_t)n_sequences * ((n + first % kKv8Block + kKv8Block - 1) / kKv8Block);
    TLC_REQUIRE(ctas <= INT_MAX, TLC_ERR_INVALID_DIMENSION, "kvcache8_rows: %d rows of %d sequences", n, n_sequences);
    const dim3 grid((unsigned)ctas, cache->n_kv_heads, 2);
    return launched(ctx, "kvcache8_rows",
                    cache->head_dim == 64 ? tlc_launch_pdl(ctx, kv8_rows_kernel<64>, grid, dim3(kThreads), 0, p)
                                          : tlc_launch_pdl(ctx, kv8_rows_kernel<128>, grid, dim3(kThreads), 0, p));
}

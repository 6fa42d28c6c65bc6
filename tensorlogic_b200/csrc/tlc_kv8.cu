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

// What the cache holds is finite: NaN as zero, infinities as the largest f16.
__device__ __forceinline__ __half finite(__half x) {
    const unsigned short b = __half_as_ushort(x);
    if ((b & 0x7C00) != 0x7C00) return x;
    return __ushort_as_half((b & 0x03FF) ? (unsigned short)0 : (unsigned short)((b & 0x8000) | 0x7BFF));
}
// rint(127 x / a), r = 127 / a: the product is off by less than 1e-4, so that only next to a border is the quotient
// itself needed.  (Correctly rounded it decides every border rightly: 127 x / a of two f16 is k + 1/2 exactly or at
// least 2^-20 of the power of two below it away, and f32 resolves 2^-24 of that.)
__device__ __forceinline__ int code_of(float x, float a, float r) {
    const float t = x * r;
    float k = rintf(t);
    if (fabsf(fabsf(t - k) - 0.5f) < 1e-4f) k = rintf(__fdiv_rn(127.f * x, a));
    return (int)k;
}

// Rows of K or V (blockIdx.z) of one KV head (blockIdx.y).  A row for each sequence: blockIdx.x is the sequence.  Rows of
// one sequence: they fall into blocks first .. last; CTA 0 takes the first and the last one, which may both live in the
// open block's place, and then the length; CTA i > 0 takes block first + i, all of whose rows are new.
// Bound by the rows' bytes and, for few of them, by the launch.
template <int D>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendParams p) {
    constexpr int PITCH = D + 8, PIECES = D / 8, PER = kKv8Block * PIECES / kThreads;
    __shared__ __align__(16) __half xs[kKv8Block * PITCH];
    __shared__ float warp_max[kThreads / 32];
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, hk = blockIdx.y, kv = blockIdx.z;
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

    auto block = [&](int b) {
        const int j0 = max(pos - b * kKv8Block, 0), j1 = min(pos + m - b * kKv8Block, kKv8Block);  // new rows
        const bool seal = j1 == kKv8Block, sealed = b < held / kKv8Block;
        // rows in front of the new ones: of the open block, or (a rewind) what the codes stand for
        if (j0 > 0 && (seal || sealed)) {
            const uint8_t *old = codes + (size_t)b * (2 * kKv8Block * D);
            const float s = sealed ? scales[2 * b] : 0.f;
            for (int i = tid; i < j0 * D; i += kThreads) {
                const int j = i / D, d = i % D;
                xs[j * PITCH + d] = sealed ? __float2half_rn(s * (float)((int)old[kv ? kv8_v_code<D>(j, d) : kv8_k_code<D>(j, d)] - 128))
                                           : open[kv ? kv8_v_open<D>(j, d) : kv8_k_open<D>(j, d)];
            }
        }
        {
            uint4 v[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int j = (tid + i * kThreads) / PIECES, d = (tid + i * kThreads) % PIECES * 8;
                if (j >= j0 && j < j1) v[i] = *reinterpret_cast<const uint4 *>(src + (size_t)(b * kKv8Block + j - pos) * row + d);
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int j = (tid + i * kThreads) / PIECES, d = (tid + i * kThreads) % PIECES * 8;
                if (j < j0 || j >= j1) continue;
                __half *h = reinterpret_cast<__half *>(&v[i]);
#pragma unroll
                for (int e = 0; e < 8; e++) h[e] = finite(h[e]);
                *reinterpret_cast<uint4 *>(xs + j * PITCH + d) = v[i];
            }
        }
        __syncthreads();
        if (!seal) {
            for (int i = (sealed ? 0 : j0 * D) + tid; i < j1 * D; i += kThreads) {
                const int j = i / D, d = i % D;
                open[kv ? kv8_v_open<D>(j, d) : kv8_k_open<D>(j, d)] = xs[j * PITCH + d];
            }
            return;
        }
        __half2 mx = __float2half2_rn(0.f);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const uint4 v = *reinterpret_cast<const uint4 *>(xs + (tid + i * kThreads) / PIECES * PITCH + (tid + i * kThreads) % PIECES * 8);
            const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
            for (int e = 0; e < 4; e++) mx = __hmax2(mx, __habs2(h[e]));
        }
        float a = fmaxf(__low2float(mx), __high2float(mx));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        if ((tid & 31) == 0) warp_max[tid >> 5] = a;
        __syncthreads();
        a = fmaxf(fmaxf(warp_max[0], warp_max[1]), fmaxf(warp_max[2], warp_max[3]));
        const float r = a > 0.f ? __fdiv_rn(127.f, a) : 0.f;
        if (tid == 0) scales[2 * b] = __fdiv_rn(a, 127.f);
        uint8_t *to = codes + (size_t)b * (2 * kKv8Block * D);
        // 16 bytes of fragment order a thread
        for (int i = tid; i < kKv8Block * D / 16; i += kThreads) {
            const int g = (i & 31) >> 2, t = i & 3, c = (i >> 5) % (D / 32), kg = (i >> 5) / (D / 32);
            __align__(16) uint8_t q[16];
            if (kv == 0) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(xs + (kg * 16 + kv8_key(g + 8 * h)) * PITCH + c * 32 + t * 8);
                    const __half *x = reinterpret_cast<const __half *>(&v);
#pragma unroll
                    for (int e = 0; e < 8; e++) q[h * 8 + e] = (uint8_t)(code_of(__half2float(x[e]), a, r) + 128);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    q[e] = (uint8_t)(code_of(__half2float(xs[(kg * 16 + 4 * t + (e & 3)) * PITCH + c * 32 + (e >> 2) * 8 + g]), a, r) + 128);
            }
            *reinterpret_cast<uint4 *>(to + (size_t)i * 16) = *reinterpret_cast<const uint4 *>(q);
        }
    };
    if (blockIdx.x > 0 && !batched) {
        block(first + blockIdx.x);
        return;
    }
    block(first);
    if (last > first) {
        __syncthreads();
        block(last);
    }
    if (tid == 0) *length = pos + m;
}

// What the cache holds of rows [first, first + n) of the view's sequences, in f16; zeros past a sequence's rows.
// A CTA for a block of one head, K or V.
struct RowsParams {
    Kv8View c;
    __half *k, *v;  // [sequence][n][kv heads][D]
    int first, n;
};
template <int D>
__global__ void __launch_bounds__(kThreads) kv8_rows_kernel(const RowsParams p) {
    constexpr int PIECES = D / 8;
    __shared__ __align__(16) uint8_t cs[kKv8Block * D * 2];
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, per = (p.n + p.first % kKv8Block + kKv8Block - 1) / kKv8Block;
    const int seq = blockIdx.x / per, b = p.first / kKv8Block + blockIdx.x % per, hk = blockIdx.y, kv = blockIdx.z;
    const size_t head = (size_t)seq * p.c.n_kv_heads + hk;
    const int held = p.c.lengths[head * 2 + kv], have = held - b * kKv8Block;  // rows of this block
    const bool sealed = have >= kKv8Block;
    const float s = sealed ? p.c.scales[(head * p.c.n_blocks + b) * 2 + kv] : 0.f;
    if (have > 0) {
        const uint4 *from = sealed ? reinterpret_cast<const uint4 *>(p.c.codes + ((head * p.c.n_blocks + b) * 2 + kv) * (size_t)(kKv8Block * D))
                                   : reinterpret_cast<const uint4 *>(p.c.open + (head * 2 + kv) * (size_t)(kKv8Block * D));
        for (int i = tid; i < kKv8Block * D / (sealed ? 16 : 8); i += kThreads) reinterpret_cast<uint4 *>(cs)[i] = from[i];
    }
    __syncthreads();
    for (int i = tid; i < kKv8Block * PIECES; i += kThreads) {
        const int j = i / PIECES, d = i % PIECES * 8, at = b * kKv8Block + j - p.first;
        if (at < 0 || at >= p.n) continue;
        __align__(16) __half h[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            h[e] = j >= have ? __float2half_rn(0.f)
                   : sealed  ? __float2half_rn(s * (float)((int)cs[kv ? kv8_v_code<D>(j, d + e) : kv8_k_code<D>(j, d + e)] - 128))
                             : reinterpret_cast<const __half *>(cs)[kv ? kv8_v_open<D>(j, d + e) : kv8_k_open<D>(j, d + e)];
        *reinterpret_cast<uint4 *>((kv ? p.v : p.k) + (((size_t)seq * p.n + at) * p.c.n_kv_heads + hk) * D + d) = *reinterpret_cast<const uint4 *>(h);
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
    const size_t open = heads * 2 * block * sizeof(__half), lengths = heads * 2 * sizeof(int), tickets = kKv8Tickets * sizeof(int);
    cudaError_t e = cudaMalloc(&c->codes, codes);
    if (e == cudaSuccess) e = cudaMalloc(&c->scales, heads * blocks * 2 * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&c->open, open);
    if (e == cudaSuccess) e = cudaMalloc(&c->lengths, lengths);
    if (e == cudaSuccess) e = cudaMalloc(&c->tickets, tickets);
    if (e == cudaSuccess) e = cudaMalloc(&c->partial, (size_t)kKv8MaxCtas * kKv8MaxRows * (head_dim + 2) * sizeof(float));
    // Codes and scales are read only after they have been written; rows of an open block past its length are
    // multiplied by zero, and have to be finite for that.
    if (e == cudaSuccess) e = cudaMemsetAsync(c->open, 0, open, ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->lengths, 0, lengths, ctx->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->tickets, 0, tickets, ctx->stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        tlc_kvcache8_destroy(c);
        return tlc_fail(TLC_ERR_ALLOCATION, "8-bit KV cache allocation of %zu bytes failed: %s", codes + open, cudaGetErrorString(e));
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
    const int blocks = (pos_offset + m - 1) / kKv8Block - pos_offset / kKv8Block + 1;  // CTA 0 takes two
    const dim3 grid(batched ? m : blocks > 1 ? blocks - 1 : 1, cache->n_kv_heads, 2);
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

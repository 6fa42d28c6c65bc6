// The 8-bit KV cache: what its append, its read-back and the attention over it share.
//
// A block is 64 consecutive positions of one KV head of one sequence and layer.  A full ("sealed") block is held as
// 8-bit codes q = rint(127 x / a), a = max |x| over the block's 64 * D values, and one f32 scale a / 127, K and V apart.
// The rows of the block that is still filling (the "open" block) are kept in f16 as they came.  So a value is
// rounded once, and what the cache holds does not depend on how many rows came with each call.
//
// Both products of the attention run on mma.sync m16n8k16 with the keys (K) and the head's values (V) on the 16-row side
// and the queries on the 8-column side (a group of up to eight query heads fills it).  Codes lie in HBM in the order in
// which a warp's lanes take them as operand fragments, 16 bytes a lane (512 a warp) in one load, as unsigned bytes
// q + 128: such a byte in the low mantissa bits of a binary16 is the subnormal (q + 128) * 2^-24, so that one PRMT makes
// two operands; the 128 goes into the accumulator's start value.
//
// Within an MMA the order of the summed index is free as long as both operands use the same one.  For Q.K^T lane t of a
// quad takes eight neighbouring values of d for two MMAs; for P.V it takes four neighbouring keys, which is why row r of
// a 16-key group holds key kv8_key(r).
#pragma once

#include <cuda_fp16.h>

#include "tlc_internal.h"

constexpr int kKv8Block = 64;     // positions per block
constexpr int kKv8MaxCtas = 640;  // CTAs of a launch that shares keys over several clusters of eight
constexpr int kKv8MaxParts = kKv8MaxCtas / 8;  // what they leave in the workspace: a part for each cluster
constexpr int kKv8MaxRows = 16;                // (query, head) rows of a part
constexpr int kKv8Tickets = 1024;

struct tlc_kvcache8 {
    tlc_ctx *ctx;
    int n_layers, max_batch, max_seq, n_kv_heads, head_dim;
    int n_blocks;     // blocks per head: max_seq / 64, rounded up
    uint8_t *codes;   // [layer][sequence][kv head][block][K, V][64 * D], fragment order
    float *scales;    // [layer][sequence][kv head][block][K, V]
    __half *open;     // [layer][sequence][kv head][K, V][64 * D], fragment order
    int *lengths;     // [layer][sequence][kv head][K, V]: rows held (a copy for each CTA that appends)
    float *partial;   // of several clusters: maximum and sum [kKv8MaxParts * kKv8MaxRows][2], then O [..][D]
    int *tickets;     // zero between launches
    // For long prompts: the blocks of one layer and sequence as f16 rows [K, V][kv head][position][D], and per block what
    // they count (kv8_widen).  Made with the cache, so that no prompt allocates, in a stream capture or out of it.
    __half *wide;
    float4 *factors;
    size_t heads() const { return (size_t)max_batch * n_kv_heads; }  // of a layer
};

// A layer's part of the cache as the kernels see it (sequence `first` and the ones after it).
struct Kv8View {
    uint8_t *codes;
    float *scales;
    __half *open;
    int *lengths;
    int n_blocks, n_kv_heads, max_seq;
};
inline Kv8View kv8_view(const tlc_kvcache8 *c, int layer, int first) {
    const size_t head = (size_t)layer * c->heads() + (size_t)first * c->n_kv_heads, block = (size_t)kKv8Block * c->head_dim;
    return {c->codes + head * c->n_blocks * 2 * block, c->scales + head * c->n_blocks * 2, c->open + head * 2 * block,
            c->lengths + head * 2, c->n_blocks, c->n_kv_heads, c->max_seq};
}
// Argument checks that every call over the cache makes: whose it is, the layer, the sequences.
int32_t kv8_check(tlc_ctx *ctx, const tlc_kvcache8 *cache, const char *what, int layer, int first, int sequences);

// Fills wide and factors with the first `blocks` blocks of a sequence.
int32_t kv8_widen(tlc_ctx *ctx, tlc_kvcache8 *cache, int layer, int sequence, int blocks);
// Attention of a prompt over that image on the 5th-generation tensor cores (tlc_attention8_tc.cu).
int32_t kv8_attention_tc(tlc_ctx *ctx, tlc_kvcache8 *cache, int layer, int sequence, const __half *q, __half *out, int I, int H,
                         int pos0, float scale);

#ifdef __CUDACC__
// Key (0..15) that row r of a 16-key group holds, and the row that holds key j.
__host__ __device__ constexpr int kv8_key(int r) { return 4 * ((r & 7) >> 1) + (r & 1) + 2 * (r >> 3); }
__host__ __device__ constexpr int kv8_row(int j) { return 2 * (j >> 2) + (j & 1) + 8 * ((j >> 1) & 1); }
// Index of (key j of the block, d) in a block's codes (bytes) ...
template <int D>
__host__ __device__ constexpr int kv8_k_code(int j, int d) {
    const int r = kv8_row(j & 15);
    return (((j >> 4) * (D / 32) + (d >> 5)) * 32 + (r & 7) * 4 + ((d & 31) >> 3)) * 16 + (r >> 3) * 8 + (d & 7);
}
template <int D>
__host__ __device__ constexpr int kv8_v_code(int j, int d) {
    return (((j >> 4) * (D / 32) + (d >> 5)) * 32 + (d & 7) * 4 + ((j & 15) >> 2)) * 16 + ((d >> 4) & 1) * 8 + ((d >> 3) & 1) * 4 + (j & 3);
}
// ... and in an open block (f16 values): the same lanes, one MMA's fragment in 16 bytes.
template <int D>
__host__ __device__ constexpr int kv8_k_open(int j, int d) {
    const int r = kv8_row(j & 15);
    return ((((j >> 4) * (D / 32) + (d >> 5)) * 2 + ((d >> 2) & 1)) * 32 + (r & 7) * 4 + ((d & 31) >> 3)) * 8 + (r >> 3) * 4 + (d & 3);
}
template <int D>
__host__ __device__ constexpr int kv8_v_open(int j, int d) {
    return ((((j >> 4) * (D / 32) + (d >> 5)) * 2 + ((d >> 4) & 1)) * 32 + (d & 7) * 4 + ((j & 15) >> 2)) * 8 + ((d >> 3) & 1) * 4 + (j & 3);
}
#endif

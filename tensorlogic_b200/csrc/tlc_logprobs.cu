// Log probabilities of given tokens, entropy and the likeliest alternatives of logit rows, in one pass.
//
//   log p(t) = x_t - ln sum e^x,   H = ln sum e^x - sum p x,   over the finite x of a row
//
// A row belongs to a cluster of 1 to 8 CTAs (any number), each with a slice of the vocabulary.  A thread streams 16-byte pieces and
// keeps a running s = sum 2^y, t = sum 2^y y with y = x log2(e) + c, one fused multiply-add, and c = -m log2(e) in f32
// for the largest x so far: whatever c is rounded to, log2 p(x) = y - log2 s, so that large logits lose nothing.
//
// Alternatives (logprob_top_kernel): the slice is taken in turns of at most 16384 logits, held in registers, 8 to 32 a
// thread, and looked at once more for them.  (value, earliest first) is one key per logit, so no two are equal.  The k-th
// largest of the best keys of 64 groups of eight threads is a bound that at least k logits reach, and none but those of
// at most k groups can: these few are collected and ranked by counting.
#include <cuda_fp16.h>

#include "tlc_internal.h"

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnroll = 4;  // 16-byte pieces of a thread in flight, twice
constexpr float kLow = -60000.f;  // 2^y of the lowest f16 is zero beside any value from here on
constexpr int kTopThreads = 512, kTopWarps = kTopThreads / 32, kGroups = 64;
constexpr int kTargetThread = 64;  // (the first threads have the row's first piece and the merging)
constexpr int kMaxTop = 32, kMaxCluster = 8;
// what k groups of threads with so many 16-byte pieces each hold
template <int PIECES> constexpr int list_size() { return kMaxTop * (kTopThreads / kGroups) * PIECES * 8; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int cluster_rank() {
    int r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ int cluster_id() {
    int i;
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(i));
    return i;
}

struct LogprobParams {
    const __half *logits;
    const int *targets;
    float *logprobs, *entropy, *top_logprobs;
    int *top_ids;
    int rows, vocab, top, cluster;
    int share;  // 16-byte pieces a CTA
    tlc_dev_status *status;
};
struct Sums {
    float c, s, t;  // c = +inf: no logits
};
// s and t as they are for another c (smaller or the same).
__device__ __forceinline__ void moved_to(Sums &a, float c) {
    if (a.c == c) return;
    const float d = fmaxf(c - a.c, -1e30f), w = exp2_of(d);
    a.t = w * (a.t + d * a.s);
    a.s *= w;
    a.c = c;
}

// Log probability of a logit, and what a row without alternatives returns.
__device__ __forceinline__ float logprob_of(float x, const Sums &run, float log2_s) { return (fmaf(x, kLog2e, run.c) - log2_s) * kLn2; }
struct Target {  // fetched behind the first loads: two trips to memory, one behind the other
    int id;
    float x;
};
__device__ __forceinline__ Target target_of(const LogprobParams &p, int row) {
    Target t = {-1, 0.f};
    if (p.logprobs) {
        t.id = p.targets[row];
        if (t.id >= 0 && t.id < p.vocab) t.x = __half2float(p.logits[(size_t)row * p.vocab + t.id]);
    }
    return t;
}
__device__ __forceinline__ void store_row(const LogprobParams &p, int row, const Target &t, const Sums &run) {
    const bool any = run.c < INFINITY;
    const float log2_s = any ? log2f(run.s) : 0.f;
    if (p.logprobs) {
        float lp = 0.f;
        if (t.id >= 0 && t.id < p.vocab) {
            lp = isfinite(t.x) ? logprob_of(t.x, run, log2_s) : -INFINITY;
        } else if (t.id != -1) {
            lp = __int_as_float(0x7FC00000);
            if (atomicCAS(&p.status->code, 0, TLC_DEV_INDEX) == 0) p.status->where = TLC_WHERE_TOKEN;
        }
        p.logprobs[row] = lp;
    }
    if (p.entropy) p.entropy[row] = any ? fmaxf((log2_s - run.t / run.s) * kLn2, 0.f) : 0.f;
}
// The sums of a warp's lanes, those of a CTA's warps.
__device__ __forceinline__ void warp_sums(Sums &run) {
    float c = run.c;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c = fminf(c, __shfl_xor_sync(0xffffffffu, c, o));
    moved_to(run, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        run.s += __shfl_xor_sync(0xffffffffu, run.s, o);
        run.t += __shfl_xor_sync(0xffffffffu, run.t, o);
    }
}
__device__ __forceinline__ void joined(Sums &run, Sums a) {
    const float c = fminf(run.c, a.c);
    moved_to(run, c);
    moved_to(a, c);
    run.s += a.s;
    run.t += a.t;
}

// A row in the 16-byte pieces of memory it lies in: the first and the last may reach into other rows and past the array.
struct Row {
    const __half *base, *lo, *hi;
    int ahead, vocab;  // values of the first piece in front of the row
    int pieces;
    // Its values of a piece; -inf for what is not finite or not the row's.
    __device__ __forceinline__ uint4 load(int at, int end) const {
        uint4 w = make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
        if (at >= end) return w;
        const __half *src = base + (size_t)at * 8;
        if (src >= lo && src + 8 <= hi) {
            w = *reinterpret_cast<const uint4 *>(src);
        } else {
            __half h[8];
#pragma unroll
            for (int e = 0; e < 8; e++) h[e] = src + e >= lo && src + e < hi ? src[e] : __ushort_as_half((unsigned short)0xFC00);
#pragma unroll
            for (int e = 0; e < 4; e++) reinterpret_cast<__half2 *>(&w)[e] = __halves2half2(h[2 * e], h[2 * e + 1]);
        }
        return w;
    }
    // A piece without what is not the row's: -inf in its place.
    __device__ __forceinline__ uint4 own(uint4 w, int at) const {
        if (at != 0 && at + 1 != pieces) return w;
        unsigned m[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const long long i = (long long)at * 8 + 2 * e - ahead;
            if (i < 0 || i >= vocab) m[e] = (m[e] & 0xFFFF0000u) | 0xFC00u;
            if (i + 1 < 0 || i + 1 >= vocab) m[e] = (m[e] & 0xFFFFu) | 0xFC000000u;
        }
        return make_uint4(m[0], m[1], m[2], m[3]);
    }
};
// The eight values of a piece, `none` for those that are not finite: x * -0 + x is NaN for them, x for the rest (+0 for
// -0), and the maximum passes over NaN and -inf.
__device__ __forceinline__ void clean(uint4 w, __half2 none, __half2 (&v)[4]) {
    const unsigned m[4] = {w.x, w.y, w.z, w.w};
    const __half2 neg_zero = __floats2half2_rn(-0.f, -0.f);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const __half2 h = *reinterpret_cast<const __half2 *>(&m[e]);
        v[e] = __hmax2(__hfma2(h, neg_zero, h), none);
    }
}

// Without alternatives.  512 x 32000 takes 9.2 us (3.6 TB/s out of the L2 and HBM, 54 % of the copy's rate): 33 MB of
// loads with 64 KB in flight an SM, and about 7 instructions a logit.
template <bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 4) logprob_kernel(const LogprobParams p) {
    __shared__ Sums sums[kMaxCluster];
    __shared__ float warp_c[kWarps], warp_s[kWarps], warp_t[kWarps];
    if (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CLUSTER ? cluster_rank() : 0, row = CLUSTER ? cluster_id() : blockIdx.x;
    const __half *x0 = p.logits + (size_t)row * p.vocab;
    Target target = {-1, 0.f};
    Row r;
    r.ahead = (int)(((uintptr_t)x0 & 15) >> 1);
    r.vocab = p.vocab;
    r.base = x0 - r.ahead;
    r.lo = p.logits;
    r.hi = p.logits + (size_t)p.rows * p.vocab;
    r.pieces = (int)(((unsigned)r.ahead + p.vocab + 7) / 8);
    const int first = rank * p.share, end = CLUSTER ? min(first + p.share, r.pieces) : r.pieces;

    // ---- one pass: the thread's largest value and its sums ----
    Sums run = {INFINITY, 0.f, 0.f};
    float most = -INFINITY;
    {
        // 1024 pieces a turn.  Turns within the row need no look at its ends.
        constexpr int kTurn = kUnroll * kThreads;
        uint4 w[kUnroll];
        auto inside = [&](int turn) { return turn > 0 && turn + kTurn < r.pieces && turn + kTurn <= end; };
        auto load = [&](int turn) {
            if (inside(turn)) {
#pragma unroll
                for (int i = 0; i < kUnroll; i++) w[i] = *reinterpret_cast<const uint4 *>(r.base + (size_t)(turn + tid + i * kThreads) * 8);
            } else {
#pragma unroll
                for (int i = 0; i < kUnroll; i++) w[i] = r.load(turn + tid + i * kThreads, end);
            }
        };
        load(first);
        if (tid == 0 && rank == 0) target = target_of(p, row);
        for (int turn = first; turn < end; turn += kTurn) {
            if (!inside(turn)) {
#pragma unroll
                for (int i = 0; i < kUnroll; i++) w[i] = r.own(w[i], turn + tid + i * kThreads);
            }
            // What is not finite becomes the lowest f16, which counts for nothing beside a larger value; a turn that
            // has none (below, the rare case) is looked at value by value.
            __half2 v[kUnroll * 4];
#pragma unroll
            for (int i = 0; i < kUnroll; i++) clean(w[i], __float2half2_rn(-65504.f), *reinterpret_cast<__half2(*)[4]>(&v[4 * i]));
            if (turn + kTurn < end) load(turn + kTurn);
            __half2 mx[2] = {v[0], v[1]};
#pragma unroll
            for (int e = 2; e < kUnroll * 4; e++) mx[e & 1] = __hmax2(mx[e & 1], v[e]);
            mx[0] = __hmax2(mx[0], mx[1]);
            const float m = fmaxf(__low2float(mx[0]), __high2float(mx[0]));
            if (fmaxf(m, most) < kLow) {
#pragma unroll 1
                for (int i = 0; i < kUnroll * 8; i++) {
                    const int at = turn + tid + (i >> 3) * kThreads;
                    const long long n = (long long)at * 8 + (i & 7) - r.ahead;
                    if (at >= end || n < 0 || n >= r.vocab) continue;
                    const float x = __half2float(r.base[(size_t)at * 8 + (i & 7)]);
                    if (!isfinite(x)) continue;
                    if (x > most) {
                        most = x;
                        moved_to(run, -(x * kLog2e));
                    }
                    const float y = fmaf(x, kLog2e, run.c), e = exp2_of(y);
                    run.s += e;
                    run.t = fmaf(e, y, run.t);
                }
                continue;
            }
            if (m > most) {
                most = m;
                moved_to(run, -(m * kLog2e));
            }
            float s4[4] = {run.s, 0.f, 0.f, 0.f}, t4[4] = {run.t, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < kUnroll * 4; e++) {
                const float2 f = __half22float2(v[e]);
                const float a = fmaf(f.x, kLog2e, run.c), b = fmaf(f.y, kLog2e, run.c);
                const float ea = exp2_of(a), eb = exp2_of(b);
                s4[2 * (e & 1)] += ea;
                s4[2 * (e & 1) + 1] += eb;
                t4[2 * (e & 1)] = fmaf(ea, a, t4[2 * (e & 1)]);
                t4[2 * (e & 1) + 1] = fmaf(eb, b, t4[2 * (e & 1) + 1]);
            }
            run.s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
            run.t = (t4[0] + t4[1]) + (t4[2] + t4[3]);
        }
    }
    // ---- the CTA's sums ----
    {
        warp_sums(run);
        if (lane == 0) {
            warp_c[warp] = run.c;
            warp_s[warp] = run.s;
            warp_t[warp] = run.t;
        }
    }
    __syncthreads();
    {
        float c = warp_c[0];
#pragma unroll
        for (int w = 1; w < kWarps; w++) c = fminf(c, warp_c[w]);
        run = {c, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            Sums a = {warp_c[w], warp_s[w], warp_t[w]};
            moved_to(a, c);
            run.s += a.s;
            run.t += a.t;
        }
    }
    // ---- the first CTA of the row joins what the others found ----
    if constexpr (CLUSTER) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA of the row runs
        __syncthreads();
        auto remote = [&](const void *at) {
            uint32_t a;
            asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)));
            return a;
        };
        if (rank > 0) {
            if (tid < 3)
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(&sums[rank].c) + 4 * tid), "f"(tid == 0 ? run.c : tid == 1 ? run.s : run.t)
                             : "memory");
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank > 0) return;
        for (int i = 1; i < p.cluster; i++) joined(run, sums[i]);
    }
    if (tid == 0) store_row(p, row, target, run);
}

// Alternatives are compared by keys: larger for a larger value, then for an earlier one, 0 for no logit.  Within a turn
// (of at most 16384 logits) value << 16 | 0xFFFF - place, in a row value << 32 | 0xFFFFFFFF - id.
__device__ __forceinline__ unsigned value_key(__half x) {
    const unsigned short b = __half_as_ushort(x);
    return (b & 0x8000) ? (unsigned short)~b : (unsigned short)(b | 0x8000);
}
__device__ __forceinline__ __half value_of(unsigned v) {
    return __ushort_as_half((v & 0x8000) ? (unsigned short)(v & 0x7FFF) : (unsigned short)~v);
}

// take(key, how many are larger) for those of n keys that fewer than `top` are larger than, a warp a key.
template <typename K, typename F>
__device__ __forceinline__ void ranked(const K *keys, int n, int top, F &&take) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int i = threadIdx.x >> 5; i < n; i += kTopWarps) {
        const K key = keys[i];
        int above = 0;
#pragma unroll 1
        for (int j = lane; j - lane < n && above < top; j += 32) above += __popc(__ballot_sync(0xffffffffu, j < n && keys[j] > key));
        if (lane == 0 && above < top) take(key, above);
    }
}

// With alternatives.  Bound by latencies: of a turn's 8000 cycles (1 x 100003 split eight ways) 1500 pass until the
// logits are there, 1200 in the exponentials (16384, at 16 a cycle of the SM), the rest between barriers -- bound,
// candidates, ranks -- and 2000 more in joining the cluster, 1700 in ranking what its CTAs found.  512 threads halve
// the steps of each against 256 and leave room for a second CTA on the SM.  1 x 32000 with 5 alternatives takes 4.8 us, of
// which a call's launch is 3.6; 37 x 100003 with 20 11.2 (seven CTAs a row: all 37 clusters find room at once).
template <int PIECES>
__global__ void __launch_bounds__(kTopThreads, 2) logprob_top_kernel(const LogprobParams p) {
    constexpr int kTurn = kTopThreads * PIECES;  // pieces
    extern __shared__ __align__(16) unsigned list[];  // [list_size<PIECES>()]
    __shared__ __align__(16) unsigned group_best[kGroups];
    __shared__ __align__(16) unsigned long long best[kMaxCluster][kMaxTop + 1];  // of this CTA's turns; in the first CTA, of all (its lists in different banks)
    __shared__ __align__(16) unsigned turn_best[kMaxTop];
    __shared__ __align__(16) Sums sums[kMaxCluster];
    __shared__ __align__(16) float warp_max[kTopWarps], warp_s[kTopWarps], warp_t[kTopWarps];
    struct Found {
        unsigned bound;
        int n;
    };
    __shared__ __align__(16) Found found;
    if (p.cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    tlc_pdl_after_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = cluster_rank(), row = cluster_id();
    const __half *x0 = p.logits + (size_t)row * p.vocab;
    Target target = {-1, 0.f};
    // The row in 16-byte pieces of memory: the first and the last may reach into other rows, and past the array.
    const int ahead = (int)(((uintptr_t)x0 & 15) >> 1);  // values of the first piece in front of the row
    const __half *base = x0 - ahead;
    const int pieces = (int)(((unsigned)ahead + p.vocab + 7) / 8), first = rank * p.share, end = min(first + p.share, pieces);
    const int whole_first = ahead > 0, whole_end = (int)(((unsigned)ahead + p.vocab) / 8);  // pieces that are all the row's

    if (tid < p.top) best[0][tid] = 0;
    if (tid < kGroups) group_best[tid] = 0;
    Sums run = {INFINITY, 0.f, 0.f};
    for (int p0 = first; p0 < end; p0 += kTurn) {
        __half2 v[PIECES * 4];
        {
            uint4 w[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
                const int at = p0 + tid + i * kTopThreads;
                w[i] = make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);  // -inf
                if (at >= whole_first && at < whole_end && at < end) w[i] = *reinterpret_cast<const uint4 *>(base + (size_t)at * 8);
            }
            // a first and a last piece of which the row has a part, value by value
#pragma unroll 1
            for (int at = whole_first ? 0 : whole_end; at < pieces; at = at < whole_end ? whole_end : pieces) {
                const int off = at - p0 - tid;
                if (at >= end || off < 0 || off >= kTurn || (off & (kTopThreads - 1))) continue;
                unsigned x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const long long n = (long long)at * 8 + e - ahead;
                    x[e] = n >= 0 && n < p.vocab ? __half_as_ushort(x0[n]) : 0xFC00;
                }
#pragma unroll
                for (int i = 0; i < PIECES; i++)
                    if (off == i * kTopThreads) w[i] = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
            }
            if (p0 == 0 && tid == kTargetThread) target = target_of(p, row);
#pragma unroll
            for (int i = 0; i < PIECES; i++) clean(w[i], __float2half2_rn(-INFINITY), *reinterpret_cast<__half2(*)[4]>(&v[4 * i]));
        }
        // the key of a turn's value: 8 places a piece
        auto key_of = [&](__half x, int e, int half) { return value_key(x) << 16 | (0xFFFF - (unsigned)((tid + (e >> 2) * kTopThreads) * 8 + 2 * (e & 3) + half)); };
        // of the values that `hit` says, one bit each (e, and 16 + e for the upper half), those of value e
        auto value_at = [&](int e, int half) {
            __half2 x = v[0];
#pragma unroll
            for (int i = 1; i < PIECES * 4; i++)
                if (e == i) x = v[i];
            return half ? __high2half(x) : __low2half(x);
        };
        __half2 mx = v[0];
#pragma unroll
        for (int e = 1; e < PIECES * 4; e++) mx = __hmax2(mx, v[e]);
        const float mine = fmaxf(__low2float(mx), __high2float(mx));
        float m = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        __syncthreads();  // (what the turn before left here has been read)
        if (lane == 0) warp_max[warp] = m;
        if (mine > -INFINITY) {
            // the first of the values equal to the thread's maximum
            const __half2 want = __float2half2_rn(mine);
            unsigned hit = 0;
#pragma unroll
            for (int e = 0; e < PIECES * 4; e++) hit |= __heq2_mask(v[e], want) & (0x10001u << e);
            const int e = __ffs((hit | hit >> 16) & 0xFFFFu) - 1, half = hit >> e & 1 ? 0 : 1;
            atomicMax(&group_best[tid & (kGroups - 1)], key_of(__low2half(want), e, half));
        }
        if (tid == 0) found = {0, 0};
        if (tid < p.top) turn_best[tid] = 0;
        __syncthreads();
        m = warp_max[0];
#pragma unroll
        for (int w = 1; w < kTopWarps; w++) m = fmaxf(m, warp_max[w]);
        {
            // group tid / 8, against an eighth of the others: the one with k - 1 better ones is the bound
            const unsigned own = group_best[tid >> 3];
            const uint4 *all = reinterpret_cast<const uint4 *>(group_best);
            int better = 0;
#pragma unroll
            for (int i = 0; i < kGroups / 32; i++) {
                const uint4 g = all[8 * i + (tid & 7)];
                better += (g.x > own) + (g.y > own) + (g.z > own) + (g.w > own);
            }
#pragma unroll
            for (int o = 1; o < 8; o *= 2) better += __shfl_xor_sync(0xffffffffu, better, o);
            if ((tid & 7) == 0 && better == p.top - 1 && own > 0) found.bound = own;
        }
        float s = 0.f, t = 0.f;
        const float c = -(m * kLog2e);
        if (m > -INFINITY) {
            float s4[4] = {0.f, 0.f, 0.f, 0.f}, t4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < PIECES * 4; e++) {
                const float2 f = __half22float2(v[e]);
                // (2^-200 is zero; e t of a logit of -inf would be NaN)
                const float a = fmaxf(fmaf(f.x, kLog2e, c), -200.f), b = fmaxf(fmaf(f.y, kLog2e, c), -200.f);
                const float ea = exp2_of(a), eb = exp2_of(b);
                s4[2 * (e & 1)] += ea;
                s4[2 * (e & 1) + 1] += eb;
                t4[2 * (e & 1)] = fmaf(ea, a, t4[2 * (e & 1)]);
                t4[2 * (e & 1) + 1] = fmaf(eb, b, t4[2 * (e & 1) + 1]);
            }
            s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
            t = (t4[0] + t4[1]) + (t4[2] + t4[3]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
        }
        if (lane == 0) {
            warp_s[warp] = s;
            warp_t[warp] = t;
        }
        __syncthreads();
        if (tid < kGroups) group_best[tid] = 0;  // for the next turn
        {
            // 0: fewer than k groups have anything.  The k-th best of the turns before (0: there are not so many) bounds
            // as well: it keeps the last, short turn, where few groups have anything, from being ranked whole.  A later
            // logit that is equal to it comes behind it.
            const unsigned long long so_far = best[0][p.top - 1];
            const unsigned above = so_far ? ((unsigned)(so_far >> 32) + 1) << 16 : 0, least = found.bound > above ? found.bound : above;
            const __half least_x = least ? value_of(least >> 16) : __ushort_as_half((unsigned short)0xFBFF);  // the lowest f16
            if (mine >= __half2float(least_x)) {
                const __half2 least2 = __half2half2(least_x);
                unsigned hit = 0;
#pragma unroll
                for (int e = 0; e < PIECES * 4; e++) hit |= __hge2_mask(v[e], least2) & (0x10001u << e);
#pragma unroll 1
                while (hit) {
                    const int bit = __ffs(hit) - 1;
                    hit &= hit - 1;
                    const unsigned key = key_of(value_at(bit & 15, bit >> 4), bit & 15, bit >> 4);
                    if (key >= least) list[atomicAdd(&found.n, 1)] = key;
                }
            }
        }
        s = t = 0.f;
#pragma unroll
        for (int w = 0; w < kTopWarps; w++) {
            s += warp_s[w];
            t += warp_t[w];
        }
        joined(run, {c, s, t});
        __syncthreads();
        ranked(list, found.n, p.top, [&](unsigned key, int above) { turn_best[above] = key; });
        __syncthreads();
        auto whole = [&](unsigned key) {
            const unsigned id = ((unsigned)p0 * 8 - ahead) + (0xFFFF - (key & 0xFFFF));
            return key ? (unsigned long long)(key >> 16) << 32 | (0xFFFFFFFFu - id) : 0;
        };
        if (p0 == first) {
            if (tid < p.top) best[0][tid] = whole(turn_best[tid]);
        } else {
            // two sorted lists, a warp each: a key's place is its own and the number of larger ones in the other
            unsigned long long key = 0;
            int above = lane;
            if (warp < 2 && lane < p.top) {
                key = warp ? whole(turn_best[lane]) : best[0][lane];
                for (int i = 0; i < p.top; i++) above += (warp ? best[0][i] : whole(turn_best[i])) > key;
            }
            __syncthreads();
            if (key > 0 && above < p.top) best[0][above] = key;
        }
    }
    const size_t out = (size_t)row * p.top;
    if (rank == 0 && tid < p.top) {  // where there are fewer logits
        p.top_ids[out + tid] = -1;
        p.top_logprobs[out + tid] = -INFINITY;
    }
    // The first CTA of the row joins what the others found.
    if (p.cluster > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA of the row runs
        __syncthreads();
        auto remote = [&](const void *at) {
            uint32_t a;
            asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)));
            return a;
        };
        if (rank == 0) {
            if (tid == 0) {
                sums[0] = run;
                found.n = 0;
            }
        } else {
            if (tid < p.top)
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(&best[rank][tid])), "l"(best[0][tid]) : "memory");
            if (tid < 3)
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(&sums[rank].c) + 4 * tid), "f"(tid == 0 ? run.c : tid == 1 ? run.s : run.t)
                             : "memory");
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank > 0) return;
        run = lane < p.cluster ? sums[lane] : Sums{INFINITY, 0.f, 0.f};
        warp_sums(run);
    }
    const float log2_s = run.c < INFINITY ? log2f(run.s) : 0.f;
    auto store = [&](int at, unsigned long long key) {
        p.top_ids[out + at] = (int)(0xFFFFFFFFu - (unsigned)key);
        p.top_logprobs[out + at] = logprob_of(__half2float(value_of((unsigned)(key >> 32))), run, log2_s);
    };
    __syncthreads();
    if (p.cluster == 1) {
        if (tid < p.top && best[0][tid] > 0) store(tid, best[0][tid]);
    } else {
        // The CTAs' sorted lists: k keys reach the least of their (k / CTAs)-th ones, and no key below it counts.
        unsigned long long *keys = reinterpret_cast<unsigned long long *>(list), least = ~0ull;
        const int nth = (p.top + p.cluster - 1) / p.cluster, at = tid % kMaxTop;
        for (int i = 0; i < p.cluster; i++) least = min(least, best[i][nth - 1]);
        const unsigned long long key = tid < p.cluster * kMaxTop && at < p.top ? best[tid / kMaxTop][at] : 0;
        if (key > 0 && key >= least) keys[atomicAdd(&found.n, 1)] = key;
        __syncthreads();
        ranked(keys, found.n, p.top, [&](unsigned long long key, int above) { store(above, key); });
    }
    if (tid == kTargetThread) store_row(p, row, target, run);
}

template <int PIECES>
cudaError_t launch_top(tlc_ctx *ctx, cudaLaunchConfig_t &cfg, const LogprobParams &p) {
    constexpr size_t smem = list_size<PIECES>() * sizeof(unsigned);
    static bool configured[64] = {};
    if (!configured[ctx->device & 63]) {
        const cudaError_t e = cudaFuncSetAttribute(logprob_top_kernel<PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        configured[ctx->device & 63] = true;
    }
    cfg.blockDim = dim3(kTopThreads);
    cfg.dynamicSmemBytes = smem;
    return cudaLaunchKernelEx(&cfg, logprob_top_kernel<PIECES>, p);
}

// How many 16-byte pieces a slice has, at most.
constexpr int slice_pieces(int vocab, int ctas) { return (int)((((long long)vocab + 14) / 8 + ctas - 1) / ctas); }

// How many clusters of c CTAs of the kernel with alternatives run at once, two CTAs an SM.  The plan takes it as the measure of
// the GPU's room for rows without alternatives too: their CTAs are half as large, and the costs below were fitted with it.
int resident_clusters(tlc_ctx *ctx, int c) {
    static int known[64][kMaxCluster + 1] = {};
    int &n = known[ctx->device & 63][c];
    if (n > 0) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c);
    cfg.blockDim = dim3(kTopThreads);
    cfg.dynamicSmemBytes = list_size<4>() * sizeof(unsigned);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)c;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, logprob_top_kernel<4>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        clusters = 0;
    }
    return n = clusters > 0 ? clusters : 1;
}

// CTAs a row, by cost in microseconds as fitted to calls of 1 to 400 rows of 16000 to 151936 logits with 1 to 8 CTAs a
// row.  A row costs the joining of its CTAs and a CTA's work: a turn of 2048 pieces with alternatives (3.45, with 512 or
// 1024 pieces 2 or 2.5), 15000 logits a microsecond without.  Half of the clusters that run at once find SMs of their own
// (of more than two CTAs, which lie in one part of the chip, a quarter); all of them take 1.5 times as long, more wait.
// With 20 alternatives 36 x 32000 takes 9.2, 6.6, 6.8, 7.4, 7.5, 7.8, 8.6 and 10.0 us with 1 to 8 CTAs a row (two are taken),
// 36 x 100003 27.3, 17.7, 13.9, 14.0, 13.7, 13.5, 9.7 and 12.3 (seven), 148 x 100003 27.7, 24.4, 35.0, 31.1, 36.2, 41.7, 29.0
// and 31.9 (two).  Without, 36 x 100003 takes 8.5, 6.6, 5.7, 6.0, 6.6, 5.9, 5.8 and 7.1 (seven), 148 x 100003 8.6, 9.1, 11.2,
// 11.8, 12.0, 13.3, 12.1 and 14.0 (two), 512 x 32000 8.8, 11.3, 15.9, 15.1, 18.1, 21.2, 24.2 and 27.7 (one).  Of 128 pairs of rows and vocabulary the
// plan is up to 18 % behind the best number, and 31 % once (16 x 151936 with alternatives).
int ctas_a_row(tlc_ctx *ctx, int rows, int vocab, bool alternatives) {
    constexpr double kJoin[2][kMaxCluster] = {{0, 1.1, 1.2, 1.3, 1.5, 1.7, 1.9, 2.1}, {0, 1.2, 1.3, 1.4, 1.45, 1.5, 1.55, 1.6}};
    int best = 1;
    double least = 1e30;
    for (int c = 1; c <= kMaxCluster; c++) {
        const int n = slice_pieces(vocab, c), held = n <= kTopThreads ? 1 : n <= 2 * kTopThreads ? 2 : 4, all = resident_clusters(ctx, c);
        const double work = alternatives ? (double)((n + held * kTopThreads - 1) / (held * kTopThreads)) * (1.5 + 0.49 * held) : n * 8 / 15000.0;
        const double times = rows <= all / (c <= 2 ? 2 : 4) ? 1.0 : rows <= all ? 1.5 : (c == 1 ? 0.3 : 0.9) + 1.6 * rows / all;
        const double cost = kJoin[alternatives][c - 1] + work * times;
        if (cost < least) {
            least = cost;
            best = c;
        }
    }
    return best;
}

}  // namespace

extern "C" int32_t tlc_token_logprobs(tlc_ctx *ctx, const void *logits_dev, int32_t rows, int32_t vocab,
                                      const int32_t *targets_dev, int32_t top_k, float *logprobs_dev, float *entropy_dev,
                                      int32_t *top_ids_dev, float *top_logprobs_dev) {
    if (int32_t rc = tlc_enter(ctx)) return rc;
    tlc_perf_scope perf(ctx, "token_logprobs(rows=%d, vocab=%d, top=%d)", rows, vocab, top_k);
    TLC_REQUIRE(logits_dev && (!logprobs_dev || targets_dev) && (top_k <= 0 || (top_ids_dev && top_logprobs_dev)),
                TLC_ERR_INVALID_OPERATION, "token_logprobs: null pointer");
    TLC_REQUIRE(rows >= 0 && rows <= INT_MAX / kMaxCluster && vocab > 0 && vocab <= INT_MAX - 8, TLC_ERR_INVALID_DIMENSION,
                "token_logprobs: bad shape [%d, %d]", rows, vocab);
    TLC_REQUIRE(top_k >= 0 && top_k <= kMaxTop, TLC_ERR_INVALID_OPERATION, "token_logprobs: top_k %d outside 0 .. %d", top_k, kMaxTop);
    TLC_REQUIRE(((uintptr_t)logits_dev & 1) == 0, TLC_ERR_INVALID_OPERATION, "token_logprobs: logits must be 2-byte aligned");
    if (rows == 0) return TLC_OK;
    LogprobParams p{};
    p.logits = static_cast<const __half *>(logits_dev);
    p.targets = targets_dev;
    p.logprobs = logprobs_dev;
    p.entropy = entropy_dev;
    p.top_ids = top_ids_dev;
    p.top_logprobs = top_logprobs_dev;
    p.rows = rows;
    p.vocab = vocab;
    p.top = top_k;
    p.status = ctx->dev_status;
    const int c = ctas_a_row(ctx, rows, vocab, top_k > 0);
    p.cluster = c;
    p.share = slice_pieces(vocab, c);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * c));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (c > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = (unsigned)c;
        attr[na].val.clusterDim.y = 1;
        attr[na++].val.clusterDim.z = 1;
    }
    if (ctx->use_pdl && ctx->pdl_small) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    const cudaError_t le = top_k == 0                  ? cudaLaunchKernelEx(&cfg, c > 1 ? logprob_kernel<true> : logprob_kernel<false>, p)
                           : p.share <= kTopThreads     ? launch_top<1>(ctx, cfg, p)
                           : p.share <= 2 * kTopThreads ? launch_top<2>(ctx, cfg, p)
                                                       : launch_top<4>(ctx, cfg, p);
    if (le != cudaSuccess) {
        cudaGetLastError();
        return tlc_fail(TLC_ERR_CUDA, "token_logprobs launch failed: %s", cudaGetErrorString(le));
    }
    TLC_CHECK_LAUNCH(ctx);
    return TLC_OK;
}

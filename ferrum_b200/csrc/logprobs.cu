// What is said of a token given the output head's logits: the log probability and rank of a given token, the entropy of the
// row's distribution and its most likely tokens.
//
//   z = log sum_j exp(l_j)     logprob = l_id - z     rank = 1 + |{j: l_j > l_id}|     entropy = z - sum_j exp(l_j - z) l_j
//
// A logit of -infinity is a token of probability 0 and adds nothing anywhere.  A row with a NaN, with +infinity or with nothing
// above -infinity has no distribution: its numbers are NaN, and its rank counts what compares above l_id.
//
// A row is read once, by a block or by a cluster of blocks (each a contiguous part; block 0 collects through distributed shared
// memory).  In powers of two, with b = log2(e) as fp32 has it and a pivot c:
//
//   S = sum 2^(b l - c)     T = sum 2^(b l - c) (b l - c)     z = (c + log2 S) / b     entropy = ln 2 (log2 S - T / S)
//
// Where one token has all of the probability, l_id - z and the entropy are what the roundings of c, S and T leave (less than 2^-21, of
// either sign).  No log probability above 0 and no entropy below it is given out: such values are 0.
//
// b l - c is one FMA with one rounding; c is the largest b l of what the block reads first and moves only when a logit is more
// than 20 / b above it (a term is 2^20 at most, far from fp32's end; a running maximum would rescale every few values).  Dividing by b as
// it is keeps its own rounding out of z.
//
// The most likely tokens: while the row is read, every thread notes the largest of each 16 or more logits it takes in.  Of the
// block's threads the k-th largest maximum (of the best of every warp) is a bound that k tokens reach and few more do, so at
// the end only the few pieces that reach it are read again, and what they hold is put in order by counting (what a piece could
// hold was looked at as it came by, against a bound that rose slowly, in the first version: 20 to 90 us more for 8 to 32
// alternatives of 1021 rows).
// Keys (value, index) are unique, of equal values the lower index is larger, so nothing depends on the order of threads.
//
// Many long rows are bound by memory (F32) or by issue and the exponentials (bf16), the alternatives' end by latency: 1021 rows
// of 151936 bf16 54 us (5.7 TB/s) without and 65 us with 8 alternatives, F32 101 us (6.2 TB/s) and 116 us; one row F32 with 20
// of them 8.3 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemv_common.cuh"
#include "internal.h"

namespace {
using namespace fqk;

constexpr uint32_t MAX_TOP = 32, MAX_CLUSTER = 8;
constexpr int UNROLL = 4; // 16-byte loads of a thread in flight
// Maxima that a thread notes; tiles share one where they are more.  Eight KB a block: with 40 the blocks' shared memory left so little
// of the L1 cache that loads waited for a place in it (20 alternatives of 1021 rows of 151936 F32: 128 us, with 20 / 12 / 8 / 6 / 4
// 122 / 121 / 121 / 122 / 125; of 300 rows of 1000000 with 12 / 8 / 4 316 / 320 / 330).
template <int NT> constexpr uint32_t NOTES = 8 * 256 / NT;
constexpr uint32_t POOL = 512;   // pieces read again, and values kept of them
constexpr float LOG2E = 1.44269502f; // b: log2(e) rounded to fp32
constexpr float SLACK = 20.f;        // how far b l may be above the pivot
// Beyond a million the rounding of c is no longer small: a row whose largest logit lies there is summed in 64 bits (sum_64).
constexpr float MOST = 1048576.f;
// Lower logits, -infinity among them, count as this: a power of two, so that b LEAST is exact, and a bf16 number.
constexpr float LEAST = -0x1p126f;

// Numbers in their order as unsigned integers: NaN below everything, the two zeros equal.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float((order & 0x80000000u) ? order ^ 0x80000000u : ~order); }
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t i) { return (uint64_t)order << 32 | (uint32_t)~i; }

__device__ __forceinline__ float exp2_fast(float d) { // within 2^-22 of itself; 0 below 2^-126
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_half(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

// Pairs of fp32 in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }

template <typename T> constexpr int PER_LOAD = 16 / (int)sizeof(T);
__device__ __forceinline__ uint32_t word(const uint4 &u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }
// The largest of 16-byte pieces; NaN if one is.
template <typename T, int N> __device__ __forceinline__ float largest(const uint4 (&u)[N]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t m = max_nan_bf16x2(max_nan_bf16x2(u[0].x, u[0].y), max_nan_bf16x2(u[0].z, u[0].w));
#pragma unroll
        for (int i = 1; i < N; i++) m = max_nan_bf16x2(m, max_nan_bf16x2(max_nan_bf16x2(u[i].x, u[i].y), max_nan_bf16x2(u[i].z, u[i].w)));
        return max_nan(low_half(m), high_half(m));
    } else {
        float m = __uint_as_float(u[0].x);
#pragma unroll
        for (int i = 0; i < N; i++)
            m = max_nan(m, max_nan(max_nan(__uint_as_float(u[i].x), __uint_as_float(u[i].y)), max_nan(__uint_as_float(u[i].z), __uint_as_float(u[i].w))));
        return m;
    }
}
// Values 2 i and 2 i + 1 of a piece.
template <typename T> __device__ __forceinline__ float2 pair_of(const uint4 &u, int i) {
    if constexpr (sizeof(T) == 2) return make_float2(low_half(word(u, i)), high_half(word(u, i)));
    else return make_float2(__uint_as_float(word(u, 2 * i)), __uint_as_float(word(u, 2 * i + 1)));
}
// The same, not below LEAST (and without NaN).
template <typename T> __device__ __forceinline__ float2 pair_from_least(const uint4 &u, int i) {
    if constexpr (sizeof(T) == 2) {
        const uint32_t w = max_bf16x2(word(u, i), 0xFE80FE80u); // LEAST
        return make_float2(low_half(w), high_half(w));
    } else {
        return make_float2(fmaxf(__uint_as_float(word(u, 2 * i)), LEAST), fmaxf(__uint_as_float(word(u, 2 * i + 1)), LEAST));
    }
}
template <typename T> __device__ __forceinline__ float load1(const T *l, uint32_t i) {
    if constexpr (sizeof(T) == 2) return low_half(__ldcg(reinterpret_cast<const unsigned short *>(l) + i));
    else return __ldcg(l + i);
}

// The 16-byte piece at elements first .. of a row's end: one element at a time, -infinity outside the row.
template <typename T> __device__ __noinline__ uint4 ends(const T *l, uint32_t n, uint32_t first) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t a = first + 2 * i, b = a + 1; // wrap in the piece that begins before the row
            const uint32_t lo = a < n ? __ldcg(reinterpret_cast<const unsigned short *>(l) + a) : 0xFF80u, hi = b < n ? __ldcg(reinterpret_cast<const unsigned short *>(l) + b) : 0xFF80u;
            w[i] = lo | hi << 16;
        } else {
            const uint32_t a = first + i;
            w[i] = a < n ? __float_as_uint(__ldcg(l + a)) : 0xFF800000u;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

struct Sums {
    float c, s, t; // pivot, sum 2^(b l - c), sum 2^(b l - c) (b l - c)
};
// The sums about another pivot.
__device__ __forceinline__ void move_pivot(Sums &a, float c) {
    const float f = exp2_fast(a.c - c);
    a.t = f > 0.f ? f * fmaf(a.c - c, a.s, a.t) : 0.f; // f = 0: nothing is left of them, whatever they were
    a.s = f > 0.f ? f * a.s : 0.f;
    a.c = c;
}
__device__ __forceinline__ void join(Sums &a, Sums b) {
    const float c = fmaxf(a.c, b.c);
    if (a.c != c) move_pivot(a, c);
    if (b.c != c) move_pivot(b, c);
    a.s += b.s;
    a.t += b.t;
}
// Over the first `lanes` lanes (a power of two).  Pivots are the same nearly always.
__device__ __forceinline__ Sums join_warp(Sums a, int lanes = 32) {
    if (__all_sync(0xffffffffu, a.c == __shfl_sync(0xffffffffu, a.c, 0))) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1)
            if (off < lanes) {
                a.s += __shfl_xor_sync(0xffffffffu, a.s, off);
                a.t += __shfl_xor_sync(0xffffffffu, a.t, off);
            }
        return a;
    }
#pragma unroll 1
    for (int off = lanes / 2; off > 0; off >>= 1) {
        const Sums b{__shfl_xor_sync(0xffffffffu, a.c, off), __shfl_xor_sync(0xffffffffu, a.s, off), __shfl_xor_sync(0xffffffffu, a.t, off)};
        join(a, b);
    }
    return a;
}
// A row of logits around numbers beyond MOST: by one warp, in 64 bits about its largest (151936 of them 1.7 ms; no model has such).
template <typename T> __device__ __noinline__ void sum_64(const T *l, uint32_t n, uint32_t lane, double &z, double &entropy) {
    double mx = -INFINITY, s = 0.0, t = 0.0;
    for (uint32_t i = lane; i < n; i += 32) mx = fmax(mx, (double)load1(l, i));
    for (int off = 16; off > 0; off >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    for (uint32_t i = lane; i < n; i += 32) {
        const double d = fmax((double)load1(l, i) - mx, -1000.0), e = exp(d);
        s += e;
        t = fma(d, e, t);
    }
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off), t += __shfl_xor_sync(0xffffffffu, t, off);
    z = mx + log(s);
    entropy = log(s) - t / s;
}

__device__ __forceinline__ float not_above_0(double v) { return v > 0.0 ? 0.f : (float)v; } // NaN stays NaN

struct Outputs {
    float *logprobs;
    uint32_t *ranks;
    float *entropy, *top_logprobs;
    uint32_t *top_ids;
};

__device__ __forceinline__ uint32_t cluster_address(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void store_cluster(uint32_t to, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(v) : "memory"); }

template <bool TOP> struct Best { // shared memory of best_of
    alignas(16) uint64_t keys[POOL + MAX_TOP];
    alignas(16) uint32_t maxima[64];
    uint64_t out[MAX_TOP];
    uint32_t work[POOL], wanted, found, bound, before[32];
};
template <> struct Best<false> {};

// The first `total` keys of the pool in order, the best MAX_TOP of them in S.out; `meanwhile` is done before the last barrier.
template <int NT, typename F> __device__ __forceinline__ void order_pool(Best<true> &S, uint32_t total, F meanwhile) {
    const uint32_t tid = threadIdx.x;
    if (tid < MAX_TOP) S.out[tid] = 0;
    if (tid == 0) S.keys[total] = 0; // they are read by twos
    __syncthreads();
    for (uint32_t i = tid; i < total; i += NT) {
        const uint64_t mine = S.keys[i];
        uint32_t higher = 0;
#pragma unroll 8
        for (uint32_t o = 0; o < total; o += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(S.keys + o);
            higher += (two.x > mine) + (two.y > mine);
        }
        if (higher < MAX_TOP) S.out[higher] = mine;
    }
    meanwhile();
    __syncthreads();
}

// The k best (value, index) keys of the block's pieces [begin, end), sorted, in the lanes of its first warp (0 where there are
// fewer); all threads call it, after what they noted (`noted` times, the largest `most`).  `meanwhile`: before its last barrier.
template <typename T, int NT, typename F>
__device__ __forceinline__ uint64_t best_of(Best<true> &S, const float *notes, uint32_t noted, float most, uint32_t shared_by, const T *l, const uint4 *aligned, uint32_t n,
                                            uint32_t skip, uint32_t begin, uint32_t end, uint32_t k, F meanwhile) {
    constexpr uint32_t W = NT / 32, V = PER_LOAD<T>, TILE = UNROLL * NT;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // This thread's first piece of a note; the threads that have one come first.
    auto piece_of = [&](uint32_t note, uint32_t thread) { return begin + note * shared_by * TILE + thread; };
    uint32_t best = order_of(most); // a logit of the thread, or 0
    // The largest maxima of every warp whose threads all have logits, 32 or (from 17 alternatives on) 64 of them, k at least.
    const uint32_t warps = max(1u, min(W, (end - begin) / 32)), m = min(32u, (k > 16 ? 64 : 32) / warps);
    if (warp < warps) {
        uint32_t high = __reduce_max_sync(0xffffffffu, best);
#pragma unroll 1
        for (uint32_t i = 0; i < m; i++) {
            if (lane == 0) S.maxima[warp * m + i] = high;
            const uint32_t holders = __ballot_sync(0xffffffffu, best == high);
            if (lane == (uint32_t)__ffs(holders) - 1) best = 0;
            high = __reduce_max_sync(0xffffffffu, best);
        }
    }
    for (uint32_t i = m * warps + tid; i < 64; i += NT) S.maxima[i] = 0;
    if (tid == 0) S.wanted = S.found = 0;
    __syncthreads();
    // The bound: the least of those that fewer than k are above.  0, below everything, where there are fewer than k.
    if (warp < 2) {
        const uint32_t mine = S.maxima[tid], last = k > 16 ? 64 : 32;
        uint32_t higher = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < last; i += 4) {
            const uint4 f = *reinterpret_cast<const uint4 *>(S.maxima + i);
            higher += (f.x > mine) + (f.y > mine) + (f.z > mine) + (f.w > mine);
        }
        const uint32_t reached = __reduce_min_sync(0xffffffffu, higher < k && tid < last ? mine : 0xFFFFFFFFu);
        if (lane == 0) S.before[warp] = reached;
    }
    __syncthreads();
    uint32_t least = min(S.before[0], S.before[1]);
    auto load = [&](uint32_t j) { return j * V - skip <= n && n - (j * V - skip) >= V ? __ldcg(aligned + j) : ends(l, n, j * V - skip); };
    auto order_at = [&](const uint4 &p, uint32_t i) {
        const uint32_t w = word(p, sizeof(T) == 2 ? i / 2 : i);
        return order_of(sizeof(T) == 4 ? __uint_as_float(w) : (i & 1) ? high_half(w) : low_half(w));
    };
    // All logits that reach the bound; where they are too many for the pool, many are equal to it, or the threads' maxima were
    // not spread: then those above it, and where these are too many, those above the k-th of the ones at hand, and so on.
    bool above = false; // only those above the bound
    uint32_t total;
    for (;;) {
        const float reach = value_of(least);
        if (__any_sync(0xffffffffu, !(most < reach)))
#pragma unroll 2
            for (uint32_t i = 0; i < noted; i++) {
                const float v = notes[i * NT + tid];
                const bool want = piece_of(i, tid) < end && (least == 0 ? !above || v == v : above ? v > reach : v >= reach);
                const uint32_t which = __ballot_sync(0xffffffffu, want);
                if (which == 0) continue;
                uint32_t at = 0;
                if (lane == 0) at = atomicAdd(&S.wanted, __popc(which));
                at = __shfl_sync(0xffffffffu, at, 0) + __popc(which & ((1u << lane) - 1));
                if (want && at < POOL) S.work[at] = i * NT + tid;
            }
        __syncthreads();
        const uint32_t wanted = S.wanted, per = UNROLL * shared_by;
        for (uint32_t i = tid; i < min(wanted, POOL) * per; i += NT) {
            const uint32_t entry = S.work[i / per], j = piece_of(entry / NT, entry % NT) + i % per * NT;
            if (j >= end) continue;
            const uint4 p = load(j);
#pragma unroll
            for (uint32_t e = 0; e < V; e++) {
                const uint32_t w = word(p, sizeof(T) == 2 ? e / 2 : e), at = j * V - skip + e;
                const float v = sizeof(T) == 4 ? __uint_as_float(w) : (e & 1) ? high_half(w) : low_half(w);
                if (v < reach || at >= n) continue;
                const uint32_t order = order_of(v);
                if (above ? order > least : order >= least) {
                    const uint32_t to = atomicAdd(&S.found, 1u);
                    if (to < POOL) S.keys[to] = key_of(order, at);
                }
            }
        }
        __syncthreads();
        total = min(S.found, POOL);
        if (S.found <= POOL && wanted <= POOL) break;
        if (above) { // POOL of them are there: the order that fewer than k of these are above
            if (tid == 0) S.bound = 0xFFFFFFFFu;
            __syncthreads();
            for (uint32_t i = tid; i < total; i += NT) {
                const uint32_t mine = (uint32_t)(S.keys[i] >> 32);
                uint32_t higher = 0;
                for (uint32_t o = 0; o < total; o++) higher += (uint32_t)(S.keys[o] >> 32) > mine;
                if (higher < k) atomicMin(&S.bound, mine);
            }
            __syncthreads();
            least = S.bound;
        }
        above = true;
        __syncthreads();
        if (tid == 0) S.wanted = S.found = 0;
        __syncthreads();
    }
    // Of those equal to the bound the first in the row, as many as are still needed.
    if (above && total < k)
        for (uint32_t j0 = begin; j0 < end && total < k; j0 += NT) {
            uint32_t equal = 0; // bits of the thread's piece
            if (j0 + tid < end) {
                const uint4 p = load(j0 + tid);
#pragma unroll 1
                for (uint32_t e = 0; e < V; e++)
                    if (order_at(p, e) == least && (j0 + tid) * V - skip + e < n) equal |= 1u << e;
            }
            uint32_t ahead = __popc(equal);
#pragma unroll
            for (uint32_t d = 1; d < 32; d *= 2) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, ahead, d);
                if (lane >= d) ahead += v;
            }
            if (lane == 31) S.before[warp] = ahead;
            __syncthreads();
            uint32_t at = total + ahead - __popc(equal);
            for (uint32_t w = 0; w < W; w++) {
                if (w < warp) at += S.before[w];
                total += S.before[w];
            }
            for (; equal && at < k; at++, equal &= equal - 1) S.keys[at] = key_of(least, (j0 + tid) * V - skip + __ffs(equal) - 1);
            total = min(total, max(k, 1u));
            __syncthreads();
        }
    order_pool<NT>(S, total, meanwhile);
    return S.out[lane];
}

// Block `rank` of the `parts` of row blockIdx.x / parts.
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, NT == 512 ? 1 : 1024 / NT)
k_token_logprobs(const T *logits, uint32_t n, size_t stride, const uint32_t *ids, uint32_t k, uint32_t parts, Outputs out) {
    constexpr int W = NT / 32, V = PER_LOAD<T>;
    extern __shared__ float notes[]; // [NOTES or fewer][NT]: the largest of a thread's logits in a tile; NaN: it has no number there
    __shared__ uint32_t first_max[W];
    __shared__ Sums sums[W];
    __shared__ uint32_t counts[W], bads[W];
    __shared__ Best<TOP> top;
    __shared__ double row_z; // log of the row's sum of exponentials
    // Of block 0: what the blocks of the cluster found.
    __shared__ Sums all_sums[MAX_CLUSTER];
    __shared__ uint32_t all_counts[MAX_CLUSTER], all_bads[MAX_CLUSTER];
    __shared__ uint64_t all_lists[TOP ? MAX_CLUSTER : 1][32];
    // Block 0's shared memory may be written once all blocks of the cluster run: arrived here, waited for before the writes.
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    pdl_trigger();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / parts, rank = blockIdx.x - row * parts;
    pdl_wait();
    // The row in whole 16-byte pieces from the boundary below its start: piece j holds elements j * V - skip ...
    const T *l = logits + (size_t)row * stride;
    const uint32_t skip = (uint32_t)(((uintptr_t)l & 15) / sizeof(T));
    const uint4 *aligned = reinterpret_cast<const uint4 *>(l - skip);
    const uint32_t pieces = (uint32_t)(((uint64_t)skip + n + V - 1) / V), per = (pieces + parts - 1) / parts;
    const uint32_t begin = min(rank * per, pieces), end = min(begin + per, pieces);
    const uint32_t whole_from = skip ? 1 : 0, whole_to = min(end, (uint32_t)(((uint64_t)skip + n) / V)); // pieces that lie in the row
    const uint32_t id = ids ? __ldcg(ids + row) : n;
    constexpr uint32_t NONE = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u; // -infinity
    // The next pieces are under way while these are added, where four blocks an SM read bf16 (8 of 1021 rows of 151936: 69 instead
    // of 74 us).  F32 pieces take longer to arrive than to add and lose by the registers (k = 20: 128 / 132 us), and so do eight blocks an
    // SM (20 of 2000 rows of 8192 bf16 19.6 / 20.6).
    constexpr bool EARLY = sizeof(T) == 2 && NT == 256;
    uint4 now[UNROLL];
    // This thread's UNROLL pieces of the block's UNROLL * NT from j0 on.
    auto fetch = [&](uint32_t j0, uint4 (&now)[UNROLL]) {
        if (j0 >= whole_from && j0 + UNROLL * NT <= whole_to) {
#pragma unroll
            for (int u = 0; u < UNROLL; u++) now[u] = __ldcg(aligned + j0 + u * NT + tid);
        } else {
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const uint32_t j = j0 + u * NT + tid;
                now[u] = make_uint4(NONE, NONE, NONE, NONE);
                if (j >= whole_from && j < whole_to) now[u] = __ldcg(aligned + j);
                else if (j < end) now[u] = ends(l, n, j * V - skip);
            }
        }
    };
    fetch(begin, now);
    const float given = id < n ? load1(l, id) : __int_as_float(0x7fc00000);

    // The largest of what is read first is the pivot.
    const uint32_t first = __reduce_max_sync(0xffffffffu, order_of(largest<T>(now))); // (a thread with a NaN does not count)
    if (lane == 0) first_max[warp] = first;
    __syncthreads();
    const float start = value_of(max(__reduce_max_sync(0xffffffffu, first_max[lane % W]), 1u << 23)); // the lowest number where there is none
    Sums a{fmaxf(start, LEAST) * LOG2E, 0.f, 0.f};
    float limit = fminf(fmaf(SLACK, 1.f / LOG2E, fmaxf(start, LEAST)), MOST); // logits above it move the pivot
    bool bad = false, beyond = false, some = false; // a NaN or +infinity; a logit above MOST; one above -infinity
    uint32_t count = 0;
    const uint32_t tiles = (end - begin + UNROLL * NT - 1) / (UNROLL * NT), shared_by = (tiles + NOTES<NT> - 1) / NOTES<NT>; // tiles of a note
    float note = __int_as_float(0x7fc00000), most = note;
    uint32_t noted = 0, at_note = 0;
    float2 s2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);

#pragma unroll 1
    for (uint32_t j0 = begin; j0 < end; j0 += UNROLL * NT) {
        [[maybe_unused]] uint4 next[UNROLL];
        if (EARLY && j0 + UNROLL * NT < end) fetch(j0 + UNROLL * NT, next);
        const float highest = largest<T>(now);
        if constexpr (TOP) {
            float h = highest;
            if (j0 < whole_from || j0 + UNROLL * NT > whole_to || h != h) { // only the row's numbers count
                h = __int_as_float(0x7fc00000);
#pragma unroll
                for (int u = 0; u < UNROLL; u++)
#pragma unroll
                    for (int i = 0; i < V / 2; i++) {
                        const float2 v = pair_of<T>(now[u], i);
                        const uint32_t j = j0 + u * NT + tid, at = j * V - skip + 2 * i;
                        if (j < end && at < n) h = fmaxf(h, v.x);
                        if (j < end && at + 1 < n) h = fmaxf(h, v.y);
                    }
            }
            note = noted ? fmaxf(note, h) : h;
            if (++noted == shared_by || j0 + UNROLL * NT >= end) {
                notes[at_note++ * NT + tid] = note;
                most = fmaxf(most, note);
                noted = 0;
            }
        }
        if (!(highest <= given)) {
            if constexpr (sizeof(T) == 2) { // ones added in bf16, 32 at most
                const __nv_bfloat162 g = __float2bfloat162_rn(given);
                __nv_bfloat162 above = __float2bfloat162_rn(0.f);
#pragma unroll
                for (int u = 0; u < UNROLL; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t w = word(now[u], i);
                        above = __hadd2(above, __hgt2(*reinterpret_cast<const __nv_bfloat162 *>(&w), g));
                    }
                count += (uint32_t)(__low2float(above) + __high2float(above));
            } else {
#pragma unroll
                for (int u = 0; u < UNROLL; u++)
#pragma unroll
                    for (int i = 0; i < V; i++) count += __uint_as_float(word(now[u], i)) > given;
            }
        }
        some |= highest > -INFINITY;
        if (!(highest <= limit)) {
            bad |= !(highest < INFINITY);
            beyond |= highest > MOST;
            if (!bad && !beyond) {
                a.s = s2.x + s2.y;
                a.t = t2.x + t2.y;
                move_pivot(a, highest * LOG2E);
                limit = fminf(fmaf(SLACK, 1.f / LOG2E, highest), MOST);
                s2 = make_float2(a.s, 0.f);
                t2 = make_float2(a.t, 0.f);
            }
        }
        const float2 b2 = make_float2(LOG2E, LOG2E), c2 = make_float2(-a.c, -a.c);
        float2 s_tile = make_float2(0.f, 0.f), t_tile = s_tile; // (a sum of short sums rounds off less)
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                const float2 d = fma2(pair_from_least<T>(now[u], i), b2, c2);
                const float2 e = make_float2(exp2_fast(d.x), exp2_fast(d.y));
                s_tile = add2(s_tile, e);
                t_tile = fma2(d, e, t_tile);
            }
        s2 = add2(s2, s_tile);
        t2 = add2(t2, t_tile);
        if constexpr (EARLY) {
#pragma unroll
            for (int u = 0; u < UNROLL; u++) now[u] = next[u];
        } else if (j0 + UNROLL * NT < end) {
            fetch(j0 + UNROLL * NT, now);
        }
    }
    a.s = s2.x + s2.y;
    a.t = t2.x + t2.y;

    // The block's sums and its best values, then the cluster's.
    a = join_warp(a);
    count = __reduce_add_sync(0xffffffffu, count);
    uint32_t flags = (__any_sync(0xffffffffu, bad) ? 1 : 0) | (__any_sync(0xffffffffu, beyond) ? 2 : 0) | (__any_sync(0xffffffffu, some) ? 4 : 0);
    if (lane == 0) {
        sums[warp] = a;
        counts[warp] = count;
        bads[warp] = flags;
    }
    // From here on the last warp has the numbers and the first one, beside it, the list.
    const bool numbers = warp == W - 1;
    auto join_block = [&] {
        a = join_warp(lane < W ? sums[lane] : Sums{sums[0].c, 0.f, 0.f});
        count = __reduce_add_sync(0xffffffffu, lane < W ? counts[lane] : 0u);
        flags = __reduce_or_sync(0xffffffffu, lane < W ? bads[lane] : 0u);
    };
    auto finish = [&] {
        double z, entropy;
        if ((flags & 1) || !(flags & 4)) z = entropy = NAN;
        else if ((flags & 2) || a.c < -MOST * LOG2E) sum_64(l, n, lane, z, entropy); // (the pivot is the row's largest or near it)
        else {
            // log2 S from its exponent and, within 2^-24, its mantissa.
            const uint32_t bits = __float_as_uint(a.s);
            const double log2_s = (double)((int)(bits >> 23) - 127) + (double)log2f(__uint_as_float((bits & 0x7FFFFFu) | 0x3F800000u));
            z = ((double)a.c + log2_s) * (1.0 / (double)LOG2E);
            entropy = 0.69314718055994531 * (log2_s - (double)a.t / (double)a.s);
        }
        if (lane == 0) {
            if (out.logprobs) out.logprobs[row] = not_above_0((double)given - z);
            if (out.ranks) out.ranks[row] = id < n ? 1 + count : 0;
            if (out.entropy) out.entropy[row] = entropy < 0.0 ? 0.f : (float)entropy;
            row_z = z;
        }
    };
    uint64_t list = 0;
    if constexpr (TOP) {
        list = best_of<T, NT>(top, notes, at_note, most, shared_by, l, aligned, n, skip, begin, end, k, [&] {
            if (!numbers) return;
            join_block();
            if (parts == 1) finish();
        });
    } else {
        __syncthreads();
        if (numbers) {
            join_block();
            if (parts == 1) finish();
        }
    }
    if (parts > 1) {
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (numbers) {
            if (lane < 3) store_cluster(cluster_address(&all_sums[rank], 0) + 4 * lane, __float_as_uint(lane == 0 ? a.c : lane == 1 ? a.s : a.t));
            if (lane == 3) store_cluster(cluster_address(&all_counts[rank], 0), count);
            if (lane == 4) store_cluster(cluster_address(&all_bads[rank], 0), flags);
        }
        if constexpr (TOP)
            if (warp == 0) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_address(&all_lists[rank][lane], 0)), "l"(list) : "memory");
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
        if (rank != 0) return;
        auto join_cluster = [&] {
            if (!numbers) return;
            a = join_warp(lane < parts ? all_sums[lane] : Sums{all_sums[0].c, 0.f, 0.f}, MAX_CLUSTER);
            a = Sums{__shfl_sync(0xffffffffu, a.c, 0), __shfl_sync(0xffffffffu, a.s, 0), __shfl_sync(0xffffffffu, a.t, 0)};
            count = __reduce_add_sync(0xffffffffu, lane < parts ? all_counts[lane] : 0u);
            flags = __reduce_or_sync(0xffffffffu, lane < parts ? all_bads[lane] : 0u);
            finish();
        };
        if constexpr (TOP) { // what reaches the largest of the lists' k-th keys, put in order by counting
            uint64_t kth = lane < parts ? all_lists[lane][k - 1] : 0;
#pragma unroll
            for (int off = MAX_CLUSTER / 2; off > 0; off /= 2) kth = max(kth, __shfl_xor_sync(0xffffffffu, kth, off));
            kth = __shfl_sync(0xffffffffu, kth, 0);
            if (tid == 0) top.found = 0;
            __syncthreads();
            for (uint32_t p = warp; p < parts; p += W) {
                const uint64_t key = all_lists[p][lane];
                const uint32_t reach = __ballot_sync(0xffffffffu, key != 0 && key >= kth); // a list's first ones
                uint32_t at = 0;
                if (lane == 0) at = atomicAdd(&top.found, __popc(reach));
                at = __shfl_sync(0xffffffffu, at, 0);
                if (reach >> lane & 1) top.keys[at + lane] = key;
            }
            __syncthreads();
            order_pool<NT>(top, top.found, join_cluster);
            list = top.out[lane];
        } else {
            join_cluster();
        }
    }
    if constexpr (TOP)
        if (warp == 0 && lane < k) {
            out.top_ids[(size_t)row * k + lane] = ~(uint32_t)list;
            out.top_logprobs[(size_t)row * k + lane] = not_above_0((double)value_of((uint32_t)(list >> 32)) - row_z);
        }
}

template <typename T, int NT, bool TOP>
cudaError_t launch_shape(fq_device *dev, const T *logits, uint32_t n, size_t stride, uint32_t rows, const uint32_t *ids, uint32_t k, uint32_t parts, const Outputs &out) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * parts);
    cfg.blockDim = dim3(NT);
    const uint32_t pieces = (n + PER_LOAD<T> - 1) / PER_LOAD<T> + 1, tiles = (pieces + parts - 1) / parts / (UNROLL * NT) + 1;
    cfg.dynamicSmemBytes = TOP ? std::min(tiles, NOTES<NT>) * NT * sizeof(float) : 0;
    auto kernel = k_token_logprobs<T, NT, TOP>;
    cfg.stream = dev->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, logits, n, stride, ids, k, parts, out);
}
template <typename T>
cudaError_t launch_rows(fq_device *dev, const T *logits, uint32_t n, size_t stride, uint32_t rows, const uint32_t *ids, uint32_t k, const Outputs &out) {
    const uint32_t sms = (uint32_t)dev->sm_count;
    // A row is cut while four blocks an SM hold all parts and a part keeps 4096 logits.  us with two / four / eight blocks an SM:
    // 64 rows of 151936 F32 without alternatives 14.3 / 10.9 / 10.9, 100 rows 23.5 / 16.2 / 18.0, 200 rows of 32000 bf16 8.0 / 6.5 / 7.7.
    uint32_t parts = 1;
    while (parts < MAX_CLUSTER && rows * (2 * parts) <= 4 * sms && n / (2 * parts) >= 4096) parts *= 2;
    // Blocks that leave half the SMs empty have 512 threads (with 20 alternatives, us with 256 / 512: one row of 151936 F32 10.1 /
    // 9.0, 16 of 32000 8.2 / 7.7; but 18 of 151936 bf16, more clusters of eight such blocks than run at once, 12.6 / 17.4).
    const bool wide = rows * parts <= sms / 2 && n > 8192;
    // Those of short rows 128, which the joins of a row cost less (128 / 256: 2000 rows of 8192 bf16 19.6 / 26.6, 512 of 4096 9.2 /
    // 9.6), and so those of longer whole rows as long as the SMs are filled about as often: eight of them an SM run at once, and
    // take up to a tenth less than four (2048 of 32000 F32 65 / 69, of 100000 163 / 169; 1500 of 65536 F32 104 / 88).  Long bf16
    // rows are faster with their pieces fetched ahead (2048 of 50257 62 / 64, of 100000 98 / 96, 1021 of 151936 79 / 72).
    const uint32_t fills_128 = (rows + 8 * sms - 1) / (8 * sms), fills_256 = (rows + 4 * sms - 1) / (4 * sms);
    const bool narrow = n <= 8192 || ((sizeof(T) == 4 || n <= 65536) && parts == 1 && 18 * fills_128 <= 10 * fills_256);
    auto go = [&](auto top) {
        constexpr bool TOP = decltype(top)::value;
        if (wide) return launch_shape<T, 512, TOP>(dev, logits, n, stride, rows, ids, k, parts, out);
        if (narrow) return launch_shape<T, 128, TOP>(dev, logits, n, stride, rows, ids, k, parts, out);
        return launch_shape<T, 256, TOP>(dev, logits, n, stride, rows, ids, k, parts, out);
    };
    return k ? go(std::true_type{}) : go(std::false_type{});
}

} // namespace

extern "C" int fq_token_logprobs(fq_device *dev, const void *logits, int dtype, uint32_t n, size_t stride, uint32_t rows, const uint32_t *ids,
                                 uint32_t k, float *logprobs, uint32_t *ranks, float *entropy, float *top_logprobs, uint32_t *top_ids) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (dtype != FQ_F32 && dtype != FQ_BF16) return fq_fail(dev, FQ_ERR_UNSUPPORTED, "element type %d", dtype);
    // (A stride whose bytes pass 64 bits would pass the check of the binding too.)
    if (n == 0 || n > 0x7fffffffu || rows == 0 || rows > 0x7fffffffu / MAX_CLUSTER || stride < n || (rows > 1 && stride > (SIZE_MAX >> 4) / (rows - 1)))
        return fq_fail(dev, FQ_ERR_SHAPE, "%u rows of %u logits, %zu apart", rows, n, stride);
    if (k > MAX_TOP || k > n) return fq_fail(dev, FQ_ERR_PARAM, "%u alternatives of %u tokens (at most %u)", k, n, MAX_TOP);
    const size_t bytes = ((size_t)(rows - 1) * stride + n) * fq_dtype_size(dtype);
    if (int rc = fq_check_binding(dev, logits, bytes, "logits", (uint32_t)fq_dtype_size(dtype))) return rc;
    if ((logprobs || ranks) && !ids) return fq_fail(dev, FQ_ERR_PARAM, "log probabilities and ranks are those of given tokens: ids is null");
    struct { const void *p; size_t bytes; const char *name; bool wanted; } out[5] = {
        {logprobs, (size_t)rows * 4, "logprobs", logprobs != nullptr}, {ranks, (size_t)rows * 4, "ranks", ranks != nullptr},
        {entropy, (size_t)rows * 4, "entropy", entropy != nullptr},    {top_logprobs, (size_t)rows * k * 4, "top_logprobs", k != 0},
        {top_ids, (size_t)rows * k * 4, "top_ids", k != 0}};
    if (ids)
        if (int rc = fq_check_binding(dev, ids, (size_t)rows * 4, "ids", 4)) return rc;
    bool any = false;
    for (int i = 0; i < 5; i++) {
        if (!out[i].wanted) continue;
        any = true;
        if (int rc = fq_check_binding(dev, out[i].p, out[i].bytes, out[i].name, 4)) return rc;
        if (int rc = fq_check_apart(dev, out[i].p, out[i].bytes, logits, bytes, out[i].name)) return rc;
        if (int rc = fq_check_apart(dev, out[i].p, out[i].bytes, ids, (size_t)rows * 4, out[i].name)) return rc;
        for (int j = 0; j < i; j++)
            if (out[j].wanted)
                if (int rc = fq_check_apart(dev, out[i].p, out[i].bytes, out[j].p, out[j].bytes, out[i].name)) return rc;
    }
    if (!any) return fq_fail(dev, FQ_ERR_PARAM, "no output is asked for");
    if (int rc = fq_check_input(dev, logits, bytes, "logits")) return rc;
    if (ids)
        if (int rc = fq_check_input(dev, ids, (size_t)rows * 4, "ids")) return rc;
    const Outputs o{logprobs, ranks, entropy, top_logprobs, top_ids};
    const cudaError_t e = dtype == FQ_BF16 ? launch_rows(dev, (const __nv_bfloat16 *)logits, n, stride, rows, ids, k, o)
                                           : launch_rows(dev, (const float *)logits, n, stride, rows, ids, k, o);
    if (int rc = fq_check_cuda(dev, e, "token_logprobs launch")) return rc;
    for (const auto &t : out)
        if (t.wanted) fq_note_write(dev, t.p, t.bytes);
    return fq_end_enqueue(dev, "token_logprobs", 1);
}

// What is said of a token given the output head's logits: the log probability and rank of a given token, the entropy of the
// row's distribution and its most likely tokens.
//
//   z = log sum_j exp(l_j)     logprob = l_id - z     rank = 1 + |{j: l_j > l_id}|     entropy = z - sum_j exp(l_j - z) l_j
//
// A logit of -infinity is a token of probability 0 and adds nothing anywhere.  A row with a NaN, with +infinity or with nothing
// above -infinity has no distribution: its numbers are NaN.
//
// A row is read once, by a block or by a cluster of blocks (each a contiguous part; block 0 collects through distributed shared
// memory).  In powers of two, with b = log2(e) as fp32 has it and a pivot c:
//
//   S = sum 2^(b l - c)     T = sum 2^(b l - c) (b l - c)     z = (c + log2 S) / b     entropy = ln 2 (log2 S - T / S)
//
// b l - c is one FMA with one rounding; c is the largest b l of what the block reads first and moves only when a logit is more
// than 20 / b above it (a term is 2^20 at most, far from fp32's end; a running maximum would rescale every few values).  Dividing by b as
// it is keeps its own rounding out of z.
//
// The most likely tokens: every warp keeps its best 32 as a sorted list, one (value, index) key per lane, and puts a value in
// only if it can still matter: above a bound that k values of the block are known to reach.  The bound starts with what is read
// first -- the k-th largest of some 64 thread maxima, the best of every warp -- so that few values pass it, and rises with the
// lists.  Keys are unique (of equal values the lower index is larger), so the result does not depend on the order of warps.  At
// the end what is left above the bound, little more than k values of all lists, is put in order by counting.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemv_common.cuh"
#include "internal.h"

namespace {
using namespace fqk;

constexpr uint32_t MAX_TOP = 32, MAX_CLUSTER = 8;
constexpr int UNROLL = 4;        // 16-byte loads of a thread in flight
constexpr uint32_t FIRSTS = 64;  // thread maxima that the first bound is taken from
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
// A number below every one whose order is at least `least`, and not below the others by more than a step: NaN where there is none.
__device__ __forceinline__ float just_below(uint32_t least) {
    const uint32_t below = least - 1 == 0x7FFFFFFFu ? 0x7FFFFFFEu : least - 1; // -0 is not below +0
    return least == 0 ? __int_as_float(0x7fc00000) : value_of(below);
}
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
// The best 32 of two sorted lists (descending by lane), sorted.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, const uint64_t *b, uint32_t lane) {
    const uint64_t o = b[31 - lane];
    uint64_t c = a > o ? a : o;
#pragma unroll 1
    for (int off = 16; off > 0; off >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, c, off);
        if ((other > c) == ((lane & off) == 0)) c = other;
    }
    return c;
}

// A row of logits around numbers beyond MOST: by one warp, in 64 bits about its largest.
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

// Block `rank` of the `parts` of row blockIdx.x / parts.
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT)
k_token_logprobs(const T *logits, uint32_t n, size_t stride, const uint32_t *ids, uint32_t k, uint32_t parts, Outputs out) {
    constexpr int W = NT / 32, V = PER_LOAD<T>;
    __shared__ uint32_t first_max[W], bound, left;
    __shared__ uint4 firsts[FIRSTS / 4];
    __shared__ Sums sums[W];
    __shared__ uint32_t counts[W], bads[W];
    __shared__ uint64_t keys[TOP ? NT : 1], list_out[32];
    // Of block 0: what the blocks of the cluster found.
    __shared__ Sums all_sums[MAX_CLUSTER];
    __shared__ uint32_t all_counts[MAX_CLUSTER], all_bads[MAX_CLUSTER];
    __shared__ uint64_t all_lists[TOP ? MAX_CLUSTER : 1][32];
    // Block 0's shared memory may be written once all blocks of the cluster run: arrived here, waited for before the writes.
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    pdl_trigger();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / parts, rank = blockIdx.x - row * parts;
    if (tid == 0) bound = left = 0;
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
    uint4 now[UNROLL];
    // This thread's UNROLL pieces of the block's UNROLL * NT from j0 on.
    auto fetch = [&](uint32_t j0) {
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
    fetch(begin);
    const float given = id < n ? load1(l, id) : __int_as_float(0x7fc00000);

    // What is read first gives the pivot and a bound that k values of the block reach.
    uint32_t best = begin + tid < end ? order_of(largest<T>(now)) : 0; // (a thread with a NaN does not count)
    const uint32_t warps = min((uint32_t)W, (end - begin + 31) / 32); // with something to read
    uint32_t high = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) first_max[warp] = high;
    if constexpr (TOP) {
        const uint32_t m = min(32u, FIRSTS / max(warps, 1u)); // of every warp, m * warps >= k
        uint32_t *mine = reinterpret_cast<uint32_t *>(firsts) + warp * m;
        if (warp < warps) {
#pragma unroll 1
            for (uint32_t i = 0; i < m; i++) {
                if (lane == 0) mine[i] = high;
                const uint32_t holders = __ballot_sync(0xffffffffu, best == high);
                if (lane == (uint32_t)__ffs(holders) - 1) best = 0;
                high = __reduce_max_sync(0xffffffffu, best);
            }
        }
        for (uint32_t i = m * warps + tid; i < FIRSTS; i += NT) reinterpret_cast<uint32_t *>(firsts)[i] = 0;
    }
    __syncthreads();
    const float top = value_of(max(__reduce_max_sync(0xffffffffu, first_max[lane % W]), 1u << 23)); // the lowest number where there is nothing (or NaN)
    Sums a{fmaxf(top, LEAST) * LOG2E, 0.f, 0.f};
    float limit = fminf(fmaf(SLACK, 1.f / LOG2E, fmaxf(top, LEAST)), MOST); // logits above it move the pivot
    uint32_t least = 0; // values of a lower order do not matter any more; 0: all do
    if constexpr (TOP) { // the least of those that fewer than k are above
        const uint32_t x = reinterpret_cast<const uint32_t *>(firsts)[lane], y = reinterpret_cast<const uint32_t *>(firsts)[lane + 32];
        uint32_t above_x = 0, above_y = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < FIRSTS / 4; i++) {
            const uint4 f = firsts[i];
            above_x += (f.x > x) + (f.y > x) + (f.z > x) + (f.w > x);
            above_y += (f.x > y) + (f.y > y) + (f.z > y) + (f.w > y);
        }
        least = __reduce_min_sync(0xffffffffu, min(above_x < k ? x : 0xFFFFFFFFu, above_y < k ? y : 0xFFFFFFFFu));
        if (tid == 0) atomicMax(&bound, least);
    }
    float below = just_below(least);
    bool bad = false, beyond = false, some = false; // a NaN or +infinity; a logit above MOST; one above -infinity
    uint32_t count = 0;
    uint64_t list = 0;
    float2 s2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);

#pragma unroll 1
    for (uint32_t j0 = begin; j0 < end; j0 += UNROLL * NT) {
        const float highest = largest<T>(now);
        if constexpr (TOP)
            if (__any_sync(0xffffffffu, !(highest <= below))) { // some pieces are looked into, in the order of their indexes
                least = max(least, *(volatile uint32_t *)&bound);
#pragma unroll 1
                for (int u = 0; u < UNROLL; u++) {
                    const uint4 own[1] = {u == 0 ? now[0] : u == 1 ? now[1] : u == 2 ? now[2] : now[3]};
                    uint32_t vote = __ballot_sync(0xffffffffu, !(largest<T>(own) <= below) && j0 + u * NT + tid < end);
#pragma unroll 1
                    while (vote) {
                        const uint32_t src = __ffs(vote) - 1, first = (j0 + u * NT + 32 * warp + src) * V - skip;
                        vote &= vote - 1;
                        const uint4 piece = make_uint4(__shfl_sync(0xffffffffu, own[0].x, src), __shfl_sync(0xffffffffu, own[0].y, src),
                                                       __shfl_sync(0xffffffffu, own[0].z, src), __shfl_sync(0xffffffffu, own[0].w, src));
                        // Lane i looks at value i; those that may matter go in one after the other.
                        const uint32_t i = lane % V, w = word(piece, sizeof(T) == 2 ? i / 2 : i), at = first + i;
                        const uint32_t order = order_of(sizeof(T) == 4 ? __uint_as_float(w) : (i & 1) ? high_half(w) : low_half(w));
                        uint32_t fit = __ballot_sync(0xffffffffu, lane < V && at < n && order >= least);
#pragma unroll 1
                        while (fit) {
                            const uint64_t key = __shfl_sync(0xffffffffu, key_of(order, at), __ffs(fit) - 1);
                            fit &= fit - 1;
                            if ((uint32_t)(key >> 32) < least) continue; // (uniform)
                            const uint32_t pos = __popc(__ballot_sync(0xffffffffu, list > key));
                            const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
                            if (lane >= pos) list = lane == pos ? key : up;
                            const uint64_t kth = __shfl_sync(0xffffffffu, list, k - 1);
                            if (kth) least = max(least, (uint32_t)(kth >> 32) + 1); // later values have higher indexes
                        }
                    }
                }
                if (lane == k - 1 && list) atomicMax(&bound, (uint32_t)(list >> 32));
                below = just_below(least);
            }
        if (!(highest <= given)) {
            if constexpr (sizeof(T) == 2) { // ones added in bf16: 4 * UNROLL at most
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
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                const float2 d = fma2(pair_from_least<T>(now[u], i), b2, c2);
                const float2 e = make_float2(exp2_fast(d.x), exp2_fast(d.y));
                s2 = add2(s2, e);
                t2 = fma2(d, e, t2);
            }
        if (j0 + UNROLL * NT < end) fetch(j0 + UNROLL * NT);
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
    __syncthreads();
    if constexpr (TOP) {
        const uint32_t kept = __ballot_sync(0xffffffffu, list != 0 && (uint32_t)(list >> 32) >= bound); // a list's first ones
        uint32_t at = 0;
        if (lane == 0 && kept) at = atomicAdd(&left, __popc(kept));
        at = __shfl_sync(0xffffffffu, at, 0);
        if (kept >> lane & 1) keys[at + lane] = list;
    }
    if (warp == 0) {
        a = join_warp(lane < W ? sums[lane] : Sums{sums[0].c, 0.f, 0.f});
        count = __reduce_add_sync(0xffffffffu, lane < W ? counts[lane] : 0u);
        flags = __reduce_or_sync(0xffffffffu, lane < W ? bads[lane] : 0u);
        if constexpr (TOP) list_out[lane] = 0;
    }
    if constexpr (TOP) {
        __syncthreads();
        const uint32_t total = left;
        if (tid < total) {
            const uint64_t mine = keys[tid];
            uint32_t above = 0;
#pragma unroll 4
            for (uint32_t i = 0; i < total; i++) above += keys[i] > mine;
            if (above < 32) list_out[above] = mine;
        }
        __syncthreads();
        if (warp == 0) list = list_out[lane];
    }
    if (parts > 1) {
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (warp == 0) {
            if (lane < 3) store_cluster(cluster_address(&all_sums[rank], 0) + 4 * lane, __float_as_uint(lane == 0 ? a.c : lane == 1 ? a.s : a.t));
            if (lane == 3) store_cluster(cluster_address(&all_counts[rank], 0), count);
            if (lane == 4) store_cluster(cluster_address(&all_bads[rank], 0), flags);
            if constexpr (TOP) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_address(&all_lists[rank][lane], 0)), "l"(list) : "memory");
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
        if (rank != 0) return;
        if (warp == 0) {
            a = join_warp(lane < parts ? all_sums[lane] : Sums{all_sums[0].c, 0.f, 0.f}, MAX_CLUSTER);
            a = Sums{__shfl_sync(0xffffffffu, a.c, 0), __shfl_sync(0xffffffffu, a.s, 0), __shfl_sync(0xffffffffu, a.t, 0)};
            count = __reduce_add_sync(0xffffffffu, lane < parts ? all_counts[lane] : 0u);
            flags = __reduce_or_sync(0xffffffffu, lane < parts ? all_bads[lane] : 0u);
        }
        if constexpr (TOP)
#pragma unroll 1
            for (uint32_t half = parts / 2; half > 0; half /= 2) { // (parts is a power of two)
                if (warp < half) all_lists[warp][lane] = list = merge_lists(all_lists[warp][lane], all_lists[warp + half], lane);
                __syncthreads();
            }
    }
    if (warp != 0) return;
    double z, entropy;
    if ((flags & 1) || !(flags & 4)) z = entropy = NAN;
    else if ((flags & 2) || a.c < -MOST * LOG2E) sum_64(l, n, lane, z, entropy); // (the pivot is the row's largest or near it)
    else {
        const double log2_s = log2((double)a.s);
        z = ((double)a.c + log2_s) / (double)LOG2E;
        entropy = 0.69314718055994531 * (log2_s - (double)a.t / (double)a.s);
    }
    if (lane == 0) {
        if (out.logprobs) out.logprobs[row] = (float)((double)given - z);
        if (out.ranks) out.ranks[row] = id < n ? 1 + count : 0;
        if (out.entropy) out.entropy[row] = (float)entropy;
    }
    if constexpr (TOP)
        if (lane < k) {
            out.top_ids[(size_t)row * k + lane] = ~(uint32_t)list;
            out.top_logprobs[(size_t)row * k + lane] = (float)((double)value_of((uint32_t)(list >> 32)) - z);
        }
}

template <typename T, int NT, bool TOP>
cudaError_t launch_shape(fq_device *dev, const T *logits, uint32_t n, size_t stride, uint32_t rows, const uint32_t *ids, uint32_t k, uint32_t parts, const Outputs &out) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * parts);
    cfg.blockDim = dim3(NT);
    cfg.stream = dev->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k_token_logprobs<T, NT, TOP>, logits, n, stride, ids, k, parts, out);
}
template <typename T>
cudaError_t launch_rows(fq_device *dev, const T *logits, uint32_t n, size_t stride, uint32_t rows, const uint32_t *ids, uint32_t k, const Outputs &out) {
    const uint32_t sms = (uint32_t)dev->sm_count;
    const bool wide = rows * MAX_CLUSTER <= sms && n > 8192; // a few rows: as many threads as there can be
    uint32_t parts = 1;
    while (parts < MAX_CLUSTER && (wide || rows * (2 * parts) <= 4 * sms) && n / (2 * parts) >= 4096) parts *= 2;
    auto go = [&](auto top) {
        constexpr bool TOP = decltype(top)::value;
        if (wide) return launch_shape<T, 512, TOP>(dev, logits, n, stride, rows, ids, k, parts, out);
        if (n > 8192) return launch_shape<T, 256, TOP>(dev, logits, n, stride, rows, ids, k, parts, out);
        return launch_shape<T, 128, TOP>(dev, logits, n, stride, rows, ids, k, parts, out);
    };
    return k ? go(std::true_type{}) : go(std::false_type{});
}

} // namespace

extern "C" int fq_token_logprobs(fq_device *dev, const void *logits, int dtype, uint32_t n, size_t stride, uint32_t rows, const uint32_t *ids,
                                 uint32_t k, float *logprobs, uint32_t *ranks, float *entropy, float *top_logprobs, uint32_t *top_ids) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (dtype != FQ_F32 && dtype != FQ_BF16) return fq_fail(dev, FQ_ERR_UNSUPPORTED, "element type %d", dtype);
    if (n == 0 || n > 0x7fffffffu || rows == 0 || rows > 0x7fffffffu / MAX_CLUSTER || stride < n) return fq_fail(dev, FQ_ERR_SHAPE, "%u rows of %u logits, %zu apart", rows, n, stride);
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
        if (int rc = fq_check_no_alias(dev, out[i].p, out[i].bytes, logits, bytes, out[i].name)) return rc;
        if (int rc = fq_check_no_alias(dev, out[i].p, out[i].bytes, ids, (size_t)rows * 4, out[i].name)) return rc;
        for (int j = 0; j < i; j++)
            if (out[j].wanted)
                if (int rc = fq_check_no_alias(dev, out[i].p, out[i].bytes, out[j].p, out[j].bytes, out[i].name)) return rc;
    }
    if (!any) return fq_fail(dev, FQ_ERR_PARAM, "no output is asked for");
    const Outputs o{logprobs, ranks, entropy, top_logprobs, top_ids};
    const cudaError_t e = dtype == FQ_BF16 ? launch_rows(dev, (const __nv_bfloat16 *)logits, n, stride, rows, ids, k, o)
                                           : launch_rows(dev, (const float *)logits, n, stride, rows, ids, k, o);
    if (int rc = fq_check_cuda(dev, e, "token_logprobs launch")) return rc;
    return fq_end_enqueue(dev, "token_logprobs", 1);
}

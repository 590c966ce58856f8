// What is said of a token given the output head's logits: the log probability and rank of a given token, the entropy of the
// row's distribution and its most likely tokens.
//
//   z = log sum_j exp(l_j)     logprob = l_id - z     rank = 1 + |{j: l_j > l_id}|     entropy = z - sum_j exp(l_j - z) l_j
//
// A logit of -infinity is a token of probability 0 and adds nothing anywhere.  A row with a NaN, with +infinity or with nothing
// above -infinity has no distribution: its numbers are NaN.
//
// A row is read once, by a block or by a cluster of up to eight (each a contiguous part; block 0 collects through distributed
// shared memory).  Per thread: S = sum exp(l - p) and T = sum exp(l - p)(l - p) with a pivot p, the largest logit of what the
// block reads first, moved only when a logit is more than 20 above it (S grows to e^20 per term at most, far from fp32's end;
// a running maximum would rescale every few values).  log S and T / S at the end give z = p + log S and the entropy log S - T / S.
//
// The most likely tokens: every warp keeps its best 32 as a sorted list, one (value, index) key per lane, and puts a value in
// only if it can still matter: above a bound that k values of the block are known to reach.  The bound starts with what is read
// first -- each warp's m-th largest thread maximum, m * warps >= k, and of these the least -- so that few values pass it, and
// rises with the lists.  Keys are unique (of equal values the lower index is larger), so the result does not depend on order.
#include <algorithm>
#include <cmath>

#include "gemv_common.cuh"
#include "internal.h"

namespace {
using namespace fqk;

constexpr uint32_t MAX_TOP = 32, MAX_CLUSTER = 8;
constexpr int UNROLL = 4; // 16-byte loads of a thread in flight

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

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp_fast(float d) { // 2^-22 of itself; 0 below 2^-126
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.44269504f));
    return r;
}

template <typename T> constexpr int PER_LOAD = 16 / (int)sizeof(T);
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

struct Sums {
    float p, s, t; // pivot, sum exp(l - p), sum exp(l - p)(l - p)
};
// The sums about another pivot.
__device__ __forceinline__ void move_pivot(Sums &a, float p) {
    const float f = exp_fast(a.p - p);
    // f = 0: nothing is left of them (and a.p - p may be -infinity)
    a.t = f > 0.f ? f * fmaf(a.p - p, a.s, a.t) : 0.f;
    a.s = f * a.s;
    a.p = p;
}
__device__ __forceinline__ void join(Sums &a, Sums b) {
    const float p = fmaxf(a.p, b.p);
    if (a.p != p) move_pivot(a, p);
    if (b.p != p) move_pivot(b, p);
    a.s += b.s;
    a.t += b.t;
}
__device__ __forceinline__ Sums join_warp(Sums a) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const Sums b{__shfl_xor_sync(0xffffffffu, a.p, off), __shfl_xor_sync(0xffffffffu, a.s, off), __shfl_xor_sync(0xffffffffu, a.t, off)};
        join(a, b);
    }
    return a;
}
// The best 32 of two sorted lists (descending by lane), sorted.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, const uint64_t *b, uint32_t lane) {
    const uint64_t o = b[31 - lane];
    uint64_t c = a > o ? a : o;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, c, off);
        if ((other > c) == ((lane & off) == 0)) c = other;
    }
    return c;
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

// Block `rank` of the `parts` of row blockIdx.x / parts.
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT)
k_token_logprobs(const T *logits, uint32_t n, size_t stride, const uint32_t *ids, uint32_t k, uint32_t parts, Outputs out) {
    constexpr int W = NT / 32, V = PER_LOAD<T>;
    __shared__ uint32_t first_max[W], first_bound[W], bound;
    __shared__ Sums sums[W];
    __shared__ uint32_t counts[W], bads[W];
    __shared__ uint64_t lists[TOP ? W : 1][32];
    // Of block 0: what the blocks of the cluster found.
    __shared__ Sums all_sums[MAX_CLUSTER];
    __shared__ uint32_t all_counts[MAX_CLUSTER], all_bads[MAX_CLUSTER];
    __shared__ uint64_t all_lists[TOP ? MAX_CLUSTER : 1][32];
    // Block 0's shared memory may be written once all blocks of the cluster run: arrived here, waited for before the writes.
    if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    pdl_trigger();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / parts, rank = blockIdx.x - row * parts;
    if (tid == 0) bound = 0;
    pdl_wait();
    // The row in whole 16-byte pieces from the boundary below its start: piece j holds elements j * V - skip ...
    const T *l = logits + (size_t)row * stride;
    const uint32_t skip = (uint32_t)(((uintptr_t)l & 15) / sizeof(T));
    const T *aligned = l - skip;
    const uint32_t pieces = (uint32_t)(((uint64_t)skip + n + V - 1) / V), per = (pieces + parts - 1) / parts;
    const uint32_t begin = min(rank * per, pieces), end = min(begin + per, pieces);
    const uint32_t id = ids ? __ldcg(ids + row) : n;
    const float none = -INFINITY;
    auto load = [&](uint32_t j, uint4 &u) {
        const uint32_t first = j * V - skip; // wraps in the piece that begins before the row
        if (first <= n && n - first >= (uint32_t)V) {
            u = __ldcg(reinterpret_cast<const uint4 *>(aligned) + j);
        } else { // the row's ends: elements one at a time, -infinity outside
            T e[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                const uint32_t at = first + i;
                if constexpr (sizeof(T) == 2) e[i] = __ushort_as_bfloat16(at < n ? __ldcg(reinterpret_cast<const unsigned short *>(l) + at) : 0xFF80u);
                else e[i] = at < n ? __ldcg(l + at) : none;
            }
            u = *reinterpret_cast<const uint4 *>(e);
        }
    };
    uint4 next[UNROLL];
    auto fetch = [&](uint32_t j0) {
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
            if (j0 + u * NT < end) load(j0 + u * NT, next[u]);
    };
    fetch(begin + tid);
    const float given = id < n ? (sizeof(T) == 2 ? __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(l) + id) << 16)
                                                 : __ldcg(reinterpret_cast<const float *>(l) + id))
                               : __int_as_float(0x7fc00000);

    // What is read first gives the pivot and a bound that k values of the block reach.
    uint32_t best = 0;
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
        if (begin + tid + u * NT < end) {
            float v[V];
            unpack(next[u], v);
#pragma unroll
            for (int i = 0; i < V; i++) best = max(best, order_of(v[i]));
        }
    const uint32_t warps = min((uint32_t)W, (end - begin + 31) / 32); // with something to read
    uint32_t high = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) first_max[warp] = high;
    if constexpr (TOP) {
        const uint32_t m = warps ? (k + warps - 1) / warps : 1; // this warp's m-th largest maximum
        uint32_t mine = best;
        for (uint32_t i = 1; i < m; i++) {
            const uint32_t holders = __ballot_sync(0xffffffffu, mine == high && mine != 0);
            if (holders && lane == (uint32_t)__ffs(holders) - 1) mine = 0;
            high = __reduce_max_sync(0xffffffffu, mine);
        }
        if (lane == 0) first_bound[warp] = high;
    }
    __syncthreads();
    Sums a{0.f, 0.f, 0.f};
    uint32_t least = 0; // values of a lower order do not matter any more; 0: all do
    {
        const uint32_t top = __reduce_max_sync(0xffffffffu, first_max[lane < W ? lane : 0]);
        a.p = top > order_of(-INFINITY) ? value_of(top) : -3.402823466e38f;
        if constexpr (TOP) least = __reduce_min_sync(0xffffffffu, lane < warps ? first_bound[lane] : 0xFFFFFFFFu);
    }
    bool bad = a.p == INFINITY;
    float limit = a.p + 20.f, below = just_below(least);
    uint32_t count = 0;
    uint64_t list = 0;

    auto take = [&](const uint4 &u, uint32_t j, bool live) {
        float v[V];
        unpack(u, v);
        float mx = v[0];
#pragma unroll
        for (int i = 1; i < V; i++) mx = max_nan(mx, v[i]);
        if (!live) mx = none;
        if constexpr (TOP) {
            uint32_t vote = __ballot_sync(0xffffffffu, live && !(mx <= below));
            if (vote) {
                while (vote) { // values in the order of their indexes
                    const uint32_t src = __ffs(vote) - 1, at = __shfl_sync(0xffffffffu, j, src) * V - skip;
                    vote &= vote - 1;
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const uint32_t order = order_of(__shfl_sync(0xffffffffu, v[i], src));
                        if (order < least || at + i >= n) continue; // uniform
                        const uint64_t key = key_of(order, at + i);
                        const uint32_t pos = __popc(__ballot_sync(0xffffffffu, list > key));
                        const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
                        if (lane >= pos) list = lane == pos ? key : up;
                        const uint64_t kth = __shfl_sync(0xffffffffu, list, k - 1);
                        if (kth) least = max(least, (uint32_t)(kth >> 32) + 1); // later values have higher indexes
                    }
                }
                if (lane == k - 1 && list) atomicMax(&bound, (uint32_t)(list >> 32));
                below = just_below(least);
            }
        }
        if (!live) return;
        if (!(mx <= given))
#pragma unroll
            for (int i = 0; i < V; i++) count += v[i] > given;
        if (!(mx <= limit)) {
            float high = none;
#pragma unroll
            for (int i = 0; i < V; i++) {
                bad |= v[i] != v[i];
                high = fmaxf(high, v[i]);
            }
            bad |= high == INFINITY;
            if (high > limit && !bad) {
                move_pivot(a, high);
                limit = high + 20.f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float d = fmaxf(v[i] - a.p, -200.f); // e^-200 is 0, and so is what -infinity adds to T
            const float e = exp_fast(d);
            a.s += e;
            a.t = fmaf(d, e, a.t);
        }
    };
    for (uint32_t j0 = begin; j0 < end; j0 += UNROLL * NT) {
        uint4 now[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) now[u] = next[u];
        fetch(j0 + UNROLL * NT + tid);
        if constexpr (TOP) {
            const uint32_t shared = *(volatile uint32_t *)&bound;
            if (shared > least) {
                least = shared;
                below = just_below(least);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) take(now[u], j0 + tid + u * NT, j0 + tid + u * NT < end);
    }

    // The block's sums and list, then the cluster's.
    a = join_warp(a);
    count = __reduce_add_sync(0xffffffffu, count);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
        sums[warp] = a;
        counts[warp] = count;
        bads[warp] = bad;
    }
    if constexpr (TOP) {
        lists[warp][lane] = list;
#pragma unroll
        for (int half = W / 2; half > 0; half >>= 1) {
            __syncthreads();
            if (warp < (uint32_t)half) lists[warp][lane] = list = merge_lists(list, lists[warp + half], lane);
        }
    }
    __syncthreads();
    if (parts > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (warp == 0) {
        a = join_warp(lane < W ? sums[lane] : Sums{-3.402823466e38f, 0.f, 0.f});
        count = __reduce_add_sync(0xffffffffu, lane < W ? counts[lane] : 0u);
        bad = __any_sync(0xffffffffu, lane < W && bads[lane]);
        if (parts > 1) {
            if (lane == 0) {
                const uint32_t to = cluster_address(&all_sums[rank], 0);
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(a.p) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(a.s) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(a.t) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_address(&all_counts[rank], 0)), "r"(count) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_address(&all_bads[rank], 0)), "r"((uint32_t)bad) : "memory");
            }
            if constexpr (TOP) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_address(&all_lists[rank][lane], 0)), "l"(list) : "memory");
        }
    }
    if (parts > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
        if (rank != 0 || warp != 0) return;
        a = join_warp(lane < parts ? all_sums[lane] : Sums{-3.402823466e38f, 0.f, 0.f});
        count = __reduce_add_sync(0xffffffffu, lane < parts ? all_counts[lane] : 0u);
        bad = __any_sync(0xffffffffu, lane < parts && all_bads[lane]);
        if constexpr (TOP)
            for (uint32_t i = 1; i < parts; i++) list = merge_lists(list, all_lists[i], lane);
    }
    if (warp != 0) return;
    bad |= !(a.s > 0.f); // nothing above -infinity
    const double log_s = bad ? NAN : log((double)a.s);
    const double p = a.p;
    if (lane == 0) {
        if (out.logprobs) out.logprobs[row] = (float)((double)given - p - log_s);
        if (out.ranks) out.ranks[row] = id < n ? 1 + count : 0;
        if (out.entropy) out.entropy[row] = (float)(log_s - (double)a.t / (double)a.s);
    }
    if constexpr (TOP)
        if (lane < k) {
            out.top_ids[(size_t)row * k + lane] = ~(uint32_t)list;
            out.top_logprobs[(size_t)row * k + lane] = (float)((double)value_of((uint32_t)(list >> 32)) - p - log_s);
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
    uint32_t parts = 1;
    while (parts < MAX_CLUSTER && rows * (2 * parts) <= 2 * (uint32_t)dev->sm_count && n / (2 * parts) >= 4096) parts *= 2;
    if (n <= 8192) return k ? launch_shape<T, 128, true>(dev, logits, n, stride, rows, ids, k, parts, out) : launch_shape<T, 128, false>(dev, logits, n, stride, rows, ids, k, parts, out);
    return k ? launch_shape<T, 512, true>(dev, logits, n, stride, rows, ids, k, parts, out) : launch_shape<T, 512, false>(dev, logits, n, stride, rows, ids, k, parts, out);
}

} // namespace

extern "C" int fq_token_logprobs(fq_device *dev, const void *logits, int dtype, uint32_t n, size_t stride, uint32_t rows, const uint32_t *ids,
                                 uint32_t k, float *logprobs, uint32_t *ranks, float *entropy, float *top_logprobs, uint32_t *top_ids) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (dtype != FQ_F32 && dtype != FQ_BF16) return fq_fail(dev, FQ_ERR_UNSUPPORTED, "element type %d", dtype);
    if (n == 0 || rows == 0 || rows > 0x7fffffffu || stride < n) return fq_fail(dev, FQ_ERR_SHAPE, "%u rows of %u logits, %zu apart", rows, n, stride);
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

// What is said of a token given the output head's logits: the log probability and rank of a given token, the entropy of the
// row's distribution and its most likely tokens.
//
//   z = log sum_j exp(l_j)     logprob = l_id - z     rank = 1 + |{j: l_j > l_id}|     entropy = z - sum_j exp(l_j - z) l_j
//
// A logit of -infinity is a token of probability 0 and adds nothing anywhere.  A row with a NaN, with +infinity or with nothing
// above -infinity has no distribution: its numbers are NaN.
#include <cmath>

#include "gemv_common.cuh"
#include "internal.h"

namespace {

constexpr uint32_t MAX_TOP = 32;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// (value, index) as one number that is larger for the larger value and, of equal values, for the lower index.  NaN is below
// everything, and the two zeros are one value.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v + 0.f);
    const uint32_t order = v != v ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (uint64_t)order << 32 | (uint32_t)~i;
}

// One block per row; the row is read for its maximum, for its sums and once per alternative.
template <typename T>
__global__ void __launch_bounds__(256)
k_token_logprobs(const T *logits, uint32_t n, size_t stride, const uint32_t *ids, uint32_t k, float *logprobs, uint32_t *ranks, float *entropy,
                 float *top_logprobs, uint32_t *top_ids) {
    __shared__ double part[8], part2[8];
    __shared__ uint64_t keys[8];
    __shared__ uint32_t above;
    const T *l = logits + (size_t)blockIdx.x * stride;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) above = 0;
    float mx = -INFINITY;
    bool nan = false;
    for (uint32_t i = tid; i < n; i += 256) {
        const float v = to_float(l[i]);
        mx = fmaxf(mx, v);
        nan |= v != v;
    }
    for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    if (lane == 0) part[warp] = mx;
    nan = __syncthreads_or(nan);
    for (int i = 0; i < 8; i++) mx = fmaxf(mx, (float)part[i]);
    __syncthreads();
    const uint32_t id = ids ? ids[blockIdx.x] : n;
    const float given = id < n ? to_float(l[id]) : NAN;
    double s = 0.0, t = 0.0;
    uint32_t count = 0;
    for (uint32_t i = tid; i < n; i += 256) {
        const float v = to_float(l[i]);
        if (v > -INFINITY) {
            const double d = (double)v - (double)mx, e = exp(d);
            s += e;
            t += e > 0.0 ? d * e : 0.0;
        }
        count += v > given;
    }
    atomicAdd(&above, count);
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off), t += __shfl_xor_sync(0xffffffffu, t, off);
    if (lane == 0) part[warp] = s, part2[warp] = t;
    __syncthreads();
    s = t = 0.0;
    for (int i = 0; i < 8; i++) s += part[i], t += part2[i];
    const bool none = nan || !(fabsf(mx) < INFINITY);
    const double z = none ? NAN : (double)mx + log(s);
    if (tid == 0) {
        if (ids && logprobs) logprobs[blockIdx.x] = (float)((double)given - z);
        if (ids && ranks) ranks[blockIdx.x] = id < n ? 1 + above : 0;
        if (entropy) entropy[blockIdx.x] = (float)(none ? NAN : log(s) - t / s);
    }
    uint64_t last = ~0ull;
    for (uint32_t j = 0; j < k; j++) {
        uint64_t best = 0;
        for (uint32_t i = tid; i < n; i += 256) {
            const uint64_t key = key_of(to_float(l[i]), i);
            if (key < last && key > best) best = key;
        }
        for (int off = 16; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor_sync(0xffffffffu, best, off);
            best = o > best ? o : best;
        }
        __syncthreads();
        if (lane == 0) keys[warp] = best;
        __syncthreads();
        for (int i = 0; i < 8; i++) best = keys[i] > best ? keys[i] : best;
        last = best;
        if (tid == 0) {
            const uint32_t at = ~(uint32_t)best;
            top_ids[(size_t)blockIdx.x * k + j] = at;
            top_logprobs[(size_t)blockIdx.x * k + j] = (float)((double)to_float(l[at]) - z);
        }
    }
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
    if (dtype == FQ_BF16)
        k_token_logprobs<<<rows, 256, 0, dev->stream>>>((const __nv_bfloat16 *)logits, n, stride, ids, k, logprobs, ranks, entropy, top_logprobs, top_ids);
    else k_token_logprobs<<<rows, 256, 0, dev->stream>>>((const float *)logits, n, stride, ids, k, logprobs, ranks, entropy, top_logprobs, top_ids);
    return fq_end_enqueue(dev, "token_logprobs", 1);
}

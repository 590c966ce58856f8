// Rows of activations as 8-bit integers with one scale per row, the inputs of the 8-bit projections: a row as it is
// (`fq_quantize_i8`), normalised, with the residual's addition or without (`fq_rmsnorm_i8`, `fq_add_rmsnorm_i8`), or the
// gated unit of two rows (`fq_glu_i8`).
//
//   v_i = x_i | h_i w_i | silu(g_i) u_i        a = max_i |v_i|        q_i = round(127 v_i / a)        scale = a c / 127
//
// with c = 1 / sqrt(mean h^2 + eps) for the norms and 1 otherwise: 1/rms is common to a row and cancels in q.  Rounding is
// to the nearest whole number, ties to even, of the exact quotient: the 8-bit values do not depend on how a row is spread
// over threads.
//
// A row is read once and stays in registers.  v is computed in 32 bits; the few values that decide are taken again in 64: those
// that may be the row's largest, and those whose quotient lies within the error of 32 bits of the border between two whole
// numbers (one in twelve thousand; of a gated unit one in five thousand).  The sum of squares is held in 64 bits: it costs a
// conversion and an FMA a value, where memory leaves time for some fifty instructions.
#include <type_traits>

#include "gemv_common.cuh"
#include "internal.h"

namespace {
using namespace fqk;

enum Op { PLAIN, NORM, ADD_NORM, GLU };

// Four values at a time.
__device__ __forceinline__ float4 load4(const float *p) { return __ldcg(reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 b = __ldcg(reinterpret_cast<const uint2 *>(p));
    return make_float4(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xFFFF0000u), __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xFFFF0000u));
}
// a + b as it is kept.
__device__ __forceinline__ float4 sum4(const float *, const float4 &a, const float4 &b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ float4 sum4(const __nv_bfloat16 *, const float4 &a, const float4 &b) {
    const float4 s = sum4((const float *)nullptr, a, b);
    auto keep = [](float v) { return __bfloat162float(__float2bfloat16_rn(v)); };
    return make_float4(keep(s.x), keep(s.y), keep(s.z), keep(s.w));
}
__device__ __forceinline__ void store4(float *p, const float4 &v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float4 &v) { // values that are bf16 already
    *reinterpret_cast<uint2 *>(p) = make_uint2(__byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632), __byte_perm(__float_as_uint(v.z), __float_as_uint(v.w), 0x7632));
}
__device__ __forceinline__ float load1(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float load1(const __nv_bfloat16 *p) { return __bfloat162float(__ushort_as_bfloat16(__ldcg(reinterpret_cast<const unsigned short *>(p)))); }
__device__ __forceinline__ float part(const float4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// silu(g) u: within 4.5 * 2^-23 of itself (2 steps of the exponential, and four roundings) while e^-g does not overflow, and
// within 2^-100 of |u| beyond.
__device__ __forceinline__ float gated(float g, float u) { return g / (1.f + expf(-g)) * u; }
__device__ __forceinline__ double gated64(double g, double u) { return g / (1.0 + exp(-g)) * u; }

// Where a row leaves these, 64 bits are used throughout: the smallest and largest |v| of a row's maximum, so that what 32 bits
// lose to underflow is nothing beside it, and for the gated unit the largest |u|, for what `gated` loses of a closed gate.
constexpr float LEAST = 1e-20f, MOST = 1e37f, MOST_UP = 1048576.f;
// How far 127 v / a in 32 bits may be from the exact quotient: 127 times 1.5 * 2^-23 of v, 127 / a and their product, and
// for the gated unit 4 * 2^-23 more.
template <int OP> constexpr float NEAR = OP == GLU ? 1e-4f : 4e-5f;
// How many steps of fp32 the exact largest value may be below the largest fp32 one: products are rounded once, which keeps
// their order; a gated unit is off by 9 half steps, and so is the largest.
template <int OP> constexpr uint32_t BELOW = OP == GLU ? 12 : 0;

// WPR warps per row, a block per row (eight rows with one warp each).  A thread holds CACHED float4s of the row's values; what
// lies beyond them in longer rows is read again for every step.
template <int OP, typename T, int WPR, int CACHED>
__global__ void __launch_bounds__(WPR == 1 ? 256 : WPR * 32)
k_rows_i8(const T *x, const T *r, const float *w, uint32_t n, float eps, uint32_t rows, T *h, int8_t *q, float *scales) {
    constexpr bool IS_NORM = OP == NORM || OP == ADD_NORM;
    __shared__ double part_ss[WPR];
    __shared__ uint32_t part_max[WPR], part_up[WPR];
    __shared__ unsigned long long most64;
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 31, warp = WPR == 1 ? 0 : threadIdx.x >> 5, tid = 32 * warp + lane;
    const uint32_t row = WPR == 1 ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x, n4 = n / 4;
    if (WPR > 1 && threadIdx.x == 0) most64 = 0;
    pdl_wait();
    if (row >= rows) return; // whole warps
    const size_t base = (size_t)row * n;
    x += base;
    if constexpr (OP == ADD_NORM || OP == GLU) r += base;
    if constexpr (OP == ADD_NORM) h += base;
    q += base;
    constexpr uint32_t STEP = WPR * 32;

    // The row: for the norms h, of which v = h w; otherwise v itself.
    float4 a[CACHED], b[OP == PLAIN ? 1 : CACHED];
#pragma unroll
    for (int j = 0; j < CACHED; j++)
        if (tid + STEP * j < n4) a[j] = load4(x + 4 * (tid + STEP * j));
    if constexpr (OP == ADD_NORM || OP == GLU)
#pragma unroll
        for (int j = 0; j < CACHED; j++)
            if (tid + STEP * j < n4) b[j] = load4(r + 4 * (tid + STEP * j));
    if constexpr (OP == ADD_NORM)
#pragma unroll
        for (int j = 0; j < CACHED; j++)
            if (tid + STEP * j < n4) store4(h + 4 * (tid + STEP * j), a[j] = sum4(x, a[j], b[j]));
    if constexpr (IS_NORM)
#pragma unroll
        for (int j = 0; j < CACHED; j++)
            if (tid + STEP * j < n4) b[j] = reinterpret_cast<const float4 *>(w)[tid + STEP * j];
    // One group of four beyond the cached ones; `first`: the sum is still to be written.
    auto beyond = [&](uint32_t i, float4 &va, float4 &vb, bool first) {
        va = load4((OP == ADD_NORM && !first ? (const T *)h : x) + 4 * i);
        if constexpr (OP == ADD_NORM)
            if (first) store4(h + 4 * i, va = sum4(x, va, load4(r + 4 * i)));
        if constexpr (OP == GLU) vb = load4(r + 4 * i);
        if constexpr (IS_NORM) vb = reinterpret_cast<const float4 *>(w)[i];
    };
    auto value = [](float va, float vb) { return OP == PLAIN ? va : OP == GLU ? gated(va, vb) : va * vb; };
    auto value64 = [](float va, float vb) { return OP == PLAIN ? (double)va : OP == GLU ? gated64(va, vb) : (double)va * (double)vb; };
    // The exact value of element i of the row (from memory: by now this thread has written h there).
    auto exact = [&](uint32_t i) {
        const float va = load1(OP == ADD_NORM ? (const T *)h + i : x + i);
        return value64(va, OP == GLU ? load1(r + i) : IS_NORM ? w[i] : 0.f);
    };

    double ss = 0.0;
    uint32_t most = 0, up = 0; // bits of non-negative numbers are ordered as the numbers, NaN above infinity
    auto take = [&](const float4 &va, const float4 &vb, float4 &v) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float e = value(part(va, i), part(vb, i));
            if constexpr (IS_NORM) ss = fma((double)part(va, i), (double)part(va, i), ss);
            most = max(most, __float_as_uint(e) & 0x7FFFFFFFu);
            if constexpr (OP == GLU) up = max(up, __float_as_uint(part(vb, i)) & 0x7FFFFFFFu);
            (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w) = e;
        }
    };
#pragma unroll
    for (int j = 0; j < CACHED; j++)
        if (tid + STEP * j < n4) {
            float4 v;
            take(a[j], b[OP == PLAIN ? 0 : j], v);
            if constexpr (!IS_NORM) a[j] = v;
        }
    for (uint32_t i = tid + STEP * CACHED; i < n4; i += STEP) {
        float4 va, vb, v;
        beyond(i, va, vb, true);
        take(va, vb, v);
    }
    if constexpr (IS_NORM)
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (OP == GLU) up = __reduce_max_sync(0xffffffffu, up);
    if constexpr (WPR > 1) {
        if (lane == 0) {
            part_ss[warp] = ss;
            part_max[warp] = most;
            part_up[warp] = up;
        }
        __syncthreads();
        const uint32_t l = lane < WPR ? lane : 0;
        most = __reduce_max_sync(0xffffffffu, part_max[l]);
        if constexpr (OP == GLU) up = __reduce_max_sync(0xffffffffu, part_up[l]);
    }

    // The row's largest |v|, exactly.
    double a64 = 0.0;
    const bool fast = __uint_as_float(most) >= LEAST && __uint_as_float(most) <= MOST && (OP != GLU || __uint_as_float(up) < MOST_UP);
    bool bad = false;
    if (fast) {
        if constexpr (OP == PLAIN) a64 = (double)__uint_as_float(most);
        else {
            const uint32_t floor = most - BELOW<OP>;
            auto look = [&](float v, uint32_t i) {
                if ((__float_as_uint(v) & 0x7FFFFFFFu) >= floor) a64 = fmax(a64, fabs(exact(i)));
            };
#pragma unroll
            for (int j = 0; j < CACHED; j++)
                if (tid + STEP * j < n4)
#pragma unroll
                    for (int i = 0; i < 4; i++) look(IS_NORM ? part(a[j], i) * part(b[j], i) : part(a[j], i), 4 * (tid + STEP * j) + i);
            for (uint32_t i = tid + STEP * CACHED; i < n4; i += STEP) {
                float4 va, vb;
                beyond(i, va, vb, false);
                for (int k = 0; k < 4; k++) look(value(part(va, k), part(vb, k)), 4 * i + k);
            }
        }
    } else {
        for (uint32_t i = tid; i < n4; i += STEP)
            for (uint32_t k = 0; k < 4; k++) {
                const double v = fabs(exact(4 * i + k));
                bad |= !(v <= 3.4028234663852886e38);
                a64 = fmax(a64, v);
            }
    }
    if (OP != PLAIN || !fast) {
        if constexpr (WPR == 1) {
            bad = __any_sync(0xffffffffu, bad);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) a64 = fmax(a64, __shfl_xor_sync(0xffffffffu, a64, off));
        } else {
            if (a64 > 0.0) atomicMax(&most64, (unsigned long long)__double_as_longlong(a64));
            bad = __syncthreads_or(bad);
            a64 = __longlong_as_double((long long)most64);
        }
    }
    if (tid == 0) {
        double c = 1.0;
        if constexpr (IS_NORM) {
            if constexpr (WPR > 1) {
                ss = 0.0;
                for (int i = 0; i < WPR; i++) ss += part_ss[i];
            }
            c = 1.0 / sqrt(ss / (double)n + (double)eps);
        }
        scales[row] = bad ? __int_as_float(0x7fc00000) : (float)(a64 * c / 127.0);
    }

    uint32_t *out = reinterpret_cast<uint32_t *>(q);
    if (!fast) {
        for (uint32_t i = tid; i < n4; i += STEP) {
            uint32_t packed = 0;
            if (!bad && a64 > 0.0)
                for (uint32_t k = 0; k < 4; k++) packed |= (uint32_t)(uint8_t)(int8_t)__double2int_rn(exact(4 * i + k) * 127.0 / a64) << (8 * k);
            out[i] = packed;
        }
        return;
    }
    const float f = (float)(127.0 / a64);
    auto quantise = [&](const float4 &v, uint32_t i) {
        uint32_t bytes[4];
        bool near = false;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // Added to 1.5 * 2^23 a number is rounded to a whole one, whose low byte is the sum's.
            const float t = part(v, k) * f, whole = __fadd_rn(t, 12582912.f);
            bytes[k] = __float_as_uint(whole);
            near |= fabsf(t - __fsub_rn(whole, 12582912.f)) > 0.5f - NEAR<OP>;
        }
        if (near)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float t = part(v, k) * f;
                if (fabsf(t - __fsub_rn(__uint_as_float(bytes[k]), 12582912.f)) > 0.5f - NEAR<OP>) bytes[k] = (uint32_t)__double2int_rn(exact(4 * i + k) * 127.0 / a64);
            }
        out[i] = __byte_perm(__byte_perm(bytes[0], bytes[1], 0x0040), __byte_perm(bytes[2], bytes[3], 0x0040), 0x5410);
    };
    auto product = [](const float4 &va, const float4 &vb) { return make_float4(va.x * vb.x, va.y * vb.y, va.z * vb.z, va.w * vb.w); };
#pragma unroll
    for (int j = 0; j < CACHED; j++)
        if (tid + STEP * j < n4) quantise(IS_NORM ? product(a[j], b[IS_NORM ? j : 0]) : a[j], tid + STEP * j);
    for (uint32_t i = tid + STEP * CACHED; i < n4; i += STEP) {
        float4 va, vb;
        beyond(i, va, vb, false);
        quantise(make_float4(value(va.x, vb.x), value(va.y, vb.y), value(va.z, vb.z), value(va.w, vb.w)), i);
    }
}

template <int OP>
int launch_rows(fq_device *dev, const char *what, const void *x, const void *r, int dtype, const float *w, uint32_t n, float eps, uint32_t rows,
                void *h, int8_t *q, float *scales) {
    auto go = [&](auto zero, auto wpr, auto cached) {
        using T = decltype(zero);
        constexpr int WPR = decltype(wpr)::value;
        return launch_pdl(k_rows_i8<OP, T, WPR, decltype(cached)::value>, dim3(WPR == 1 ? (rows + 7) / 8 : rows), dim3(WPR == 1 ? 256 : WPR * 32), 0, dev->stream,
                          (const T *)x, (const T *)r, w, n, eps, rows, (T *)h, q, scales);
    };
    auto shape = [&](auto zero) {
        using std::integral_constant;
        constexpr integral_constant<int, 8> eight;
        if (n <= 1024) return go(zero, integral_constant<int, 1>{}, eight);
        if (rows <= 2 * (uint32_t)dev->sm_count || n > 8192) return go(zero, integral_constant<int, 16>{}, integral_constant<int, 10>{});
        if (n > 4096) return go(zero, eight, eight);
        return go(zero, integral_constant<int, 4>{}, eight);
    };
    const cudaError_t e = dtype == FQ_BF16 ? shape(__nv_bfloat16{}) : shape(float{});
    if (int rc = fq_check_cuda(dev, e, what)) return rc;
    return fq_end_enqueue(dev, what, 1);
}

// Shapes and bindings all four share; `x` and `r` (may be null) are the row inputs, `w` (may be null) the norm's weights.
int check_rows(fq_device *dev, const void *x, const void *r, int dtype, const float *w, bool norm, uint32_t n, uint32_t rows, const int8_t *q,
               const float *scales) {
    if (dtype != FQ_F32 && dtype != FQ_BF16) return fq_fail(dev, FQ_ERR_UNSUPPORTED, "element type %d", dtype);
    if (n == 0 || n % 4 || rows == 0) return fq_fail(dev, FQ_ERR_SHAPE, "%u rows of %u values in 8 bits (a multiple of 4)", rows, n);
    if (rows > 0x7fffffffu) return fq_fail(dev, FQ_ERR_SHAPE, "too many rows");
    const size_t count = (size_t)rows * n, bytes = count * fq_dtype_size(dtype);
    if (int rc = fq_check_binding(dev, x, bytes, "x")) return rc;
    if (r)
        if (int rc = fq_check_binding(dev, r, bytes, "r")) return rc;
    if (norm)
        if (int rc = fq_check_binding(dev, w, (size_t)n * 4, "w")) return rc;
    if (int rc = fq_check_binding(dev, q, count, "q")) return rc;
    if (int rc = fq_check_binding(dev, scales, (size_t)rows * 4, "scales")) return rc;
    const struct { const void *p; size_t bytes; } in[3] = {{x, bytes}, {r, bytes}, {w, (size_t)n * 4}};
    for (const auto &i : in) {
        if (int rc = fq_check_no_alias(dev, q, count, i.p, i.bytes, "q")) return rc;
        if (int rc = fq_check_no_alias(dev, scales, (size_t)rows * 4, i.p, i.bytes, "scales")) return rc;
    }
    return fq_check_no_alias(dev, scales, (size_t)rows * 4, q, count, "scales");
}

} // namespace

extern "C" int fq_quantize_i8(fq_device *dev, const void *x, int x_dtype, uint32_t n, uint32_t rows, int8_t *q, float *scales) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (int rc = check_rows(dev, x, nullptr, x_dtype, nullptr, false, n, rows, q, scales)) return rc;
    return launch_rows<PLAIN>(dev, "quantize_i8", x, nullptr, x_dtype, nullptr, n, 0.f, rows, nullptr, q, scales);
}

extern "C" int fq_rmsnorm_i8(fq_device *dev, const void *x, int x_dtype, const float *w, uint32_t n, float eps, uint32_t rows, int8_t *q,
                             float *scales) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (int rc = check_rows(dev, x, nullptr, x_dtype, w, true, n, rows, q, scales)) return rc;
    return launch_rows<NORM>(dev, "rmsnorm_i8", x, nullptr, x_dtype, w, n, eps, rows, nullptr, q, scales);
}

extern "C" int fq_add_rmsnorm_i8(fq_device *dev, const void *x, const void *r, int x_dtype, const float *w, uint32_t n, float eps, uint32_t rows,
                                 void *h, int8_t *q, float *scales) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (!r) return fq_fail(dev, FQ_ERR_RANGE, "r: null binding");
    if (int rc = check_rows(dev, x, r, x_dtype, w, true, n, rows, q, scales)) return rc;
    const size_t count = (size_t)rows * n, bytes = count * fq_dtype_size(x_dtype);
    if (int rc = fq_check_binding(dev, h, bytes, "h")) return rc;
    // h may be x or r itself: a value of h is written by the thread that read it.
    if (h != x)
        if (int rc = fq_check_no_alias(dev, h, bytes, x, bytes, "h")) return rc;
    if (h != r)
        if (int rc = fq_check_no_alias(dev, h, bytes, r, bytes, "h")) return rc;
    if (int rc = fq_check_no_alias(dev, h, bytes, w, (size_t)n * 4, "h")) return rc;
    if (int rc = fq_check_no_alias(dev, q, count, h, bytes, "q")) return rc;
    if (int rc = fq_check_no_alias(dev, scales, (size_t)rows * 4, h, bytes, "scales")) return rc;
    return launch_rows<ADD_NORM>(dev, "add_rmsnorm_i8", x, r, x_dtype, w, n, eps, rows, h, q, scales);
}

extern "C" int fq_glu_i8(fq_device *dev, const void *gate, const void *up, int dtype, uint32_t n, uint32_t rows, int8_t *q, float *scales) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (!up) return fq_fail(dev, FQ_ERR_RANGE, "up: null binding");
    if (int rc = check_rows(dev, gate, up, dtype, nullptr, false, n, rows, q, scales)) return rc;
    return launch_rows<GLU>(dev, "glu_i8", gate, up, dtype, nullptr, n, 0.f, rows, nullptr, q, scales);
}

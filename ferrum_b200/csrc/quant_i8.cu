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
// A row is read from memory once and kept in shared memory, every thread its own values of it.  v is computed in 32 bits; the
// few values that decide are taken again in 64: those that may be the row's largest, by one thread while the others round, and
// after it those whose quotient lies within the error of 32 bits of the border between two whole numbers.  Squares are added by fours in 32 bits and from there in 64.
// (Held in registers, unrolled over a row, the same took 105 registers and 63 instructions a value, a third of the time
// waiting for instructions: 2048 x 5120 bf16 45 us.)
#include <atomic>
#include <type_traits>

#include "gemv_common.cuh"
#include "internal.h"

namespace {
using namespace fqk;

enum Op { PLAIN, NORM, ADD_NORM, GLU };

// Four values at a time.
__device__ __forceinline__ float4 raw4(const float *p) { return __ldcg(reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ uint2 raw4(const __nv_bfloat16 *p) { return __ldcg(reinterpret_cast<const uint2 *>(p)); }
__device__ __forceinline__ float4 floats(const float4 &v) { return v; }
__device__ __forceinline__ float4 floats(const uint2 &b) {
    return make_float4(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xFFFF0000u), __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xFFFF0000u));
}
template <typename T> __device__ __forceinline__ float4 load4(const T *p) { return floats(raw4(p)); }
__device__ __forceinline__ float load1(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float load1(const __nv_bfloat16 *p) { return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(p)) << 16); }
// a + b, stored as its type keeps it, and as it is kept.
__device__ __forceinline__ float4 add4(float *p, const float4 &a, const float4 &b) {
    const float4 s = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
    *reinterpret_cast<float4 *>(p) = s;
    return s;
}
__device__ __forceinline__ float4 add4(__nv_bfloat16 *p, const float4 &a, const float4 &b) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(a.x + b.x, a.y + b.y), hi = __floats2bfloat162_rn(a.z + b.z, a.w + b.w);
    const uint2 u = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    *reinterpret_cast<uint2 *>(p) = u;
    return floats(u);
}
__device__ __forceinline__ float max_abs(float a, float b) { // NaN if one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}
__device__ __forceinline__ float max_abs(const float4 &v) { return max_abs(max_abs(v.x, v.y), max_abs(v.z, v.w)); }
// Two values an instruction.
__device__ __forceinline__ float4 mul4(const float4 &a, const float4 &b) {
    const float2 lo = __fmul2_rn(make_float2(a.x, a.y), make_float2(b.x, b.y)), hi = __fmul2_rn(make_float2(a.z, a.w), make_float2(b.z, b.w));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ float4 fma4(const float4 &a, float b, const float4 &c) {
    const float2 b2 = make_float2(b, b);
    const float2 lo = __ffma2_rn(make_float2(a.x, a.y), b2, make_float2(c.x, c.y)), hi = __ffma2_rn(make_float2(a.z, a.w), b2, make_float2(c.z, c.w));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ float4 rsub4(float a, const float4 &b) { // a - b
    const float2 lo = __fadd2_rn(make_float2(-b.x, -b.y), make_float2(a, a)), hi = __fadd2_rn(make_float2(-b.z, -b.w), make_float2(a, a));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}

// silu(g) u.  Relative error: 2 steps (2^-22) of the exponential and as much of the quotient, two roundings: 10 * 2^-24; beyond
// g = -87, where e^-g leaves the range of the quotient, 0 instead of less than 2^-118 |u|.
__device__ __forceinline__ float gated(float g, float u) { return __fdividef(g, 1.f + expf(-g)) * u; }
__device__ __forceinline__ double gated64(double g, double u) { return g / (1.0 + exp(-g)) * u; }

// The part of a quotient t = 127 v / a that its computation in 32 bits may be off: v and a as above or (norms) once rounded,
// 127 / a rounded.
template <int OP> constexpr float OFF = OP == GLU ? 24 * 0x1p-24f : 4 * 0x1p-24f;
// How many steps of fp32 the exact largest value may lie below the largest fp32 one: single roundings keep their order; a
// gated unit is off by at most 10 steps, and so is the largest.
template <int OP> constexpr uint32_t BELOW = OP == GLU ? 24 : 0;
// Rows that leave these go through 64 bits throughout: the largest |v|, so that what 32 bits lose to underflow is nothing
// beside it; and of the norms the largest sum of four squares, of the gated unit the largest |u|, for the same reason.
constexpr float LEAST = 1e-20f, MOST = 1e37f;
template <int OP> constexpr float LEAST_2 = OP == NORM || OP == ADD_NORM ? 1e-20f : 0.f;
template <int OP> constexpr float MOST_2 = OP == GLU ? 1048576.f : 1e37f;

// NT threads per row: a block, or one of its eight warps.  STAGED: the row is kept in shared memory (for the norms h, otherwise
// v); longer rows are computed again from memory for every step.
template <int OP, typename T, int NT, bool STAGED>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT, NT == 512 ? 2 : 5)
k_rows_i8(const T *x, const T *r, const float *w, uint32_t n, float eps, uint32_t rows, T *h, int8_t *q, float *scales) {
    constexpr bool IS_NORM = OP == NORM || OP == ADD_NORM, ONE_WARP = NT == 32;
    constexpr int W = NT / 32;
    extern __shared__ float4 stage[];
    __shared__ double part_ss[W];
    __shared__ uint32_t part_max[W], part_2[W];
    __shared__ unsigned long long largest;
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 31, warp = ONE_WARP ? 0 : threadIdx.x >> 5, tid = ONE_WARP ? lane : threadIdx.x;
    const uint32_t row = ONE_WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x, n4 = n / 4;
    if (!ONE_WARP && tid == 0) largest = 0;
    pdl_wait();
    if (row >= rows) return; // whole warps
    float4 *const kept = stage + (ONE_WARP ? (threadIdx.x >> 5) * n4 : 0);
    x += (size_t)row * n;
    if constexpr (OP == ADD_NORM || OP == GLU) r += (size_t)row * n;
    if constexpr (OP == ADD_NORM) h += (size_t)row * n;
    uint32_t *const out = reinterpret_cast<uint32_t *>(q + (size_t)row * n);
    const float4 *const w4 = reinterpret_cast<const float4 *>(w);

    auto values = [&](const float4 &a, const float4 &b) {
        if constexpr (OP == PLAIN) return a;
        else if constexpr (OP == GLU) return make_float4(gated(a.x, b.x), gated(a.y, b.y), gated(a.z, b.z), gated(a.w, b.w));
        else return mul4(a, b);
    };
    // v of group i of four, after the row has been read once.
    auto again = [&](uint32_t i) {
        if constexpr (STAGED) return IS_NORM ? values(kept[i], w4[i]) : kept[i];
        else if constexpr (OP == ADD_NORM) return values(load4((const T *)h + 4 * i), w4[i]);
        else if constexpr (OP == NORM) return values(load4(x + 4 * i), w4[i]);
        else if constexpr (OP == GLU) return values(load4(x + 4 * i), load4(r + 4 * i));
        else return load4(x + 4 * i);
    };
    // Value i in 64 bits.  (In memory a thread has written its own values of h.)
    auto exact = [&](uint32_t i) {
        const float a = STAGED && OP != GLU ? reinterpret_cast<const float *>(kept)[i] : load1(OP == ADD_NORM ? (const T *)h + i : x + i);
        if constexpr (OP == PLAIN) return (double)a;
        else if constexpr (OP == GLU) return gated64((double)a, (double)load1(r + i));
        else return (double)a * (double)w[i];
    };

    double ss = 0.0;
    float own = 0.f, own_2 = 0.f;
    auto take = [&](uint32_t i, float4 a, float4 b) {
        if constexpr (OP == ADD_NORM) a = add4(h + 4 * i, a, b);
        if constexpr (IS_NORM) {
            const float squares = fmaf(a.x, a.x, a.y * a.y) + fmaf(a.z, a.z, a.w * a.w);
            ss += (double)squares;
            own_2 = max_abs(own_2, squares);
        }
        if constexpr (OP == GLU) own_2 = max_abs(own_2, max_abs(b));
        const float4 v = IS_NORM ? values(a, w4[i]) : values(a, b);
        own = max_abs(own, max_abs(v));
        if constexpr (STAGED) kept[i] = IS_NORM ? a : v;
    };
    constexpr uint32_t AHEAD = sizeof(T) == 2 ? 4 : 2; // loads of either input that are under way together
    for (uint32_t i = tid; i < n4; i += AHEAD * NT) {
        decltype(raw4(x)) a[AHEAD], b[AHEAD];
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; j++)
            if (i + j * NT < n4) {
                a[j] = raw4(x + 4 * (i + j * NT));
                if constexpr (OP == ADD_NORM || OP == GLU) b[j] = raw4(r + 4 * (i + j * NT));
            }
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; j++)
            if (i + j * NT < n4) take(i + j * NT, floats(a[j]), floats(b[j]));
    }
    if constexpr (IS_NORM)
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    // Bits of numbers that are not negative are ordered as the numbers, NaN above infinity.
    uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(own)), most_2 = OP == PLAIN ? 0 : __reduce_max_sync(0xffffffffu, __float_as_uint(own_2));
    if constexpr (!ONE_WARP) {
        if (lane == 0) {
            part_ss[warp] = ss;
            part_max[warp] = most;
            part_2[warp] = most_2;
        }
        __syncthreads();
        most = __reduce_max_sync(0xffffffffu, part_max[lane % W]);
        if constexpr (OP != PLAIN) most_2 = __reduce_max_sync(0xffffffffu, part_2[lane % W]);
    }

    const bool fast = __uint_as_float(most) >= LEAST && __uint_as_float(most) <= MOST &&
                      (OP == PLAIN || (__uint_as_float(most_2) >= LEAST_2<OP> && __uint_as_float(most_2) <= MOST_2<OP>));
    double a64 = 0.0; // the row's largest |v|, exactly: of the thread's own values first
    bool bad = false;
    uint32_t near = 0; // groups of the thread with a value next to a border
    if (fast) {
        if (__float_as_uint(own) >= most - BELOW<OP>)
            for (uint32_t i = tid; i < n4; i += NT) {
                const float4 v = again(i);
#pragma unroll 1
                for (uint32_t k = 0; k < 4; k++)
                    if (__float_as_uint(fabsf(k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w)) >= most - BELOW<OP>) a64 = fmax(a64, fabs(exact(4 * i + k)));
            }
        if (!ONE_WARP && a64 > 0.0) atomicMax(&largest, (unsigned long long)__double_as_longlong(a64));
    } else {
        ss = 0.0;
        for (uint32_t i = tid; i < n4; i += NT)
#pragma unroll 1
            for (uint32_t k = 0; k < 4; k++) {
                const double v = fabs(exact(4 * i + k));
                bad |= !(v <= 3.4028234663852886e38);
                a64 = fmax(a64, v);
                if constexpr (IS_NORM) {
                    const double a = (double)load1(OP == ADD_NORM ? (const T *)h + 4 * i + k : x + 4 * i + k);
                    ss = fma(a, a, ss);
                }
            }
        if (!ONE_WARP && a64 > 0.0) atomicMax(&largest, (unsigned long long)__double_as_longlong(a64));
        if constexpr (IS_NORM) {
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
            if (!ONE_WARP && lane == 0) part_ss[warp] = ss;
        }
    }
    // t = 127 v / a: added to 1.5 * 2^23 it is rounded to a whole number, whose low byte is the sum's; `rest` is what that took.
    constexpr float MAGIC = 12582912.f;
    const float f = 127.f / __uint_as_float(most);
    auto rests = [&](const float4 &v, const float4 &whole) { return fma4(v, f, rsub4(MAGIC, whole)); };
    auto wholes = [&](const float4 &v) { return fma4(v, f, make_float4(MAGIC, MAGIC, MAGIC, MAGIC)); };
    if (fast) { // while the largest value is taken in 64 bits elsewhere
        uint32_t at = 0;
#pragma unroll 2
        for (uint32_t i = tid; i < n4; i += NT, at++) {
            const float4 v = again(i), whole = wholes(v);
            out[i] = __byte_perm(__byte_perm(__float_as_uint(whole.x), __float_as_uint(whole.y), 0x0040), __byte_perm(__float_as_uint(whole.z), __float_as_uint(whole.w), 0x0040), 0x5410);
            if (max_abs(rests(v, whole)) > 0.5f - 128 * OFF<OP>) near |= 1u << (at & 31);
        }
    }
    if constexpr (ONE_WARP) {
        bad = __any_sync(0xffffffffu, bad);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) a64 = fmax(a64, __shfl_xor_sync(0xffffffffu, a64, off));
    } else {
        bad = __syncthreads_or(bad);
        a64 = __longlong_as_double((long long)largest);
    }
    if (tid == NT - 1) { // not the first warp, which may have one group more of the row than the last
        double c = 1.0;
        if constexpr (IS_NORM) {
            if constexpr (!ONE_WARP) {
                ss = 0.0;
                for (int i = 0; i < W; i++) ss += part_ss[i];
            }
            c = 1.0 / sqrt(ss / (double)n + (double)eps);
        }
        scales[row] = bad ? __int_as_float(0x7fc00000) : (float)(a64 * c / 127.0);
    }

    auto rounded = [&](uint32_t i) { return (uint32_t)__double2int_rn(exact(i) * 127.0 / a64) & 0xFFu; };
    if (fast) {
        // Values that may be on the wrong side of a border, by their own size (bit b of `near`: groups b, b + 32, ...).
        while (near) {
            const uint32_t b = __ffs(near) - 1;
            near &= near - 1;
            for (uint32_t i = tid + b * NT; i < n4; i += 32 * NT) {
                const float4 v = again(i), whole = wholes(v), rest = rests(v, whole);
#pragma unroll 1
                for (uint32_t k = 0; k < 4; k++) {
                    const float e = k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w, part = k == 0 ? rest.x : k == 1 ? rest.y : k == 2 ? rest.z : rest.w;
                    if (fabsf(part) > 0.5f - (fabsf(e * f) + 0.5f) * OFF<OP>) reinterpret_cast<uint8_t *>(out)[4 * i + k] = (uint8_t)rounded(4 * i + k);
                }
            }
        }
    } else {
        for (uint32_t i = tid; i < n4; i += NT) {
            uint32_t packed = 0;
            if (!bad && a64 > 0.0)
#pragma unroll 1
                for (uint32_t k = 0; k < 4; k++) packed |= rounded(4 * i + k) << (8 * k);
            out[i] = packed;
        }
    }
}

constexpr size_t STAGE_MOST = 200 << 10;

template <int OP, typename T, int NT>
cudaError_t launch_nt(fq_device *dev, const T *x, const T *r, const float *w, uint32_t n, float eps, uint32_t rows, T *h, int8_t *q, float *scales) {
    const size_t bytes = (size_t)n * 4 * (NT == 32 ? 8 : 1);
    const dim3 grid(NT == 32 ? (rows + 7) / 8 : rows), block(NT == 32 ? 256 : NT);
    if (bytes > STAGE_MOST) return launch_pdl(k_rows_i8<OP, T, NT, false>, grid, block, 0, dev->stream, x, r, w, n, eps, rows, h, q, scales);
    auto kernel = k_rows_i8<OP, T, NT, true>;
    if (bytes > (40 << 10)) { // beyond what a kernel may use unasked (48 KB with its own arrays): asked for once per device
        static std::atomic<uint64_t> asked{0};
        const uint64_t bit = 1ull << (dev->ordinal & 63);
        if (!(asked.load(std::memory_order_relaxed) & bit) || dev->ordinal > 63) {
            if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)STAGE_MOST)) return e;
            asked.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    return launch_pdl(kernel, grid, block, bytes, dev->stream, x, r, w, n, eps, rows, h, q, scales);
}

template <int OP>
int launch_rows(fq_device *dev, const char *what, const void *x, const void *r, int dtype, const float *w, uint32_t n, float eps, uint32_t rows,
                void *h, int8_t *q, float *scales) {
    auto shape = [&](auto zero) {
        using T = decltype(zero);
        const T *tx = (const T *)x, *tr = (const T *)r;
        if (n <= 1024) return launch_nt<OP, T, 32>(dev, tx, tr, w, n, eps, rows, (T *)h, q, scales);
        if (n > 8192 || rows <= 2 * (uint32_t)dev->sm_count) return launch_nt<OP, T, 512>(dev, tx, tr, w, n, eps, rows, (T *)h, q, scales);
        return launch_nt<OP, T, 256>(dev, tx, tr, w, n, eps, rows, (T *)h, q, scales);
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

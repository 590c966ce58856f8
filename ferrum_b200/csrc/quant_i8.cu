// Rows of activations as 8-bit integers with one scale per row, the inputs of the 8-bit projections: a row as it is
// (`fq_quantize_i8`), normalised, with the residual's addition or without (`fq_rmsnorm_i8`, `fq_add_rmsnorm_i8`), or the
// gated unit of two rows (`fq_glu_i8`).
//
//   v_i = x_i | h_i w_i | silu(g_i) u_i        a = max_i |v_i|        q_i = round(127 v_i / a)        scale = a c / 127
//
// with c = 1 / sqrt(mean h^2 + eps) for the norms and 1 otherwise: 1/rms is common to a row and cancels in q.  Rounding is
// to the nearest whole number, ties to even, of the exact quotient.
#include <type_traits>

#include "gemv_common.cuh"
#include "internal.h"

namespace {
using namespace fqk;

enum Op { PLAIN, NORM, ADD_NORM, GLU };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// One block per row, everything in 64 bits, the row read again for every step.
template <int OP, typename T>
__global__ void __launch_bounds__(256)
k_rows_i8(const T *x, const T *r, const float *w, uint32_t n, float eps, T *h, int8_t *q, float *scales) {
    __shared__ double part[8], part_max[8];
    const size_t base = (size_t)blockIdx.x * n;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto value = [&](uint32_t i) -> double {
        if constexpr (OP == PLAIN) return (double)to_float(x[base + i]);
        else if constexpr (OP == NORM) return (double)to_float(x[base + i]) * (double)w[i];
        else if constexpr (OP == ADD_NORM) return (double)to_float(h[base + i]) * (double)w[i];
        else {
            const double g = (double)to_float(x[base + i]);
            return g / (1.0 + exp(-g)) * (double)to_float(r[base + i]);
        }
    };
    double ss = 0.0, most = 0.0;
    bool bad = false;
    for (uint32_t i = tid; i < n; i += 256) {
        if constexpr (OP == ADD_NORM) put(h + base + i, to_float(x[base + i]) + to_float(r[base + i]));
        if constexpr (OP == NORM || OP == ADD_NORM) {
            const double a = (double)to_float(OP == NORM ? x[base + i] : h[base + i]);
            ss += a * a;
        }
        const double v = fabs(value(i));
        bad |= !(v <= 3.402823466e38);
        most = fmax(most, v);
    }
    for (int off = 16; off > 0; off >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, off);
        most = fmax(most, __shfl_xor_sync(0xffffffffu, most, off));
    }
    if (lane == 0) part[warp] = ss, part_max[warp] = most;
    bad = __syncthreads_or(bad);
    ss = 0.0;
    for (int i = 0; i < 8; i++) ss += part[i], most = fmax(most, part_max[i]);
    const double c = OP == NORM || OP == ADD_NORM ? 1.0 / sqrt(ss / (double)n + (double)eps) : 1.0;
    if (tid == 0) scales[blockIdx.x] = bad ? __int_as_float(0x7fc00000) : (float)(most * c / 127.0);
    for (uint32_t i = tid; i < n; i += 256) q[base + i] = bad || most == 0.0 ? 0 : (int8_t)__double2int_rn(value(i) * 127.0 / most);
}

template <int OP>
int launch_rows(fq_device *dev, const char *what, const void *x, const void *r, int dtype, const float *w, uint32_t n, float eps, uint32_t rows,
                void *h, int8_t *q, float *scales) {
    auto go = [&](auto zero) {
        using T = decltype(zero);
        k_rows_i8<OP, T><<<rows, 256, 0, dev->stream>>>((const T *)x, (const T *)r, w, n, eps, (T *)h, q, scales);
    };
    if (dtype == FQ_BF16) go(__nv_bfloat16{});
    else go(float{});
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

// Projections of 8-bit rows by 8-bit matrices:
//
//   y[t][o] = (sum_k x[t][k] w[o][k]) * x_scale[t] * w_scale[o]
//
// The sum is a whole number of at most 2^14 * 65536 < 2^31 and exact; it is converted to fp32 once (rounded past 2^24), multiplied by the
// token's scale and then by the row's, and rounded to the output's type.
#include <cmath>
#include <vector>

#include "gemv_common.cuh"
#include "internal.h"

namespace {

constexpr uint32_t TILE = 64;

// 64 weight rows x 64 tokens a block, 4 x 4 outputs a thread, 64 bytes of K at a time through shared memory.
template <typename YT>
__global__ void __launch_bounds__(256)
k_project_i8(const int8_t *__restrict__ w, const float *__restrict__ ws, uint32_t rows, uint32_t cols, const int8_t *__restrict__ x,
             const float *__restrict__ xs, uint32_t m, YT *__restrict__ y) {
    __shared__ int a[TILE][17], b[TILE][17];
    const uint32_t tid = threadIdx.x, r0 = blockIdx.x * TILE, t0 = blockIdx.y * TILE;
    int acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < cols; k0 += 64) {
        for (uint32_t i = tid; i < TILE * 16; i += 256) {
            const uint32_t row = i / 16, k = k0 + 4 * (i % 16);
            a[row][i % 16] = r0 + row < rows && k < cols ? *(const int *)(w + (size_t)(r0 + row) * cols + k) : 0;
            b[row][i % 16] = t0 + row < m && k < cols ? *(const int *)(x + (size_t)(t0 + row) * cols + k) : 0;
        }
        __syncthreads();
        for (uint32_t k = 0; k < 16; k++)
            for (uint32_t i = 0; i < 4; i++)
                for (uint32_t j = 0; j < 4; j++) acc[i][j] = __dp4a(a[(tid & 15) + 16 * i][k], b[(tid >> 4) + 16 * j][k], acc[i][j]);
        __syncthreads();
    }
    for (uint32_t i = 0; i < 4; i++)
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t row = r0 + (tid & 15) + 16 * i, t = t0 + (tid >> 4) + 16 * j;
            if (row >= rows || t >= m) continue;
            const float v = (float)acc[i][j] * xs[t] * ws[row];
            if constexpr (sizeof(YT) == 2) y[(size_t)t * rows + row] = __float2bfloat16_rn(v);
            else y[(size_t)t * rows + row] = v;
        }
}

int launch_one(fq_device *dev, const fq_matrix *w, const int8_t *x, const float *xs, uint32_t m, void *y, int y_dtype) {
    const uint32_t rows = (uint32_t)w->rows, cols = (uint32_t)w->cols;
    const dim3 grid((rows + TILE - 1) / TILE, (m + TILE - 1) / TILE);
    if (y_dtype == FQ_BF16)
        k_project_i8<<<grid, 256, 0, dev->stream>>>((const int8_t *)w->data, w->scales, rows, cols, x, xs, m, (__nv_bfloat16 *)y);
    else k_project_i8<<<grid, 256, 0, dev->stream>>>((const int8_t *)w->data, w->scales, rows, cols, x, xs, m, (float *)y);
    return FQ_OK;
}

} // namespace

extern "C" int fq_matrix_create_i8(fq_device *dev, uint64_t rows, uint64_t cols, const int8_t *values, const float *scales, fq_matrix **out) {
    if (!dev || !out) return FQ_ERR_PARAM;
    *out = nullptr;
    if (!values || !scales) return fq_fail(dev, FQ_ERR_PARAM, "null payload");
    if (rows == 0 || cols == 0) return fq_fail(dev, FQ_ERR_SHAPE, "empty matrix geometry");
    if (cols % 16) return fq_fail(dev, FQ_ERR_SHAPE, "rows of %llu 8-bit values (a multiple of 16)", (unsigned long long)cols);
    if (cols > FQ_MAX_COLS || rows > 0x7fffffffull / 128) return fq_fail(dev, FQ_ERR_SHAPE, "matrix geometry is out of range");
    if (dev->capturing) return fq_fail(dev, FQ_ERR_PARAM, "a matrix cannot be created inside a graph capture");
    if (int rc = fq_check_cuda(dev, cudaSetDevice(dev->ordinal), "cudaSetDevice")) return rc;
    for (const void *p : {(const void *)values, (const void *)scales}) {
        cudaPointerAttributes attr{};
        if (int rc = fq_check_cuda(dev, cudaPointerGetAttributes(&attr, p), "payload")) return rc;
        if (attr.type == cudaMemoryTypeDevice && attr.device != dev->ordinal) return fq_fail(dev, FQ_ERR_DEVICE, "the payload is on device %d", attr.device);
    }
    std::vector<float> host(rows);
    cudaError_t e = cudaMemcpyAsync(host.data(), scales, rows * 4, cudaMemcpyDefault, dev->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(dev->stream);
    if (e != cudaSuccess) return fq_check_cuda(dev, e, "weight scales");
    for (uint64_t r = 0; r < rows; r++)
        if (!std::isfinite(host[r])) return fq_fail(dev, FQ_ERR_WEIGHT, "the scale of row %llu is not finite", (unsigned long long)r);
    fq_matrix *w = new fq_matrix();
    w->dev = dev;
    w->format = FQ_I8;
    w->rows = rows;
    w->cols = cols;
    w->row_bytes = w->pitch = cols;
    w->byte_size = rows * (cols + 4);
    w->block_elems = w->block_bytes = 1;
    const size_t len = rows * cols;
    e = cudaMalloc((void **)&w->data, len + rows * 4);
    w->scales = (float *)(w->data + len);
    if (e == cudaSuccess) e = cudaMemcpyAsync(w->data, values, len, cudaMemcpyDefault, dev->stream);
    if (e == cudaSuccess) e = cudaMemcpyAsync(w->scales, host.data(), rows * 4, cudaMemcpyHostToDevice, dev->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(dev->stream);
    if (e != cudaSuccess) {
        if (w->data) cudaFree(w->data);
        delete w;
        return fq_check_cuda(dev, e, "weight upload");
    }
    dev->counters.bytes_uploaded += w->byte_size;
    *out = w;
    return FQ_OK;
}

extern "C" int fq_project_many_i8(fq_device *dev, const fq_matrix *const *w, size_t count, const int8_t *x, size_t x_elems, const float *x_scales,
                                  size_t m, void *const *y, int y_dtype) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    constexpr size_t MAX = 8;
    if (!w || !y || count == 0) return fq_fail(dev, FQ_ERR_PARAM, "projection list");
    if (count > MAX) return fq_fail(dev, FQ_ERR_PARAM, "at most %zu projections share an input", MAX);
    if (y_dtype != FQ_F32 && y_dtype != FQ_BF16) return fq_fail(dev, FQ_ERR_UNSUPPORTED, "element type %d", y_dtype);
    for (size_t i = 0; i < count; i++) {
        if (!w[i]) return fq_fail(dev, FQ_ERR_PARAM, "null matrix");
        if (w[i]->dev != dev) return fq_fail(dev, FQ_ERR_DEVICE, "matrix belongs to another device handle");
        if (w[i]->format != FQ_I8) return fq_fail(dev, FQ_ERR_UNSUPPORTED, "8-bit rows are multiplied by matrices of fq_matrix_create_i8");
        if (m == 0 || x_elems != m * w[i]->cols)
            return fq_fail(dev, FQ_ERR_SHAPE, "projection [%zu, %llu] from %zu values", m, (unsigned long long)w[i]->cols, x_elems);
        if (m > 0x7fffffffu / 8) return fq_fail(dev, FQ_ERR_SHAPE, "too many activation rows");
        const size_t yb = m * w[i]->rows * fq_dtype_size(y_dtype);
        if (int rc = fq_check_binding(dev, x, x_elems, "x")) return rc;
        if (int rc = fq_check_binding(dev, x_scales, m * 4, "x_scales")) return rc;
        if (int rc = fq_check_binding(dev, y[i], yb, "y")) return rc;
        if (int rc = fq_check_no_alias(dev, y[i], yb, x, x_elems, "y")) return rc;
        if (int rc = fq_check_no_alias(dev, y[i], yb, x_scales, m * 4, "y")) return rc;
        for (size_t j = 0; j < i; j++)
            if (int rc = fq_check_no_alias(dev, y[i], yb, y[j], m * w[j]->rows * fq_dtype_size(y_dtype), "y")) return rc;
    }
    for (size_t i = 0; i < count; i++) launch_one(dev, w[i], x, x_scales, (uint32_t)m, y[i], y_dtype);
    return fq_end_enqueue(dev, "project_i8", (int)count);
}

extern "C" int fq_project_i8(fq_device *dev, const fq_matrix *w, const int8_t *x, size_t x_elems, const float *x_scales, size_t m, void *y,
                             int y_dtype, size_t y_elems) {
    if (w && y_elems != m * w->rows) {
        if (int rc = fq_begin_enqueue(dev)) return rc;
        return fq_fail(dev, FQ_ERR_SHAPE, "projection of %zu rows by [%llu, %llu]^T into %zu values", m, (unsigned long long)w->rows,
                       (unsigned long long)w->cols, y_elems);
    }
    return fq_project_many_i8(dev, &w, 1, x, x_elems, x_scales, m, &y, y_dtype);
}

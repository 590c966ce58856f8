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
// after it those whose quotient lies within the error of 32 bits of the border between two whole numbers.  Squares are added by fours or
// eights in 32 bits and from there in 64.
// (Held in registers, unrolled over a row, the same took 105 registers and 63 instructions a value, a third of the time
// waiting for instructions: 2048 x 5120 bf16 45 us.)
//
// What bounds it is a row's chain of dependent steps, of which the blocks of an SM cover a part.  2048 x 5120, bf16 / F32: quantize
// 11.5 / 14.8 us (2.7 / 3.6 TB/s), rmsnorm 13.1 / 16.1 (2.4 / 3.3), add_rmsnorm 20.0 / 28.1 (3.7 / 4.8); the gated unit of 1021 x
// 17408 22.3 / 39.1 (4.0 / 4.1), of 28672 values a row, of which an SM holds one or two, 49 / 63 (3.0 / 4.1), of 53248, computed
// twice, 111 / 195 (2.5 / 2.5); one row of 5120 F32 2.2, 2.5 and 3.4.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gemv_common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace {
using namespace fqk;
using namespace fqtc;

struct Arrivals { // of a block's bulk copies
    uint64_t full;
    uint32_t abort_flag;
};

enum Op { PLAIN, NORM, ADD_NORM, GLU };

// VEC values of a row at a time: 16 bytes, or 8 of bf16 rows whose length is no multiple of eight.
template <int VEC> struct Vec { float2 p[VEC / 2]; };
template <int VEC> struct Raw; // as they lie in memory
template <> struct Raw<4> { uint2 u; };
template <> struct Raw<8> { uint4 u; };
__device__ __forceinline__ uint32_t word(const uint2 &u, int i) { return i == 0 ? u.x : u.y; }
__device__ __forceinline__ uint32_t word(const uint4 &u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }
__device__ __forceinline__ float2 floats(uint32_t bf16x2) { return make_float2(__uint_as_float(bf16x2 << 16), __uint_as_float(bf16x2 & 0xFFFF0000u)); }
template <int VEC> __device__ __forceinline__ Vec<VEC> floats(const Raw<VEC> &r) {
    Vec<VEC> v;
#pragma unroll
    for (int i = 0; i < VEC / 2; i++) v.p[i] = floats(word(r.u, i));
    return v;
}
template <int VEC> __device__ __forceinline__ const Vec<VEC> &floats(const Vec<VEC> &v) { return v; }
template <int VEC> __device__ __forceinline__ Vec<VEC> load(const float *p) { // (in shared memory too)
    Vec<VEC> v;
#pragma unroll
    for (int i = 0; i < VEC / 4; i++) {
        const float4 f = reinterpret_cast<const float4 *>(p)[i];
        v.p[2 * i] = make_float2(f.x, f.y);
        v.p[2 * i + 1] = make_float2(f.z, f.w);
    }
    return v;
}
template <int VEC> __device__ __forceinline__ void store(float *p, const Vec<VEC> &v) {
#pragma unroll
    for (int i = 0; i < VEC / 4; i++) reinterpret_cast<float4 *>(p)[i] = make_float4(v.p[2 * i].x, v.p[2 * i].y, v.p[2 * i + 1].x, v.p[2 * i + 1].y);
}
// Activations: of a kernel that may still run when this one starts, so past L1.
template <int VEC> __device__ __forceinline__ Vec<VEC> fetch(const float *p) {
    static_assert(VEC == 4, "16 bytes");
    const float4 f = __ldcg(reinterpret_cast<const float4 *>(p));
    return Vec<VEC>{make_float2(f.x, f.y), make_float2(f.z, f.w)};
}
template <int VEC> __device__ __forceinline__ Raw<VEC> fetch(const __nv_bfloat16 *p) {
    if constexpr (VEC == 8) return Raw<VEC>{__ldcg(reinterpret_cast<const uint4 *>(p))};
    else return Raw<VEC>{__ldcg(reinterpret_cast<const uint2 *>(p))};
}
__device__ __forceinline__ float load1(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float load1(const __nv_bfloat16 *p) { return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(p)) << 16); }
// a + b as its type keeps it; stored.  (Of bf16 numbers it is the same rounded once or by way of fp32: one that reaches below
// the 24 bits of the other's sum is less than a 2^7th of half a step of it.)
__device__ __forceinline__ Vec<4> sum_to(float *p, const Vec<4> &a, const Vec<4> &b) {
    const Vec<4> s{__fadd2_rn(a.p[0], b.p[0]), __fadd2_rn(a.p[1], b.p[1])};
    store<4>(p, s);
    return s;
}
__device__ __forceinline__ uint32_t sum_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 s = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&s);
}
template <int VEC> __device__ __forceinline__ Vec<VEC> sum_to(__nv_bfloat16 *p, const Raw<VEC> &a, const Raw<VEC> &b) {
    Raw<VEC> s;
    s.u.x = sum_bf16x2(a.u.x, b.u.x);
    s.u.y = sum_bf16x2(a.u.y, b.u.y);
    if constexpr (VEC == 8) {
        s.u.z = sum_bf16x2(a.u.z, b.u.z);
        s.u.w = sum_bf16x2(a.u.w, b.u.w);
    }
    *reinterpret_cast<decltype(s.u) *>(p) = s.u;
    return floats(s);
}
// The largest of |a|, |b|, |c|; NaN if one is.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int VEC> __device__ __forceinline__ float max_abs(float m, const Vec<VEC> &v) {
#pragma unroll
    for (int i = 0; i < VEC / 2; i++) m = max_abs(m, v.p[i].x, v.p[i].y);
    return m;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 minus(const float2 &v) { return make_float2(-v.x, -v.y); }

__device__ __forceinline__ float ex2(float v) { // within 2^-22.5 of itself
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp(float v) { // within 2^-23 of itself
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// silu(g) u for two values, e^-g = 2^t (1 + d ln 2) with t = -g log2 e rounded and d what the rounding took.  Relative error at
// most 10 * 2^-24: 5 of the exponential, 1 of 1 + e^-g, 2 of its reciprocal and one of each product.  Below g = -87.34, where the
// reciprocal is below 2^-126 and flushed, it is 0 and off by less than 2^-119 |u|.  For that g is held at -127 ln 2 in t and in d
// alike: of t alone, d of a g past 2^24 is the rounding of a t that is not used, and 1 + d ln 2 can be next to nothing.  The factor g
// is as it is, so that an infinite one gives NaN.
__device__ __forceinline__ float2 gated(const float2 &g, const float2 &u) {
    constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.92596299e-8f, LN2 = 0.693147182f, LOWEST = -88.0296936f;
    const float2 held = make_float2(fmaxf(g.x, LOWEST), fmaxf(g.y, LOWEST));
    const float2 t = __fmul2_rn(held, both(-LOG2E));
    const float2 d = __ffma2_rn(held, both(-LOG2E_REST), __ffma2_rn(held, both(-LOG2E), minus(t)));
    const float2 e = make_float2(ex2(t.x), ex2(t.y));
    const float2 s = __fadd2_rn(__ffma2_rn(__fmul2_rn(d, both(LN2)), e, e), both(1.f));
    return __fmul2_rn(__fmul2_rn(g, make_float2(rcp(s.x), rcp(s.y))), u);
}
__device__ __forceinline__ double gated64(double g, double u) { return g / (1.0 + exp(-g)) * u; }

// The part of a quotient t = 127 v / a that its computation in 32 bits may be off: v and a as above or (norms) once rounded,
// 127 / a rounded.
template <int OP> constexpr float OFF = OP == GLU ? 24 * 0x1p-24f : 4 * 0x1p-24f;
// How many steps of fp32 the exact largest value may lie below the largest fp32 one: single roundings keep their order; a
// gated unit is off by at most 10 steps, and so is the largest.
template <int OP> constexpr uint32_t BELOW = OP == GLU ? 24 : 0;
// Rows that leave these go through 64 bits throughout: the largest |v|, so that what 32 bits lose to underflow is nothing
// beside it; and of the norms the largest sum of four squares, of the gated unit the largest |u|, for the same reason.  Of a
// row as it is products of up to 127.5 and the largest |v| are taken in 32 bits (`settle`): fp32 ends at 127.5 * 2.66e36.
constexpr float LEAST = 1e-20f;
template <int OP> constexpr float MOST = OP == PLAIN ? 2.5e36f : 1e37f;
template <int OP> constexpr float LEAST_2 = OP == NORM || OP == ADD_NORM ? 1e-20f : 0.f;
template <int OP> constexpr float MOST_2 = OP == GLU ? 1048576.f : 1e37f;

// Where a thread's values of a row are between its steps.
enum Mode {
    DIRECT, // nowhere: v is computed again from memory (rows longer than shared memory)
    KEPT,   // v in shared memory, read from memory by the threads
    BULK    // bulk copies bring the inputs to shared memory, where v takes their place (bf16: a group's 16 bytes of each)
};

// NT threads per row: a block, or one of its eight warps.
template <int OP, typename T, int VEC, int NT, int MODE>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT, NT == 512 ? 3 : NT == 32 ? 5 : 1280 / NT)
k_rows_i8(const T *x, const T *r, const float *w, uint32_t n, float eps, uint32_t rows, T *h, int8_t *q, float *scales, double inv_n, int *status) {
    constexpr bool IS_NORM = OP == NORM || OP == ADD_NORM, TWO = OP == ADD_NORM || OP == GLU, ONE_WARP = NT == 32;
    constexpr int W = NT / 32;
    extern __shared__ float4 stage[];
    __shared__ double part_ss[W];
    __shared__ uint32_t part_max[W], part_2[W];
    __shared__ unsigned long long largest;
    __shared__ Arrivals arrivals;
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 31, warp = ONE_WARP ? 0 : threadIdx.x >> 5, tid = ONE_WARP ? lane : threadIdx.x;
    const uint32_t row = ONE_WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x, groups = n / VEC, half = n * (uint32_t)sizeof(T);
    // Of group i, BULK: the 16 bytes at i and at `half` + i; KEPT: VEC floats.
    uint8_t *const kept = reinterpret_cast<uint8_t *>(stage) + (ONE_WARP ? (threadIdx.x >> 5) * n * 4 : 0);
    if (!ONE_WARP && tid == 0) largest = 0;
    if (MODE == BULK && tid == 0) {
        mbar_init(&arrivals.full, 1);
        arrivals.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    if (row >= rows) return; // whole warps
    x += (size_t)row * n;
    if constexpr (TWO) r += (size_t)row * n;
    if constexpr (OP == ADD_NORM) h += (size_t)row * n;
    q += (size_t)row * n;
    bool late = false;
    if constexpr (MODE == BULK) {
        if (tid == 0) {
            mbar_expect_tx(&arrivals.full, TWO ? 2 * half : half);
            bulk_load(kept, x, half, &arrivals.full);
            if constexpr (TWO) bulk_load(kept + half, r, half, &arrivals.full);
        }
        __syncthreads();
        late = !mbar_wait(&arrivals.full, 0, &arrivals, status);
    }

    auto product = [](const Vec<VEC> &a, const Vec<VEC> &b) {
        Vec<VEC> v;
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) v.p[i] = OP == GLU ? gated(a.p[i], b.p[i]) : __fmul2_rn(a.p[i], b.p[i]);
        return v;
    };
    // v of group i, after the row has been read once.
    auto again = [&](uint32_t i) {
        if constexpr (MODE == KEPT) return load<VEC>(reinterpret_cast<const float *>(kept) + VEC * i);
        else if constexpr (MODE == BULK && VEC == 8) {
            const Vec<4> lo = load<4>(reinterpret_cast<const float *>(kept) + 4 * i), hi = load<4>(reinterpret_cast<const float *>(kept + half) + 4 * i);
            return Vec<VEC>{lo.p[0], lo.p[1], hi.p[0], hi.p[1]};
        } else if constexpr (OP == PLAIN) return Vec<VEC>(floats(fetch<VEC>(x + VEC * i)));
        else if constexpr (OP == GLU) return product(floats(fetch<VEC>(x + VEC * i)), floats(fetch<VEC>(r + VEC * i)));
        else return product(floats(fetch<VEC>((OP == ADD_NORM ? (const T *)h : x) + VEC * i)), load<VEC>(w + VEC * i));
    };
    // Value i in 64 bits, from memory.  (Of h this thread has written its own values there.)
    auto exact = [&](uint32_t i) {
        const float a = load1(OP == ADD_NORM ? (const T *)h + i : x + i);
        if constexpr (OP == PLAIN) return (double)a;
        else if constexpr (OP == GLU) return gated64((double)a, (double)load1(r + i));
        else return (double)a * (double)w[i];
    };

    double ss = 0.0;
    float own = 0.f, own_2 = 0.f;
    auto take = [&](uint32_t i, const decltype(fetch<VEC>(x)) &a, const decltype(fetch<VEC>(x)) &b) {
        const uint32_t at = VEC * i;
        Vec<VEC> v;
        if constexpr (OP == ADD_NORM) v = sum_to(h + at, a, b);
        else v = floats(a);
        if constexpr (IS_NORM) {
            float2 squares = __fmul2_rn(v.p[0], v.p[0]);
#pragma unroll
            for (int k = 1; k < VEC / 2; k++) squares = __ffma2_rn(v.p[k], v.p[k], squares);
            const float sum = squares.x + squares.y;
            ss += (double)sum;
            own_2 = max_abs(own_2, sum, sum);
            v = product(v, load<VEC>(w + at));
        }
        if constexpr (OP == GLU) {
            const Vec<VEC> u = floats(b);
            own_2 = max_abs(own_2, u);
            v = product(v, u);
        }
        own = max_abs(own, v);
        if constexpr (MODE == KEPT) store<VEC>(reinterpret_cast<float *>(kept) + at, v);
        if constexpr (MODE == BULK && VEC == 8) {
            store<4>(reinterpret_cast<float *>(kept) + 4 * i, Vec<4>{v.p[0], v.p[1]});
            store<4>(reinterpret_cast<float *>(kept + half) + 4 * i, Vec<4>{v.p[2], v.p[3]});
        }
    };
    if constexpr (MODE == BULK) {
        using In = decltype(fetch<VEC>(x));
        static_assert(sizeof(In) == 16 && VEC == 8, "a group is 16 bytes of each input, and 32 of v");
#pragma unroll 2
        for (uint32_t i = tid; i < groups; i += NT)
            take(i, reinterpret_cast<const In *>(kept)[i], reinterpret_cast<const In *>(kept + (TWO ? half : 0))[i]);
    } else {
        constexpr uint32_t AHEAD = sizeof(T) * VEC == 16 ? 2 : 4; // loads of either input that are under way together
        for (uint32_t i = tid; i < groups; i += AHEAD * NT) {
            decltype(fetch<VEC>(x)) a[AHEAD], b[AHEAD];
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; j++)
                if (i + j * NT < groups) {
                    a[j] = fetch<VEC>(x + VEC * (i + j * NT));
                    if constexpr (TWO) b[j] = fetch<VEC>(r + VEC * (i + j * NT));
                }
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; j++)
                if (i + j * NT < groups) take(i + j * NT, a[j], b[j]);
        }
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
        if constexpr (MODE == BULK) {
            if (__syncthreads_or(late)) { // a copy did not come, and the status says so: time for it to land before the memory is another's
                for (const uint64_t t0 = now_ns(); now_ns() - t0 < 200000;) {}
                return;
            }
        } else {
            __syncthreads();
        }
        most = __reduce_max_sync(0xffffffffu, part_max[lane % W]);
        if constexpr (OP != PLAIN) most_2 = __reduce_max_sync(0xffffffffu, part_2[lane % W]);
    }

    const bool fast = __uint_as_float(most) >= LEAST && __uint_as_float(most) <= MOST<OP> &&
                      (OP == PLAIN || (__uint_as_float(most_2) >= LEAST_2<OP> && __uint_as_float(most_2) <= MOST_2<OP>));
    double a64 = 0.0; // the row's largest |v|, exactly: of the thread's own values first
    bool bad = false;
    uint32_t near = 0; // groups of the thread with a value next to a border
    if (fast) {
        if (__float_as_uint(own) >= most - BELOW<OP>)
            for (uint32_t i = tid; i < groups; i += NT) {
                const Vec<VEC> v = again(i);
                const float floor = __uint_as_float(most - BELOW<OP>);
                uint32_t which = 0;
#pragma unroll
                for (int k = 0; k < VEC / 2; k++) which |= (fabsf(v.p[k].x) >= floor ? 1u : 0u) << (2 * k) | (fabsf(v.p[k].y) >= floor ? 2u : 0u) << (2 * k);
                for (; which; which &= which - 1) a64 = fmax(a64, fabs(exact(VEC * i + __ffs(which) - 1)));
            }
        if (!ONE_WARP && a64 > 0.0) atomicMax(&largest, (unsigned long long)__double_as_longlong(a64));
    } else {
        ss = 0.0;
        for (uint32_t i = tid; i < groups; i += NT)
#pragma unroll 1
            for (uint32_t k = 0; k < VEC; k++) {
                const double v = fabs(exact(VEC * i + k));
                bad |= !(v <= 3.4028234663852886e38);
                a64 = fmax(a64, v);
                if constexpr (IS_NORM) {
                    const double a = (double)load1(OP == ADD_NORM ? (const T *)h + VEC * i + k : x + VEC * i + k);
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
    const float2 magic = both(12582912.f), f = both(127.f / __uint_as_float(most));
    auto whole_of = [&](const float2 &v) { return __ffma2_rn(v, f, magic); };
    auto rest_of = [&](const float2 &v, const float2 &whole) { return __ffma2_rn(v, f, __fadd2_rn(minus(whole), magic)); };
    auto low_bytes = [](const float2 &a, const float2 &b) {
        return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
    };
    // A value of a row as it is, v, against the border b that its quotient is next to: 127 v - b a from products and what their
    // roundings took (where it decides the products differ by little, and exactly).
    auto settle = [&](float v, int8_t *to, float whole) {
        const float a = __uint_as_float(most), near = whole - magic.x, rest = fmaf(v, f.x, -near);
        const float b = near + copysignf(0.5f, rest), p = 127.f * v, m = b * a;
        const float over = copysignf(1.f, rest) * ((p - m) + (fmaf(127.f, v, -p) - fmaf(b, a, -m)));
        const bool odd = __float_as_uint(whole) & 1;
        if (fabsf(rest) > 0.25f && (over > 0.f || (over == 0.f && odd))) *to = (int8_t)(near + copysignf(1.f, rest));
    };
    if (fast) { // while the largest value is taken in 64 bits elsewhere
        uint32_t at = 0;
#pragma unroll 2
        for (uint32_t i = tid; i < groups; i += NT, at++) {
            const Vec<VEC> v = again(i);
            Vec<VEC> whole, rest;
#pragma unroll
            for (int k = 0; k < VEC / 2; k++) {
                whole.p[k] = whole_of(v.p[k]);
                rest.p[k] = rest_of(v.p[k], whole.p[k]);
            }
            if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(q + VEC * i) = make_uint2(low_bytes(whole.p[0], whole.p[1]), low_bytes(whole.p[2], whole.p[3]));
            else *reinterpret_cast<uint32_t *>(q + VEC * i) = low_bytes(whole.p[0], whole.p[1]);
            if (max_abs(0.f, rest) > 0.5f - 128 * OFF<OP>) {
                if constexpr (OP == PLAIN) { // v and a are what they are, and bf16 rows hold many halves of a: 63.5
#pragma unroll
                    for (int k = 0; k < VEC / 2; k++) {
                        settle(v.p[k].x, q + VEC * i + 2 * k, whole.p[k].x);
                        settle(v.p[k].y, q + VEC * i + 2 * k + 1, whole.p[k].y);
                    }
                } else {
                    near |= 1u << (at & 31);
                }
            }
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
            const double mean = fma(ss, inv_n, (double)eps);
            if (fast) { // (in the range of fp32) a step of Newton's method squares the error of 2^-22
                const double y = (double)rsqrtf((float)mean);
                c = y * fma(-0.5 * mean * y, y, 1.5);
            } else {
                c = 1.0 / sqrt(mean);
            }
        }
        scales[row] = bad ? __int_as_float(0x7fc00000) : a64 > 0.0 ? (float)(a64 * c * (1.0 / 127.0)) : 0.f; // (c of zeros without eps is infinite)
    }

    // 127 v / a rounded, from the whole number next to it or nearly so: 127 v is compared with its borders times a.
    auto rounded = [&](double v, int near) {
        const double t = 127.0 * v, up = ((double)near + 0.5) * a64, down = ((double)near - 0.5) * a64;
        if (t > up || (t == up && (near & 1))) return (int8_t)(near + 1);
        return (int8_t)(t < down || (t == down && (near & 1)) ? near - 1 : near);
    };
    if (fast) {
        // Values that may be on the wrong side of a border, by their own size (bit b of `near`: groups b, b + 32, ...).
        while (near) {
            const uint32_t b = __ffs(near) - 1;
            near &= near - 1;
            for (uint32_t i = tid + b * NT; i < groups; i += 32 * NT) {
                const Vec<VEC> v = again(i);
                auto look = [&](uint32_t k, float e) {
                    const float whole = fmaf(e, f.x, magic.x), rest = fmaf(e, f.x, magic.x - whole);
                    if (fabsf(rest) > 0.5f - (fabsf(e * f.x) + 0.5f) * OFF<OP>)
                        q[VEC * i + k] = rounded(exact(VEC * i + k), (int8_t)__float_as_uint(whole));
                };
#pragma unroll
                for (int k = 0; k < VEC / 2; k++) {
                    look(2 * k, v.p[k].x);
                    look(2 * k + 1, v.p[k].y);
                }
            }
        }
    } else {
        for (uint32_t i = tid; i < groups; i += NT)
#pragma unroll 1
            for (uint32_t k = 0; k < VEC; k++) {
                const double v = bad ? 0.0 : exact(VEC * i + k); // (a quotient is rounded twice, and a tie falls to either side)
                q[VEC * i + k] = a64 > 0.0 ? rounded(v, __double2int_rn(v * 127.0 / a64)) : 0;
            }
    }
}

constexpr size_t STAGE_MOST = 200 << 10, BULK_MOST = 74 << 10; // bytes of v of a row: what fits, and three blocks an SM
constexpr uint32_t NARROW_GROUPS = 1600;                       // of a row, for blocks of fewer than 512 threads
static_assert(NARROW_GROUPS * 8 * 4 <= BULK_MOST && 8 * 1024 * 4 <= BULK_MOST, "only blocks of 512 threads get longer rows");

// What a kernel may use of an SM's shared memory beyond what it may unasked (48 KB with its own arrays): asked for once per device.
template <typename K> cudaError_t allow(fq_device *dev, K kernel, size_t bytes, std::atomic<uint64_t> &asked) {
    if (bytes <= (40 << 10)) return cudaSuccess;
    const uint64_t bit = 1ull << (dev->ordinal & 63);
    if ((asked.load(std::memory_order_relaxed) & bit) && dev->ordinal <= 63) return cudaSuccess;
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)STAGE_MOST)) return e;
    asked.fetch_or(bit, std::memory_order_relaxed);
    return cudaSuccess;
}

template <int OP, typename T, int VEC, int NT>
cudaError_t launch_nt(fq_device *dev, const T *x, const T *r, const float *w, uint32_t n, float eps, uint32_t rows, T *h, int8_t *q, float *scales) {
    const size_t bytes = (size_t)n * 4 * (NT == 32 ? 8 : 1);
    const dim3 grid(NT == 32 ? (rows + 7) / 8 : rows), block(NT == 32 ? 256 : NT);
    const double inv_n = 1.0 / n;
    auto go = [&](auto kernel, size_t smem, std::atomic<uint64_t> &asked) {
        if (const cudaError_t e = allow(dev, kernel, smem, asked)) return e;
        return launch_pdl(kernel, grid, block, smem, dev->stream, x, r, w, n, eps, rows, h, q, scales, inv_n, dev->status_dev);
    };
    // Each mode for the rows that it gets: bulk copies bring in eight bf16 values a thread at a time, and only 512 threads get rows
    // past BULK_MOST.
    constexpr bool BULKS = NT != 32 && VEC == 8;
    if constexpr (BULKS)
        if (NT != 512 || bytes <= BULK_MOST) {
            static std::atomic<uint64_t> asked{0};
            return go(k_rows_i8<OP, T, VEC, NT, BULK>, bytes, asked);
        }
    if constexpr (NT == 512)
        if (bytes > STAGE_MOST) {
            static std::atomic<uint64_t> asked{0};
            return go(k_rows_i8<OP, T, VEC, NT, DIRECT>, 0, asked);
        }
    if constexpr (!BULKS || NT == 512) {
        static std::atomic<uint64_t> asked{0};
        return go(k_rows_i8<OP, T, VEC, NT, KEPT>, bytes, asked);
    }
}

template <int OP, typename T, int VEC>
cudaError_t launch_vec(fq_device *dev, const void *x, const void *r, const float *w, uint32_t n, float eps, uint32_t rows, void *h, int8_t *q, float *scales) {
    const T *tx = (const T *)x, *tr = (const T *)r;
    const bool few = rows <= 2 * (uint32_t)dev->sm_count;
    const uint32_t groups = n / VEC;
    if (n <= 1024) return launch_nt<OP, T, VEC, 32>(dev, tx, tr, w, n, eps, rows, (T *)h, q, scales);
    // With many rows the threads that a row's sums are joined over cost more than the time a row waits for itself; a few rows wait.
    // us with 128 / 256 / 512 threads: add_rmsnorm bf16 2048 x 5120 21.1 / 19.5 / -, gated unit 14.8 / 16.4 / -, 1021 x 17408 - /
    // 24.5 / 22.2; add_rmsnorm F32 of one row of 5120 - / 4.1 / 3.5, of 200 - / 6.5 / 5.3.
    if (groups > (few ? 512 : NARROW_GROUPS)) return launch_nt<OP, T, VEC, 512>(dev, tx, tr, w, n, eps, rows, (T *)h, q, scales);
    if (groups > (few ? 256 : OP == ADD_NORM ? 400 : 800)) return launch_nt<OP, T, VEC, 256>(dev, tx, tr, w, n, eps, rows, (T *)h, q, scales);
    return launch_nt<OP, T, VEC, 128>(dev, tx, tr, w, n, eps, rows, (T *)h, q, scales);
}

template <int OP>
int launch_rows(fq_device *dev, const char *what, const void *x, const void *r, int dtype, const float *w, uint32_t n, float eps, uint32_t rows,
                void *h, int8_t *q, float *scales) {
    const cudaError_t e = dtype == FQ_F32 ? launch_vec<OP, float, 4>(dev, x, r, w, n, eps, rows, h, q, scales)
                          : n % 8 == 0    ? launch_vec<OP, __nv_bfloat16, 8>(dev, x, r, w, n, eps, rows, h, q, scales)
                                          : launch_vec<OP, __nv_bfloat16, 4>(dev, x, r, w, n, eps, rows, h, q, scales);
    if (int rc = fq_check_cuda(dev, e, what)) return rc;
    const size_t count = (size_t)rows * n;
    if (h) fq_note_write(dev, h, count * fq_dtype_size(dtype));
    fq_note_write(dev, q, count);
    fq_note_write(dev, scales, (size_t)rows * 4);
    return fq_end_enqueue(dev, what, 1);
}

// Shapes and bindings all four share; `x` and `r` (may be null) are the row inputs, `w` (may be null) the norm's weights.
int check_rows(fq_device *dev, const void *x, const void *r, int dtype, const float *w, bool norm, uint32_t n, uint32_t rows, const int8_t *q,
               const float *scales) {
    if (dtype != FQ_F32 && dtype != FQ_BF16) return fq_fail(dev, FQ_ERR_UNSUPPORTED, "element type %d", dtype);
    if (n == 0 || n % 4 || rows == 0) return fq_fail(dev, FQ_ERR_SHAPE, "%u rows of %u values in 8 bits (a multiple of 4)", rows, n);
    const size_t count = (size_t)rows * n;
    if (rows > 0x7fffffffu || count > SIZE_MAX >> 4) return fq_fail(dev, FQ_ERR_SHAPE, "too many rows"); // (bytes that pass 64 bits would pass the checks)
    const size_t bytes = count * fq_dtype_size(dtype);
    if (int rc = fq_check_binding(dev, x, bytes, "x")) return rc;
    if (r)
        if (int rc = fq_check_binding(dev, r, bytes, "r")) return rc;
    if (norm)
        if (int rc = fq_check_binding(dev, w, (size_t)n * 4, "w")) return rc;
    if (int rc = fq_check_binding(dev, q, count, "q")) return rc;
    if (int rc = fq_check_binding(dev, scales, (size_t)rows * 4, "scales", 4)) return rc;
    const struct { const void *p; size_t bytes; const char *name; } in[3] = {{x, bytes, "x"}, {r, bytes, "r"}, {w, (size_t)n * 4, "w"}};
    for (const auto &i : in) {
        if (!i.p) continue;
        if (int rc = fq_check_apart(dev, q, count, i.p, i.bytes, "q")) return rc;
        if (int rc = fq_check_apart(dev, scales, (size_t)rows * 4, i.p, i.bytes, "scales")) return rc;
        if (int rc = fq_check_input(dev, i.p, i.bytes, i.name)) return rc;
    }
    return fq_check_apart(dev, scales, (size_t)rows * 4, q, count, "scales");
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
        if (int rc = fq_check_apart(dev, h, bytes, x, bytes, "h")) return rc;
    if (h != r)
        if (int rc = fq_check_apart(dev, h, bytes, r, bytes, "h")) return rc;
    if (int rc = fq_check_apart(dev, h, bytes, w, (size_t)n * 4, "h")) return rc;
    if (int rc = fq_check_apart(dev, q, count, h, bytes, "q")) return rc;
    if (int rc = fq_check_apart(dev, scales, (size_t)rows * 4, h, bytes, "scales")) return rc;
    return launch_rows<ADD_NORM>(dev, "add_rmsnorm_i8", x, r, x_dtype, w, n, eps, rows, h, q, scales);
}

extern "C" int fq_glu_i8(fq_device *dev, const void *gate, const void *up, int dtype, uint32_t n, uint32_t rows, int8_t *q, float *scales) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    if (!up) return fq_fail(dev, FQ_ERR_RANGE, "up: null binding");
    if (int rc = check_rows(dev, gate, up, dtype, nullptr, false, n, rows, q, scales)) return rc;
    return launch_rows<GLU>(dev, "glu_i8", gate, up, dtype, nullptr, n, 0.f, rows, nullptr, q, scales);
}

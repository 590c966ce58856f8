// Projections of 8-bit rows by 8-bit matrices on the fifth-generation tensor cores (kind::i8, sums in tensor memory):
//
//   y[t][o] = (sum_k x[t][k] w[o][k]) * x_scale[t] * w_scale[o]
//
// The sum is a whole number of at most 2^14 * 65536 < 2^31 and exact at every width and however it is cut; it is converted to
// fp32 once, multiplied by the token's scale and then by the row's, and rounded to the output's type.
//
// Weights sit on the MMA's M side (128 rows), tokens on its N side (16..256), so one kernel serves one token and a prompt.
// `fq_matrix_create_i8` lays the matrix out in tiles of 128 rows x 128 bytes of K, each stored in the 128-byte-swizzled order
// in which the MMA reads shared memory, one after the other along K: a tile is one contiguous copy of 16 KB without a tensor
// map, and a block's share of the weights is one run of memory.
//
//   warp 0       one thread copies the weight tiles (cp.async.bulk) and, by TMA, the tokens' 128 bytes of K beside them;
//   warp 1       one thread issues tcgen05.mma (M = 128, N = the token tile, K = 32, four per stage);
//   warps 2..5   read the accumulator, scale and store.  The accumulator is double: the next tile's MMAs run meanwhile.
//
// Blocks walk (row tile, token tile) items.  Where there are fewer items than blocks the machine holds, a cluster of up to
// eight blocks cuts an item's K and adds the partial sums (whole numbers, so in any order) through distributed shared memory:
// block r of the cluster collects and stores the tokens of its share, which the others send as one bulk copy each (value by
// value, remote stores took 45 us for q|k|v of 128 rows where these took 24).  All waits are bounded (tcgen05.cuh).
//
// Up to about 128 tokens HBM bounds it (gate|up, 2 x 17408 x 5120: 16 tokens 27.7 us, 6.5 TB/s), from there the tensor pipe (2048
// tokens 215 us, 3.4 POP/s, 95 % active); small matrices the launch and the filling of the ring (q|k|v of one token 9.1 us).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>

#include "gemv_common.cuh"
#include "internal.h"
#include "tcgen05.cuh"

namespace {
using namespace fqtc;
using fqk::pdl_trigger;
using fqk::pdl_wait;

constexpr uint32_t BM = 128;              // weight rows of a tile (MMA M)
constexpr uint32_t BK = 128;              // bytes of K of a stage: one swizzle row
constexpr uint32_t TILE_BYTES = BM * BK;
constexpr uint32_t MAX_STAGES = 12;
constexpr uint32_t MAX_MANY = 8, MAX_SLICES = 8;
constexpr uint32_t EPILOGUE_WARPS = 4, THREADS = (2 + EPILOGUE_WARPS) * 32;
constexpr uint32_t SMEM_MAX = 227 * 1024;
constexpr uint64_t DRAIN_NS = 200000;

struct Target {
    const uint8_t *w; // tiles
    const float *scales;
    void *y;
    uint32_t rows;
    uint32_t tile_end; // row tiles up to and including this matrix
};
struct Job {
    Target t[MAX_MANY];
    const float *x_scales;
    uint32_t count, m;
    uint32_t k_blocks;           // of the whole K
    uint32_t bn, token_tiles;    // tokens of a tile (a multiple of 16) and how many tiles cover m
    uint32_t items;              // row tiles of all matrices * token_tiles
    uint32_t slices, per;        // blocks of a cluster, k-blocks each
    uint32_t stages, box_bytes;  // of the ring; bytes of one TMA box of tokens
    uint32_t tmem_cols;
    int bf16;
};

struct Ctl {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2], drained, received;
    uint32_t tmem_base, abort_flag;
};

// kind::i8: D = s32, A = B = s8, both K-major.
__device__ __forceinline__ uint32_t idesc_i8(uint32_t m, uint32_t n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24); }
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_address(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
// From this block's shared memory to another's, whose barrier learns of it (cluster addresses).
__device__ __forceinline__ void bulk_send(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(smem_u32(src)), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

// Where an item lies: its matrix, row tile and token tile.  Token tiles run fastest, so that blocks that run together share
// weight tiles in L2.
struct Place {
    uint32_t which, tile, m0;
};
__device__ __forceinline__ Place place_of(const Job &J, uint32_t item) {
    Place p;
    uint32_t tile = item / J.token_tiles, first = 0;
    p.m0 = (item - tile * J.token_tiles) * J.bn;
    p.which = 0;
    for (uint32_t i = 0; i + 1 < J.count; i++)
        if (tile >= J.t[i].tile_end) {
            p.which = i + 1;
            first = J.t[i].tile_end;
        }
    p.tile = tile - first;
    return p;
}

__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
// The scales of a token tile, in shared memory of the warp's own; asked for before the accumulator is waited for.
__device__ __forceinline__ void stage_scales(const Job &J, uint32_t m0, uint32_t live, float *xs, uint32_t lane) {
    __syncwarp(); // the tile before has been stored
    for (uint32_t c = lane; c < live; c += 32) xs[c] = __ldcg(J.x_scales + m0 + c);
    __syncwarp();
}
// `live` tokens from m0 of the accumulator at `acc`: one weight row a lane, so that a warp's stores of a token are contiguous.
template <typename YT>
__device__ __forceinline__ void store_rows(YT *y, uint32_t rows, uint32_t acc, uint32_t live, bool in, float ws, const float *xs) {
    for (uint32_t c0 = 0; c0 < live; c0 += 16) {
        int v[16];
        tmem_ld16(acc + c0, v);
        if (!in) continue;
        const float4 *x4 = reinterpret_cast<const float4 *>(xs + c0);
#pragma unroll
        for (uint32_t c = 0; c < 16; c++) {
            const float4 x = x4[c / 4];
            if (c0 + c < live) put(y, (float)v[c] * (c % 4 == 0 ? x.x : c % 4 == 1 ? x.y : c % 4 == 2 ? x.z : x.w) * ws);
            y += rows;
        }
    }
}
__device__ __forceinline__ void store_tile(const Job &J, const Target &T, uint32_t acc, uint32_t m0, uint32_t live, uint32_t row, float ws, const float *xs) {
    const size_t at = (size_t)m0 * T.rows + row;
    if (J.bf16) store_rows(static_cast<__nv_bfloat16 *>(T.y) + at, T.rows, acc, live, row < T.rows, ws, xs);
    else store_rows(static_cast<float *>(T.y) + at, T.rows, acc, live, row < T.rows, ws, xs);
}

// The same of partial sums in shared memory, [token][row]: this block's and, `stride` apart, those of the others.
template <typename YT>
__device__ __forceinline__ void store_sums(YT *y, uint32_t rows, uint32_t tokens, const int *sums, const int *others, uint32_t blocks, uint32_t stride, const float *xs, float ws) {
    constexpr uint32_t AHEAD = 8; // tokens whose loads are under way together (one at a time took 150 clocks each)
    for (uint32_t c0 = 0; c0 < tokens; c0 += AHEAD) {
        int v[AHEAD];
#pragma unroll
        for (uint32_t c = 0; c < AHEAD; c++) v[c] = c0 + c < tokens ? sums[(c0 + c) * BM] : 0;
        for (uint32_t from = 0; from < blocks; from++)
#pragma unroll
            for (uint32_t c = 0; c < AHEAD; c++)
                if (c0 + c < tokens) v[c] += others[from * stride + (c0 + c) * BM];
#pragma unroll
        for (uint32_t c = 0; c < AHEAD; c++) {
            if (c0 + c < tokens) put(y, (float)v[c] * xs[c0 + c] * ws);
            y += rows;
        }
    }
}

template <bool SLICED>
__global__ void __launch_bounds__(THREADS)
k_gemm_i8(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ Job J, int *status) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ Ctl ctl;
    __shared__ __align__(16) float xs[EPILOGUE_WARPS][256];
    uint8_t *ring = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stage_bytes = TILE_BYTES + J.bn * BK;
    const uint32_t slice = SLICED ? blockIdx.x % J.slices : 0, unit = SLICED ? blockIdx.x / J.slices : blockIdx.x, units = SLICED ? gridDim.x / J.slices : gridDim.x;
    const uint32_t k_first = slice * J.per, k_iters = min(J.per, J.k_blocks - k_first);
    pdl_trigger();
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < J.stages; s++) {
            mbar_init(&ctl.full[s], 1);
            mbar_init(&ctl.empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&ctl.acc_full[b], 1);
            mbar_init(&ctl.acc_empty[b], EPILOGUE_WARPS * 32);
        }
        mbar_init(&ctl.drained, 1);
        mbar_init(&ctl.received, 1);
        ctl.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&xmap) : "memory");
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"(J.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *(volatile uint32_t *)&ctl.tmem_base;

    if (warp == 0) {
        if (elect_one()) {
            auto weights = [&](const Place &p, uint32_t it) {
                return J.t[p.which].w + ((size_t)p.tile * J.k_blocks + k_first + it) * TILE_BYTES;
            };
            // The weights are nobody's output: the first ones are under way before the kernel ahead has finished.
            const uint32_t primed = unit < J.items ? min(J.stages, k_iters) : 0;
            for (uint32_t it = 0; it < primed; it++) {
                mbar_expect_tx(&ctl.full[it], TILE_BYTES + J.box_bytes);
                bulk_load(ring + it * stage_bytes, weights(place_of(J, unit), it), TILE_BYTES, &ctl.full[it]);
            }
            pdl_wait();
            uint32_t s = 0, phase = 0, issued = 0;
            bool ok = true;
            for (uint32_t item = unit; item < J.items && ok; item += units) {
                const Place p = place_of(J, item);
                for (uint32_t it = 0; it < k_iters; it++) {
                    if (issued >= primed) {
                        if (!(ok = mbar_wait(&ctl.empty[s], phase ^ 1, &ctl, status))) break;
                        mbar_expect_tx(&ctl.full[s], TILE_BYTES + J.box_bytes);
                        bulk_load(ring + s * stage_bytes, weights(p, it), TILE_BYTES, &ctl.full[s]);
                    }
                    tma_load_2d(ring + s * stage_bytes + TILE_BYTES, &xmap, (int)((k_first + it) * BK), (int)p.m0, &ctl.full[s]);
                    issued++;
                    if (++s == J.stages) s = 0, phase ^= 1;
                }
            }
            // After an abort the copies under way still land: wait for them (bounded) before the shared memory goes away.
            if (*(volatile uint32_t *)&ctl.abort_flag)
                for (uint32_t ib = issued > J.stages ? issued - J.stages : 0; ib < issued; ib++)
                    for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try(&ctl.full[ib % J.stages], (ib / J.stages) & 1); i++) {}
        }
    } else if (warp == 1) {
        if (elect_one()) {
            pdl_wait(); // the clock of the bounded waits starts when there is something to wait for
            const uint32_t idesc = idesc_i8(BM, J.bn);
            uint32_t s = 0, phase = 0, buf = 0, buf_phase = 0;
            bool ok = true;
            for (uint32_t item = unit; item < J.items && ok; item += units) {
                if (!mbar_wait(&ctl.acc_empty[buf], buf_phase ^ 1, &ctl, status)) break;
                const uint32_t acc = tmem + buf * J.bn;
                for (uint32_t it = 0; it < k_iters; it++) {
                    if (!(ok = mbar_wait(&ctl.full[s], phase, &ctl, status))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_u32(ring + s * stage_bytes);
                    const uint64_t a = umma_desc(at), b = umma_desc(at + TILE_BYTES);
#pragma unroll
                    for (uint32_t k = 0; k < BK / 32; k++) umma_i8(acc, a + 2 * k, b + 2 * k, idesc, (it | k) != 0);
                    umma_commit(&ctl.empty[s]);
                    if (++s == J.stages) s = 0, phase ^= 1;
                }
                if (ok) umma_commit(&ctl.acc_full[buf]);
                if (++buf == 2) buf = 0, buf_phase ^= 1;
            }
            // Everything this thread issued has finished (after an abort too) before the accumulators are released.
            umma_commit(&ctl.drained);
            for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try(&ctl.drained, 0, WAIT_HINT_NS); i++) {}
        }
    } else {
        pdl_wait(); // x_scales may be, and what y held may still be in use by, the kernel ahead
    }

    const uint32_t quarter = warp & 3; // the tensor-memory lanes a warp may read
    if constexpr (!SLICED) {
        if (warp >= 2) {
            uint32_t buf = 0, buf_phase = 0;
            for (uint32_t item = unit; item < J.items; item += units) {
                const Place p = place_of(J, item);
                const Target &T = J.t[p.which];
                const uint32_t row = p.tile * BM + 32 * quarter + lane, live = min(J.bn, J.m - p.m0);
                const float ws = row < T.rows ? T.scales[row] : 0.f;
                stage_scales(J, p.m0, live, xs[quarter], lane);
                if (!__all_sync(0xffffffffu, mbar_wait(&ctl.acc_full[buf], buf_phase, &ctl, status))) break; // the warp agrees
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                store_tile(J, T, tmem + buf * J.bn + ((32 * quarter) << 16), p.m0, live, row, ws, xs[quarter]);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                mbar_arrive(&ctl.acc_empty[buf]);
                if (++buf == 2) buf = 0, buf_phase ^= 1;
            }
        }
    } else { // one item per cluster; every thread passes both barriers whatever happened
        const Place p = place_of(J, unit);
        const Target &T = J.t[p.which];
        const uint32_t live = min(J.bn, J.m - p.m0), share = (live + J.slices - 1) / J.slices;
        const uint32_t mine = min(live, slice * share), mine_end = min(live, mine + share), acc = tmem + ((32 * quarter) << 16);
        const uint32_t row = p.tile * BM + 32 * quarter + lane;
        int *sums = reinterpret_cast<int *>(ring) + 32 * quarter + lane, *others = sums + J.bn * BM; // [token][row]; [block][token][row]
        float ws = 0.f;
        if (threadIdx.x == 0 && mine_end > mine) mbar_expect_tx(&ctl.received, (J.slices - 1) * (mine_end - mine) * BM * 4);
        if (warp >= 2) {
            if (row < T.rows) ws = T.scales[row];
            stage_scales(J, p.m0, live, xs[quarter], lane);
            if (mbar_wait(&ctl.acc_full[0], 0, &ctl, status)) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        __syncthreads();
        cluster_sync(); // every block's MMAs have read their ring (or given up): it takes the sums now
        if (warp >= 2 && *(volatile uint32_t *)&ctl.abort_flag == 0) {
            for (uint32_t c0 = 0; c0 < live; c0 += 16) {
                int v[16];
                tmem_ld16(acc + c0, v);
#pragma unroll
                for (uint32_t c = 0; c < 16; c++)
                    if (c0 + c < live) sums[(c0 + c) * BM] = v[c];
            }
            asm volatile("fence.proxy.async.shared::cta;\nbar.sync 1, 128;" ::: "memory");
            if (threadIdx.x == 64)
                for (uint32_t to = 0; to < J.slices; to++) {
                    const uint32_t first = min(live, to * share), n = min(live, first + share) - first;
                    if (to == slice || n == 0) continue;
                    const uint32_t from = slice < to ? slice : slice - 1;
                    bulk_send(cluster_address(smem_u32(ring), to) + (J.bn + from * share) * BM * 4, ring + first * BM * 4, n * BM * 4, cluster_address(smem_u32(&ctl.received), to));
                }
            if (mine_end > mine && mbar_wait(&ctl.received, 0, &ctl, status) && row < T.rows) {
                const size_t at = (size_t)(p.m0 + mine) * T.rows + row;
                if (J.bf16) store_sums(static_cast<__nv_bfloat16 *>(T.y) + at, T.rows, mine_end - mine, sums + mine * BM, others, J.slices - 1, share * BM, xs[quarter] + mine, ws);
                else store_sums(static_cast<float *>(T.y) + at, T.rows, mine_end - mine, sums + mine * BM, others, J.slices - 1, share * BM, xs[quarter] + mine, ws);
            }
        }
        __syncwarp();
        cluster_sync(); // what a block sent has been received
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(J.tmem_cols) : "memory");
}

// Many tokens: two blocks of a cluster share one MMA (cta_group::2, M = 256): each holds 128 of the 256 weight rows and half of
// the tokens in its shared memory, and the sums of its own rows in its tensor memory.  A block then takes in 16 KB of weights
// and only half of a token tile for as many products, and what it takes in per product is what binds the kernel above.
//
// The even block issues the MMAs.  Both blocks' copies report to its barriers (TMA with .cta_group::2; through a thread of the
// other block that waits and passes the arrival on, down, 509 tokens by 5120 x 17408, took 50 instead of then 48 us); the commits
// that release a stage and hand over an accumulator arrive in both blocks; both blocks' epilogues return the accumulator to the even one.
struct PairMaps {
    CUtensorMap x, w[MAX_MANY]; // tokens; the tiles of each matrix as rows of 128 bytes
};
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) { // bar: cluster address
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint64_t *bar) { // arrives at this barrier in both blocks
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive_at(uint64_t *bar, uint32_t rank) { // the same barrier of block `rank` of the cluster
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_address(smem_u32(bar), rank)) : "memory");
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS)
k_gemm_i8_pair(const __grid_constant__ PairMaps maps, const __grid_constant__ Job J, int *status) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ Ctl ctl;
    __shared__ __align__(16) float xs[EPILOGUE_WARPS][256];
    uint8_t *ring = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023); // the same place in both blocks
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x & 1, unit = blockIdx.x >> 1, units = gridDim.x >> 1;
    const uint32_t half = J.bn / 2, stage_bytes = TILE_BYTES + half * BK;
    pdl_trigger();
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < J.stages; s++) {
            mbar_init(&ctl.full[s], 1);
            mbar_init(&ctl.empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&ctl.acc_full[b], 1);
            mbar_init(&ctl.acc_empty[b], 2 * EPILOGUE_WARPS);
        }
        mbar_init(&ctl.drained, 1);
        ctl.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.x) : "memory");
    }
    __syncthreads();
    cluster_sync(); // both blocks run and their barriers are there
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"(J.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync(); // both have their accumulators
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *(volatile uint32_t *)&ctl.tmem_base;

    if (warp == 0) {
        if (elect_one()) {
            const uint32_t both = 2 * (TILE_BYTES + J.box_bytes);
            auto weights = [&](const Place &p, uint32_t it, uint32_t s) {
                if (rank == 0) mbar_expect_tx(&ctl.full[s], both); // (the other block's copies may report before)
                tma_load_pair(ring + s * stage_bytes, &maps.w[p.which], 0, (int)(((2 * p.tile + rank) * J.k_blocks + it) * BM), cluster_address(smem_u32(&ctl.full[s]), 0));
            };
            const uint32_t primed = unit < J.items ? min(J.stages, J.k_blocks) : 0;
            for (uint32_t it = 0; it < primed; it++) weights(place_of(J, unit), it, it);
            pdl_wait();
            uint32_t s = 0, phase = 0, issued = 0;
            bool ok = true;
            for (uint32_t item = unit; item < J.items && ok; item += units) {
                const Place p = place_of(J, item);
                for (uint32_t it = 0; it < J.k_blocks; it++) {
                    if (issued >= primed) {
                        if (!(ok = mbar_wait(&ctl.empty[s], phase ^ 1, &ctl, status))) break;
                        weights(p, it, s);
                    }
                    tma_load_pair(ring + s * stage_bytes + TILE_BYTES, &maps.x, (int)(it * BK), (int)(p.m0 + rank * half), cluster_address(smem_u32(&ctl.full[s]), 0));
                    issued++;
                    if (++s == J.stages) s = 0, phase ^= 1;
                }
            }
            // After an abort the copies under way still land, some of them reporting to the other block: they are given time.
            if (*(volatile uint32_t *)&ctl.abort_flag)
                for (const uint64_t t0 = now_ns(); now_ns() - t0 < DRAIN_NS;) {}
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            pdl_wait();
            const uint32_t idesc = idesc_i8(2 * BM, J.bn);
            uint32_t s = 0, phase = 0, buf = 0, buf_phase = 0;
            bool ok = true;
            for (uint32_t item = unit; item < J.items && ok; item += units) {
                if (!mbar_wait(&ctl.acc_empty[buf], buf_phase ^ 1, &ctl, status)) break;
                const uint32_t acc = tmem + buf * J.bn;
                for (uint32_t it = 0; it < J.k_blocks; it++) {
                    if (!(ok = mbar_wait(&ctl.full[s], phase, &ctl, status))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_u32(ring + s * stage_bytes);
                    const uint64_t a = umma_desc(at), b = umma_desc(at + TILE_BYTES);
#pragma unroll
                    for (uint32_t k = 0; k < BK / 32; k++) umma_i8_pair(acc, a + 2 * k, b + 2 * k, idesc, (it | k) != 0);
                    umma_commit_pair(&ctl.empty[s]);
                    if (++s == J.stages) s = 0, phase ^= 1;
                }
                if (ok) umma_commit_pair(&ctl.acc_full[buf]);
                if (++buf == 2) buf = 0, buf_phase ^= 1;
            }
            // Everything this thread issued has finished before either block goes on to its end.
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&ctl.drained)) : "memory");
            for (uint32_t i = 0; i < WAIT_LIMIT && !mbar_try(&ctl.drained, 0, WAIT_HINT_NS); i++) {}
        }
    } else {
        pdl_wait();
        const uint32_t quarter = warp & 3;
        uint32_t buf = 0, buf_phase = 0;
        for (uint32_t item = unit; item < J.items; item += units) {
            const Place p = place_of(J, item);
            const Target &T = J.t[p.which];
            const uint32_t row = (2 * p.tile + rank) * BM + 32 * quarter + lane, live = min(J.bn, J.m - p.m0);
            const float ws = row < T.rows ? T.scales[row] : 0.f;
            stage_scales(J, p.m0, live, xs[quarter], lane);
            if (!__all_sync(0xffffffffu, mbar_wait(&ctl.acc_full[buf], buf_phase, &ctl, status))) break; // the warp agrees
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            store_tile(J, T, tmem + buf * J.bn + ((32 * quarter) << 16), p.m0, live, row, ws, xs[quarter]);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_at(&ctl.acc_empty[buf], 0);
            if (++buf == 2) buf = 0, buf_phase ^= 1;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync(); // no MMA reads, and no arrival is on its way to, a block that is gone
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(J.tmem_cols) : "memory");
    }
}

// A matrix of rows of `cols` bytes as swizzled tiles: 16 bytes a thread, zero past the matrix's end.
__global__ void __launch_bounds__(256) k_tile_i8(const uint8_t *__restrict__ src, uint64_t rows, uint64_t cols, uint32_t k_blocks,
                                                        uint8_t *__restrict__ dst) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; // 1024 chunks a tile, eight a row; four blocks a tile
    const uint64_t tile = i >> 10, row = (tile / k_blocks) * BM + ((i >> 3) & 127), k = (tile % k_blocks) * BK + (i & 7) * 16;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < rows && k < cols) v = *reinterpret_cast<const uint4 *>(src + row * cols + k);
    const uint32_t r = (uint32_t)(i >> 3) & 127, chunk = (uint32_t)(i & 7) ^ (r & 7);
    *reinterpret_cast<uint4 *>(dst + (tile << 14) + r * 128 + chunk * 16) = v;
}

// How a product is cut: tokens of a tile, the blocks among which an item's K is shared, pairs or single blocks.
struct Plan {
    uint32_t bn, token_tiles, slices, per, stages;
    bool pair;
};
uint32_t stage_bytes(const Plan &p) { return TILE_BYTES + (p.pair ? p.bn / 2 : p.bn) * BK; }
// By an estimate of clocks, one block per SM (two with half the ring each were slower wherever they differed):
//   - a k-block takes its four MMAs (40 / 48 / 64 / 128 clocks each at N = 32 / 64 / 128 / 256, and 1.3 times that with the
//     waits between them), or as long as its bytes need: one
//     SM streams weights at 57 bytes a clock, L2 feeds all of them 6500 a clock; the first ring of it comes at once;
//   - HBM delivers 3440 bytes of weights a clock;
//   - a cluster's exchange takes 1300 clocks and 55 a token; a pair's start 1000.
// us, estimated best against the other (rows x cols, tokens): 5120 x 17408, 1: three slices 16.3, two 17.1, one 21.1; 8192 x 5120, 1: one
// 9.1, two 9.9, 64: one 10.8, two 13.2; 34816 x 5120, 2048: pairs 224, single blocks 335.
Plan plan(const fq_device *dev, const fq_matrix *const *w, uint32_t count, uint32_t k_blocks, uint32_t m) {
    const uint32_t sms = (uint32_t)dev->sm_count;
    uint32_t tiles = 0, pairs = 0;
    for (uint32_t i = 0; i < count; i++) {
        tiles += (uint32_t)((w[i]->rows + BM - 1) / BM);
        pairs += (uint32_t)((w[i]->rows + 2 * BM - 1) / (2 * BM));
    }
    const double hbm = (double)tiles * k_blocks * TILE_BYTES / 3440.0;
    Plan p{};
    double best = 0.0;
    auto consider = [&](uint32_t token_tiles, bool pair, uint32_t slices) {
        const uint32_t step = pair ? 32 : 16;
        Plan c{};
        c.pair = pair;
        c.bn = ((m + token_tiles - 1) / token_tiles + step - 1) / step * step;
        if (c.bn > 256) return;
        c.token_tiles = (m + c.bn - 1) / c.bn;
        c.per = (k_blocks + slices - 1) / slices;
        c.slices = (k_blocks + c.per - 1) / c.per; // no slice is left without work
        c.stages = std::min((SMEM_MAX - 8192) / stage_bytes(c), MAX_STAGES);
        const uint32_t items = (pair ? pairs : tiles) * c.token_tiles, slots = pair ? sms / 2 : sms;
        if (c.slices > 1) { // all at once, and the sums fit where the ring was
            if (items > dev->i8_clusters[c.slices]) return;
            if ((c.bn + (c.slices - 1) * ((c.bn + c.slices - 1) / c.slices)) * BM * 4 > c.stages * stage_bytes(c)) return;
        }
        const double active = std::min(items * c.slices, slots) * (pair ? 2.0 : 1.0), mma = 5.2 * std::max(32.0 + c.bn / 4.0, c.bn / 2.0);
        const double feed = std::max(TILE_BYTES / 57.0 + (stage_bytes(c) - TILE_BYTES) / 300.0, stage_bytes(c) * active / 6500.0);
        const double rounds = (items + slots - 1) / slots, ring = std::min(c.per, 8u) * std::max(0.0, feed - mma);
        const double cost = std::max(hbm, rounds * c.per * std::max(mma, feed) - ring) + 6.0 * c.bn + (c.slices > 1 ? 1300.0 + 55.0 * c.bn : 0.0) + (pair ? 1000.0 : 0.0);
        if (p.bn == 0 || cost <= best) { // (of equals the one with more blocks)
            best = cost;
            p = c;
        }
    };
    for (uint32_t t = (m + 255) / 256; t <= (m + 255) / 256 + 7 && t <= (m + 15) / 16; t++) {
        for (uint32_t slices = 1; slices <= std::min(MAX_SLICES, k_blocks) && (slices == 1 || tiles * t * slices <= sms); slices++) consider(t, false, slices);
        consider(t, true, 1);
    }
    return p;
}

// Once per handle: the kernels may use all of an SM's shared memory, and how many clusters of each size run at once (a cluster's
// blocks share a GPC, so fewer than blocks would).
cudaError_t prepare_device(fq_device *dev) {
    if (dev->i8_clusters[1]) return cudaSuccess;
    for (const void *kernel : {(const void *)k_gemm_i8<false>, (const void *)k_gemm_i8<true>, (const void *)k_gemm_i8_pair})
        if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(SMEM_MAX - 6144))) return e;
    for (uint32_t slices = MAX_SLICES; slices >= 1; slices--) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(slices * (uint32_t)dev->sm_count);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = SMEM_MAX - 8192 + 1024;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = slices;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, k_gemm_i8<true>, &cfg)) return e;
        dev->i8_clusters[slices] = (uint16_t)clusters; // [1], the last, is never 0
    }
    return cudaSuccess;
}

// Rows of `cols` bytes for boxes of 128 bytes of `box_rows` rows.
int encode_bytes(fq_device *dev, CUtensorMap *map, const void *p, uint64_t cols, uint64_t rows, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    EncodeTiled encode = encode_fn();
    if (!encode) return fq_fail(dev, FQ_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols};
    const cuuint32_t box[2] = {BK, box_rows}, step[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FQ_OK : fq_fail(dev, FQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

int launch(fq_device *dev, const fq_matrix *const *w, uint32_t count, const int8_t *x, const float *x_scales, uint32_t m, void *const *y, int y_dtype) {
    const uint32_t cols = (uint32_t)w[0]->cols, k_blocks = (cols + BK - 1) / BK;
    const Plan p = plan(dev, w, count, k_blocks, m);
    Job J{};
    uint32_t tiles = 0; // of 128 rows, or for pairs of 256
    for (uint32_t i = 0; i < count; i++) {
        const uint32_t bm = p.pair ? 2 * BM : BM;
        tiles += (uint32_t)((w[i]->rows + bm - 1) / bm);
        J.t[i] = {w[i]->data, w[i]->scales, y[i], (uint32_t)w[i]->rows, tiles};
    }
    J.x_scales = x_scales;
    J.count = count;
    J.m = m;
    J.k_blocks = k_blocks;
    J.bn = p.bn;
    J.token_tiles = p.token_tiles;
    J.items = tiles * p.token_tiles;
    J.slices = p.slices;
    J.per = p.per;
    J.stages = p.stages;
    J.bf16 = y_dtype == FQ_BF16;
    for (J.tmem_cols = 32; J.tmem_cols < 2 * p.bn;) J.tmem_cols *= 2;
    CUtensorMap map;
    const uint32_t box_rows = std::min(m, p.pair ? p.bn / 2 : p.bn);
    if (int rc = encode_bytes(dev, &map, x, cols, m, box_rows, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    J.box_bytes = box_rows * BK;
    cudaLaunchConfig_t cfg{};
    const uint32_t sms = (uint32_t)dev->sm_count;
    cfg.gridDim = dim3(p.pair ? 2 * std::min(J.items, sms / 2) : p.slices > 1 ? J.items * p.slices : std::min(J.items, sms));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = 1024 + p.stages * stage_bytes(p);
    cfg.stream = dev->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.slices;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.slices > 1 ? 2 : 1;
    cudaError_t e;
    if (p.pair) {
        PairMaps maps;
        maps.x = map;
        for (uint32_t i = 0; i < count; i++) memcpy(&maps.w[i], w[i]->tile_map, sizeof(CUtensorMap));
        e = cudaLaunchKernelEx(&cfg, k_gemm_i8_pair, maps, J, dev->status_dev);
    } else {
        e = cudaLaunchKernelEx(&cfg, p.slices > 1 ? k_gemm_i8<true> : k_gemm_i8<false>, map, J, dev->status_dev);
    }
    return fq_check_cuda(dev, e, "8-bit projection launch");
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
    bool on_device = false; // the values
    const struct { const void *p; size_t bytes; const char *name; } payload[2] = {{scales, rows * 4, "scales"}, {values, rows * cols, "values"}};
    for (const auto &t : payload) {
        cudaPointerAttributes attr{};
        if (int rc = fq_check_cuda(dev, cudaPointerGetAttributes(&attr, t.p), "payload")) return rc;
        on_device = attr.type == cudaMemoryTypeDevice;
        if (!on_device) continue;
        if (attr.device != dev->ordinal) return fq_fail(dev, FQ_ERR_DEVICE, "the payload is on device %d", attr.device);
        if (int rc = fq_check_binding(dev, t.p, t.bytes, t.name, 1)) return rc;
        // What makes the payload has to have ended well: no later call would see that a matrix was made of anything else.
        if (int rc = fq_synchronize(dev)) return rc;
        if (int rc = fq_check_input(dev, t.p, t.bytes, t.name)) return rc;
    }
    const std::unique_ptr<float[]> host(new (std::nothrow) float[rows]);
    if (!host) return fq_fail(dev, FQ_ERR_CUDA, "no host memory for %llu scales", (unsigned long long)rows);
    cudaError_t e = cudaMemcpyAsync(host.get(), scales, rows * 4, cudaMemcpyDefault, dev->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(dev->stream);
    if (e != cudaSuccess) return fq_check_cuda(dev, e, "weight scales");
    for (uint64_t r = 0; r < rows; r++)
        if (!std::isfinite(host[r])) return fq_fail(dev, FQ_ERR_WEIGHT, "the scale of row %llu is not finite", (unsigned long long)r);
    fq_matrix *w = new (std::nothrow) fq_matrix();
    if (!w) return fq_fail(dev, FQ_ERR_CUDA, "no host memory for a matrix");
    w->dev = dev;
    w->format = FQ_I8;
    w->rows = rows;
    w->cols = cols;
    w->row_bytes = w->pitch = cols;
    w->byte_size = rows * (cols + 4);
    w->block_elems = w->block_bytes = 1;
    const uint32_t k_blocks = (uint32_t)((cols + BK - 1) / BK);
    const uint64_t tiles = (rows + 2 * BM - 1) / (2 * BM) * 2 * k_blocks; // an even number of row tiles, for pairs of blocks
    const size_t len = tiles * TILE_BYTES;
    // The tiles are laid out on the device; rows in host memory (or off their 16 bytes) go through a copy of their own.
    uint8_t *staged = nullptr;
    const uint8_t *src = (const uint8_t *)values;
    e = prepare_device(dev);
    if (e == cudaSuccess) e = cudaMalloc((void **)&w->data, len + rows * 4);
    w->scales = (float *)(w->data + len);
    if (e == cudaSuccess && (!on_device || ((uintptr_t)values & 15))) {
        e = cudaMalloc((void **)&staged, rows * cols);
        if (e == cudaSuccess) e = cudaMemcpyAsync(staged, values, rows * cols, cudaMemcpyDefault, dev->stream);
        src = staged;
    }
    if (e == cudaSuccess) {
        k_tile_i8<<<(unsigned)(tiles * 4), 256, 0, dev->stream>>>(src, rows, cols, k_blocks, w->data);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaMemcpyAsync(w->scales, host.get(), rows * 4, cudaMemcpyHostToDevice, dev->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(dev->stream);
    if (staged) cudaFree(staged);
    int rc = fq_check_cuda(dev, e, "weight upload");
    static_assert(sizeof(CUtensorMap) == sizeof w->tile_map, "fq_matrix holds a tensor map");
    if (!rc) rc = encode_bytes(dev, (CUtensorMap *)w->tile_map, w->data, BK, tiles * BM, BM, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc) {
        if (w->data) cudaFree(w->data);
        delete w;
        return rc;
    }
    dev->counters.bytes_uploaded += w->byte_size;
    *out = w;
    return FQ_OK;
}

extern "C" int fq_project_many_i8(fq_device *dev, const fq_matrix *const *w, size_t count, const int8_t *x, size_t x_elems, const float *x_scales,
                                  size_t m, void *const *y, int y_dtype) {
    if (int rc = fq_begin_enqueue(dev)) return rc;
    constexpr size_t MAX = MAX_MANY;
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
        if (int rc = fq_check_binding(dev, x_scales, m * 4, "x_scales", 4)) return rc;
        if (int rc = fq_check_binding(dev, y[i], yb, "y")) return rc;
        if (int rc = fq_check_apart(dev, y[i], yb, x, x_elems, "y")) return rc;
        if (int rc = fq_check_apart(dev, y[i], yb, x_scales, m * 4, "y")) return rc;
        for (size_t j = 0; j < i; j++)
            if (int rc = fq_check_apart(dev, y[i], yb, y[j], m * w[j]->rows * fq_dtype_size(y_dtype), "y")) return rc;
    }
    if (int rc = fq_check_input(dev, x, x_elems, "x")) return rc;
    if (int rc = fq_check_input(dev, x_scales, m * 4, "x_scales")) return rc;
    if (int rc = launch(dev, w, (uint32_t)count, x, x_scales, (uint32_t)m, y, y_dtype)) return rc;
    for (size_t i = 0; i < count; i++) fq_note_write(dev, y[i], m * w[i]->rows * fq_dtype_size(y_dtype));
    return fq_end_enqueue(dev, "project_i8", 1);
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

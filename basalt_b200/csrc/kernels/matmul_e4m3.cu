// e4m3 matmul with row scales for sm_100a:
//
//   C[m, n] = (sum_k A[m, k] * B[n, k]) * a_scales[m] * b_scales[n]
//
// A [M x K] and B [N x K] are e4m3 rows, the sums f32 in tensor memory (tcgen05.mma.kind::f8f6f4), the product with the
// two scales and the one rounding to C's type in the epilogue. Rows of B (a layer's weights) lie along the MMA's 128
// accumulator lanes and rows of A (tokens) along its columns, so one token costs a 16-column tile, not a 128-row one.
//
// A CTA computes 128 rows of B x TN rows of A over its share of K: thread 0 of warp 0 feeds a ring of shared-memory
// stages (128 bytes of K each) by bulk-tensor loads, thread 0 of warp 1 issues the MMAs, and all four warps drain
// the accumulator. Where there are fewer tiles than the GPU has room for, a cluster of up to eight
// CTAs shares one tile, each taking a run of K slabs: the partial sums meet in distributed shared memory and are added in
// the order of the CTAs, so the result depends on no race and needs no workspace. (Two such CTAs fit an SM, and their tensor memory,
// 256 columns at most, with them; no CTA that waits for its cluster can be kept from starting by another's.)
// Ragged edges are the tensor maps' business: what lies outside a matrix is read as zero.
// What bounds it: for one row the weights, 14.2 us for 8192 x 8192 (4.7 TB/s; a plain stream of as many bytes takes 11.4 to 12.3, the rest is the
// way of the first and the last slab); for many rows see the pairs of CTAs below, 8192^3 in 374 to 382 us in a burst (2.9 PFLOP/s) and 419 to 445 at the 1.2 GHz
// that the power cap leaves.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "../../../include/basalt_b200_kernels.h"
#include "common.cuh"
#include "tensor_core.cuh"

namespace {

using namespace basalt_k::tc;

constexpr int BN = 128, BK = 128, THREADS = 128, B_BYTES = BN * BK, MMA_K = 32;

__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <class T>
__device__ __forceinline__ uint32_t two_as(float a, float b) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

template <int TN>
__host__ __device__ constexpr int stages_of() { return TN == 16 ? 5 : TN <= 64 ? 4 : 3; }
template <int TN>
__host__ __device__ constexpr int ring_of() { return stages_of<TN>() * (B_BYTES + TN * BK); }
// Where the partial sums of a cluster meet: behind the ring where there is room, so that no CTA waits for the others' rings; else in it.
template <int TN>
__host__ __device__ constexpr int sums_at() { return TN <= 32 ? ring_of<TN>() : 0; }
template <int TN>
__host__ __device__ constexpr int smem_of() { return ring_of<TN>() + (TN <= 32 ? TN * BN * 4 : 0) + 1024; }   // at most 99 KB: two CTAs fit an SM

// C = v, or C += v (f32 alone: a later part of a long K, see launch_type)
template <class T>
__device__ __forceinline__ void store_sum(T* c, float v, int add) {
    if constexpr (sizeof(T) == 4)
        if (add) v += *c;
    store_as(c, v);
}

// The scales are no __restrict__ pointers here and below: the kernel before, which may still run when this one begins, writes them, and a pointer that
// promises memory nobody writes could be read before the wait for it.
template <class T, int TN>
__global__ void __launch_bounds__(THREADS) matmul_e4m3_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
                                                              const float* a_scales, const float* b_scales, T* __restrict__ C,
                                                              int64_t ldc, int M, int N, int K, int shift, int add, int32_t* status) {
    constexpr int STAGES = stages_of<TN>(), A_BYTES = TN * BK, STAGE_BYTES = B_BYTES + A_BYTES;
    constexpr uint32_t TMEM_COLS = TN < 32 ? 32 : TN;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], acc_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t gave_up;
    __shared__ float scale[TN];   // of the tile's rows of A: in the epilogue each would be a trip to memory
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int splits = 1 << shift, split = blockIdx.x & (splits - 1), n0 = (blockIdx.x >> shift) * BN, m0 = blockIdx.y * TN;
    const int slabs = (K - 1) / BK + 1, first = slabs * split >> shift, count = (slabs * (split + 1) >> shift) - first;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        mbar_init(smem_u32(&acc_bar), 1);
        prefetch_map(&map_a);
        prefetch_map(&map_b);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_arrive();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_acc = tmem_slot;
    wait_for_predecessor();
    if (threadIdx.x == 0 && status && *reinterpret_cast<volatile int32_t*>(status) != 0) gave_up = 1;   // an earlier CTA gave up: do not pile on
    bool ok = true;
    const float b_scale = n0 + (int)threadIdx.x < N ? b_scales[n0 + threadIdx.x] : 0.0f;

    if (warp == 0 && lane == 0) {
        for (int i = 0; i < count; i++) {
            const int s = i % STAGES;
            ok &= mbar_wait(smem_u32(&empty_bar[s]), ((i / STAGES) & 1) ^ 1, &gave_up);
            if (!ok) break;
            const uint32_t fb = smem_u32(&full_bar[s]), b_dst = tiles + s * STAGE_BYTES, a_dst = b_dst + B_BYTES;
            mbar_expect_tx(fb, STAGE_BYTES);
            tma_load_2d(b_dst, &map_b, fb, (first + i) * BK, n0);
            tma_load_2d(a_dst, &map_a, fb, (first + i) * BK, m0);
        }
        if (!ok) {   // let the copies already issued land before the CTA can exit
            const uint64_t t0 = global_ns();
            while (global_ns() - t0 < 2000000ull) {}
        }
    } else if (warp == 1 && lane == 0) {
        // D = f32 (bits 4-5 = 1), both operands e4m3 (0) and K-major, N/8 in bits 17-22, M/16 in bits 24-28
        const uint32_t idesc = (1u << 4) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(BN >> 4) << 24);
        for (int i = 0; i < count; i++) {
            const int s = i % STAGES;
            ok &= mbar_wait(smem_u32(&full_bar[s]), (i / STAGES) & 1, &gave_up);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t b_src = tiles + s * STAGE_BYTES, a_src = b_src + B_BYTES;
            const uint64_t db = smem_desc(b_src, 16, 1024), da = smem_desc(a_src, 16, 1024);
#pragma unroll
            for (int k = 0; k < BK / MMA_K; k++) umma_f8(tmem_acc, db + (uint64_t)(2 * k), da + (uint64_t)(2 * k), idesc, (i | k) != 0);
            umma_commit(smem_u32(&empty_bar[s]));
        }
        umma_commit(smem_u32(&acc_bar));
        if (!ok) {   // let the products already issued end before tensor memory is given back
            const uint64_t t0 = global_ns();
            while (global_ns() - t0 < 2000000ull) {}
        }
    } else if (warp >= 2) {
        for (int m = threadIdx.x - 64; m < TN; m += 64) scale[m] = m0 + m < M ? a_scales[m0 + m] : 0.0f;
    }
    __syncthreads();

    ok &= mbar_wait(smem_u32(&acc_bar), 0, &gave_up);   // on give-up the drain still runs (warp-uniformly) on whatever TMEM holds
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int n = n0 + threadIdx.x, tokens = min(TN, M - m0), each = TN >> shift;
    const uint32_t src = tmem_acc + ((uint32_t)(warp * 32) << 16);
    __syncwarp();
    cluster_wait();   // every CTA of the cluster runs, so its shared memory is there
    if (splits > 1 && sums_at<TN>() == 0) cluster_sync_all();   // and is through with its ring
    const uint32_t mine = tiles + sums_at<TN>() + (split * each * BN + threadIdx.x) * 4;   // in the CTA that adds up column c: [CTA][c >> shift][row of B]
#pragma unroll 1
    for (int c = 0; c < TN; c += 16) {
        if (c >= tokens) break;
        uint32_t r[16];
        __syncwarp();   // the load is the whole warp's
        tmem_load_16(src + (uint32_t)c, r);
        if (splits > 1) {   // stores that nobody waits for, and not loads: the way between two SMs' memories is paid once, at the barrier
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (c + j < tokens) store_cluster_f32(map_to_cta(mine + ((c + j) >> shift) * BN * 4, (c + j) & (splits - 1)), __uint_as_float(r[j]));
        } else if (n < N) {
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (c + j < tokens) store_sum(C + (m0 + c + j) * ldc + n, __uint_as_float(r[j]) * scale[c + j] * b_scale, add);
        }
    }
    if (splits > 1) {
        __syncwarp();
        cluster_sync_all();
        const float* sums = reinterpret_cast<const float*>(smem_raw + (tiles - smem_u32(smem_raw)) + sums_at<TN>());
        if (n < N) {
            for (int c = split; c < tokens; c += splits) {
                float total = 0.0f;
                for (int q = 0; q < splits; q++) total += sums[(q * each + (c >> shift)) * BN + threadIdx.x];
                store_sum(C + (m0 + c) * ldc + n, total * scale[c] * b_scale, add);
            }
        }
    }
    if (!ok && status) atomicExch(status, 1);

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_acc), "r"(TMEM_COLS) : "memory");
}

// ---- many tokens: a pair of CTAs per 256 x 256 tile, tcgen05.mma.cta_group::2 ----
//
// Rows of A (tokens) along the accumulator's lanes. CTA r of the pair loads rows 128 r .. of the tile's A and columns 128 r .. of its
// B, 32 KB a slab of 128 bytes of K, and holds its 128 rows of the accumulator; the even CTA issues every
// MMA, two slabs for each wait (one: 443 us where two take 413, 8192^3 under the power cap; the tensor cores run dry over a wait). Persistent: one warp feeds the ring, one issues, four drain the accumulator of the tile before (two of them
// in tensor memory), so the stores of a tile hide behind the next one's products.
namespace pair {
constexpr int TM = 256, TN = 256, HALF = 128, SLABS = 2, STAGES = 3, SLAB_BYTES = 2 * HALF * BK, STAGE_BYTES = SLABS * SLAB_BYTES, PIECE_BYTES = 32 * 128, PAIR_THREADS = 192, GROUP_M = 8;
constexpr int SMEM = STAGES * STAGE_BYTES + 4 * (PIECE_BYTES + TN * 4) + 1024;
constexpr uint32_t TMEM_COLS = 512;

// Tiles in bands of GROUP_M tile rows, so that the tiles in flight share panels of A and B in L2.
__device__ __forceinline__ void tile_at(int t, int tiles_m, int tiles_n, int* m, int* n) {
    const int per_band = GROUP_M * tiles_n, band = t / per_band, first = band * GROUP_M, rows = min(GROUP_M, tiles_m - first), r = t - band * per_band;
    *m = first + r % rows;
    *n = r / rows;
}

// VECTORS: C's rows are whole 16-byte pieces from an aligned start.
template <class T, bool VECTORS>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
    matmul_e4m3_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const float* a_scales,
                     const float* b_scales, T* __restrict__ C, int64_t ldc, int M, int N, int K, int add, int32_t* status) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], tfull_bar[2], tempty_bar[2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t gave_up;
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles_m = (M - 1) / TM + 1, tiles_n = (N - 1) / TN + 1, num_tiles = tiles_m * tiles_n, steps = (K - 1) / (BK * SLABS) + 1;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(smem_u32(&full_bar[s]), 1);    // the leader's producer; bytes arrive from both CTAs
            mbar_init(smem_u32(&empty_bar[s]), 1);   // one commit of the leader's MMA warp
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(smem_u32(&tfull_bar[b]), 1);
            mbar_init(smem_u32(&tempty_bar[b]), 8);   // four epilogue warps in each CTA (used in the leader only)
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    cluster_sync_all();   // the peer runs and its barriers are initialised: only from here on may anything reach into it, and allocating for the pair does
    if (warp == 1) {      // the same warp of both CTAs
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();   // the peer's tensor memory is allocated
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_slot;
    wait_for_predecessor();
    if (threadIdx.x == 0 && status && *reinterpret_cast<volatile int32_t*>(status) != 0) gave_up = 1;   // an earlier CTA gave up: do not pile on
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (int t = pair; t < num_tiles && ok; t += pairs) {
                int mi, ni;
                tile_at(t, tiles_m, tiles_n, &mi, &ni);
                const int m0 = mi * TM + (int)rank * HALF, n0 = ni * TN + (int)rank * HALF;
                for (int kb = 0; kb < steps; kb++) {
                    ok &= mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, &gave_up);
                    if (!ok) break;
                    const uint32_t fb_local = smem_u32(&full_bar[s]), fb = map_to_cta(fb_local, 0), a_dst = tiles + s * STAGE_BYTES;
                    if (leader) mbar_expect_tx(fb_local, 2 * STAGE_BYTES);
#pragma unroll
                    for (int h = 0; h < SLABS; h++) {   // a slab behind the end of K arrives as zeros
                        tma_load_2d_pair(a_dst + h * SLAB_BYTES, &map_a, fb, (kb * SLABS + h) * BK, m0);
                        tma_load_2d_pair(a_dst + h * SLAB_BYTES + HALF * BK, &map_b, fb, (kb * SLABS + h) * BK, n0);
                    }
                    if (++s == STAGES) s = 0, ph ^= 1;
                }
            }
            if (!ok) {   // let the copies already issued land before the CTA can exit
                const uint64_t t0 = global_ns();
                while (global_ns() - t0 < 2000000ull) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            const uint32_t idesc = (1u << 4) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
            uint32_t s = 0, ph = 0, local = 0;
            for (int t = pair; t < num_tiles && ok; t += pairs, local++) {
                const uint32_t buf = local & 1, use = local >> 1;
                ok &= mbar_wait(smem_u32(&tempty_bar[buf]), (use & 1) ^ 1, &gave_up);   // both epilogues have drained this accumulator
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; kb < steps; kb++) {
                    ok &= mbar_wait(smem_u32(&full_bar[s]), ph, &gave_up);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t a_src = tiles + s * STAGE_BYTES;
                    const uint64_t da = smem_desc(a_src, 16, 1024), db = smem_desc(a_src + HALF * BK, 16, 1024);
#pragma unroll
                    for (int h = 0; h < SLABS; h++)
#pragma unroll
                        for (int k = 0; k < BK / MMA_K; k++)
                            umma_f8_pair(tmem_base + buf * TN, da + (uint64_t)(h * (SLAB_BYTES >> 4) + 2 * k), db + (uint64_t)(h * (SLAB_BYTES >> 4) + 2 * k), idesc, (kb | h | k) != 0);
                    umma_commit_pair(smem_u32(&empty_bar[s]));
                    if (++s == STAGES) s = 0, ph ^= 1;
                }
                umma_commit_pair(smem_u32(&tfull_bar[buf]));
            }
            if (!ok) {   // let the products already issued end before tensor memory is given back
                const uint64_t t0 = global_ns();
                while (global_ns() - t0 < 2000000ull) {}
            }
        }
    } else {
        // Each 32-row piece of 128 bytes a row is transposed through shared memory and stored as whole lines.
        constexpr int COLS = 128 / sizeof(T), W = 16 / sizeof(T);
        const int ew = warp & 3;   // this warp may touch lanes 32 ew .. 32 ew + 31
        uint8_t* stage = smem_raw + (tiles - smem_u32(smem_raw)) + STAGES * STAGE_BYTES + ew * PIECE_BYTES;
        float* scale = reinterpret_cast<float*>(smem_raw + (tiles - smem_u32(smem_raw)) + STAGES * STAGE_BYTES + 4 * PIECE_BYTES) + ew * TN;
        uint32_t local = 0;
        for (int t = pair; t < num_tiles && ok; t += pairs, local++) {
            int mi, ni;
            tile_at(t, tiles_m, tiles_n, &mi, &ni);
            const uint32_t buf = local & 1, use = local >> 1;
            const int m0 = mi * TM + (int)rank * HALF + ew * 32, n0 = ni * TN;
            const float a_scale = m0 + lane < M ? a_scales[m0 + lane] : 0.0f;
            __syncwarp();   // the tile before has been read out of `scale`
#pragma unroll
            for (int i = 0; i < TN / 32; i++) scale[lane + 32 * i] = n0 + lane + 32 * i < N ? b_scales[n0 + lane + 32 * i] : 0.0f;
            ok &= mbar_wait(smem_u32(&tfull_bar[buf]), use & 1, &gave_up);
            ok = __all_sync(0xffffffffu, ok);   // the warp stays together: the loads of tensor memory are warp-collective
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = tmem_base + buf * TN + ((uint32_t)(ew * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < TN; c += COLS) {
#pragma unroll
                for (int part = 0; part < COLS / 32; part++) {
                    uint32_t r[32];
                    tmem_load_32(src + (uint32_t)(c + 32 * part), r);
#pragma unroll
                    for (int q = 0; q < 32 / W; q++) {   // 16-byte piece q of this lane's row, at a place rotated by the row: no bank conflicts
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < W; i += 4) {
                            const float4 b = *reinterpret_cast<const float4*>(scale + c + 32 * part + W * q + i);
                            const float v0 = __uint_as_float(r[W * q + i]) * a_scale * b.x, v1 = __uint_as_float(r[W * q + i + 1]) * a_scale * b.y;
                            const float v2 = __uint_as_float(r[W * q + i + 2]) * a_scale * b.z, v3 = __uint_as_float(r[W * q + i + 3]) * a_scale * b.w;
                            if constexpr (sizeof(T) == 4) w[0] = __float_as_uint(v0), w[1] = __float_as_uint(v1), w[2] = __float_as_uint(v2), w[3] = __float_as_uint(v3);
                            else w[i / 2] = two_as<T>(v0, v1), w[i / 2 + 1] = two_as<T>(v2, v3);
                        }
                        *reinterpret_cast<uint4*>(stage + lane * 128 + (((32 / W * part + q) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                __syncwarp();
                if (c + COLS == TN) {   // the accumulator is drained: the MMA warp may overwrite it while the stores go out
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tempty_bar[buf]), 0));
                }
                const int row = lane >> 3, piece = lane & 7, n = n0 + c + W * piece;   // eight lanes to a row
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int m = m0 + 4 * i + row;
                    uint4 v = *reinterpret_cast<const uint4*>(stage + (4 * i + row) * 128 + ((piece ^ ((4 * i + row) & 7)) << 4));
                    T* to = C + m * ldc + n;
                    if constexpr (sizeof(T) == 4) {
                        if (add && m < M) {
                            float* e = reinterpret_cast<float*>(&v);
#pragma unroll
                            for (int j = 0; j < W; j++)
                                if (n + j < N) e[j] += to[j];
                        }
                    }
                    if (VECTORS && m < M && n + W <= N) *reinterpret_cast<uint4*>(to) = v;
                    else if (m < M) {
                        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
                        for (int j = 0; j < W; j++)
                            if (n + j < N) to[j] = e[j];
                    }
                }
                __syncwarp();   // the next piece may overwrite the staging rows
            }
        }
    }
    if (!ok && status) atomicExch(status, 1);
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();   // the peer has stopped naming this CTA's barriers, shared and tensor memory
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    __syncwarp();
    cluster_sync_all();   // neither leaves while the other still frees the pair's
}
}  // namespace pair

struct Args {
    const void *a, *b;
    const float *a_scales, *b_scales;
    void* c;
    int64_t lda, ldb, ldc;
    int M, N, K, add;
    int32_t* status;
    cudaStream_t stream;
};

const char* const WHO = "matmul_e4m3";
constexpr int PART_K = 8192;   // of one launch into an f32 C

// How many CTAs share a tile's K, as a power of two: two CTAs fit an SM; split while the tiles leave room and every share keeps four slabs.
int split_shift(int64_t tiles, int slabs) {
    int shift = 0;
    while (shift < 3 && tiles << (shift + 1) <= 2 * basalt_k::sm_count() && slabs >= 8 << shift) shift++;
    return shift;
}

template <class T, int TN>
int launch(const Args& p) {
    CUtensorMap ma, mb;
    if (const int rc = make_tensor_map(&mb, WHO, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.b, p.N, p.K, p.ldb, BK, BN)) return rc;
    if (const int rc = make_tensor_map(&ma, WHO, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.a, p.M, p.K, p.lda, BK, TN)) return rc;
    constexpr auto kern = matmul_e4m3_kernel<T, TN>;
    constexpr int smem = smem_of<TN>();
    if (const int rc = basalt_k::allow_smem<kern>(WHO, smem)) return rc;
    const int tiles_n = (p.N - 1) / BN + 1, slabs = (p.K - 1) / BK + 1;
    const int64_t tiles = (int64_t)tiles_n * ((p.M - 1) / TN + 1);
    const int shift = split_shift(tiles, slabs);
    const dim3 grid(tiles_n << shift, (p.M - 1) / TN + 1);
    return basalt_k::launch_clusters(WHO, kern, grid, THREADS, smem, 1 << shift, p.stream, mb, ma, p.a_scales, p.b_scales, (T*)p.c, p.ldc, p.M, p.N, p.K, shift, p.add, p.status);
}

template <class T, bool VECTORS>
int launch_pair(const Args& p) {
    CUtensorMap ma, mb;
    if (const int rc = make_tensor_map(&ma, WHO, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.a, p.M, p.K, p.lda, BK, pair::HALF)) return rc;
    if (const int rc = make_tensor_map(&mb, WHO, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.b, p.N, p.K, p.ldb, BK, pair::HALF)) return rc;
    constexpr auto kern = pair::matmul_e4m3_pair<T, VECTORS>;
    if (const int rc = basalt_k::allow_smem<kern>(WHO, pair::SMEM)) return rc;
    const int64_t tiles = (int64_t)((p.M - 1) / pair::TM + 1) * ((p.N - 1) / pair::TN + 1);
    if (tiles > INT32_MAX / 2) return basalt_k::record_msg(1, WHO, "M * N is too large");
    const int pairs = (int)(tiles < basalt_k::sm_count() / 2 ? tiles : basalt_k::sm_count() / 2);
    return basalt_k::launch_clusters(WHO, kern, 2 * pairs, pair::PAIR_THREADS, pair::SMEM, 2, p.stream, ma, mb, p.a_scales, p.b_scales, (T*)p.c, p.ldc, p.M, p.N, p.K, p.add, p.status);
}

// What a call takes, in microseconds, by the kernel above with tiles of TN rows of A: a slab takes a round of CTAs 0.31 to 0.51; the weights
// come from memory at 6.3 TB/s, and a third of them again for each further tile over M; the join of a split tile takes 0.055 a column.
// (Measured / estimated: 8192 x 8192 for 1 row 15.0 / 13.9, 64 rows 19.5 / 18.2; 4096 x 4096 for 64 rows in tiles of 16, 32
// and 64: 10.5 / 10.3, 8.8 / 9.4, 9.3 / 10.2; for 128 rows 13.5 / 13.1, 12.6 / 11.2, 11.4 / 11.1 and in tiles of 128 12.9 / 13.7.)
double time_of_tiles(int M, int N, int K, int TN) {
    const int64_t tiles_m = (M - 1) / TN + 1, tiles = tiles_m * ((N - 1) / BN + 1), slabs = (K - 1) / BK + 1;
    const int shift = split_shift(tiles, (int)slabs);
    const double slab = TN == 16 ? 0.31 : TN == 32 ? 0.32 : TN == 64 ? 0.37 : 0.51;
    const double rounds = (double)(((tiles << shift) - 1) / (2 * basalt_k::sm_count()) + 1), compute = rounds * slab * (double)((slabs - 1 >> shift) + 1);
    const double memory = (double)N * K * (1.0 + 0.35 * (double)(tiles_m - 1)) / 6.3e6;
    return 3.2 + (compute > memory ? compute : memory) + (shift ? 1.5 + 0.055 * (M < TN ? M : TN) : 0.0);
}
// By the pairs of CTAs: 0.305 a slab and round of 74 tiles, and the weights at 5.4 TB/s. (16384 x 16384 for 64 rows 52.7 / 55.2; 4096 x 4096 for 256 rows 15.0 / 15.3, where tiles of 32 rows take 14.0; 8192 x 8192
// for 256 rows 25.5 / 25.0, where tiles of 64 take 27.3; for 2048 rows 84 / 83.6, where tiles of 128 take 142.)
double time_of_pairs(int M, int N, int K) {
    const int64_t tiles = (int64_t)((M - 1) / pair::TM + 1) * ((N - 1) / pair::TN + 1);
    const double compute = 0.305 * (double)((tiles - 1) / (basalt_k::sm_count() / 2) + 1) * (double)((K - 1) / BK + 1), memory = (double)N * K / 5.4e6;
    return 5.5 + (compute > memory ? compute : memory);
}

template <class T>
int launch_type(const Args& p) {
    int best = 0;
    double least = time_of_pairs(p.M, p.N, p.K);
    for (int TN = 16; TN <= 128; TN *= 2) {
        if (TN > 16 && TN >= 2 * p.M) break;
        if ((p.M - 1) / TN >= 65535) continue;   // a grid's second dimension
        const double t = time_of_tiles(p.M, p.N, p.K, TN);
        if (t < least) least = t, best = TN;
    }
    if (best == 16) return launch<T, 16>(p);
    if (best == 32) return launch<T, 32>(p);
    if (best == 64) return launch<T, 64>(p);
    if (best == 128) return launch<T, 128>(p);
    const bool vectors = (uintptr_t)p.c % 16 == 0 && p.ldc * sizeof(T) % 16 == 0;
    return vectors ? launch_pair<T, true>(p) : launch_pair<T, false>(p);
}

}  // namespace

extern "C" int basalt_k_matmul_e4m3(const void* A, int64_t lda, const float* a_scales, const void* B, int64_t ldb, const float* b_scales, int c_type, void* C,
                                    int64_t ldc, int M, int N, int K, int32_t* status, void* stream) {
    if (c_type != BASALT_K_TYPE_F16 && c_type != BASALT_K_TYPE_BF16 && c_type != BASALT_K_TYPE_F32) return basalt_k::record_msg(1, WHO, "unknown type of C");
    if (M < 0 || N < 0) return basalt_k::record_msg(1, WHO, "M and N must not be negative");
    if (K < 1) return basalt_k::record_msg(1, WHO, "K must be at least 1");
    if (M > 1 << 30 || N > 1 << 30 || K > 1 << 30) return basalt_k::record_msg(1, WHO, "M, N and K must not exceed 2^30");
    if (!M || !N) return 0;
    if (!A || !B || !C || !a_scales || !b_scales) return basalt_k::record_msg(1, WHO, "A, B, C and both scales are needed");
    const int size = c_type == BASALT_K_TYPE_F32 ? 4 : 2;
    if (((uintptr_t)A | (uintptr_t)B) & 15 || (lda | ldb) & 15) return basalt_k::record_msg(1, WHO, "A and B and their row strides must be multiples of 16 bytes");
    if (lda < K || ldb < K || ldc < N) return basalt_k::record_msg(1, WHO, "a row stride lies below the row");
    if (lda >= (int64_t)1 << 31 || ldb >= (int64_t)1 << 31 || ldc >= (int64_t)1 << 31) return basalt_k::record_msg(1, WHO, "a row stride lies above 2^31 - 1");
    if ((uintptr_t)C % size || ((uintptr_t)a_scales | (uintptr_t)b_scales | (uintptr_t)status) % 4) return basalt_k::record_msg(1, WHO, "C, the scales or the status are not aligned to their elements");
    const basalt_k::Span c = {C, M, N, ldc, size};
    if (overlap(c, {A, M, K, lda, 1}) || overlap(c, {B, N, K, ldb, 1}) || overlap(c, {a_scales, 1, M, M, 4}) || overlap(c, {b_scales, 1, N, N, 4}))
        return basalt_k::record_msg(1, WHO, "C overlaps an input");
    if (const int rc = basalt_k::check_device_pointers(WHO, {A, a_scales, B, b_scales, C, status})) return rc;
    const Args p = {A, B, a_scales, b_scales, C, lda, ldb, ldc, M, N, K, 0, status, (cudaStream_t)stream};
    if (c_type == BASALT_K_TYPE_F16) return launch_type<__half>(p);
    if (c_type == BASALT_K_TYPE_BF16) return launch_type<__nv_bfloat16>(p);
    // The tensor cores' f32 sums are truncated, term by term, which costs some 9e-11 of the result for each k: 1.4e-6 at 16,384. An f32 result
    // shows it, so K goes in equal parts of at most 8192, each rounded and added to C in turn. (What that and the wider C cost, f32 / f16: 2048 rows,
    // 16384 -> 4096, 172 / 92 us; one row 19.4 / 14.8.)
    const int parts = (K - 1) / PART_K + 1, part = ((K - 1) / parts / BK + 1) * BK;
    for (int k = 0; k < K; k += part) {
        Args q = p;
        q.a = (const uint8_t*)A + k, q.b = (const uint8_t*)B + k, q.K = K - k < part ? K - k : part, q.add = k > 0;
        if (const int rc = launch_type<float>(q)) return rc;
    }
    return 0;
}

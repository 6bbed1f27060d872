// Product with 4-bit weights for sm_100a:
//
//   C[m, n] = sum_k X[m, k] * (q[n, k] - z[n, k / group]) * s[n, k / group]
//
// X [M x K] and C [M x N] are f16 or bf16; q is four bits, two to a byte along k (even k in the low half); s has X's type,
// z is an integer (8 where none are given). Two kernels: few rows of X are bound by reading (and unpacking) N K / 2 bytes of weights, many rows by
// the products. Both read the weights once for a tile of rows, unpack them by putting four bits into the mantissa
// of a power of two and subtracting, exactly, and add in f32. A cluster of up to eight CTAs shares a tile's K where tiles are few; the
// partial sums meet in distributed shared memory and are added in a fixed order: no workspace, no atomics, the same bits every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "../../../include/basalt_b200_kernels.h"
#include "common.cuh"
#include "tensor_core.cuh"

namespace {

using namespace basalt_k::tc;

constexpr int ROWS = 128, UNIT_K = 32;

template <class T>
__device__ __forceinline__ T as_type(uint32_t bits) {
    if constexpr (std::is_same_v<T, __half>) return __ushort_as_half((unsigned short)bits);
    else return __ushort_as_bfloat16((unsigned short)bits);
}
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// BYTES (4, 8 or 16, and so aligned) from global to shared memory, asynchronously. The first `valid` of them are read (none, if it is
// negative; the address has to be aligned all the same); the others arrive as zeros.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const uint8_t* from, int valid = BYTES) {
    const int n = max(0, min(BYTES, valid));
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
// Arrives on the barrier when every copy that this thread has begun is done.
__device__ __forceinline__ void copies_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory"); }

// For every reader of a ring's place, before the warp hands it back: orders what the thread has read there before the bulk loads that fill it again. They write
// through the async proxy, which an arrival on a barrier alone does not order against plain reads: without this, reads that queued behind the copies' cache
// misses saw the next slab (14720 -> 14931 in groups of 32, bf16, from cold memory, with a warp that only carries scales: one launch in four missed 32 k of X
// in the rows of a warp on that warp's scheduler).
// It costs 0.6 us of 20.5 for 17 rows through 8192 x 8192, nothing that shows for one row.
__device__ __forceinline__ void reads_done() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A slab's scales and zero points in shared memory: of each of the tile's 128 rows the groups that 256 k touch, at most 8 / FLUSH where
// FLUSH * 32 k certainly share a group. They travel with the slab's weights. (A load by each thread that wants a scale touches 32
// rows, so 32 lines of the cache, in an instruction: with those, one row through 8192 x 8192 in groups of 32 took 34 us.)
// ALIGNED: every slab begins with a group and its groups are whole pieces of 4, 8 or 16 bytes; else as many 4-byte words as hold
// them from any start.
template <class T, int FLUSH, bool ZEROS>
struct SlabScales {
    static constexpr int GROUPS = 8 / FLUSH, SCALE_WORDS = GROUPS / 2 + 1, ZERO_WORDS = ZEROS ? (GROUPS + 6) / 4 : 0, ZERO_PIECE = GROUPS < 4 ? 4 : GROUPS;
    static constexpr int ZERO_AT = ROWS * SCALE_WORDS * 4, BYTES = (ZERO_AT + ROWS * ZERO_WORDS * 4 + 1023) / 1024 * 1024;

    static bool aligned(const void* scales, const void* zeros, int group, int groups) {
        return group * GROUPS == 256 && groups % GROUPS == 0 && (uintptr_t)scales % (2 * GROUPS) == 0 && (uintptr_t)zeros % ZERO_PIECE == 0;
    }

    // One warp's copies of the rows from n0; lane l has rows l, l + 32, l + 64 and l + 96.
    struct Copies {
        const uint8_t *scale_row[4], *zero_row[4], *scale_base, *zero_base, *scale_end, *zero_end;
        __device__ __forceinline__ Copies(const void* scales, const uint8_t* zeros, int n0, int N, int groups, int lane) {
            scale_base = (const uint8_t*)scales, zero_base = zeros;
            scale_end = scale_base + (int64_t)N * groups * 2, zero_end = zeros + (ZEROS ? (int64_t)N * groups : 0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int64_t first = (int64_t)min(n0 + lane + 32 * r, N - 1) * groups;   // rows past the last get its scales
                scale_row[r] = (const uint8_t*)scales + first * 2, zero_row[r] = zeros + (ZEROS ? first : 0);
            }
        }
        // those of the groups from `start`, to `at` in shared memory
        __device__ __forceinline__ void operator()(uint32_t at, int start, int lane, bool aligned) const {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = lane + 32 * r;
                const uint8_t *s = scale_row[r] + 2 * start, *z = zero_row[r] + start;
                if (aligned) {
                    copy_async<2 * GROUPS>(at + row * 2 * GROUPS, s);
                    if (ZEROS) {
                        const uint8_t* piece = (const uint8_t*)((uintptr_t)z & ~(uintptr_t)(ZERO_PIECE - 1));
                        copy_async<ZERO_PIECE>(at + ZERO_AT + row * ZERO_PIECE, piece, (int)min((int64_t)ZERO_PIECE, zero_end - piece));
                    }
                } else {
                    const uint8_t *sw = (const uint8_t*)((uintptr_t)s & ~(uintptr_t)3), *zw = (const uint8_t*)((uintptr_t)z & ~(uintptr_t)3);
#pragma unroll
                    for (int w = 0; w < SCALE_WORDS; w++) {
                        const bool in = sw + 4 * w < scale_end;
                        copy_async<4>(at + (row * SCALE_WORDS + w) * 4, in ? sw + 4 * w : scale_base, in ? (int)min((int64_t)4, scale_end - sw - 4 * w) : 0);
                    }
#pragma unroll
                    for (int w = 0; w < ZERO_WORDS; w++) {
                        const bool in = zw + 4 * w < zero_end;
                        copy_async<4>(at + ZERO_AT + (row * ZERO_WORDS + w) * 4, in ? zw + 4 * w : zero_base, in ? (int)min((int64_t)4, zero_end - zw - 4 * w) : 0);
                    }
                }
            }
        }
    };
    // The scale (its bits) and the zero point of row `row` in group start + ahead; row_group: the row's first group, modulo 4 at least.
    static __device__ __forceinline__ uint32_t scale_bits(const uint8_t* at, int row, uint32_t row_group, int start, int ahead, bool aligned) {
        return *reinterpret_cast<const uint16_t*>(at + (aligned ? row * 2 * GROUPS : row * SCALE_WORDS * 4 + ((row_group + start) & 1) * 2) + ahead * 2);
    }
    static __device__ __forceinline__ int zero(const uint8_t* at, int row, uint32_t row_group, int start, int ahead, bool aligned) {
        return at[ZERO_AT + (aligned ? row * ZERO_PIECE + ((row_group + start) & (ZERO_PIECE - 1)) : row * ZERO_WORDS * 4 + ((row_group + start) & 3)) + ahead];
    }
};

// (a & mask) | magic in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t magic) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(magic));
    return d;
}

// The zero point of a weight row as the two constants that unpacking subtracts, in both halves of a register.
template <class T>
struct Zero;
template <>
struct Zero<__half> {
    __half2 low, high;
    __device__ __forceinline__ void set(int z) {
        low = __half2half2(__ushort_as_half((unsigned short)(0x6400 + z)));   // 1024 + z: z counts the last bits of the mantissa
        high = __hsub2(__half2half2(__int2half_rn(960)), low);   // -64 - z
    }
    __device__ __forceinline__ Zero of_lane(int lane) const {
        Zero v;
        v.low = __shfl_sync(0xffffffffu, low, lane);
        v.high = __hsub2(__half2half2(__int2half_rn(960)), v.low);
        return v;
    }
};
template <>
struct Zero<__nv_bfloat16> {
    __nv_bfloat162 low;
    __device__ __forceinline__ void set(int z) { low = __bfloat162bfloat162(__ushort_as_bfloat16((unsigned short)(0x4300 + z))); }   // 128 + z, likewise
    __device__ __forceinline__ Zero of_lane(int lane) const {
        Zero v;
        v.low = __shfl_sync(0xffffffffu, low, lane);
        return v;
    }
};

// Eight packed weights -> q - z as pairs of k: (0, 4), (1, 5), (2, 6), (3, 7). The four bits are put into the mantissa of a
// power of two (1024 + q in f16, 128 + q in bf16; 1024 + 16 q for the upper half of a byte), and the subtraction is exact.
__device__ __forceinline__ void unpack(uint32_t w, const Zero<__half>& z, uint32_t (&p)[4]) {
    const __half2 sixteenth = __half2half2(__ushort_as_half((unsigned short)0x2C00));   // 2^-4
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t lo = and_or(w >> (8 * i), 0x000F000Fu, 0x64006400u), hi = and_or(w >> (8 * i), 0x00F000F0u, 0x64006400u);
        const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), z.low);
        const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, z.high);
        p[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
        p[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
}
__device__ __forceinline__ void unpack(uint32_t w, const Zero<__nv_bfloat16>& z, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t v = and_or(w >> (4 * i), 0x000F000Fu, 0x43004300u);
        const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), z.low);
        p[i] = *reinterpret_cast<const uint32_t*>(&a);
    }
}

// The power of two whose last bits of mantissa four bits become: 1024 in f16, 128 in bf16.
template <class T>
constexpr uint32_t MAGIC = std::is_same_v<T, __half> ? 0x64006400u : 0x43004300u;

template <class T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- few rows of X ----
//
// A CTA takes 128 rows of the weights over its share of K: one warp feeds a ring of stages (256 k) by bulk-tensor loads, eight
// warps compute, 32 rows x half a stage each. Operands are exact: q - z is a small integer, exact in f16 and in bf16, so
// mma.sync m16n8k16 adds (q - z) * x over a group in f32 and the group's scale multiplies that sum in f32. Nothing but C is
// rounded to 16 bits. The instruction's order of k is free as long as both operands share it; it is chosen so that one
// 32-bit word of packed weights (eight k) and one 16-byte load of X (eight k) feed two instructions without a shuffle
// between threads. (tcgen05.mma would save the products, which are not what bounds this: its instructions are 128 rows high, and
// a group's sum would have to leave tensor memory before its scale.)
// What bounds it: no unit by itself. One row through 8192 x 8192 takes 11.8 to 12.2 us (2.9 TB/s of packed weights; a plain stream of as many bytes takes
// 6.5) with the memory 28 % busy, the issue slots 44 % and the logic unit, which unpacks, 36 %: a warp has one slab's chain of barrier, scales, unpacking,
// product and scaled sum in flight, and shares of K in powers of two leave places empty (256 CTAs on 148 SMs that hold two each).
// 16 rows, 4096 -> 14336 in groups of 64 with zero points, bf16: 18.9 us; one row in groups of 32: 14.3, bf16 with zero points 17.6.
namespace few {
constexpr int SLAB_K = 256, W_BYTES = ROWS * SLAB_K / 2, CONSUMERS = 8, THREADS = 32 * (CONSUMERS + 1), X_BOX_K = 32;

// A stage: 128 rows of weights, 8 NT rows of X, the scales. JOIN: the sums of both halves of the warps, for every row of X.
template <class T, int NT, int FLUSH, bool ZEROS>
struct Stage {
    using Scales = SlabScales<T, FLUSH, ZEROS>;
    static constexpr int X = W_BYTES, SCALES = X + 8 * NT * SLAB_K * 2, BYTES = SCALES + Scales::BYTES, COUNT = NT == 1 ? 4 : 3, JOIN = 2 * 8 * NT * ROWS * 4;
    static constexpr int SMEM = COUNT * BYTES + JOIN + 1024;   // at most 109 KB: two CTAs fit an SM
};

// NT: tiles of eight rows of X. FLUSH: units (32 k) that certainly share a group, 1, 2 or 4.
template <class T, int NT, int FLUSH, bool ZEROS>
__global__ void __launch_bounds__(THREADS, 2) matmul_w4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                               const T* __restrict__ scales, const uint8_t* __restrict__ zeros, T* __restrict__ C, int64_t ldc,
                                                               int M, int N, int K, int group, int groups, int aligned, int shift, int32_t* status) {
    using S = Stage<T, NT, FLUSH, ZEROS>;
    using Scales = typename S::Scales;
    constexpr int STAGES = S::COUNT, TOKENS = 8 * NT, STAGE_BYTES = S::BYTES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES];
    __shared__ volatile uint32_t gave_up;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (ring - smem_u32(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // 1 << shift CTAs share a tile's K. (No division is done here that the host can do: on the way to the first load their latencies add up.)
    const int splits = 1 << shift, split = blockIdx.x & (splits - 1), n0 = (blockIdx.x >> shift) * ROWS, m0 = blockIdx.y * TOKENS;
    const int slabs = (K - 1) / SLAB_K + 1, first = slabs * split >> shift, count = (slabs * (split + 1) >> shift) - first;

    if (threadIdx.x == 0) {
        prefetch_map(&map_w);
        prefetch_map(&map_x);
        gave_up = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(smem_u32(&full_bar[s]), 1 + 32);   // the bulk loads, and each lane's copies of scales
            mbar_init(smem_u32(&empty_bar[s]), CONSUMERS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    cluster_arrive();
    wait_for_predecessor();
    if (threadIdx.x == 0 && status && *reinterpret_cast<volatile int32_t*>(status) != 0) gave_up = 1;   // an earlier CTA gave up: do not pile on
    bool ok = true;
    float total[2][NT][4] = {};

    const int first_group = (unsigned)(first * SLAB_K) / (unsigned)group;
    if (warp == CONSUMERS) {
        const typename Scales::Copies copies(scales, zeros, n0, N, groups, lane);
        int start = first_group, in_group = first * SLAB_K - start * group;
        for (int i = 0; i < count; i++) {
            const int s = i % STAGES;
            ok &= mbar_wait<LONG_WAIT>(smem_u32(&empty_bar[s]), ((i / STAGES) & 1) ^ 1, &gave_up);
            if (!ok) break;
            const uint32_t fb = smem_u32(&full_bar[s]), at = ring + s * STAGE_BYTES;
            const int k = (first + i) * SLAB_K;
            if (lane == 0) {
                mbar_expect_tx(fb, W_BYTES + min(M, TOKENS) * SLAB_K * 2);
                tma_load_2d(at, &map_w, fb, k / 2, n0);
#pragma unroll
                for (int b = 0; b < SLAB_K / X_BOX_K; b++) tma_load_2d(at + S::X + b * TOKENS * X_BOX_K * 2, &map_x, fb, k + b * X_BOX_K, m0);
            }
            copies(at + S::SCALES, start, lane, aligned);
            copies_arrive(fb);
            for (in_group += SLAB_K; in_group >= group; in_group -= group) start++;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (!ok) {   // let the copies already issued land before the CTA can exit
            const uint64_t t0 = global_ns();
            while (global_ns() - t0 < 2000000ull) {}
        }
        __syncwarp();
    } else {
        const int half = warp >> 2, row0 = (warp & 3) * 32, g = lane >> 2, t = lane & 3;
        // Of the four weight rows g, g + 8, g + 16 and g + 24 that four lanes share, lane t reads the scales of row g + 8 t and the
        // lanes exchange them.
        const int my_row = row0 + g + 8 * t;
        const uint32_t row_group = (uint32_t)min(n0 + my_row, N - 1) * (uint32_t)groups;
        int start = first_group, in_start = first * SLAB_K - start * group, s = 0;
        uint32_t ph = 0;
        for (int i = 0; i < count; i++) {
            ok &= mbar_wait(smem_u32(&full_bar[s]), ph, &gave_up);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint8_t* my_scales = smem + s * STAGE_BYTES + S::SCALES;
            float by[4 / FLUSH];
            Zero<T> z[ZEROS ? 4 / FLUSH : 1];
            if (!ZEROS) z[0].set(8);
            if (aligned) {   // this half's groups follow one another, and all of them exist
                const uint8_t* from = my_scales + my_row * 2 * Scales::GROUPS + half * Scales::GROUPS;
                T scale[4 / FLUSH];
                memcpy(scale, __builtin_assume_aligned(from, sizeof scale), sizeof scale);
#pragma unroll
                for (int f = 0; f < 4 / FLUSH; f++) by[f] = to_float(scale[f]);
                if constexpr (ZEROS) {
                    const uint8_t* zero = my_scales + Scales::ZERO_AT + my_row * Scales::ZERO_PIECE + ((row_group + start) & (Scales::ZERO_PIECE - 1)) + half * (Scales::GROUPS / 2);
#pragma unroll
                    for (int f = 0; f < 4 / FLUSH; f++) z[f].set(zero[f]);
                }
                start += Scales::GROUPS;
            } else {
                int ahead = 0, k = in_start + half * 128;   // the group of this half's next part, counted from the slab's first
#pragma unroll
                for (int f = 0; f < 4 / FLUSH; f++) {
                    for (; k >= group; k -= group) ahead++;
                    const bool in = start + ahead < groups;   // past the end of K: X is zero there, and so is the scale
                    by[f] = in ? to_float(as_type<T>(Scales::scale_bits(my_scales, my_row, row_group, start, ahead, false))) : 0.0f;
                    if (ZEROS) z[f].set(in ? Scales::zero(my_scales, my_row, row_group, start, ahead, false) : 0);
                    k += FLUSH * UNIT_K;
                }
                for (in_start += SLAB_K; in_start >= group; in_start -= group) start++;
            }
            const uint8_t* w_at = smem + s * STAGE_BYTES + (row0 + g) * 128 + t * 4;
            const uint8_t* x_at = smem + s * STAGE_BYTES + S::X + half * 4 * TOKENS * X_BOX_K * 2 + lane * 16;
#pragma unroll
            for (int f = 0; f < 4 / FLUSH; f++) {
                float acc[2][NT][4] = {};
                Zero<T> row_z[4];
#pragma unroll
                for (int r = 0; r < 4; r++) row_z[r] = ZEROS ? z[ZEROS ? f : 0].of_lane((lane & ~3) | r) : z[0];
#pragma unroll
                for (int v = 0; v < FLUSH; v++) {
                    const int u = f * FLUSH + v;
                    uint32_t a[4][4];
#pragma unroll
                    for (int r = 0; r < 4; r++) unpack(*reinterpret_cast<const uint32_t*>(w_at + r * 8 * 128 + (((half * 4 + u) ^ g) << 4)), row_z[r], a[r]);   // 128-byte swizzle: piece ^ (row & 7)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const uint4 x = *reinterpret_cast<const uint4*>(x_at + u * TOKENS * X_BOX_K * 2 + nt * 8 * X_BOX_K * 2);   // row 8 nt + g of X, its k 8 t .. 8 t + 7 of the unit
                        const uint32_t b0 = __byte_perm(x.x, x.z, 0x5410), b1 = __byte_perm(x.x, x.z, 0x7632);
                        const uint32_t b2 = __byte_perm(x.y, x.w, 0x5410), b3 = __byte_perm(x.y, x.w, 0x7632);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            mma_16816<T>(acc[h][nt], a[2 * h][0], a[2 * h + 1][0], a[2 * h][1], a[2 * h + 1][1], b0, b1);
                            mma_16816<T>(acc[h][nt], a[2 * h][2], a[2 * h + 1][2], a[2 * h][3], a[2 * h + 1][3], b2, b3);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float b = __shfl_sync(0xffffffffu, by[f], (lane & ~3) | r);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 2; j++) total[r >> 1][nt][2 * (r & 1) + j] += b * acc[r >> 1][nt][2 * (r & 1) + j];
                }
            }
            reads_done();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty_bar[s]));
            if (++s == STAGES) s = 0, ph ^= 1;
        }
    }

    // Every row of X has a CTA of the cluster that adds up its sums: both halves of the warps, CTA by CTA, in that order. Each
    // warp stores its sums where that CTA will read them.
    __syncwarp();
    cluster_wait();   // every CTA of the cluster runs, so its shared memory is there
    const int tokens = min(TOKENS, M - m0), each = TOKENS >> shift;
    float* join = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES);   // [CTA][half][row of X, of those this CTA adds up][row of the weights]
    if (warp < CONSUMERS) {
        const uint32_t mine = smem_u32(join + (split * 2 + (warp >> 2)) * each * ROWS + (warp & 3) * 32 + (lane >> 2));
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c = 8 * nt + 2 * (lane & 3) + e;
                if (c >= tokens) continue;
                const uint32_t to = map_to_cta(mine + (c >> shift) * ROWS * 4, c & (splits - 1));
#pragma unroll
                for (int r = 0; r < 4; r++) store_cluster_f32(to + 8 * r * 4, total[r >> 1][nt][2 * (r & 1) + e]);
            }
    }
    __syncwarp();
    cluster_sync_all();
    for (int i = threadIdx.x; i < ((tokens - split + splits - 1) >> shift) * ROWS; i += THREADS) {
        const int row = i % ROWS, c = (i / ROWS << shift) + split;
        if (n0 + row >= N) continue;
        float v = 0.0f;
        for (int q = 0; q < 2 * splits; q++) v += join[(q * each + i / ROWS) * ROWS + row];
        store_as(C + (m0 + c) * ldc + n0 + row, v);
    }
    if (!ok && status) atomicExch(status, 1);
}
}  // namespace few

// ---- many rows of X: the weights unpacked into tensor memory for tcgen05.mma ----
//
// The weights lie along the accumulator's 128 lanes and up to 256 rows of X along its columns (the width of a tile is the
// host's choice, a multiple of 16). Teams of four warps unpack 64 k each, a thread one row, straight into the tensor memory
// that the MMA takes its first operand from: (q - z) * s rounded to X's type. Unlike the kernel above, which scales sums, this one
// scales the operand, because a group's sum would have to leave tensor memory for every group. That is one rounding of half
// a step a weight, of random sign, beside the one of C: the error of C grows by less than the root of two.
// (Through shared memory, written once and read by every MMA, the operand made that memory the bound: 2048 rows, 11008 -> 4096, 149 us
// where this took 122.) Persistent where there are more tiles than SMs; a cluster shares a tile's K where there are fewer.
// What bounds it: for wide tiles the tensor cores at the clock the power cap leaves (2048 rows, 11008 -> 4096: 1.3 PFLOP/s at 141 to 142 us in a burst,
// 1.12 at 165 in a longer run); for narrow ones the way of a slab from barrier to barrier, some 0.28 us of 64 k (64 rows,
// 8192 x 8192: 22.9 us, where the weights alone would take 5.3).
namespace tall {
constexpr int SLAB_K = 256, TILE_K = 64, PACKED_BYTES = ROWS * SLAB_K / 2, MAX_STAGES = 8, MAX_RAW = 4, MAX_M = 256;
constexpr int WARP_X = 0, WARP_MMA = 1, WARP_RAW = 2, TEAMS = SLAB_K / TILE_K, TEAM = 4, FIRST_UNPACKER = 4, EPILOGUE = 4;
constexpr int FIRST_EPILOGUE = FIRST_UNPACKER + TEAMS * TEAM;
constexpr int TALL_THREADS = 32 * (FIRST_EPILOGUE + EPILOGUE), SMEM_MOST = 231936;
// Tensor memory: 256 columns of accumulators (two of up to 128, or one), and 32 columns for each 64 k of unpacked weights in a stage.
constexpr uint32_t TMEM_COLS = 512, WEIGHTS_AT = 256, WEIGHT_COLS = TILE_K / 2;

// Eight packed weights of one group -> (q - z) * s in the order of k, two to a register.
template <class T>
__device__ __forceinline__ void unpack_scaled(uint32_t w, uint32_t zero, uint32_t scale, uint32_t* p) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const uint32_t up = w >> 4;
#pragma unroll
    for (int b = 0; b < 4; b++) {
        const uint32_t v = and_or(__byte_perm(w, up, b | (4 + b) << 8), 0x000F000Fu, MAGIC<T>);
        const T2 a = __hmul2(__hsub2(*reinterpret_cast<const T2*>(&v), *reinterpret_cast<const T2*>(&zero)), *reinterpret_cast<const T2*>(&scale));
        p[b] = *reinterpret_cast<const uint32_t*>(&a);
    }
}
struct Shape {
    int M, N, K, group, tile_m, tiles_n, tiles, stages, raws, groups, split_shift, aligned;
};

// HALVES: 64-k tiles in a stage. Two, wherever three such stages fit (tiles of up to 240 columns): the tensor cores run dry while the
// issuing thread waits for a stage and its barrier's answer, some 250 clocks (before reads_done() was needed, 64 rows, 8192 x 8192: 24.5 us with one, 22.4 with
// two; 2048 rows, 11008 -> 4096, under the power cap: 170 and 156).
template <class T, int FLUSH, bool ZEROS, int HALVES>
__global__ void __launch_bounds__(TALL_THREADS, 1) matmul_w4_tall(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                  const T* __restrict__ scales, const uint8_t* __restrict__ zeros, T* __restrict__ C,
                                                                  int64_t ldc, const Shape p, int32_t* status) {
    using Scales = SlabScales<T, FLUSH, ZEROS>;
    constexpr int RAW_BYTES = PACKED_BYTES + Scales::BYTES, STAGE_K = TILE_K * HALVES, STAGE_COLS = WEIGHT_COLS * HALVES, SLAB_STAGES = SLAB_K / STAGE_K;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], raw_full[MAX_RAW], raw_empty[MAX_RAW], tfull_bar[2], tempty_bar[2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t gave_up;
    const uint32_t raw = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = raw + p.raws * RAW_BYTES;
    uint8_t* smem = smem_raw + (raw - smem_u32(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int shift = p.split_shift, splits = 1 << shift, split = blockIdx.x & (splits - 1);
    const int my_tile = blockIdx.x >> shift, step = gridDim.x >> shift;
    const int slabs = (p.K - 1) / SLAB_K + 1, first = slabs * split >> shift, slabs_here = (slabs * (split + 1) >> shift) - first;
    // Stages of a tile. A team's stages must follow one another by no more than the ring holds (three at least, five of 64 k), or its wait's parity
    // would name the phase after the next and let it through too early. Each has every fourth 64-k tile; a team whose share of the last slab lay
    // behind the end of K and was left out would next be needed three stages on where a stage is two tiles, seven where it is one:
    // there the slab is walked to its end, on zeros.
    const int count = HALVES == 1 ? slabs_here * SLAB_STAGES : min(slabs_here * SLAB_STAGES, (p.K - 1) / STAGE_K + 1 - first * SLAB_STAGES);
    const int first_group = (unsigned)(first * SLAB_K) / (unsigned)p.group;
    const int half_bytes = p.tile_m * TILE_K * 2, stage_bytes = half_bytes * HALVES, accs = p.tile_m <= 128 ? 2 : 1;   // with one accumulator, its drain is not hidden

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < p.stages; s++) {
            mbar_init(smem_u32(&full_bar[s]), 1 + TEAM * HALVES);   // the rows of X, and each warp of the teams that unpack it
            mbar_init(smem_u32(&empty_bar[s]), 1);
        }
        for (int s = 0; s < p.raws; s++) {
            mbar_init(smem_u32(&raw_full[s]), 1 + 32);   // the bulk load, and each lane's copies of scales
            mbar_init(smem_u32(&raw_empty[s]), TEAMS * TEAM);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(smem_u32(&tfull_bar[b]), 1);
            mbar_init(smem_u32(&tempty_bar[b]), EPILOGUE);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == WARP_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_slot;
    wait_for_predecessor();
    if (threadIdx.x == 0 && status && *reinterpret_cast<volatile int32_t*>(status) != 0) gave_up = 1;   // an earlier CTA gave up: do not pile on
    bool ok = true;

    if (warp == WARP_X) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            for (int t = my_tile; t < p.tiles && ok; t += step) {
                const int m0 = t / p.tiles_n * p.tile_m;
                for (int i = 0; i < count; i++) {
                    ok &= mbar_wait<LONG_WAIT>(smem_u32(&empty_bar[s]), ph ^ 1, &gave_up);
                    if (!ok) break;
                    const uint32_t fb = smem_u32(&full_bar[s]);
                    mbar_expect_tx(fb, stage_bytes);
#pragma unroll
                    for (int h = 0; h < HALVES; h++) tma_load_2d(ring + s * stage_bytes + h * half_bytes, &map_x, fb, first * SLAB_K + i * STAGE_K + h * TILE_K, m0);
                    if (++s == p.stages) s = 0, ph ^= 1;
                }
            }
            if (!ok) {   // let the copies already issued land before the CTA can exit
                const uint64_t t0 = global_ns();
                while (global_ns() - t0 < 2000000ull) {}
            }
        }
    } else if (warp == WARP_RAW) {
        int s = 0;
        uint32_t ph = 0;
        for (int t = my_tile; t < p.tiles && ok; t += step) {
            const int n0 = t % p.tiles_n * ROWS;
            const typename Scales::Copies copies(scales, zeros, n0, p.N, p.groups, lane);
            int start = first_group, in_group = first * SLAB_K - start * p.group;
            for (int i = 0; i < slabs_here; i++) {
                ok &= mbar_wait<LONG_WAIT>(smem_u32(&raw_empty[s]), ph ^ 1, &gave_up);
                if (!ok) break;
                const uint32_t fb = smem_u32(&raw_full[s]), at = raw + s * RAW_BYTES;
                if (lane == 0) {
                    mbar_expect_tx(fb, PACKED_BYTES);
                    tma_load_2d(at, &map_w, fb, (first + i) * SLAB_K / 2, n0);
                }
                copies(at + PACKED_BYTES, start, lane, p.aligned);
                copies_arrive(fb);
                for (in_group += SLAB_K; in_group >= p.group; in_group -= p.group) start++;
                if (++s == p.raws) s = 0, ph ^= 1;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (!ok) {
            const uint64_t t0 = global_ns();
            while (global_ns() - t0 < 2000000ull) {}
        }
    } else if (warp == WARP_MMA) {
        // The warp stays together (see umma_f16_tmem). It shares its scheduler with warps that unpack, every instruction waits its
        // turn, and a tile of 64 k has at most 512 clocks: no vote on the waits (after one that gave up, the rest of the way
        // is walked on whatever the memories hold), descriptors stepped by one addition a tile.
        const uint32_t type = std::is_same_v<T, __half> ? 0u : 1u;
        const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(p.tile_m >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
        const uint32_t full0 = smem_u32(&full_bar[0]), empty0 = smem_u32(&empty_bar[0]), end = full0 + 8 * p.stages, w0 = tmem_base + WEIGHTS_AT;
        const uint64_t x0 = smem_desc(ring, 16, 1024), x_step = stage_bytes >> 4, x_half = half_bytes >> 4;
        uint32_t bar = full0, w = w0, ph = 0, buf = 0, use = 0;
        uint64_t x = x0;
        for (int t = my_tile; t < p.tiles; t += step) {
            ok &= mbar_wait(smem_u32(&tempty_bar[buf]), (use & 1) ^ 1, &gave_up);
            const uint32_t acc = tmem_base + buf * 128;
            uint32_t accumulate = 0;
            for (int i = 0; i < count; i++) {
                ok &= mbar_wait(bar, ph, &gave_up);
                __syncwarp();
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int h = 0; h < HALVES; h++) {
#pragma unroll
                    for (int k = 0; k < TILE_K / 16; k++) {
                        umma_f16_tmem(acc, w + h * WEIGHT_COLS + 8 * k, x + h * x_half + (uint64_t)(2 * k), idesc, accumulate);
                        accumulate = 1;
                    }
                }
                umma_commit_elected(bar - full0 + empty0);
                bar += 8, w += STAGE_COLS, x += x_step;
                if (bar == end) bar = full0, w = w0, x = x0, ph ^= 1;
            }
            umma_commit_elected(smem_u32(&tfull_bar[buf]));
            if (++buf == (uint32_t)accs) buf = 0, use++;
        }
        if (!ok) {   // let the products already issued end before tensor memory is given back
            const uint64_t t0 = global_ns();
            while (global_ns() - t0 < 2000000ull) {}
        }
    } else if (warp >= FIRST_UNPACKER && warp < FIRST_EPILOGUE) {
        // Four teams of four warps take the four tiles of a slab of packed weights, so that each has four tiles' time for
        // the way from its barrier to the MMA's. This thread: row `row`, two 16-byte pieces in, its lane's 32 columns out.
        const int team = (warp - FIRST_UNPACKER) / TEAM, row = (warp & 3) * 32 + lane, groups = p.groups;
        const uint32_t row_at = row * 128, turn = row & 7;
        constexpr int PARTS = FLUSH == 1 ? 2 : 1;   // groups that 64 k may touch
        const bool whole = p.group <= SLAB_K && SLAB_K % p.group == 0;
        const int whole_shift = p.group == 32 ? 0 : p.group == 64 ? 1 : p.group == 128 ? 2 : 3;
        int steady[PARTS];   // groups from the slab's first to this thread's, where all slabs begin with a group
#pragma unroll
        for (int h = 0; h < PARTS; h++) steady[h] = (team * 2 + h) >> whole_shift;
        int rs = 0, at = 0;                         // `at`: the ring's place of this tile's first 64 k
        uint32_t rph = 0, ph = 0;
        const auto forward = [&](int& place, uint32_t& parity, int by) {
            for (place += by; place >= p.stages; place -= p.stages) parity ^= 1;
        };
        for (int t = my_tile; t < p.tiles && ok; t += step) {
            const uint32_t row_group = (uint32_t)min(t % p.tiles_n * ROWS + row, p.N - 1) * (uint32_t)groups;
            int place = at, start = first_group, in_start = first * SLAB_K - start * p.group;
            uint32_t parity = ph;
            forward(place, parity, team / HALVES);
            for (int j = 0; j < slabs_here; j++) {
                ok &= mbar_wait(smem_u32(&raw_full[rs]), rph, &gave_up);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint8_t* stage = smem + rs * RAW_BYTES;
                uint32_t s2[2], z2[2];
#pragma unroll
                for (int h = 0; h < PARTS; h++) {
                    int ahead = steady[h];
                    if (!whole) {   // groups that do not divide a slab
                        ahead = 0;
                        for (int k = in_start + team * TILE_K + h * UNIT_K; k >= p.group; k -= p.group) ahead++;
                    }
                    const bool in = start + ahead < groups;   // past the end of K: X is zero there, and so is the scale
                    const uint32_t scale = Scales::scale_bits(stage + PACKED_BYTES, row, row_group, start, ahead, p.aligned);
                    s2[h] = in ? scale * 0x10001u : 0u;
                    z2[h] = MAGIC<T> + 0x10001u * (ZEROS && in ? Scales::zero(stage + PACKED_BYTES, row, row_group, start, ahead, p.aligned) : 8);
                }
                if (PARTS == 1) s2[1] = s2[0], z2[1] = z2[0];
                if (whole) start += SLAB_K / 32 >> whole_shift;
                else for (in_start += SLAB_K; in_start >= p.group; in_start -= p.group) start++;
                uint32_t out[32];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(stage + row_at + (((2 * team + h) ^ turn) << 4));
                    unpack_scaled<T>(w.x, z2[h], s2[h], out + 16 * h), unpack_scaled<T>(w.y, z2[h], s2[h], out + 16 * h + 4);
                    unpack_scaled<T>(w.z, z2[h], s2[h], out + 16 * h + 8), unpack_scaled<T>(w.w, z2[h], s2[h], out + 16 * h + 12);
                }
                reads_done();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&raw_empty[rs]));
                if (++rs == p.raws) rs = 0, rph ^= 1;
                if (j * SLAB_STAGES + team / HALVES >= count) continue;   // this stage lies behind the end of K
                ok &= mbar_wait(smem_u32(&empty_bar[place]), parity ^ 1, &gave_up);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                tmem_store_32(tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + WEIGHTS_AT + place * STAGE_COLS + team % HALVES * WEIGHT_COLS, out);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&full_bar[place]));
                forward(place, parity, SLAB_STAGES);
            }
            forward(at, ph, count);
        }
    } else if (warp >= FIRST_EPILOGUE && splits == 1) {
        const int ew = warp & 3;   // this warp may touch lanes 32 ew .. 32 ew + 31
        uint32_t buf = 0, use = 0;
        for (int t = my_tile; t < p.tiles && ok; t += step) {
            const int n = t % p.tiles_n * ROWS + ew * 32 + lane, m0 = t / p.tiles_n * p.tile_m, rows = min(p.tile_m, p.M - m0);
            ok &= mbar_wait<LONG_WAIT>(smem_u32(&tfull_bar[buf]), use & 1, &gave_up);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = tmem_base + buf * 128 + ((uint32_t)(ew * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < rows; c += 16) {
                uint32_t r[16];
                __syncwarp();
                tmem_load_16(src + (uint32_t)c, r);
                if (n < p.N) {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (c + j < rows) store_as(C + (m0 + c + j) * ldc + n, __uint_as_float(r[j]));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&tempty_bar[buf]));
            if (++buf == (uint32_t)accs) buf = 0, use++;
        }
    }
    __syncwarp();

    if (splits > 1) {   // one tile a cluster: the CTAs' sums, added in the order of the CTAs
        __syncthreads();   // the ring is done with: its memory takes the sums
        float* sums = reinterpret_cast<float*>(smem);
        const int n0 = my_tile % p.tiles_n * ROWS, m0 = my_tile / p.tiles_n * p.tile_m, rows = min(p.tile_m, p.M - m0);
        if (warp >= FIRST_EPILOGUE) {
            const int ew = warp & 3;
            ok &= mbar_wait<LONG_WAIT>(smem_u32(&tfull_bar[0]), 0, &gave_up);   // on give-up the drain still runs on whatever tensor memory holds
            ok = __all_sync(0xffffffffu, ok);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < rows; c += 16) {
                uint32_t r[16];
                tmem_load_16(tmem_base + ((uint32_t)(ew * 32) << 16) + (uint32_t)c, r);
#pragma unroll
                for (int j = 0; j < 16; j++) sums[(c + j) * ROWS + ew * 32 + lane] = __uint_as_float(r[j]);
            }
        }
        __syncwarp();
        cluster_sync_all();
        for (int i = threadIdx.x; i < ((rows - split + splits - 1) >> shift) * ROWS; i += TALL_THREADS) {
            const int row = i % ROWS, c = (i / ROWS << shift) + split;
            if (n0 + row >= p.N) continue;
            const uint32_t at = smem_u32(&sums[c * ROWS + row]);
            float v = 0.0f;
            for (int q = 0; q < splits; q++) v += load_cluster_f32(map_to_cta(at, q));
            store_as(C + (m0 + c) * ldc + n0 + row, v);
        }
        __syncwarp();
        cluster_sync_all();   // no CTA leaves while another reads its sums
    }
    if (!ok && status) atomicExch(status, 1);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == WARP_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}
}  // namespace tall

struct Args {
    const void *x, *w, *scales;
    const uint8_t* zeros;
    void* c;
    int64_t ldx, ldw, ldc;
    int M, N, K, group;
    int32_t* status;
    cudaStream_t stream;
};

const char* const WHO = "matmul_w4";

template <class T>
constexpr CUtensorMapDataType MAP_TYPE = std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;

// CTAs that share a tile's K, as a power of two, in the kernel for few rows: two fit an SM; split while the tiles leave room and every share
// keeps two slabs.
int few_shift(int64_t tiles, int slabs) {
    int shift = 0;
    while (shift < 3 && tiles << (shift + 1) <= 2 * basalt_k::sm_count() && slabs >= 4 << shift) shift++;
    return shift;
}

template <class T, int NT, int FLUSH, bool ZEROS>
int launch_few(const Args& p) {
    constexpr int TOKENS = 8 * NT, smem = few::Stage<T, NT, FLUSH, ZEROS>::SMEM;
    constexpr auto kern = few::matmul_w4_kernel<T, NT, FLUSH, ZEROS>;
    if (const int rc = basalt_k::allow_smem<kern>(WHO, smem)) return rc;
    const int tiles_n = (p.N - 1) / ROWS + 1, slabs = (p.K - 1) / few::SLAB_K + 1, groups = (p.K - 1) / p.group + 1;
    const int64_t tiles = (int64_t)tiles_n * ((p.M - 1) / TOKENS + 1);
    const int shift = few_shift(tiles, slabs);
    CUtensorMap mw, mx;
    if (const int rc = make_tensor_map(&mw, WHO, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, p.N, ((int64_t)p.K + 1) / 2, p.ldw, few::SLAB_K / 2, ROWS)) return rc;
    // one launch takes 65535 tiles of rows of X
    for (int m = 0; m < p.M; m += 65535 * TOKENS) {
        const int rows = p.M - m < 65535 * TOKENS ? p.M - m : 65535 * TOKENS;
        if (const int rc = make_tensor_map(&mx, WHO, MAP_TYPE<T>, (const T*)p.x + m * p.ldx, rows, p.K, p.ldx * 2, few::X_BOX_K, rows < TOKENS ? rows : TOKENS, CU_TENSOR_MAP_SWIZZLE_NONE))
            return rc;
        const dim3 grid(tiles_n << shift, (rows - 1) / TOKENS + 1);
        if (const int rc = basalt_k::launch_clusters(WHO, kern, grid, few::THREADS, smem, 1 << shift, p.stream, mw, mx, (const T*)p.scales, p.zeros, (T*)p.c + m * p.ldc, p.ldc, rows,
                                                     p.N, p.K, p.group, groups, (int)SlabScales<T, FLUSH, ZEROS>::aligned(p.scales, p.zeros, p.group, groups), shift, p.status))
            return rc;
    }
    return 0;
}

// The width of a tile of the tcgen05 kernel and the CTAs that share its K (one CTA fits an SM): of the few counts of tiles over M that come near
// 256 columns each, the one that costs least. A slab costs what its products do, two clocks a column and 64 k, and not less than
// its unpacking, about 112 columns' worth. (128 rows through 8192 x 8192: tiles of 128 with K shared 25.4 us, of 64 without some 37.)
struct TallPlan {
    int width, tiles, shift;
    double time;   // us
};
TallPlan plan_tall(int M, int N, int K) {
    const int sms = basalt_k::sm_count(), slabs = (K - 1) / tall::SLAB_K + 1;
    TallPlan best = {0, 0, 0, 1e300};
    for (int tiles_m = (M - 1) / tall::MAX_M + 1, tries = 0; tries < 4; tries++, tiles_m++) {
        const int width = ((M - 1) / tiles_m + 16) / 16 * 16;
        const int64_t tiles = (int64_t)((M - 1) / width + 1) * ((N - 1) / ROWS + 1);
        if (tiles > INT32_MAX / 2) continue;
        int shift = 0;
        while (shift < 3 && tiles << (shift + 1) <= sms && slabs >= 4 << shift) shift++;
        const double units = (double)((tiles - 1) / sms + 1) * ((slabs - 1 >> shift) + 1) * (width > 112 ? width : 112);
        const double time = 6.5 + 0.9 / 112 * units + (shift ? 0.5 * (1 << shift) : 0.0);
        if (time < best.time) best = {width, (int)tiles, shift, time};
    }
    return best;
}

template <class T, int FLUSH, bool ZEROS>
int launch_tall(const Args& p, const TallPlan& plan) {
    constexpr int RAW_BYTES = tall::PACKED_BYTES + SlabScales<T, FLUSH, ZEROS>::BYTES;
    const int sms = basalt_k::sm_count(), groups = (p.K - 1) / p.group + 1;
    tall::Shape q = {p.M, p.N, p.K, p.group, plan.width, (p.N - 1) / ROWS + 1, plan.tiles, 0, 0, groups, plan.shift, SlabScales<T, FLUSH, ZEROS>::aligned(p.scales, p.zeros, p.group, groups)};
    const int halves = q.tile_m <= 240 ? 2 : 1, stage = q.tile_m * tall::TILE_K * 2 * halves;
    q.raws = q.tile_m > 160 ? 2 : tall::MAX_RAW;
    q.stages = (tall::SMEM_MOST - 1024 - q.raws * RAW_BYTES) / stage;
    if (q.stages > tall::MAX_STAGES / halves) q.stages = tall::MAX_STAGES / halves;   // as many as tensor memory has columns for
    // The whole SM's shared memory is asked for, used or not. The kernel takes all of the SM's tensor memory, and its clusters' CTAs wait for
    // one another: beside a kernel of another stream that does the same, each could hold what the other's CTA waits for.
    const int smem = tall::SMEM_MOST;
    const int splits = 1 << q.split_shift;
    CUtensorMap mw, mx;
    if (const int rc = make_tensor_map(&mw, WHO, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, p.N, ((int64_t)p.K + 1) / 2, p.ldw, tall::SLAB_K / 2, ROWS)) return rc;
    if (const int rc = make_tensor_map(&mx, WHO, MAP_TYPE<T>, p.x, p.M, p.K, p.ldx * 2, tall::TILE_K, q.tile_m)) return rc;
    const auto go = [&](auto two) {
        constexpr auto kern = tall::matmul_w4_tall<T, FLUSH, ZEROS, decltype(two)::value>;
        if (const int rc = basalt_k::allow_smem<kern>(WHO, tall::SMEM_MOST)) return rc;
        return basalt_k::launch_clusters(WHO, kern, splits > 1 || q.tiles < sms ? q.tiles * splits : sms, tall::TALL_THREADS, smem, splits, p.stream, mw, mx, (const T*)p.scales,
                                         p.zeros, (T*)p.c, p.ldc, q, p.status);
    };
    return halves == 2 ? go(std::integral_constant<int, 2>()) : go(std::integral_constant<int, 1>());
}

// Up to 16 rows go through the kernel for few rows. More do so in tiles of 16, where that is the shorter way: 2.5 us and 1.6 a slab and
// round of CTAs against the estimate above. (Tiles of 16 / tcgen05, measured: 48 rows, 4096 -> 1024: 7.2 / 8.9 us; 64 rows, 4096 -> 4096:
// 13.9 / 10.5; 17 rows, 8192 -> 8192: 24.4 / 21.1; 64 rows, 2048 -> 2048: 7.1 / 7.5.) Under 128 rows of weights most of the tcgen05 kernel's lanes would idle.
template <class T, int FLUSH, bool ZEROS>
int launch_rows(const Args& p) {
    if (p.M <= 8) return launch_few<T, 1, FLUSH, ZEROS>(p);
    if (p.M > 16 && p.N >= ROWS) {
        const int slabs = (p.K - 1) / few::SLAB_K + 1;
        const int64_t tiles = (int64_t)((p.M - 1) / 16 + 1) * ((p.N - 1) / ROWS + 1);
        const int shift = few_shift(tiles, slabs);
        const TallPlan plan = plan_tall(p.M, p.N, p.K);
        if (!plan.tiles) return basalt_k::record_msg(1, WHO, "M * N is too large");
        if (plan.time < 2.5 + 1.6 * (double)(((tiles << shift) - 1) / (2 * basalt_k::sm_count()) + 1) * ((slabs - 1 >> shift) + 1)) return launch_tall<T, FLUSH, ZEROS>(p, plan);
    }
    return launch_few<T, 2, FLUSH, ZEROS>(p);
}

template <class T, int FLUSH>
int launch_zeros(const Args& p) { return p.zeros ? launch_rows<T, FLUSH, true>(p) : launch_rows<T, FLUSH, false>(p); }

template <class T>
int launch_type(const Args& p) {
    const int units = p.group / UNIT_K;
    return units % 4 == 0 ? launch_zeros<T, 4>(p) : units % 2 == 0 ? launch_zeros<T, 2>(p) : launch_zeros<T, 1>(p);
}

}  // namespace

extern "C" int basalt_k_matmul_w4(int type, const void* X, int64_t ldx, const void* W, int64_t ldw, const void* scales, const uint8_t* zeros, int group, void* C,
                                  int64_t ldc, int M, int N, int K, int32_t* status, void* stream) {
    if (type != BASALT_K_TYPE_F16 && type != BASALT_K_TYPE_BF16) return basalt_k::record_msg(1, WHO, "X must be f16 or bf16");
    if (M < 0 || N < 0) return basalt_k::record_msg(1, WHO, "M and N must not be negative");
    if (K < 1) return basalt_k::record_msg(1, WHO, "K must be at least 1");
    if (M > 1 << 30 || N > 1 << 30 || K > 1 << 30) return basalt_k::record_msg(1, WHO, "M, N and K must not exceed 2^30");
    if (group < UNIT_K || group % UNIT_K) return basalt_k::record_msg(1, WHO, "the group must be a multiple of 32");
    if (!M || !N) return 0;
    if (!X || !W || !C || !scales) return basalt_k::record_msg(1, WHO, "X, W, C and the scales are needed");
    if (((uintptr_t)X | (uintptr_t)W) & 15 || ldw & 15 || ldx & 7) return basalt_k::record_msg(1, WHO, "X and W and their row strides must be multiples of 16 bytes");
    if (ldx < K || ldw < ((int64_t)K + 1) / 2 || ldc < N) return basalt_k::record_msg(1, WHO, "a row stride lies below the row");
    if (ldx >= (int64_t)1 << 31 || ldw >= (int64_t)1 << 31 || ldc >= (int64_t)1 << 31) return basalt_k::record_msg(1, WHO, "a row stride lies above 2^31 - 1");
    if (((uintptr_t)scales | (uintptr_t)zeros) % 4) return basalt_k::record_msg(1, WHO, "the scales and the zero points must start at a multiple of 4 bytes");
    if ((uintptr_t)C % 2 || (uintptr_t)status % 4) return basalt_k::record_msg(1, WHO, "C or the status is not aligned to its elements");
    const int64_t groups = (K - 1) / group + 1, packed = ((int64_t)K + 1) / 2;
    const basalt_k::Span c = {C, M, N, ldc, 2};
    if (overlap(c, {X, M, K, ldx, 2}) || overlap(c, {W, N, packed, ldw, 1}) || overlap(c, {scales, N, groups, groups, 2}) || overlap(c, {zeros, N, groups, groups, 1}))
        return basalt_k::record_msg(1, WHO, "C overlaps an input");
    if (const int rc = basalt_k::check_device_pointers(WHO, {X, W, scales, zeros, C, status})) return rc;
    const Args p = {X, W, scales, zeros, C, ldx, ldw, ldc, M, N, K, group, status, (cudaStream_t)stream};
    return type == BASALT_K_TYPE_F16 ? launch_type<__half>(p) : launch_type<__nv_bfloat16>(p);
}

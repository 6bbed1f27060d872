// Row operators in front of a quantised product: root-mean-square norm with the residual's addition, and the
// quantisation of rows to e4m3.
//
//   h = x + residual                              (f32)          total = h rounded to the rows' type
//   y = h * w / sqrt(mean(h^2) + eps)             (f32)
//   s = max(max_k |y_k| / 448, 2^-126)            one per row    q = y / s (f32) rounded to e4m3
//
// Both need one number of the whole row before the first output: the sum of squares and, because
// rounding is monotone (max_k |h_k w_k| * r is exactly max_k |h_k w_k r|), the largest |h_k w_k|. So one pass reads the
// row, one exchange between the row's threads joins both numbers, and the row is written from registers:
// every input is read once and every output written once.
//
// What bounds it: memory. 8192 x 8192 in f16 with a residual to e4m3: 470 MB in 72.2 us, 6.5 TB/s, what a plain copy reaches; 4096 x 14336 bf16 to
// e4m3: 176 MB in 30.8 us, 5.7 TB/s, with 69 % of the issue slots taken. One row of 4096 takes 2.1 us, a launch's time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "../../../include/basalt_b200_kernels.h"
#include "common.cuh"
#include "tensor_core.cuh"

namespace {

constexpr float E4M3_MAX = 448.0f;
constexpr float SCALE_MIN = 1.17549435e-38f;   // 2^-126: a row of zeros has a scale whose reciprocal is finite

struct Rows {
    const void *x, *residual, *weight;
    void *total, *y;
    float* scales;
    int ldx, ldr, ldt, ldy, rows, cols;   // (88 bytes of parameters; with 64-bit strides a launch took the host 0.3 us longer)
    float eps, per_col_high, per_col_low;   // 1 / cols, as a sum of two
};

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <class T>
__device__ __forceinline__ T rounded(float v) {
    if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
    else return v;
}

template <class T>
constexpr int VEC = 16 / sizeof(T);

__device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
template <class T>
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float2 p;
        if constexpr (std::is_same_v<T, __half>) p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
        f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
}
template <class T>
__device__ __forceinline__ void values(const uint4& u, float (&f)[VEC<T>]) {
    if constexpr (sizeof(T) == 4) unpack(u, f);
    else unpack<T>(u, f);
}
template <class T>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VEC<T>]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
        else if constexpr (std::is_same_v<T, __half>) {
            const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
            const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
// Two f32 in a 64-bit register, and arithmetic on both at once.
__device__ __forceinline__ uint64_t two(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ uint64_t mul_two(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint32_t four_e4m3(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
template <int N>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[N]) {
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = four_e4m3(f[0], f[1], f[2], f[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(four_e4m3(f[0], f[1], f[2], f[3]), four_e4m3(f[4], f[5], f[6], f[7]));
}
__device__ __forceinline__ uint8_t one_e4m3(float f) { return (uint8_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3); }

// The larger of two, NaN where either is: a NaN in a row reaches the row's scale instead of vanishing in it.
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// Joins the sum of squares and the largest magnitude over the blockDim.x threads of a row (a power of two below 32, or
// whole warps), in an order that does not change. blockDim.y rows share the block, so every thread of it has to call this.
__device__ __forceinline__ void join_row(float& sum, float& top) {
    const int width = blockDim.x < 32 ? blockDim.x : 32;
    for (int d = width / 2; d; d /= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
    }
    if (blockDim.x <= 32) return;
    __shared__ float sums[32], tops[32];   // rows of more than a warp: warps in the block <= 32
    const int warp = (threadIdx.y * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, first = threadIdx.y * warps;
    if (lane == 0) sums[warp] = sum, tops[warp] = top;
    __syncthreads();
    sum = lane < warps ? sums[first + lane] : 0.0f;
    top = lane < warps ? tops[first + lane] : 0.0f;
    for (int d = 16; d; d /= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
    }
}

// What the joined numbers make of a row's values: y = v * r and, for e4m3, y / scale = v * (r / scale). The row's first thread stores the scale.
//
// The quotient is the f32 one by the stored scale, so that a y half-way between two e4m3 numbers is rounded as a tie, which a product with a
// rounded reciprocal is not (8 bits of x over 8 bits of the maximum meet ties often: 8 bytes in 10,000 of bf16 rows went to the other neighbour).
// A division each would cost more than everything else that is done for an element. So r / scale is kept as a sum of two f32,
// high + low, that is off by 2^-45 of it (2^-30 where the row's largest number lies near f32's, because low is subnormal then), and
// v * high + (v * low) is one product and one fused multiply-add, rounded once: a quotient that f32 holds is exact, and no other is off by more than half a step
// and 2^-30 of it. `high` lies a little below, so that `low` is positive and a zero keeps its sign.
// (Calls behind one another from cold memory, so / with the product alone: 4096 x 14336 bf16 32.7 / 31.6 us; 8192 x 8192 f16 norm with residual 76.1 / 76.0;
// 1023 x 5003 bf16 norm, element by element, 9.7 / 9.1.)
template <bool NORM, bool E4M3>
struct Factor {
    float lift, high, low;
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) const {
        if (NORM && E4M3 && lift != 1.0f)   // all threads of a row go one way
#pragma unroll
            for (int j = 0; j < N; j++) v[j] *= lift;
        // Two at a time, the norm into e4m3 is left more of the issue slots (8192 x 8192: 76.4 us, one at a time 77.3); rows that are only
        // quantised come out of 16-bit pairs and lose more to moves between registers (4096 x 14336: 34.0 us, one at a time 33.3).
        if constexpr (NORM && E4M3) {
            const uint64_t h = two(high, high), l = two(low, low);
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const uint64_t pair = two(v[j], v[j + 1]), q = fma_two(pair, h, mul_two(pair, l));
                v[j] = __uint_as_float((uint32_t)q), v[j + 1] = __uint_as_float((uint32_t)(q >> 32));
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = E4M3 ? fmaf(v[j], high, v[j] * low) : v[j] * high;
        }
    }
};
constexpr float BELOW = 1.0f - 0x1p-22f;   // more than the hardware's reciprocal is off by
constexpr float MAX_HIGH = (float)(1.0 / 448.0) * BELOW, MAX_LOW = (float)(1.0 / 448.0 - (double)MAX_HIGH);
template <bool NORM, bool E4M3>
__device__ __forceinline__ Factor<NORM, E4M3> row_factor(const Rows& p, int64_t row, bool active, float sum, float top) {
    float r = 1.0f;
    if (NORM) {
        const float square = fmaf(sum, p.per_col_high, sum * p.per_col_low) + p.eps;
        r = rsqrtf(square);   // the hardware's, two steps off at most; after one of Newton's one
        if (square >= 0x1p-126f && square <= FLT_MAX) r = fmaf(0.5f * r, fmaf(-square * r, r, 1.0f), r);
    }
    if (!E4M3) return {1.0f, r, 0.0f};
    const float most = top * r;
    float scale = most < 0x1p-80f ? most / E4M3_MAX : fmaf(most, MAX_HIGH, most * MAX_LOW);   // the nearest to the quotient, which is 1 / 14 of a step or more from any middle
    if (scale < SCALE_MIN) scale = SCALE_MIN;   // false for a NaN, which stays
    if (active && threadIdx.x == 0) p.scales[row] = scale;
    // A norm of rows so small that r / scale could exceed f32 lifts them first, exactly: zeros, first of all, whose r is 1 / sqrt(eps) and whose scale is
    // 2^-126. Their bytes are zeros, and 0 * inf is none.
    const float lift = NORM && top < 0x1p-90f ? 0x1p100f : 1.0f;
    const float divisor = scale * lift;   // 2^-126 to 2^119.2: its reciprocal is a normal number (that of the row's maximum is subnormal above 2^126)
    float high;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(high) : "f"(divisor));
    high *= BELOW;
    float low = fmaf(-high, divisor, 1.0f) * high;
    if (isinf(divisor)) low = 0.0f;   // a row with an infinity: finite values give 0 * (0 + 0), the infinity NaN
    if (NORM) {
        const float product = r * high * BELOW;
        low = fmaf(r, low, fmaf(r, high, -product));
        high = product;
    }
    return {lift, high, low};
}

// The largest magnitude in a vector of T; 16-bit values are compared two at a time as they are.
template <class T>
__device__ __forceinline__ float magnitude(const uint4& u) {
    if constexpr (sizeof(T) == 4) {
        return max_nan(max_nan(fabsf(__uint_as_float(u.x)), fabsf(__uint_as_float(u.y))), max_nan(fabsf(__uint_as_float(u.z)), fabsf(__uint_as_float(u.w))));
    } else {
        using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
        const uint32_t w[4] = {u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu, u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu};
        const T2* v = reinterpret_cast<const T2*>(w);
        const T2 m = __hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3]));
        return max_nan(load_one(&m.x), load_one(&m.y));
    }
}

// Rows whose pointers, strides and width are whole 16-byte vectors, V of them in each thread's registers. Every load of the
// row is issued before its first use and before any store (an output may be an input's buffer, so the compiler
// keeps their order): the loads in flight are what the memory is kept busy with (8192 x 8192 with a residual: 102.6 us with the
// residual's loads between total's stores, 72.0 so). Without a residual the row stays
// in its own type until it is written; with one, h is kept in f32.
template <class T, bool NORM, bool RESIDUAL, bool E4M3, int V>
__global__ void __launch_bounds__(V == 1 ? 1024 : 512) rows_in_registers(const Rows p) {
    constexpr int W = VEC<T>;
    basalt_k::tc::wait_for_predecessor();
    const int64_t row64 = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const bool active = row64 < p.rows;
    const int64_t row = active ? row64 : 0;   // times a stride in 64 bits
    const int vectors = active ? p.cols / W : 0;
    const uint4* x = (const uint4*)((const T*)p.x + row * p.ldx) + threadIdx.x;
    uint4 raw[V];
#pragma unroll
    for (int v = 0; v < V; v++)
        if (threadIdx.x + v * blockDim.x < vectors) raw[v] = x[v * blockDim.x];
    float h[RESIDUAL ? V : 1][W], sum = 0.0f, top = 0.0f;
    if constexpr (RESIDUAL) {
        const uint4* residual = (const uint4*)((const T*)p.residual + row * p.ldr) + threadIdx.x;
        uint4 more[V];
#pragma unroll
        for (int v = 0; v < V; v++)
            if (threadIdx.x + v * blockDim.x < vectors) more[v] = residual[v * blockDim.x];
        T* total = (T*)p.total + row * p.ldt + threadIdx.x * W;
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (threadIdx.x + v * blockDim.x >= vectors) continue;
            float r[W];
            values<T>(raw[v], h[v]);
            values<T>(more[v], r);
#pragma unroll
            for (int j = 0; j < W; j++) h[v][j] += r[j];
            if (p.total) store_vec(total + v * blockDim.x * W, h[v]);
        }
    }
    const uint4* weight = (const uint4*)p.weight + threadIdx.x;
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (threadIdx.x + v * blockDim.x >= vectors) continue;
        if constexpr (!NORM) top = max_nan(top, magnitude<T>(raw[v]));
        else {
            float once[W];
            float(&e)[W] = RESIDUAL ? h[v] : once;
            if (!RESIDUAL) values<T>(raw[v], e);
#pragma unroll
            for (int j = 0; j < W; j++) sum += e[j] * e[j];
            if (p.weight && (E4M3 || RESIDUAL)) {
                float w[W];
                values<T>(weight[v * blockDim.x], w);
#pragma unroll
                for (int j = 0; j < W; j++) e[j] *= w[j];
            }
            if (E4M3) {
#pragma unroll
                for (int j = 0; j < W; j++) top = max_nan(top, fabsf(e[j]));
            }
        }
    }
    join_row(sum, top);
    const auto f = row_factor<NORM, E4M3>(p, row, active, sum, top);
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (threadIdx.x + v * blockDim.x >= vectors) continue;
        float once[W];
        float(&e)[W] = RESIDUAL ? h[v] : once;
        if (!RESIDUAL) {
            values<T>(raw[v], e);
            if (NORM && p.weight) {
                float w[W];
                values<T>(weight[v * blockDim.x], w);
#pragma unroll
                for (int j = 0; j < W; j++) e[j] *= w[j];
            }
        }
        f(e);
        const int at = (threadIdx.x + v * blockDim.x) * W;
        if constexpr (E4M3) store_e4m3((uint8_t*)p.y + row * p.ldy + at, e);
        else store_vec((T*)p.y + row * p.ldy + at, e);
    }
}

// Rows that start at no vector boundary, or whose width is no whole number of vectors, up to EACH * 512 elements: a block per
// row, element by element, one read of the row. Bound by its instructions (1023 x 5003 bf16 to e4m3: 9.7 us, 1.6 TB/s).
constexpr int EACH = 16;
template <class T, bool NORM, bool RESIDUAL, bool E4M3>
__global__ void __launch_bounds__(512) rows_by_element(const Rows p) {
    basalt_k::tc::wait_for_predecessor();
    const int64_t row = blockIdx.x;
    const T* x = (const T*)p.x + row * p.ldx + threadIdx.x;
    const int left = p.cols - threadIdx.x, step = blockDim.x;   // element v of this thread is in the row where v * step < left
    T raw[EACH], more[RESIDUAL ? EACH : 1];
#pragma unroll
    for (int v = 0; v < EACH; v++)
        if (v * step < left) raw[v] = x[v * step];
    if constexpr (RESIDUAL) {
        const T* residual = (const T*)p.residual + row * p.ldr + threadIdx.x;
#pragma unroll
        for (int v = 0; v < EACH; v++)
            if (v * step < left) more[v] = residual[v * step];
    }
    T by[NORM ? EACH : 1];
    const bool weighted = NORM && p.weight;
    if constexpr (NORM) {
        const T* weight = (const T*)p.weight + threadIdx.x;
#pragma unroll
        for (int v = 0; v < EACH; v++)
            if (weighted && v * step < left) by[v] = weight[v * step];
    }
    T* total = RESIDUAL && p.total ? (T*)p.total + row * p.ldt + threadIdx.x : nullptr;
    float h[EACH], sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int v = 0; v < EACH; v++) {
        const bool in = v * step < left;
        h[v] = in ? load_one(&raw[v]) : 0.0f;
        if constexpr (RESIDUAL) {
            if (in) h[v] += load_one(&more[v]);
            if (in && total) total[v * step] = rounded<T>(h[v]);
        }
        sum += h[v] * h[v];
        if constexpr (NORM)
            if (in && weighted) h[v] *= load_one(&by[v]);
        if (E4M3) top = max_nan(top, fabsf(h[v]));
    }
    join_row(sum, top);
    const auto f = row_factor<NORM, E4M3>(p, row, true, sum, top);
    f(h);
    T* y = (T*)p.y + row * p.ldy + threadIdx.x;
    uint8_t* bytes = (uint8_t*)p.y + row * p.ldy + threadIdx.x;
#pragma unroll
    for (int v = 0; v < EACH; v++) {
        if (v * step >= left) continue;
        if constexpr (E4M3) bytes[v * step] = one_e4m3(h[v]);
        else y[v * step] = rounded<T>(h[v]);
    }
}

// Any alignment, any width: a block per row, element by element, the row read twice (the second time from
// cache). Only the second pass writes, so that total may be the residual's own buffer.
template <class T, bool NORM, bool E4M3>
__global__ void __launch_bounds__(512) rows_twice(const Rows p) {
    basalt_k::tc::wait_for_predecessor();
    const int64_t row = blockIdx.x;
    const T* x = (const T*)p.x + row * p.ldx;
    const T* residual = NORM && p.residual ? (const T*)p.residual + row * p.ldr : nullptr;
    const T* weight = NORM ? (const T*)p.weight : nullptr;
    float sum = 0.0f, top = 0.0f;
    for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
        float h = load_one(x + i);
        if (residual) h += load_one(residual + i);
        sum += h * h;
        if (weight) h *= load_one(weight + i);
        top = max_nan(top, fabsf(h));
    }
    join_row(sum, top);
    const auto f = row_factor<NORM, E4M3>(p, row, true, sum, top);
    for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
        float h = load_one(x + i);
        if (residual) {
            h += load_one(residual + i);
            if (p.total) ((T*)p.total)[row * p.ldt + i] = rounded<T>(h);
        }
        if (weight) h *= load_one(weight + i);
        float v[2] = {h, h};
        f(v);
        if (E4M3) ((uint8_t*)p.y)[row * p.ldy + i] = one_e4m3(v[0]);
        else ((T*)p.y)[row * p.ldy + i] = rounded<T>(v[0]);
    }
}

template <class T, bool NORM, bool E4M3>
int launch(const Rows& p, const char* who, cudaStream_t s) {
    constexpr int W = VEC<T>;
    const bool eight = E4M3;
    uintptr_t all = (uintptr_t)p.x | (uintptr_t)p.residual | (uintptr_t)p.weight | (uintptr_t)p.total;
    int64_t strides = p.ldx | p.cols;
    if (p.residual) strides |= p.ldr;
    if (p.total) strides |= p.ldt;
    const bool y_vec = eight ? (uintptr_t)p.y % W == 0 && p.ldy % W == 0 : (uintptr_t)p.y % 16 == 0 && p.ldy % W == 0;
    const int64_t vectors = p.cols / W;
    const bool by_vector = all % 16 == 0 && strides % W == 0 && y_vec;
    if (!by_vector && p.cols <= EACH * 512) {
        auto kern = rows_by_element<T, NORM, false, E4M3>;
        if constexpr (NORM)
            if (p.residual) kern = rows_by_element<T, NORM, true, E4M3>;
        // every slot of a thread is worked through, used or not: as few threads as hold a long row, more for a short one
        const int each = p.cols > 4 * 256 ? EACH : 4, threads = ((p.cols + each - 1) / each + 31) / 32 * 32;
        return basalt_k::launch_clusters(who, kern, p.rows, threads, 0, 1, s, p);
    }
    if (!by_vector || vectors > 8 * 512) {
        return basalt_k::launch_clusters(who, rows_twice<T, NORM, E4M3>, p.rows, 512, 0, 1, s, p);
    }
    // Vectors a thread: one where the rows are few and each should be over soon; four where there are rows for every SM, so that
    // what a thread spends on joining and on the row's factor is shared by more elements (8192 x 8192: a thousand threads of one
    // vector each executed 41 instructions an element and took 105 us, of four 22 and 102, before the loads were put first).
    const bool few = p.rows <= basalt_k::sm_count();
    const int v = vectors <= 1024 && few ? 1 : vectors <= 4 * 512 ? 4 : 8;
    int tpr = (int)((vectors + v - 1) / v);
    if (tpr > 32) tpr = (tpr + 31) / 32 * 32;
    else {
        int t = 1;
        while (t < tpr) t *= 2;
        tpr = t;
    }
    const int per_block = tpr >= 128 ? 1 : 128 / tpr;
    const dim3 block(tpr, per_block), grid((unsigned)(((int64_t)p.rows + per_block - 1) / per_block));
    const auto pick = [&](auto residual) {
        constexpr bool R = decltype(residual)::value;
        return v == 1 ? rows_in_registers<T, NORM, R, E4M3, 1> : v == 4 ? rows_in_registers<T, NORM, R, E4M3, 4> : rows_in_registers<T, NORM, R, E4M3, 8>;
    };
    auto kern = pick(std::false_type());
    if constexpr (NORM)
        if (p.residual) kern = pick(std::true_type());
    return basalt_k::launch_clusters(who, kern, grid, block, 0, 1, s, p);
}

template <bool NORM, bool E4M3>
int launch_type(int type, const Rows& p, const char* who, cudaStream_t s) {
    if (type == BASALT_K_TYPE_F16) return launch<__half, NORM, E4M3>(p, who, s);
    if (type == BASALT_K_TYPE_BF16) return launch<__nv_bfloat16, NORM, E4M3>(p, who, s);
    return launch<float, NORM, E4M3>(p, who, s);
}

using basalt_k::Span;

int check_rows(const char* who, int type, int64_t rows, int64_t cols, const Span& x, const Span& residual, const Span& total, const Span& y, const float* scales,
               const void* weight) {
    if (type != BASALT_K_TYPE_F16 && type != BASALT_K_TYPE_BF16 && type != BASALT_K_TYPE_F32) return basalt_k::record_msg(1, who, "unknown type");
    if (rows < 0 || rows > INT32_MAX) return basalt_k::record_msg(1, who, "rows must lie in 0 .. 2^31 - 1");
    if (cols < 1 || cols > INT32_MAX) return basalt_k::record_msg(1, who, "cols must lie in 1 .. 2^31 - 1");
    if (!x.p || !y.p) return basalt_k::record_msg(1, who, "the input and the output are needed");
    for (const Span* m : {&x, &residual, &total, &y}) {
        if (!m->p) continue;
        if (m->ld < cols || m->ld >= (int64_t)1 << 31) return basalt_k::record_msg(1, who, "a row stride lies below cols or above 2^31 - 1");
        if ((uintptr_t)m->p % m->size) return basalt_k::record_msg(1, who, "a matrix is not aligned to its elements");
    }
    if ((uintptr_t)scales % 4 || (uintptr_t)weight % x.size) return basalt_k::record_msg(1, who, "the scales or the weight are not aligned to their elements");
    // Rows are read and written in no order: an output may be an input's own buffer, element for element, and must not overlap it otherwise.
    const Span w = {weight, 1, cols, cols, x.size}, s = {scales, 1, rows, rows, 4};
    for (const Span* out : {&total, &y})
        for (const Span* in : {&x, &residual})
            if (overlap(*out, *in) && !(out->p == in->p && out->ld == in->ld && out->size == in->size))
                return basalt_k::record_msg(1, who, "an output overlaps an input without being the same matrix");
    if (overlap(total, y)) return basalt_k::record_msg(1, who, "the outputs overlap");
    if (overlap(w, total) || overlap(w, y) || overlap(w, s)) return basalt_k::record_msg(1, who, "an output overlaps the weight");
    for (const Span* m : {&x, &residual, &total, &y})
        if (overlap(s, *m)) return basalt_k::record_msg(1, who, "the scales overlap a matrix");
    return 0;
}

}  // namespace

extern "C" int basalt_k_rms_norm(int type, const void* x, int64_t ldx, const void* residual, int64_t ldr, void* total, int64_t ldt, const void* weight,
                                 float eps, void* y, int64_t ldy, float* scales, int64_t rows, int64_t cols, void* stream) {
    const char* who = "rms_norm";
    const int size = type == BASALT_K_TYPE_F32 ? 4 : 2;
    if (const int rc = check_rows(who, type, rows, cols, {x, rows, cols, ldx, size}, {residual, rows, cols, ldr, size}, {total, rows, cols, ldt, size},
                                {y, rows, cols, ldy, scales ? 1 : size}, scales, weight)) return rc;
    if (total && !residual) return basalt_k::record_msg(1, who, "total is written only where a residual is added");
    if (!(eps >= 0.0f)) return basalt_k::record_msg(1, who, "eps must not be negative");
    if (rows == 0) return 0;
    if (const int rc = basalt_k::check_device_pointers(who, {x, residual, total, weight, y, scales})) return rc;
    const float high = (float)(1.0 / (double)cols) * (1.0f - 0x1p-22f);
    const Rows p = {x, residual, weight, total, y, scales, (int)ldx, (int)ldr, (int)ldt, (int)ldy, (int)rows, (int)cols, eps, high, (float)(1.0 / (double)cols - (double)high)};
    return scales ? launch_type<true, true>(type, p, who, (cudaStream_t)stream) : launch_type<true, false>(type, p, who, (cudaStream_t)stream);
}

extern "C" int basalt_k_quantize_e4m3(int type, const void* x, int64_t ldx, void* q, int64_t ldq, float* scales, int64_t rows, int64_t cols, void* stream) {
    const char* who = "quantize_e4m3";
    if (!scales) return basalt_k::record_msg(1, who, "the scales are needed");
    if (const int rc = check_rows(who, type, rows, cols, {x, rows, cols, ldx, type == BASALT_K_TYPE_F32 ? 4 : 2}, {}, {}, {q, rows, cols, ldq, 1}, scales, nullptr)) return rc;
    if (rows == 0) return 0;
    if (const int rc = basalt_k::check_device_pointers(who, {x, q, scales})) return rc;
    const Rows p = {x, nullptr, nullptr, nullptr, q, scales, (int)ldx, 0, 0, (int)ldq, (int)rows, (int)cols, 0.0f, 0.0f, 0.0f};
    return launch_type<false, true>(type, p, who, (cudaStream_t)stream);
}

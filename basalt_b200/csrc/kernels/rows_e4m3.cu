// Row operators in front of a quantised product: root-mean-square norm with the residual's addition, and the
// quantisation of rows to e4m3.
//
//   h = x + residual                              (f32)          total = h rounded to the rows' type
//   y = h * w / sqrt(mean(h^2) + eps)             (f32)
//   s = max(max_k |y_k| / 448, 2^-126)            one per row    q = y / s rounded to e4m3
//
// Both need one number of the whole row before the first output: the sum of squares and, because
// rounding is monotone (max_k |h_k w_k| * r is exactly max_k |h_k w_k r|), the largest |h_k w_k|. So one pass reads the
// row, one exchange between the row's threads joins both numbers, and the row is written from registers:
// every input is read once and every output written once.
//
// What bounds it: memory. 8192 x 8192 in f16 with a residual to e4m3: 470 MB in 72.0 us, 6.5 TB/s, what a plain copy reaches; 4096 x 14336 bf16 to
// e4m3: 176 MB in 29.7 us, 5.9 TB/s. One row of 4096 takes 2.1 us, a launch's time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../../include/basalt_b200_kernels.h"
#include "common.cuh"
#include "tensor_core.cuh"

namespace {

constexpr float E4M3_MAX = 448.0f;
constexpr float SCALE_MIN = 1.17549435e-38f;   // 2^-126: a row of zeros has a scale whose reciprocal is finite
constexpr float SMALL = 1e-15f;   // 448 / SMALL * r stays below 2^127 while r, which is at most 1 / sqrt(eps), does not exceed 1e20

struct Rows {
    const void *x, *residual, *weight;
    void *total, *y;
    float* scales;
    int64_t ldx, ldr, ldt, ldy;
    int rows, cols;
    float eps, per_col;   // per_col: 1 / cols
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

// What the row's outputs are multiplied by, from the joined numbers, in two factors; the row's first thread stores the scale. The reciprocal
// square root is the hardware's, off by at most two f32 steps, 2^-22 of the value. The reciprocal is that of the scale, which lies between 2^-126 and
// 2^119.2: the row's maximum goes up to 2^128, and the reciprocal of one above 2^126 would be subnormal. The second factor is one but for rows so small that the product of both could exceed f32
// (zeros, first of all, whose r is 1 / sqrt(eps) and whose scale is 2^-126: their bytes are zeros, and 0 * inf is none).
struct Factor {
    float first, second;
};
__device__ __forceinline__ float operator*(float v, const Factor& f) {
    v *= f.first;
    return f.second == 1.0f ? v : v * f.second;   // all threads of a row go one way
}
template <bool NORM, bool E4M3>
__device__ __forceinline__ Factor row_factor(const Rows& p, int row, bool active, float sum, float top) {
    const float r = NORM ? rsqrtf(sum * p.per_col + p.eps) : 1.0f;
    if (!E4M3) return {r, 1.0f};
    float most = top * r;
    if (most < E4M3_MAX * SCALE_MIN) most = E4M3_MAX * SCALE_MIN;   // false for a NaN, which stays
    if (active && threadIdx.x == 0) p.scales[row] = most / E4M3_MAX;
    const float inverse = __frcp_rn(most / E4M3_MAX);   // of the scale: the maximum's own would be a subnormal number above 2^126
    if (NORM && most < SMALL) return {r, inverse};
    return {r * inverse, 1.0f};
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
    const int row = active ? (int)row64 : 0, vectors = active ? p.cols / W : 0;
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
    const Factor f = row_factor<NORM, E4M3>(p, row, active, sum, top);
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
#pragma unroll
        for (int j = 0; j < W; j++) e[j] = e[j] * f;
        const int at = (threadIdx.x + v * blockDim.x) * W;
        if constexpr (E4M3) store_e4m3((uint8_t*)p.y + row * p.ldy + at, e);
        else store_vec((T*)p.y + row * p.ldy + at, e);
    }
}

// Rows that start at no vector boundary, or whose width is no whole number of vectors, up to EACH * 512 elements: a block per
// row, element by element, one read of the row. Bound by its instructions (1023 x 5003 bf16 to e4m3: 8.7 us, 1.8 TB/s; reading twice 14.3).
constexpr int EACH = 16;
template <class T, bool NORM, bool RESIDUAL, bool E4M3>
__global__ void __launch_bounds__(512) rows_by_element(const Rows p) {
    basalt_k::tc::wait_for_predecessor();
    const int row = blockIdx.x;
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
    const Factor f = row_factor<NORM, E4M3>(p, row, true, sum, top);
    T* y = (T*)p.y + row * p.ldy + threadIdx.x;
    uint8_t* bytes = (uint8_t*)p.y + row * p.ldy + threadIdx.x;
#pragma unroll
    for (int v = 0; v < EACH; v++) {
        if (v * step >= left) continue;
        if constexpr (E4M3) bytes[v * step] = (uint8_t)__nv_cvt_float_to_fp8(h[v] * f, __NV_SATFINITE, __NV_E4M3);
        else y[v * step] = rounded<T>(h[v] * f);
    }
}

// Any alignment, any width: a block per row, element by element, the row read twice (the second time from
// cache). Only the second pass writes, so that total may be the residual's own buffer.
template <class T, bool NORM, bool E4M3>
__global__ void __launch_bounds__(512) rows_twice(const Rows p) {
    basalt_k::tc::wait_for_predecessor();
    const int row = blockIdx.x;
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
    const Factor f = row_factor<NORM, E4M3>(p, row, true, sum, top);
    for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
        float h = load_one(x + i);
        if (residual) {
            h += load_one(residual + i);
            if (p.total) ((T*)p.total)[row * p.ldt + i] = rounded<T>(h);
        }
        if (weight) h *= load_one(weight + i);
        if (E4M3) ((uint8_t*)p.y)[row * p.ldy + i] = (uint8_t)__nv_cvt_float_to_fp8(h * f, __NV_SATFINITE, __NV_E4M3);
        else ((T*)p.y)[row * p.ldy + i] = rounded<T>(h * f);
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
    const Rows p = {x, residual, weight, total, y, scales, ldx, ldr, ldt, ldy, (int)rows, (int)cols, eps, 1.0f / (float)cols};
    return scales ? launch_type<true, true>(type, p, who, (cudaStream_t)stream) : launch_type<true, false>(type, p, who, (cudaStream_t)stream);
}

extern "C" int basalt_k_quantize_e4m3(int type, const void* x, int64_t ldx, void* q, int64_t ldq, float* scales, int64_t rows, int64_t cols, void* stream) {
    const char* who = "quantize_e4m3";
    if (!scales) return basalt_k::record_msg(1, who, "the scales are needed");
    if (const int rc = check_rows(who, type, rows, cols, {x, rows, cols, ldx, type == BASALT_K_TYPE_F32 ? 4 : 2}, {}, {}, {q, rows, cols, ldq, 1}, scales, nullptr)) return rc;
    if (rows == 0) return 0;
    if (const int rc = basalt_k::check_device_pointers(who, {x, q, scales})) return rc;
    const Rows p = {x, nullptr, nullptr, nullptr, q, scales, ldx, 0, 0, ldq, (int)rows, (int)cols, 0.0f, 0.0f};
    return launch_type<false, true>(type, p, who, (cudaStream_t)stream);
}

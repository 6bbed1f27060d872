// Shared helpers of the hand-written kernels' host launchers.
#pragma once
#include <cuda_runtime.h>

#include <stdint.h>

#include <initializer_list>

namespace basalt_k {

// SM count of the current device (148 on a B200), cached per device.
int sm_count();
// Stores a failing error code with its text for basalt_k_last_error(); returns the code.
int record(cudaError_t e, const char* what);
int record_msg(int code, const char* what, const char* msg);

// Refuses pointers that do not lie in memory of the current device (NULL passes): a kernel that followed one would fault.
int check_device_pointers(const char* who, std::initializer_list<const void*> pointers);

// Rows of a matrix as the argument checks see them: `ld` and `cols` in elements of `size` bytes.
struct Span {
    const void* p;
    int64_t rows, cols, ld;
    int size;
};
// Whether the address ranges of two matrices meet.
inline bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || a.rows < 1 || b.rows < 1) return false;
    const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
    return a0 < b0 + (uintptr_t)(((b.rows - 1) * b.ld + b.cols) * b.size) && b0 < a0 + (uintptr_t)(((a.rows - 1) * a.ld + a.cols) * a.size);
}

// Resident CTAs per SM for `kernel` at the given block size, from the occupancy calculator.
template <class K>
int resident_ctas(K kernel, int threads, size_t dyn_smem = 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, dyn_smem) != cudaSuccess || n < 1) n = 1;
    return n;
}

}  // namespace basalt_k

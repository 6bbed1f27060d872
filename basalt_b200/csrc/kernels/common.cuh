// Shared helpers of the hand-written kernels' host launchers.
#pragma once
#include <cuda_runtime.h>

#include <stdint.h>

#include <atomic>
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
// Whether two matrices have bytes in common. Two of one stride whose columns lie beside one another (the halves of a wider buffer's rows) have none.
inline bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || a.rows < 1 || b.rows < 1) return false;
    const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
    if (a0 >= b0 + (uintptr_t)(((b.rows - 1) * b.ld + b.cols) * b.size) || b0 >= a0 + (uintptr_t)(((a.rows - 1) * a.ld + a.cols) * a.size)) return false;
    if (a.ld * a.size != b.ld * b.size || a.cols > a.ld || b.cols > b.ld) return true;
    const int64_t stride = a.ld * a.size, step = (int64_t)(b0 - a0) % stride, at = step < 0 ? step + stride : step;   // of b's first column, from a's
    return at < a.cols * a.size || at + b.cols * b.size > stride;
}

// Lets KERNEL have `bytes` of dynamic shared memory on the current device; asked of the runtime once a kernel and device.
template <auto KERNEL>
int allow_smem(const char* who, int bytes) {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    if (const cudaError_t e = cudaGetDevice(&device)) return record(e, who);
    if (device < 64 && (done.load(std::memory_order_relaxed) >> device & 1)) return 0;
    if (const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return record(e, who);
    if (device < 64) done.fetch_or((uint64_t)1 << device, std::memory_order_relaxed);
    return 0;
}

// Launches `kernel` on `grid` CTAs in clusters of `cluster`, with programmatic stream serialisation: its prologue may run
// while the kernel before it in the stream drains, so it has to call tc::wait_for_predecessor() before it touches global memory.
template <class... P, class... A>
int launch_clusters(const char* who, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return record(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...), who);
}

// Resident CTAs per SM for `kernel` at the given block size, from the occupancy calculator.
template <class K>
int resident_ctas(K kernel, int threads, size_t dyn_smem = 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, dyn_smem) != cudaSuccess || n < 1) n = 1;
    return n;
}

}  // namespace basalt_k

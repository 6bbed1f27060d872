#include "common.cuh"

#include <cstdio>
#include <cstring>

#include "../../../include/basalt_b200_kernels.h"
#include "tensor_core.cuh"

namespace basalt_k {

static thread_local char g_msg[256] = "";

int sm_count() {
    static int cached[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!cached[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
        cached[dev] = n;
    }
    return cached[dev];
}

int record(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return 0;
    snprintf(g_msg, sizeof g_msg, "%s: %s", what, cudaGetErrorString(e));
    return (int)e;
}

int record_msg(int code, const char* what, const char* msg) {
    snprintf(g_msg, sizeof g_msg, "%s: %s", what, msg);
    return code;
}

namespace {

template <class Fn>
Fn driver_entry(const char* name) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) return (Fn)p;
    return nullptr;
}

}  // namespace

int tc::make_tensor_map(CUtensorMap* map, const char* who, CUtensorMapDataType type, const void* base, uint64_t rows, uint64_t cols, uint64_t stride,
                        uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    static const auto enc = driver_entry<decltype(&cuTensorMapEncodeTiled)>("cuTensorMapEncodeTiled");
    if (!enc) return record_msg(1, who, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {stride};
    const cuuint32_t box[2] = {box_cols, box_rows}, estr[2] = {1, 1};
    const CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return record_msg((int)r, who, "cuTensorMapEncodeTiled failed");
    return 0;
}

int check_device_pointers(const char* who, std::initializer_list<const void*> pointers) {
    static const auto get = driver_entry<decltype(&cuPointerGetAttribute)>("cuPointerGetAttribute");
    int current = 0;
    if (const cudaError_t e = cudaGetDevice(&current)) return record(e, who);
    if (!get) return record_msg(1, who, "cuPointerGetAttribute is not available from this driver");
    for (const void* p : pointers) {
        int device = -1;
        if (!p) continue;
        if (get(&device, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, (CUdeviceptr)p) != CUDA_SUCCESS) return record_msg(1, who, "an argument does not point to device memory");
        if (device != current) return record_msg(1, who, "an argument points to memory of another device than the current one");
    }
    return 0;
}

}  // namespace basalt_k

extern "C" const char* basalt_k_last_error(void) { return basalt_k::g_msg; }

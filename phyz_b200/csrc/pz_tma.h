// Tensor maps and launch setup of the recurrent-block operators' kernels: host
// side.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace pz {

// cuTensorMapEncodeTiled through the runtime's entry point lookup (the library
// links no driver stub).
inline CUresult encode_tiled(CUtensorMap* map, CUtensorMapDataType type, unsigned rank, void* base,
                             const cuuint64_t* size, const cuuint64_t* stride_bytes, const cuuint32_t* box,
                             CUtensorMapSwizzle swizzle) {
    using Fn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Fn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (Fn)p;
    }();
    if (!fn) return CUDA_ERROR_NOT_FOUND;
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    return fn(map, type, rank, base, size, stride_bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// A kernel's dynamic shared memory, set once per device (two threads that both do
// so set the same).
struct SmemOnce {
    std::atomic<bool> ready[64];
    template <class F>
    cudaError_t smem(F* kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess || (dev < 64 && ready[dev].load(std::memory_order_acquire))) return e;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && dev < 64) ready[dev].store(true, std::memory_order_release);
        return e;
    }
};

// The device address of a file's fault word (`symbol`), looked up once per device.
struct FaultWord {
    std::atomic<unsigned int*> at[64];
    template <class S>
    unsigned int* get(const S& symbol) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return nullptr;
        unsigned int* p = at[dev].load(std::memory_order_acquire);
        if (!p) {
            void* q = nullptr;
            if (cudaGetSymbolAddress(&q, symbol) != cudaSuccess) return nullptr;
            at[dev].store(p = (unsigned int*)q, std::memory_order_release);
        }
        return p;
    }
};

}  // namespace pz

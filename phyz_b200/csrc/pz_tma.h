// Tensor maps of the recurrent-block operators' TMA copies: host side.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

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

}  // namespace pz

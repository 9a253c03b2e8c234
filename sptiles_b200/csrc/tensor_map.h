// tensor_map.h -- tiled tensor maps (TMA descriptors) by the driver's encoder.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <string>

#include "common.h"

namespace st {

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// Boxes (128-byte-swizzled, unless told otherwise) of a tensor of `rank` dimensions, the first one
// contiguous; strides in bytes, of the second dimension on.
inline int make_tensor_map(CUtensorMap *map, const char *what, CUtensorMapDataType type, int rank, const void *base,
                           const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                           CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    auto fn = tensor_map_encoder();
    if (!fn) return fail(ST_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, type, static_cast<cuuint32_t>(rank), const_cast<void *>(base), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string("cuTensorMapEncodeTiled rejected ") + what + " (error " +
                                                 std::to_string(static_cast<int>(r)) + ")");
    return ST_OK;
}

}  // namespace st

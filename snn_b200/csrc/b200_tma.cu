// Tensor maps: the driver's encoder, found through the runtime.
#include "b200_tma.h"

namespace b200 {
namespace tma {
namespace {

using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                            const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                            CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {
    static const Encode f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (Encode)p;
    }();
    return f;
}

}  // namespace

cudaError_t encode(CUtensorMap *map, CUtensorMapDataType type, uint32_t rank, const void *base, const cuuint64_t *dims,
                   const cuuint64_t *strides, const cuuint32_t *box, CUtensorMapSwizzle swizzle) {
    const Encode f = encoder();
    if (f == nullptr) return cudaErrorNotSupported;
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    return f(map, type, rank, const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

}  // namespace tma
}  // namespace b200

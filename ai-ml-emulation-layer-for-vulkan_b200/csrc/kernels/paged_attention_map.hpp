// Tensor maps over the paged int8 cache.
#pragma once

#include <string>

#include "paged_attention.hpp"
#include "tcgen05_common.cuh"

namespace mlel {

// Rows of `headDim` bytes of one half of the cache, in boxes of `width` bytes by `rows` rows: plain, or swizzled over the width (64
// or 128 bytes).  What lies behind the end of a row reads as zero.
inline bool makeCacheMap(CUtensorMap *map, const void *base, const PagedCache &c, int width, int rowsOfBox, bool swizzled) {
    tc::EncodeTiledFn fn = tc::encodeTiled();
    if (fn == nullptr) {
        setLastError("cuTensorMapEncodeTiled is not available from the driver");
        return false;
    }
    const cuuint64_t rows = cuuint64_t(c.pages) * c.heads * c.page;
    const cuuint64_t dims[3] = {cuuint64_t(c.headDim), rows, 1}, strides[2] = {cuuint64_t(c.headDim), rows * c.headDim};
    const cuuint32_t box[3] = {cuuint32_t(width), cuuint32_t(rowsOfBox), 1}, elemStrides[3] = {1, 1, 1};
    const tc::MapKey key{{6, reinterpret_cast<uint64_t>(base), dims[0], rows, uint64_t(width), uint64_t(rowsOfBox), swizzled ? 1u : 0u}};
    return tc::rememberedMap(map, key, [&](CUtensorMap *m) {
        const CUresult rc = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), dims, strides, box, elemStrides,
                               CU_TENSOR_MAP_INTERLEAVE_NONE,
                               !swizzled     ? CU_TENSOR_MAP_SWIZZLE_NONE
                               : width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                             : CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (rc != CUDA_SUCCESS) {
            setLastError("cuTensorMapEncodeTiled failed with code " + std::to_string(int(rc)));
        }
        return rc == CUDA_SUCCESS;
    });
}

} // namespace mlel

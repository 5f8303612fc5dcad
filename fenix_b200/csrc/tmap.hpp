// tmap.hpp — 2-D tensor maps for TMA loads. The encoder is the driver's, reached through the runtime, so the
// library links no driver stub.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

namespace fxk {

inline PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// Rows of 16-bit (elem = 2) or 8-byte (elem = 8) elements: `cols` of them in a row of `pitch` bytes (a multiple of
// 16, as the base is), boxes of box_cols x box_rows with 128 bytes in a box row, 128-byte swizzled in shared memory
// (16-byte cell c of row r lies at cell c ^ (r % 8)). Out of range reads as zero.
inline cudaError_t tmap_rows(CUtensorMap* map, const void* base, int elem, int64_t cols, int64_t rows, int64_t pitch,
                             int box_rows) {
    if (!tmap_encoder()) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / elem), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t steps[2] = {1, 1};
    const CUtensorMapDataType type = elem == 8 ? CU_TENSOR_MAP_DATA_TYPE_INT64 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    return tmap_encoder()(map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

#ifdef __CUDACC__
// One box of a 2-D map into shared memory (128-byte aligned, 1024 for whole swizzle patterns); its bytes are counted
// on the mbarrier. x in elements: x * elem a multiple of 16 bytes.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
#endif

}  // namespace fxk

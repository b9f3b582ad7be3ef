// Host side of the TMA tile loads: the driver's tensor-map encoder, found once
// through the runtime (no link against libcuda), and the one map shape the
// attention kernels' page loads use.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

namespace rfx {
namespace tma {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// A [rows, cols] row-major bfloat16 matrix read in boxes of `box_rows` rows x 64
// columns (128 bytes) with the 128-byte swizzle: 16-byte chunk c of row r lands
// at chunk c ^ (r & 7) of that row's 128 bytes.  `cols` a multiple of 8, `base`
// 16-byte aligned.  `ld` (a multiple of 8): the elements from one row to the next, `cols` where it is 0.
inline bool make_map_rows64(CUtensorMap* map, const void* base, long long rows, int cols, int box_rows, long long ld = 0) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld ? ld : cols) * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tma
}  // namespace rfx

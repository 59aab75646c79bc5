// Tensor maps of the tensor-core kernels.
#include "umma.cuh"

namespace sgnn {

static int tensor_map(CUtensorMap *map, CUtensorMapDataType type, int bytes, const void *base, int64_t cols, int64_t rows, int64_t ld,
                      int planes, int64_t plane_stride, int box_cols, int box_rows, CUtensorMapSwizzle swizzle)
{
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;  // same value for every thread that finds it
    if (encode == nullptr) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        SGNN_CUDA_OK(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
        SGNN_REQUIRE(fn != nullptr && found == cudaDriverEntryPointSuccess, SGNN_ERR_CUDA, "cuTensorMapEncodeTiled is not there");
        encode = reinterpret_cast<Encode>(fn);
    }
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * bytes, (cuuint64_t)plane_stride * bytes};
    const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUresult rc = encode(map, type, 3, const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    SGNN_REQUIRE(rc == CUDA_SUCCESS, SGNN_ERR_CUDA, "tensor map of %lld x %lld (ld %lld) refused: %d", (long long)rows,
                 (long long)cols, (long long)ld, (int)rc);
    return SGNN_OK;
}

int umma_tensor_map(CUtensorMap *map, const void *base, bool bf16, int64_t cols, int64_t rows, int64_t ld, int planes,
                    int64_t plane_stride, int box_rows)
{
    return tensor_map(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, cols, rows, ld, planes,
                      plane_stride, 64, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

int raw_tensor_map(CUtensorMap *map, const void *base, int elem_bytes, int64_t cols, int64_t rows, int64_t ld, int box_cols, int box_rows)
{
    const CUtensorMapDataType t = elem_bytes == 4   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    return tensor_map(map, t, elem_bytes, base, cols, rows, ld, 1, rows * ld, box_cols, box_rows, CU_TENSOR_MAP_SWIZZLE_NONE);
}

int umma_store_map(CUtensorMap *map, void *base, StoreType type, int64_t cols, int64_t rows, int64_t ld, int planes,
                   int64_t plane_stride, int box_cols)
{
    const CUtensorMapDataType t = type == StoreType::kF32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : type == StoreType::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int bytes = type == StoreType::kF32 ? 4 : 2;
    return tensor_map(map, t, bytes, base, cols, rows, ld, planes, plane_stride, box_cols, 32,
                      box_cols * bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace sgnn

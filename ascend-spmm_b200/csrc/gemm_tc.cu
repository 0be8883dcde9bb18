// Host side of gemm_tc.cuh: tensor maps.
#include "gemm_tc.cuh"

#include "engine.h"

namespace spmmb {
namespace tc {

namespace {

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, found through the runtime (no link against libcuda).
EncodeTiled encoder()
{
    static const EncodeTiled f = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
                cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return f;
}

bool encode(CUtensorMap *map, const void *p, CUtensorMapDataType type, int rank, const cuuint64_t *dims,
            const cuuint64_t *strides, const cuuint32_t *box, CUtensorMapSwizzle swizzle)
{
    const EncodeTiled encode = encoder();
    if (!encode) return false;
    const cuuint32_t step[4] = {1, 1, 1, 1};
    for (int attempt = 0; attempt < 2; ++attempt) {
        const CUresult r = encode(map, type, rank, const_cast<void *>(p), dims, strides, box, step,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r == CUDA_SUCCESS) return true;
        // a thread that has made no runtime call yet (an autograd worker) has no
        // current context: setting its device binds the primary one
        int dev = 0;
        if (r != CUDA_ERROR_INVALID_CONTEXT || cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
            return false;
    }
    return false;
}

bool encode_map(CUtensorMap *map, const void *p, CUtensorMapDataType type, int size, int64_t inner, int64_t rows,
                int64_t batch, int64_t ld, int64_t batch_stride, int box_inner, int box_rows, CUtensorMapSwizzle swizzle)
{
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)batch};
    const cuuint64_t strides[2] = {(cuuint64_t)(ld * size), (cuuint64_t)((batch > 1 ? batch_stride : ld) * size)};
    const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, 1};
    return encode(map, p, type, 3, dims, strides, box, swizzle);
}

CUtensorMapDataType type16(bool bf16)
{
    return bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

}  // namespace

bool make_map(CUtensorMap *map, const void *p, int64_t inner, int64_t rows, int64_t batch, int64_t ld,
              int64_t batch_stride, int box_rows, bool bf16)
{
    return encode_map(map, p, type16(bf16), 2, inner, rows, batch, ld, batch_stride, kBK, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool make_blocked_map(CUtensorMap *map, const void *p, int64_t inner, int64_t rows, int64_t batch, int64_t ld,
                      int64_t batch_stride, int blocks, bool bf16)
{
    const cuuint64_t dims[4] = {64, (cuuint64_t)rows, (cuuint64_t)(inner / 64), (cuuint64_t)batch};
    const cuuint64_t strides[3] = {(cuuint64_t)(ld * 2), 128, (cuuint64_t)((batch > 1 ? batch_stride : ld) * 2)};
    const cuuint32_t box[4] = {64, 64, (cuuint32_t)blocks, 1};
    return encode(map, p, type16(bf16), 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool make_out_map(CUtensorMap *map, void *p, int64_t inner, int64_t rows, int64_t batch, int64_t ld,
                  int64_t batch_stride, int out_type)
{
    if (out_type == kOutF32)
        return encode_map(map, p, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, inner, rows, batch, ld, batch_stride, 32, 32,
                          CU_TENSOR_MAP_SWIZZLE_128B);
    return encode_map(map, p, type16(out_type == kOutBf16), 2, inner, rows, batch, ld, batch_stride, 32, 32,
                      CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace tc
}  // namespace spmmb

// Tensor maps of tiled copies. The driver's function is looked up through the runtime: the library is not linked with libcuda.
#ifndef ASP_TENSOR_MAP_H
#define ASP_TENSOR_MAP_H
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace asp
{
inline cudaError_t tensor_map(CUtensorMap *out, CUtensorMapDataType type, const void *p, uint64_t width, uint64_t height, uint64_t pitch_bytes, uint32_t box_width, uint32_t box_height,
                              bool swizzle = true)
{
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? (Encode)f : nullptr;
    }();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t size[2] = {width, height}, pitch[1] = {pitch_bytes};
    const cuuint32_t box[2] = {box_width, box_height}, step[2] = {1, 1};
    const CUresult r = encode(out, type, 2, const_cast<void *>(p), size, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
// rows of bytes, 128 columns a copy; what lies outside is read as zero
inline cudaError_t byte_map(CUtensorMap *out, const void *p, uint64_t width, uint64_t height, uint64_t pitch, uint32_t box_height, bool swizzle = true)
{
    return tensor_map(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, width, height, pitch, 128, box_height, swizzle);
}
} // namespace asp
#endif

// Tensor maps: descriptions of operands in device memory for TMA loads, made on the host.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace cutespmm {

// cuTensorMapEncodeTiled on the current device.  It is looked up through the runtime: the library does not link libcuda.  Being a call of the
// driver, it wants a context that is bound to the calling thread.  The runtime binds one with a thread's first call that does anything, and a
// thread whose memory is there already (an autograd engine's, a server's worker) may come here before any such call: setting the device that is
// current anyway binds it, also during a capture.
inline cudaError_t encode_tiled(CUtensorMap *out, CUtensorMapDataType type, uint32_t rank, const void *p, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                                CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion)
{
    using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                       const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                       CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeTiledFn enc = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    if (!enc) return cudaErrorNotSupported;
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    auto encode = [&] {
        return enc(out, type, rank, const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (encode()) return cudaSuccess;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e != cudaSuccess) return e;
    return encode() ? cudaSuccess : cudaErrorInvalidValue;
}

// The dense operand B for gather4 loads: a 2-D fp32 tensor (columns innermost, extent N; rows extent K, pitch ldb), and one
// cp.async.bulk.tensor...tile::gather4 brings four arbitrary rows of it, `box_cols` columns wide, into consecutive rows of shared
// memory.  Columns beyond N are filled with zeros without touching memory.
inline cudaError_t make_b_tensor_map(CUtensorMap *out, const float *B, uint64_t N, uint64_t K, uint64_t ldb, uint32_t box_cols,
                                     CUtensorMapSwizzle swizzle)
{
    const cuuint64_t dims[2] = {N, K};
    const cuuint64_t strides[1] = {ldb * sizeof(float)};
    const cuuint32_t box[2] = {box_cols, 1};
    return encode_tiled(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, B, dims, strides, box, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

}  // namespace cutespmm

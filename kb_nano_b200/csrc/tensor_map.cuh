// Tensor maps of the MXFP4 GEMM and of the few-row kernels, encoded with every call (a few hundredths of a
// microsecond each: remembering them by address saved nothing that could be measured).
#pragma once
#include <cuda.h>
#include <string.h>

#include <atomic>

#include "common.cuh"

namespace kbn {

struct TensorMapSpec {
    const void* base;
    uint64_t dims[3], strides[2];      // bytes; dimension 0 is contiguous
    uint32_t box[3];
    uint32_t rank, swizzle, promo;
};

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Byte-typed tiled map, out-of-range parts of a box filled with zeros.
static inline int encode_tensor_map(CUtensorMap* tm, const TensorMapSpec& s) {
    static std::atomic<EncodeTiled> known{nullptr};
    EncodeTiled encode = known.load(std::memory_order_acquire);
    if (encode == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        KBN_REQUIRE(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess,
                    KBN_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
        encode = reinterpret_cast<EncodeTiled>(p);
        known.store(encode, std::memory_order_release);
    }
    cuuint64_t dims[3], strides[2];
    cuuint32_t box[3], one[3] = {1, 1, 1};
    for (int i = 0; i < 3; ++i) dims[i] = s.dims[i], box[i] = s.box[i];
    for (int i = 0; i < 2; ++i) strides[i] = s.strides[i];
    const CUresult r = encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.rank, const_cast<void*>(s.base), dims, strides, box, one,
                                                        CU_TENSOR_MAP_INTERLEAVE_NONE, static_cast<CUtensorMapSwizzle>(s.swizzle),
                                                        static_cast<CUtensorMapL2promotion>(s.promo), CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    KBN_REQUIRE(r == CUDA_SUCCESS, KBN_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%llu x %llu x %llu)", (int)r,
                (unsigned long long)s.dims[0], (unsigned long long)s.dims[1], (unsigned long long)s.dims[2]);
    return KBN_OK;
}

}  // namespace kbn

// Tensor maps of the MXFP4 GEMM and of the few-row kernels, with a small per-thread cache.  A map depends on nothing but
// the arguments it was encoded from (address, extents, strides, box), so an entry stays valid whatever happens to the
// memory behind the address.
#pragma once
#include <cuda.h>
#include <string.h>

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
    struct Entry {
        TensorMapSpec spec;
        CUtensorMap tm;
        bool used;
    };
    static thread_local Entry cache[64];
    uint64_t h = 0x9e3779b97f4a7c15ull;
    const uint64_t key[] = {reinterpret_cast<uintptr_t>(s.base), s.dims[0], s.dims[1], s.dims[2], s.strides[0], s.strides[1], s.box[1], s.swizzle};
    for (uint64_t k : key) h = (h ^ k) * 0xff51afd7ed558ccdull, h ^= h >> 29;
    Entry& e = cache[(h >> 40) & 63];
    if (e.used && memcmp(&e.spec, &s, sizeof(s)) == 0) {
        *tm = e.tm;
        return KBN_OK;
    }
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    KBN_REQUIRE(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess,
                KBN_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[3], strides[2];
    cuuint32_t box[3], one[3] = {1, 1, 1};
    for (int i = 0; i < 3; ++i) dims[i] = s.dims[i], box[i] = s.box[i];
    for (int i = 0; i < 2; ++i) strides[i] = s.strides[i];
    const CUresult r = reinterpret_cast<EncodeTiled>(p)(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.rank, const_cast<void*>(s.base), dims, strides, box, one,
                                                        CU_TENSOR_MAP_INTERLEAVE_NONE, static_cast<CUtensorMapSwizzle>(s.swizzle),
                                                        static_cast<CUtensorMapL2promotion>(s.promo), CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    KBN_REQUIRE(r == CUDA_SUCCESS, KBN_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%llu x %llu x %llu)", (int)r,
                (unsigned long long)s.dims[0], (unsigned long long)s.dims[1], (unsigned long long)s.dims[2]);
    e.spec = s;
    e.tm = *tm;
    e.used = true;
    return KBN_OK;
}

}  // namespace kbn

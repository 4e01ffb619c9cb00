// Arithmetic of the MXFP4 format (blocks of 32 values along K: e2m1 codes, two per byte with the even element in the low
// nibble, and one E8M0 scale byte b = 2^(b-127) per block), shared by the quantisers and the kernels that quantise or
// dequantise on the way.
//
// Scale rule: the smallest power of two under which no value is clipped, 2^ceil(log2(amax / 6)).  With
// amax = 1.m * 2^(E-127) that is exponent byte E - 2, plus one iff 1.m > 1.5; a byte below 0 (amax under 2^-125) is
// raised to 0, which only makes the codes smaller.  The format has no zero scale: an all-zero block has byte 0 and codes 0.
// A block that holds an infinity or a NaN gets byte 255, the format's NaN: every value read back from it is NaN.
#pragma once
#include "common.cuh"

namespace kbn {
namespace mxfp4 {

constexpr int kBlock = 32;

// Per 16-bit half the larger of two unsigned values: on |bf16| bit patterns the order is that of the values, infinities
// above every finite value and NaNs above infinities, so that neither is lost in a maximum.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// |bf16| bit pattern of a block's largest magnitude -> E8M0 byte.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
    const int e = (int)(amax >> 7) - 2 + ((amax & 0x7fu) > 0x40u ? 1 : 0);
    return amax >= 0x7f80u ? 255u : (uint32_t)max(e, 0);
}

// 2^(127 - b), what a block's values are multiplied by before they are rounded to e2m1 (0 for the NaN byte: codes 0).
__device__ __forceinline__ float inv_scale(uint32_t b) { return b == 255u ? 0.0f : __uint_as_float((254u - b) << 23); }

// 2^(b - 127), exactly, with the subnormal 2^-127 and the NaN.
__device__ __forceinline__ float scale_value(uint32_t b) {
    return __uint_as_float(b == 0u ? 0x00400000u : (b == 255u ? 0x7fc00000u : b << 23));
}

// Two E8M0 bytes (the low half of w) -> two packed bf16 values, with the subnormal and the NaN.  Exact.
__device__ __forceinline__ uint32_t scale_bf16x2(uint32_t w) {
    uint32_t d;
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %1;\n\t"
        "cvt.rn.bf16x2.ue8m0x2 %0, a;\n\t}"
        : "=r"(d)
        : "r"(w));
    return d;
}

// Two fp32 values -> one byte of two e2m1 codes (lo in the low nibble), round to nearest even, saturating at +-6.
__device__ __forceinline__ uint32_t pack_e2m1x2(float lo, float hi) {
    uint32_t d;
    asm("{\n\t.reg .b8 c, z;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n\t"
        "mov.b16 {z, _}, 0;\n\t"
        "mov.b32 %0, {c, z, z, z};\n\t}"
        : "=r"(d)
        : "f"(lo), "f"(hi));
    return d;
}

// Eight bf16 values (packed pairs) times `inv` -> eight codes in one word.
__device__ __forceinline__ uint32_t quant8(const uint32_t (&w)[4], float inv, bool nan_block) {
    if (nan_block) return 0u;          // inf * 0 would be a NaN, which the conversion has no code for
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= pack_e2m1x2(__fmul_rn(bf16_lo(w[i]), inv), __fmul_rn(bf16_hi(w[i]), inv)) << (8 * i);
    return r;
}

// One byte of two codes -> two f16 values.  Exact.
__device__ __forceinline__ uint32_t unpack_e2m1x2(uint32_t byte) {
    uint32_t d;
    asm("{\n\t.reg .b8 c, x, y, z;\n\t"
        "mov.b32 {c, x, y, z}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, c;\n\t}"
        : "=r"(d)
        : "r"(byte));
    return d;
}
// Four bytes of codes -> eight f16 values.
__device__ __forceinline__ void unpack_e2m1x8(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

// kbn_quant_mxfp4 (mxfp4_quant.cu).  behind_gemm: the calls come in a row with GEMMs.
int quantise(const void* x, int64_t M, int64_t K, int64_t ld_x, void* q, int64_t ld_q, void* scale, int64_t s_row, void* sf_packed, bool behind_gemm, cudaStream_t st);

// Position of a row's scale word for 128-K block kb in the packed layout the tensor core reads: per 128 rows and 128 of K
// 128 words, word (l, i) <-> row 32 i + l; the word's four bytes are the scales of the block's four 32-value groups.
__host__ __device__ __forceinline__ size_t packed_word(int64_t row, int64_t kb, int64_t kblocks) {
    return ((size_t)(row >> 7) * (size_t)kblocks + (size_t)kb) * 128u + (size_t)((row & 31) * 4 + ((row & 127) >> 5));
}

}  // namespace mxfp4
}  // namespace kbn

// MXFP4 quantisers and their inverse: bf16 -> e2m1 codes + E8M0 scales (plain and behind SiLU(gate)*up), codes -> bf16,
// and the repacking of row-major scales into the layout of the tensor core.  The 4-bit counterparts of the 1x128 FP8
// quantisers (kb-nano has FP8 only: tasks/baseline/L1/fp8_linear.py:181-215, tasks/baseline/L1/silu_mul_quant_fp8.py:23-76).
//
// All four are HBM-bound: 2 B in and 17/32 B out per element (4 B in with the activation), the inverse the other way round.
// A half-warp takes 128 consecutive values of a row (16 bytes a lane), so a block of 32 is four lanes: two shuffles give
// its largest magnitude, and the four scale bytes of the 128 values meet in one word, which is stored whole, both in the
// row-major scales and in the packed layout.
#include "mxfp4.cuh"
#include "silu_exact.cuh"

namespace kbn {
namespace mxfp4 {

// Where the results go.  scale and packed may each be null.
struct QuantOut {
    uint8_t* q;
    int64_t ld_q;          // bytes between rows
    uint8_t* scale;        // [M, K/32], row stride s_row
    int64_t s_row;
    uint32_t* packed;
    int64_t kblocks;
    bool word_scales;      // the row-major scales allow 4-byte stores
};

// The 16 lanes of a half-warp hold 8 values each of columns [128 g, 128 g + 128) of `row` (lanes past K hold zeros and
// live == false).  Quantises and stores them.
__device__ __forceinline__ void quant_group(const uint32_t (&w)[4], bool live, int64_t row, uint32_t g, uint32_t j, uint32_t K, const QuantOut& o) {
    uint32_t m = max_u16x2(max_u16x2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), max_u16x2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    m = max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t b = scale_byte(max(m & 0xffffu, m >> 16));
    // the four blocks' bytes in one word, in every lane; blocks past K count as 2^0, so that nothing read there is a NaN
    uint32_t word = (g * 128u + j * 8u < K ? b : 127u) << (8u * (j >> 2));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if (live) {
        *reinterpret_cast<uint32_t*>(o.q + row * o.ld_q + g * 64u + j * 4u) = quant8(w, inv_scale(b), b == 255u);
        if (o.scale != nullptr) {
            uint8_t* s = o.scale + row * o.s_row + g * 4u;
            if (o.word_scales && g * 128u + 128u <= K) {
                if (j == 0) *reinterpret_cast<uint32_t*>(s) = word;
            } else if ((j & 3u) == 0) {
                s[j >> 2] = (uint8_t)b;
            }
        }
        if (o.packed != nullptr && j == 0) o.packed[packed_word(row, g, o.kblocks)] = word;
    }
}

// VEC: rows of x start on 16-byte boundaries.  U groups of 128 per half-warp, all loads issued before the first use.
template <bool VEC, int U>
__global__ void __launch_bounds__(256)
quant_mxfp4_kernel(const __nv_bfloat16* __restrict__ x, uint32_t K, int64_t ld_x, QuantOut o, uint32_t G, uint32_t chunks_per_row, uint32_t n_chunks) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // a GEMM behind this kernel waits before it reads
    const uint32_t j = threadIdx.x & 15u;
    const uint32_t chunk = blockIdx.x * 16u + (threadIdx.x >> 4);
    const bool valid = chunk < n_chunks;
    const uint32_t row = valid ? chunk / chunks_per_row : 0u;
    const uint32_t g0 = (chunk - row * chunks_per_row) * U;
    const uint16_t* xr = reinterpret_cast<const uint16_t*>(x) + (int64_t)row * ld_x;
    uint32_t w[U][4];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t col = (g0 + u) * 128u + j * 8u;
        live[u] = valid && g0 + u < G && col < K;
        if (VEC) {
            const uint4 v = live[u] ? __ldcs(reinterpret_cast<const uint4*>(xr + col)) : make_uint4(0, 0, 0, 0);
            w[u][0] = v.x; w[u][1] = v.y; w[u][2] = v.z; w[u][3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[u][i] = live[u] ? (uint32_t)xr[col + 2 * i] | ((uint32_t)xr[col + 2 * i + 1] << 16) : 0u;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) quant_group(w[u], live[u], row, g0 + u, j, K, o);
}

// bf16(bf16(silu(gate)) * up) with the exactly rounded SiLU of the FP8 activation kernel (silu_exact.cuh), then as above.
// The two roundings to bf16 are those of an unfused activation in the model's type, so that fused and unfused layers agree.
template <bool VEC, int U>
__global__ void __launch_bounds__(256)
silu_mul_quant_mxfp4_kernel(const __nv_bfloat16* __restrict__ in, uint32_t N2, int64_t ld_in, QuantOut o, uint32_t G, uint32_t chunks_per_row,
                            uint32_t n_chunks, const uint16_t* __restrict__ table) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t j = threadIdx.x & 15u;
    const uint32_t chunk = blockIdx.x * 16u + (threadIdx.x >> 4);
    const bool valid = chunk < n_chunks;
    const uint32_t row = valid ? chunk / chunks_per_row : 0u;
    const uint32_t g0 = (chunk - row * chunks_per_row) * U;
    const uint16_t* gr = reinterpret_cast<const uint16_t*>(in) + (int64_t)row * ld_in;
    uint4 gate[U], up[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t col = (g0 + u) * 128u + j * 8u;
        live[u] = valid && g0 + u < G && col < N2;
        gate[u] = up[u] = make_uint4(0, 0, 0, 0);
        if (live[u]) {
            if (VEC) {
                gate[u] = __ldcs(reinterpret_cast<const uint4*>(gr + col));
                up[u] = __ldcs(reinterpret_cast<const uint4*>(gr + N2 + col));
            } else {
                uint32_t a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = (uint32_t)gr[col + 2 * i] | ((uint32_t)gr[col + 2 * i + 1] << 16);
                    b[i] = (uint32_t)gr[N2 + col + 2 * i] | ((uint32_t)gr[N2 + col + 2 * i + 1] << 16);
                }
                gate[u] = make_uint4(a[0], a[1], a[2], a[3]);
                up[u] = make_uint4(b[0], b[1], b[2], b[3]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        uint32_t y[4];
        silu_mul_8(gate[u], up[u], table, y);
        quant_group(y, live[u], row, g0 + u, j, N2, o);
    }
}

// 32 codes (16 bytes) per thread and step -> 32 bf16 values.  e2m1 times a power of two is exact in bf16 except where it
// leaves bf16's range (6 * 2^126 and above becomes infinity).
template <bool VEC>
__global__ void __launch_bounds__(256)
dequant_mxfp4_kernel(const uint8_t* __restrict__ q, int64_t ld_q, const uint8_t* __restrict__ scale, int64_t s_row, uint32_t vecs_per_row, int64_t n_vecs,
                     __nv_bfloat16* __restrict__ out, int64_t ld_out) {
    // one vector = 8 values: 4 bytes of codes, a quarter of a block
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v >= n_vecs) return;
    const int64_t row = v / vecs_per_row;
    const uint32_t c = (uint32_t)(v - row * vecs_per_row);
    uint32_t w;
    const uint8_t* qp = q + row * ld_q + (int64_t)c * 4;
    if (VEC) {
        w = *reinterpret_cast<const uint32_t*>(qp);
    } else {
        w = (uint32_t)qp[0] | ((uint32_t)qp[1] << 8) | ((uint32_t)qp[2] << 16) | ((uint32_t)qp[3] << 24);
    }
    const float s = scale_value(scale[row * s_row + (c >> 2)]);
    uint32_t h[4], r[4];
    unpack_e2m1x8(w, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 p = *reinterpret_cast<const __half2*>(&h[i]);
        r[i] = pack_bf16x2(__low2float(p) * s, __high2float(p) * s);
    }
    uint16_t* op = reinterpret_cast<uint16_t*>(out) + row * ld_out + (int64_t)c * 8;
    if (VEC) {
        *reinterpret_cast<uint4*>(op) = make_uint4(r[0], r[1], r[2], r[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            op[2 * i] = (uint16_t)(r[i] & 0xffffu);
            op[2 * i + 1] = (uint16_t)(r[i] >> 16);
        }
    }
}

// Row-major scale bytes [rows, K/32] -> packed words; bytes of blocks past K and rows past the last one are 2^0.
__global__ void __launch_bounds__(256)
pack_mxfp4_scales_kernel(const uint8_t* __restrict__ scale, int64_t rows, uint32_t kb32, int64_t s_row, uint32_t kblocks, int64_t n_words, uint32_t* __restrict__ packed) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n_words) return;
    // word i belongs to (row block, kb, l, quarter); neighbouring threads take neighbouring words
    const uint32_t in = (uint32_t)(i & 127);
    const int64_t blk = i >> 7;
    const int64_t rb = blk / kblocks;
    const uint32_t kb = (uint32_t)(blk - rb * kblocks);
    const int64_t row = rb * 128 + (in & 3u) * 32 + (in >> 2);
    uint32_t w = 0x7f7f7f7fu;
    if (row < rows) {
        w = 0;
#pragma unroll
        for (uint32_t b = 0; b < 4; ++b) {
            const uint32_t col = kb * 4 + b;
            w |= (col < kb32 ? (uint32_t)scale[row * s_row + col] : 127u) << (8 * b);
        }
    }
    packed[i] = w;
}

static int fill_out(QuantOut& o, const char* who, int64_t M, int64_t K, void* q, int64_t ld_q, void* scale, int64_t s_row, void* sf_packed) {
    KBN_REQUIRE(K % 32 == 0, KBN_ERR_ARG, "%s: K=%lld must be a multiple of 32", who, (long long)K);
    KBN_REQUIRE(q, KBN_ERR_ARG, "%s: null pointer", who);
    KBN_REQUIRE(ld_q >= K / 2 && ld_q % 4 == 0 && (reinterpret_cast<uintptr_t>(q) & 3u) == 0, KBN_ERR_ARG,
                "%s: code rows must start on 4-byte boundaries and hold K/2 bytes", who);
    KBN_REQUIRE(scale || sf_packed, KBN_ERR_ARG, "%s: no place for the scales (row-major or packed)", who);
    KBN_REQUIRE(!scale || s_row >= K / 32, KBN_ERR_ARG, "%s: scale row stride below K/32", who);
    KBN_REQUIRE(!sf_packed || aligned16(sf_packed), KBN_ERR_ARG, "%s: the packed scale buffer must be 16-byte aligned", who);
    KBN_REQUIRE(K < (1ll << 31) && M < (1ll << 31), KBN_ERR_ARG, "%s: M and K must be below 2^31", who);
    o.q = static_cast<uint8_t*>(q);
    o.ld_q = ld_q;
    o.scale = static_cast<uint8_t*>(scale);
    o.s_row = s_row;
    o.packed = static_cast<uint32_t*>(sf_packed);
    o.kblocks = (K + 127) / 128;
    o.word_scales = scale && s_row % 4 == 0 && (reinterpret_cast<uintptr_t>(scale) & 3u) == 0;
    return KBN_OK;
}

}  // namespace mxfp4
}  // namespace kbn

extern "C" int64_t kbn_packed_mxfp4_bytes(int64_t rows, int64_t K) {
    if (rows <= 0 || K <= 0) return 0;
    return (rows + 127) / 128 * ((K + 127) / 128) * 512;
}

extern "C" int kbn_quant_mxfp4(const void* x, int64_t M, int64_t K, int64_t ld_x, void* q, int64_t ld_q, void* scale, int64_t s_row, void* sf_packed,
                               kbn_stream_t stream) {
    using namespace kbn;
    using namespace kbn::mxfp4;
    KBN_REQUIRE(M >= 0 && K >= 0, KBN_ERR_ARG, "kbn_quant_mxfp4: negative size (M=%lld K=%lld)", (long long)M, (long long)K);
    if (M == 0 || K == 0) return KBN_OK;
    KBN_REQUIRE(x && (reinterpret_cast<uintptr_t>(x) & 1u) == 0, KBN_ERR_ARG, "kbn_quant_mxfp4: null or odd pointer");
    KBN_REQUIRE(ld_x >= K || M == 1, KBN_ERR_ARG, "kbn_quant_mxfp4: row stride smaller than K");
    QuantOut o;
    const int rc = fill_out(o, "kbn_quant_mxfp4", M, K, q, ld_q, scale, s_row, sf_packed);
    if (rc != KBN_OK) return rc;
    const auto* xb = static_cast<const __nv_bfloat16*>(x);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    constexpr int U = 4;
    const int64_t G = (K + 127) / 128, cpr = (G + U - 1) / U, n_chunks = M * cpr;
    KBN_REQUIRE(n_chunks < (1ll << 31), KBN_ERR_ARG, "kbn_quant_mxfp4: more than 2^31 groups");
    const unsigned blocks = (unsigned)((n_chunks + 15) / 16);
    if (ld_x % 8 == 0 && aligned16(x))
        quant_mxfp4_kernel<true, U><<<blocks, 256, 0, st>>>(xb, (uint32_t)K, ld_x, o, (uint32_t)G, (uint32_t)cpr, (uint32_t)n_chunks);
    else
        quant_mxfp4_kernel<false, U><<<blocks, 256, 0, st>>>(xb, (uint32_t)K, ld_x, o, (uint32_t)G, (uint32_t)cpr, (uint32_t)n_chunks);
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

extern "C" int kbn_silu_mul_quant_mxfp4(const void* in, int64_t M, int64_t N2, int64_t ld_in, void* q, int64_t ld_q, void* scale, int64_t s_row,
                                        void* sf_packed, kbn_stream_t stream) {
    using namespace kbn;
    using namespace kbn::mxfp4;
    KBN_REQUIRE(M >= 0 && N2 >= 0, KBN_ERR_ARG, "kbn_silu_mul_quant_mxfp4: negative size (M=%lld N2=%lld)", (long long)M, (long long)N2);
    if (M == 0 || N2 == 0) return KBN_OK;
    KBN_REQUIRE(in && (reinterpret_cast<uintptr_t>(in) & 1u) == 0, KBN_ERR_ARG, "kbn_silu_mul_quant_mxfp4: null or odd pointer");
    KBN_REQUIRE(ld_in >= 2 * N2 || M == 1, KBN_ERR_ARG, "kbn_silu_mul_quant_mxfp4: row stride smaller than 2*N2");
    QuantOut o;
    int rc = fill_out(o, "kbn_silu_mul_quant_mxfp4", M, N2, q, ld_q, scale, s_row, sf_packed);
    if (rc != KBN_OK) return rc;
    const uint16_t* table = nullptr;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = silu_table_for_stream(st, &table);
    if (rc != KBN_OK) return rc;
    const auto* xb = static_cast<const __nv_bfloat16*>(in);
    constexpr int U = 2;
    const int64_t G = (N2 + 127) / 128, cpr = (G + U - 1) / U, n_chunks = M * cpr;
    KBN_REQUIRE(n_chunks < (1ll << 31), KBN_ERR_ARG, "kbn_silu_mul_quant_mxfp4: more than 2^31 groups");
    const unsigned blocks = (unsigned)((n_chunks + 15) / 16);
    if (ld_in % 8 == 0 && aligned16(in))
        silu_mul_quant_mxfp4_kernel<true, U><<<blocks, 256, 0, st>>>(xb, (uint32_t)N2, ld_in, o, (uint32_t)G, (uint32_t)cpr, (uint32_t)n_chunks, table);
    else
        silu_mul_quant_mxfp4_kernel<false, U><<<blocks, 256, 0, st>>>(xb, (uint32_t)N2, ld_in, o, (uint32_t)G, (uint32_t)cpr, (uint32_t)n_chunks, table);
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

extern "C" int kbn_dequant_mxfp4(const void* q, int64_t ld_q, const void* scale, int64_t s_row, int64_t M, int64_t K, void* out, int64_t ld_out,
                                 kbn_stream_t stream) {
    using namespace kbn;
    using namespace kbn::mxfp4;
    KBN_REQUIRE(M >= 0 && K >= 0, KBN_ERR_ARG, "kbn_dequant_mxfp4: negative size (M=%lld K=%lld)", (long long)M, (long long)K);
    if (M == 0 || K == 0) return KBN_OK;
    KBN_REQUIRE(q && scale && out && (reinterpret_cast<uintptr_t>(out) & 1u) == 0, KBN_ERR_ARG, "kbn_dequant_mxfp4: null or odd pointer");
    KBN_REQUIRE(K % 32 == 0, KBN_ERR_ARG, "kbn_dequant_mxfp4: K=%lld must be a multiple of 32", (long long)K);
    KBN_REQUIRE(M == 1 || (ld_q >= K / 2 && s_row >= K / 32 && ld_out >= K), KBN_ERR_ARG, "kbn_dequant_mxfp4: a row stride is too small");
    const int64_t n = M * (K / 8);
    KBN_REQUIRE(K < (1ll << 31) && (n + 255) / 256 < (1ll << 31), KBN_ERR_ARG, "kbn_dequant_mxfp4: too many values");
    const bool vec = ld_q % 4 == 0 && (reinterpret_cast<uintptr_t>(q) & 3u) == 0 && ld_out % 8 == 0 && aligned16(out);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned blocks = (unsigned)((n + 255) / 256);
    auto* ob = static_cast<__nv_bfloat16*>(out);
    const auto *qb = static_cast<const uint8_t*>(q), *sb = static_cast<const uint8_t*>(scale);
    if (vec)
        dequant_mxfp4_kernel<true><<<blocks, 256, 0, st>>>(qb, ld_q, sb, s_row, (uint32_t)(K / 8), n, ob, ld_out);
    else
        dequant_mxfp4_kernel<false><<<blocks, 256, 0, st>>>(qb, ld_q, sb, s_row, (uint32_t)(K / 8), n, ob, ld_out);
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

extern "C" int kbn_pack_mxfp4_scales(const void* scale, int64_t rows, int64_t K, int64_t s_row, void* packed, kbn_stream_t stream) {
    using namespace kbn;
    using namespace kbn::mxfp4;
    KBN_REQUIRE(rows >= 0 && K >= 0, KBN_ERR_ARG, "kbn_pack_mxfp4_scales: negative size");
    if (rows == 0 || K == 0) return KBN_OK;
    KBN_REQUIRE(scale && packed && aligned16(packed), KBN_ERR_ARG, "kbn_pack_mxfp4_scales: null pointer, or packed not 16-byte aligned");
    KBN_REQUIRE(K % 32 == 0 && K < (1ll << 31), KBN_ERR_ARG, "kbn_pack_mxfp4_scales: K=%lld must be a multiple of 32", (long long)K);
    KBN_REQUIRE(s_row >= K / 32 || rows == 1, KBN_ERR_ARG, "kbn_pack_mxfp4_scales: row stride below K/32");
    const int64_t words = kbn_packed_mxfp4_bytes(rows, K) / 4;
    KBN_REQUIRE((words + 255) / 256 < (1ll << 31), KBN_ERR_ARG, "kbn_pack_mxfp4_scales: too many scales");
    pack_mxfp4_scales_kernel<<<(unsigned)((words + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(scale), rows, (uint32_t)(K / 32), s_row, (uint32_t)((K + 127) / 128), words, static_cast<uint32_t*>(packed));
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

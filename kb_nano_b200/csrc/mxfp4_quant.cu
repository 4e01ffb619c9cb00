// MXFP4 quantisers and their inverse: bf16 -> e2m1 codes + E8M0 scales (plain and behind SiLU(gate)*up), codes -> bf16,
// and the repacking of row-major scales into the layout of the tensor core.  The 4-bit counterparts of the 1x128 FP8
// quantisers (kb-nano has FP8 only: tasks/baseline/L1/fp8_linear.py:181-215, tasks/baseline/L1/silu_mul_quant_fp8.py:23-76).
//
// All four are HBM-bound: 2 B in and 17/32 B out per element (4 B in with the activation), the inverse the other way round.
// A lane takes 16 consecutive values (one 32-byte access), eight lanes 128 of a row: a block of 32 is two lanes, one shuffle
// gives its largest magnitude, and the four scale bytes of the 128 values meet in one word, which is stored whole, both in
// the row-major scales and in the packed layout.  Measured inside a graph (share of a copy's 6.57 TB/s), 8192 x 7168: quantise 23.7 us (95 %),
// dequantise 24.8 (91 %), activation and quantise (8192 x 2 * 7168 in) 44.4 (91 %); 16384 x 2048: 14.9, 13.6, 27.0; 512 x 7168:
// 3.1, 2.6, 4.9, where the launch is most of it.  With 8 values a lane (16-byte accesses) the first were 33.9 and 34.4; the
// activation took 73 with those and with every gate's SiLU from the table.
#include "mxfp4.cuh"
#include "silu_exact.cuh"

namespace kbn {
namespace mxfp4 {

// All of these are launched with programmatic stream serialisation: resident, as far as there is room, while the kernel in front
// of them ends, and the kernel behind them in its turn.  It is let in only after the wait: a kernel that reads its weights
// before its own wait then still finds what was written two kernels ahead of it.  Calls in a row, against plain launches: quantise
// and back 8192 x 7168 52.2 -> 48.4 us, 1 x 7168 6.7 -> 5.7; SiLU*up, quantise and back 129 x 2048 8.2 -> 6.2.
// What they read may be written while they are already resident: their pointers are not __restrict__ and no load takes the
// read-only path, which the wait does not hold back.
__device__ __forceinline__ void begin_kernel() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Where the results go.  scale and packed may each be null.
struct QuantOut {
    uint8_t* q;
    int64_t ld_q;          // bytes between rows
    uint8_t* scale;        // [M, K/32], row stride s_row
    int64_t s_row;
    uint32_t* packed;
    int64_t kblocks;
    bool word_scales;      // the row-major scales allow 4-byte stores
    bool pair_codes;       // the codes allow 8-byte stores
};

struct Vec16 {             // 16 bf16 values
    uint32_t w[8];
};
__device__ __forceinline__ Vec16 load16(const void* p) {       // 32-byte aligned, read once
    Vec16 v;
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
                 : "l"(p)
                 : "memory");
    return v;
}
__device__ __forceinline__ void store16(void* p, const Vec16& v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]),
                 "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
                 : "memory");
}
// ALIGN: what the rows' start allows, 32, 16 or 2 bytes.
template <int ALIGN>
__device__ __forceinline__ Vec16 load_values(const uint16_t* p) {
    Vec16 v;
    if (ALIGN == 32) {
        v = load16(p);
    } else if (ALIGN == 16) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p)), b = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
        v.w[0] = a.x; v.w[1] = a.y; v.w[2] = a.z; v.w[3] = a.w;
        v.w[4] = b.x; v.w[5] = b.y; v.w[6] = b.z; v.w[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    }
    return v;
}

// The eight lanes of a team hold 16 values each of columns [128 g, 128 g + 128) of `row` (lanes past K hold zeros and
// live == false).  Quantises and stores them; returns the word of the group's four scale bytes, in every lane of the team.
// A value times the block's power of two is exact in bf16 wherever it does not round to code 0 anyway, so the products are
// packed ones.
__device__ __forceinline__ uint32_t quant_group(const Vec16& v, bool live, int64_t row, uint32_t g, uint32_t j, uint32_t K, const QuantOut& o) {
    uint32_t m = v.w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_u16x2(m, v.w[i] & 0x7fff7fffu);
    m = max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const uint32_t b = scale_byte(max(m & 0xffffu, m >> 16));
    // blocks past K count as 2^0, so that nothing read there is a NaN
    uint32_t word = (g * 128u + j * 16u < K ? b : 127u) << (8u * (j >> 1));
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    if (live) {
        uint32_t q[2] = {0, 0};
        if (b != 255u) {
            const uint32_t inv = (uint32_t)(254u - b) * 0x00800080u;      // 2^(127 - b) in both halves
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t s = mul_bf16x2(v.w[i], inv);
                q[i >> 2] |= pack_e2m1x2(bf16_lo(s), bf16_hi(s)) << (8 * (i & 3));
            }
        }
        uint32_t* qp = reinterpret_cast<uint32_t*>(o.q + row * o.ld_q + g * 64u + j * 8u);
        if (o.pair_codes) *reinterpret_cast<uint2*>(qp) = make_uint2(q[0], q[1]);
        else qp[0] = q[0], qp[1] = q[1];
    }
    return word;
}

// The scale words of U consecutive groups g0 .. of one row, stored by lanes 0 .. U - 1 of the team.
template <int U>
__device__ __forceinline__ void store_scales(const uint32_t (&word)[U], bool valid, int64_t row, uint32_t g0, uint32_t j, uint32_t G, uint32_t K, const QuantOut& o) {
    uint32_t w = word[0];
#pragma unroll
    for (int u = 1; u < U; ++u)
        if (j == (uint32_t)u) w = word[u];
    const uint32_t g = g0 + j;
    if (!valid || j >= U || g >= G) return;
    if (o.packed != nullptr) o.packed[packed_word(row, g, o.kblocks)] = w;
    if (o.scale != nullptr) {
        uint8_t* s = o.scale + row * o.s_row + g * 4u;
        if (o.word_scales && g * 128u + 128u <= K) {
            *reinterpret_cast<uint32_t*>(s) = w;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (g * 128u + i * 32u < K) s[i] = (uint8_t)(w >> (8 * i));
        }
    }
}

// U groups of 128 per team, all loads issued before the first use.
template <int ALIGN, int U>
__global__ void __launch_bounds__(256)
quant_mxfp4_kernel(const __nv_bfloat16* x, uint32_t K, int64_t ld_x, QuantOut o, uint32_t G, uint32_t chunks_per_row, uint32_t n_chunks) {
    begin_kernel();
    const uint32_t j = threadIdx.x & 7u;
    const uint32_t chunk = blockIdx.x * 32u + (threadIdx.x >> 3);
    const bool valid = chunk < n_chunks;
    const uint32_t row = valid ? chunk / chunks_per_row : 0u;
    const uint32_t g0 = (chunk - row * chunks_per_row) * U;
    const uint16_t* xr = reinterpret_cast<const uint16_t*>(x) + (int64_t)row * ld_x;
    Vec16 v[U];
    bool live[U];
    uint32_t word[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t col = (g0 + u) * 128u + j * 16u;
        live[u] = valid && g0 + u < G && col < K;
        if (live[u]) v[u] = load_values<ALIGN>(xr + col);
        else v[u] = Vec16{};
    }
#pragma unroll
    for (int u = 0; u < U; ++u) word[u] = quant_group(v[u], live[u], row, g0 + u, j, K, o);
    store_scales<U>(word, valid, row, g0, j, G, K, o);
}

// Eight gates times eight ups -> four packed bf16x2 y = bf16(bf16(silu(g)) * up).  silu(g) is g / (1 + exp(-g)) in fp32 with an
// exactly rounded exponential: the exactly rounded SiLU for gates from -60 on (of an odd subnormal gate, whose half is a tie,
// the even neighbour), -0 below -88.7, where fp32's exponential overflows.  For every finite gate of at least -60 the
// five-instruction approximation lies on the right side of its rounding boundary, so only gates below that come from the
// table.  Every finite gate is tested against the definition, by itself and, beside one below -60, from the table.
__device__ __forceinline__ void silu_mul_exact8(const uint32_t* g, const uint32_t* u, const uint16_t* __restrict__ table, uint32_t* y) {
    const uint32_t gm = min_bf16x2(min_bf16x2(g[0], g[1]), min_bf16x2(g[2], g[3]));
    uint32_t s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = pack_bf16x2(silu_approx(bf16_lo(g[i])), silu_approx(bf16_hi(g[i])));
    if (fminf(bf16_lo(gm), bf16_hi(gm)) < -60.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = silu_table_pair(g[i], table);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = mul_bf16x2(s[i], u[i]);
}

// bf16(bf16(silu(gate)) * up) with the SiLU of the FP8 activation kernel (silu_exact.cuh), then as above.
// The two roundings to bf16 are those of an unfused activation in the model's type, so that fused and unfused layers agree.
template <int ALIGN, int U>
__global__ void __launch_bounds__(256)
silu_mul_quant_mxfp4_kernel(const __nv_bfloat16* in, uint32_t N2, int64_t ld_in, QuantOut o, uint32_t G, uint32_t chunks_per_row,
                            uint32_t n_chunks, const uint16_t* table) {
    begin_kernel();
    const uint32_t j = threadIdx.x & 7u;
    const uint32_t chunk = blockIdx.x * 32u + (threadIdx.x >> 3);
    const bool valid = chunk < n_chunks;
    const uint32_t row = valid ? chunk / chunks_per_row : 0u;
    const uint32_t g0 = (chunk - row * chunks_per_row) * U;
    const uint16_t* gr = reinterpret_cast<const uint16_t*>(in) + (int64_t)row * ld_in;
    Vec16 gate[U], up[U];
    bool live[U];
    uint32_t word[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t col = (g0 + u) * 128u + j * 16u;
        live[u] = valid && g0 + u < G && col < N2;
        gate[u] = up[u] = Vec16{};
        if (live[u]) {
            gate[u] = load_values<ALIGN>(gr + col);
            up[u] = load_values<ALIGN>(gr + N2 + col);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        Vec16 y;
#pragma unroll
        for (int h = 0; h < 2; ++h) silu_mul_exact8(gate[u].w + 4 * h, up[u].w + 4 * h, table, y.w + 4 * h);
        word[u] = quant_group(y, live[u], row, g0 + u, j, N2, o);
    }
    store_scales<U>(word, valid, row, g0, j, G, N2, o);
}

// 16 codes (8 bytes) per thread and vector -> 16 bf16 values.  e2m1 times a power of two is exact in bf16 except where it
// leaves bf16's range (6 * 2^126 and above becomes infinity).  FLAT: everything is contiguous, rows do not matter.
template <bool FLAT, bool VEC, int U>
__global__ void __launch_bounds__(256)
dequant_mxfp4_kernel(const uint8_t* q, int64_t ld_q, const uint8_t* scale, int64_t s_row, uint32_t vecs_per_row, uint32_t n_vecs,
                     __nv_bfloat16* out, int64_t ld_out) {
    begin_kernel();
    uint32_t w[U][2], sb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t v = blockIdx.x * (256u * U) + u * 256u + threadIdx.x;
        w[u][0] = w[u][1] = sb[u] = 0;
        if (v >= n_vecs) continue;
        const uint32_t row = FLAT ? 0u : v / vecs_per_row, c = v - row * vecs_per_row;
        const uint8_t* qp = q + (FLAT ? (int64_t)v * 8 : (int64_t)row * ld_q + (int64_t)c * 8);
        if (VEC) {
            const uint2 p = __ldcs(reinterpret_cast<const uint2*>(qp));
            w[u][0] = p.x; w[u][1] = p.y;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[u][i >> 2] |= (uint32_t)qp[i] << (8 * (i & 3));
        }
        sb[u] = FLAT ? scale[v >> 1] : scale[(int64_t)row * s_row + (c >> 1)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t v = blockIdx.x * (256u * U) + u * 256u + threadIdx.x;
        if (v >= n_vecs) continue;
        const uint32_t row = FLAT ? 0u : v / vecs_per_row, c = v - row * vecs_per_row;
        const float s = scale_value(sb[u]);
        Vec16 r;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t p[4];
            unpack_e2m1x8(w[u][h], p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2 f = *reinterpret_cast<const __half2*>(&p[i]);
                r.w[4 * h + i] = pack_bf16x2(__low2float(f) * s, __high2float(f) * s);
            }
        }
        uint16_t* op = reinterpret_cast<uint16_t*>(out) + (FLAT ? (int64_t)v * 16 : (int64_t)row * ld_out + (int64_t)c * 16);
        if (VEC) {
            store16(op, r);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                op[2 * i] = (uint16_t)(r.w[i] & 0xffffu);
                op[2 * i + 1] = (uint16_t)(r.w[i] >> 16);
            }
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

// What the starts of a bf16 matrix's rows allow: accesses of 32, 16 or 2 bytes.
static int row_alignment(const void* p, int64_t ld, int64_t rows) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | (rows > 1 ? (uintptr_t)(ld * 2) : 0);
    return (bits & 31u) == 0 ? 32 : ((bits & 15u) == 0 ? 16 : 2);
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
    o.pair_codes = ld_q % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
    o.word_scales = scale && s_row % 4 == 0 && (reinterpret_cast<uintptr_t>(scale) & 3u) == 0;
    return KBN_OK;
}

}  // namespace mxfp4
}  // namespace kbn

extern "C" int64_t kbn_packed_mxfp4_bytes(int64_t rows, int64_t K) {
    if (rows <= 0 || K <= 0) return 0;
    return (rows + 127) / 128 * ((K + 127) / 128) * 512;
}

namespace kbn {
namespace mxfp4 {

int quantise(const void* x, int64_t M, int64_t K, int64_t ld_x, void* q, int64_t ld_q, void* scale, int64_t s_row, void* sf_packed, bool behind_gemm, cudaStream_t st) {
    KBN_REQUIRE(M >= 0 && K >= 0, KBN_ERR_ARG, "kbn_quant_mxfp4: negative size (M=%lld K=%lld)", (long long)M, (long long)K);
    if (M == 0 || K == 0) return KBN_OK;
    KBN_REQUIRE(x && (reinterpret_cast<uintptr_t>(x) & 1u) == 0, KBN_ERR_ARG, "kbn_quant_mxfp4: null or odd pointer");
    KBN_REQUIRE(ld_x >= K || M == 1, KBN_ERR_ARG, "kbn_quant_mxfp4: row stride smaller than K");
    QuantOut o;
    const int rc = fill_out(o, "kbn_quant_mxfp4", M, K, q, ld_q, scale, s_row, sf_packed);
    if (rc != KBN_OK) return rc;
    const auto* xb = static_cast<const __nv_bfloat16*>(x);
    const int64_t G = (K + 127) / 128;
    KBN_REQUIRE(M * G < (1ll << 31), KBN_ERR_ARG, "kbn_quant_mxfp4: more than 2^31 groups");
    // Four groups per team where that still gives every SM work; a few rows are spread over more teams.
    const bool many = M * G >= 32 * 4 * (int64_t)sm_count();
    // In a row of linear layers the kernel in front is a GEMM that holds every SM to its end: a large quantiser's blocks, let in
    // early, then crowd the SMs that come free first (with that, 512 x 4096 x 7168 17.8 -> 19.7 us, 8192 x 7168 x 7168 173 -> 179;
    // a small one gains, 77 x 2056 x 1440 10.2 -> 8.7).
    const bool early = !(behind_gemm && many);
    auto go = [&](auto kernel, int U) {
        const int64_t cpr = (G + U - 1) / U, n_chunks = M * cpr;
        const dim3 grid((unsigned)((n_chunks + 31) / 32));
        if (!early) {
            kernel<<<grid, 256, 0, st>>>(xb, (uint32_t)K, ld_x, o, (uint32_t)G, (uint32_t)cpr, (uint32_t)n_chunks);
            return cudaSuccess;
        }
        return launch_pdl(kernel, grid, dim3(256), 0, st, xb, (uint32_t)K, ld_x, o, (uint32_t)G, (uint32_t)cpr, (uint32_t)n_chunks);
    };
    const int align = row_alignment(x, ld_x, M);
    cudaError_t e;
    if (align == 32) e = many ? go(quant_mxfp4_kernel<32, 4>, 4) : go(quant_mxfp4_kernel<32, 1>, 1);
    else if (align == 16) e = many ? go(quant_mxfp4_kernel<16, 4>, 4) : go(quant_mxfp4_kernel<16, 1>, 1);
    else e = go(quant_mxfp4_kernel<2, 1>, 1);
    KBN_CUDA(e);
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

}  // namespace mxfp4
}  // namespace kbn

extern "C" int kbn_quant_mxfp4(const void* x, int64_t M, int64_t K, int64_t ld_x, void* q, int64_t ld_q, void* scale, int64_t s_row, void* sf_packed,
                               kbn_stream_t stream) {
    return kbn::mxfp4::quantise(x, M, K, ld_x, q, ld_q, scale, s_row, sf_packed, false, static_cast<cudaStream_t>(stream));
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
    const int64_t G = (N2 + 127) / 128;
    KBN_REQUIRE(M * G < (1ll << 31), KBN_ERR_ARG, "kbn_silu_mul_quant_mxfp4: more than 2^31 groups");
    auto go = [&](auto kernel, int U) {
        const int64_t cpr = (G + U - 1) / U, n_chunks = M * cpr;
        return launch_pdl(kernel, dim3((unsigned)((n_chunks + 31) / 32)), dim3(256), 0, st, xb, (uint32_t)N2, ld_in, o, (uint32_t)G, (uint32_t)cpr, (uint32_t)n_chunks, table);
    };
    // the up half starts N2 * 2 bytes, a multiple of 64, behind the gate half
    const int align = row_alignment(in, ld_in, M);
    const bool many = M * G >= 32 * 2 * (int64_t)sm_count();
    cudaError_t e;
    if (align == 32) e = many ? go(silu_mul_quant_mxfp4_kernel<32, 2>, 2) : go(silu_mul_quant_mxfp4_kernel<32, 1>, 1);
    else if (align == 16) e = many ? go(silu_mul_quant_mxfp4_kernel<16, 2>, 2) : go(silu_mul_quant_mxfp4_kernel<16, 1>, 1);
    else e = go(silu_mul_quant_mxfp4_kernel<2, 1>, 1);
    KBN_CUDA(e);
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
    const int64_t n = M * (K / 16);
    KBN_REQUIRE(n < (1ll << 31), KBN_ERR_ARG, "kbn_dequant_mxfp4: more than 2^35 values");
    const bool vec = (ld_q % 8 == 0 || M == 1) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && row_alignment(out, ld_out, M) == 32;
    const bool flat = M == 1 || (ld_q == K / 2 && s_row == K / 32 && ld_out == K);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto* ob = static_cast<__nv_bfloat16*>(out);
    const auto *qb = static_cast<const uint8_t*>(q), *sb = static_cast<const uint8_t*>(scale);
    auto go = [&](auto kernel, int U) {
        return launch_pdl(kernel, dim3((unsigned)((n + 256 * U - 1) / (256 * U))), dim3(256), 0, st, qb, ld_q, sb, s_row, (uint32_t)(K / 16), (uint32_t)n, ob, ld_out);
    };
    const bool many = n >= 256 * 4 * (int64_t)sm_count();
    cudaError_t e;
    if (vec && flat) e = many ? go(dequant_mxfp4_kernel<true, true, 4>, 4) : go(dequant_mxfp4_kernel<true, true, 1>, 1);
    else if (vec) e = many ? go(dequant_mxfp4_kernel<false, true, 4>, 4) : go(dequant_mxfp4_kernel<false, true, 1>, 1);
    else e = go(dequant_mxfp4_kernel<false, false, 1>, 1);
    KBN_CUDA(e);
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

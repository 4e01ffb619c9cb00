// The MXFP4 linear layer: bf16 rows in, quantised to MXFP4 on the way, times MXFP4 weights.
//
// At most eight rows (a decode step): one launch.  Every CTA quantises the rows itself -- a few thousand values, under a
// microsecond a row -- into f16 rows in shared memory and streams its share of the weight rows (few_rows.cuh).  The values are
// the ones the quantiser would have stored: the codes, exact in f16, and each block's power of two beside them.
// More rows, or K no multiple of 128: the quantiser and the tensor-core GEMM.
// Measured inside a graph, one row, 4096 x 7168 (15.6 MB, 2.4 us at a copy's rate): 6.5 us (a call among others 6.7), against
// 14.9 for quantiser and GEMM; 7168 x 2048, one to eight rows, 5.3 to 6.5 and 8.4 to 8.5.  Every row adds what its quantisation
// takes in every CTA: 4096 x 7168, four rows, 9.2 us, eight 11.9.
#include <algorithm>

#include "few_rows.cuh"

namespace kbn {
namespace few {

// Rows that leave a shorter ring go through the GEMM.  Weight stream against quantiser and GEMM, with four stages: 8 rows,
// 4096 x 7168 11.9 and 14.2 us, 7 rows, 4096 x 8192 12.4 and 15.2, 16384 x 8192 25.3 and 21.9; with three (measured while a power
// served 128 values): 8 rows, 4096 x 8192 14.1 and 15.5, 16384 x 8192 27.5 and 22.7; with two: 8 rows, 7168 x 9216 24.0 and 17.8.
constexpr int kLinearMinStages = 4;
constexpr int kUnitRows = 2 * kBoxRows<kMxfp4>;
constexpr int kLinearFixed = 1024 + kRedBytes<kMxfp4> + 256 + 128;      // alignment, partial sums, barriers, flag

struct LinearArgs {
    const __nv_bfloat16* x;
    int64_t ld_x;
    const void* sfb;               // packed weight scales
    const __nv_bfloat16* bias;
    __nv_bfloat16* C;
    int64_t ldc;
    int32_t* status;
    int32_t M, N, K, stages, token_stride;
};

// x rows -> MXFP4 codes as f16 (times 2^-kLift, see few_rows.cuh) and their blocks' powers, by all consumer threads.
__device__ __forceinline__ void quantise_tokens(const Smem& s, const LinearArgs& a, bool vec, int tid) {
    constexpr int NT = 32 * kConsumerWarps, BATCH = 4;
    const uint32_t vecs = (uint32_t)a.K / 8u, total = (uint32_t)a.M * vecs;      // four consecutive threads share a block
    const uint32_t row_powers = (uint32_t)power_bytes<kMxfp4>(a.K) / 4u;
    const __half2 lift = __float2half2_rn(1.0f / (1 << Fmt<kMxfp4>::kLift));
    const uint32_t magic = 0xffffffffu / vecs + 1u;      // i / vecs == umulhi(i, magic): i * vecs < 2^32 here
    for (uint32_t i0 = 0; i0 < total; i0 += BATCH * NT) {
        uint32_t w[BATCH][4];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const uint32_t i = i0 + (uint32_t)(k * NT + tid), row = __umulhi(i, magic);
            const uint16_t* p = reinterpret_cast<const uint16_t*>(a.x) + (int64_t)row * a.ld_x + (size_t)(i - row * vecs) * 8;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[k][j] = 0;
            if (i < total) {
                if (vec) {
                    const uint4 u = *reinterpret_cast<const uint4*>(p);
                    w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[k][j] = (uint32_t)p[2 * j] | ((uint32_t)p[2 * j + 1] << 16);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const uint32_t i = i0 + (uint32_t)(k * NT + tid), row = __umulhi(i, magic), v = i - row * vecs;
            if (i0 + (uint32_t)(k * NT) >= total) break;      // whole warps
            uint32_t m = mxfp4::max_u16x2(mxfp4::max_u16x2(w[k][0] & 0x7fff7fffu, w[k][1] & 0x7fff7fffu),
                                          mxfp4::max_u16x2(w[k][2] & 0x7fff7fffu, w[k][3] & 0x7fff7fffu));
            m = mxfp4::max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = mxfp4::max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const uint32_t b = mxfp4::scale_byte(max(m & 0xffffu, m >> 16));
            uint32_t h[4];
            mxfp4::unpack_e2m1x8(mxfp4::quant8(w[k], mxfp4::inv_scale(b), b == 255u), h);
            if (i < total) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&h[j]), lift);
                    h[j] = b == 255u ? 0x7e007e00u : *reinterpret_cast<const uint32_t*>(&r);      // a block with an infinity or a NaN is all NaN
                }
                *reinterpret_cast<uint4*>(s.tokens + (size_t)row * (uint32_t)a.token_stride + (size_t)v * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                if ((tid & 3) == 0) s.token_scales[row * row_powers + v / 4] = mxfp4::scale_value(b);
            }
        }
    }
}

__global__ void __launch_bounds__(kThreads, 1)
mxfp4_linear_few_kernel(const __grid_constant__ CUtensorMap tm, const LinearArgs a, const int vec) {
    extern __shared__ uint8_t raw[];
    Smem s;
    uint8_t* p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    s.ring = p;
    p += (size_t)a.stages * kStageBytes;
    s.scales = p;
    p += (size_t)a.stages * Fmt<kMxfp4>::kScaleBytes;
    s.red = reinterpret_cast<float*>(p);
    p += kRedBytes<kMxfp4>;
    s.bars = reinterpret_cast<uint64_t*>(p);
    p += 256;
    int* abort_flag = reinterpret_cast<int*>(p);
    p += 128;
    s.tokens = p;
    s.token_scales = reinterpret_cast<float*>(p + (size_t)a.M * a.token_stride);
    s.stages = a.stages;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        init_ring(s);
        *abort_flag = 0;
        ptx::prefetch_tensormap(&tm);
    }
    __syncthreads();
    ptx::grid_dependency_wait();
    ptx::launch_dependents();

    const int32_t units = (a.N + kUnitRows - 1) / kUnitRows, KC = a.K / 128;
    const int32_t u0 = (int32_t)((int64_t)units * blockIdx.x / gridDim.x), u1 = (int32_t)((int64_t)units * (blockIdx.x + 1) / gridDim.x);
    if (warp == kProducerWarp) {
        const WaitCtx w{abort_flag, a.status, 17};
        RingPos pos;
        for (int32_t u = u0; u < u1; ++u) produce_unit<kMxfp4, true>(s, pos, &tm, ScaleSource{a.sfb, nullptr}, kUnitRows * u, kUnitRows * u + kUnitRows / 2, a.N, KC, 0, KC, lane, w);
    } else if (warp < kConsumerWarps) {
        const WaitCtx w{abort_flag, a.status, 18};
        OwnPos pos(warp);
        quantise_tokens(s, a, vec != 0, tid);
        consumer_sync();
        const TokenColumns columns = token_columns<kMxfp4>(s, (uint32_t)a.token_stride, KC, a.M, lane, [](int col) { return col; });
        for (int32_t u = u0; u < u1; ++u) {
            float acc[Fmt<kMxfp4>::kTiles][4] = {};
            consume_unit<kMxfp4>(s, pos, KC, warp, lane, columns, acc, w);
            hand_over(s, (uint32_t)(u - u0), warp, lane, acc, w);
        }
    } else {
        const WaitCtx w{abort_flag, a.status, 21};
        for (int32_t u = u0 + warp - kFirstFinisher; u < u1; u += kFinishers) {
            float v[Fmt<kMxfp4>::kTiles][4];
            take_over<kMxfp4>(s, warp - kFirstFinisher, (uint32_t)(u - u0) / kFinishers, lane, v, w);
            const int tok0 = 4 * (lane & 1);
#pragma unroll
            for (int tile = 0; tile < Fmt<kMxfp4>::kTiles; ++tile) {
                const int n = kUnitRows * u + row_of_lane<kMxfp4>(tile, lane);
                if (n >= a.N) continue;
                const float bias = a.bias != nullptr ? __bfloat162float(a.bias[n]) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tok0 + i < a.M) a.C[(int64_t)(tok0 + i) * a.ldc + n] = __float2bfloat16_rn(v[tile][i] + bias);
            }
        }
    }
    if (*abort_flag != 0)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

static int linear_few(const void* x, int64_t ld_x, int64_t M, int64_t K, const void* B, const void* sfb_packed, const void* bias, void* C, int64_t ldc,
                      int64_t N, int stages, cudaStream_t st) {
    LinearArgs a{};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ld_x = ld_x;
    a.sfb = sfb_packed;
    a.bias = static_cast<const __nv_bfloat16*>(bias);
    a.C = static_cast<__nv_bfloat16*>(C);
    a.ldc = ldc;
    a.M = (int32_t)M; a.N = (int32_t)N; a.K = (int32_t)K;
    a.stages = stages;
    a.token_stride = (int32_t)(K * 2 + Fmt<kMxfp4>::kTokenPad);
    int rc = gemm_status_ptr(&a.status);
    if (rc != KBN_OK) return rc;
    CUtensorMap tm;
    rc = weight_map<kMxfp4>(&tm, B, N, K);
    if (rc != KBN_OK) return rc;
    static std::atomic<uint64_t> allowed{0};
    rc = allow_smem(mxfp4_linear_few_kernel, allowed);
    if (rc != KBN_OK) return rc;
    const int64_t units = (N + kUnitRows - 1) / kUnitRows;
    const unsigned grid = (unsigned)std::min<int64_t>(units, sm_count());
    const size_t smem = (size_t)(kLinearFixed + M * (a.token_stride + power_bytes<kMxfp4>(K)) + stages * (kStageBytes + Fmt<kMxfp4>::kScaleBytes));
    const int vec = (ld_x % 8 == 0 || M == 1) && aligned16(x);
    KBN_CUDA(launch_pdl(mxfp4_linear_few_kernel, dim3(grid), dim3(kThreads), smem, st, tm, a, vec));
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

// Whether M rows of na and of nb bf16 values share memory.  Rows that lie side by side in
// one wider matrix (equal strides) do not; with unequal strides the whole extents count.
static bool rows_overlap(const void* a, int64_t ld_a, int64_t na, const void* b, int64_t ld_b, int64_t nb, int64_t M) {
    const int64_t pa = (int64_t)reinterpret_cast<uintptr_t>(a), pb = (int64_t)reinterpret_cast<uintptr_t>(b);
    if (M == 1) ld_a = ld_b = 0;
    if (pa + 2 * (ld_a * (M - 1) + na) <= pb || pb + 2 * (ld_b * (M - 1) + nb) <= pa) return false;
    if (ld_a != ld_b || M == 1) return true;
    const int64_t ld = 2 * ld_a, d = ((pb - pa) % ld + ld) % ld;      // where b's rows start in a's
    return d < 2 * na || d + 2 * nb > ld;
}

}  // namespace few
}  // namespace kbn

extern "C" int kbn_mxfp4_linear(const void* x, int64_t ld_x, int64_t M, int64_t K, void* a_q, void* a_sf, const void* B, const void* sfb_packed,
                                const void* bias, void* C, int64_t ldc, int64_t N, kbn_stream_t stream) {
    using namespace kbn;
    using namespace kbn::few;
    KBN_REQUIRE(M >= 0 && N >= 0 && K > 0, KBN_ERR_ARG, "kbn_mxfp4_linear: bad sizes (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
    if (M == 0 || N == 0) return KBN_OK;
    KBN_REQUIRE(x && a_q && a_sf && B && sfb_packed && C, KBN_ERR_ARG, "kbn_mxfp4_linear: null pointer");
    KBN_REQUIRE(K % 32 == 0, KBN_ERR_ARG, "kbn_mxfp4_linear: K=%lld must be a multiple of 32", (long long)K);
    KBN_REQUIRE(aligned16(B) && aligned16(sfb_packed) && aligned16(a_q) && aligned16(a_sf), KBN_ERR_ARG, "kbn_mxfp4_linear: pointers must be 16-byte aligned");
    KBN_REQUIRE((reinterpret_cast<uintptr_t>(x) & 1u) == 0 && (reinterpret_cast<uintptr_t>(C) & 1u) == 0 && ((ld_x >= K && ldc >= N) || M == 1), KBN_ERR_ARG,
                "kbn_mxfp4_linear: odd pointer or a row stride too small");
    KBN_REQUIRE(aligned_to(bias, 2), KBN_ERR_ARG, "kbn_mxfp4_linear: odd bias pointer");
    // the one-launch form still reads x where it already writes C
    KBN_REQUIRE(!rows_overlap(x, ld_x, K, C, ldc, N, M), KBN_ERR_ARG, "kbn_mxfp4_linear: x and the output overlap");
    // The weight stream serves up to eight rows, as long as their f16 values leave room for the ring.
    if (M <= kMaxGroup && K % 128 == 0 && K < (1ll << 17) && N < (1ll << 27)) {
        const int64_t left = kSmemMax - kLinearFixed - M * (K * 2 + Fmt<kMxfp4>::kTokenPad + power_bytes<kMxfp4>(K));
        const int64_t stages = std::min<int64_t>(left / (kStageBytes + Fmt<kMxfp4>::kScaleBytes), kMaxStages);
        if (stages >= kLinearMinStages) return linear_few(x, ld_x, M, K, B, sfb_packed, bias, C, ldc, N, (int)stages, static_cast<cudaStream_t>(stream));
    }
    const int rc = mxfp4::quantise(x, M, K, ld_x, a_q, K / 2, nullptr, 0, a_sf, true, static_cast<cudaStream_t>(stream));
    if (rc != KBN_OK) return rc;
    return kbn_mxfp4_gemm_nt(a_q, a_sf, B, sfb_packed, bias, C, ldc, M, N, K, stream);
}

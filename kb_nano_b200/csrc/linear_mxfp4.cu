// The MXFP4 linear layer: bf16 rows in, quantised to MXFP4 on the way, times MXFP4 weights.
//
// At most eight rows (a decode step): one launch.  Every CTA quantises the rows itself -- a few thousand values, under a
// microsecond -- into f16 rows in shared memory and streams its share of the weight rows (few_rows.cuh).  The values are
// the ones the quantiser would have stored: a code times 2^(b - b_max), b_max the row's largest scale byte, is exact in f16
// down to 2^-36 of the row's largest block, and the power is taken out after the sum.
// More rows, or K no multiple of 128: the quantiser and the tensor-core GEMM.
#include <algorithm>

#include "few_rows.cuh"

namespace kbn {
namespace few {

constexpr int kRedBytes = kFinishers * kConsumerWarps * 128 * 4;
constexpr int kLinearFixed = 1024 + kRedBytes + 256 + 128;      // alignment, partial sums, barriers, row exponents and flag

struct LinearArgs {
    const __nv_bfloat16* x;
    int64_t ld_x;
    ScaleSource s;
    const __nv_bfloat16* bias;
    __nv_bfloat16* C;
    int64_t ldc;
    int32_t* status;
    int32_t M, N, K, stages, token_stride;
};

// x rows -> MXFP4 values as f16, by all consumer threads; b_max[i]: row i's largest scale byte.  VEC: 16-byte loads.
__device__ __forceinline__ void quantise_tokens(uint8_t* tokens, uint32_t stride, const LinearArgs& a, bool vec, uint32_t* b_max, int tid) {
    const int vecs = a.K / 8, total = a.M * vecs;      // K % 128 == 0: sixteen consecutive threads share a row, four a block
    auto load = [&](int i, uint32_t (&w)[4]) {
        const int row = i / vecs, v = i - row * vecs;
        const uint16_t* p = reinterpret_cast<const uint16_t*>(a.x) + (int64_t)row * a.ld_x + (int64_t)v * 8;
        if (vec) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (uint32_t)p[2 * j] | ((uint32_t)p[2 * j + 1] << 16);
        }
        return row;
    };
    auto block_byte = [&](const uint32_t (&w)[4]) {
        uint32_t m = mxfp4::max_u16x2(mxfp4::max_u16x2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), mxfp4::max_u16x2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
        m = mxfp4::max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = mxfp4::max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
        return mxfp4::scale_byte(max(m & 0xffffu, m >> 16));
    };
    if (tid < a.M) b_max[tid] = 0;
    consumer_sync();
    for (int i0 = 0; i0 < total; i0 += 32 * kConsumerWarps) {
        const int i = i0 + tid;
        uint32_t w[4] = {0, 0, 0, 0};
        const int row = i < total ? load(i, w) : 0;
        const uint32_t b = block_byte(w);
        uint32_t m = b == 255u ? 0u : b;
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
        if ((tid & 15) == 0 && i < total) atomicMax(b_max + row, m);
    }
    consumer_sync();
    for (int i0 = 0; i0 < total; i0 += 32 * kConsumerWarps) {
        const int i = i0 + tid;
        uint32_t w[4] = {0, 0, 0, 0};
        const int row = i < total ? load(i, w) : 0;
        const uint32_t b = block_byte(w);
        uint32_t h[4];
        mxfp4::unpack_e2m1x8(mxfp4::quant8(w, mxfp4::inv_scale(b), b == 255u), h);
        if (i < total) {
            // 2^(b - b_max + 13): the largest code, 6, becomes 49152
            const int e = max((int)b - (int)b_max[row] + 13, -126);
            const float f = b == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(e + 127) << 23);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __half2 c = *reinterpret_cast<const __half2*>(&h[j]);
                const __half2 r = __floats2half2_rn(__low2float(c) * f, __high2float(c) * f);
                h[j] = *reinterpret_cast<const uint32_t*>(&r);
            }
            *reinterpret_cast<uint4*>(tokens + (size_t)row * stride + (size_t)(i - row * vecs) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
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
    p += kRedBytes;
    s.bars = reinterpret_cast<uint64_t*>(p);
    p += 256;
    uint32_t* b_max = reinterpret_cast<uint32_t*>(p);
    int* abort_flag = reinterpret_cast<int*>(p) + kMaxGroup;
    p += 128;
    s.tokens = p;
    s.stages = a.stages;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        init_ring(s, Fmt<kMxfp4>::kArrivals);
        *abort_flag = 0;
        ptx::prefetch_tensormap(&tm);
    }
    __syncthreads();
    ptx::grid_dependency_wait();
    ptx::launch_dependents();

    const int32_t units = (a.N + 15) / 16, KC = a.K / 128;
    const int32_t u0 = (int32_t)((int64_t)units * blockIdx.x / gridDim.x), u1 = (int32_t)((int64_t)units * (blockIdx.x + 1) / gridDim.x);
    if (warp == kProducerWarp) {
        const WaitCtx w{abort_flag, a.status, 17};
        RingPos pos;
        for (int32_t u = u0; u < u1; ++u) produce_unit<kMxfp4>(s, pos, &tm, a.s, 16 * u, 16 * u + 8, a.N, KC, lane, w);
    } else if (warp < kConsumerWarps) {
        const WaitCtx w{abort_flag, a.status, 18};
        RingPos pos;
        quantise_tokens(s.tokens, (uint32_t)a.token_stride, a, vec != 0, b_max, tid);
        consumer_sync();
        const uint32_t token_row = ptx::smem_u32(s.tokens) + (uint32_t)min(lane >> 2, a.M - 1) * (uint32_t)a.token_stride;
        for (int32_t u = u0; u < u1; ++u) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            consume_unit<kMxfp4>(s, pos, KC, warp, lane, token_row, acc, w);
            hand_over(s, u - u0, warp, lane, acc, w);
        }
    } else {
        const WaitCtx w{abort_flag, a.status, 21};
        for (int32_t u = u0 + warp - kFirstFinisher; u < u1; u += kFinishers) {
            float v[4];
            take_over(s, u - u0, lane, v, w);          // the row exponents were there before the first partial sum
            const int n = 16 * u + (lane >> 1), tok0 = 4 * (lane & 1);
            if (n < a.N) {
                const float bias = a.bias != nullptr ? __bfloat162float(a.bias[n]) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tok0 + i < a.M)
                        a.C[(int64_t)(tok0 + i) * a.ldc + n] = __float2bfloat16_rn(scale_pow2(v[i], (int)b_max[tok0 + i] - 127 - 13) + bias);
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
    a.s = ScaleSource{sfb_packed, 1};
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
    KBN_CUDA(cudaFuncSetAttribute(mxfp4_linear_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax));
    const int64_t units = (N + 15) / 16;
    const unsigned grid = (unsigned)std::min<int64_t>(units, sm_count());
    const size_t smem = (size_t)(kLinearFixed + M * a.token_stride + stages * (kStageBytes + Fmt<kMxfp4>::kScaleBytes));
    const int vec = (ld_x % 8 == 0 || M == 1) && aligned16(x);
    KBN_CUDA(launch_pdl(mxfp4_linear_few_kernel, dim3(grid), dim3(kThreads), smem, st, tm, a, vec));
    KBN_CHECK_LAUNCH();
    return KBN_OK;
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
    // The weight stream serves up to eight rows, as long as their f16 values leave room for the ring.
    if (M <= kMaxGroup && K % 128 == 0 && K < (1ll << 24) && N < (1ll << 27)) {
        const int64_t left = kSmemMax - kLinearFixed - M * (K * 2 + Fmt<kMxfp4>::kTokenPad);
        const int64_t stages = std::min<int64_t>(left / (kStageBytes + Fmt<kMxfp4>::kScaleBytes), kMaxStages);
        if (stages >= kMinStages) return linear_few(x, ld_x, M, K, B, sfb_packed, bias, C, ldc, N, (int)stages, static_cast<cudaStream_t>(stream));
    }
    const int rc = kbn_quant_mxfp4(x, M, K, ld_x, a_q, K / 2, nullptr, 0, a_sf, stream);
    if (rc != KBN_OK) return rc;
    return kbn_mxfp4_gemm_nt(a_q, a_sf, B, sfb_packed, bias, C, ldc, M, N, K, stream);
}

// The mixture-of-experts layer behind the router's logits for at most 16 tokens, in two kernels:
//
//   few_gate_up   every CTA routes all tokens (one warp each, moe_route.cuh) and groups the chosen (token, slot) pairs into
//                 jobs of one expert and at most eight tokens; then streams the gate and up rows of the jobs' experts and
//                 writes silu(gate) * up, fp32, for every pair
//   few_down      streams the down rows and adds up each token's rows with the router weights, in slot order, where the
//                 last of an output column block's jobs ends
//
// out[t] = sum_s w[t, s] * W2_e (silu(W1_e x_t) * (W3_e x_t)), e = e[t, s]; kb-nano runs it as routing, permutation, two
// grouped GEMMs, activation and reduction (tasks/baseline/L2/qwen3_moe.py:161-188, tasks/baseline/L2/fused_experts.py:208-283).
// The activations are not quantised here: with a few tokens that saves no bytes (the weights are everything), so the result
// is closer to the real-number one than the W8A8 pipeline's.  Roundings: the tokens and the activated rows to 11 bits
// beside their row's power of two (few_rows.cuh), the result to bf16; everything between is fp32.
//
// Bound: the chosen experts' weights, once.  A CTA's range of units is contiguous over (job, row block), so the tokens of
// a job are loaded into shared memory once or twice per CTA and the ring keeps filling meanwhile.
#include <algorithm>

#include "few_rows.cuh"
#include "moe_route.cuh"

namespace kbn {
namespace few {

// Routing and jobs, in shared memory of every CTA and (written by CTA 0 of the first kernel) in the workspace.
struct Jobs {
    int32_t n_jobs;
    int32_t expert[kMaxPairs];
    int32_t count[kMaxPairs];
    int16_t pair[kMaxPairs][kMaxGroup];
    float weight[kMaxPairs];       // router weight of every pair; NaN for a pair without an expert (NaN logits)
};

struct MoeArgs {
    const __nv_bfloat16* x;
    int64_t ld_x;
    int32_t T, topk, H, I, E, group;
    ScaleSource s13, s2;
    float* y;                      // [pairs, I]
    float* rows;                   // [pairs, H]
    Jobs* jobs;
    int32_t* counters;             // [H / 16], zeroed by the first kernel
    __nv_bfloat16* out;
    int64_t ld_out;
    float* out_w;                  // may be null
    int32_t* out_ids;
    int32_t* status;
    int32_t stages, token_stride;
};

struct Scratch {                   // small shared-memory state beside the ring
    Jobs jobs;
    int32_t id[kMaxPairs];
    int32_t leader[kMaxPairs];
    uint32_t max_bits[kMaxGroup];
    int expo[2][kMaxGroup];        // by the job's parity: a finisher may be a unit or two behind the consumers
    int abort_flag;
};

__host__ __device__ constexpr int scratch_bytes() { return (int)((sizeof(Scratch) + 127) / 128 * 128); }
constexpr int kRedBytes = kFinishers * kConsumerWarps * 128 * 4;
constexpr int kBarBytes = (2 * kMaxStages + 2 * kFinishers) * 8;

template <int FMT>
__device__ __forceinline__ Smem carve(uint8_t* raw, int stages, int group, int token_stride, Scratch** scratch) {
    Smem s;
    uint8_t* p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    s.ring = p;
    p += (size_t)stages * kStageBytes;
    s.scales = p;
    p += (size_t)stages * Fmt<FMT>::kScaleBytes;
    s.red = reinterpret_cast<float*>(p);
    p += kRedBytes;
    *scratch = reinterpret_cast<Scratch*>(p);
    p += scratch_bytes();
    s.bars = reinterpret_cast<uint64_t*>(p);
    p += kBarBytes;
    s.tokens = p;
    s.stages = stages;
    (void)group;
    (void)token_stride;
    return s;
}

// Pairs -> jobs.  A job is up to `group` pairs of one expert, in pair order; jobs are numbered by their first pair.  All
// threads of the block take part (blockDim >= pairs).
__device__ __forceinline__ void build_jobs(Scratch& sc, int pairs, int E, int group, int tid) {
    int before = 0, leader = -1;
    const int e = tid < pairs ? sc.id[tid] : -1;
    const bool valid = e >= 0 && e < E;
    if (valid) {
        for (int q = 0; q < tid; ++q)
            if (sc.id[q] == e) {
                if (before % group == 0) leader = q;
                ++before;
            }
        if (before % group == 0) leader = tid;
    }
    if (tid < pairs) sc.leader[tid] = leader;
    __syncthreads();
    if (valid) {
        int job = 0;
        for (int q = 0; q < leader; ++q) job += sc.leader[q] == q;
        sc.jobs.pair[job][before % group] = (int16_t)tid;
        if (leader == tid) {
            int n = 0;
            for (int q = tid; q < pairs; ++q) n += sc.leader[q] == tid;
            sc.jobs.expert[job] = e;
            sc.jobs.count[job] = n;
        }
    }
    if (tid == 0) {
        int n = 0;
        for (int q = 0; q < pairs; ++q) n += sc.leader[q] == q;
        sc.jobs.n_jobs = n;
    }
    __syncthreads();
}

// A copy that was asked for may still be on its way when a bounded wait has run out: give it time to land before the
// shared memory is given back.
__device__ __forceinline__ void drain_after_abort(const volatile int* abort_flag) {
    if (*abort_flag != 0)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

template <int FMT, int PER>
__global__ void __launch_bounds__(kThreads, 1)
few_gate_up_kernel(const __grid_constant__ CUtensorMap tm, const RouteArgs ra, const int logits_bf16, const MoeArgs a) {
    extern __shared__ uint8_t raw[];
    Scratch* scp;
    const Smem s = carve<FMT>(raw, a.stages, a.group, a.token_stride, &scp);
    Scratch& sc = *scp;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        init_ring(s, Fmt<FMT>::kArrivals);
        sc.abort_flag = 0;
        ptx::prefetch_tensormap(&tm);
    }
    __syncthreads();
    ptx::grid_dependency_wait();          // the logits, the tokens and the weights are final from here on
    ptx::launch_dependents();

    const int pairs = a.T * a.topk;
    if (warp < a.T) {
        float w;
        int id;
        if (logits_bf16) route_token<PER, true>(ra, warp, lane, w, id);
        else route_token<PER, false>(ra, warp, lane, w, id);
        if (lane < a.topk) {
            const bool ok = id >= 0 && id < a.E;
            sc.id[warp * a.topk + lane] = ok ? id : -1;
            sc.jobs.weight[warp * a.topk + lane] = ok ? w : __uint_as_float(0x7fc00000u);
            if (blockIdx.x == 0 && a.out_w != nullptr) {
                a.out_w[warp * a.topk + lane] = w;
                a.out_ids[warp * a.topk + lane] = ok ? id : -1;
            }
        }
    }
    __syncthreads();
    build_jobs(sc, pairs, a.E, a.group, tid);
    if (blockIdx.x == 0) {                // for the second kernel
        const uint32_t* src = reinterpret_cast<const uint32_t*>(&sc.jobs);
        uint32_t* dst = reinterpret_cast<uint32_t*>(a.jobs);
        for (int i = tid; i < (int)(sizeof(Jobs) / 4); i += kThreads) dst[i] = src[i];
        for (int i = tid; i < a.H / 16; i += kThreads) a.counters[i] = 0;
    }

    const int32_t blocks = a.I / 8, KC = a.H / 128;
    const int64_t units = (int64_t)sc.jobs.n_jobs * blocks;
    const int64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
    int32_t job = (int32_t)(u0 / blocks), rb = (int32_t)(u0 - (int64_t)job * blocks);
    if (warp == kProducerWarp) {
        const WaitCtx w{&sc.abort_flag, a.status, 8};
        RingPos pos;
        for (int64_t u = u0; u < u1; ++u) {
            const int32_t row = sc.jobs.expert[job] * 2 * a.I + 8 * rb;
            produce_unit<FMT>(s, pos, &tm, a.s13, row, row + a.I, 2 * a.I * a.E, KC, lane, w);
            if (++rb == blocks) rb = 0, ++job;
        }
    } else if (warp < kConsumerWarps) {
        const WaitCtx w{&sc.abort_flag, a.status, 9};
        RingPos pos;
        int32_t loaded = -1;
        for (int64_t u = u0; u < u1; ++u) {
            const int count = sc.jobs.count[job];
            if (job != loaded) {
                load_tokens<__nv_bfloat16>(s.tokens, (uint32_t)a.token_stride, count, a.H,
                                           [&](int i) { return a.x + (int64_t)(sc.jobs.pair[job][i] / a.topk) * a.ld_x; }, sc.max_bits, sc.expo[job & 1], tid);
                consumer_sync();
                loaded = job;
            }
            // columns without a token compute the last token's again; nothing reads them
            const uint32_t token_row = ptx::smem_u32(s.tokens) + (uint32_t)min(lane >> 2, count - 1) * (uint32_t)a.token_stride;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            consume_unit<FMT>(s, pos, KC, warp, lane, token_row, acc, w);
            hand_over(s, u - u0, warp, lane, acc, w);
            if (++rb == blocks) rb = 0, ++job;
        }
    } else {
        const WaitCtx w{&sc.abort_flag, a.status, 19};
        for (int64_t u = u0; u < u1; ++u) {
            if ((u - u0) % kFinishers == warp - kFirstFinisher) {
                float v[4];
                take_over(s, u - u0, lane, v, w);
                const int count = sc.jobs.count[job], tok0 = 4 * (lane & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float other = __shfl_down_sync(0xffffffffu, v[i], 16);      // rows 8-15 are the up projection's
                    if (lane < 16 && tok0 + i < count) {
                        const int e = sc.expo[job & 1][tok0 + i];
                        const float g = scale_pow2(v[i], e), up = scale_pow2(other, e);
                        a.y[(int64_t)sc.jobs.pair[job][tok0 + i] * a.I + 8 * rb + (lane >> 1)] = __fdiv_rn(g, 1.0f + expf(-g)) * up;
                    }
                }
            }
            if (++rb == blocks) rb = 0, ++job;
        }
    }
    drain_after_abort(&sc.abort_flag);
}

// out[:, 16 rb .. + 15]: each token's rows with their router weights, in slot order, by one warp.
__device__ __forceinline__ void add_up(const MoeArgs& a, const float* weight, int rb, int lane) {
    const int col = 16 * rb + (lane & 15);
    for (int t = lane >> 4; t < a.T; t += 2) {
        float v = 0.f;
        const float* rp = a.rows + (int64_t)t * a.topk * a.H + col;
#pragma unroll 8
        for (int k = 0; k < a.topk; ++k) v = fmaf(weight[t * a.topk + k], __ldcg(rp + (int64_t)k * a.H), v);
        a.out[(int64_t)t * a.ld_out + col] = __float2bfloat16_rn(v);
    }
}

constexpr int kCountBatch = 4;

template <int FMT>
__global__ void __launch_bounds__(kThreads, 1)
few_down_kernel(const __grid_constant__ CUtensorMap tm, const MoeArgs a) {
    extern __shared__ uint8_t raw[];
    Scratch* scp;
    const Smem s = carve<FMT>(raw, a.stages, a.group, a.token_stride, &scp);
    Scratch& sc = *scp;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        init_ring(s, Fmt<FMT>::kArrivals);
        sc.abort_flag = 0;
        ptx::prefetch_tensormap(&tm);
    }
    __syncthreads();
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(a.jobs);
        uint32_t* dst = reinterpret_cast<uint32_t*>(&sc.jobs);
        for (int i = tid; i < (int)(sizeof(Jobs) / 4); i += kThreads) dst[i] = __ldcg(src + i);
    }
    __syncthreads();

    const int32_t blocks = a.H / 16, KC = a.I / 128, n_jobs = sc.jobs.n_jobs;
    if (n_jobs == 0) {                    // no token has an expert: every logit row held a NaN
        for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < (int64_t)a.T * a.H; i += (int64_t)gridDim.x * kThreads)
            a.out[i / a.H * a.ld_out + i % a.H] = __float2bfloat16_rn(__uint_as_float(0x7fc00000u));
        return;
    }
    const int64_t units = (int64_t)n_jobs * blocks;
    const int64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
    int32_t job = (int32_t)(u0 / blocks), rb = (int32_t)(u0 - (int64_t)job * blocks);
    if (warp == kProducerWarp) {
        const WaitCtx w{&sc.abort_flag, a.status, 10};
        RingPos pos;
        for (int64_t u = u0; u < u1; ++u) {
            const int32_t row = sc.jobs.expert[job] * a.H + 16 * rb;
            produce_unit<FMT>(s, pos, &tm, a.s2, row, row + 8, a.H * a.E, KC, lane, w);
            if (++rb == blocks) rb = 0, ++job;
        }
    } else if (warp < kConsumerWarps) {
        const WaitCtx w{&sc.abort_flag, a.status, 11};
        RingPos pos;
        int32_t loaded = -1;
        for (int64_t u = u0; u < u1; ++u) {
            const int count = sc.jobs.count[job];
            if (job != loaded) {
                load_tokens<float>(s.tokens, (uint32_t)a.token_stride, count, a.I,
                                   [&](int i) { return a.y + (int64_t)sc.jobs.pair[job][i] * a.I; }, sc.max_bits, sc.expo[job & 1], tid);
                consumer_sync();
                loaded = job;
            }
            const uint32_t token_row = ptx::smem_u32(s.tokens) + (uint32_t)min(lane >> 2, count - 1) * (uint32_t)a.token_stride;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            consume_unit<FMT>(s, pos, KC, warp, lane, token_row, acc, w);
            hand_over(s, u - u0, warp, lane, acc, w);
            if (++rb == blocks) rb = 0, ++job;
        }
    } else {
        const WaitCtx w{&sc.abort_flag, a.status, 20};
        int pending = 0, mine = 0;            // column blocks stored but not yet counted; lane i holds the i-th
        for (int64_t u = u0; u < u1; ++u) {
            if ((u - u0) % kFinishers == warp - kFirstFinisher) {
                float v[4];
                take_over(s, u - u0, lane, v, w);
                const int count = sc.jobs.count[job], tok0 = 4 * (lane & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tok0 + i < count)
                        a.rows[(int64_t)sc.jobs.pair[job][tok0 + i] * a.H + 16 * rb + (lane >> 1)] = scale_pow2(v[i], sc.expo[job & 1][tok0 + i]);
                if (lane == pending) mine = rb;
                ++pending;
            }
            // One fence and one round of counting for several units.  Who completes a column block (every job once) adds it up.
            if (pending == kCountBatch || (pending > 0 && u + kFinishers >= u1)) {
                __threadfence();
                __syncwarp();
                unsigned last = __ballot_sync(0xffffffffu, lane < pending && atomicAdd(a.counters + mine, 1) == n_jobs - 1);
                if (last) __threadfence();
                for (; last; last &= last - 1) add_up(a, sc.jobs.weight, __shfl_sync(0xffffffffu, mine, __ffs((int)last) - 1), lane);
                pending = 0;
            }
            if (++rb == blocks) rb = 0, ++job;
        }
    }
    drain_after_abort(&sc.abort_flag);
}

// ---- host ----------------------------------------------------------------------------------------

struct Plan {
    int group, stages, token_stride;
    size_t smem;
};

// Largest group of tokens (up to `want`) whose rows of K values leave room for a ring of at least kMinStages.
template <int FMT>
static bool plan(int64_t K, int want, Plan* p) {
    const int64_t stride = K * 2 + Fmt<FMT>::kTokenPad, per_stage = kStageBytes + Fmt<FMT>::kScaleBytes;
    const int64_t fixed = 1024 + kRedBytes + scratch_bytes() + kBarBytes;
    for (int g = std::min(want, kMaxGroup); g >= 1; --g) {
        const int64_t left = kSmemMax - fixed - g * stride;
        if (left < kMinStages * per_stage) continue;
        p->group = g;
        p->token_stride = (int)stride;
        p->stages = (int)std::min<int64_t>(left / per_stage, kMaxStages);
        p->smem = (size_t)(fixed + g * stride + p->stages * per_stage);
        return true;
    }
    return false;
}

template <typename Kernel>
static int allow_smem(Kernel kernel) {
    KBN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax));
    return KBN_OK;
}

struct WorkspaceLayout {
    int64_t jobs, counters, y, rows, total;
};
static WorkspaceLayout workspace_layout(int64_t T, int64_t topk, int64_t H, int64_t I) {
    WorkspaceLayout w;
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    w.jobs = 0;
    w.counters = up((int64_t)sizeof(Jobs));
    w.y = w.counters + up(H / 16 * 4);
    w.rows = w.y + up(T * topk * I * 4);
    w.total = w.rows + up(T * topk * H * 4);
    return w;
}

template <int FMT>
static int run_moe(const void* w13, const void* w2, MoeArgs a, const RouteArgs& ra, int logits_bf16, cudaStream_t st) {
    Plan p1, p2;
    KBN_REQUIRE(plan<FMT>(std::max(a.H, a.I), a.T, &p1), KBN_ERR_UNSUPPORTED,
                "kbn_moe_few_tokens: a row of %d values does not fit the shared memory", std::max(a.H, a.I));
    a.group = p1.group;                    // one grouping for both kernels
    KBN_REQUIRE(plan<FMT>(a.H, a.group, &p1) && plan<FMT>(a.I, a.group, &p2), KBN_ERR_UNSUPPORTED, "kbn_moe_few_tokens: shared memory");
    CUtensorMap t13, t2;
    int rc = weight_map<FMT>(&t13, w13, (int64_t)a.E * 2 * a.I, a.H);
    if (rc != KBN_OK) return rc;
    rc = weight_map<FMT>(&t2, w2, (int64_t)a.E * a.H, a.I);
    if (rc != KBN_OK) return rc;
    rc = gemm_status_ptr(&a.status);
    if (rc != KBN_OK) return rc;
    auto up_kernel = a.E <= 256 ? few_gate_up_kernel<FMT, 8> : few_gate_up_kernel<FMT, 32>;
    rc = allow_smem(up_kernel);
    if (rc != KBN_OK) return rc;
    rc = allow_smem(few_down_kernel<FMT>);
    if (rc != KBN_OK) return rc;
    const unsigned grid = (unsigned)sm_count();
    a.stages = p1.stages;
    a.token_stride = p1.token_stride;
    KBN_CUDA(launch_pdl(up_kernel, dim3(grid), dim3(kThreads), p1.smem, st, t13, ra, logits_bf16, a));
    KBN_CHECK_LAUNCH();
    a.stages = p2.stages;
    a.token_stride = p2.token_stride;
    KBN_CUDA(launch_pdl(few_down_kernel<FMT>, dim3(grid), dim3(kThreads), p2.smem, st, t2, a));
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

}  // namespace few
}  // namespace kbn

extern "C" int64_t kbn_moe_few_tokens_workspace_bytes(int64_t T, int64_t topk, int64_t H, int64_t I) {
    using namespace kbn::few;
    if (T <= 0 || topk <= 0 || H <= 0 || I <= 0 || T > kMaxTokens || topk > kMaxTopk || H >= (1ll << 31) || I >= (1ll << 31)) return 0;
    return workspace_layout(T, topk, H, I).total;
}

extern "C" int kbn_moe_few_tokens(const void* x, int64_t ld_x, int64_t T, const void* logits, int logits_bf16, int64_t ld, int64_t E, int softmax,
                                  const float* bias, int64_t n_group, int64_t topk_group, int64_t topk, int renormalize, float renorm_floor,
                                  float scale, int round_bf16, int weight_format, const void* w13, const void* w13_s, const void* w2,
                                  const void* w2_s, int64_t H, int64_t I, void* out, int64_t ld_out, float* out_w, int32_t* out_ids,
                                  void* workspace, int64_t workspace_bytes, kbn_stream_t stream) {
    using namespace kbn;
    using namespace kbn::few;
    KBN_REQUIRE(T >= 0 && E > 0 && topk > 0 && H > 0 && I > 0, KBN_ERR_ARG, "kbn_moe_few_tokens: bad sizes");
    KBN_REQUIRE(T <= kMaxTokens, KBN_ERR_UNSUPPORTED, "kbn_moe_few_tokens: at most %d tokens (got %lld)", kMaxTokens, (long long)T);
    KBN_REQUIRE(E <= 32 * kRouteMaxPerLane, KBN_ERR_UNSUPPORTED, "kbn_moe_few_tokens: at most %d experts", 32 * kRouteMaxPerLane);
    KBN_REQUIRE(topk <= kMaxTopk && topk <= E, KBN_ERR_ARG, "kbn_moe_few_tokens: topk=%lld must be at most %d and at most E", (long long)topk, kMaxTopk);
    KBN_REQUIRE(H % 128 == 0 && I % 128 == 0, KBN_ERR_ARG, "kbn_moe_few_tokens: H=%lld and I=%lld must be multiples of 128", (long long)H, (long long)I);
    KBN_REQUIRE(weight_format == kFp8 || weight_format == kMxfp4, KBN_ERR_ARG, "kbn_moe_few_tokens: weight_format must be 0 (FP8) or 1 (MXFP4)");
    KBN_REQUIRE(n_group >= 1 && n_group <= 32 && E % n_group == 0 && topk_group >= 1 && topk_group <= n_group, KBN_ERR_ARG,
                "kbn_moe_few_tokens: n_group=%lld must divide E and be at most 32, topk_group=%lld in [1, n_group]", (long long)n_group, (long long)topk_group);
    KBN_REQUIRE(topk <= topk_group * (E / n_group), KBN_ERR_ARG, "kbn_moe_few_tokens: fewer experts in the kept groups than topk");
    if (T == 0) return KBN_OK;
    KBN_REQUIRE(x && logits && w13 && w13_s && w2 && w2_s && out && workspace, KBN_ERR_ARG, "kbn_moe_few_tokens: null pointer");
    KBN_REQUIRE((out_w == nullptr) == (out_ids == nullptr), KBN_ERR_ARG, "kbn_moe_few_tokens: out_w and out_ids come together");
    KBN_REQUIRE((ld_x >= H && ld_out >= H && ld >= E) || T == 1, KBN_ERR_ARG, "kbn_moe_few_tokens: a row stride is too small");
    KBN_REQUIRE(aligned16(x) && (ld_x % 8 == 0 || T == 1), KBN_ERR_ARG, "kbn_moe_few_tokens: rows of x must start on 16-byte boundaries");
    KBN_REQUIRE(aligned16(w13) && aligned16(w2) && (reinterpret_cast<uintptr_t>(w13_s) & 3u) == 0 && (reinterpret_cast<uintptr_t>(w2_s) & 3u) == 0, KBN_ERR_ARG,
                "kbn_moe_few_tokens: weights must be 16-byte aligned, their scales 4-byte aligned");
    KBN_REQUIRE(E * 2 * I < (1ll << 31) && E * H < (1ll << 31), KBN_ERR_UNSUPPORTED, "kbn_moe_few_tokens: more than 2^31 weight rows");
    const WorkspaceLayout wl = workspace_layout(T, topk, H, I);
    KBN_REQUIRE(workspace_bytes >= wl.total && aligned16(workspace), KBN_ERR_ARG, "kbn_moe_few_tokens: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                (long long)wl.total, (long long)workspace_bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    MoeArgs a{};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ld_x = ld_x;
    a.T = (int32_t)T; a.topk = (int32_t)topk; a.H = (int32_t)H; a.I = (int32_t)I; a.E = (int32_t)E;
    a.s13 = ScaleSource{w13_s, 0};
    a.s2 = ScaleSource{w2_s, 0};
    a.jobs = reinterpret_cast<Jobs*>(ws + wl.jobs);
    a.counters = reinterpret_cast<int32_t*>(ws + wl.counters);
    a.y = reinterpret_cast<float*>(ws + wl.y);
    a.rows = reinterpret_cast<float*>(ws + wl.rows);
    a.out = static_cast<__nv_bfloat16*>(out);
    a.ld_out = ld_out;
    a.out_w = out_w;
    a.out_ids = out_ids;
    const RouteArgs ra{logits, ld, (int)E, softmax, bias, (int)n_group, (int)topk_group, (int)topk, renormalize, renorm_floor, scale, round_bf16};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return weight_format == kFp8 ? run_moe<kFp8>(w13, w2, a, ra, logits_bf16, st) : run_moe<kMxfp4>(w13, w2, a, ra, logits_bf16, st);
}

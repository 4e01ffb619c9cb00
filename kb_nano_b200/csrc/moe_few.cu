// The mixture-of-experts layer behind the router's logits for at most 16 tokens, in two kernels:
//
//   few_gate_up   every CTA routes all tokens (one warp each, moe_route.cuh) and groups the chosen (token, slot) pairs into
//                 jobs of one expert and at most eight tokens; then streams the gate and up rows of the jobs' experts and
//                 writes silu(gate) * up, fp32, for every pair
//   few_down      streams the down rows, for at most four tokens at a time (their rows take two columns each, see below), and
//                 adds up each token's rows with the router weights, in slot order, where the last of an output column block's
//                 jobs ends
//
// out[t] = sum_s w[t, s] * W2_e (silu(W1_e x_t) * (W3_e x_t)), e = e[t, s]; kb-nano runs it as routing, permutation, two
// grouped GEMMs, activation and reduction (tasks/baseline/L2/qwen3_moe.py:161-188, tasks/baseline/L2/fused_experts.py:208-283).
// The activations are not quantised here: with a few tokens that saves no bytes (the weights are everything), so the result
// is closer to the real-number one than the W8A8 pipeline's.  Roundings: the activated rows to 22 bits beside a power of two per
// block of 128 or 32 values (few_rows.cuh; the bf16 tokens are exact there), the result to bf16; everything between is fp32.
// 22 bits, in two f16 pieces side by side in the product's columns, and not 11: with 11 the layer's error against 64 bits was 1 %
// above that of fp32 arithmetic.  An expert of more than four tokens then has its down rows streamed twice, by CTAs that run side by
// side, mostly from L2 (I 14336, 8 experts, 16 tokens: MXFP4 228 -> 232 us, FP8 286 -> 299); products of their own for the second
// pieces needed twice the shared memory (300 and 349).
//
// Bound: the chosen experts' weights, once.  A CTA's range of units is contiguous over (job, row block), so the tokens of
// a job are loaded into shared memory once or twice per CTA and the ring keeps filling meanwhile.  What a small call takes
// beyond its bytes is latency: one token, 8 of 128 experts, H 2048, I 768 (38 MB, 5.7 us at a copy's rate) takes 22 to 24 us, of which
// logits, routing and jobs 4, the first stages' way to the first sums 2, the streams themselves 8, the second kernel's start
// behind the first's last block 2, its jobs, tokens and first stages 3, and the last sums' way through finisher, count and
// weighted sum 3.  Both kernels on one SM at a time (shorter rings, the second filling its own under the first) was slower: 78 ->
// 83 us for one token on 8 of 256.
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
    int32_t T, topk, H, I, E, group;      // group: most tokens of a job of the first kernel
    const void *s13, *s2;          // weight scales
    int32_t tiled13, tiled2;       // their loads are tiled (MXFP4, K % 512 == 0)
    float* y;                      // [pairs, I]
    float* rows;                   // [pairs, 2^log_parts, H]
    Jobs* jobs;
    int32_t* counters;             // one per column block of the second kernel, zeroed by the first
    __nv_bfloat16* out;
    int64_t ld_out;
    float* out_w;                  // may be null
    int32_t* out_ids;
    int32_t* status;
    int32_t stages, token_stride, token_rows;
    int32_t log_parts;             // second kernel: parts of K per job
};

constexpr int kMaxExperts = 32 * kRouteMaxPerLane;
struct Scratch {                   // small shared-memory state beside the ring
    Jobs jobs;
    int32_t id[kMaxPairs];
    int16_t taken[kMaxExperts], open_job[kMaxExperts];      // by expert: pairs so far, the job that takes the next one
    int abort_flag;
};

__host__ __device__ constexpr int scratch_bytes() { return (int)((sizeof(Scratch) + 127) / 128 * 128); }
constexpr int kBarBytes = (2 * kMaxStages + 2 * kBuffers) * 8;

template <int FMT>
__device__ __forceinline__ Smem carve(uint8_t* raw, int stages, int rows, int token_stride, Scratch** scratch) {
    Smem s;
    uint8_t* p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    s.ring = p;
    p += (size_t)stages * kStageBytes;
    s.scales = p;
    p += (size_t)stages * Fmt<FMT>::kScaleBytes;
    s.red = reinterpret_cast<float*>(p);
    p += kRedBytes<FMT>;
    *scratch = reinterpret_cast<Scratch*>(p);
    p += scratch_bytes();
    s.bars = reinterpret_cast<uint64_t*>(p);
    p += kBarBytes;
    s.tokens = p;
    s.token_scales = reinterpret_cast<float*>(p + (size_t)rows * token_stride);
    s.stages = stages;
    return s;
}

// Pairs -> jobs, by one warp.  A job is up to `group` pairs of one expert, in pair order; jobs are numbered by their first
// pair.  sc.taken is all zero.  One step per token: its experts are distinct, as a rule; where one occurs twice (equal
// choices of a router that has run out of experts) the later slot waits for a step of its own.
__device__ __forceinline__ void build_jobs(Scratch& sc, int T, int topk, int group, int lane) {
    int n = 0;
    for (int t = 0; t < T; ++t) {
        const int p = t * topk + lane;
        const int e = lane < topk ? sc.id[p] : -1;
        unsigned todo = __ballot_sync(0xffffffffu, e >= 0);
        const unsigned same = __match_any_sync(0xffffffffu, e);
        while (todo) {
            const bool now = ((todo >> lane) & 1u) && __ffs((int)(same & todo)) - 1 == lane;
            const int k = now ? sc.taken[e] : 1;
            const bool opens = now && k == 0;
            const unsigned opening = __ballot_sync(0xffffffffu, opens);
            if (now) {
                const int job = opens ? n + __popc(opening & ((1u << lane) - 1u)) : sc.open_job[e];
                if (opens) {
                    sc.open_job[e] = (int16_t)job;
                    sc.jobs.expert[job] = e;
                }
                sc.jobs.pair[job][k] = (int16_t)p;
                sc.jobs.count[job] = k + 1;
                sc.taken[e] = (int16_t)(k + 1 == group ? 0 : k + 1);
            }
            n += __popc(opening);
            todo &= ~__ballot_sync(0xffffffffu, now);
            __syncwarp();
        }
    }
    if (lane == 0) sc.jobs.n_jobs = n;
    __syncwarp();
}
constexpr int kJobsBarrier = 3;

// The second kernel's jobs, by one warp: those of more than kPieceGroup tokens in two halves.
__device__ __forceinline__ void write_down_jobs(const Jobs& jobs, Jobs* out, int lane) {
    static_assert(kMaxGroup <= 2 * kPieceGroup, "a job has two halves at most");
    const unsigned before = (1u << lane) - 1u;
    int n = 0;
    for (int base = 0; base < jobs.n_jobs; base += 32) {
        const int job = base + lane, count = job < jobs.n_jobs ? jobs.count[job] : 0;
        const unsigned any = __ballot_sync(0xffffffffu, count > 0), split = __ballot_sync(0xffffffffu, count > kPieceGroup);
        const int at = n + __popc(any & before) + __popc(split & before), first = count > kPieceGroup ? (count + 1) / 2 : count;
        for (int k = 0; k < count; ++k) out->pair[k < first ? at : at + 1][k < first ? k : k - first] = jobs.pair[job][k];
        if (count > 0) {
            out->expert[at] = jobs.expert[job];
            out->count[at] = first;
        }
        if (count > first) {
            out->expert[at + 1] = jobs.expert[job];
            out->count[at + 1] = count - first;
        }
        n += __popc(any) + __popc(split);
    }
    if (lane == 0) out->n_jobs = n;
}

// A copy that was asked for may still be on its way when a bounded wait has run out: give it time to land before the
// shared memory is given back.
__device__ __forceinline__ void drain_after_abort(const volatile int* abort_flag) {
    if (*abort_flag != 0)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

template <int FMT, int PER>
__global__ void __launch_bounds__(kThreads, 1)
few_gate_up_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tm_scales, const RouteArgs ra, const int logits_bf16, const MoeArgs a) {
    extern __shared__ uint8_t raw[];
    Scratch* scp;
    const Smem s = carve<FMT>(raw, a.stages, a.token_rows, a.token_stride, &scp);
    Scratch& sc = *scp;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        init_ring(s);
        sc.abort_flag = 0;
        ptx::prefetch_tensormap(&tm);
    }
    for (int i = tid; i < a.E; i += kThreads) sc.taken[i] = 0;
    __syncthreads();
    ptx::grid_dependency_wait();          // the logits, the tokens and the weights are final from here on
    ptx::launch_dependents();

    // Where all tokens fit they stay in shared memory for every job; with at most eight, half of the consumers fetch them
    // while the other half routes.
    const bool resident = a.T <= a.token_rows;
    const bool at_once = resident && a.T <= kConsumerWarps / 2;
    const int router = at_once ? warp - kConsumerWarps / 2 : warp;
    auto token = [&](int i) { return a.x + (int64_t)i * a.ld_x; };
    if (warp < kConsumerWarps && router >= 0 && router < a.T) {
        float logit[PER], w;
        int id;
        load_logits<PER>(ra, logits_bf16 != 0, router, lane, logit);
        route_logits<PER>(ra, lane, logit, w, id);
        if (lane < a.topk) {
            const bool ok = id >= 0 && id < a.E;
            sc.id[router * a.topk + lane] = ok ? id : -1;
            sc.jobs.weight[router * a.topk + lane] = ok ? w : __uint_as_float(0x7fc00000u);
            if (blockIdx.x == 0 && a.out_w != nullptr) {
                a.out_w[router * a.topk + lane] = w;
                a.out_ids[router * a.topk + lane] = ok ? id : -1;
            }
        }
    }
    if (at_once && warp < kConsumerWarps / 2) load_tokens<FMT, __nv_bfloat16, 16 * kConsumerWarps>(s, (uint32_t)a.token_stride, a.T, a.H, token, tid);
    __syncthreads();
    // The producer groups the pairs and starts on the weights at once; the others join as soon as the jobs are there.
    if (warp == kProducerWarp) {
        build_jobs(sc, a.T, a.topk, a.group, lane);
        asm volatile("bar.arrive %0, %1;" ::"n"(kJobsBarrier), "n"(kThreads) : "memory");
    } else {
        if (resident && !at_once && warp < kConsumerWarps) load_tokens<FMT, __nv_bfloat16, 32 * kConsumerWarps>(s, (uint32_t)a.token_stride, a.T, a.H, token, tid);
        asm volatile("bar.sync %0, %1;" ::"n"(kJobsBarrier), "n"(kThreads) : "memory");
        if (blockIdx.x == 0) {            // for the second kernel
            const int i0 = tid - (warp > kProducerWarp ? 32 : 0);      // the producer is not here
            for (int i = i0; i < a.T * a.topk; i += kThreads - 32) a.jobs->weight[i] = sc.jobs.weight[i];
            for (int i = i0; i < a.H / (2 * kBoxRows<FMT>); i += kThreads - 32) a.counters[i] = 0;
            if (warp == kFirstFinisher) write_down_jobs(sc.jobs, a.jobs, lane);
        }
    }

    constexpr int kRows = kBoxRows<FMT>;      // gate rows, and as many up rows, of a unit
    const int32_t blocks = a.I / kRows, KC = a.H / 128;
    const int64_t units = (int64_t)sc.jobs.n_jobs * blocks;      // below 2^31: at most 16 E jobs, E * 2 I rows below 2^31
    const int32_t u0 = (int32_t)(units * blockIdx.x / gridDim.x), u1 = (int32_t)(units * (blockIdx.x + 1) / gridDim.x);
    int32_t job = u0 / blocks, rb = u0 - job * blocks;
    if (warp == kProducerWarp) {
        const WaitCtx w{&sc.abort_flag, a.status, 8};
        RingPos pos;
        for (int32_t u = u0; u < u1; ++u) {
            const int32_t row = sc.jobs.expert[job] * 2 * a.I + kRows * rb;
            produce_unit<FMT>(s, pos, &tm, ScaleSource{a.s13, a.tiled13 ? &tm_scales : nullptr}, row, row + a.I, 2 * a.I * a.E, KC, 0, KC, lane, w);
            if (++rb == blocks) rb = 0, ++job;
        }
    } else if (warp < kConsumerWarps) {
        const WaitCtx w{&sc.abort_flag, a.status, 9};
        OwnPos pos(warp);
        int32_t loaded = -1;
        TokenColumns columns{};
        for (int32_t u = u0; u < u1; ++u) {
            const int count = sc.jobs.count[job];
            if (job != loaded) {
                if (!resident) {
                    consumer_sync();          // everybody is done with the last job's tokens
                    load_tokens<FMT, __nv_bfloat16, 32 * kConsumerWarps>(s, (uint32_t)a.token_stride, count, a.H,
                                                                    [&](int i) { return token(sc.jobs.pair[job][i] / a.topk); }, tid);
                    consumer_sync();
                }
                loaded = job;
                columns = token_columns<FMT>(s, (uint32_t)a.token_stride, KC, count, lane, [&](int col) { return resident ? sc.jobs.pair[job][col] / a.topk : col; });
            }
            float acc[Fmt<FMT>::kTiles][4] = {};
            consume_unit<FMT>(s, pos, KC, warp, lane, columns, acc, w);
            hand_over(s, (uint32_t)(u - u0), warp, lane, acc, w);
            if (++rb == blocks) rb = 0, ++job;
        }
    } else {
        const WaitCtx w{&sc.abort_flag, a.status, 19};
        for (int32_t u = u0; u < u1; ++u) {
            if ((u - u0) % kFinishers == warp - kFirstFinisher) {
                float v[Fmt<FMT>::kTiles][4];
                take_over<FMT>(s, warp - kFirstFinisher, (uint32_t)(u - u0) / kFinishers, lane, v, w);
                const int count = sc.jobs.count[job], tok0 = 4 * (lane & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int tile = 0; tile < Fmt<FMT>::kTiles; ++tile) {
                        const float gate = v[tile][i], up = __shfl_down_sync(0xffffffffu, gate, 16);      // box 1 is the up projection's
                        if (lane < 16 && tok0 + i < count)
                            a.y[(int64_t)sc.jobs.pair[job][tok0 + i] * a.I + kRows * rb + row_of_lane<FMT>(tile, lane)] = __fdiv_rn(gate, 1.0f + expf(-gate)) * up;
                    }
            }
            if (++rb == blocks) rb = 0, ++job;
        }
    }
    drain_after_abort(&sc.abort_flag);
}

// COLS output columns of every token: its rows with their router weights, in slot order, by one warp.  Two columns a lane,
// so that several tokens' rows are under way at once: this is the last thing a block does, and round trips to L2 count.
template <int COLS>
__device__ __forceinline__ void add_up(const MoeArgs& a, int log_parts, const float* weight, int rb, int lane) {
    const int col = COLS * rb + 2 * (lane % (COLS / 2));
    const int n = a.topk << log_parts;
    for (int t = lane / (COLS / 2); t < a.T; t += 64 / COLS) {
        float2 v = make_float2(0.f, 0.f);
        const float2* rp = reinterpret_cast<const float2*>(a.rows + (int64_t)t * n * a.H + col);
#pragma unroll 8
        for (int k = 0; k < n; ++k) {
            const float2 r = __ldcg(rp + (int64_t)k * (a.H / 2));
            const float wk = weight[t * a.topk + (k >> log_parts)];
            v.x = fmaf(wk, r.x, v.x);
            v.y = fmaf(wk, r.y, v.y);
        }
        __nv_bfloat16* o = a.out + (int64_t)t * a.ld_out + col;
        o[0] = __float2bfloat16_rn(v.x);
        o[1] = __float2bfloat16_rn(v.y);
    }
}

constexpr int kCountBatch = 4;
__device__ __forceinline__ int add_acq_rel_gpu(int32_t* p) {
    int old;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
    return old;
}

// kWhole: a unit is the whole K.  kHalves: a unit is a single stage, see few_rows.cuh.  kParts: K in parts.
enum DownMode : int { kWhole, kHalves, kParts };
template <int FMT, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
few_down_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tm_scales, const MoeArgs a) {
    extern __shared__ uint8_t raw[];
    constexpr bool HALVES = MODE == kHalves;
    Scratch* scp;
    const Smem s = carve<FMT>(raw, a.stages, a.token_rows, a.token_stride, &scp);
    Scratch& sc = *scp;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        init_ring<HALVES>(s);
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

    constexpr int kRows = 2 * kBoxRows<FMT>;      // output columns of a unit
    const int32_t blocks = a.H / kRows, KC = a.I / 128, n_jobs = sc.jobs.n_jobs;
    if (n_jobs == 0) {                    // no token has an expert: every logit row held a NaN
        for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < (int64_t)a.T * a.H; i += (int64_t)gridDim.x * kThreads)
            a.out[i / a.H * a.ld_out + i % a.H] = __float2bfloat16_rn(__uint_as_float(0x7fc00000u));
        return;
    }
    // A job's K is worked on in parts of whole stages; vj = (job << log_parts) + part.
    const int32_t lp = MODE == kParts ? a.log_parts : 0, n_parts = n_jobs << lp, k_stages = (KC + kChunks - 1) / kChunks;
    auto first_chunk = [&](int32_t part) { return min(KC, (k_stages * part >> lp) * kChunks); };
    const int64_t units = (int64_t)n_parts * blocks;      // below 2^31: each has 64 bytes of workspace or more
    const int32_t u0 = (int32_t)(units * blockIdx.x / gridDim.x), u1 = (int32_t)(units * (blockIdx.x + 1) / gridDim.x);
    int32_t vj = u0 / blocks, rb = u0 - vj * blocks;
    if (warp == kProducerWarp) {
        const WaitCtx w{&sc.abort_flag, a.status, 10};
        RingPos pos;
        for (int32_t u = u0; u < u1; ++u) {
            const int32_t row = sc.jobs.expert[vj >> lp] * a.H + kRows * rb, part = vj & ((1 << lp) - 1);
            produce_unit<FMT>(s, pos, &tm, ScaleSource{a.s2, a.tiled2 ? &tm_scales : nullptr}, row, row + kRows / 2, a.H * a.E, KC, first_chunk(part), first_chunk(part + 1), lane, w);
            if (++rb == blocks) rb = 0, ++vj;
        }
    } else if (warp < kConsumerWarps) {
        const WaitCtx w{&sc.abort_flag, a.status, 11};
        OwnPos pos(warp);
        int32_t loaded = -1, kc = 0;
        uint32_t handed = 0;
        TokenColumns columns{};
        for (int32_t u = u0; u < u1; ++u) {
            if (vj != loaded) {
                const int job = vj >> lp, part = vj & ((1 << lp) - 1), count = sc.jobs.count[job];
                const int32_t c0 = first_chunk(part);
                kc = first_chunk(part + 1) - c0;
                consumer_sync();
                load_tokens<FMT, float, 32 * kConsumerWarps>(s, (uint32_t)a.token_stride, count, 128 * kc,
                                                        [&](int i) { return a.y + (int64_t)sc.jobs.pair[job][i] * a.I + 128 * c0; }, tid);
                consumer_sync();
                loaded = vj;
                columns = piece_columns<FMT>(s, (uint32_t)a.token_stride, kc, count, lane);
            }
            float acc[Fmt<FMT>::kTiles][4] = {};
            const bool part = !HALVES || pos.ahead == 0;      // a unit is one stage
            consume_unit<FMT>(s, pos, kc, warp, lane, columns, acc, w);
            if (part) hand_over<HALVES>(s, handed++, warp, lane, acc, w);
            if (++rb == blocks) rb = 0, ++vj;
        }
    } else {
        const WaitCtx w{&sc.abort_flag, a.status, 20};
        const int finisher = warp - kFirstFinisher;
        uint32_t taken = 0;
        RingPos pos;
        int pending = 0, mine = 0;            // column blocks stored but not yet counted; lane i holds the i-th
        for (int32_t u = u0; u < u1; ++u) {
            if ((HALVES ? half_of(pos) : (int)((u - u0) % kFinishers)) == finisher) {
                float v[Fmt<FMT>::kTiles][4];
                take_over<FMT, HALVES>(s, finisher, taken++, lane, v, w);
                const int job = vj >> lp, part = vj & ((1 << lp) - 1), count = sc.jobs.count[job];
#pragma unroll
                for (int tile = 0; tile < Fmt<FMT>::kTiles; ++tile)
#pragma unroll
                    for (int i = 0; i < kPieceGroup; ++i) v[tile][i] += __shfl_down_sync(0xffffffffu, v[tile][i], 1);      // the odd lanes hold the second pieces' sums
#pragma unroll
                for (int i = 0; i < kPieceGroup; ++i)
#pragma unroll
                    for (int tile = 0; tile < Fmt<FMT>::kTiles; ++tile)
                        if ((lane & 1) == 0 && i < count) a.rows[(((int64_t)sc.jobs.pair[job][i] << lp) + part) * a.H + kRows * rb + row_of_lane<FMT>(tile, lane)] = v[tile][i];
                if (lane == pending) mine = rb;
                ++pending;
            }
            // One round of counting for several units; the release half of the atomic publishes the warp's rows, its acquire
            // half makes the others' visible.  Who completes a column block (every job once) adds it up.
            if (pending == kCountBatch || (pending > 0 && u + (HALVES ? 1 : kFinishers) >= u1)) {
                __syncwarp();
                int before = -1;
                if (lane < pending) before = add_acq_rel_gpu(a.counters + mine);
                unsigned last = __ballot_sync(0xffffffffu, before == n_parts - 1);
                __syncwarp();
                for (; last; last &= last - 1) add_up<kRows>(a, lp, sc.jobs.weight, __shfl_sync(0xffffffffu, mine, __ffs((int)last) - 1), lane);
                pending = 0;
            }
            if (HALVES) pos.advance((uint32_t)s.stages);      // a stage per unit
            if (++rb == blocks) rb = 0, ++vj;
        }
    }
    drain_after_abort(&sc.abort_flag);
}

// ---- host ----------------------------------------------------------------------------------------

struct Plan {
    int rows, stages, token_stride;
    size_t smem;
};

template <int FMT>
static int64_t row_bytes(int64_t K, int pieces) {      // of a token with its powers; the second kernel's in two pieces
    return pieces * (K * 2 + Fmt<FMT>::kTokenPad) + power_bytes<FMT>(K);
}
template <int FMT>
static int64_t fixed_bytes() {
    return 1024 + kRedBytes<FMT> + scratch_bytes() + kBarBytes;
}

// As many tokens of K values (with their powers), up to `want`, as leave room for a ring of at least kMinStages; a single token
// whose row does not, at least three.
template <int FMT>
static bool plan(int64_t K, int want, int pieces, Plan* p) {
    const int64_t row = row_bytes<FMT>(K, pieces), per_stage = kStageBytes + Fmt<FMT>::kScaleBytes, fixed = fixed_bytes<FMT>();
    for (int g = want; g >= 1; --g) {
        const int64_t left = kSmemMax - fixed - g * row;
        if (left < kMinStages * per_stage && (g > 1 || left < 3 * per_stage)) continue;
        p->rows = g;
        p->token_stride = (int)(K * 2 + Fmt<FMT>::kTokenPad);
        p->stages = (int)std::min<int64_t>(left / per_stage, kMaxStages);
        p->smem = (size_t)(fixed + g * row + p->stages * per_stage);
        return true;
    }
    return false;
}

// Parts of K per job of the second kernel, as a power of two, and the longest part's length.  The rows of a job's tokens
// share the shared memory with the ring.  So: one part if that leaves a ring beside a full job, else the fewest parts, of three
// stages or more, that leave a ring of seven, else the fewest, of a stage or more, that leave a ring.  8 experts, two / four / eight
// parts (whole rows do not fit): I 14336, MXFP4, 5 tokens - / 157 / 173 us, 16 tokens - / 232 / 253; FP8, 5 tokens 207 / 208 / 225, 16
// tokens 306 / 299 / 331; I 7168, MXFP4, 5 tokens 96 / 93 / 112, where the rule takes two.  Where a full job fits whole, parts cost:
// I 6144, FP8, 5 tokens 100 / 106 with two.
template <int FMT>
static int log_parts(int64_t T, int64_t I, int64_t* longest) {
    const int64_t S = (I / 128 + kChunks - 1) / kChunks;
    for (int lp = 0;; ++lp) {
        *longest = std::min(I, ((S + ((int64_t)1 << lp) - 1) >> lp) * kChunks * 128);
        const int64_t ring = (kSmemMax - fixed_bytes<FMT>() - std::min<int64_t>(T, kPieceGroup) * row_bytes<FMT>(*longest, 2)) / (kStageBytes + Fmt<FMT>::kScaleBytes);
        const int64_t shorter = S >> (lp + 1);      // stages of a part with twice as many
        if (ring >= (lp == 0 ? kMinStages : 7) || shorter < 1 || (shorter < 3 && ring >= kMinStages)) return lp;
    }
}

struct WorkspaceLayout {
    int64_t jobs, counters, y, rows, total;
};
static WorkspaceLayout workspace_layout(int64_t T, int64_t topk, int64_t H, int64_t I) {
    WorkspaceLayout w;
    int64_t longest;
    const int parts = std::max(log_parts<kFp8>(T, I, &longest), log_parts<kMxfp4>(T, I, &longest));      // whichever the weights are
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    w.jobs = 0;
    w.counters = up((int64_t)sizeof(Jobs));
    w.y = w.counters + up(H / 16 * 4);
    w.rows = w.y + up(T * topk * I * 4);
    w.total = w.rows + up((T * topk * H * 4) << parts);
    return w;
}

template <int FMT>
static int run_moe(const void* w13, const void* w2, MoeArgs a, const RouteArgs& ra, int logits_bf16, cudaStream_t st) {
    // The first kernel keeps all tokens in shared memory if it can, else those of one job at a time.
    Plan p1, p2;
    int64_t longest;
    a.log_parts = log_parts<FMT>(a.T, a.I, &longest);
    KBN_REQUIRE(plan<FMT>(a.H, a.T, 1, &p1) && plan<FMT>(longest, std::min(a.T, kPieceGroup), 2, &p2), KBN_ERR_UNSUPPORTED,
                "kbn_moe_few_tokens: a row of %d values does not fit the shared memory", std::max(a.H, a.I));
    KBN_REQUIRE(p2.rows == std::min(a.T, kPieceGroup), KBN_ERR_UNSUPPORTED, "kbn_moe_few_tokens: shared memory");
    a.group = std::min(p1.rows, kMaxGroup);
    if (p1.rows < a.T) plan<FMT>(a.H, a.group, 1, &p1);
    CUtensorMap t13, t2;
    int rc = weight_map<FMT>(&t13, w13, (int64_t)a.E * 2 * a.I, a.H);
    if (rc != KBN_OK) return rc;
    rc = weight_map<FMT>(&t2, w2, (int64_t)a.E * a.H, a.I);
    if (rc != KBN_OK) return rc;
    // FP8: never read; the kernels take a map all the same
    CUtensorMap t13s = t13, t2s = t2;
    a.tiled13 = FMT == kMxfp4 && a.H % 512 == 0 && aligned16(a.s13);
    a.tiled2 = FMT == kMxfp4 && a.I % 512 == 0 && aligned16(a.s2);
    if (a.tiled13 && (rc = scale_rows_map(&t13s, a.s13, (int64_t)a.E * 2 * a.I, a.H)) != KBN_OK) return rc;
    if (a.tiled2 && (rc = scale_rows_map(&t2s, a.s2, (int64_t)a.E * a.H, a.I)) != KBN_OK) return rc;
    rc = gemm_status_ptr(&a.status);
    if (rc != KBN_OK) return rc;
    auto up_kernel = a.E <= 256 ? few_gate_up_kernel<FMT, 8> : few_gate_up_kernel<FMT, 32>;
    static std::atomic<uint64_t> up_small{0}, up_large{0}, down{0}, down_halves{0}, down_parts{0};
    rc = allow_smem(up_kernel, a.E <= 256 ? up_small : up_large);
    if (rc != KBN_OK) return rc;
    // one token, 8 of 128 experts, H 2048, I 768: 24.6 us without halves, 23.5 with them; four tokens, I 1024: 81.3 and 80.3
    const bool halves = a.I <= 128 * kChunks;
    auto down_kernel = halves ? few_down_kernel<FMT, kHalves> : (a.log_parts > 0 ? few_down_kernel<FMT, kParts> : few_down_kernel<FMT, kWhole>);
    rc = allow_smem(down_kernel, halves ? down_halves : (a.log_parts > 0 ? down_parts : down));
    if (rc != KBN_OK) return rc;
    const unsigned grid = (unsigned)sm_count();
    a.stages = p1.stages;
    a.token_rows = p1.rows;
    a.token_stride = p1.token_stride;
    KBN_CUDA(launch_pdl(up_kernel, dim3(grid), dim3(kThreads), p1.smem, st, t13, t13s, ra, logits_bf16, a));
    KBN_CHECK_LAUNCH();
    a.stages = p2.stages;
    a.token_rows = 2 * p2.rows;
    a.token_stride = p2.token_stride;
    KBN_CUDA(launch_pdl(down_kernel, dim3(grid), dim3(kThreads), p2.smem, st, t2, t2s, a));
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
    KBN_REQUIRE(aligned_to(logits, logits_bf16 ? 2 : 4) && aligned_to(bias, 4) && aligned_to(out, 2) && aligned_to(out_w, 4) && aligned_to(out_ids, 4), KBN_ERR_ARG,
                "kbn_moe_few_tokens: logits, bias, out, out_w and out_ids must be aligned to their elements");
    KBN_REQUIRE(E * 2 * I < (1ll << 31) && E * H < (1ll << 31), KBN_ERR_UNSUPPORTED, "kbn_moe_few_tokens: more than 2^31 weight rows");
    const WorkspaceLayout wl = workspace_layout(T, topk, H, I);
    KBN_REQUIRE(workspace_bytes >= wl.total && aligned16(workspace), KBN_ERR_ARG, "kbn_moe_few_tokens: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                (long long)wl.total, (long long)workspace_bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    MoeArgs a{};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ld_x = ld_x;
    a.T = (int32_t)T; a.topk = (int32_t)topk; a.H = (int32_t)H; a.I = (int32_t)I; a.E = (int32_t)E;
    a.s13 = w13_s;
    a.s2 = w2_s;
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

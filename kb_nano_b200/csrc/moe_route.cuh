// Expert routing, warp-level: scores (softmax or sigmoid of the router logits), optional selection bias, optional
// group-limited selection, top-k, renormalisation and scaling for one token per warp.  Used by the stand-alone routing
// kernel and by the expert-parallel dispatch kernel when it routes on the way.
#pragma once
#include "common.cuh"

namespace kbn {

constexpr int kRouteMaxPerLane = 32;      // experts per lane: E <= 1024

// Selection works on order-preserving keys, unsigned integers that compare as the floats do, so that a warp finds its
// largest value with one redux instruction instead of five rounds of shuffles (the whole selection of 8 of 256 experts in
// 8 groups: 13.6 -> 3.4 us of latency).  A NaN has key 0, below everything, and is never chosen.
__device__ __forceinline__ uint32_t route_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);         // -0 counts as +0
    return f != f ? 0u : ((u & 0x80000000u) ? ~u : (u | 0x80000000u));
}
__device__ __forceinline__ float route_unkey(uint32_t k) {
    return k == 0u ? -INFINITY : __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kRouteKeyNegInf = 0x007fffffu;         // route_key(-infinity)

// Routing arguments shared by the stand-alone kernel and the expert-parallel dispatch kernel that routes on the way.
struct RouteArgs {
    const void* logits;
    int64_t ld;
    int E, softmax;
    const float* bias;
    int n_group, topk_group, topk, renorm;
    float renorm_floor, scale;
    int round_bf16;
};

// One warp routes a token whose logits it holds in s (expert of slot (j, lane) is j * 32 + lane; -infinity past E): on return
// lane r < topk holds the r-th choice (weight, expert id).  PER = ceil(E / 32) rounded up to a power of two by the host
// (compile-time unrolling).
template <int PER>
__device__ __forceinline__ void route_logits(const RouteArgs& a, int lane, float (&s)[PER], float& out_weight, int& out_id) {
    const int E = a.E, softmax = a.softmax, n_group = a.n_group, topk_group = a.topk_group, topk = a.topk, renorm = a.renorm;
    const int round_bf16 = a.round_bf16;
    const float* bias = a.bias;
    const float renorm_floor = a.renorm_floor, scale = a.scale;
    float c[PER];
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) mx = fmaxf(mx, s[j]);
    if (softmax) {
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            s[j] = (j * 32 + lane < E) ? expf(s[j] - mx) : 0.0f;
            sum += s[j];
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
        for (int j = 0; j < PER; ++j) s[j] = j * 32 < E ? __fdiv_rn(s[j], sum) : 0.0f * sum;      // a division of zero takes its slow path
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) s[j] = __fdiv_rn(1.0f, 1.0f + expf(-s[j]));
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = j * 32 + lane;
        if (round_bf16) s[j] = __bfloat162float(__float2bfloat16_rn(s[j]));
        c[j] = e < E ? (bias != nullptr ? s[j] + bias[e] : s[j]) : -INFINITY;      // a fp32 bias promotes the sum to fp32
    }
    uint32_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = route_key(c[j]);
    // group-limited selection: experts of the groups that are not among the topk_group best are masked out
    if (n_group > 1 && topk_group < n_group) {
        const uint32_t gs = (uint32_t)(E / n_group), magic = ((1u << 20) + gs - 1u) / gs;      // e / gs == e * magic >> 20 for e, gs <= 1024
        uint32_t gkey = kRouteKeyNegInf;          // lane g holds the score of group g (n_group <= 32)
        for (int g = 0; g < n_group; ++g) {
            uint32_t k1 = 0, k2 = 0;              // two largest choice values of group g seen by this lane
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const uint32_t e = (uint32_t)(j * 32 + lane);
                if (e < (uint32_t)E && ((e * magic) >> 20) == (uint32_t)g) {
                    k2 = max(k2, min(k1, key[j]));
                    k1 = max(k1, key[j]);
                }
            }
            const uint32_t m1 = __reduce_max_sync(0xffffffffu, k1);
            float sc = route_unkey(m1);
            if (bias != nullptr) {
                const unsigned holders = __ballot_sync(0xffffffffu, k1 == m1);
                const uint32_t rest = __reduce_max_sync(0xffffffffu, k1 == m1 ? k2 : k1);
                sc += route_unkey(__popc(holders) > 1 ? m1 : rest);
            }
            if (lane == g) gkey = route_key(sc);
        }
        unsigned keep = 0;                        // bit g set: group g survives
        for (int r = 0; r < topk_group; ++r) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, gkey);
            const int i = __ffs((int)__ballot_sync(0xffffffffu, gkey == m)) - 1;
            keep |= 1u << i;
            if (lane == i) gkey = kRouteKeyNegInf;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t e = (uint32_t)(j * 32 + lane);
            if (e < (uint32_t)E && !((keep >> ((e * magic) >> 20)) & 1u)) key[j] = kRouteKeyNegInf;
        }
    }
    // k rounds: the warp's largest key, the lowest expert that has it
    float wsum = 0.0f, my_w = 0.0f;
    int my_id = 0;
    for (int r = 0; r < topk; ++r) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) best = max(best, key[j]);
        const uint32_t m = __reduce_max_sync(0xffffffffu, best);
        uint32_t at = 0x7fffffffu;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j)
            if (key[j] == m) at = (uint32_t)(j * 32 + lane);
        const int i = m == 0u ? 0x7fffffff : (int)__reduce_min_sync(0xffffffffu, at);
        float w = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j * 32 + lane == i) {
                w = s[j];
                key[j] = kRouteKeyNegInf;
            }
        w = __shfl_sync(0xffffffffu, w, i & 31);
        wsum += w;
        if (lane == r) {                          // lane r keeps the r-th choice (topk <= 32)
            my_w = w;
            my_id = i;
        }
    }
    float w = my_w;
    if (lane < topk) {
        if (round_bf16) {
            if (renorm) w = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(w, __bfloat162float(__float2bfloat16_rn(fmaxf(wsum, renorm_floor))))));
            if (scale != 1.0f) w = __bfloat162float(__float2bfloat16_rn(w * scale));
        } else {
            if (renorm) w = __fdiv_rn(w, fmaxf(wsum, renorm_floor));
            if (scale != 1.0f) w *= scale;
        }
    }
    out_weight = w;
    out_id = my_id;
}

template <int PER>
__device__ __forceinline__ void load_logits(const RouteArgs& a, bool bf16_in, int64_t t, int lane, float (&s)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = j * 32 + lane;
        s[j] = -INFINITY;
        if (e < a.E)
            s[j] = bf16_in ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.logits)[t * a.ld + e]) : static_cast<const float*>(a.logits)[t * a.ld + e];
    }
}

template <int PER, bool BF16_IN>
__device__ __forceinline__ void route_token(const RouteArgs& a, int64_t t, int lane, float& out_weight, int& out_id) {
    float s[PER];
    load_logits<PER>(a, BF16_IN, t, lane, s);
    route_logits<PER>(a, lane, s, out_weight, out_id);
}

}  // namespace kbn

// Dense MXFP4 GEMM, C[m,n] = sum_k A[m,k] B[n,k] (+ bias[n]), A [M,K] and B [N,K] in MXFP4, fp32 accumulation, bf16 out:
// the 4-bit counterpart of the block-scaled FP8 linear (tasks/baseline/L1/fp8_linear.py:371-450; kb-nano has no 4-bit path).
//
// tcgen05.mma kind::mxf4 with block scales multiplies the codes and applies both operands' power-of-two scales itself, one
// per 32 K-values (scale_vec::2X: two scale bytes per row and instruction of K = 64).
//
// At 4 bits the tensor cores eat 93 B/clk and SM of operands from a 128 x 256 tile on one SM, more than L2 delivers (about 64);
// so two SMs share a 256 x 256 tile (cta_group::2): each loads its own 128 rows of A and half of the tile's 256 rows of B, 62
// B/clk.  One K-step is 256 values (128 bytes a row): 32 KB of codes and 3 KB of scales per SM, five steps in the ring (seven of
// 24 + 2 KB with 128-column tiles).  All copies are plain tiled TMA loads into the issuing CTA's own shared memory, counted on
// the even CTA's barrier.
//
//   warps       loads; products; epilogue (eight); scales.  A step is four products of K = 64; its scales are copied from shared
//               to tensor memory by a warp of their own, into columns of the step's ring slot, because the products' warp, with
//               the copies' instructions between its own, took longer to issue a step than the tensor cores to run it
//               (8192 x 7168 x 7168: 197 -> 153 us with the rest of this list).
//   many tiles  persistent CTA pairs over the tiles.  The epilogue warps drain the accumulator into registers (128 columns a
//               thread), release it, and convert and store while the next tile's products run.  (Two 256-column accumulators
//               and the scales do not fit the 512 columns of tensor memory.)  The results go through shared memory to tiled
//               stores where the output's rows allow it, else straight to global memory.
//   few tiles   256 x 128 tiles while every pair then has one tile at most.
//   few tiles, long K   one 256 x 256 tile per cluster of 2 S CTAs, whose S pairs split K.  Each pair owns 256 / S columns and
//               receives the other pairs' partial sums of them as one bulk copy each through the cluster's shared memory;
//               partials are added in slice order, so results are reproducible.
//
// Measured inside a graph: 8192 x 7168 x 7168 153 us, 5.5 PFLOP/s, 82 % of four times the measured bf16 rate of cuBLAS.  What is missing is
// the drain of the accumulator between two tiles (1 to 2 us of 11.8) and the last round (896 tiles on 74 pairs: 8 in the
// thirteenth round, which run as 16 halves).  In a loop of seconds the
// power cap sets the clock (calls in a row, with the quantiser: 203 to 211 us).  512 x 4096 x 7168: 17.5 us with the quantiser (3.2)
// in front (calls in a row 19.2 to 20.2), against 4.5 for the products alone: one tile per pair has nothing to hide its first loads and its drain behind.
#include <algorithm>

#include "gemm_common.cuh"
#include "mxfp4.cuh"
#include "tensor_map.cuh"

namespace kbn {
namespace mxfp4 {

constexpr int kTileM = 256;
constexpr int kABytes = 128 * 128;                             // this CTA's rows of A, one K-step of 256 values
constexpr int kEpiWarps = 8;
constexpr int kScaleWarp = 2 + kEpiWarps;                      // warps: loads, products, epilogue, scales
constexpr int kGemmThreads = 32 * (kScaleWarp + 1);
constexpr int kStagingBytes = kEpiWarps * 32 * 128;            // 32 rows x 64 bf16 columns per epilogue warp
constexpr int kTmemColumns = 512, kColScales = 256;            // accumulators in columns 0-255, scales behind them
constexpr int kSplitGain = 18;                                 // K-steps a split over the cluster has to save
constexpr int kGroupM = 8;                                     // tile rows that run side by side, for reuse of B in L2

// BN: tile columns, 256 or 128.
template <int BN>
struct Cfg {
    static constexpr int kBBytes = BN / 2 * 128;               // this CTA's half of the tile's rows of B
    static constexpr int kOperandBytes = kABytes + kBBytes;
    static constexpr int kSfBlocks = 1 + BN / 128;             // row blocks whose scales a step needs: A's own, all of B's
    static constexpr int kSfBytes = kSfBlocks * 1024;          // two 128-K blocks each
    static constexpr int kStages = BN == 256 ? 5 : 7;
    static constexpr uint32_t kTxPair = 2u * (kOperandBytes + kSfBytes);
    static constexpr int kAccs = 256 / BN;                     // accumulators: a 128-column tile is drained under the next one
    static constexpr int kScaleCols = 4 * kSfBlocks;           // scale columns of 128 of K; every ring slot has its own
    static_assert(kColScales + kStages * 2 * kScaleCols <= kTmemColumns, "tensor memory");
    static constexpr int kSmem = kStages * (kOperandBytes + kSfBytes) + kStagingBytes + 1024 + 256;
    static constexpr int kExchange = 2 * 3 * 128 * (BN / 4) * 4;      // split K: partial sums sent and received, S = 4
    static_assert(kExchange <= kStages * (kOperandBytes + kSfBytes) + kStagingBytes && kSmem <= 232448, "shared memory");
};

struct GemmArgs {
    const __nv_bfloat16* bias;
    __nv_bfloat16* C;
    int64_t ldc;
    int32_t* status;
    int32_t M, N, kblocks, steps;      // kblocks: 128-K blocks (scales), steps: 256-K steps
    int32_t m_tiles, n_tiles, S;
    int32_t whole;                     // tiles from this one on are worked on as two halves of 128 columns each
    int32_t tiled_out;                 // the output's rows allow tiled stores
};

// Instruction descriptor, kind::mxf4: A = B = e2m1 K-major, UE8M0 scales, K = 64 dense.
__host__ __device__ constexpr uint32_t idesc_mxf4(uint32_t m, uint32_t n, uint32_t sf_id) {
    return (sf_id << 4)          // scale bytes of B: 0 or 2
           | (1u << 7)           // A format: e2m1
           | (1u << 10)          // B format: e2m1
           | ((n >> 3) << 17)    // N / 8
           | (1u << 23)          // scale format: UE8M0
           | ((m >> 7) << 27)    // M / 128
           | (sf_id << 29);      // scale bytes of A
}
// The issuing warps run their loops whole, every lane with the same values, and elect one lane inside each instruction.  With
// one lane branched off instead, the operands cannot stay in uniform registers and each tcgen05 or TMA instruction cost its
// issuer about 70 cycles: more, over a step, than the tensor cores need for it (8192 x 7168 x 7168, with the quantiser:
// 259 -> 197 us).
#define KBN_ELECT "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
__device__ __forceinline__ void mma_mxf4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(KBN_ELECT
                 ".reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
                 : "memory");
}
__device__ __forceinline__ void copy_scales_pair(uint32_t dst_tmem, uint64_t src_desc) {
    asm volatile(KBN_ELECT "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(dst_tmem), "l"(src_desc) : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar, uint16_t cta_mask) {
    asm volatile(KBN_ELECT "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
                 ::"r"(bar), "h"(cta_mask) : "memory");
}
__device__ __forceinline__ void load_pair(uint32_t dst, const void* tmap, int32_t x, int32_t y, uint32_t bar_cluster) {
    asm volatile(KBN_ELECT
                 "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar_cluster), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
    asm volatile(KBN_ELECT "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
}
// Tiled store of a box from shared memory; completion by bulk groups of the elected lane.
__device__ __forceinline__ void store_box(const void* tmap, int32_t x, int32_t y, uint32_t src) {
    asm volatile(KBN_ELECT
                 "@e cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\t"
                 "@e cp.async.bulk.commit_group;\n\t}"
                 ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void stores_have_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void arrive_cluster(uint32_t bar_cluster) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// `half`: 0 or 1 of a halved tile, -1 of a whole one.
__device__ __forceinline__ void tile_of(int32_t t, const GemmArgs& p, int32_t& m_tile, int32_t& n_tile, int32_t& half) {
    half = -1;
    if (t >= p.whole) {
        half = (t - p.whole) & 1;
        t = p.whole + ((t - p.whole) >> 1);
    }
    const int32_t per_group = kGroupM * p.n_tiles;
    const int32_t grp = t / per_group, first = grp * kGroupM;
    const int32_t size = min(kGroupM, p.m_tiles - first);
    const int32_t in = t - grp * per_group;
    m_tile = first + in % size;
    n_tile = in / size;
}

// + bias, 32 columns.
__device__ __forceinline__ void add_bias(float (&f)[32], const GemmArgs& p, int32_t n0) {
    if (p.bias == nullptr) return;
    if (n0 + 32 <= p.N && (reinterpret_cast<uintptr_t>(p.bias + n0) & 15u) == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint4 b = *reinterpret_cast<const uint4*>(p.bias + n0 + 8 * j);
            const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[8 * j + 2 * i] += bf16_lo(w[i]);
                f[8 * j + 2 * i + 1] += bf16_hi(w[i]);
            }
        }
    } else {
#pragma unroll
        for (int q = 0; q < 32; ++q)
            if (n0 + q < p.N) f[q] += __bfloat162float(p.bias[n0 + q]);
    }
}
// 32 columns of one row -> bf16, straight to global memory.
__device__ __forceinline__ void store_row(const float (&f)[32], const GemmArgs& p, int32_t row, int32_t n0) {
    __nv_bfloat16* c = p.C + (int64_t)row * p.ldc + n0;
    const bool vec = (reinterpret_cast<uintptr_t>(c) & 15u) == 0;
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
        if (n0 + j + 8 <= p.N && vec) {
            uint4 v;
            v.x = pack_bf16x2(f[j + 0], f[j + 1]); v.y = pack_bf16x2(f[j + 2], f[j + 3]);
            v.z = pack_bf16x2(f[j + 4], f[j + 5]); v.w = pack_bf16x2(f[j + 6], f[j + 7]);
            *reinterpret_cast<uint4*>(c + j) = v;
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (n0 + j + q < p.N) c[j + q] = __float2bfloat16_rn(f[j + q]);
        }
    }
}
// 32 columns of one row -> bf16 in a warp's staging rows (64 columns, 128 bytes, swizzled as the tensor map expects).
__device__ __forceinline__ void stage_row(const float (&f)[32], uint32_t staging, int row, int half) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        ptx::st_shared_v4(staging + (uint32_t)row * 128u + (uint32_t)(((4 * half + j) ^ (row & 7)) << 4), pack_bf16x2(f[8 * j + 0], f[8 * j + 1]),
                          pack_bf16x2(f[8 * j + 2], f[8 * j + 3]), pack_bf16x2(f[8 * j + 4], f[8 * j + 5]), pack_bf16x2(f[8 * j + 6], f[8 * j + 7]));
}

template <int BN, bool SPLIT>
__global__ void __launch_bounds__(kGemmThreads, 1)
mxfp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSfa,
                  const __grid_constant__ CUtensorMap tmSfb, const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmBh, const GemmArgs p) {
    using F = Cfg<BN>;
    constexpr int kStages = F::kStages, kOperandBytes = F::kOperandBytes, kSfBytes = F::kSfBytes;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    uint8_t* sf = smem + (size_t)kStages * kOperandBytes;
    uint8_t* staging = sf + (size_t)kStages * kSfBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kStagingBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * kStages + 5);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t bar_full = ptx::smem_u32(bars), bar_empty = ptx::smem_u32(bars + kStages);
    const uint32_t bar_scales = ptx::smem_u32(bars + 2 * kStages);             // a slot's scales are in tensor memory
    const uint32_t bar_tfull = ptx::smem_u32(bars + 3 * kStages), bar_tempty = bar_tfull + 16, bar_xchg = bar_tfull + 32;      // two accumulators each
    const uint32_t tiles_smem = ptx::smem_u32(smem), sf_smem = ptx::smem_u32(sf);

    const uint32_t rank = ptx::cluster_ctarank();
    const uint32_t pr = rank & 1u, ks = rank >> 1, leader = rank & ~1u;      // place in the pair, K-slice, issuing CTA
    const uint16_t pair_mask = (uint16_t)(3u << leader);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(bar_full + 8 * s, 1);         // armed by the even CTA for both CTAs' copies
            ptx::mbar_init(bar_empty + 8 * s, 1);        // one commit, delivered to both
            ptx::mbar_init(bar_scales + 8 * s, 1);       // one commit, in the even CTA
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(bar_tfull + 8 * i, 1);
            ptx::mbar_init(bar_tempty + 8 * i, 2 * kEpiWarps);       // used in the even CTA: the epilogue warps of both
        }
        ptx::mbar_init(bar_xchg, 1);
        if (SPLIT) ptx::mbar_arrive_expect_tx(bar_xchg, (uint32_t)(p.S - 1) * (uint32_t)(128 * (BN / p.S) * 4));
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
        ptx::prefetch_tensormap(&tmA);
        ptx::prefetch_tensormap(&tmB);
        ptx::prefetch_tensormap(&tmSfa);
        ptx::prefetch_tensormap(&tmSfb);
        if (p.tiled_out) ptx::prefetch_tensormap(&tmC);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), kTmemColumns);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();              // the partner's barriers exist before anything is sent to them
    ptx::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    // Everything this kernel reads, the weights too, may have been written by the kernel before it.
    ptx::grid_dependency_wait();
    ptx::launch_dependents();

    const int32_t tiles = 2 * p.m_tiles * p.n_tiles - p.whole;      // halves count for themselves
    const int32_t cluster = (int32_t)(blockIdx.x / (SPLIT ? 2u * (uint32_t)p.S : 2u));
    const int32_t stride = SPLIT ? tiles : (int32_t)(gridDim.x / 2);          // split: one tile per cluster
    const int32_t per_slice = SPLIT ? (p.steps + p.S - 1) / p.S : p.steps;
    const int32_t k0 = (int32_t)ks * per_slice, k1 = min(p.steps, k0 + per_slice);      // not empty: the host sees to it

    if (warp == 0) {
        const WaitCtx w{abort_flag, p.status, 12};
        uint32_t slot = 0, phase = 0;
        bool ok = true;
        for (int32_t t = cluster; ok && t < tiles; t += stride) {
            int32_t mt, nt, half;
            tile_of(t, p, mt, nt, half);
            const bool halved = half >= 0;
            const int32_t row_a = mt * kTileM + (int32_t)pr * 128, row_b = nt * BN + (halved ? half * (BN / 2) + (int32_t)pr * (BN / 4) : (int32_t)pr * (BN / 2));
            const int32_t sfa_row = (row_a >> 7) * p.kblocks, sfb_row = nt * (BN / 128) * p.kblocks;
            for (int32_t k = k0; k < k1; ++k) {
                ok = __all_sync(0xffffffffu, wait_bar(bar_empty + 8 * slot, phase ^ 1u, w));
                if (!ok) break;
                if (pr == 0) expect_bytes(bar_full + 8 * slot, halved ? F::kTxPair - F::kBBytes : F::kTxPair);
                const uint32_t bar = ptx::mapa(bar_full + 8 * slot, leader);
                const uint32_t dst = tiles_smem + slot * kOperandBytes, sdst = sf_smem + slot * kSfBytes;
                load_pair(dst, &tmA, k * 128, row_a, bar);
                load_pair(dst + kABytes, halved ? &tmBh : &tmB, k * 128, row_b, bar);
                // scales: the packed array as rows of 256 bytes, two per 512-byte block
                load_pair(sdst, &tmSfa, 0, 2 * (sfa_row + 2 * k), bar);
#pragma unroll
                for (int b = 0; b < BN / 128; ++b) load_pair(sdst + 1024 * (1 + b), &tmSfb, 0, 2 * (sfb_row + b * p.kblocks + 2 * k), bar);
                if (++slot == kStages) slot = 0, phase ^= 1u;
            }
        }
    } else if (warp == 1) {
        if (pr == 0) {
            const WaitCtx w{abort_flag, p.status, 13};
            uint32_t slot = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (int32_t t = cluster; ok && t < tiles; t += stride) {
                if (!SPLIT) {                 // the accumulator has been drained (passes at once while it is fresh)
                    const long long t0 = clock64();
                    while (!__all_sync(0xffffffffu, try_wait_cluster(bar_tempty + 8 * acc, acc_phase ^ 1u))) {
                        ok = __all_sync(0xffffffffu, *abort_flag == 0 && clock64() - t0 <= kWaitLimitCycles);
                        if (!ok) {
                            *abort_flag = 1;
                            if (lane == 0) atomicCAS(p.status, 0, w.code | (int)(blockIdx.x << 8));
                            break;
                        }
                    }
                    if (!ok) break;
                    ptx::tc_fence_after();
                }
                const uint32_t d = tmem + acc * BN;
                int32_t mt, nt, half;
                tile_of(t, p, mt, nt, half);
                const uint32_t id0 = half >= 0 ? idesc_mxf4(kTileM, BN / 2, 0) : idesc_mxf4(kTileM, BN, 0), id2 = id0 | idesc_mxf4(0, 0, 2);
                const uint32_t sfb_at = half > 0 ? 8u : 4u;      // the second half's scales are the tile's second block
                for (int32_t k = k0; k < k1; ++k) {
                    ok = __all_sync(0xffffffffu, wait_bar(bar_scales + 8 * slot, phase, w));      // operands and scales are there
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint32_t a = tiles_smem + slot * kOperandBytes, scales = tmem + kColScales + slot * 2 * F::kScaleCols;
                    const uint64_t a_desc = ptx::umma_desc_k_sw128(a), b_desc = ptx::umma_desc_k_sw128(a + kABytes);
                    const int halves = min(2, p.kblocks - 2 * k);      // the last step may hold one 128-K block only
                    for (int h = 0; h < halves; ++h) {
                        const uint32_t sfa = scales + F::kScaleCols * h, sfb = sfa + sfb_at;
                        mma_mxf4_pair(d, a_desc + 4 * h, b_desc + 4 * h, id0, sfa, sfb, (k > k0 || h > 0) ? 1u : 0u);
                        mma_mxf4_pair(d, a_desc + 4 * h + 2, b_desc + 4 * h + 2, id2, sfa, sfb, 1u);
                    }
                    commit_pair(bar_empty + 8 * slot, pair_mask);
                    if (++slot == kStages) slot = 0, phase ^= 1u;
                }
                if (ok) commit_pair(bar_tfull + 8 * acc, pair_mask);
                if (++acc == F::kAccs) acc = 0, acc_phase ^= 1u;
            }
        }
    } else if (warp == kScaleWarp) {
        // Scales, shared memory -> tensor memory, by a warp of its own: beside the products' warp, whose four instructions a
        // step then take less time to issue than the tensor cores need for them.
        if (pr == 0) {
            const WaitCtx w{abort_flag, p.status, 22};
            uint32_t slot = 0, phase = 0;
            bool ok = true;
            for (int32_t t = cluster; ok && t < tiles; t += stride) {
                for (int32_t k = k0; k < k1; ++k) {
                    ok = __all_sync(0xffffffffu, wait_bar(bar_full + 8 * slot, phase, w));
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint32_t s = sf_smem + slot * kSfBytes, scales = tmem + kColScales + slot * 2 * F::kScaleCols;
#pragma unroll
                    for (int h = 0; h < 2; ++h)        // of a last step's missing block: never used
#pragma unroll
                        for (int b = 0; b < F::kSfBlocks; ++b) copy_scales_pair(scales + F::kScaleCols * h + 4 * b, ptx::umma_desc_sf(s + 1024 * b + 512 * h));
                    commit_pair(bar_scales + 8 * slot, (uint16_t)(1u << leader));
                    if (++slot == kStages) slot = 0, phase ^= 1u;
                }
            }
        }
    } else if (!SPLIT) {
        const WaitCtx w{abort_flag, p.status, 14};
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t mine = ptx::smem_u32(staging) + (uint32_t)(warp - 2) * (32 * 128);
        uint32_t acc = 0, phase = 0;
        constexpr int kCols = BN / 2, kChunks = kCols / 32;      // of this warp
        for (int32_t t = cluster; t < tiles; t += stride) {
            if (!__all_sync(0xffffffffu, wait_bar(bar_tfull + 8 * acc, phase, w))) break;
            ptx::tc_fence_after();
            int32_t mt, nt, part;
            tile_of(t, p, mt, nt, part);
            const int cols = part >= 0 ? kCols / 2 : kCols;      // of this warp, in this tile
            uint32_t r[kChunks][32];
#pragma unroll
            for (int c = 0; c < kChunks; ++c) ptx::tmem_ld_32x32(tmem + ((uint32_t)(quarter * 32) << 16) + acc * BN + half * cols + c * 32, r[c]);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) ptx::tmem_ld_wait(r[c]);
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(ptx::mapa(bar_tempty + 8 * acc, leader));
            if (++acc == F::kAccs) acc = 0, phase ^= 1u;
            const int32_t row0 = mt * kTileM + (int32_t)pr * 128 + quarter * 32;
            if (row0 >= p.M || *abort_flag != 0) continue;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                if (c * 32 >= cols) break;
                const int32_t n0 = nt * BN + max(part, 0) * (BN / 2) + half * cols + c * 32;
                float f[32];
#pragma unroll
                for (int q = 0; q < 32; ++q) f[q] = __uint_as_float(r[c][q]);
                add_bias(f, p, n0);
                if (p.tiled_out) {
                    if ((c & 1) == 0) {
                        stores_have_read();      // nothing to wait for in lanes that stored nothing
                        __syncwarp();
                    }
                    stage_row(f, mine, lane, c & 1);
                    if ((c & 1) == 1 && n0 - 32 < p.N) {
                        ptx::fence_proxy_async();
                        __syncwarp();
                        store_box(&tmC, (n0 - 32) * 2, row0, mine);
                    }
                } else if (row0 + lane < p.M) {
                    store_row(f, p, row0 + lane, n0);
                }
            }
        }
        stores_have_read();              // the shared memory may go once they have
    } else {
        const WaitCtx w{abort_flag, p.status, 15};
        wait_bar(bar_tfull, 0u, w);
        __syncwarp();
        ptx::tc_fence_after();
    }

    if (SPLIT) {
        int32_t mt, nt, half_tile;
        tile_of(cluster, p, mt, nt, half_tile);
        const int32_t row0 = mt * kTileM + (int32_t)pr * 128;
        const int32_t live = max(0, min(p.M - row0, 128));
        __syncwarp();
        ptx::cluster_sync();              // every CTA of the cluster is done with its stages: they may be overwritten
        const int W = BN / p.S;
        const uint32_t slot_bytes = (uint32_t)(128 * W * 4), units = (uint32_t)W / 4u;
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int r_in_tile = quarter * 32 + lane;
        const uint32_t swz = (uint32_t)r_in_tile & (units - 1u);
        // partial sums of the columns other slices own: rows of W floats, 16-byte units XOR-swizzled by the row so that a
        // lane per row stores without bank conflicts; one bulk copy per owner
        const bool epilogue = warp >= 2 && warp < kScaleWarp;
        if (epilogue) {
#pragma unroll 1
            for (int cc = half; cc < BN / 32; cc += 2) {
                const uint32_t o = (uint32_t)(32 * cc / W);
                if (o == ks) continue;
                uint32_t r[32];
                ptx::tmem_ld_32x32(tmem + ((uint32_t)(quarter * 32) << 16) + 32 * cc, r);
                ptx::tmem_ld_wait(r);
                const uint32_t send = o < ks ? o : o - 1u;
                const uint32_t base = tiles_smem + send * slot_bytes + (uint32_t)r_in_tile * (uint32_t)W * 4u;
                const uint32_t u0 = (uint32_t)(32 * cc % W) / 4u;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    ptx::st_shared_v4(base + (((u0 + (uint32_t)j) ^ swz) << 4), r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
            }
            ptx::fence_proxy_async();     // the bulk copies below read what was just stored
        }
        __syncthreads();
        if (threadIdx.x == 64) {
            for (uint32_t o = 0; o < (uint32_t)p.S; ++o) {
                if (o == ks) continue;
                const uint32_t send = o < ks ? o : o - 1u, recv = ks < o ? ks : ks - 1u, owner = (o << 1) | pr;
                ptx::bulk_copy_to_cluster(ptx::mapa(tiles_smem + ((uint32_t)(p.S - 1) + recv) * slot_bytes, owner), tiles_smem + send * slot_bytes, slot_bytes,
                                          ptx::mapa(bar_xchg, owner));
            }
        }
        if (epilogue) {
            const WaitCtx w{abort_flag, p.status, 16};
            wait_bar(bar_xchg, 0u, w);
            __syncwarp();
            if (quarter * 32 < live && *abort_flag == 0) {
                // this warp's half of the owned band; two slices leave the staging rows free and hand whole boxes to the TMA
                const bool boxes = p.S == 2 && p.tiled_out;
                const uint32_t mine = ptx::smem_u32(staging) + (uint32_t)(warp - 2) * (32 * 128);
                const int32_t c0 = (int32_t)ks * W + half * (W / 2);
#pragma unroll 1
                for (int c = 0; c < W / 64; ++c) {
                    const int32_t col = c0 + 32 * c, n0 = nt * BN + col;
                    uint32_t r[32];
                    ptx::tmem_ld_32x32(tmem + ((uint32_t)(quarter * 32) << 16) + col, r);
                    ptx::tmem_ld_wait(r);
                    float f[32];
#pragma unroll
                    for (int q = 0; q < 32; ++q) f[q] = 0.f;
                    const uint32_t u0 = (uint32_t)(col % W) / 4u;
                    for (uint32_t sl = 0; sl < (uint32_t)p.S; ++sl) {
                        if (sl == ks) {
#pragma unroll
                            for (int q = 0; q < 32; ++q) f[q] += __uint_as_float(r[q]);
                            continue;
                        }
                        const uint32_t recv = sl < ks ? sl : sl - 1u;
                        const uint32_t base = tiles_smem + ((uint32_t)(p.S - 1) + recv) * slot_bytes + (uint32_t)r_in_tile * (uint32_t)W * 4u;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float4 v = ptx::ld_shared_v4(base + (((u0 + (uint32_t)i) ^ swz) << 4));
                            f[4 * i + 0] += v.x; f[4 * i + 1] += v.y; f[4 * i + 2] += v.z; f[4 * i + 3] += v.w;
                        }
                    }
                    add_bias(f, p, n0);
                    if (boxes) {
                        stage_row(f, mine, lane, c & 1);
                        if ((c & 1) == 1 && n0 - 32 < p.N) {
                            ptx::fence_proxy_async();
                            __syncwarp();
                            store_box(&tmC, (n0 - 32) * 2, row0 + quarter * 32, mine);
                        }
                    } else if (r_in_tile < live) {
                        store_row(f, p, row0 + r_in_tile, n0);
                    }
                }
                stores_have_read();
            }
        }
    }

    if (*abort_flag != 0)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);      // copies that were asked for may still be on their way
    ptx::tc_fence_before();
    __syncthreads();
    // no CTA leaves while its partner's copies, products or arrivals may still touch its memory
    ptx::cluster_sync();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem, kTmemColumns);
    }
}

// ---- host ----------------------------------------------------------------------------------------

// Codes [rows, K]: boxes of box_rows x 256 values (128 bytes, 128-byte swizzle).
static int code_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t K, int box_rows, bool weights) {
    TensorMapSpec t;
    memset(&t, 0, sizeof(t));
    t.base = base;
    t.rank = 2;
    t.dims[0] = (uint64_t)(K / 2); t.dims[1] = (uint64_t)rows; t.dims[2] = 1;
    t.strides[0] = (uint64_t)(K / 2);
    t.box[0] = 128; t.box[1] = (uint32_t)box_rows; t.box[2] = 1;
    t.swizzle = CU_TENSOR_MAP_SWIZZLE_128B;
    t.promo = weights ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
    return encode_tensor_map(tm, t);
}
// Packed scales as rows of 256 bytes: boxes of two 512-byte blocks.
static int scale_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t kblocks) {
    TensorMapSpec t;
    memset(&t, 0, sizeof(t));
    t.base = base;
    t.rank = 2;
    t.dims[0] = 256; t.dims[1] = (uint64_t)((rows + 127) / 128 * kblocks * 2); t.dims[2] = 1;
    t.strides[0] = 256;
    t.box[0] = 256; t.box[1] = 4; t.box[2] = 1;
    t.swizzle = CU_TENSOR_MAP_SWIZZLE_NONE;
    t.promo = CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
    return encode_tensor_map(tm, t);
}

// Output [M, N] bf16, row stride ldc: boxes of 32 rows x 64 columns.
static int out_map(CUtensorMap* tm, const void* base, int64_t M, int64_t N, int64_t ldc) {
    TensorMapSpec t;
    memset(&t, 0, sizeof(t));
    t.base = base;
    t.rank = 2;
    t.dims[0] = (uint64_t)N * 2; t.dims[1] = (uint64_t)M; t.dims[2] = 1;
    t.strides[0] = (uint64_t)ldc * 2;
    t.box[0] = 128; t.box[1] = 32; t.box[2] = 1;
    t.swizzle = CU_TENSOR_MAP_SWIZZLE_128B;
    t.promo = CU_TENSOR_MAP_L2_PROMOTION_NONE;
    return encode_tensor_map(tm, t);
}

template <int BN, bool SPLIT>
static int max_clusters(int size) {
    static std::atomic<int> cache[64][9];      // calls come from several threads at once, without the interpreter's lock
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int known = cache[dev][size].load(std::memory_order_acquire);
    if (known == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(size * 16));
        cfg.blockDim = dim3(kGemmThreads);
        cfg.dynamicSmemBytes = Cfg<BN>::kSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(mxfp4_gemm_kernel<BN, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::kSmem) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, mxfp4_gemm_kernel<BN, SPLIT>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
        }
        known = n > 0 ? n : -1;
        cache[dev][size].store(known, std::memory_order_release);
    }
    return known > 0 ? known : 0;
}

template <int BN, bool SPLIT>
static int launch(const void* A, const void* sfa, const void* B, const void* sfb, int64_t K, const GemmArgs& p, unsigned clusters, cudaStream_t st) {
    CUtensorMap a, b, sa, sb, c, bh;
    int rc;
    if ((rc = code_map(&a, A, p.M, K, 128, false)) != KBN_OK || (rc = code_map(&b, B, p.N, K, BN / 2, true)) != KBN_OK ||
        (rc = scale_map(&sa, sfa, p.M, p.kblocks)) != KBN_OK || (rc = scale_map(&sb, sfb, p.N, p.kblocks)) != KBN_OK)
        return rc;
    c = bh = a;                          // never read without tiled_out, without halved tiles
    if (p.whole < p.m_tiles * p.n_tiles && (rc = code_map(&bh, B, p.N, K, BN / 4, true)) != KBN_OK) return rc;
    if (p.tiled_out && (rc = out_map(&c, p.C, p.M, p.N, p.ldc)) != KBN_OK) return rc;
    const unsigned size = SPLIT ? 2u * (unsigned)p.S : 2u;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(clusters * size);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = Cfg<BN>::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    KBN_CUDA(cudaLaunchKernelEx(&cfg, mxfp4_gemm_kernel<BN, SPLIT>, a, b, sa, sb, c, bh, p));
    KBN_CHECK_LAUNCH();
    return KBN_OK;
}

template <int BN>
static int launch_persistent(const void* A, const void* sfa, const void* B, const void* sfb, int64_t K, const GemmArgs& p, cudaStream_t st) {
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    const int pairs = max_clusters<BN, false>(2);
    KBN_REQUIRE(pairs > 0, KBN_ERR_UNSUPPORTED, "kbn_mxfp4_gemm_nt: no CTA pair fits this device");
    // A last round that at most half of the pairs have a tile in is worked on in halves, by twice as many (with the quantiser):
    // 1280 x 4096 x 2048 (80 tiles on 74 pairs) 14.9 -> 13.8 us, x 7168 32.8 -> 30.8, 8192 x 7168 x 1024 (896) 51.7 -> 48.6,
    // x 7168 180 either way, where power is the bound.  As a launch of their own the halves cost more than they saved.
    GemmArgs q = p;
    q.whole = (int32_t)tiles;
    const int64_t rest = tiles % pairs;
    if (BN == 256 && tiles > pairs && rest > 0 && 2 * rest <= pairs) q.whole = (int32_t)(tiles - rest);
    return launch<BN, false>(A, sfa, B, sfb, K, q, (unsigned)std::min<int64_t>(tiles, pairs), st);
}

}  // namespace mxfp4
}  // namespace kbn

extern "C" int kbn_mxfp4_gemm_nt(const void* A, const void* sfa_packed, const void* B, const void* sfb_packed, const void* bias, void* C, int64_t ldc,
                                 int64_t M, int64_t N, int64_t K, kbn_stream_t stream) {
    using namespace kbn;
    using namespace kbn::mxfp4;
    KBN_REQUIRE(M >= 0 && N >= 0 && K > 0, KBN_ERR_ARG, "kbn_mxfp4_gemm_nt: bad sizes (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
    if (M == 0 || N == 0) return KBN_OK;
    KBN_REQUIRE(A && sfa_packed && B && sfb_packed && C, KBN_ERR_ARG, "kbn_mxfp4_gemm_nt: null pointer");
    KBN_REQUIRE(K % 32 == 0, KBN_ERR_ARG, "kbn_mxfp4_gemm_nt: K=%lld must be a multiple of 32", (long long)K);
    KBN_REQUIRE(aligned16(A) && aligned16(B) && aligned16(sfa_packed) && aligned16(sfb_packed), KBN_ERR_ARG, "kbn_mxfp4_gemm_nt: pointers must be 16-byte aligned");
    KBN_REQUIRE((reinterpret_cast<uintptr_t>(C) & 1u) == 0 && (ldc >= N || M == 1), KBN_ERR_ARG, "kbn_mxfp4_gemm_nt: odd output pointer or row stride below N");
    KBN_REQUIRE(aligned_to(bias, 2), KBN_ERR_ARG, "kbn_mxfp4_gemm_nt: odd bias pointer");
    const int64_t kblocks = (K + 127) / 128;
    // packed-scale rows and tile numbers are 32-bit in the kernel
    KBN_REQUIRE(K < (1ll << 31) && M < (1ll << 30) && N < (1ll << 30) && (M / 128 + 3) * kblocks * 2 < (1ll << 31) && (N / 128 + 3) * kblocks * 2 < (1ll << 31) &&
                    ((M + 255) / 256) * ((N + 255) / 256) < (1ll << 30), KBN_ERR_UNSUPPORTED, "kbn_mxfp4_gemm_nt: problem too large");
    GemmArgs p{};
    p.bias = static_cast<const __nv_bfloat16*>(bias);
    p.C = static_cast<__nv_bfloat16*>(C);
    p.ldc = ldc;
    p.M = (int32_t)M; p.N = (int32_t)N;
    p.kblocks = (int32_t)kblocks;
    p.steps = (int32_t)((kblocks + 1) / 2);
    p.m_tiles = (int32_t)((M + kTileM - 1) / kTileM);
    int rc = gemm_status_ptr(&p.status);
    if (rc != KBN_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (M == 1) p.ldc = (N + 7) / 8 * 8;      // the stride of a single row is free
    p.tiled_out = aligned16(C) && p.ldc % 8 == 0;
    const int64_t wide = p.m_tiles * ((N + 255) / 256), narrow = p.m_tiles * ((N + 127) / 128);
    // Few tiles: K split over the cluster, the most slices that are resident at once and leave each a step.  The exchange of
    // partial sums takes as long as 18 steps, so a split has to save as many: measured with the quantiser, split and not:
    // 512 x 4096 x 7168 (S = 2 saves 14 of 28 steps) 17.6 and 17.1 us, x 9216 (18 of 36) 20.3 and 20.2, x 12288 (24 of 48) 23.3
    // and 24.4; 64 x 4096 x 7168 (S = 4, 21 of 28) 13.4 and 13.6, 64 x 2048 x 16384 (48 of 64) 17.1 and 23.7.
    p.n_tiles = (int32_t)((N + 255) / 256);
    for (int S = 4; S >= 2; S /= 2) {
        const int per = (p.steps + S - 1) / S;
        if (2 * S * wide > sm_count() || (S - 1) * per >= p.steps || p.steps - per < kSplitGain || wide > max_clusters<256, true>(2 * S)) continue;
        p.S = S;
        p.whole = (int32_t)wide;
        return launch<256, true>(A, sfa_packed, B, sfb_packed, K, p, (unsigned)wide, st);
    }
    const int64_t pairs = sm_count() / 2;
    // 128 columns a tile while every pair then has one tile at most; more rounds of them cost 0.75 of a round of wide ones each.
    if (narrow <= pairs) {
        p.n_tiles = (int32_t)((N + 127) / 128);
        return launch_persistent<128>(A, sfa_packed, B, sfb_packed, K, p, st);
    }
    return launch_persistent<256>(A, sfa_packed, B, sfb_packed, K, p, st);
}

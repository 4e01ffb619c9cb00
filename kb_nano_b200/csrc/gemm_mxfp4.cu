// Dense MXFP4 GEMM, C[m,n] = sum_k A[m,k] B[n,k] (+ bias[n]), A [M,K] and B [N,K] in MXFP4, fp32 accumulation, bf16 out:
// the 4-bit counterpart of the block-scaled FP8 linear (tasks/baseline/L1/fp8_linear.py:371-450; kb-nano has no 4-bit path).
//
// tcgen05.mma kind::mxf4 with block scales multiplies the codes and applies both operands' power-of-two scales itself, one
// per 32 K-values (scale_vec::2X: two scale bytes per row and instruction of K = 64).
//
// At 4 bits the tensor cores eat 93 B/clk and SM of operands from a 128 x 256 tile on one SM, more than L2 delivers (about 64);
// so two SMs share a 256 x 256 tile (cta_group::2): each loads its own 128 rows of A and half of the tile's 256 rows of B, 62
// B/clk.  One K-step is 256 values (128 bytes a row): 32 KB of codes and 3 KB of scales per SM, six steps in the ring.  All
// copies are plain tiled TMA loads into the issuing CTA's own shared memory, counted on the even CTA's barrier.
//
//   many tiles  persistent CTA pairs over the tiles.  The epilogue warps drain the accumulator into registers (128 columns a
//               thread), release it, and convert and store while the next tile's products run.  (Two 256-column accumulators
//               and the scales do not fit the 512 columns of tensor memory.)
//   few tiles   (a few hundred rows or fewer) one tile per cluster of 2 S CTAs, whose S pairs split K.  Each pair owns 256 / S
//               columns and receives the other pairs' partial sums of them as one bulk copy each through the cluster's shared
//               memory; partials are added in slice order, so results are reproducible.
#include "gemm_common.cuh"
#include "mxfp4.cuh"
#include "tensor_map.cuh"

namespace kbn {
namespace mxfp4 {

constexpr int kTileM = 256, kTileN = 256;
constexpr int kStages = 6;                                    // K-steps of 256 values in the ring
constexpr int kABytes = 128 * 128, kBBytes = 128 * 128;      // this CTA's rows of A and of B, one K-step
constexpr int kOperandBytes = kABytes + kBBytes;
constexpr int kSfBytes = 3 * 1024;                            // own A row block, both B row blocks, two 128-K blocks each
constexpr uint32_t kTxPair = 2u * (kOperandBytes + kSfBytes);
constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 32 * (2 + kEpiWarps);
constexpr int kGemmSmem = kStages * (kOperandBytes + kSfBytes) + 1024 + 256;
constexpr int kTmemColumns = 512, kColSfa = 256, kColSfb = 264;      // scale columns: 4 per row block and 128-K block
constexpr int kGroupM = 8;                                     // tile rows that run side by side, for reuse of B in L2

struct GemmArgs {
    const __nv_bfloat16* bias;
    __nv_bfloat16* C;
    int64_t ldc;
    int32_t* status;
    int32_t M, N, kblocks, steps;      // kblocks: 128-K blocks (scales), steps: 256-K steps
    int32_t m_tiles, n_tiles, S;
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
__device__ __forceinline__ void mma_mxf4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}
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

__device__ __forceinline__ void tile_of(int32_t t, const GemmArgs& p, int32_t& m_tile, int32_t& n_tile) {
    const int32_t per_group = kGroupM * p.n_tiles;
    const int32_t grp = t / per_group, first = grp * kGroupM;
    const int32_t size = min(kGroupM, p.m_tiles - first);
    const int32_t in = t - grp * per_group;
    m_tile = first + in % size;
    n_tile = in / size;
}

// 32 accumulator columns of one row (+ bias) -> bf16.
__device__ __forceinline__ void store_row(float (&f)[32], const GemmArgs& p, int32_t row, int32_t n0) {
    if (p.bias != nullptr) {
#pragma unroll
        for (int q = 0; q < 32; ++q)
            if (n0 + q < p.N) f[q] += __bfloat162float(p.bias[n0 + q]);
    }
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

template <bool SPLIT>
__global__ void __launch_bounds__(kGemmThreads, 1)
mxfp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSfa,
                  const __grid_constant__ CUtensorMap tmSfb, const GemmArgs p) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    uint8_t* sf = smem + (size_t)kStages * kOperandBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sf + (size_t)kStages * kSfBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 3);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bar_full = ptx::smem_u32(bars), bar_empty = ptx::smem_u32(bars + kStages);
    const uint32_t bar_tfull = ptx::smem_u32(bars + 2 * kStages), bar_tempty = bar_tfull + 8, bar_xchg = bar_tfull + 16;
    const uint32_t tiles_smem = ptx::smem_u32(smem), sf_smem = ptx::smem_u32(sf);

    const uint32_t rank = ptx::cluster_ctarank();
    const uint32_t pr = rank & 1u, ks = rank >> 1, leader = rank & ~1u;      // place in the pair, K-slice, issuing CTA
    const uint16_t pair_mask = (uint16_t)(3u << leader);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(bar_full + 8 * s, 1);         // armed by the even CTA for both CTAs' copies
            ptx::mbar_init(bar_empty + 8 * s, 1);        // one commit, delivered to both
        }
        ptx::mbar_init(bar_tfull, 1);
        ptx::mbar_init(bar_tempty, 2 * kEpiWarps);       // used in the even CTA: the epilogue warps of both
        ptx::mbar_init(bar_xchg, 1);
        if (SPLIT) ptx::mbar_arrive_expect_tx(bar_xchg, (uint32_t)(p.S - 1) * (uint32_t)(128 * (kTileN / p.S) * 4));
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
        ptx::prefetch_tensormap(&tmA);
        ptx::prefetch_tensormap(&tmB);
        ptx::prefetch_tensormap(&tmSfa);
        ptx::prefetch_tensormap(&tmSfb);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), kTmemColumns);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();              // the partner's barriers exist before anything is sent to them
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Everything this kernel reads, the weights too, may have been written by the kernel before it.
    ptx::grid_dependency_wait();
    ptx::launch_dependents();

    const int32_t tiles = p.m_tiles * p.n_tiles;
    const int32_t cluster = (int32_t)(blockIdx.x / (SPLIT ? 2u * (uint32_t)p.S : 2u));
    const int32_t stride = SPLIT ? tiles : (int32_t)(gridDim.x / 2);          // split: one tile per cluster
    const int32_t per_slice = SPLIT ? (p.steps + p.S - 1) / p.S : p.steps;
    const int32_t k0 = (int32_t)ks * per_slice, k1 = min(p.steps, k0 + per_slice);      // not empty: the host sees to it

    if (warp == 0) {
        if (lane == 0) {
            const WaitCtx w{abort_flag, p.status, 12};
            uint32_t slot = 0, phase = 0;
            bool ok = true;
            for (int32_t t = cluster; ok && t < tiles; t += stride) {
                int32_t mt, nt;
                tile_of(t, p, mt, nt);
                const int32_t row_a = mt * kTileM + (int32_t)pr * 128, row_b = nt * kTileN + (int32_t)pr * 128;
                const int32_t sfa_row = (row_a >> 7) * p.kblocks, sfb_row = (nt * 2) * p.kblocks;
                for (int32_t k = k0; k < k1; ++k) {
                    if (!wait_bar(bar_empty + 8 * slot, phase ^ 1u, w)) { ok = false; break; }
                    if (pr == 0) ptx::mbar_arrive_expect_tx(bar_full + 8 * slot, kTxPair);
                    const uint32_t bar = ptx::mapa(bar_full + 8 * slot, leader);
                    const uint32_t dst = tiles_smem + slot * kOperandBytes, sdst = sf_smem + slot * kSfBytes;
                    ptx::tma_load_2d_pair(dst, &tmA, k * 128, row_a, bar);
                    ptx::tma_load_2d_pair(dst + kABytes, &tmB, k * 128, row_b, bar);
                    // scales: the packed array as rows of 256 bytes, two per 512-byte block
                    ptx::tma_load_2d_pair(sdst, &tmSfa, 0, 2 * (sfa_row + 2 * k), bar);
                    ptx::tma_load_2d_pair(sdst + 1024, &tmSfb, 0, 2 * (sfb_row + 2 * k), bar);
                    ptx::tma_load_2d_pair(sdst + 2048, &tmSfb, 0, 2 * (sfb_row + p.kblocks + 2 * k), bar);
                    if (++slot == kStages) slot = 0, phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && pr == 0) {
            const WaitCtx w{abort_flag, p.status, 13};
            uint32_t slot = 0, phase = 0, acc_phase = 0;
            bool ok = true;
            for (int32_t t = cluster; ok && t < tiles; t += stride, acc_phase ^= 1u) {
                if (!SPLIT) {                 // the accumulator has been drained (passes at once for the first tile)
                    const long long t0 = clock64();
                    while (!try_wait_cluster(bar_tempty, acc_phase ^ 1u)) {
                        if (*abort_flag) { ok = false; break; }
                        if (clock64() - t0 > kWaitLimitCycles) {
                            *abort_flag = 1;
                            atomicCAS(p.status, 0, w.code | (int)(blockIdx.x << 8));
                            ok = false;
                            break;
                        }
                    }
                    if (!ok) break;
                    ptx::tc_fence_after();
                }
                for (int32_t k = k0; k < k1; ++k) {
                    if (!wait_bar(bar_full + 8 * slot, phase, w)) { ok = false; break; }
                    ptx::tc_fence_after();
                    const uint32_t a = tiles_smem + slot * kOperandBytes, s = sf_smem + slot * kSfBytes;
                    const uint64_t a_desc = ptx::umma_desc_k_sw128(a), b_desc = ptx::umma_desc_k_sw128(a + kABytes);
                    const int halves = min(2, p.kblocks - 2 * k);      // the last step may hold one 128-K block only
                    for (int h = 0; h < halves; ++h) {
                        const uint32_t sfa = tmem + kColSfa + 4 * h, sfb = tmem + kColSfb + 8 * h;
                        ptx::tmem_cp_32x128b_warpx4_pair(sfa, ptx::umma_desc_sf(s + 512 * h));
                        ptx::tmem_cp_32x128b_warpx4_pair(sfb, ptx::umma_desc_sf(s + 1024 + 512 * h));
                        ptx::tmem_cp_32x128b_warpx4_pair(sfb + 4, ptx::umma_desc_sf(s + 2048 + 512 * h));
                        mma_mxf4_pair(tmem, a_desc + 4 * h, b_desc + 4 * h, idesc_mxf4(kTileM, kTileN, 0), sfa, sfb, (k > k0 || h > 0) ? 1u : 0u);
                        mma_mxf4_pair(tmem, a_desc + 4 * h + 2, b_desc + 4 * h + 2, idesc_mxf4(kTileM, kTileN, 2), sfa, sfb, 1u);
                    }
                    ptx::mma_commit_pair(bar_empty + 8 * slot, pair_mask);
                    if (++slot == kStages) slot = 0, phase ^= 1u;
                }
                if (ok) ptx::mma_commit_pair(bar_tfull, pair_mask);
            }
        }
    } else if (!SPLIT) {
        const WaitCtx w{abort_flag, p.status, 14};
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t release = ptx::mapa(bar_tempty, leader);
        uint32_t phase = 0;
        for (int32_t t = cluster; t < tiles; t += stride, phase ^= 1u) {
            if (!wait_bar(bar_tfull, phase, w)) break;
            __syncwarp();
            ptx::tc_fence_after();
            int32_t mt, nt;
            tile_of(t, p, mt, nt);
            uint32_t r[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(tmem + ((uint32_t)(quarter * 32) << 16) + half * 128 + c * 32, r[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) ptx::tmem_ld_wait(r[c]);
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(release);
            const int32_t row = mt * kTileM + (int32_t)pr * 128 + quarter * 32 + lane;
            if (row < p.M && *abort_flag == 0) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float f[32];
#pragma unroll
                    for (int q = 0; q < 32; ++q) f[q] = __uint_as_float(r[c][q]);
                    store_row(f, p, row, nt * kTileN + half * 128 + c * 32);
                }
            }
        }
    } else {
        const WaitCtx w{abort_flag, p.status, 15};
        wait_bar(bar_tfull, 0u, w);
        ptx::tc_fence_after();
    }

    if (SPLIT) {
        int32_t mt, nt;
        tile_of(cluster, p, mt, nt);
        const int32_t row0 = mt * kTileM + (int32_t)pr * 128;
        const int32_t live = max(0, min(p.M - row0, 128));
        __syncwarp();
        ptx::cluster_sync();              // every CTA of the cluster is done with its stages: they may be overwritten
        const int W = kTileN / p.S;
        const uint32_t slot_bytes = (uint32_t)(128 * W * 4), units = (uint32_t)W / 4u;
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int r_in_tile = quarter * 32 + lane;
        const uint32_t swz = (uint32_t)r_in_tile & (units - 1u);
        // partial sums of the columns other slices own: rows of W floats, 16-byte units XOR-swizzled by the row so that a
        // lane per row stores without bank conflicts; one bulk copy per owner
        if (warp >= 2) {
#pragma unroll 1
            for (int cc = half; cc < kTileN / 32; cc += 2) {
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
        if (warp >= 2) {
            const WaitCtx w{abort_flag, p.status, 16};
            wait_bar(bar_xchg, 0u, w);
            __syncwarp();
            if (quarter * 32 < live) {
#pragma unroll 1
                for (int cc = half; cc < kTileN / 32; cc += 2) {
                    if ((uint32_t)(32 * cc / W) != ks) continue;
                    uint32_t r[32];
                    ptx::tmem_ld_32x32(tmem + ((uint32_t)(quarter * 32) << 16) + 32 * cc, r);
                    ptx::tmem_ld_wait(r);
                    if (r_in_tile < live && *abort_flag == 0) {
                        float f[32];
#pragma unroll
                        for (int q = 0; q < 32; ++q) f[q] = 0.f;
                        const uint32_t u0 = (uint32_t)(32 * cc % W) / 4u;
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
                        store_row(f, p, row0 + r_in_tile, nt * kTileN + 32 * cc);
                    }
                }
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

// Codes [rows, K]: boxes of 128 rows x 256 values (128 bytes, 128-byte swizzle).
static int code_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t K, bool weights) {
    TensorMapSpec t;
    memset(&t, 0, sizeof(t));
    t.base = base;
    t.rank = 2;
    t.dims[0] = (uint64_t)(K / 2); t.dims[1] = (uint64_t)rows; t.dims[2] = 1;
    t.strides[0] = (uint64_t)(K / 2);
    t.box[0] = 128; t.box[1] = 128; t.box[2] = 1;
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

template <bool SPLIT>
static int max_clusters(int size) {
    static int cache[64][9] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (cache[dev][size] == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(size * 16));
        cfg.blockDim = dim3(kGemmThreads);
        cfg.dynamicSmemBytes = kGemmSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(mxfp4_gemm_kernel<SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, mxfp4_gemm_kernel<SPLIT>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
        }
        cache[dev][size] = n > 0 ? n : -1;
    }
    return cache[dev][size] > 0 ? cache[dev][size] : 0;
}

// K-slices for a problem with too few tiles for one pair each: the most that are resident at once and leave every slice a
// step; 1: persistent pairs.
static int plan_split(const GemmArgs& p) {
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    for (int S = 4; S >= 2; S /= 2) {
        const int per = (p.steps + S - 1) / S;
        if (2 * S * tiles > sm_count() || (S - 1) * per >= p.steps) continue;
        if (tiles <= max_clusters<true>(2 * S)) return S;
    }
    return 1;
}

template <bool SPLIT>
static int launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& sa, const CUtensorMap& sb, const GemmArgs& p, unsigned grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = kGemmSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)(SPLIT ? 2 * p.S : 2);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    KBN_CUDA(cudaLaunchKernelEx(&cfg, mxfp4_gemm_kernel<SPLIT>, a, b, sa, sb, p));
    KBN_CHECK_LAUNCH();
    return KBN_OK;
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
    p.n_tiles = (int32_t)((N + kTileN - 1) / kTileN);
    int rc = gemm_status_ptr(&p.status);
    if (rc != KBN_OK) return rc;
    CUtensorMap a, b, sa, sb;
    if ((rc = code_map(&a, A, M, K, false)) != KBN_OK || (rc = code_map(&b, B, N, K, true)) != KBN_OK || (rc = scale_map(&sa, sfa_packed, M, kblocks)) != KBN_OK ||
        (rc = scale_map(&sb, sfb_packed, N, kblocks)) != KBN_OK)
        return rc;
    p.S = plan_split(p);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    if (p.S > 1) return launch<true>(a, b, sa, sb, p, (unsigned)(tiles * 2 * p.S), st);
    const int pairs = max_clusters<false>(2);
    KBN_REQUIRE(pairs > 0, KBN_ERR_UNSUPPORTED, "kbn_mxfp4_gemm_nt: no CTA pair fits this device");
    return launch<false>(a, b, sa, sb, p, (unsigned)(2 * (tiles < pairs ? tiles : pairs)), st);
}

// Weight streaming for a few activation rows: the core of the MoE layer for a few tokens and of the MXFP4 linear layer
// on at most eight rows.
//
// With at most eight rows (tokens) per weight matrix a product is a weight stream, 2 to 16 flop per weight byte, and what
// counts is that enough weight bytes are in flight on every SM all the time.  One CTA per SM walks a contiguous range of
// units; a unit is 16 (FP8) or 32 (MXFP4) weight rows, in two boxes, over the whole K.  A producer warp keeps a ring of
// 16 KB stages full with 3-D tiled TMA loads (the rows of a box, eight chunks of 128 K-values each, one instruction) and
// the block scales beside them (tiled loads too where their rows allow it, else 4-byte asynchronous copies, which cost the
// one producer warp about as many instructions as everything else); sixteen consumer warps split the chunks, eight per stage.
//
//   product    mma.sync.m16n8k16, f16 x f16 -> fp32: the 16 weight rows are its M, the tokens its N.  (tcgen05 would spend a
//              128-row tile on them and needs its operands in fp8 or fp4; at this intensity the legacy instruction is far
//              from being the bound.)  e4m3 and e2m1 codes are converted to f16 exactly, two per instruction.
//   tokens     held in shared memory as f16, every block of a row (the K-values that share a weight scale: 128 with FP8, 32 with
//              MXFP4) multiplied by a power of two that brings its largest magnitude into [2^14, 2^15); the power is taken out
//              of the block's partial sum.  bf16 has 8 significant bits and f16 has 11, so a value is kept exactly down to
//              2^-32 of its block's largest, and below that to within 2^-39 of it.  One power per block, not per row, so that a
//              row is converted in one pass, without a barrier, and values that the weights' scales make up for are kept.
//              fp32 rows (the MoE layer's activated ones) are held in two pieces, the f16 value and what it leaves, 22 bits: the
//              columns of a product are then up to four tokens and their second pieces, which cost no instruction.
//   scales     FP8: one fp32 factor per 128 x 128 block.  MXFP4: one power of two per row and 32 K-values.  A block's partial
//              sum is multiplied first by the tokens' power, then by the weights' scale, both in fp32.  So that neither step
//              leaves fp32's range where the result does not, the tokens' power lacks a constant factor 2^kLift, which the
//              sums get back at the end: partial sum times power stays below 2^128 (2^31 * 2^(113 - 16) with FP8, 2^23 *
//              2^(113 - 9) with MXFP4), powers go down to fp32's smallest.  Nothing overflows before 2^128, and a zero sum stays
//              zero under any scale; sums below 2^-120 (FP8) and 2^-127 carry fp32's smallest step times 2^kLift.  For MXFP4 that is four multiplications a tile and block more than one power per 128 values
//              behind the blocks' scales, which overflowed from scales of 2^101 on.
//   K order    a dot product does not care: lane t of a quad takes 16 consecutive K-values of a row per load (FP8) or
//              eight (MXFP4), and reads the same K-values of its token.
//   sums       fp32; the warps' partial results meet in shared memory, where two finisher warps (one per buffer, every other
//              unit) add them in warp order (bit-reproducible) and do what the unit's results need, so that no consumer
//              waits for a store, a fence or another consumer.  HALVES (a unit is a single stage, K <= 1024, and so belongs to
//              eight warps): each half of the consumers has a finisher and two buffers of eight partial sums to itself.
//
// Bound: the weights' bytes, once, wherever there are enough units to keep 80 to 190 KB per SM in flight.  One token on 8 of
// 256 experts (FP8, H 7168, I 2048): 352 MB in 76.4 us (all times inside a graph), 4.61 TB/s over the whole layer, 7.0 to 7.5 TB/s
// while the weights stream; 16 tokens: 4.5 GB in 724 us, 95 % of a copy's 6.57 TB/s.  MXFP4 is bound by its conversions (a byte
// holds two codes, a conversion yields two f16 values): 5 tokens on 8 experts (H 4096, I 14336) take 157 us at 52 to 54 % of all
// issue slots, 3.6 TB/s.  Converting with integer shifts and masks instead of cvt was slower (175 -> 224 us, one tile per warp), and
// so were packed fp32 multiplications for the tokens' powers (163.9 -> 166.7).
#pragma once
#include "gemm_common.cuh"
#include "mxfp4.cuh"
#include "tensor_map.cuh"

namespace kbn {
namespace few {

enum WeightFormat : int { kFp8 = 0, kMxfp4 = 1 };

constexpr int kConsumerWarps = 16, kFinishers = 2, kBuffers = 4;      // HALVES uses all four buffers, else the first two
constexpr int kProducerWarp = kConsumerWarps, kFirstFinisher = kConsumerWarps + 1;
constexpr int kThreads = 32 * (kConsumerWarps + 1 + kFinishers);
constexpr int kStageBytes = 16384;                        // two boxes of 8 KB
constexpr int kMaxGroup = 8;                              // tokens per job: the N of the matrix instruction
constexpr int kPieceGroup = kMaxGroup / 2;                // tokens per job whose rows are held in two pieces
constexpr int kMaxTokens = 16, kMaxTopk = 16, kMaxPairs = kMaxTokens * kMaxTopk;
constexpr int kMaxStages = 12;
constexpr int kMinStages = 5;                             // 80 KB in flight per SM: what 6.5 TB/s needs at about 1.5 us

constexpr int kChunks = 8;                                // 128-K chunks per stage, one consumer warp each

template <int FMT>
struct Fmt;
template <>
struct Fmt<kFp8> {
    static constexpr int kTiles = 1;                      // 16-row tiles of the matrix instruction per unit
    static constexpr int kChunkBytes = 128, kScaleBytes = 512, kTokenPad = 16;
    static constexpr int kBlock = 128, kLift = 16;        // K-values that share a weight scale; sums are held times 2^-kLift
};
template <>
struct Fmt<kMxfp4> {
    static constexpr int kTiles = 2;                      // half the bytes a row: two tiles share a warp's token loads and waits
    static constexpr int kChunkBytes = 64, kScaleBytes = 1024, kTokenPad = 64;
    static constexpr int kBlock = 32, kLift = 9;
};
template <int FMT>
constexpr int kBoxRows = 8 * Fmt<FMT>::kTiles;            // rows of each of a unit's two boxes
// Bytes of a token row's powers: an fp32 per block.  MXFP4 reads four at once; 16 bytes more keep a warp's rows on different banks.
template <int FMT>
__host__ __device__ constexpr int64_t power_bytes(int64_t K) { return K / Fmt<FMT>::kBlock * 4 + (FMT == kMxfp4 ? 16 : 0); }
template <int FMT>
constexpr int kRedBytes = kFinishers * kConsumerWarps * 128 * Fmt<FMT>::kTiles * 4;

// Where a weight matrix's scales lie.  FP8: fp32 [rows / 128, KC].  MXFP4: one 32-bit word per row and chunk, row-major
// (word (row, c) at row * KC + c) or, PACKED, in the packed layout of the tensor core.
// MXFP4 row-major scales with 16-byte row strides (K % 512 == 0) also have a tensor map (boxes of 16 rows x 32 bytes, 32-byte
// swizzle).  In the ring a stage's word (row of 32, chunk) is always where that box puts it, see scale_word().
struct ScaleSource {
    const void* base;
    const CUtensorMap* map;      // null: asynchronous copies
};
__device__ __forceinline__ uint32_t scale_word(int row, int chunk) {      // byte offset; no bank conflicts over eight rows
    return (uint32_t)(row * 32 + ((((chunk >> 2) ^ (row >> 2)) & 1) << 4) + (chunk & 3) * 4);
}

struct Smem {
    uint8_t* ring;         // stages, 1024-byte aligned
    uint8_t* scales;       // one area per stage
    uint8_t* tokens;       // f16 rows, stride token_stride
    float* token_scales;   // a row of power_bytes each: what the blocks' partial sums are multiplied by
    float* red;            // 32 x 128 partial sums (times tiles): two buffers of 16 warps or four of 8
    uint64_t* bars;        // full[stages], empty[stages], partials full[kBuffers], partials empty[kBuffers]
    int32_t stages;
};

__device__ __forceinline__ void mma_f16_m16n8k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with a zero C operand, so that a fresh partial sum costs no register moves.
__device__ __forceinline__ void mma_f16_m16n8k16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Four e4m3 bytes -> two packed f16 pairs.  Exact.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, int32_t x, int32_t y, int32_t z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival on `bar` once this thread's earlier cp.async copies have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumerWarps) : "memory"); }

// Bounded wait of a warp on one of this file's barriers.  The hint lets the hardware keep the warp suspended for longer than
// its default, so that waiting warps take fewer issue slots from working ones.
__device__ __forceinline__ void wait_ring(uint32_t bar, uint32_t parity, const WaitCtx& w) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (!ok) wait_bar(bar, parity, w);
}

// Ring position, advanced one stage at a time.
struct RingPos {
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void advance(uint32_t stages) {
        if (++slot == stages) {
            slot = 0;
            phase ^= 1u;
        }
    }
};

// A consumer warp's place in the ring: its next slot (one of its half's), and how many stages ahead of the current unit's
// first that is.
struct OwnPos {
    uint32_t slot, phase;
    int32_t ahead;
    __device__ __forceinline__ explicit OwnPos(int warp) : slot((uint32_t)warp >> 3), phase(0), ahead(warp >> 3) {}
    __device__ __forceinline__ void advance(uint32_t stages) {      // two on, or to the first of the half's slots in the next lap
        const uint32_t half = slot & 1u, next = slot + 2u;
        if (next < stages) {
            slot = next;
            ahead += 2;
        } else {
            ahead += (int32_t)(stages - slot + half);
            slot = half;
            phase ^= 1u;
        }
    }
};

template <bool HALVES = false>
__device__ __forceinline__ void init_ring(const Smem& s) {
    for (int i = 0; i < s.stages; ++i) {
        ptx::mbar_init(ptx::smem_u32(s.bars + i), 1 + 32);                    // the producer's bytes, its 32 lanes' scale copies
        ptx::mbar_init(ptx::smem_u32(s.bars + s.stages + i), kChunks);
    }
    for (int i = 0; i < kBuffers; ++i) {
        ptx::mbar_init(ptx::smem_u32(s.bars + 2 * s.stages + i), HALVES ? 8 : kConsumerWarps);
        ptx::mbar_init(ptx::smem_u32(s.bars + 2 * s.stages + kBuffers + i), 1);
    }
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
}

// Producer warp: all stages of one unit's chunks c_begin (a multiple of kChunks) .. c_end - 1 (up to a multiple, or KC).
// row_a, row_b: first rows of the two boxes (in rows of the tensor map; a box past the last row is filled with zeros by the
// TMA).  n_rows: rows the scale array covers.
template <int FMT, bool PACKED = false>
__device__ __forceinline__ void produce_unit(const Smem& s, RingPos& pos, const void* tmap, const ScaleSource& sc, int32_t row_a, int32_t row_b,
                                             int32_t n_rows, int32_t KC, int32_t c_begin, int32_t c_end, int lane, const WaitCtx& w) {
    using F = Fmt<FMT>;
    for (int32_t c0 = c_begin; c0 < c_end; c0 += kChunks) {
        const uint32_t full = ptx::smem_u32(s.bars + pos.slot), empty = ptx::smem_u32(s.bars + s.stages + pos.slot);
        wait_ring(empty, pos.phase ^ 1u, w);
        const uint32_t dst = ptx::smem_u32(s.ring) + pos.slot * kStageBytes;
        const uint32_t sdst = ptx::smem_u32(s.scales) + pos.slot * F::kScaleBytes;
        const bool tiled = FMT == kMxfp4 && !PACKED && sc.map != nullptr;
        if (lane == 0) {
            ptx::mbar_arrive_expect_tx(full, tiled ? kStageBytes + F::kScaleBytes : kStageBytes);
            tma_load_3d(dst, tmap, 0, row_a, c0, full);
            tma_load_3d(dst + kStageBytes / 2, tmap, 0, row_b, c0, full);
            if (tiled) {
                ptx::tma_load_2d(sdst, sc.map, c0 * 4, row_a, full);
                ptx::tma_load_2d(sdst + F::kScaleBytes / 2, sc.map, c0 * 4, row_b, full);
            }
        }
        if (FMT == kFp8) {
            // lane = 8 * box + chunk
            const int32_t c = c0 + (lane & 7);
            if (lane < 16 && c < KC) {
                const int32_t row = lane < 8 ? row_a : row_b;
                cp_async4(sdst + lane * 4, static_cast<const float*>(sc.base) + (int64_t)(row >> 7) * KC + c);
            }
        } else if (!tiled) {
            // a row per lane, eight words each
            const int32_t row = min((lane < 16 ? row_a : row_b - 16) + lane, n_rows - 1);
            const uint32_t* src = static_cast<const uint32_t*>(sc.base) + (PACKED ? (int64_t)mxfp4::packed_word(row, c0, KC) : (int64_t)row * KC + c0);
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
                if (c0 + i < KC) cp_async4(sdst + scale_word(lane, i), src + i * (PACKED ? 128 : 1));
        }
        cp_async_arrive(full);
        pos.advance((uint32_t)s.stages);
    }
}

// What a consumer lane reads of the tokens: the f16 row of column g, the powers of columns 2t and 2t + 1 (shared-memory
// addresses).  Columns without a token repeat the last one's; nothing reads their results.
struct TokenColumns {
    uint32_t row, scale0, scale1;
};
template <int FMT, typename RowOf>
__device__ __forceinline__ TokenColumns token_columns(const Smem& s, uint32_t stride, int32_t KC, int count, int lane, RowOf row_of) {
    const int g = min(lane >> 2, count - 1), t0 = min(2 * (lane & 3), count - 1), t1 = min(2 * (lane & 3) + 1, count - 1);
    const uint32_t powers = ptx::smem_u32(s.token_scales), row_bytes = (uint32_t)power_bytes<FMT>(128 * (int64_t)KC);
    return TokenColumns{ptx::smem_u32(s.tokens) + (uint32_t)row_of(g) * stride, powers + (uint32_t)row_of(t0) * row_bytes, powers + (uint32_t)row_of(t1) * row_bytes};
}

// The same of up to four rows in two pieces, row r's second one in row count + r: columns 4 to 7 are the second pieces of 0 to 3.
template <int FMT>
__device__ __forceinline__ TokenColumns piece_columns(const Smem& s, uint32_t stride, int32_t KC, int count, int lane) {
    const int g = lane >> 2, t = 2 * (lane & 1), row = min(g & (kPieceGroup - 1), count - 1) + (g < kPieceGroup ? 0 : count);
    const uint32_t powers = ptx::smem_u32(s.token_scales), row_bytes = (uint32_t)power_bytes<FMT>(128 * (int64_t)KC);
    return TokenColumns{ptx::smem_u32(s.tokens) + (uint32_t)row * stride, powers + (uint32_t)min(t, count - 1) * row_bytes,
                        powers + (uint32_t)min(t + 1, count - 1) * row_bytes};
}

// Consumer warp: its chunks of one unit, added to acc.  acc[i][0..1]: row 8 i + g of box 0 with tokens 2t, 2t + 1; acc[i][2..3]:
// row 8 i + g of box 1.  A stage has work for eight warps: slots with an even number belong to warps 0-7, the others to warps
// 8-15.  A slot must always have the same readers: a warp may only test a barrier for a phase if it has seen the phase
// before it complete, because the test tells two phases apart by their parity alone.
template <int FMT>
__device__ __forceinline__ void consume_unit(const Smem& s, OwnPos& here, int32_t KC, int warp, int lane, const TokenColumns& tc,
                                             float (&acc)[Fmt<FMT>::kTiles][4], const WaitCtx& w) {
    using F = Fmt<FMT>;
    const int g = lane >> 2, t = lane & 3, cw = warp & 7;
    const int32_t n = (KC + kChunks - 1) / kChunks;
    for (; here.ahead < n; here.advance((uint32_t)s.stages)) {
        wait_ring(ptx::smem_u32(s.bars + here.slot), here.phase, w);
        const int32_t c = here.ahead * kChunks + cw;
        if (c < KC) {
            const uint32_t box0 = ptx::smem_u32(s.ring) + here.slot * kStageBytes + (uint32_t)(cw * kBoxRows<FMT> + g) * F::kChunkBytes;
            const uint32_t box1 = box0 + kStageBytes / 2;
            const uint32_t sdst = ptx::smem_u32(s.scales) + here.slot * F::kScaleBytes;
            if constexpr (FMT == kFp8) {
                const float x0s = __uint_as_float(lds32(tc.scale0 + (uint32_t)c * 4u)), x1s = __uint_as_float(lds32(tc.scale1 + (uint32_t)c * 4u));
                float p[4], q[4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t piece = (uint32_t)(t + 4 * j);
                    const uint4 wa = lds128(box0 + ((piece ^ (uint32_t)g) << 4)), wb = lds128(box1 + ((piece ^ (uint32_t)g) << 4));
                    const uint32_t ta = tc.row + (uint32_t)(c * 128 + (int)piece * 16) * 2u;
                    const uint4 x0 = lds128(ta), x1 = lds128(ta + 16);
                    uint32_t a0, a1, a2, a3;
                    e4m3x4_to_f16(wa.x, a0, a2); e4m3x4_to_f16(wb.x, a1, a3);
                    if (j == 0) mma_f16_m16n8k16_first(p, a0, a1, a2, a3, x0.x, x0.y);
                    else mma_f16_m16n8k16(p, a0, a1, a2, a3, x0.x, x0.y);
                    e4m3x4_to_f16(wa.y, a0, a2); e4m3x4_to_f16(wb.y, a1, a3);
                    if (j == 0) mma_f16_m16n8k16_first(q, a0, a1, a2, a3, x0.z, x0.w);
                    else mma_f16_m16n8k16(q, a0, a1, a2, a3, x0.z, x0.w);
                    e4m3x4_to_f16(wa.z, a0, a2); e4m3x4_to_f16(wb.z, a1, a3);
                    mma_f16_m16n8k16(p, a0, a1, a2, a3, x1.x, x1.y);
                    e4m3x4_to_f16(wa.w, a0, a2); e4m3x4_to_f16(wb.w, a1, a3);
                    mma_f16_m16n8k16(q, a0, a1, a2, a3, x1.z, x1.w);
                }
                const float s0 = __uint_as_float(lds32(sdst + cw * 4)), s1 = __uint_as_float(lds32(sdst + 32 + cw * 4));
                acc[0][0] = fmaf((p[0] + q[0]) * x0s, s0, acc[0][0]);
                acc[0][1] = fmaf((p[1] + q[1]) * x1s, s0, acc[0][1]);
                acc[0][2] = fmaf((p[2] + q[2]) * x0s, s1, acc[0][2]);
                acc[0][3] = fmaf((p[3] + q[3]) * x1s, s1, acc[0][3]);
            } else {
                const uint32_t w0 = box0 + (uint32_t)(((g >> 1) & 3) << 4) + (uint32_t)t * 4u;      // 16-byte piece b of the row at w0 ^ 16 b
                const uint32_t xa = tc.row + (uint32_t)(c * 128 + t * 8) * 2u;
                uint32_t sw[F::kTiles][2];        // tile, box: four scale bytes
#pragma unroll
                for (int i = 0; i < F::kTiles; ++i)
#pragma unroll
                    for (int box = 0; box < 2; ++box) sw[i][box] = lds32(sdst + scale_word(8 * i + g, cw) + box * 512);
                const uint4 v0 = lds128(tc.scale0 + (uint32_t)c * 16u), v1 = lds128(tc.scale1 + (uint32_t)c * 16u);
                const uint32_t x0s[4] = {v0.x, v0.y, v0.z, v0.w}, x1s[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int pair = 0; pair < 2; ++pair) {
                    uint32_t e[F::kTiles][2];
#pragma unroll
                    for (int i = 0; i < F::kTiles; ++i)
#pragma unroll
                        for (int box = 0; box < 2; ++box) {
                            e[i][box] = mxfp4::scale_bf16x2(sw[i][box]);
                            sw[i][box] >>= 16;
                        }
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t at = w0 ^ (uint32_t)(32 * pair + 16 * b);
                        const uint4 x = lds128(xa + 64 * b + 128 * pair);
#pragma unroll
                        for (int i = 0; i < F::kTiles; ++i) {
                            uint32_t ha[4], hb[4];
                            mxfp4::unpack_e2m1x8(lds32(at + i * 8 * F::kChunkBytes), ha);
                            mxfp4::unpack_e2m1x8(lds32(at + i * 8 * F::kChunkBytes + kStageBytes / 2), hb);
                            float p[4];
                            mma_f16_m16n8k16_first(p, ha[0], hb[0], ha[1], hb[1], x.x, x.y);
                            mma_f16_m16n8k16(p, ha[2], hb[2], ha[3], hb[3], x.z, x.w);
                            const float s0 = b & 1 ? bf16_hi(e[i][0]) : bf16_lo(e[i][0]);
                            const float s1 = b & 1 ? bf16_hi(e[i][1]) : bf16_lo(e[i][1]);
                            const float t0 = __uint_as_float(x0s[2 * pair + b]), t1 = __uint_as_float(x1s[2 * pair + b]);
                            acc[i][0] = fmaf(p[0] * t0, s0, acc[i][0]);
                            acc[i][1] = fmaf(p[1] * t1, s0, acc[i][1]);
                            acc[i][2] = fmaf(p[2] * t0, s1, acc[i][2]);
                            acc[i][3] = fmaf(p[3] * t1, s1, acc[i][3]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(s.bars + s.stages + here.slot));
    }
    here.ahead -= n;
}

// Consumer warp: its partial sums of its n-th unit to a finisher; per tile element (row of 16) * 8 + token, rows 0-7 box 0's,
// rows 8-15 box 1's.  Each buffer always has the same writers, for the reason given above.
template <bool HALVES = false, int TILES>
__device__ __forceinline__ void hand_over(const Smem& s, uint32_t n, int warp, int lane, const float (&acc)[TILES][4], const WaitCtx& w) {
    const int buf = (int)(n & 1u) + (HALVES ? 2 * (warp >> 3) : 0);
    wait_ring(ptx::smem_u32(s.bars + 2 * s.stages + kBuffers + buf), (n >> 1 & 1u) ^ 1u, w);
    float* r = s.red + (HALVES ? buf * 8 + (warp & 7) : buf * kConsumerWarps + warp) * (128 * TILES);
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        *reinterpret_cast<float2*>(r + i * 128 + g * 8 + 2 * t) = make_float2(acc[i][0], acc[i][1]);
        *reinterpret_cast<float2*>(r + i * 128 + (g + 8) * 8 + 2 * t) = make_float2(acc[i][2], acc[i][3]);
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(s.bars + 2 * s.stages + buf));
}
// HALVES: whose unit is the one at this ring slot (0: warps 0-7, 1: warps 8-15).  The finishers follow the ring with a RingPos.
__device__ __forceinline__ int half_of(const RingPos& pos) { return (int)(pos.slot & 1u); }
// Finisher: the sums of its n-th unit.  Lane l receives, of each tile, row l / 2, tokens 4 (l % 2) .. + 3.
template <int FMT, bool HALVES = false>
__device__ __forceinline__ void take_over(const Smem& s, int finisher, uint32_t n, int lane, float (&v)[Fmt<FMT>::kTiles][4], const WaitCtx& w) {
    constexpr int TILES = Fmt<FMT>::kTiles;
    constexpr float kUnlift = (float)(1 << Fmt<FMT>::kLift);
    constexpr int kPartials = HALVES ? 8 : kConsumerWarps;
    const int buf = HALVES ? 2 * finisher + (int)(n & 1u) : finisher;
    wait_ring(ptx::smem_u32(s.bars + 2 * s.stages + buf), (HALVES ? n >> 1 : n) & 1u, w);
    const float4* r = reinterpret_cast<const float4*>(s.red + buf * kPartials * (128 * TILES)) + lane;
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
#pragma unroll
        for (int j = 0; j < kPartials; ++j) {
            const float4 p = r[(j * TILES + i) * 32];
            v[i][0] += p.x; v[i][1] += p.y; v[i][2] += p.z; v[i][3] += p.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] *= kUnlift;
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(s.bars + 2 * s.stages + kBuffers + buf));
}
// Row of a unit, counted over its two boxes, that lane l's value of tile i belongs to.
template <int FMT>
__device__ __forceinline__ int row_of_lane(int tile, int lane) {
    const int r = lane >> 1;
    return 8 * tile + (r & 7) + (r >> 3) * kBoxRows<FMT>;
}

// x * 2^e for |e| up to 254, in two exact steps (one factor alone may leave fp32's range).
__device__ __forceinline__ float scale_pow2(float x, int e) {
    const int h = e >> 1;
    return x * __uint_as_float((uint32_t)(h + 127) << 23) * __uint_as_float((uint32_t)(e - h + 127) << 23);
}
// Exponent that brings the largest finite magnitude (fp32 bit pattern) of some values into [2^14, 2^15); 0 if all are zero.
__device__ __forceinline__ int token_exponent(uint32_t amax_bits) {
    if (amax_bits == 0u) return 0;
    int e = (int)(amax_bits >> 23) - 127;
    if (amax_bits < 0x00800000u) e = -118 - __clz((int)amax_bits);      // subnormal: 2^(31 - clz - 149)
    return 14 - e;
}

// Rows of K values -> f16 rows and the blocks' powers in shared memory, normalised as described above, by NT threads.  T: fp32 or
// bf16; fp32 rows leave two f16 rows each, the second pieces in rows n to 2n - 1.  row_ptr(i): row i < n, 16-byte aligned.  No
// barrier inside: the caller sees to it that nobody reads the rows that are replaced, and publishes the new ones.  BATCH vectors
// of eight are under way at once in every thread; no more, because a CTA comes here once or twice and fetches the unrolled code
// from L2 (BATCH 8 and 4 to 4 and 1: one token of 256 experts 78.7 -> 76.4 us, 16 tokens 739 -> 723).
template <int FMT, typename T, int NT, typename RowPtr>
__device__ __forceinline__ void load_tokens(const Smem& s, uint32_t stride, int n, int K, RowPtr row_ptr, int tid) {
    constexpr int kTeam = Fmt<FMT>::kBlock / 8;   // consecutive threads that share a block of a row: K % 128 == 0
    constexpr int kMaxExponent = 149 - Fmt<FMT>::kLift;      // so that a power is never below fp32's smallest value
    const uint32_t row_powers = (uint32_t)power_bytes<FMT>(K) / 4u;
    constexpr int W = sizeof(T) / 2;              // 16-byte loads per eight values
    constexpr int BATCH = W == 2 ? 1 : 4;
    const uint32_t vecs = (uint32_t)K / 8u;
    const uint32_t total = (uint32_t)n * vecs;
    const uint32_t magic = 0xffffffffu / vecs + 1u;      // i / vecs == umulhi(i, magic): i * vecs < 2^32 here
    for (uint32_t i0 = 0; i0 < total; i0 += BATCH * NT) {
        uint4 u[BATCH][W];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const uint32_t i = i0 + (uint32_t)(k * NT + tid), row = __umulhi(i, magic);
            if (i < total) {
                const uint4* p = reinterpret_cast<const uint4*>(row_ptr((int)row)) + (size_t)(i - row * vecs) * W;
#pragma unroll
                for (int j = 0; j < W; ++j) u[k][j] = __ldcg(p + j);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) u[k][j] = make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const uint32_t i = i0 + (uint32_t)(k * NT + tid), row = __umulhi(i, magic), v = i - row * vecs;
            if (i0 + (uint32_t)(k * NT) >= total) break;      // whole warps
            float f[8];
            const uint32_t w[4] = {u[k][0].x, u[k][0].y, u[k][0].z, u[k][0].w}, w2[4] = {u[k][W - 1].x, u[k][W - 1].y, u[k][W - 1].z, u[k][W - 1].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[W == 1 ? 2 * j : j] = W == 1 ? bf16_lo(w[j]) : __uint_as_float(w[j]);
                f[W == 1 ? 2 * j + 1 : j + 4] = W == 1 ? bf16_hi(w[j]) : __uint_as_float(w2[j]);
            }
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = __float_as_uint(f[j]) & 0x7fffffffu;
                m = max(m, b < 0x7f800000u ? b : 0u);         // infinities and NaNs keep their place, the finite values set the scale
            }
#pragma unroll
            for (int o = kTeam / 2; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (i < total) {
                const int e = min(token_exponent(m), kMaxExponent);
                uint32_t h[4], l[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float a = scale_pow2(f[2 * j], e), b = scale_pow2(f[2 * j + 1], e);
                    const __half2 p = __floats2half2_rn(a, b);
                    h[j] = *reinterpret_cast<const uint32_t*>(&p);
                    if constexpr (sizeof(T) == 4) {           // what is left is at most 8; fminf: an infinity's would be a NaN, 16 does no harm beside it
                        const float ra = a - __low2float(p), rb = b - __high2float(p);
                        const __half2 r = __floats2half2_rn(fminf(ra, 16.0f), fminf(rb, 16.0f));
                        l[j] = *reinterpret_cast<const uint32_t*>(&r);
                    }
                }
                *reinterpret_cast<uint4*>(s.tokens + (size_t)row * stride + (size_t)v * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(s.tokens + (size_t)(row + n) * stride + (size_t)v * 16) = make_uint4(l[0], l[1], l[2], l[3]);
                if ((tid & (kTeam - 1)) == 0) s.token_scales[row * row_powers + v / kTeam] = scale_pow2(1.0f, -e - Fmt<FMT>::kLift);
            }
        }
    }
}

constexpr int kSmemMax = 232448;      // shared memory a CTA may ask for

// Lets a kernel use all of an SM's shared memory; asked of the driver once per kernel and device.
template <typename Kernel>
static int allow_smem(Kernel kernel, std::atomic<uint64_t>& done) {
    int dev = 0;
    KBN_CUDA(cudaGetDevice(&dev));
    KBN_REQUIRE(dev >= 0 && dev < 64, KBN_ERR_UNSUPPORTED, "device ordinal %d out of range", dev);
    if (done.load(std::memory_order_acquire) >> dev & 1u) return KBN_OK;
    KBN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax));
    done.fetch_or(1ull << dev, std::memory_order_release);
    return KBN_OK;
}

// Weight matrix [rows, K] as (chunk, row, chunk number): one box is kBoxRows rows of kChunks chunks, each chunk's rows side by
// side and swizzled, so that a warp reading one chunk of eight rows touches every bank once.
template <int FMT>
static int weight_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t K) {
    using F = Fmt<FMT>;
    TensorMapSpec t;
    memset(&t, 0, sizeof(t));
    const uint64_t row_bytes = (uint64_t)(FMT == kFp8 ? K : K / 2);
    t.base = base;
    t.rank = 3;
    t.dims[0] = F::kChunkBytes; t.dims[1] = (uint64_t)rows; t.dims[2] = (uint64_t)(K / 128);
    t.strides[0] = row_bytes; t.strides[1] = F::kChunkBytes;
    t.box[0] = F::kChunkBytes; t.box[1] = kBoxRows<FMT>; t.box[2] = kChunks;
    t.swizzle = FMT == kFp8 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    t.promo = CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
    return encode_tensor_map(tm, t);
}

// Row-major MXFP4 scales [rows, K / 32]; only with K % 512 == 0.
static int scale_rows_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t K) {
    TensorMapSpec t;
    memset(&t, 0, sizeof(t));
    t.base = base;
    t.rank = 2;
    t.dims[0] = (uint64_t)(K / 32); t.dims[1] = (uint64_t)rows; t.dims[2] = 1;
    t.strides[0] = (uint64_t)(K / 32);
    t.box[0] = 4 * kChunks; t.box[1] = kBoxRows<kMxfp4>; t.box[2] = 1;
    t.swizzle = CU_TENSOR_MAP_SWIZZLE_32B;
    t.promo = CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
    return encode_tensor_map(tm, t);
}

}  // namespace few
}  // namespace kbn

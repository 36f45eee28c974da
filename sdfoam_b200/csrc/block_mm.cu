// out = (a * a_scales) (b * b_scales)^T + bias: the product of two e4m3
// matrices with a scale per block of 128 along the reduction.
//
//   out[m, n] = sum over blocks j of 128 of  sa[m, j] sb[n, j] * (sum over k in j of a[m, k] b[n, k])  + bias[n]
//
// The inner sum runs on the tensor cores (tcgen05.mma kind::f8f6f4, fp32
// accumulation in TMEM); the scales differ from block to block, so each
// block's 128-wide product is read back from TMEM and added, times its scale,
// to fp32 sums in registers, whatever the scales' sizes (scale_factors).  A persistent CTA per SM walks units of (tile of
// 128 x TN, slice of the reduction):
//   * warp 0 (one lane) streams 128-byte wide tiles of both operands through
//     a ring with TMA (128-byte swizzle; rows and columns past the ends read
//     as zero);
//   * warp 1 (one lane) issues four MMAs (K 32 each) per block into the next
//     of the TMEM accumulators, releasing ring stages and finished
//     accumulators with tcgen05.commit;
//   * warps 2 and 3 bring the blocks' scales of the tile's rows of P and of Q
//     into a ring of their own (cp.async), several blocks ahead;
//   * warps 4-11 read the accumulators back (warp w: TMEM lanes 32 (w % 4)
//     .., half of the TN columns; one row per thread) and multiply-add them
//     into registers while the tensor cores fill the next accumulator.  Their
//     sums take the registers that the first four warps give up.
//
// The operand with the rows on the TMEM lanes is P, the other Q.  Q is b
// unless a has few rows (a single token to 64): then a's rows are the narrow
// side, so that a weight is read once with 128 of its rows per tile and TN
// columns of tokens.  When the tiles do not fill the GPU, the reduction is
// cut into slices, whose fp32 sums are added in order (no atomics: the same
// bits every run): up to 8 slices of a narrow tile are a cluster that adds
// them through its shared memory, otherwise they go to the workspace and a
// second launch adds them.
//
// What bounds it.  Small reductions (sites x 256): HBM -- 1048576 x 256 x 256
// in 135 us, 6.0 TB/s, 1048577 x 217 x 256 with a bias in 173 (162 without).
// Large products: the pass over the accumulators between two blocks.  In short
// runs 8192^3 takes 399 us when the tensor cores add up the whole reduction
// (2750 TFLOP/s), 427 with an accumulator per block that nobody reads, and 510
// with the scaled sums (2150); back to back, at the power limit, 589 (1870).
// TMEM holds two accumulators of a 256-column tile, so the MMAs of a block
// wait for the reads of the block before last.  A CTA pair halves the operand
// bytes per SM (one CTA per tile, short runs: 565 us).  No kernel spills.
//
// Every wait is bounded: a CTA that gives up sets *error, writes NaN, waits
// (bounded) for its own copies and MMAs and frees its TMEM.  No TMA multicast.
#include <algorithm>
#include <cfloat>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "foam_internal.h"
#include "tcgen05.cuh"

namespace sdfoam_b200 {

namespace {

constexpr int kSms = 148;
constexpr int kTileP = 128;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (4 + kEpiWarps);
// Registers: launched with 168 each (384 threads), the first four warps keep
// 56 and the others grow to 224: 128 x 56 + 256 x 224 = 384 x 168.
constexpr int kControlRegs = 56, kEpiRegs = 224;
constexpr int kBlockK = 128;  // bytes of a row per stage: one swizzle span, one block of scales
constexpr uint32_t kPBytes = kTileP * kBlockK;  // 16 KB
constexpr int kSwizzleTiles = 16;               // tiles of P that are walked together (L2)

// TN columns of Q per tile, shared by the CTAs of a pair: ring stages that
// fit, TMEM accumulators, the epilogue's staging.
template <int TN, bool PAIR>
struct Shape {
    static constexpr int kCtas = PAIR ? 2 : 1;
    static constexpr uint32_t kQBytes = TN / kCtas * kBlockK;
    static constexpr uint32_t kStageBytes = kPBytes + kQBytes;  // per CTA
    static constexpr int kStages = TN == 256 ? 4 : TN == 128 ? 5 : TN == 64 ? 7 : 8;
    static constexpr int kAccs = TN == 256 ? 2 : 4;
    static constexpr uint32_t kTmemCols = uint32_t(TN) * kAccs;
    static constexpr int kGroups = 2, kCols = TN / kGroups;  // groups of four epilogue warps, their columns
    // per epilogue warp: its 32 rows x kCols columns of 16 bits, at least a box of 32 x 128 bytes
    static constexpr uint32_t kBoxBytes = kCols < 32 ? 0 : kCols == 128 ? 8192 : 4096;
    static constexpr int kScaleStages = 8;
    static constexpr uint32_t kScaleFloats = kTileP + TN;  // of a block: P's rows, Q's rows
    static constexpr uint32_t kSmem =
        kStages * kStageBytes + kEpiWarps * kBoxBytes + (kScaleStages * kScaleFloats + TN) * 4 + 512 + 1024;
    static_assert(kSmem <= 232448, "shared memory of a block");
    static_assert((2 * kStages + 2 * kAccs + 2 * kScaleStages + 1) * 8 + 4 <= 512, "room for the barriers");
};

// How a tile's rows reach out.
enum : int {
    kStoreRows,  // element by element, consecutive lanes on consecutive columns
    kStoreBox,   // TMA boxes of 32 rows x 128 bytes: rows of out are 16-byte aligned
    kStoreSpan,  // one tile covers whole contiguous rows, both groups: 32 rows are one bulk copy
};

struct BlockParams {
    uint32_t p_rows, q_rows;
    uint32_t tiles_p, tiles_q;
    uint32_t k_blocks, splits, units;
    const float *p_scales, *q_scales;  // of row r and block j: scales[(r >> shift) * row + j * block]
    int p_shift, q_shift;              // 0 or 7: rows per scale as a power of two
    uint64_t p_scale_row, p_scale_block, q_scale_row, q_scale_block;
    const void *bias;                  // over b's rows (n), or null
    uint32_t bias_dtype;
    void *out;                         // [m, n]
    uint64_t ldo;
    uint32_t out_dtype;
    int store;
    float4 *parts;                     // splits > 1: sums of the slices
    int cluster_join;                  // splits > 1: a tile's slices are a cluster, joined in it
    int *error;
};

// tcgen05 instruction descriptor, kind::f8f6f4: D fp32 (bits 4-5 = 1), A and
// B e4m3 (0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
template <int N, bool PAIR>
__device__ __forceinline__ constexpr uint32_t idesc() {
    return (1u << 4) | (uint32_t(N >> 3) << 17) | (uint32_t((PAIR ? 2 * kTileP : kTileP) >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t id,
                                         uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(id), "r"(accumulate));
    else
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(id), "r"(accumulate));
}

// An arrival at the barrier of both CTAs of the pair (the same place in
// their shared memory), or of the one CTA, when the MMAs so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit_to_all(uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                bar),
            "h"(uint16_t(3))
            : "memory");
    else
        mma_commit(bar);
}

// A pair's copies complete on the first CTA's barrier (bit 24 of a shared
// address is the rank in the pair).
template <bool PAIR>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
            "%3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar & 0xfeffffffu)
            : "memory");
    else
        tma_load_2d(dst, map, x, y, bar);
}

// An arrival at the first CTA's barrier.  Relaxed: what it orders are reads of
// TMEM, which the tcgen05 fence before it covers; a release at cluster scope
// waits for every other access too (8192^3: 1084 us with it, 524 without).
template <bool PAIR>
__device__ __forceinline__ void arrive_at_first(uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "{\n"
            ".reg .b32 a;\n"
            "mapa.shared::cluster.u32 a, %0, 0;\n"
            "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n"
            "}\n" ::"r"(bar)
            : "memory");
    else
        mbar_arrive(bar);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Consecutive columns of the warp's 32 lanes; the values may be used after
// tmem_wait, which names them so that no use moves before it.
__device__ __forceinline__ void tmem_load(uint32_t (&r)[8], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(addr));
}
// 16 lanes x 16 columns: thread t holds columns 2 (t % 4) and + 1 of rows t / 4
// (r[0], r[1]) and t / 4 + 8 (r[2], r[3]), and of the columns 8 further (r[4..7]).
__device__ __forceinline__ void tmem_load_patch(uint32_t (&r)[8], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8]) {
    asm volatile(
        "tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
        :
        : "memory");
}

// Two fp32 lanes in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 unpair(uint64_t d) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(d));
    return f;
}
__device__ __forceinline__ void fma_pair(uint64_t &acc, uint64_t x, uint64_t s) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(x), "l"(s));
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// A sum x of a block is 0 or from 2^-18 to 2^25 in size.  Its scaled value
// x * p * q may be a number of fp32 (or zero) where a step on the way, p * q or
// x * q, is not: there it is multiplied by two factors that share the exponent.

// Whether p * q leaves fp32's normal numbers, with neither zero, infinite or NaN.
__device__ __forceinline__ bool product_leaves(float p, float q) {
    const float size = fabsf(__fmul_rn(p, q));
    return !(size >= FLT_MIN && size <= FLT_MAX) && p != 0.0f && q != 0.0f && isfinite(p) && isfinite(q);
}

// False only where x * q stays within them for every such x: q from 2^-108 to 2^102.
__device__ __forceinline__ bool scale_is_far(float q) {
    return (__float_as_uint(q) & 0x7fffffffu) - __float_as_uint(0x1p-108f) > __float_as_uint(0x1p102f) - __float_as_uint(0x1p-108f);
}

// x * first * second, rounded after each step, for finite p and q.  A call:
// inlined for each column it slows the loop beside it (4096^3 with a scale per
// column: 112 to 117 us).
__device__ __noinline__ float2 scale_factors(float p, float q) {
    int i, j;
    const float a = frexpf(p, &i), b = frexpf(q, &j);
    const int e = i + j, first = max(-100, min(100, e));
    return make_float2(ldexpf(__fmul_rn(a, b), first), ldexpf(1.0f, max(-149, min(127, e - first))));
}

// acc + x * q * p, the same bits as without the factors where they are not needed.
__device__ __forceinline__ float add_scaled(float acc, float x, float p, float q) {
    if (!scale_is_far(q) || !isfinite(p) || !isfinite(q)) return __fmaf_rn(__fmul_rn(x, q), p, acc);
    const float2 f = scale_factors(p, q);
    return __fmaf_rn(__fmul_rn(x, f.x), f.y, acc);
}

__device__ __forceinline__ float bias_at(const BlockParams &P, uint32_t n) {
    if (P.bias_dtype == SDFOAM_F32) return __ldg(static_cast<const float *>(P.bias) + n);
    if (P.bias_dtype == SDFOAM_F16) return __half2float(static_cast<const __half *>(P.bias)[n]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(P.bias)[n]);
}

__device__ __forceinline__ void store_value(void *out, uint32_t dtype, uint64_t at, float v) {
    if (dtype == SDFOAM_F32) static_cast<float *>(out)[at] = v;
    else if (dtype == SDFOAM_F16) static_cast<__half *>(out)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(out)[at] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t pack2(uint32_t dtype, float a, float b) {
    if (dtype == SDFOAM_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

struct Unit {
    uint32_t tp, tq, k0, k1;  // tile, blocks of the reduction
};

// Units in the order of their tiles (16 tiles of P by all of Q at a time, so
// that the CTAs at work read few rows of either operand), a tile's slices
// one after another.
__device__ __forceinline__ Unit unit_of(const BlockParams &P, uint32_t u) {
    const uint32_t tile = u / P.splits, s = u - tile * P.splits;
    const uint32_t per = kSwizzleTiles * P.tiles_q, g = tile / per, in = tile - g * per;
    const uint32_t rows = min(uint32_t(kSwizzleTiles), P.tiles_p - g * kSwizzleTiles);
    Unit r;
    r.tq = in / rows;
    r.tp = g * kSwizzleTiles + (in - r.tq * rows);
    r.k0 = uint32_t(uint64_t(P.k_blocks) * s / P.splits);
    r.k1 = uint32_t(uint64_t(P.k_blocks) * (s + 1) / P.splits);
    return r;
}

// Stores a warp's 32 rows x kCols columns (lane = row), at least 32 columns.
// `stage` is the warp's staging buffer, `row_stage` that of the warps of its
// rows.  Rows go to shared memory in pieces of 16 bytes, swizzled as the TMA
// unit (or the element-wise reader) expects: piece q of row r of a box of 128
// bytes at q ^ (r & 7), of 64 bytes at q ^ ((r / 2) & 3).  PATCH: the thread
// holds columns 2 (lane % 4) and + 1 of each 8 (cg) of rows 8 j + lane / 4, at
// acc[4 cg + j].
template <int kCols, int kGroups, bool PATCH>
__device__ __forceinline__ void store_rows(const BlockParams &P, const CUtensorMap *map, unsigned char *stage,
                                           unsigned char *row_stage, const uint64_t (&acc)[kCols / 2], uint32_t row0,
                                           uint32_t col0, uint32_t lane, uint32_t group, uint32_t quarter) {
    // this warp's previous stores have read the buffer
    if (P.store != kStoreRows && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    if (!PATCH && P.store == kStoreSpan) {
        // 16-bit rows of q_rows columns one after another: kCols < q_rows <= 2
        // kCols.  The second group stores all its columns, past its rows'
        // ends into the next rows' first columns; the first group's, which
        // are all in the row, come after it (bounds for each column instead
        // of the order: 260 us for 1M x 217 x 256, 161 so).  Whole words: a
        // row that starts on half a word stores its first column alone, then
        // the pairs of columns 2 i - 1 and 2 i, then its last.
        const uint32_t n = P.q_rows, odd = (lane * n + group * kCols) & 1u;
        uint16_t *dst = reinterpret_cast<uint16_t *>(row_stage) + lane * n + group * kCols;
        uint32_t w[kCols / 2 + 1];
        w[0] = 0;
#pragma unroll
        for (int i = 0; i < kCols / 2; ++i) {
            const float2 x = unpair(acc[i]);
            w[i + 1] = pack2(P.out_dtype, x.x, x.y);
        }
        const uint16_t head = uint16_t(w[1]), tail = uint16_t(w[kCols / 2] >> 16);
        if (odd) {
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) w[i] = __byte_perm(w[i], w[i + 1], 0x5432);
        } else {
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) w[i] = w[i + 1];
        }
        __syncwarp();
        asm volatile("bar.sync %0, %1;" ::"r"(2 + quarter), "n"(32 * kGroups) : "memory");
#pragma unroll
        for (uint32_t turn = 0; turn < uint32_t(kGroups); ++turn) {
            __syncwarp();
            if (turn > 0) asm volatile("bar.sync %0, %1;" ::"r"(2 + quarter), "n"(32 * kGroups) : "memory");
            if (group == turn) continue;
            if (odd) {
                dst[0] = head;
                dst[kCols - 1] = tail;
            } else {
                *reinterpret_cast<uint32_t *>(dst) = w[0];
            }
#pragma unroll
            for (int i = 1; i < kCols / 2; ++i) *reinterpret_cast<uint32_t *>(dst + 2 * i - odd) = w[i];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        asm volatile("bar.sync %0, %1;" ::"r"(2 + quarter), "n"(32 * kGroups) : "memory");
        if (group == 0 && row0 < P.p_rows) {
            const uint32_t bytes = min(32u, P.p_rows - row0) * n * 2, whole = bytes & ~15u;
            unsigned char *to = static_cast<unsigned char *>(P.out) + uint64_t(row0) * n * 2;
            if (lane == 0 && whole) {
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to),
                             "r"(smem_u32(row_stage)), "r"(whole)
                             : "memory");
            }
            if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            if (lane < (bytes - whole) / 2)
                reinterpret_cast<uint16_t *>(to + whole)[lane] = reinterpret_cast<uint16_t *>(row_stage + whole)[lane];
        }
        return;
    }
    __syncwarp();
    const bool wide = P.out_dtype == SDFOAM_F32;
    constexpr int kCols16 = kCols >= 64 ? 64 : 32;  // columns of a box of 16-bit elements
    constexpr int kBoxes16 = kCols / kCols16, kBoxes32 = kCols / 32, kFit32 = kBoxes32 >= 2 ? kBoxes32 / 2 : 1;
    const uint32_t sw16 = kCols16 == 64 ? (lane & 7u) : ((lane >> 1) & 3u);
    if (!wide) {
        if constexpr (PATCH) {
            static_assert(kCols16 == 64, "a patch stores boxes of 128 bytes");
#pragma unroll
            for (int cg = 0; cg < kCols / 8; ++cg) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 x = unpair(acc[4 * cg + j]);
                    unsigned char *row = stage + cg / 8 * 4096 + (8 * j + (lane >> 2)) * 128;
                    *reinterpret_cast<uint32_t *>(row + (((cg % 8) ^ (lane >> 2)) << 4) + (lane & 3u) * 4) =
                        pack2(P.out_dtype, x.x, x.y);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < (PATCH ? 0 : kBoxes16); ++b) {
            unsigned char *box = stage + b * (32 * kCols16 * 2) + lane * (kCols16 * 2);
#pragma unroll
            for (int q = 0; q < kCols16 / 8; ++q) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = unpair(acc[(b * kCols16 + q * 8) / 2 + e]);
                    w[e] = pack2(P.out_dtype, x.x, x.y);
                }
                *reinterpret_cast<uint4 *>(box + ((q ^ sw16) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        if (P.store == kStoreBox) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
#pragma unroll
                for (int b = 0; b < kBoxes16; ++b)
                    if (col0 + b * kCols16 < P.q_rows && row0 < P.p_rows)
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                                         reinterpret_cast<uint64_t>(map)),
                                     "r"(int(col0 + b * kCols16)), "r"(int(row0)),
                                     "r"(smem_u32(stage + b * (32 * kCols16 * 2)))
                                     : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            return;
        }
        __syncwarp();
        for (uint32_t r = 0; r < 32 && row0 + r < P.p_rows; ++r) {
            const uint32_t sw = kCols16 == 64 ? (r & 7u) : ((r >> 1) & 3u);
            uint16_t *dst = static_cast<uint16_t *>(P.out) + uint64_t(row0 + r) * P.ldo;
#pragma unroll
            for (int j = 0; j < kCols / 32; ++j) {
                const uint32_t c = j * 32 + lane, b = c / kCols16, in = c % kCols16;
                const uint16_t v = *reinterpret_cast<const uint16_t *>(
                    stage + b * (32 * kCols16 * 2) + r * (kCols16 * 2) + (((in >> 3) ^ sw) << 4) + (in & 7u) * 2u);
                if (col0 + c < P.q_rows) dst[col0 + c] = v;
            }
        }
        __syncwarp();
        return;
    }
    // fp32: boxes of 32 columns, kFit32 of them at a time
#pragma unroll
    for (int b0 = 0; b0 < kBoxes32; b0 += kFit32) {
        if (b0 > 0) {
            if (P.store == kStoreBox && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
        }
#pragma unroll
        for (int b = b0; b < b0 + kFit32; ++b) {
            if constexpr (PATCH) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int cg = i / 4, j = i % 4;  // of the box's 32 columns
                    const float2 x = unpair(acc[16 * b + 4 * cg + j]);
                    unsigned char *row = stage + (b - b0) * 4096 + (8 * j + (lane >> 2)) * 128;
                    const uint32_t q = 2 * cg + ((lane & 3u) >> 1);
                    *reinterpret_cast<float2 *>(row + ((q ^ (lane >> 2)) << 4) + (lane & 1u) * 8) = x;
                }
            }
            unsigned char *box = stage + (b - b0) * 4096 + lane * 128;
#pragma unroll
            for (int q = 0; q < (PATCH ? 0 : 8); ++q) {
                const float2 x = unpair(acc[b * 16 + q * 2]), y = unpair(acc[b * 16 + q * 2 + 1]);
                *reinterpret_cast<float4 *>(box + ((q ^ (lane & 7u)) << 4)) = make_float4(x.x, x.y, y.x, y.y);
            }
        }
        if (P.store == kStoreBox) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
#pragma unroll
                for (int b = b0; b < b0 + kFit32; ++b)
                    if (col0 + b * 32 < P.q_rows && row0 < P.p_rows)
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                                         reinterpret_cast<uint64_t>(map)),
                                     "r"(int(col0 + b * 32)), "r"(int(row0)), "r"(smem_u32(stage + (b - b0) * 4096))
                                     : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            __syncwarp();
            for (uint32_t r = 0; r < 32 && row0 + r < P.p_rows; ++r) {
                float *dst = static_cast<float *>(P.out) + uint64_t(row0 + r) * P.ldo;
#pragma unroll
                for (int b = b0; b < b0 + kFit32; ++b) {
                    const float v = *reinterpret_cast<const float *>(stage + (b - b0) * 4096 + r * 128 +
                                                                     (((lane >> 2) ^ (r & 7u)) << 4) + (lane & 3u) * 4u);
                    if (col0 + b * 32 + lane < P.q_rows) dst[col0 + b * 32 + lane] = v;
                }
            }
            __syncwarp();
        }
    }
}

// Float4 number i of a tile's sums (the epilogue's order), plus the bias, to
// its four places of out.
template <int TN, bool SWAP>
__device__ __forceinline__ void store_four(const BlockParams &P, const Unit &t, uint32_t i, const float (&v)[4]) {
    constexpr int kCols = Shape<TN, false>::kCols;
    // warp w of the epilogue: quarter w % 4, group w / 4
    const uint32_t lane = i & 31, c4 = (i >> 5) % (kCols / 4), w = (i >> 5) / (kCols / 4);
    const uint32_t row = t.tp * kTileP + (w & 3) * 32 + lane;
    const uint32_t col = t.tq * TN + (w / 4) * kCols + c4 * 4;
    if (row >= P.p_rows) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= P.q_rows) return;
        const uint32_t n = SWAP ? row : col + e, m = SWAP ? col + e : row;
        store_value(P.out, P.out_dtype, uint64_t(m) * P.ldo + n, P.bias ? v[e] + bias_at(P, n) : v[e]);
    }
}

// QROWS: a scale per row of Q (per column of the tile) instead of one per 128.
// SWAP: P is b and Q is a; the tile is stored turned.
// PAIR: two CTAs share a tile of 256 rows of P; each brings its 128 rows and
// half of the tile's rows of Q, and the first one issues the MMAs
// (cta_group::2) over both CTAs' shared memory, so that each operand byte
// brought in feeds twice the work.
template <int TN, bool QROWS, bool SWAP, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) block_mm_kernel(const __grid_constant__ CUtensorMap map_p,
                                                               const __grid_constant__ CUtensorMap map_q,
                                                               const __grid_constant__ CUtensorMap map_out,
                                                               const BlockParams P) {
    using S = Shape<TN, PAIR>;
    constexpr int kCols = S::kCols;
    constexpr int kChunk = 8;
    // A scale per column is a value per column for every thread that holds one
    // row: at 128 bytes a cycle shared memory takes twice the MMAs' time to
    // hand them out (4096^3: 111 to 134 us in two runs, 75 to 89 without those
    // reads).  Where the tile is wide, a thread holds 4 rows of a quarter of the
    // columns instead (93 to 112; 74 with a scale per 128 columns).
    constexpr bool kPatch = QROWS && !SWAP && TN >= 128;
    constexpr uint32_t kPart = kTileP * TN / 4;  // float4 of a CTA's sums: [warp][columns / 4][lane]
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char *boxes = smem + S::kStages * S::kStageBytes;
    float *scales = reinterpret_cast<float *>(boxes + kEpiWarps * S::kBoxBytes);  // [kScaleStages][kTileP + TN]
    float *bias_s = scales + S::kScaleStages * S::kScaleFloats;                    // [TN]
    uint64_t *bars = reinterpret_cast<uint64_t *>(bias_s + TN);
    // bars: full[stages], empty[stages], acc_full[accs], acc_empty[accs],
    // scale_full[scale stages], scale_empty[scale stages], drain
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S::kStages + 2 * S::kAccs + 2 * S::kScaleStages + 1);
    __shared__ volatile int abort_flag;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const uint32_t first_unit = PAIR ? blockIdx.x / 2 : blockIdx.x, unit_step = PAIR ? gridDim.x / 2 : gridDim.x;
    const uint32_t full = smem_u32(bars), empty = full + 8 * S::kStages;
    const uint32_t acc_full = empty + 8 * S::kStages, acc_empty = acc_full + 8 * S::kAccs;
    const uint32_t scale_full = acc_empty + 8 * S::kAccs, scale_empty = scale_full + 8 * S::kScaleStages;
    const uint32_t drain = scale_empty + 8 * S::kScaleStages;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < S::kAccs; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, kEpiWarps * S::kCtas);
        }
        for (int s = 0; s < S::kScaleStages; ++s) {
            mbar_init(scale_full + 8 * s, 64);
            mbar_init(scale_empty + 8 * s, kEpiWarps);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        abort_flag = 0;
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(S::kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(S::kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = *tmem_slot;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == 0 && lane == 0) {
            // ---- producer ----
            uint32_t issued = 0;
            bool ok = true;
            for (uint32_t u = first_unit; u < P.units && ok; u += unit_step) {
                const Unit t = unit_of(P, u);
                const int p0 = int((t.tp * S::kCtas + rank) * kTileP), q0 = int(t.tq * TN + rank * (TN / S::kCtas));
                for (uint32_t kb = t.k0; kb < t.k1; ++kb, ++issued) {
                    const uint32_t s = issued % S::kStages, use = issued / S::kStages;
                    if (use > 0 && !mbar_wait(empty + 8 * s, (use - 1) & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = smem_u32(smem + s * S::kStageBytes);
                    if (rank == 0) mbar_expect_tx(full + 8 * s, S::kCtas * S::kStageBytes);
                    load_tile<PAIR>(dst, &map_p, int(kb * kBlockK), p0, full + 8 * s);
                    load_tile<PAIR>(dst + kPBytes, &map_q, int(kb * kBlockK), q0, full + 8 * s);
                }
            }
            // the pair's copies, and the MMAs' releases of the stages, which
            // arrive here: the last use of every stage
            for (uint32_t l = issued > uint32_t(S::kStages) ? issued - S::kStages : 0; l < issued; ++l) {
                if (rank == 0) mbar_wait(full + 8 * (l % S::kStages), (l / S::kStages) & 1, nullptr);
                if (ok) mbar_wait(empty + 8 * (l % S::kStages), (l / S::kStages) & 1, &abort_flag);
            }
        } else if (warp == 1 && lane == 0 && rank == 0) {
            // ---- MMA issuer: one accumulator per block of 128 ----
            uint32_t done = 0;
            bool ok = true;
            for (uint32_t u = first_unit; u < P.units && ok; u += unit_step) {
                const Unit t = unit_of(P, u);
                for (uint32_t kb = t.k0; kb < t.k1; ++kb, ++done) {
                    const uint32_t s = done % S::kStages, use = done / S::kStages;
                    const uint32_t b = done % S::kAccs, turn = done / S::kAccs;
                    if ((turn > 0 && !mbar_wait(acc_empty + 8 * b, (turn - 1) & 1, &abort_flag)) ||
                        !mbar_wait(full + 8 * s, use & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t base = smem_u32(smem + s * S::kStageBytes);
                    const uint64_t ad = sw128_desc(base), bd = sw128_desc(base + kPBytes);
#pragma unroll
                    for (int k = 0; k < kBlockK / 32; ++k)
                        mma_e4m3<PAIR>(tmem + b * TN, ad + uint64_t(2 * k), bd + uint64_t(2 * k), idesc<TN, PAIR>(),
                                       k > 0 ? 1u : 0u);
                    commit_to_all<PAIR>(acc_full + 8 * b);
                    commit_to_all<PAIR>(empty + 8 * s);
                }
            }
            // no MMA may still be running when the accumulators are freed
            if constexpr (PAIR)
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain) : "memory");
            else
                mma_commit(drain);
            mbar_wait(drain, 0, nullptr);
        } else if (warp >= 2) {
            // ---- scales: warp 2 P's, warp 3 Q's (one per row, or one for the
            // 128 rows that a group of epilogue warps has) ----
            const uint64_t step = warp == 2 ? P.p_scale_block : P.q_scale_block;
            const uint32_t to = smem_u32(scales + (warp == 2 ? 0 : kTileP) + lane);
            uint32_t done = 0;
            bool ok = true;
            for (uint32_t u = first_unit; u < P.units && ok; u += unit_step) {
                const Unit t = unit_of(P, u);
                constexpr int kQPer = QROWS ? (TN + 31) / 32 : 1, kPer = kQPer > 4 ? kQPer : 4;
                const float *src[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const uint32_t at = i * 32 + lane;
                    src[i] = nullptr;
                    if (warp == 2 && i < 4) {
                        const uint32_t row = min((t.tp * S::kCtas + rank) * kTileP + at, P.p_rows - 1);
                        src[i] = P.p_scales + (row >> P.p_shift) * P.p_scale_row + t.k0 * P.p_scale_block;
                    } else if (warp == 3 && i < kQPer && at < uint32_t(QROWS ? TN : S::kGroups)) {
                        const uint32_t row = min(t.tq * TN + (QROWS ? at : at * kCols), P.q_rows - 1);
                        src[i] = P.q_scales + (row >> P.q_shift) * P.q_scale_row + t.k0 * P.q_scale_block;
                    }
                }
                for (uint32_t kb = t.k0; kb < t.k1; ++kb, ++done) {
                    const uint32_t s = done % S::kScaleStages, use = done / S::kScaleStages;
                    if (use > 0 && !mbar_wait(scale_empty + 8 * s, (use - 1) & 1, &abort_flag)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (src[i]) {
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + (s * S::kScaleFloats + i * 32) * 4),
                                         "l"(src[i])
                                         : "memory");
                            src[i] += step;
                        }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(scale_full + 8 * s) : "memory");
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        // ---- sums and stores; every warp takes every block, also after a
        // wait gave up (the barriers below stay matched) ----
        const uint32_t quarter = warp & 3, group = (warp - 4) / 4, et = threadIdx.x - 128;
        // the warps of a quarter have their staging next to each other
        unsigned char *row_stage = boxes + quarter * S::kGroups * S::kBoxBytes, *stage = row_stage + group * S::kBoxBytes;
        uint32_t done = 0, bias_tq = 0xffffffffu;
        bool bad = false;
        // this warp has read an accumulator and its scales
        auto release = [&](uint32_t b, uint32_t ss) {
            asm volatile("tcgen05.fence::before_thread_sync;");
            __syncwarp();
            if (lane == 0) {
                arrive_at_first<PAIR>(acc_empty + 8 * b);
                mbar_arrive(scale_empty + 8 * ss);
            }
        };
        for (uint32_t u = first_unit; u < P.units; u += unit_step) {
            const Unit t = unit_of(P, u);
            const uint32_t row0 = (t.tp * S::kCtas + rank) * kTileP + quarter * 32, row = row0 + lane;
            const uint32_t col0 = t.tq * TN + group * kCols;
            uint64_t acc[kCols / 2];
            if (!SWAP && P.bias && P.splits == 1) {
                // the sums start from the bias
                if (t.tq != bias_tq) {
                    __syncwarp();
                    asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
                    if (et < TN) bias_s[et] = t.tq * TN + et < P.q_rows ? bias_at(P, t.tq * TN + et) : 0.0f;
                    __syncwarp();
                    asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
                    bias_tq = t.tq;
                }
                const float *own = bias_s + group * kCols;
                if constexpr (kPatch) {
#pragma unroll
                    for (int i = 0; i < kCols / 2; ++i)
                        acc[i] = *reinterpret_cast<const uint64_t *>(own + i / 4 * 8 + (lane & 3u) * 2);
                } else {
#pragma unroll
                    for (int i = 0; i < kCols / 2; i += 2) {
                        const float4 x = *reinterpret_cast<const float4 *>(own + 2 * i);
                        acc[i] = pair(x.x, x.y);
                        acc[i + 1] = pair(x.z, x.w);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < kCols / 2; ++i) acc[i] = 0;
            }
            bool far = false;
            for (uint32_t kb = t.k0; kb < t.k1; ++kb, ++done) {
                for (; kb < t.k1; ++kb, ++done) {
                    const uint32_t b = done % S::kAccs, turn = done / S::kAccs;
                    const uint32_t ss = done % S::kScaleStages;
                    if (!mbar_wait(scale_full + 8 * ss, (done / S::kScaleStages) & 1, &abort_flag)) bad = true;
                    const float *sc = scales + ss * S::kScaleFloats;
                    const float *q_sc = sc + kTileP + (QROWS ? group * kCols : group);
                    if constexpr (QROWS) {
                        // any of the warp's columns
                        constexpr int kPer = kCols < 32 ? 1 : kCols / 32;
                        struct alignas(4 * kPer) Piece { float q[kPer]; };
                        const Piece piece = reinterpret_cast<const Piece *>(q_sc)[kCols < 32 ? lane % kCols : lane];
                        far = false;
#pragma unroll
                        for (int i = 0; i < kPer; ++i) far |= scale_is_far(piece.q[i]);
                    }
                    float one = 0.0f;
                    uint64_t p4[kPatch ? 4 : 1];
                    if constexpr (kPatch) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float p = sc[quarter * 32 + 8 * j + (lane >> 2)];
                            p4[j] = pair(p, p);
                        }
                    } else {
                        one = sc[quarter * 32 + lane];
                        if constexpr (!QROWS) {
                            // this row, which then adds nothing
                            far = product_leaves(one, *q_sc);
                            one = far ? 0.0f : one * *q_sc;
                        }
                    }
                    if (!mbar_wait(acc_full + 8 * b, turn & 1, &abort_flag)) bad = true;
                    __syncwarp();
                    const bool some = __any_sync(0xffffffffu, far);
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    if (QROWS && some) break;
                    const uint32_t addr = tmem + ((quarter * 32) << 16) + b * TN + group * kCols;
                    if constexpr (kPatch) {
#pragma unroll
                        for (int c = 0; c < kCols / 16; ++c) {
                            const uint64_t *qp = reinterpret_cast<const uint64_t *>(q_sc + c * 16 + (lane & 3u) * 2);
                            const uint64_t q2[2] = {qp[0], qp[4]};
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t v[8];
                                tmem_load_patch(v, addr + (uint32_t(16 * h) << 16) + c * 16);
                                tmem_wait(v);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int g = i / 2, j = 2 * h + i % 2;
                                    const uint64_t x = pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                                    fma_pair(acc[4 * (2 * c + g) + j], mul_pair(x, q2[g]), p4[j]);
                                }
                            }
                        }
                    } else {
                        const uint64_t s2 = pair(one, one);
#pragma unroll
                        for (int c = 0; c < kCols / kChunk; ++c) {
                            uint32_t v[kChunk];
                            tmem_load(v, addr + c * kChunk);
                            tmem_wait(v);
#pragma unroll
                            for (int i = 0; i < kChunk; i += 4) {
                                uint64_t x = pair(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                                uint64_t y = pair(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
                                if (QROWS) {
                                    const float4 q = *reinterpret_cast<const float4 *>(q_sc + c * kChunk + i);
                                    x = mul_pair(x, pair(q.x, q.y));
                                    y = mul_pair(y, pair(q.z, q.w));
                                }
                                fma_pair(acc[(c * kChunk + i) / 2], x, s2);
                                fma_pair(acc[(c * kChunk + i) / 2 + 1], y, s2);
                            }
                        }
                    }
                    if (!QROWS && some) break;
                    release(b, ss);
                }
                if (kb == t.k1) break;
                // a block with scales that need the factors: with a scale per
                // column the whole of it, element by element, else the rows
                // that the loop above left out.  In that loop this code costs
                // a tenth although it does not run (4096^3: 76 to 85 us; out
                // here 74, and 112 with a scale per column, as without any
                // check; 1M x 217 x 256 166 to 173)
                const uint32_t b = done % S::kAccs, ss = done % S::kScaleStages;
                const float *sc = scales + ss * S::kScaleFloats;
                const uint32_t addr = tmem + ((quarter * 32) << 16) + b * TN + group * kCols;
                if constexpr (QROWS) {
                    const float *q_sc = sc + kTileP + group * kCols;
#pragma unroll
                    for (int i = 0; i < kCols / 8; ++i) {
                        // as many loads as in the loop above
                        const int c = kPatch ? i / 2 * 16 : i * 8, h = i % 2;
                        uint32_t v[8];
                        if constexpr (kPatch) tmem_load_patch(v, addr + (uint32_t(16 * h) << 16) + c);
                        else tmem_load(v, addr + c);
                        tmem_wait(v);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int g = e / 2, j = 2 * h + e % 2;
                            const float p = sc[quarter * 32 + (kPatch ? 8 * j + (lane >> 2) : lane)];
                            const float *q = q_sc + c + (kPatch ? 8 * g + (lane & 3u) * 2 : 2 * e);
                            uint64_t &sum = acc[kPatch ? 4 * (c / 8 + g) + j : c / 2 + e];
                            const float2 was = unpair(sum);
                            sum = pair(add_scaled(was.x, __uint_as_float(v[2 * e]), p, q[0]),
                                       add_scaled(was.y, __uint_as_float(v[2 * e + 1]), p, q[1]));
                        }
                    }
                } else {
                    float2 f = make_float2(0.0f, 0.0f);
                    if (far) f = scale_factors(sc[quarter * 32 + lane], sc[kTileP + group]);
#pragma unroll
                    for (int c = 0; c < kCols / kChunk; ++c) {
                        uint32_t v[kChunk];
                        tmem_load(v, addr + c * kChunk);
                        tmem_wait(v);
#pragma unroll
                        for (int i = 0; i < kChunk; i += 2) {
                            const uint64_t x = pair(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                            if (far) fma_pair(acc[(c * kChunk + i) / 2], mul_pair(x, pair(f.x, f.x)), pair(f.y, f.y));
                        }
                    }
                }
                release(b, ss);
            }
            if (bad) {
#pragma unroll
                for (int i = 0; i < kCols / 2; ++i) acc[i] = 0x7fc000007fc00000ull;
            }
            if (!PAIR && P.splits > 1) {
                // in a cluster: over the operands' ring, which is done with
                float4 *dst = TN <= 64 && P.cluster_join ? reinterpret_cast<float4 *>(smem) : P.parts + size_t(u) * kPart;
                dst += (warp - 4) * (kCols / 4) * 32;
                if constexpr (kPatch) {
#pragma unroll
                    for (int i = 0; i < kCols / 2; ++i) {
                        const int c4 = i / 4 * 2, j = i % 4;
                        float4 *at = dst + (c4 + ((lane & 3u) >> 1)) * 32 + 8 * j + (lane >> 2);
                        reinterpret_cast<float2 *>(at)[lane & 1u] = unpair(acc[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kCols / 4; ++i) {
                        const float2 x = unpair(acc[2 * i]), y = unpair(acc[2 * i + 1]);
                        dst[i * 32 + lane] = make_float4(x.x, x.y, y.x, y.y);
                    }
                }
            } else if constexpr (SWAP) {
                // lane = column of out: the warp writes 32 consecutive elements
                const float bias = P.bias && row < P.p_rows ? bias_at(P, row) : 0.0f;
#pragma unroll
                for (int i = 0; i < kCols / 2; ++i) {
                    const float2 x = unpair(acc[i]);
                    if (row < P.p_rows && col0 + 2 * i < P.q_rows)
                        store_value(P.out, P.out_dtype, uint64_t(col0 + 2 * i) * P.ldo + row, x.x + bias);
                    if (row < P.p_rows && col0 + 2 * i + 1 < P.q_rows)
                        store_value(P.out, P.out_dtype, uint64_t(col0 + 2 * i + 1) * P.ldo + row, x.y + bias);
                }
            } else if constexpr (kCols >= 32) {
                store_rows<kCols, S::kGroups, kPatch>(P, &map_out, stage, row_stage, acc, row0, col0, lane, group, quarter);
            } else if (row < P.p_rows && P.out_dtype != SDFOAM_F32 && col0 + kCols <= P.q_rows &&
                       ((reinterpret_cast<uintptr_t>(P.out) | (P.ldo * 2)) & 15u) == 0) {
                // 8 or 16 columns per thread, 16 bytes at a time
                uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(P.out) + uint64_t(row) * P.ldo + col0);
#pragma unroll
                for (int q = 0; q < kCols / 8; ++q) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 x = unpair(acc[q * 4 + e]);
                        w[e] = pack2(P.out_dtype, x.x, x.y);
                    }
                    dst[q] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else if (row < P.p_rows) {
#pragma unroll
                for (int i = 0; i < kCols / 2; ++i) {
                    const float2 x = unpair(acc[i]);
                    const uint64_t at = uint64_t(row) * P.ldo + col0 + 2 * i;
                    if (col0 + 2 * i < P.q_rows) store_value(P.out, P.out_dtype, at, x.x);
                    if (col0 + 2 * i + 1 < P.q_rows) store_value(P.out, P.out_dtype, at + 1, x.y);
                }
            }
        }
        // the bulk stores are complete
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    if (abort_flag && threadIdx.x == 0) {
        *static_cast<volatile int *>(P.error) = 1;
        __threadfence_system();
    }
    if constexpr (TN <= 64 && !PAIR) {
        if (P.cluster_join) {
            // one unit per CTA: the slices of a tile, each CTA adds its share
            // of them in order
            cluster_sync();
            const Unit t = unit_of(P, blockIdx.x);
            const uint32_t own = cluster_rank(), mine = smem_u32(smem);
            for (uint32_t i = own * kThreads + threadIdx.x; i < kPart; i += P.splits * kThreads) {
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (uint32_t s = 0; s < P.splits; ++s) {
                    float4 x;
                    asm volatile(
                        "{\n"
                        ".reg .b32 a;\n"
                        "mapa.shared::cluster.u32 a, %4, %5;\n"
                        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n"
                        "}\n"
                        : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                        : "r"(mine + i * 16), "r"(s)
                        : "memory");
                    v[0] += x.x;
                    v[1] += x.y;
                    v[2] += x.z;
                    v[3] += x.w;
                }
                store_four<TN, SWAP>(P, t, i, v);
            }
            cluster_sync();  // the others have read this CTA's sums
        }
    }
    // the other CTA's copies, commits and arrivals are done before either leaves
    if constexpr (PAIR) cluster_sync();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;");
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmemCols));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmemCols));
    }
}

// Adds the slices of a tile in order (parts: [tile][slice][warp][columns / 4]
// [lane] float4) and the bias.  A block takes the 32 rows x kCols columns of
// one epilogue warp, or 16 columns of them where there are MANY slices, read
// as that warp wrote them: groups of threads take consecutive runs of the
// slices, their sums are added in order and turned in shared memory, so that
// consecutive threads store consecutive elements (512 x 2048 of two slices:
// 12 us stored straight from the parts' order, 4.7 so; 256 x 256 of 37: 7.5
// and 3.5).
constexpr int kJoinThreads = 512;

template <int TN, bool MANY>
constexpr int join_columns() {
    return MANY && Shape<TN, false>::kCols > 16 ? 16 : Shape<TN, false>::kCols;
}

template <int TN, bool SWAP, bool MANY>
__global__ void __launch_bounds__(kJoinThreads) join_slices_kernel(const BlockParams P) {
    constexpr int kCols = Shape<TN, false>::kCols, kTake = join_columns<TN, MANY>(), kPieces = kCols / kTake;
    constexpr uint32_t kPerTile = kTileP * TN / 4, kItems = kTake / 4 * 32, kRuns = kJoinThreads / kItems;
    __shared__ float sums[kRuns][32][kTake + 1];
    const uint32_t piece = blockIdx.x % kPieces, w = blockIdx.x / kPieces % kEpiWarps, tile = blockIdx.x / (kPieces * kEpiWarps);
    const uint32_t run = threadIdx.x / kItems, i = threadIdx.x % kItems;
    const float4 *src = P.parts + size_t(tile) * P.splits * kPerTile + (w * kPieces + piece) * kItems + i;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t s1 = (run + 1) * P.splits / kRuns;
#pragma unroll 4
    for (uint32_t s = run * P.splits / kRuns; s < s1; ++s) {
        const float4 x = __ldcs(src + size_t(s) * kPerTile);
        v[0] += x.x;
        v[1] += x.y;
        v[2] += x.z;
        v[3] += x.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[run][i & 31][(i >> 5) * 4 + e] = v[e];
    __syncthreads();
    const Unit t = unit_of(P, tile * P.splits);
    const uint32_t row0 = t.tp * kTileP + (w & 3) * 32, col0 = t.tq * TN + (w / 4) * kCols + piece * kTake;
    for (uint32_t o = threadIdx.x; o < 32 * kTake; o += kJoinThreads) {
        const uint32_t r = SWAP ? o % 32 : o / kTake, c = SWAP ? o / 32 : o % kTake;
        const uint32_t row = row0 + r, col = col0 + c;
        if (row >= P.p_rows || col >= P.q_rows) continue;
        const uint32_t n = SWAP ? row : col, m = SWAP ? col : row;
        float x = sums[0][r][c];
#pragma unroll
        for (uint32_t q = 1; q < kRuns; ++q) x += sums[q][r][c];
        store_value(P.out, P.out_dtype, uint64_t(m) * P.ldo + n, P.bias ? x + bias_at(P, n) : x);
    }
}

// The bias (or zero) everywhere: a product over nothing.
__global__ void __launch_bounds__(256) fill_bias_kernel(const BlockParams P, uint32_t m, uint32_t n) {
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < uint64_t(m) * n; i += uint64_t(gridDim.x) * 256) {
        const uint32_t r = uint32_t(i / n), c = uint32_t(i % n);
        store_value(P.out, P.out_dtype, uint64_t(r) * P.ldo + c, P.bias ? bias_at(P, c) : 0.0f);
    }
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------

struct Plan {
    bool swap, pair, cluster_join;
    int tn;
    uint32_t tiles_p, tiles_q, k_blocks, splits;
};

Plan plan_of(uint32_t m, uint32_t n, uint32_t k) {
    Plan l{};
    l.swap = m <= 64 && m < n;
    const uint32_t p = l.swap ? n : m, q = l.swap ? m : n;
    l.tiles_p = (p + kTileP - 1) / kTileP;
    l.tn = q <= 16 ? 16 : q <= 32 ? 32 : q <= 64 ? 64 : q <= 128 ? 128 : 256;
    if (l.tn == 256 && uint64_t(l.tiles_p) * ((q + 255) / 256) < kSms) l.tn = 128;
    l.tiles_q = (q + l.tn - 1) / l.tn;
    l.k_blocks = (k + kBlockK - 1) / kBlockK;
    uint64_t tiles = uint64_t(l.tiles_p) * l.tiles_q;
    // pairs where there is a tile of 256 x 256 for each of them
    l.pair = l.tn == 256;
    if (l.pair) l.tiles_p = (l.tiles_p + 1) / 2;
    l.splits = !l.pair && tiles < kSms ? std::min<uint32_t>(l.k_blocks, uint32_t(kSms / tiles)) : 1;
    // narrow tiles: a cluster of up to 8 slices (the portable size), and no
    // more slices where 16 blocks or fewer are left to each: a second launch
    // costs about as much as 8 blocks
    if (l.tn <= 64 && l.splits > 8 && l.k_blocks <= 128) l.splits = 8;
    l.cluster_join = l.tn <= 64 && l.splits > 1 && l.splits <= 8;
    return l;
}

// [rows, k] e4m3, row stride ld bytes, boxes of box_rows x 128 bytes.
bool operand_map(CUtensorMap *map, const void *base, uint32_t rows, uint32_t k, uint64_t ld, uint32_t box_rows) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {k, rows};
    const cuuint64_t strides[1] = {ld};
    const cuuint32_t box[2] = {uint32_t(kBlockK), box_rows};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// out [rows, cols] in boxes of 32 rows x 128 bytes (64 for tiles of 32 16-bit
// columns per warp), swizzled over the same width.
bool output_map(CUtensorMap *map, void *base, uint32_t rows, uint32_t cols, uint64_t ld, uint32_t dtype, int tn) {
    auto fn = encode_fn();
    if (!fn) return false;
    const uint32_t size = dtype == SDFOAM_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {ld * size};
    const uint32_t bytes = dtype != SDFOAM_F32 && tn == 64 ? 64 : 128;
    const cuuint32_t box[2] = {bytes / size, 32};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, dtype == SDFOAM_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base,
              dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TN, bool QROWS, bool SWAP, bool PAIR>
cudaError_t launch_tiles(const CUtensorMap &mp, const CUtensorMap &mq, const CUtensorMap &mo, const BlockParams &P,
                         cudaStream_t stream) {
    using S = Shape<TN, PAIR>;
    auto kernel = block_mm_kernel<TN, QROWS, SWAP, PAIR>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::kSmem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min<uint32_t>(P.units, kSms / S::kCtas) * S::kCtas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : P.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR || P.cluster_join ? 1 : 0;
    if ((e = cudaLaunchKernelEx(&cfg, kernel, mp, mq, mo, P)) != cudaSuccess || P.splits == 1 || P.cluster_join) return e;
    if constexpr (!PAIR) {
        const unsigned warps = P.tiles_p * P.tiles_q * kEpiWarps;
        if (P.splits > 8)
            join_slices_kernel<TN, SWAP, true><<<warps * (S::kCols / join_columns<TN, true>()), kJoinThreads, 0, stream>>>(P);
        else if constexpr (TN > 64)  // narrow tiles of so few slices are a cluster
            join_slices_kernel<TN, SWAP, false><<<warps, kJoinThreads, 0, stream>>>(P);
    }
    return cudaGetLastError();
}

template <int TN>
cudaError_t launch_tn(const Plan &l, const CUtensorMap &mp, const CUtensorMap &mq, const CUtensorMap &mo,
                      const BlockParams &P, cudaStream_t stream) {
    const bool rows = P.q_shift == 0;
    if constexpr (TN <= 64) {
        if (l.swap)
            return rows ? launch_tiles<TN, true, true, false>(mp, mq, mo, P, stream)
                        : launch_tiles<TN, false, true, false>(mp, mq, mo, P, stream);
    }
    if constexpr (TN == 256)
        return rows ? launch_tiles<TN, true, false, true>(mp, mq, mo, P, stream)
                    : launch_tiles<TN, false, false, true>(mp, mq, mo, P, stream);
    else
        return rows ? launch_tiles<TN, true, false, false>(mp, mq, mo, P, stream)
                    : launch_tiles<TN, false, false, false>(mp, mq, mo, P, stream);
}

}  // namespace

size_t block_matmul_workspace_bytes(uint32_t m, uint32_t n, uint32_t k) {
    if (m == 0 || n == 0 || k == 0) return 0;
    const Plan l = plan_of(m, n, k);
    return l.splits > 1 && !l.cluster_join ? size_t(l.tiles_p) * l.tiles_q * l.splits * kTileP * l.tn * 4 : 0;
}

cudaError_t launch_block_matmul(const void *a, uint64_t lda, const float *a_scales, uint64_t a_scale_row,
                                uint64_t a_scale_block, int a_block_rows, uint32_t m, const void *b, uint64_t ldb,
                                const float *b_scales, uint64_t b_scale_row, uint64_t b_scale_block, int b_block_rows,
                                uint32_t n, uint32_t k, const void *bias, uint32_t bias_dtype, void *out, uint64_t ldo,
                                uint32_t out_dtype, void *workspace, int *error, cudaStream_t stream) {
    if (m == 0 || n == 0) return cudaSuccess;
    BlockParams P{};
    P.bias = bias;
    P.bias_dtype = bias_dtype;
    P.out = out;
    P.ldo = ldo;
    P.out_dtype = out_dtype;
    if (k == 0) {
        fill_bias_kernel<<<unsigned(std::min<uint64_t>((uint64_t(m) * n + 255) / 256, kSms * 32)), 256, 0, stream>>>(P, m, n);
        return cudaGetLastError();
    }
    const Plan l = plan_of(m, n, k);
    P.p_rows = l.swap ? n : m;
    P.q_rows = l.swap ? m : n;
    P.tiles_p = l.tiles_p;
    P.tiles_q = l.tiles_q;
    P.k_blocks = l.k_blocks;
    P.splits = l.splits;
    P.units = l.tiles_p * l.tiles_q * l.splits;
    P.p_scales = l.swap ? b_scales : a_scales;
    P.q_scales = l.swap ? a_scales : b_scales;
    P.p_scale_row = l.swap ? b_scale_row : a_scale_row;
    P.p_scale_block = l.swap ? b_scale_block : a_scale_block;
    P.q_scale_row = l.swap ? a_scale_row : b_scale_row;
    P.q_scale_block = l.swap ? a_scale_block : b_scale_block;
    P.p_shift = (l.swap ? b_block_rows : a_block_rows) == 128 ? 7 : 0;
    P.q_shift = (l.swap ? a_block_rows : b_block_rows) == 128 ? 7 : 0;
    P.parts = static_cast<float4 *>(workspace);
    P.cluster_join = l.cluster_join;
    P.error = error;
    const uint32_t size = out_dtype == SDFOAM_F32 ? 4 : 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(out);
    P.store = l.tn < 64 || l.swap || l.splits > 1                   ? kStoreRows
              : ((at | (ldo * size)) & 15u) == 0                   ? kStoreBox
              : size == 2 && l.tiles_q == 1 && P.q_shift != 0 && n > uint32_t(l.tn) / 2 && ldo == n && !(at & 15u) ? kStoreSpan
                                                                   : kStoreRows;
    CUtensorMap mp, mq, mo{};
    if (!operand_map(&mp, l.swap ? b : a, P.p_rows, k, l.swap ? ldb : lda, kTileP) ||
        !operand_map(&mq, l.swap ? a : b, P.q_rows, k, l.swap ? lda : ldb, uint32_t(l.pair ? l.tn / 2 : l.tn)) ||
        (P.store == kStoreBox && !output_map(&mo, out, m, n, ldo, out_dtype, l.tn)))
        return cudaErrorInvalidValue;
    switch (l.tn) {
        case 16: return launch_tn<16>(l, mp, mq, mo, P, stream);
        case 32: return launch_tn<32>(l, mp, mq, mo, P, stream);
        case 64: return launch_tn<64>(l, mp, mq, mo, P, stream);
        case 128: return launch_tn<128>(l, mp, mq, mo, P, stream);
        default: return launch_tn<256>(l, mp, mq, mo, P, stream);
    }
}

}  // namespace sdfoam_b200

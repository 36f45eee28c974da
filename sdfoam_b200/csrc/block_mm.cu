// out = (a * a_scales) (b * b_scales)^T + bias: the product of two e4m3
// matrices with a scale per block of 128 along the reduction.
//
//   out[m, n] = sum over blocks j of 128 of  sa[m, j] sb[n, j] * (sum over k in j of a[m, k] b[n, k])  + bias[n]
//
// The inner sum runs on the tensor cores (tcgen05.mma kind::f8f6f4, fp32
// accumulation in TMEM); the scales differ from block to block, so each
// block's 128-wide product is read back from TMEM and added, times its scale,
// to fp32 sums in registers.  A persistent CTA per SM walks units of (tile of
// 128 x TN, slice of the reduction):
//   * warp 0 (one lane) streams 128-byte wide tiles of both operands through
//     a ring with TMA (128-byte swizzle; rows and columns past the ends read
//     as zero);
//   * warp 1 (one lane) issues four MMAs (K 32 each) per block into the next
//     of the TMEM accumulators, releasing ring stages and finished
//     accumulators with tcgen05.commit;
//   * warps 2-9 read the accumulators back (warp w: TMEM lanes 32 (w % 4)
//     .., half of the TN columns; one row per thread) and multiply-add them
//     into registers while the tensor cores fill the next accumulator.
//
// The operand with the rows on the TMEM lanes is P, the other Q.  Q is b
// unless a has few rows (a single token to 64): then a's rows are the narrow
// side, so that a weight is read once with 128 of its rows per tile and TN
// columns of tokens.  When the tiles do not fill the GPU, the reduction is
// cut into slices; their fp32 sums go to the workspace and a second launch
// adds them in order (no atomics: the same bits every run).
//
// Every wait is bounded: a CTA that gives up sets *error, writes NaN, waits
// (bounded) for its own copies and MMAs and frees its TMEM.  No TMA multicast.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "foam_internal.h"
#include "tcgen05.cuh"

namespace sdfoam_b200 {

namespace {

constexpr int kSms = 148;
constexpr int kTileP = 128;
constexpr int kBlockK = 128;  // bytes of a row per stage: one swizzle span, one block of scales
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);
constexpr uint32_t kPBytes = kTileP * kBlockK;  // 16 KB
constexpr uint32_t kBoxBytes = 32 * 64;         // an epilogue warp's output box: 32 rows of 64 bytes
constexpr int kSwizzleTiles = 16;               // tiles of P that are walked together (L2)

// TN columns of Q per tile: ring stages that fit, TMEM accumulators.
template <int TN>
struct Shape {
    static constexpr uint32_t kQBytes = TN * kBlockK;
    static constexpr uint32_t kStageBytes = kPBytes + kQBytes;
    static constexpr int kStages = TN == 256 ? 4 : TN == 128 ? 6 : 8;
    static constexpr int kAccs = TN == 256 ? 2 : 4;
    static constexpr uint32_t kTmemCols = uint32_t(TN) * kAccs;
    static constexpr int kHalf = TN / 2;  // columns of an epilogue warp
    static constexpr uint32_t kSmem = kStages * kStageBytes + kEpiWarps * kBoxBytes + 2 * TN * 4 + 256 + 1024;
};

struct BlockParams {
    uint32_t p_rows, q_rows;
    uint32_t tiles_p, tiles_q;
    uint32_t k_blocks, splits, units;
    const float *p_scales, *q_scales;  // [ceil(rows >> shift), k_blocks]
    int p_shift, q_shift;              // 0 or 7: rows per scale as a power of two
    const void *bias;                  // over b's rows (n), or null
    uint32_t bias_dtype;
    void *out;                         // [m, n]
    uint64_t ldo;
    uint32_t out_dtype;
    int box_store;                     // rows of out allow TMA stores
    float4 *parts;                     // splits > 1: sums of the slices
    int *error;
};

// tcgen05 instruction descriptor, kind::f8f6f4: D fp32 (bits 4-5 = 1), A and
// B e4m3 (0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24.
template <int TN>
__device__ __forceinline__ constexpr uint32_t idesc() {
    return (1u << 4) | (uint32_t(TN >> 3) << 17) | (uint32_t(kTileP >> 4) << 24);
}

__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t id,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(id), "r"(accumulate));
}

// 16 (or 8) consecutive columns of the warp's 32 lanes; the values may be
// used after tmem_wait, which names them so that no use moves before it.
__device__ __forceinline__ void tmem_load(uint32_t (&r)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load(uint32_t (&r)[8], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
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

// One 64-byte row per lane (32 rows) of the output through the warp's box:
// TMA where the rows of out are 16-byte aligned, else whole rows of the box
// by consecutive lanes.
__device__ __forceinline__ void store_box(const BlockParams &P, const CUtensorMap *map, unsigned char *box,
                                          const uint32_t (&w)[16], uint32_t row0, uint32_t col0, uint32_t lane) {
    const uint32_t sw = (lane >> 1) & 3u;
    if (P.box_store && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q)
        *reinterpret_cast<uint4 *>(box + lane * 64u + ((q ^ sw) << 4)) =
            make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    if (P.box_store) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                             reinterpret_cast<uint64_t>(map)),
                         "r"(int(col0)), "r"(int(row0)), "r"(smem_u32(box))
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        return;
    }
    __syncwarp();
    if (P.out_dtype == SDFOAM_F32) {
        const uint32_t c = lane & 15u;
#pragma unroll 4
        for (uint32_t r = lane >> 4; r < 32; r += 2) {
            const uint32_t v = *reinterpret_cast<const uint32_t *>(box + r * 64u + (((c >> 2) ^ ((r >> 1) & 3u)) << 4) + (c & 3u) * 4u);
            if (row0 + r < P.p_rows && col0 + c < P.q_rows)
                static_cast<uint32_t *>(P.out)[uint64_t(row0 + r) * P.ldo + col0 + c] = v;
        }
    } else {
#pragma unroll 4
        for (uint32_t r = 0; r < 32; ++r) {
            const uint16_t v = *reinterpret_cast<const uint16_t *>(box + r * 64u + (((lane >> 3) ^ ((r >> 1) & 3u)) << 4) + (lane & 7u) * 2u);
            if (row0 + r < P.p_rows && col0 + lane < P.q_rows)
                static_cast<uint16_t *>(P.out)[uint64_t(row0 + r) * P.ldo + col0 + lane] = v;
        }
    }
}

// QROWS: a scale per row of Q (per column of the tile) instead of one per 128.
// SWAP: P is b and Q is a; the tile is stored turned.
template <int TN, bool QROWS, bool SWAP>
__global__ void __launch_bounds__(kThreads, 1) block_mm_kernel(const __grid_constant__ CUtensorMap map_p,
                                                               const __grid_constant__ CUtensorMap map_q,
                                                               const __grid_constant__ CUtensorMap map_out,
                                                               const BlockParams P) {
    using S = Shape<TN>;
    constexpr int kHalf = S::kHalf;
    constexpr int kChunk = kHalf < 16 ? kHalf : 16;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char *boxes = smem + S::kStages * S::kStageBytes;
    float *q_scale = reinterpret_cast<float *>(boxes + kEpiWarps * kBoxBytes);  // [2][TN]
    uint64_t *bars = reinterpret_cast<uint64_t *>(q_scale + 2 * TN);
    // bars: full[stages], empty[stages], acc_full[accs], acc_empty[accs], drain
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S::kStages + 2 * S::kAccs + 1);
    __shared__ volatile int abort_flag;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_u32(bars), empty = full + 8 * S::kStages;
    const uint32_t acc_full = empty + 8 * S::kStages, acc_empty = acc_full + 8 * S::kAccs;
    const uint32_t drain = acc_empty + 8 * S::kAccs;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < S::kAccs; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, kEpiWarps);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        abort_flag = 0;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(S::kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        // ---- producer ----
        uint32_t issued = 0;
        bool ok = true;
        for (uint32_t u = blockIdx.x; u < P.units && ok; u += gridDim.x) {
            const Unit t = unit_of(P, u);
            for (uint32_t kb = t.k0; kb < t.k1; ++kb, ++issued) {
                const uint32_t s = issued % S::kStages, use = issued / S::kStages;
                if (use > 0 && !mbar_wait(empty + 8 * s, (use - 1) & 1, &abort_flag)) {
                    ok = false;
                    break;
                }
                unsigned char *dst = smem + s * S::kStageBytes;
                mbar_expect_tx(full + 8 * s, S::kStageBytes);
                tma_load_2d(smem_u32(dst), &map_p, int(kb * kBlockK), int(t.tp * kTileP), full + 8 * s);
                tma_load_2d(smem_u32(dst + kPBytes), &map_q, int(kb * kBlockK), int(t.tq * TN), full + 8 * s);
            }
        }
        // own copies: the last use of every stage
        for (uint32_t l = issued > uint32_t(S::kStages) ? issued - S::kStages : 0; l < issued; ++l)
            mbar_wait(full + 8 * (l % S::kStages), (l / S::kStages) & 1, nullptr);
    } else if (warp == 1 && lane == 0) {
        // ---- MMA issuer: one accumulator per block of 128 ----
        uint32_t done = 0;
        bool ok = true;
        for (uint32_t u = blockIdx.x; u < P.units && ok; u += gridDim.x) {
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
                    mma_e4m3(tmem + b * TN, ad + uint64_t(2 * k), bd + uint64_t(2 * k), idesc<TN>(), k > 0 ? 1u : 0u);
                mma_commit(empty + 8 * s);
                mma_commit(acc_full + 8 * b);
            }
        }
        // no MMA may still be running when the accumulators are freed
        mma_commit(drain);
        mbar_wait(drain, 0, nullptr);
    } else if (warp >= 2) {
        // ---- sums and stores; every warp takes every block, also after a
        // wait gave up (the barriers below stay matched) ----
        const uint32_t quarter = warp & 3, half = (warp - 2) / 4, et = threadIdx.x - 64;
        unsigned char *box = boxes + (warp - 2) * kBoxBytes;
        uint32_t done = 0;
        bool bad = false;
        for (uint32_t u = blockIdx.x; u < P.units; u += gridDim.x) {
            const Unit t = unit_of(P, u);
            const uint32_t row0 = t.tp * kTileP + quarter * 32, row = row0 + lane;
            const uint32_t col0 = t.tq * TN + half * kHalf;
            const float *ps = P.p_scales + size_t(min(row, P.p_rows - 1) >> P.p_shift) * P.k_blocks;
            // QROWS: this thread's column of the tile; else the warp's columns' scale
            const uint32_t q_row = min(QROWS ? t.tq * TN + et : col0, P.q_rows - 1);
            const float *qs = P.q_scales + size_t(q_row >> P.q_shift) * P.k_blocks;
            float p_next = __ldg(ps + t.k0);
            float q_next = (!QROWS || et < TN) ? __ldg(qs + t.k0) : 0.0f;
            uint64_t acc[kHalf / 2];
#pragma unroll
            for (int i = 0; i < kHalf / 2; ++i) acc[i] = 0;
            for (uint32_t kb = t.k0; kb < t.k1; ++kb, ++done) {
                const uint32_t b = done % S::kAccs, turn = done / S::kAccs;
                const float p_cur = p_next, q_cur = q_next;
                float *q_buf = q_scale + (done & 1) * TN;
                if (QROWS && et < TN) q_buf[et] = q_cur;
                if (kb + 1 < t.k1) {
                    p_next = __ldg(ps + kb + 1);
                    if (!QROWS || et < TN) q_next = __ldg(qs + kb + 1);
                }
                if (!mbar_wait(acc_full + 8 * b, turn & 1, &abort_flag)) bad = true;
                asm volatile("tcgen05.fence::after_thread_sync;");
                if (QROWS) asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
                const uint32_t addr = tmem + ((quarter * 32) << 16) + b * TN + half * kHalf;
                const float one = QROWS ? p_cur : p_cur * q_cur;
                const uint64_t s2 = pair(one, one);
                uint32_t r[2][kChunk];
                tmem_load(r[0], addr);
#pragma unroll
                for (int c = 0; c < kHalf / kChunk; ++c) {
                    tmem_wait(r[c & 1]);
                    if (c + 1 < kHalf / kChunk) tmem_load(r[(c + 1) & 1], addr + (c + 1) * kChunk);
#pragma unroll
                    for (int i = 0; i < kChunk; i += 2) {
                        const uint64_t x = pair(__uint_as_float(r[c & 1][i]), __uint_as_float(r[c & 1][i + 1]));
                        uint64_t s = s2;
                        if (QROWS)
                            s = mul_pair(s2, *reinterpret_cast<const uint64_t *>(q_buf + half * kHalf + c * kChunk + i));
                        fma_pair(acc[(c * kChunk + i) / 2], x, s);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty + 8 * b);
            }
            if (bad) {
#pragma unroll
                for (int i = 0; i < kHalf / 2; ++i) acc[i] = 0x7fc000007fc00000ull;
            }
            if (P.splits > 1) {
                float4 *dst = P.parts + ((size_t(u) * kEpiWarps + (warp - 2)) * (kHalf / 4)) * 32 + lane;
#pragma unroll
                for (int i = 0; i < kHalf / 4; ++i) {
                    const float2 x = unpair(acc[2 * i]), y = unpair(acc[2 * i + 1]);
                    dst[i * 32] = make_float4(x.x, x.y, y.x, y.y);
                }
                continue;
            }
            if (SWAP) {
                // lane = column of out: the warp writes 32 consecutive elements
                const float bias = P.bias && row < P.p_rows ? bias_at(P, row) : 0.0f;
#pragma unroll
                for (int i = 0; i < kHalf / 2; ++i) {
                    const float2 x = unpair(acc[i]);
                    if (row < P.p_rows && col0 + 2 * i < P.q_rows)
                        store_value(P.out, P.out_dtype, uint64_t(col0 + 2 * i) * P.ldo + row, x.x + bias);
                    if (row < P.p_rows && col0 + 2 * i + 1 < P.q_rows)
                        store_value(P.out, P.out_dtype, uint64_t(col0 + 2 * i + 1) * P.ldo + row, x.y + bias);
                }
                continue;
            }
            if (P.bias) {
#pragma unroll
                for (int i = 0; i < kHalf / 2; ++i) {
                    const uint32_t n = col0 + 2 * i;
                    const float2 x = unpair(acc[i]);
                    acc[i] = pair(x.x + (n < P.q_rows ? bias_at(P, n) : 0.0f),
                                  x.y + (n + 1 < P.q_rows ? bias_at(P, n + 1) : 0.0f));
                }
            }
            if constexpr (kHalf >= 32) {
                if (P.out_dtype == SDFOAM_F32) {
#pragma unroll
                    for (int c = 0; c < kHalf / 16; ++c) {
                        if (col0 + c * 16 >= P.q_rows || row0 >= P.p_rows) continue;  // the same for every lane
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float2 x = unpair(acc[c * 8 + i]);
                            w[2 * i] = __float_as_uint(x.x);
                            w[2 * i + 1] = __float_as_uint(x.y);
                        }
                        store_box(P, &map_out, box, w, row0, col0 + c * 16, lane);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kHalf / 32; ++c) {
                        if (col0 + c * 32 >= P.q_rows || row0 >= P.p_rows) continue;
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float2 x = unpair(acc[c * 16 + i]);
                            w[i] = pack2(P.out_dtype, x.x, x.y);
                        }
                        store_box(P, &map_out, box, w, row0, col0 + c * 32, lane);
                    }
                }
            } else if (row < P.p_rows) {
                // at most 16 columns per thread
#pragma unroll
                for (int i = 0; i < kHalf / 2; ++i) {
                    const float2 x = unpair(acc[i]);
                    const uint64_t at = uint64_t(row) * P.ldo + col0 + 2 * i;
                    if (col0 + 2 * i < P.q_rows) store_value(P.out, P.out_dtype, at, x.x);
                    if (col0 + 2 * i + 1 < P.q_rows) store_value(P.out, P.out_dtype, at + 1, x.y);
                }
            }
        }
        // the TMA stores have read their boxes and are complete
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    if (abort_flag && threadIdx.x == 0) {
        *static_cast<volatile int *>(P.error) = 1;
        __threadfence_system();
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmemCols));
    }
}

// Adds the slices of a tile in order (parts: [tile][slice][warp][columns / 4]
// [lane] float4, the epilogue's own order) and the bias; also the product
// with an empty reduction (no slices).
template <int TN, bool SWAP>
__global__ void __launch_bounds__(256) join_slices_kernel(const BlockParams P) {
    constexpr int kHalf = TN / 2;
    constexpr uint32_t kPerTile = kEpiWarps * (kHalf / 4) * 32;
    const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
    const uint32_t tile = uint32_t(i / kPerTile), in = uint32_t(i % kPerTile);
    if (tile >= P.tiles_p * P.tiles_q) return;
    const uint32_t lane = in & 31, c4 = (in >> 5) % (kHalf / 4), w = (in >> 5) / (kHalf / 4);
    const Unit t = unit_of(P, tile * P.splits);
    const float4 *src = P.parts + size_t(tile) * P.splits * kPerTile + in;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t s = 0; s < P.splits; ++s) {
        const float4 x = __ldcs(src + size_t(s) * kPerTile);
        v[0] += x.x;
        v[1] += x.y;
        v[2] += x.z;
        v[3] += x.w;
    }
    // warp w of the epilogue: TMEM quarter (w + 2) % 4, half w / 4
    const uint32_t row = t.tp * kTileP + ((w + 2) & 3) * 32 + lane;
    const uint32_t col = t.tq * TN + (w / 4) * kHalf + c4 * 4;
    if (row >= P.p_rows) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= P.q_rows) return;
        const uint32_t n = SWAP ? row : col + e, m = SWAP ? col + e : row;
        if (P.bias) v[e] += bias_at(P, n);
        store_value(P.out, P.out_dtype, uint64_t(m) * P.ldo + n, v[e]);
    }
}

// The bias (or zero) everywhere: a product over nothing.
__global__ void __launch_bounds__(256) fill_bias_kernel(const BlockParams P, uint32_t m, uint32_t n) {
    const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= uint64_t(m) * n) return;
    const uint32_t r = uint32_t(i / n), c = uint32_t(i % n);
    store_value(P.out, P.out_dtype, uint64_t(r) * P.ldo + c, P.bias ? bias_at(P, c) : 0.0f);
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------

struct Plan {
    bool swap;
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
    const uint64_t tiles = uint64_t(l.tiles_p) * l.tiles_q;
    l.splits = tiles < kSms ? std::min<uint32_t>(l.k_blocks, uint32_t(kSms / tiles)) : 1;
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

// out [rows, cols] in boxes of 32 rows x 64 bytes, 64-byte swizzle.
bool output_map(CUtensorMap *map, void *base, uint32_t rows, uint32_t cols, uint64_t ld, uint32_t dtype) {
    auto fn = encode_fn();
    if (!fn) return false;
    const uint32_t size = dtype == SDFOAM_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {ld * size};
    const cuuint32_t box[2] = {64 / size, 32};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, dtype == SDFOAM_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base,
              dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TN, bool QROWS, bool SWAP>
cudaError_t launch_tiles(const CUtensorMap &mp, const CUtensorMap &mq, const CUtensorMap &mo, const BlockParams &P,
                         cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(block_mm_kernel<TN, QROWS, SWAP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         int(Shape<TN>::kSmem));
    if (e != cudaSuccess) return e;
    block_mm_kernel<TN, QROWS, SWAP><<<std::min<uint32_t>(P.units, kSms), kThreads, Shape<TN>::kSmem, stream>>>(mp, mq, mo, P);
    if ((e = cudaGetLastError()) != cudaSuccess || P.splits == 1) return e;
    const uint64_t threads = uint64_t(P.tiles_p) * P.tiles_q * kTileP * TN / 4;
    join_slices_kernel<TN, SWAP><<<unsigned((threads + 255) / 256), 256, 0, stream>>>(P);
    return cudaGetLastError();
}

template <int TN>
cudaError_t launch_tn(bool swap, const CUtensorMap &mp, const CUtensorMap &mq, const CUtensorMap &mo,
                      const BlockParams &P, cudaStream_t stream) {
    if constexpr (TN <= 64) {
        if (swap) {
            if (P.q_shift == 0) return launch_tiles<TN, true, true>(mp, mq, mo, P, stream);
            return launch_tiles<TN, false, true>(mp, mq, mo, P, stream);
        }
    }
    if (P.q_shift == 0) return launch_tiles<TN, true, false>(mp, mq, mo, P, stream);
    return launch_tiles<TN, false, false>(mp, mq, mo, P, stream);
}

}  // namespace

size_t block_matmul_workspace_bytes(uint32_t m, uint32_t n, uint32_t k) {
    if (m == 0 || n == 0 || k == 0) return 0;
    const Plan l = plan_of(m, n, k);
    return l.splits > 1 ? size_t(l.tiles_p) * l.tiles_q * l.splits * kTileP * l.tn * 4 : 0;
}

cudaError_t launch_block_matmul(const void *a, uint64_t lda, const float *a_scales, int a_block_rows, uint32_t m,
                                const void *b, uint64_t ldb, const float *b_scales, int b_block_rows, uint32_t n,
                                uint32_t k, const void *bias, uint32_t bias_dtype, void *out, uint64_t ldo,
                                uint32_t out_dtype, void *workspace, int *error, cudaStream_t stream) {
    if (m == 0 || n == 0) return cudaSuccess;
    BlockParams P{};
    P.bias = bias;
    P.bias_dtype = bias_dtype;
    P.out = out;
    P.ldo = ldo;
    P.out_dtype = out_dtype;
    if (k == 0) {
        fill_bias_kernel<<<unsigned((uint64_t(m) * n + 255) / 256), 256, 0, stream>>>(P, m, n);
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
    P.p_shift = (l.swap ? b_block_rows : a_block_rows) == 128 ? 7 : 0;
    P.q_shift = (l.swap ? a_block_rows : b_block_rows) == 128 ? 7 : 0;
    P.parts = static_cast<float4 *>(workspace);
    P.error = error;
    const uint32_t size = out_dtype == SDFOAM_F32 ? 4 : 2;
    P.box_store = !l.swap && l.splits == 1 && l.tn >= 64 && ((reinterpret_cast<uintptr_t>(out) | (ldo * size)) & 15u) == 0;
    CUtensorMap mp, mq, mo{};
    if (!operand_map(&mp, l.swap ? b : a, P.p_rows, k, l.swap ? ldb : lda, kTileP) ||
        !operand_map(&mq, l.swap ? a : b, P.q_rows, k, l.swap ? lda : ldb, uint32_t(l.tn)) ||
        (P.box_store && !output_map(&mo, out, m, n, ldo, out_dtype)))
        return cudaErrorInvalidValue;
    switch (l.tn) {
        case 16: return launch_tn<16>(l.swap, mp, mq, mo, P, stream);
        case 32: return launch_tn<32>(l.swap, mp, mq, mo, P, stream);
        case 64: return launch_tn<64>(l.swap, mp, mq, mo, P, stream);
        case 128: return launch_tn<128>(l.swap, mp, mq, mo, P, stream);
        default: return launch_tn<256>(l.swap, mp, mq, mo, P, stream);
    }
}

}  // namespace sdfoam_b200

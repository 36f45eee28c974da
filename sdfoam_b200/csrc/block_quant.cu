// e4m3 values with one scale per block of 128, from and to wider types.
//
// A block is `block_rows` x 128 elements, block_rows 1 (activations) or 128
// (weights).  Its scale is the smallest power of two s with s * 448 >= the
// block's largest magnitude (not below 2^-126; 1 for a block of zeros), and an
// element's value is x / s rounded to the nearest e4m3, ties to even.  Powers
// of two cost e4m3 no precision -- it is a floating type -- and make the
// division exact, so the values follow from the input alone, whatever the
// order or the kernel that computes them.  Infinities and NaN are left out of
// the largest magnitude and stored as NaN: they reach the products that read
// them and no other element of their block.
//
// A training step needs a matrix twice: in rows for the product and turned
// for the weight gradient, whose reduction runs over the rows, with blocks
// along that axis.  One pass over 128 x 128 tiles in registers writes either
// or both, so the input is read once.  Scales are stored block by block, the
// rows of one block of columns next to each other, as a product's tile reads
// them.  HBM bounds it (2 or 4 bytes in, one or two out per element):
// 1048576 x 256 bf16 turned in 141 us, 5.7 TB/s, in rows in 133, fp32 237 and
// 199 (turned 276 when each tile waited for its own loads).  Rows that are not
// whole 16-byte pieces are read element by element: 1048576 x 217 bf16 244 us
// in rows, fp32 273.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "foam_internal.h"

namespace sdfoam_b200 {

namespace {

constexpr int kThreads = 512;
constexpr uint32_t kTile = 128;
constexpr int kRows = 4;  // of a thread's piece of the tile, 8 columns wide

struct QuantParams {
    const void *x;
    size_t ld;  // elements
    uint32_t m, k;
    unsigned char *values, *turned;  // [m, ldv], [k, ldt]; either may be null
    size_t ldv, ldt;
    float *scales, *turned_scales;
    float *sums;                     // [ceil(m / 128), k] or null: sums of 128 rows
    uint32_t k_blocks, m_blocks;     // ceil(k / 128), ceil(m / 128)
};

// Scale of a block from its largest magnitude, as the bits of the scale's
// exponent: 448 = 1.75 * 2^8, so the scale is 2^(e - 8) when the magnitude
// 2^e * f has f <= 1.75 and 2^(e - 7) above.
__device__ __forceinline__ uint32_t scale_exponent(float largest) {
    const uint32_t bits = __float_as_uint(largest);
    if (bits == 0) return 127;
    const int e = int(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1u : uint32_t(e);
}
__device__ __forceinline__ float scale_value(uint32_t exponent) { return __uint_as_float(exponent << 23); }
__device__ __forceinline__ float scale_inverse(uint32_t exponent) { return __uint_as_float((254u - exponent) << 23); }

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Starts the copy of eight consecutive elements (zeros past `left`) into
// this thread's place of the staging buffer.
template <typename T>
__device__ __forceinline__ void stage8(unsigned char *dst, const T *src, int left) {
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) {
        const int bytes = max(0, min(16, left * int(sizeof(T)) - 16 * i));
        // a copy of nothing still needs an address of the matrix
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 16 * i),
                     "l"(bytes > 0 ? reinterpret_cast<const char *>(src) + 16 * i : reinterpret_cast<const char *>(src)),
                     "r"(bytes)
                     : "memory");
    }
}

// 128 x 128 tiles, one after another.  Thread (g, c) holds rows 4 g .. 4 g + 3
// and columns 8 c .. 8 c + 7: a row of the tile is 16 lanes' 16-byte copies,
// and the thread's 4 rows of one column are 4 consecutive bytes of the turned
// tile, which goes out through shared memory.  32 elements a thread keep it
// at 64 registers, two blocks of 16 warps to an SM; the next tile's copies
// (VEC: rows of 16-byte pieces) run while this one is worked on, each thread
// reading only what it copied itself.
template <typename T, bool VEC, int BLOCK_ROWS, bool NORMAL, bool TURNED>
__global__ void __launch_bounds__(kThreads, 2) quantize_kernel(const QuantParams P) {
    constexpr int kWarps = kThreads / 32;
    extern __shared__ __align__(16) unsigned char staged[];  // VEC: [2][kTile][kTile] of T
    __shared__ __align__(16) uint32_t tile[TURNED ? kTile * kTile / 4 : 4];
    __shared__ __align__(16) float tops[TURNED && BLOCK_ROWS == 1 ? kWarps : 1][kTile];
    __shared__ __align__(16) float inverses[TURNED && BLOCK_ROWS == 1 ? kTile : 4];
    __shared__ float top_all[kWarps];
    const uint32_t g = threadIdx.x >> 4, c = threadIdx.x & 15, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t tiles = P.k_blocks * P.m_blocks;

    auto prefetch = [&](uint32_t t, uint32_t buffer) {
        const uint32_t kb = t % P.k_blocks, mb = t / P.k_blocks;
        const uint32_t row = mb * kTile + g * kRows, col = kb * kTile + c * 8;
        unsigned char *dst = staged + ((buffer * kTile + g * kRows) * kTile + c * 8) * sizeof(T);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const bool in = row + r < P.m && col < P.k;
            const T *src = static_cast<const T *>(P.x) + (in ? size_t(row + r) * P.ld + col : 0);
            stage8<T>(dst + r * kTile * sizeof(T), src, in ? int(min(P.k - col, 8u)) : 0);
        }
    };
    if (VEC) {
        if (blockIdx.x < tiles) prefetch(blockIdx.x, 0);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    uint32_t buffer = 0;
    for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x, buffer ^= 1) {
        const uint32_t kb = t % P.k_blocks, mb = t / P.k_blocks;
        const uint32_t row0 = mb * kTile + g * kRows, col0 = kb * kTile + c * 8;
        const int left = int(P.k) - int(col0);

        float v[kRows][8];
        if (VEC) {
            if (t + gridDim.x < tiles) prefetch(t + gridDim.x, buffer ^ 1);
            asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;" ::: "memory");
            const unsigned char *src = staged + ((buffer * kTile + g * kRows) * kTile + c * 8) * sizeof(T);
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                union Eight {
                    uint4 q[sizeof(T) / 2];
                    T e[8];
                    __device__ Eight() {}
                } u;
#pragma unroll
                for (int i = 0; i < int(sizeof(T) / 2); ++i)
                    u.q[i] = *reinterpret_cast<const uint4 *>(src + r * kTile * sizeof(T) + 16 * i);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[r][i] = as_float(u.e[i]);
            }
        } else {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const T *src = static_cast<const T *>(P.x) + size_t(row0 + r) * P.ld + col0;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[r][i] = row0 + r < P.m && i < left ? as_float(src[i]) : 0.0f;
            }
        }
        if (TURNED && P.sums) {
            // column sums of the tile, rows in a fixed order
            float sum[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum[i] = (v[0][i] + v[1][i]) + (v[2][i] + v[3][i]);
                sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 16);
            }
            float *sums = reinterpret_cast<float *>(tile);  // [kWarps][kTile]
            if (lane < 16) {
#pragma unroll
                for (int i = 0; i < 8; i += 4)
                    *reinterpret_cast<float4 *>(sums + warp * kTile + c * 8 + i) =
                        make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
            }
            __syncthreads();
            if (threadIdx.x < kTile && kb * kTile + threadIdx.x < P.k) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) s += sums[w * kTile + threadIdx.x];
                P.sums[size_t(mb) * P.k + kb * kTile + threadIdx.x] = s;
            }
            __syncthreads();
        }
        // infinities become NaN, which the maxima below pass over (0 * v is 0
        // for every finite v, so most threads find none)
        float any = 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) any = fmaf(v[r][i], 0.0f, any);
        if (any != 0.0f) {
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (fabsf(v[r][i]) == __int_as_float(0x7f800000)) v[r][i] = __int_as_float(0x7fc00000);
        }

        uint32_t whole = 127;  // scale exponent of the 128 x 128 block
        if (BLOCK_ROWS == 128) {
            float top = 0.0f;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[r][i]));
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
            if (lane == 0) top_all[warp] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, top_all[w]);
            whole = scale_exponent(top);
            if (threadIdx.x == 0) {
                if (NORMAL) P.scales[size_t(kb) * P.m_blocks + mb] = scale_value(whole);
                if (TURNED) P.turned_scales[size_t(mb) * P.k_blocks + kb] = scale_value(whole);
            }
        }
        if (TURNED && BLOCK_ROWS == 1) {
            float top[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                top[i] = fmaxf(fmaxf(fabsf(v[0][i]), fabsf(v[1][i])), fmaxf(fabsf(v[2][i]), fabsf(v[3][i])));
                top[i] = fmaxf(0.0f, top[i]);  // four NaN
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
            }
            if (lane < 16) {
#pragma unroll
                for (int i = 0; i < 8; i += 4)
                    *reinterpret_cast<float4 *>(&tops[warp][c * 8 + i]) = make_float4(top[i], top[i + 1], top[i + 2], top[i + 3]);
            }
            __syncthreads();
            if (threadIdx.x < kTile) {
                float t = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) t = fmaxf(t, tops[w][threadIdx.x]);
                const uint32_t e = scale_exponent(t), col = kb * kTile + threadIdx.x;
                inverses[threadIdx.x] = scale_inverse(e);
                if (col < P.k) P.turned_scales[size_t(mb) * P.k + col] = scale_value(e);
            }
        }

        if (NORMAL) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                uint32_t exponent = whole;
                if (BLOCK_ROWS == 1) {
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[r][i]));
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    exponent = scale_exponent(top);
                }
                const float inv = scale_inverse(exponent);
                if (row0 + r < P.m) {
                    if (BLOCK_ROWS == 1 && c == 0) P.scales[size_t(kb) * P.m + row0 + r] = scale_value(exponent);
                    // whole 16-byte pieces of the row are written, zeros past k
                    if (col0 < ((P.k + 15u) & ~15u)) {
                        uint2 q;
                        q.x = pack4(v[r][0] * inv, v[r][1] * inv, v[r][2] * inv, v[r][3] * inv);
                        q.y = pack4(v[r][4] * inv, v[r][5] * inv, v[r][6] * inv, v[r][7] * inv);
                        *reinterpret_cast<uint2 *>(P.values + size_t(row0 + r) * P.ldv + col0) = q;
                    }
                }
            }
        }

        if (TURNED) {
            float inv[8];
            if (BLOCK_ROWS == 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 q = *reinterpret_cast<const float4 *>(&inverses[c * 8 + i]);
                    inv[i] = q.x;
                    inv[i + 1] = q.y;
                    inv[i + 2] = q.z;
                    inv[i + 3] = q.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) inv[i] = scale_inverse(whole);
            }
            // column j of the tile: 32 words of 4 rows, word g at place
            // g ^ 2 (j / 8), so that the lanes of a store fall on different banks
#pragma unroll
            for (int i = 0; i < 8; ++i)
                tile[(c * 8 + i) * 32 + (g ^ (2 * c))] = pack4(v[0][i] * inv[i], v[1][i] * inv[i], v[2][i] * inv[i], v[3][i] * inv[i]);
            __syncthreads();
            // 16 bytes per thread and turn: whole 16-byte pieces of the turned
            // rows, zeros past m
            const uint32_t m16 = (P.m + 15u) & ~15u;
#pragma unroll
            for (int i = 0; i < int(kTile * 8 / kThreads); ++i) {
                const uint32_t at = i * kThreads + threadIdx.x, j = at >> 3, s = at & 7, turn = (j >> 3) & 15;
                uint4 q = *reinterpret_cast<const uint4 *>(tile + j * 32 + ((s ^ (turn >> 1)) << 2));
                if (turn & 1) q = make_uint4(q.z, q.w, q.x, q.y);
                const uint32_t row = kb * kTile + j, col = mb * kTile + 16 * s;
                if (row < P.k && col < m16) *reinterpret_cast<uint4 *>(P.turned + size_t(row) * P.ldt + col) = q;
            }
        }
        if (TURNED || BLOCK_ROWS == 128) __syncthreads();  // the next tile takes the shared memory
    }
}

// out[c] = the sums of 128 rows, added up in order.
template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 32 columns per block, 32 runs of consecutive rows each; the runs' sums are
// added in order.
template <typename T>
__global__ void __launch_bounds__(1024) add_sums_kernel(const float *__restrict__ sums, uint32_t rows, uint32_t k,
                                                        T *__restrict__ out) {
    __shared__ float part[32][33];
    const uint32_t x = threadIdx.x & 31, y = threadIdx.x >> 5, col = blockIdx.x * 32 + x;
    const uint32_t per = (rows + 31) / 32, beg = min(rows, y * per), end = min(rows, beg + per);
    float s = 0.0f;
    if (col < k) {
#pragma unroll 8
        for (uint32_t r = beg; r < end; ++r) s += sums[size_t(r) * k + col];
    }
    part[y][x] = s;
    __syncthreads();
    if (y == 0 && col < k) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += part[i][x];
        out[col] = round_to<T>(t);
    }
}

// out[r, c] = values[r, c] * scales[r / block_rows, c / 128], in flat order:
// 16 bytes of out per thread and turn.  Where rows of values are as aligned
// (ALIGNED), a turn is one load of values and one of a scale, all turns' loads
// before the first store; elsewhere a byte per element, and a scale where a
// block or a row begins.  1048576 x 256 turned into fp32 201 us, 6.7 TB/s, in
// rows into bf16 126: HBM (1000000 x 256: 195 and 116; 2 turns 221 and 129; 4
// bytes of values to a turn, each turn waiting for its loads, 247 and 216).
// 1048576 x 217 into bf16 316, bound by the byte loads (1000000 rows: 302, and
// 544 with one element and one division per turn).
template <typename T>
__device__ __forceinline__ void store16(T *p, const float *v);
template <>
__device__ __forceinline__ void store16<float>(float *p, const float *v) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <>
__device__ __forceinline__ void store16<__half>(__half *p, const float *v) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}
template <>
__device__ __forceinline__ void store16<__nv_bfloat16>(__nv_bfloat16 *p, const float *v) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}

__device__ __forceinline__ float e4m3_float(uint32_t byte) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
    return __half2float(__half(h));
}

constexpr int kDequantThreads = 256, kDequantItems = 4;

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kDequantThreads) dequantize_kernel(const unsigned char *__restrict__ values, size_t ldv,
                                                              const float *__restrict__ scales, uint32_t shift,
                                                              size_t scale_row, size_t scale_block, uint64_t total,
                                                              uint32_t k, bool wide, T *__restrict__ out) {
    constexpr int kVec = 16 / sizeof(T);  // elements per turn
    const uint64_t first = uint64_t(blockIdx.x) * (kDequantThreads * kDequantItems * kVec);
    const uint64_t row0 = first / k;
    const uint32_t col0 = uint32_t(first - row0 * k);
    auto scale_at = [&](uint64_t row, uint32_t col) {
        return __ldg(scales + (row >> shift) * scale_row + (col >> 7) * scale_block);
    };
    if constexpr (ALIGNED) {
        uint32_t w[kDequantItems][kVec / 4];
        float s[kDequantItems];
#pragma unroll
        for (int t = 0; t < kDequantItems; ++t) {
            const uint32_t e = (t * kDequantThreads + threadIdx.x) * kVec;
            if (first + e < total) {
                const uint32_t r = (col0 + e) / k, col = (col0 + e) - r * k;
                const uint32_t *src = reinterpret_cast<const uint32_t *>(values + (row0 + r) * ldv + col);
                if constexpr (kVec == 8) {
                    const uint2 q = __ldg(reinterpret_cast<const uint2 *>(src));
                    w[t][0] = q.x;
                    w[t][1] = q.y;
                } else {
                    w[t][0] = __ldg(src);
                }
                s[t] = scale_at(row0 + r, col);
            }
        }
#pragma unroll
        for (int t = 0; t < kDequantItems; ++t) {
            const uint32_t e = (t * kDequantThreads + threadIdx.x) * kVec;
            if (first + e < total) {
                float v[kVec];
#pragma unroll
                for (int i = 0; i < kVec; ++i) v[i] = s[t] * e4m3_float((w[t][i / 4] >> (8 * (i % 4))) & 255u);
                store16<T>(out + first + e, v);
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < kDequantItems; ++t) {
            const uint32_t e = (t * kDequantThreads + threadIdx.x) * kVec;
            if (first + e >= total) return;
            const int left = int(min(uint64_t(kVec), total - first - e));
            uint32_t col = (col0 + e) / k;
            uint64_t row = row0 + col;
            col = (col0 + e) - col * k;
            float v[kVec], s = scale_at(row, col);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (i < left) {
                    v[i] = s * e4m3_float(__ldg(values + row * ldv + col));
                    if (++col == k) {
                        col = 0;
                        ++row;
                    }
                    if ((col & 127u) == 0 && i + 1 < left) s = scale_at(row, col);
                }
            }
            T *const dst = out + first + e;
            if (wide && left == kVec) {
                store16<T>(dst, v);
            } else {
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                    if (i < left) dst[i] = round_to<T>(v[i]);
            }
        }
    }
}

template <typename T, bool VEC, int BLOCK_ROWS, bool NORMAL, bool TURNED>
cudaError_t quantize_launch(const QuantParams &P, cudaStream_t stream) {
    auto kernel = quantize_kernel<T, VEC, BLOCK_ROWS, NORMAL, TURNED>;
    constexpr size_t kStaged = VEC ? 2 * kTile * kTile * sizeof(T) : 0;
    // two blocks of an SM where their staging fits, one for fp32
    constexpr unsigned kResident = sizeof(T) == 4 && VEC ? 148 : 2 * 148;
    if (kStaged > 0) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kStaged));
        if (e != cudaSuccess) return e;
    }
    kernel<<<std::min(P.k_blocks * P.m_blocks, kResident), kThreads, kStaged, stream>>>(P);
    return cudaGetLastError();
}

template <typename T, bool VEC, int BLOCK_ROWS>
cudaError_t quantize_out(const QuantParams &P, cudaStream_t stream) {
    if (P.values && P.turned) return quantize_launch<T, VEC, BLOCK_ROWS, true, true>(P, stream);
    if (P.values) return quantize_launch<T, VEC, BLOCK_ROWS, true, false>(P, stream);
    return quantize_launch<T, VEC, BLOCK_ROWS, false, true>(P, stream);
}

template <typename T>
cudaError_t quantize_typed(const QuantParams &P, int block_rows, cudaStream_t stream) {
    const bool vec = ((reinterpret_cast<uintptr_t>(P.x) | (P.ld * sizeof(T))) & 15u) == 0;
    if (vec) return block_rows == 1 ? quantize_out<T, true, 1>(P, stream) : quantize_out<T, true, 128>(P, stream);
    return block_rows == 1 ? quantize_out<T, false, 1>(P, stream) : quantize_out<T, false, 128>(P, stream);
}

template <typename T>
void dequantize_typed(const void *values, size_t ldv, const float *scales, size_t scale_row, size_t scale_block,
                      int block_rows, uint32_t m, uint32_t k, void *out, cudaStream_t stream) {
    constexpr uint32_t kVec = 16 / sizeof(T);
    const bool wide = (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
    const bool aligned = wide && ((k | ldv | reinterpret_cast<uintptr_t>(values)) & (kVec - 1)) == 0;
    const uint32_t shift = block_rows == 128 ? 7 : 0;
    const uint64_t per = kDequantThreads * kDequantItems * kVec, total = uint64_t(m) * k;
    const unsigned blocks = unsigned((total + per - 1) / per);
    const unsigned char *v = static_cast<const unsigned char *>(values);
    if (aligned) dequantize_kernel<T, true><<<blocks, kDequantThreads, 0, stream>>>(v, ldv, scales, shift, scale_row, scale_block, total, k, wide, static_cast<T *>(out));
    else dequantize_kernel<T, false><<<blocks, kDequantThreads, 0, stream>>>(v, ldv, scales, shift, scale_row, scale_block, total, k, wide, static_cast<T *>(out));
}

}  // namespace

cudaError_t launch_block_quantize(const void *x, size_t ld, uint32_t dtype, uint32_t m, uint32_t k, int block_rows,
                                  void *values, size_t ldv, float *scales, void *turned, size_t ldt,
                                  float *turned_scales, float *sums, void *column_sums, uint32_t sums_dtype,
                                  cudaStream_t stream) {
    if (m == 0 || k == 0) return cudaSuccess;
    QuantParams P{};
    P.x = x;
    P.ld = ld;
    P.m = m;
    P.k = k;
    P.values = static_cast<unsigned char *>(values);
    P.turned = static_cast<unsigned char *>(turned);
    P.ldv = ldv;
    P.ldt = ldt;
    P.scales = scales;
    P.turned_scales = turned_scales;
    P.sums = column_sums ? sums : nullptr;
    P.k_blocks = (k + kTile - 1) / kTile;
    P.m_blocks = (m + kTile - 1) / kTile;
    const cudaError_t e = dtype == SDFOAM_F32   ? quantize_typed<float>(P, block_rows, stream)
                          : dtype == SDFOAM_F16 ? quantize_typed<__half>(P, block_rows, stream)
                                                : quantize_typed<__nv_bfloat16>(P, block_rows, stream);
    if (e != cudaSuccess || !column_sums) return e;
    const unsigned columns = (k + 31) / 32;
    switch (sums_dtype) {
        case SDFOAM_F32: add_sums_kernel<<<columns, 1024, 0, stream>>>(sums, P.m_blocks, k, static_cast<float *>(column_sums)); break;
        case SDFOAM_F16: add_sums_kernel<<<columns, 1024, 0, stream>>>(sums, P.m_blocks, k, static_cast<__half *>(column_sums)); break;
        default: add_sums_kernel<<<columns, 1024, 0, stream>>>(sums, P.m_blocks, k, static_cast<__nv_bfloat16 *>(column_sums)); break;
    }
    return cudaGetLastError();
}

cudaError_t launch_block_dequantize(const void *values, size_t ldv, const float *scales, size_t scale_row,
                                    size_t scale_block, int block_rows, uint32_t m, uint32_t k, uint32_t dtype,
                                    void *out, cudaStream_t stream) {
    if (m == 0 || k == 0) return cudaSuccess;
    switch (dtype) {
        case SDFOAM_F32: dequantize_typed<float>(values, ldv, scales, scale_row, scale_block, block_rows, m, k, out, stream); break;
        case SDFOAM_F16: dequantize_typed<__half>(values, ldv, scales, scale_row, scale_block, block_rows, m, k, out, stream); break;
        default: dequantize_typed<__nv_bfloat16>(values, ldv, scales, scale_row, scale_block, block_rows, m, k, out, stream); break;
    }
    return cudaGetLastError();
}

}  // namespace sdfoam_b200

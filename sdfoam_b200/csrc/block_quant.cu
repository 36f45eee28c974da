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
// them.  HBM bounds it (2 or 4 bytes in, one
// or two out per element).
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "foam_internal.h"

namespace sdfoam_b200 {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kTile = 128;
constexpr int kRows = 8;  // rows and columns of a thread's piece of the tile

struct QuantParams {
    const void *x;
    size_t ld;  // elements
    uint32_t m, k;
    unsigned char *values, *turned;  // [m, ldv], [k, ldt]; either may be null
    size_t ldv, ldt;
    float *scales, *turned_scales;
    uint32_t k_blocks, m_blocks;     // ceil(k / 128), ceil(m / 128)
};

// Scale of a block from the bits of its largest magnitude, as the bits of
// the scale's exponent: 448 = 1.75 * 2^8, so the scale is 2^(e - 8) when the
// magnitude 2^e * f has f <= 1.75 and 2^(e - 7) above.
__device__ __forceinline__ uint32_t scale_exponent(uint32_t largest) {
    if (largest == 0) return 127;
    const int e = int(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1u : uint32_t(e);
}
__device__ __forceinline__ float scale_value(uint32_t exponent) { return __uint_as_float(exponent << 23); }
__device__ __forceinline__ float scale_inverse(uint32_t exponent) { return __uint_as_float((254u - exponent) << 23); }

// The magnitude's bits, 0 for infinities and NaN.
__device__ __forceinline__ uint32_t magnitude(float v) {
    const uint32_t a = __float_as_uint(v) & 0x7fffffffu;
    return a < 0x7f800000u ? a : 0u;
}

// v / scale; NaN for infinities and NaN (v - v is 0 for every other v).
__device__ __forceinline__ float scaled(float v, float inverse) { return fmaf(v, inverse, v - v); }

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Eight consecutive elements, zeros past k.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *src, int left, float *v) {
    if (VEC && left >= 8) {
        union {
            uint4 q[sizeof(T) / 2];
            T e[8];
            __device__ uint4 &operator[](int i) { return q[i]; }
        } u = {};
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) u.q[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = as_float(u.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? as_float(src[i]) : 0.0f;
    }
}

// One 128 x 128 tile per block.  Thread (g, c) holds rows 8 g .. 8 g + 7 and
// columns 8 c .. 8 c + 7: a row of the tile is 16 lanes' 16-byte loads, and
// the thread's 8 rows of one column are 8 consecutive bytes of the turned
// tile, which goes out through shared memory.
template <typename T, bool VEC, int BLOCK_ROWS, bool NORMAL, bool TURNED>
__global__ void __launch_bounds__(kThreads, 2) quantize_kernel(const QuantParams P) {
    __shared__ __align__(16) unsigned char tile[TURNED ? kTile * kTile : 16];
    __shared__ uint32_t tops[TURNED && BLOCK_ROWS == 1 ? 8 : 1][kTile];
    __shared__ uint32_t top_all[8];
    const uint32_t g = threadIdx.x >> 4, c = threadIdx.x & 15, warp = threadIdx.x >> 5;
    const uint32_t kb = blockIdx.x % P.k_blocks, mb = blockIdx.x / P.k_blocks;
    const uint32_t row0 = mb * kTile + g * kRows, col0 = kb * kTile + c * 8;
    const int left = int(P.k) - int(col0);

    float v[kRows][8];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (row0 + r < P.m && left > 0) {
            load8<T, VEC>(static_cast<const T *>(P.x) + size_t(row0 + r) * P.ld + col0, left, v[r]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = 0.0f;
        }
    }

    uint32_t whole = 127;  // scale exponent of the 128 x 128 block
    if (BLOCK_ROWS == 128) {
        uint32_t top = 0;
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[r][i]));
        top = __reduce_max_sync(0xffffffffu, top);
        if ((threadIdx.x & 31) == 0) top_all[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) top = max(top, top_all[w]);
        whole = scale_exponent(top);
        if (threadIdx.x == 0) {
            if (NORMAL) P.scales[size_t(kb) * P.m_blocks + mb] = scale_value(whole);
            if (TURNED) P.turned_scales[size_t(mb) * P.k_blocks + kb] = scale_value(whole);
        }
    }

    if (NORMAL) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            uint32_t exponent = whole;
            if (BLOCK_ROWS == 1) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[r][i]));
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                exponent = scale_exponent(top);
            }
            const float inv = scale_inverse(exponent);
            if (row0 + r < P.m) {
                if (BLOCK_ROWS == 1 && c == 0) P.scales[size_t(kb) * P.m + row0 + r] = scale_value(exponent);
                // whole 16-byte pieces of the row are written, zeros past k
                if (col0 < ((P.k + 15u) & ~15u)) {
                    uint2 q;
                    q.x = pack4(scaled(v[r][0], inv), scaled(v[r][1], inv), scaled(v[r][2], inv), scaled(v[r][3], inv));
                    q.y = pack4(scaled(v[r][4], inv), scaled(v[r][5], inv), scaled(v[r][6], inv), scaled(v[r][7], inv));
                    *reinterpret_cast<uint2 *>(P.values + size_t(row0 + r) * P.ldv + col0) = q;
                }
            }
        }
    }

    if (TURNED) {
        uint32_t exponent[8];
        if (BLOCK_ROWS == 1) {
            uint32_t top[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                top[i] = 0;
#pragma unroll
                for (int r = 0; r < kRows; ++r) top[i] = max(top[i], magnitude(v[r][i]));
                top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
            }
            if ((threadIdx.x & 31) < 16) {
#pragma unroll
                for (int i = 0; i < 8; ++i) tops[warp][c * 8 + i] = top[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int w = 0; w < 8; ++w) top[i] = max(top[i], tops[w][c * 8 + i]);
                exponent[i] = scale_exponent(top[i]);
            }
            if (g == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < left) P.turned_scales[size_t(mb) * P.k + col0 + i] = scale_value(exponent[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) exponent[i] = whole;
        }
        // column j of the tile: 16 pieces of 8 rows, piece g at place
        // g ^ (j / 8), so that the lanes of a store fall on different banks
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float inv = scale_inverse(exponent[i]);
            uint2 q;
            q.x = pack4(scaled(v[0][i], inv), scaled(v[1][i], inv), scaled(v[2][i], inv), scaled(v[3][i], inv));
            q.y = pack4(scaled(v[4][i], inv), scaled(v[5][i], inv), scaled(v[6][i], inv), scaled(v[7][i], inv));
            *reinterpret_cast<uint2 *>(tile + (c * 8 + i) * kTile + ((g ^ c) << 3)) = q;
        }
        __syncthreads();
        // 16 bytes (two pieces) per thread and turn: whole 16-byte pieces of
        // the turned rows, zeros past m
        const uint32_t m16 = (P.m + 15u) & ~15u;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t at = t * kThreads + threadIdx.x, j = at >> 3, s = at & 7, turn = (j >> 3) & 15;
            uint4 q = *reinterpret_cast<const uint4 *>(tile + j * kTile + (((2 * s) ^ (turn & ~1u)) << 3));
            if (turn & 1) q = make_uint4(q.z, q.w, q.x, q.y);
            const uint32_t row = kb * kTile + j, col = mb * kTile + 16 * s;
            if (row < P.k && col < m16) *reinterpret_cast<uint4 *>(P.turned + size_t(row) * P.ldt + col) = q;
        }
    }
}

// out[r, c] = values[r, c] * scales[r / block_rows, c / 128], four columns
// per thread where the rows allow it.
template <typename T>
__device__ __forceinline__ void store4(T *p, const float *v);
template <>
__device__ __forceinline__ void store4<float>(float *p, const float *v) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <>
__device__ __forceinline__ void store4<__half>(__half *p, const float *v) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16 *p, const float *v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

__device__ __forceinline__ void store1(float *p, float v) { *p = v; }
__device__ __forceinline__ void store1(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float e4m3_float(uint32_t byte) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
    return __half2float(__half(h));
}

constexpr int kDequantItems = 4;

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const unsigned char *__restrict__ values, size_t ldv,
                                                              const float *__restrict__ scales, uint32_t shift,
                                                              size_t scale_row, size_t scale_block, uint32_t m,
                                                              uint32_t k, uint32_t units,
                                                              T *__restrict__ out) {
    const uint64_t total = uint64_t(m) * units;
    const uint64_t first = uint64_t(blockIdx.x) * (kThreads * kDequantItems);
    const uint64_t row0 = first / units;
    const uint32_t col0 = uint32_t(first - row0 * units);
#pragma unroll
    for (int t = 0; t < kDequantItems; ++t) {
        const uint32_t e = t * kThreads + threadIdx.x;
        if (first + e >= total) return;
        const uint32_t r = (col0 + e) / units, u = (col0 + e) - r * units, col = u * VEC;
        const uint64_t row = row0 + r;
        const float s = __ldg(scales + (row >> shift) * scale_row + (col >> 7) * scale_block);
        const unsigned char *src = values + row * ldv + col;
        T *dst = out + row * k + col;
        if (VEC == 4) {
            const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(src));
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = s * e4m3_float((w >> (8 * i)) & 255u);
            store4<T>(dst, v);
        } else {
            store1(dst, s * e4m3_float(*src));
        }
    }
}

template <typename T, bool VEC, int BLOCK_ROWS>
void quantize_out(const QuantParams &P, unsigned blocks, cudaStream_t stream) {
    if (P.values && P.turned) quantize_kernel<T, VEC, BLOCK_ROWS, true, true><<<blocks, kThreads, 0, stream>>>(P);
    else if (P.values) quantize_kernel<T, VEC, BLOCK_ROWS, true, false><<<blocks, kThreads, 0, stream>>>(P);
    else quantize_kernel<T, VEC, BLOCK_ROWS, false, true><<<blocks, kThreads, 0, stream>>>(P);
}

template <typename T>
void quantize_typed(const QuantParams &P, int block_rows, unsigned blocks, cudaStream_t stream) {
    const bool vec = ((reinterpret_cast<uintptr_t>(P.x) | (P.ld * sizeof(T))) & 15u) == 0;
    if (vec && block_rows == 1) quantize_out<T, true, 1>(P, blocks, stream);
    else if (vec) quantize_out<T, true, 128>(P, blocks, stream);
    else if (block_rows == 1) quantize_out<T, false, 1>(P, blocks, stream);
    else quantize_out<T, false, 128>(P, blocks, stream);
}

template <typename T>
void dequantize_typed(const void *values, size_t ldv, const float *scales, size_t scale_row, size_t scale_block,
                      int block_rows, uint32_t m, uint32_t k, void *out, cudaStream_t stream) {
    const bool vec = k % 4 == 0 && ldv % 4 == 0 && (reinterpret_cast<uintptr_t>(values) & 3u) == 0 &&
                     (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
    const uint32_t units = vec ? k / 4 : k, shift = block_rows == 128 ? 7 : 0;
    const uint64_t per = kThreads * kDequantItems;
    const unsigned blocks = unsigned((uint64_t(m) * units + per - 1) / per);
    const unsigned char *v = static_cast<const unsigned char *>(values);
    if (vec) dequantize_kernel<T, 4><<<blocks, kThreads, 0, stream>>>(v, ldv, scales, shift, scale_row, scale_block, m, k, units, static_cast<T *>(out));
    else dequantize_kernel<T, 1><<<blocks, kThreads, 0, stream>>>(v, ldv, scales, shift, scale_row, scale_block, m, k, units, static_cast<T *>(out));
}

}  // namespace

cudaError_t launch_block_quantize(const void *x, size_t ld, uint32_t dtype, uint32_t m, uint32_t k, int block_rows,
                                  void *values, size_t ldv, float *scales, void *turned, size_t ldt,
                                  float *turned_scales, cudaStream_t stream) {
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
    P.k_blocks = (k + kTile - 1) / kTile;
    P.m_blocks = (m + kTile - 1) / kTile;
    const unsigned blocks = P.k_blocks * P.m_blocks;
    switch (dtype) {
        case SDFOAM_F32: quantize_typed<float>(P, block_rows, blocks, stream); break;
        case SDFOAM_F16: quantize_typed<__half>(P, block_rows, blocks, stream); break;
        default: quantize_typed<__nv_bfloat16>(P, block_rows, blocks, stream); break;
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

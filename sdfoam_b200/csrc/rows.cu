// Rows of a table at given ids, and the table's gradient by sorted ids.
//
//   lookup    out[i, :] = scale * table[ids[i], :]
//   gradient  grad_table[v, :] = scale * sum over i with ids[i] = v of grad[i, :]
//
// An id outside [0, rows) names no row: its output row is zero and it adds
// to no gradient (sdfoam_nn and the walks write UINT32_MAX for "none").
// Products and sums are fp32, rounded once to the table's type.
//
// Both are bound by HBM: a lookup moves each row once in and once out.  The
// gradient sorts (id, position) pairs -- a stable sort, so the rows of one id
// are added in ascending position and the result is the same every run --
// and then streams the gradient rows once, in id order:
//   * the sorted entries are cut into equal chunks; a group of lanes, one
//     lane per 16 bytes of a row, adds a chunk's rows in registers and writes
//     a row of the result whenever the id changes;
//   * a segment that crosses a chunk's end leaves its parts in the workspace
//     (at most two per chunk), and a second launch adds them in order;
//   * rows that no id names are written as zeros by blocks of the same
//     launch, from a byte per row that the sort's first pass sets -- the
//     result is written exactly once.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "foam_internal.h"

namespace sdfoam_b200 {

namespace {

// --------------------------------------------------------------------------
// element and index types
// --------------------------------------------------------------------------

template <typename I>
__device__ __forceinline__ uint32_t row_of(I id, uint32_t rows) {
    // the id as a row number, or `rows` when it names none
    if constexpr (sizeof(I) == 8) return static_cast<unsigned long long>(id) < rows ? uint32_t(id) : rows;
    else return uint32_t(id) < rows ? uint32_t(id) : rows;
}

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VB bytes of a row: what one lane loads at a time.
template <int VB>
struct Word;
template <>
struct Word<16> { using type = uint4; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<2> { using type = uint16_t; };

template <typename T, int VB>
union Unit {
    typename Word<VB>::type word;
    T item[VB / sizeof(T)];
    __device__ Unit() {}
};

// --------------------------------------------------------------------------
// lookup
// --------------------------------------------------------------------------

constexpr int kLookupThreads = 256;

// Units of VB bytes in the flat order of the output, ITEMS per thread: the
// block's first unit is divided by the units per row in 64 bits, the rest of
// the positions follow from 32-bit offsets.  Consecutive lanes write
// consecutive units whatever the row length.
template <typename T, typename I, int VB, int ITEMS>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(const char *__restrict__ table, uint32_t rows,
                                                                size_t row_bytes, const I *__restrict__ ids,
                                                                uint64_t total, uint32_t units, float scale,
                                                                char *__restrict__ out) {
    using W = typename Word<VB>::type;
    const uint64_t first = uint64_t(blockIdx.x) * (kLookupThreads * ITEMS);
    const uint64_t row0 = first / units;
    const uint32_t col0 = uint32_t(first - row0 * units);
    uint32_t col[ITEMS], row[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const uint32_t e = col0 + j * kLookupThreads + threadIdx.x;  // < units + 2048: fits
        const uint32_t r = e / units;
        col[j] = e - r * units;
        row[j] = first + j * kLookupThreads + threadIdx.x < total ? row_of(ids[row0 + r], rows) : rows;
    }
    Unit<T, VB> u[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        u[j].word = W{};
        if (row[j] < rows) u[j].word = *reinterpret_cast<const W *>(table + size_t(row[j]) * row_bytes + size_t(col[j]) * VB);
    }
    W *dst = reinterpret_cast<W *>(out) + first + threadIdx.x;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        if (scale != 1.0f) {
#pragma unroll
            for (int e = 0; e < int(VB / sizeof(T)); ++e)
                if (row[j] < rows) u[j].item[e] = from_f<T>(scale * to_f<T>(u[j].item[e]));
        }
        if (first + j * kLookupThreads + threadIdx.x < total) dst[j * kLookupThreads] = u[j].word;
    }
}

// --------------------------------------------------------------------------
// gradient: keys
// --------------------------------------------------------------------------

// keys[i] = the row id i names, or `rows` (sorts last); vals[i] = i; touched
// rows are marked.
template <typename I>
__global__ void __launch_bounds__(256) row_keys_kernel(const I *__restrict__ ids, uint32_t n, uint32_t rows,
                                                       uint32_t *__restrict__ keys, uint32_t *__restrict__ vals,
                                                       unsigned char *__restrict__ touched) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t k = row_of(ids[i], rows);
    keys[i] = k;
    vals[i] = i;
    if (k < rows) touched[k] = 1;
}

// --------------------------------------------------------------------------
// gradient: sums of sorted rows
// --------------------------------------------------------------------------

constexpr int kSumThreads = 256;
constexpr int kAhead = 4;            // rows in flight per lane and unit
constexpr uint32_t kNoPart = 0xffffffffu;

struct SumParams {
    const uint32_t *keys, *vals;  // sorted
    uint32_t n, rows;
    const char *grad;             // [n] rows of units * VB bytes, grad_bytes apart
    size_t grad_bytes;
    uint32_t units;               // per row
    int lane_bits;                // log2 of the lanes of a group
    int lane_units;               // units that a group takes of a row: R << lane_bits
    uint32_t chunk, chunks;       // entries per chunk, number of chunks
    float scale;
    char *out;                    // [rows][units] contiguous
    const unsigned char *touched;
    float *parts;                 // [2 * chunks][columns]: the chunk's first and last segment
    uint32_t columns;             // elements per row
    uint32_t sum_blocks;          // blocks of sums; the others write zero rows
};

// The blocks behind the sums': zeros for the rows that no id names.
template <int VB>
__device__ __forceinline__ void zero_rows(const SumParams &P, uint32_t block, uint32_t blocks) {
    using W = typename Word<VB>::type;
    const uint64_t total = uint64_t(P.rows) * P.units;
    constexpr int kItems = 8;
    const uint64_t step = uint64_t(blocks) * kSumThreads * kItems;
    W *dst = reinterpret_cast<W *>(P.out);
    for (uint64_t first = uint64_t(block) * kSumThreads * kItems; first < total; first += step) {
        const uint64_t row0 = first / P.units;
        const uint32_t col0 = uint32_t(first - row0 * P.units);
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const uint32_t e = j * kSumThreads + threadIdx.x;
            if (first + e < total && !P.touched[row0 + (col0 + e) / P.units]) dst[first + e] = W{};
        }
    }
}

// A group of 1 << lane_bits lanes adds one chunk, R units per lane; the
// columns past lane_units are other blocks' (blockIdx.y).  parts: a segment
// that starts before the chunk goes to part 2c, one that ends after it to
// 2c + 1 (a segment that does both only to 2c).
template <typename T, int VB, int R>
__global__ void __launch_bounds__(kSumThreads) sum_rows_kernel(const SumParams P) {
    using W = typename Word<VB>::type;
    constexpr int E = VB / int(sizeof(T));
    if (blockIdx.x >= P.sum_blocks) {
        if (blockIdx.y == 0) zero_rows<VB>(P, blockIdx.x - P.sum_blocks, gridDim.x - P.sum_blocks);
        return;
    }
    const uint32_t lanes = 1u << P.lane_bits, lane = threadIdx.x & (lanes - 1);
    const uint32_t c = blockIdx.x * (kSumThreads >> P.lane_bits) + (threadIdx.x >> P.lane_bits);
    if (c >= P.chunks) return;
    const uint32_t beg = c * P.chunk, end = min(P.n, beg + P.chunk);
    const uint32_t u0 = blockIdx.y * P.lane_units + lane;  // this lane's units: u0 + r * lanes

    float acc[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = 0.0f;

    uint32_t cur = P.keys[beg];
    bool open = beg > 0 && P.keys[beg - 1] == cur;  // the segment began before this chunk

    auto flush = [&](uint32_t key, bool more) {
        if (key >= P.rows) return;  // ids that name no row
        if (open || more) {
            float *part = P.parts + size_t(2 * c + (open ? 0 : 1)) * P.columns;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t u = u0 + r * lanes;
                if (u < P.units)
#pragma unroll
                    for (int e = 0; e < E; ++e) part[size_t(u) * E + e] = acc[r][e];
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t u = u0 + r * lanes;
                if (u < P.units) {
                    Unit<T, VB> w;
#pragma unroll
                    for (int e = 0; e < E; ++e) w.item[e] = from_f<T>(P.scale * acc[r][e]);
                    reinterpret_cast<W *>(P.out)[size_t(key) * P.units + u] = w.word;
                }
            }
        }
    };

    for (uint32_t j0 = beg; j0 < end; j0 += kAhead) {
        uint32_t key[kAhead];
        Unit<T, VB> w[kAhead][R];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t j = min(j0 + a, end - 1);
            key[a] = P.keys[j];
            const bool named = key[a] < P.rows && j0 + a < end;
            const char *src = P.grad + size_t(P.vals[j]) * P.grad_bytes;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t u = u0 + r * lanes;
                w[a][r].word = W{};
                if (named && u < P.units) w[a][r].word = *reinterpret_cast<const W *>(src + size_t(u) * VB);
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (j0 + a >= end) break;
            if (key[a] != cur) {
                flush(cur, false);
                cur = key[a];
                open = false;
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[r][e] = 0.0f;
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[r][e] += to_f<T>(w[a][r].item[e]);
        }
    }
    flush(cur, end < P.n && P.keys[end] == cur);
}

// Adds the parts of the segments that cross chunk ends.  The chunk a segment
// starts in owns it: its last part, then the first parts of the chunks that
// follow while they continue the segment.  A block takes kJoinChunks chunks;
// segments of many chunks (hot ids) are shared by the block's threads, each
// taking a contiguous run of the parts, and their sums are added in order.
constexpr int kJoinThreads = 256;
constexpr int kJoinChunks = 8;
constexpr int kJoinSlices = 16;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_parts_kernel(const SumParams P) {
    __shared__ float partial[kJoinSlices][kJoinThreads / kJoinSlices];
    constexpr uint32_t kCols = kJoinThreads / kJoinSlices;  // columns of a slice's threads
    const uint32_t slice = threadIdx.x / kCols, tc = threadIdx.x % kCols;
    for (uint32_t i = 0; i < uint32_t(kJoinChunks); ++i) {
        const uint32_t c = blockIdx.x * kJoinChunks + i;
        if (c + 1 >= P.chunks) return;
        const uint32_t end = (c + 1) * P.chunk, beg = end - P.chunk;
        const uint32_t key = P.keys[end - 1];
        if (key >= P.rows || P.keys[end] != key) continue;                             // nothing crosses this end
        if (beg > 0 && P.keys[beg] == key && P.keys[beg - 1] == key) continue;         // another chunk owns it
        // last chunk with entries of this segment: the first entry past it by bisection
        uint32_t lo = end, hi = P.n;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (P.keys[mid] <= key) lo = mid + 1;
            else hi = mid;
        }
        const uint32_t last = (lo - 1) / P.chunk;
        const uint32_t count = last - c;  // first parts of chunks c + 1 .. last
        if (count < 4 * kJoinSlices) {
            for (uint32_t col = threadIdx.x; col < P.columns; col += kJoinThreads) {
                float s = P.parts[size_t(2 * c + 1) * P.columns + col];
                for (uint32_t k = 1; k <= count; ++k) s += P.parts[size_t(2 * (c + k)) * P.columns + col];
                reinterpret_cast<T *>(P.out)[size_t(key) * P.columns + col] = from_f<T>(P.scale * s);
            }
            continue;
        }
        const uint32_t per = (count + kJoinSlices - 1) / kJoinSlices;
        const uint32_t k0 = 1 + slice * per, k1 = min(count + 1, k0 + per);
        for (uint32_t col0 = 0; col0 < P.columns; col0 += kCols) {
            const uint32_t col = col0 + tc;
            float s = 0.0f;
            if (col < P.columns)
                for (uint32_t k = k0; k < k1; ++k) s += P.parts[size_t(2 * (c + k)) * P.columns + col];
            partial[slice][tc] = s;
            __syncthreads();
            if (slice == 0 && col < P.columns) {
                float t = P.parts[size_t(2 * c + 1) * P.columns + col];
                for (int q = 0; q < kJoinSlices; ++q) t += partial[q][tc];
                reinterpret_cast<T *>(P.out)[size_t(key) * P.columns + col] = from_f<T>(P.scale * t);
            }
            __syncthreads();
        }
    }
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------

size_t type_size(uint32_t dtype) { return dtype == SDFOAM_F32 ? 4 : 2; }

// The widest unit that rows of `bytes` bytes, `stride` bytes apart from
// `base`, are whole numbers of.
int unit_bytes(const void *base, size_t stride, size_t bytes) {
    const size_t all = reinterpret_cast<uintptr_t>(base) | stride | bytes;
    return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// Entries per chunk: enough chunks to fill the GPU (a chunk is a warp or
// less; 148 SMs x 64), and no more parts than needed.
uint32_t chunk_of(uint32_t n) {
    uint32_t c = 4;
    while (c < 128 && uint64_t(c) * 148 * 64 < n) c *= 2;
    return c;
}

struct RowGradLayout {
    size_t keys[2], vals[2], hist, totals, touched, parts, total;
    uint32_t chunk, chunks;
};

RowGradLayout grad_layout(uint32_t n, uint32_t rows, uint32_t columns) {
    RowGradLayout l{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes, 256);
        return here;
    };
    for (int i = 0; i < 2; ++i) {
        l.keys[i] = take(size_t(n) * 4);
        l.vals[i] = take(size_t(n) * 4);
    }
    l.hist = take(radix_hist_entries(n) * 4);
    l.totals = take(256 * 4);
    l.touched = take(rows);
    l.chunk = chunk_of(n);
    l.chunks = (n + l.chunk - 1) / l.chunk;
    l.parts = take(size_t(2) * l.chunks * columns * 4);
    l.total = at;
    return l;
}

template <typename T, typename I, int VB>
cudaError_t lookup_typed(const void *table, uint32_t rows, size_t row_bytes, const void *ids, uint64_t n,
                         uint32_t units, float scale, void *out, cudaStream_t stream) {
    const uint64_t total = n * units;
    // few units: more blocks of fewer items
    if (total < 148ull * 2048 * 4) {
        lookup_kernel<T, I, VB, 2><<<unsigned((total + 511) / 512), kLookupThreads, 0, stream>>>(
            static_cast<const char *>(table), rows, row_bytes, static_cast<const I *>(ids), total, units, scale,
            static_cast<char *>(out));
    } else {
        lookup_kernel<T, I, VB, 8><<<unsigned((total + 2047) / 2048), kLookupThreads, 0, stream>>>(
            static_cast<const char *>(table), rows, row_bytes, static_cast<const I *>(ids), total, units, scale,
            static_cast<char *>(out));
    }
    return cudaGetLastError();
}

template <typename T, typename I>
cudaError_t lookup_unit(int vb, const void *table, uint32_t rows, size_t row_bytes, const void *ids, uint64_t n,
                        uint32_t columns, float scale, void *out, cudaStream_t stream) {
    const uint32_t units = uint32_t(columns * sizeof(T) / vb);
    switch (vb) {
        case 16: return lookup_typed<T, I, 16>(table, rows, row_bytes, ids, n, units, scale, out, stream);
        case 8: return lookup_typed<T, I, 8>(table, rows, row_bytes, ids, n, units, scale, out, stream);
        case 4: return lookup_typed<T, I, 4>(table, rows, row_bytes, ids, n, units, scale, out, stream);
        default: break;
    }
    if constexpr (sizeof(T) == 2) return lookup_typed<T, I, 2>(table, rows, row_bytes, ids, n, units, scale, out, stream);
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t lookup_index(uint32_t itype, int vb, const void *table, uint32_t rows, size_t row_bytes, const void *ids,
                         uint64_t n, uint32_t columns, float scale, void *out, cudaStream_t stream) {
    // 32-bit ids: a signed one below 0 is past every row as an unsigned one
    if (itype == SDFOAM_I64)
        return lookup_unit<T, long long>(vb, table, rows, row_bytes, ids, n, columns, scale, out, stream);
    return lookup_unit<T, uint32_t>(vb, table, rows, row_bytes, ids, n, columns, scale, out, stream);
}

template <typename T, int VB>
cudaError_t sum_typed(SumParams &P, cudaStream_t stream) {
    P.units = uint32_t(P.columns * sizeof(T) / VB);
    P.lane_bits = 0;
    while (P.lane_bits < 5 && (1u << P.lane_bits) < P.units) ++P.lane_bits;
    const uint32_t lanes = 1u << P.lane_bits;
    const uint32_t per_lane = (P.units + lanes - 1) / lanes;
    const int R = per_lane >= 3 && VB < 16 ? 4 : per_lane >= 2 ? 2 : 1;
    P.lane_units = int(lanes) * R;
    const uint32_t groups = kSumThreads / lanes;
    P.sum_blocks = (P.chunks + groups - 1) / groups;
    const uint64_t zero_units = uint64_t(P.rows) * P.units;
    const uint32_t zero_blocks = uint32_t(std::min<uint64_t>((zero_units + 2047) / 2048, 148 * 4));
    const dim3 grid(P.sum_blocks + zero_blocks, (P.units + P.lane_units - 1) / P.lane_units);
    if (R == 4) sum_rows_kernel<T, VB, (VB < 16 ? 4 : 2)><<<grid, kSumThreads, 0, stream>>>(P);
    else if (R == 2) sum_rows_kernel<T, VB, 2><<<grid, kSumThreads, 0, stream>>>(P);
    else sum_rows_kernel<T, VB, 1><<<grid, kSumThreads, 0, stream>>>(P);
    if (P.chunks > 1)
        join_parts_kernel<T><<<(P.chunks + kJoinChunks - 1) / kJoinChunks, kJoinThreads, 0, stream>>>(P);
    return cudaGetLastError();
}

template <typename T>
cudaError_t sum_unit(int vb, SumParams &P, cudaStream_t stream) {
    switch (vb) {
        case 16: return sum_typed<T, 16>(P, stream);
        case 8: return sum_typed<T, 8>(P, stream);
        case 4: return sum_typed<T, 4>(P, stream);
        default: break;
    }
    if constexpr (sizeof(T) == 2) return sum_typed<T, 2>(P, stream);
    return cudaErrorInvalidValue;
}

}  // namespace

size_t lookup_grad_workspace_bytes(uint32_t n, uint32_t rows, uint32_t columns) {
    return n == 0 ? 0 : grad_layout(n, rows, columns).total;
}

cudaError_t launch_lookup_rows(const void *table, uint32_t rows, uint32_t columns, size_t ld, uint32_t dtype,
                               const void *ids, uint64_t n, uint32_t itype, float scale, void *out,
                               cudaStream_t stream) {
    if (n == 0 || columns == 0) return cudaSuccess;
    const size_t bytes = size_t(columns) * type_size(dtype), row_bytes = ld * type_size(dtype);
    const int vb = std::min(unit_bytes(table, row_bytes, bytes), unit_bytes(out, bytes, bytes));
    switch (dtype) {
        case SDFOAM_F32: return lookup_index<float>(itype, vb, table, rows, row_bytes, ids, n, columns, scale, out, stream);
        case SDFOAM_F16: return lookup_index<__half>(itype, vb, table, rows, row_bytes, ids, n, columns, scale, out, stream);
        default: return lookup_index<__nv_bfloat16>(itype, vb, table, rows, row_bytes, ids, n, columns, scale, out, stream);
    }
}

cudaError_t launch_lookup_rows_backward(const void *grad, size_t ld, uint32_t columns, uint32_t dtype, const void *ids,
                                        uint32_t n, uint32_t itype, float scale, void *out, uint32_t rows,
                                        void *workspace, cudaStream_t stream) {
    if (rows == 0 || columns == 0) return cudaSuccess;
    const size_t size = type_size(dtype);
    if (n == 0) return cudaMemsetAsync(out, 0, size_t(rows) * columns * size, stream);
    const RowGradLayout l = grad_layout(n, rows, columns);
    char *ws = static_cast<char *>(workspace);
    uint32_t *keys[2], *vals[2];
    for (int i = 0; i < 2; ++i) {
        keys[i] = reinterpret_cast<uint32_t *>(ws + l.keys[i]);
        vals[i] = reinterpret_cast<uint32_t *>(ws + l.vals[i]);
    }
    unsigned char *touched = reinterpret_cast<unsigned char *>(ws + l.touched);
    cudaError_t e = cudaMemsetAsync(touched, 0, rows, stream);
    if (e != cudaSuccess) return e;
    const unsigned blocks = (n + 255) / 256;
    if (itype == SDFOAM_I64)
        row_keys_kernel<<<blocks, 256, 0, stream>>>(static_cast<const long long *>(ids), n, rows, keys[0], vals[0], touched);
    else
        row_keys_kernel<<<blocks, 256, 0, stream>>>(static_cast<const uint32_t *>(ids), n, rows, keys[0], vals[0], touched);
    int bits = 0;  // of the largest key, `rows`
    while (bits < 32 && (uint64_t(rows) >> bits) != 0) ++bits;
    int cur = 0;
    e = launch_radix_sort_pairs(keys, vals, n, reinterpret_cast<uint32_t *>(ws + l.hist),
                                reinterpret_cast<uint32_t *>(ws + l.totals), cur, stream, bits);
    if (e != cudaSuccess) return e;
    SumParams P{};
    P.keys = keys[cur];
    P.vals = vals[cur];
    P.n = n;
    P.rows = rows;
    P.grad = static_cast<const char *>(grad);
    P.grad_bytes = ld * size;
    P.chunk = l.chunk;
    P.chunks = l.chunks;
    P.scale = scale;
    P.out = static_cast<char *>(out);
    P.touched = touched;
    P.parts = reinterpret_cast<float *>(ws + l.parts);
    P.columns = columns;
    const size_t bytes = size_t(columns) * size;
    const int vb = std::min(unit_bytes(grad, P.grad_bytes, bytes), unit_bytes(out, bytes, bytes));
    switch (dtype) {
        case SDFOAM_F32: return sum_unit<float>(vb, P, stream);
        case SDFOAM_F16: return sum_unit<__half>(vb, P, stream);
        default: return sum_unit<__nv_bfloat16>(vb, P, stream);
    }
}

}  // namespace sdfoam_b200

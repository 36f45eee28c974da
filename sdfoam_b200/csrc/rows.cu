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
//   * rows that no id names are written as zeros by more blocks of that
//     launch, from a byte per row that the sums set -- the result is written
//     exactly once.
// Measured: 1M rows of 49 floats at skewed ids of a 4M-row table in 97 us
// (312 MB at least; 425 move, since 196-byte rows start anywhere in a 64-byte
// line); the gradient of 2M rows of 48 floats in 190 us, of which the sums
// take 104 (5.4 TB/s), the sort 68 and the joins 17; of 512k bf16 rows of 256
// into 1M in 193 (sums 86, zeros and joins 65, sort 42).  The lookups of 16-bit
// elements by 16 bytes, 8 units a thread, spill 4 bytes; no other kernel does.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "foam_internal.h"

namespace sdfoam_b200 {

namespace {

// --------------------------------------------------------------------------
// element and index types
// --------------------------------------------------------------------------

// The id as a row number below `limit`, or `none` when it names no such row.
template <typename I>
__device__ __forceinline__ uint32_t row_of(I id, uint32_t limit, uint32_t none) {
    if constexpr (sizeof(I) == 8) return static_cast<unsigned long long>(id) < limit ? uint32_t(id) : none;
    else return uint32_t(id) < limit ? uint32_t(id) : none;
}

// The rows that ids of a type can name: 32-bit ids are compared as unsigned
// numbers, where a negative signed one is 2^31 or more.
uint32_t nameable_rows(uint32_t rows, uint32_t itype) {
    return itype == SDFOAM_I32 ? std::min(rows, 1u << 31) : rows;
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

// x / d and x % d, in 32 bits where x allows.
__device__ __forceinline__ uint64_t divide(uint64_t x, uint32_t d, uint32_t &rem) {
    if (x >> 32) {
        const uint64_t q = x / d;
        rem = uint32_t(x - q * d);
        return q;
    }
    const uint32_t q = uint32_t(x) / d;
    rem = uint32_t(x) - q * d;
    return q;
}

// Units of VB bytes in the flat order of the output, ITEMS per thread, 256
// apart: consecutive lanes write consecutive units whatever the row length.
// A thread divides its first unit by the units per row; the others follow by
// step_row rows and step_col units (256 divided by the units per row).
template <typename T, typename I, int VB, int ITEMS>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(const char *__restrict__ table, uint32_t rows,
                                                                size_t row_bytes, const I *__restrict__ ids,
                                                                uint64_t total, uint32_t units, uint32_t step_row,
                                                                uint32_t step_col, float scale,
                                                                char *__restrict__ out) {
    using W = typename Word<VB>::type;
    const uint64_t first = uint64_t(blockIdx.x) * (kLookupThreads * ITEMS);
    uint32_t col[ITEMS], row[ITEMS];
    {
        uint32_t c;
        const uint64_t r0 = divide(first + threadIdx.x, units, c);
        const I *id = ids + r0;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            col[j] = c;
            row[j] = first + j * kLookupThreads + threadIdx.x < total ? row_of(*id, rows, rows) : rows;
            c += step_col;
            id += step_row;
            if (c >= units) {
                c -= units;
                ++id;
            }
        }
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
        if (first + j * kLookupThreads + threadIdx.x < total) __stcs(dst + j * kLookupThreads, u[j].word);
    }
}

// --------------------------------------------------------------------------
// gradient: a stable sort of (row, position)
// --------------------------------------------------------------------------
//
// Least significant digit first, digits of at most 9 bits (as few passes as
// the number of rows needs, of equal width).  A pass over tiles of 2048
// counts the digits of each tile, scans the counts, and scatters: every warp
// ranks its 256 consecutive entries by ballots over the digit's bits and its
// own digit counts (with __match_any_sync a pass over 2M entries takes 33 to
// 38 us instead of 21), the tile is put in order in shared memory and leaves
// in runs of equal digits.  The first pass reads the ids themselves.
//
// Launches count where there are few ids.  Up to 96 tiles need no scan: every
// block adds up the counts of the tiles before its own, and a pass counts the
// next one's digits while it writes (integer atomics: the same counts in any
// order).  180k ids with the scan and without it, the call: 47 and 42 us for
// 41450 rows of 3 bf16, 137 and 125 us for 1M rows of 49 floats, 33 and 34 us
// for 300 rows of 16; replayed in a graph 31 and 34, 117 and 116, 24 and 29.
// 250k ids (123 tiles): the call 49 and 50, 148 and 143, 36 and 42.  Up to
// 8192 entries are sorted by one block in one launch (4097: the same time on
// the GPU as five launches, 8 us less with the call).

constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;
constexpr uint32_t kSortTile = kSortThreads * kSortItems;
constexpr int kMaxBins = 512;
constexpr uint32_t kBlockSort = 8192;  // entries that one block sorts
constexpr uint32_t kFewTiles = 96;
constexpr int kMaxPasses = 4;          // 32 bits by 9

uint32_t sort_tiles(uint32_t n) { return (n + kSortTile - 1) / kSortTile; }

struct SortPass {
    const void *ids;               // the first pass's input
    const uint32_t *keys_in, *vals_in;
    uint32_t *keys_out, *vals_out;
    uint32_t *counts;              // [bins][tiles], then its exclusive scan along the tiles;
                                   // few tiles: [tiles][bins]
    uint32_t *next_counts;         // few tiles: the next pass's, or null
    uint32_t clear_counts;         // few tiles, first pass: words behind counts that later passes add to
    uint32_t *totals;              // [bins]
    uint32_t n, rows, tiles;
    uint32_t named;                // rows that an id of the type can name; an id without a row sorts as `rows`
    int shift, bins;
    unsigned char *touched;        // cleared by the first pass
};

template <typename I, bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const SortPass &P, uint32_t i) {
    if constexpr (FIRST) return row_of(static_cast<const I *>(P.ids)[i], P.named, P.rows);
    else return P.keys_in[i];
}

// Clears bytes [block * share, ...) of the rows' marks.
__device__ __forceinline__ void clear_touched(unsigned char *touched, uint32_t rows, uint32_t block, uint32_t blocks) {
    const uint64_t words = (uint64_t(rows) + 15) / 16;  // the array is padded to 256 bytes
    for (uint64_t w = uint64_t(block) * blockDim.x + threadIdx.x; w < words; w += uint64_t(blocks) * blockDim.x)
        reinterpret_cast<uint4 *>(touched)[w] = make_uint4(0, 0, 0, 0);
}

template <typename I, bool FIRST, bool FEW>
__global__ void __launch_bounds__(kSortThreads) digit_counts_kernel(const SortPass P) {
    __shared__ uint32_t count[kMaxBins];
    for (int b = threadIdx.x; b < P.bins; b += kSortThreads) count[b] = 0;
    if (FIRST) clear_touched(P.touched, P.rows, blockIdx.x, gridDim.x);
    if (FEW)
        for (uint32_t w = blockIdx.x * kSortThreads + threadIdx.x; w < P.clear_counts; w += gridDim.x * kSortThreads)
            P.counts[P.tiles * P.bins + w] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kSortTile, mask = P.bins - 1;
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const uint32_t i = base + r * kSortThreads + threadIdx.x;
        if (i < P.n) atomicAdd(&count[(sort_key<I, FIRST>(P, i) >> P.shift) & mask], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < P.bins; b += kSortThreads)
        P.counts[FEW ? blockIdx.x * P.bins + b : size_t(b) * P.tiles + blockIdx.x] = count[b];
}

// Exclusive scan of each digit's counts along the tiles, one warp per digit.
__global__ void __launch_bounds__(256) scan_counts_kernel(const SortPass P) {
    const uint32_t b = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (b >= uint32_t(P.bins)) return;
    uint32_t *row = P.counts + size_t(b) * P.tiles;
    uint32_t carry = 0;
    for (uint32_t t0 = 0; t0 < P.tiles; t0 += 128) {
        uint32_t v[4], incl[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t t = t0 + q * 32 + lane;
            v[q] = t < P.tiles ? row[t] : 0u;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            incl[q] = v[q];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, incl[q], o);
                if (lane >= uint32_t(o)) incl[q] += y;
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t t = t0 + q * 32 + lane;
            if (t < P.tiles) row[t] = carry + incl[q] - v[q];
            carry += __shfl_sync(0xffffffffu, incl[q], 31);
        }
    }
    if (lane == 0) P.totals[b] = carry;
}

// The lanes whose digit (of at most 9 bits) is this lane's, among the valid ones.
__device__ __forceinline__ uint32_t same_digit(uint32_t digit, bool valid, int width) {
    uint32_t peers = __ballot_sync(0xffffffffu, valid);
#pragma unroll
    for (int b = 0; b < 9; ++b) {
        if (b >= width) break;
        const uint32_t set = __ballot_sync(0xffffffffu, (digit >> b) & 1u);
        peers &= (digit >> b) & 1u ? set : ~set;
    }
    return peers;
}

// Ranks WARPS x items x 32 entries (warp w's are consecutive) by their digit
// and puts them in order in shared memory: rank[] are this thread's places.
// counts: [WARPS][bins], start: [bins + 1] first place of each digit.
template <int WARPS, int ITEMS>
__device__ __forceinline__ void rank_digits(const uint32_t (&digit)[ITEMS], uint32_t (&rank)[ITEMS], uint16_t *counts,
                                            uint32_t *start, uint32_t *warp_sums, int bins, int items = ITEMS) {
    const int width = 31 - __clz(bins);
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lt = (1u << lane) - 1u;
    constexpr uint32_t kThreads = WARPS * 32;
    for (uint32_t i = threadIdx.x; i < uint32_t(WARPS * bins); i += kThreads) counts[i] = 0;
    __syncthreads();
    uint16_t *mine = counts + warp * bins;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        if (r >= items) break;  // the same for every thread
        const uint32_t d = digit[r];
        const bool valid = d < uint32_t(bins);
        const uint32_t peers = same_digit(d, valid, width);
        uint32_t before = 0;
        if (valid) before = mine[d];
        __syncwarp();
        if (valid && (peers & lt) == 0) mine[d] = uint16_t(before + __popc(peers));
        __syncwarp();
        rank[r] = before + __popc(peers & lt);
    }
    __syncthreads();
    // per digit: where each warp's entries start within the digit, and the
    // digit's total; then the digits' starts
    uint32_t carry = 0;
    for (int b0 = 0; b0 < bins; b0 += int(kThreads)) {
        const int b = b0 + int(threadIdx.x);
        uint32_t total = 0;
        if (b < bins) {
#pragma unroll 8
            for (int w = 0; w < WARPS; ++w) {
                const uint32_t c = counts[w * bins + b];
                counts[w * bins + b] = uint16_t(total);
                total += c;
            }
        }
        uint32_t incl = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= uint32_t(o)) incl += y;
        }
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        uint32_t before = carry, all = 0;
#pragma unroll 8
        for (int w = 0; w < WARPS; ++w) {
            if (uint32_t(w) < warp) before += warp_sums[w];
            all += warp_sums[w];
        }
        if (b < bins) start[b] = before + incl - total;
        carry += all;
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (digit[r] < uint32_t(bins)) rank[r] += mine[digit[r]] + start[digit[r]];
}

template <typename I, bool FIRST, bool FEW>
__global__ void __launch_bounds__(kSortThreads) scatter_digits_kernel(const SortPass P) {
    constexpr int kWarps = kSortThreads / 32;
    __shared__ uint32_t keys[kSortTile];
    __shared__ union {
        uint16_t counts[kWarps * kMaxBins];
        uint32_t vals[kSortTile];
    } u;
    __shared__ uint32_t start[kMaxBins], base[kMaxBins], warp_sums[kWarps];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mask = P.bins - 1;
    const uint32_t tile0 = blockIdx.x * kSortTile, valid = min(kSortTile, P.n - tile0);
    const uint32_t first = warp * (32 * kSortItems) + lane;
    // everything this block reads, before the ranking
    uint32_t key[kSortItems], val[kSortItems], digit[kSortItems], rank[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const uint32_t i = first + r * 32;
        key[r] = i < valid ? sort_key<I, FIRST>(P, tile0 + i) : 0u;
        val[r] = FIRST ? tile0 + i : i < valid ? P.vals_in[tile0 + i] : 0u;
        digit[r] = i < valid ? (key[r] >> P.shift) & mask : 0xffffffffu;
    }
    constexpr int kBinsPer = kMaxBins / kSortThreads;
    uint32_t total[kBinsPer], earlier[kBinsPer];
#pragma unroll
    for (int q = 0; q < kBinsPer; ++q) {
        const int b = q * kSortThreads + int(threadIdx.x);
        total[q] = earlier[q] = 0;
        if (b < P.bins) {
            if (FEW) {
#pragma unroll 8
                for (uint32_t t = 0; t < P.tiles; ++t) {
                    const uint32_t x = P.counts[t * P.bins + b];
                    total[q] += x;
                    if (t < blockIdx.x) earlier[q] += x;
                }
            } else {
                total[q] = P.totals[b];
                earlier[q] = P.counts[size_t(b) * P.tiles + blockIdx.x];
            }
        }
    }
    rank_digits<kWarps, kSortItems>(digit, rank, u.counts, start, warp_sums, P.bins);
    // the digit's first place in the output: entries of smaller digits, this
    // digit's in earlier tiles, less the tile's own start
    __syncthreads();
    uint32_t carry = 0;
#pragma unroll
    for (int q = 0; q < kBinsPer; ++q) {
        const int b = q * kSortThreads + int(threadIdx.x);
        uint32_t incl = total[q];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= uint32_t(o)) incl += y;
        }
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        uint32_t before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (uint32_t(w) < warp) before += warp_sums[w];
            all += warp_sums[w];
        }
        if (b < P.bins) base[b] = before + incl - total[q] + earlier[q] - start[b];
        carry += all;
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kSortItems; ++r)
        if (first + r * 32 < valid) keys[rank[r]] = key[r];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < valid; i += kSortThreads) {
        const uint32_t k = keys[i], at = base[(k >> P.shift) & mask] + i;
        if (at < P.n) {  // always, for consistent counts; keeps the store in bounds
            P.keys_out[at] = k;
            if (FEW && P.next_counts)
                atomicAdd(P.next_counts + at / kSortTile * P.bins + ((k >> P.shift) / P.bins & mask), 1u);
        }
    }
    // the values, in the order of their keys (the counts are no longer needed)
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const uint32_t i = first + r * 32;
        if (i < valid) u.vals[rank[r]] = val[r];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < valid; i += kSortThreads) {
        const uint32_t at = base[(keys[i] >> P.shift) & mask] + i;
        if (at < P.n) P.vals_out[at] = u.vals[i];
    }
}

// Up to kBlockSort entries: block 0 sorts them, digits of 8 bits; the others
// clear the rows' marks.
constexpr int kBlockSortThreads = 1024;
constexpr int kBlockSortBins = 256;
constexpr size_t block_sort_smem(int items) {
    return size_t(kBlockSortThreads) * items * 8 + kBlockSortThreads / 32 * kBlockSortBins * 2 + kBlockSortBins * 4 + 128;
}

template <typename I, int kItems>
__global__ void __launch_bounds__(kBlockSortThreads) sort_block_kernel(const SortPass P, int bits) {
    extern __shared__ __align__(16) unsigned char raw[];
    if (blockIdx.x > 0) {
        clear_touched(P.touched, P.rows, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    constexpr int kWarps = kBlockSortThreads / 32;
    uint32_t *keys = reinterpret_cast<uint32_t *>(raw), *vals = keys + kBlockSortThreads * kItems;
    uint16_t *counts = reinterpret_cast<uint16_t *>(vals + kBlockSortThreads * kItems);
    uint32_t *start = reinterpret_cast<uint32_t *>(counts + kWarps * kBlockSortBins), *warp_sums = start + kBlockSortBins;
    // no more items per thread than there are: warp w's are consecutive
    const int items = int((P.n + kBlockSortThreads - 1) / kBlockSortThreads);
    const uint32_t first = (threadIdx.x >> 5) * (32 * items) + (threadIdx.x & 31);
    uint32_t key[kItems], val[kItems], digit[kItems], rank[kItems];
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
        val[r] = first + r * 32;
        key[r] = r < items && val[r] < P.n ? sort_key<I, true>(P, val[r]) : 0u;
    }
    for (int shift = 0; shift < bits; shift += 8) {
#pragma unroll
        for (int r = 0; r < kItems; ++r)
            digit[r] = r < items && first + r * 32 < P.n ? (key[r] >> shift) & (kBlockSortBins - 1) : 0xffffffffu;
        rank_digits<kWarps, kItems>(digit, rank, counts, start, warp_sums, kBlockSortBins, items);
#pragma unroll
        for (int r = 0; r < kItems; ++r)
            if (r < items && first + r * 32 < P.n) {
                keys[rank[r]] = key[r];
                vals[rank[r]] = val[r];
            }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kItems; ++r)
            if (r < items && first + r * 32 < P.n) {
                key[r] = keys[first + r * 32];
                val[r] = vals[first + r * 32];
            }
    }
#pragma unroll
    for (int r = 0; r < kItems; ++r)
        if (r < items && first + r * 32 < P.n) {
            P.keys_out[first + r * 32] = key[r];
            P.vals_out[first + r * 32] = val[r];
        }
}

// --------------------------------------------------------------------------
// gradient: sums of sorted rows
// --------------------------------------------------------------------------

constexpr int kSumThreads = 128;
constexpr int kJoinThreads = 512;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr uint32_t kJoinSlices = 32;
constexpr uint32_t kJoinLong = 16;  // chunks that a warp adds alone
constexpr int kAhead = 4;            // rows in flight per lane and unit

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
    unsigned char *touched;       // [rows]: 1 for the rows that an id names
    float *parts;                 // [2 * chunks][columns]: the chunk's first and last segment
    uint32_t columns;             // elements per row
    uint32_t join_blocks;         // of the join's launch; the others write zero rows
};

// The blocks behind the join's: zeros for the rows that no id names.
template <int VB>
__device__ __forceinline__ void zero_rows(const SumParams &P, uint32_t block, uint32_t blocks) {
    using W = typename Word<VB>::type;
    const uint64_t total = uint64_t(P.rows) * P.units;
    constexpr int kItems = 8;
    const uint64_t step = uint64_t(blocks) * kJoinThreads * kItems;
    const uint32_t step_row = kJoinThreads / P.units, step_col = kJoinThreads % P.units;
    W *dst = reinterpret_cast<W *>(P.out);
    for (uint64_t first = uint64_t(block) * kJoinThreads * kItems; first < total; first += step) {
        uint32_t col;
        uint64_t row = divide(first + threadIdx.x, P.units, col);
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const uint64_t at = first + j * kJoinThreads + threadIdx.x;
            if (at < total && !P.touched[row]) dst[at] = W{};
            col += step_col;
            row += step_row;
            if (col >= P.units) {
                col -= P.units;
                ++row;
            }
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
        if (lane == 0 && blockIdx.y == 0) P.touched[key] = 1;
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

    // the entries of the next rows are read while these rows are on their way
    uint32_t next_key[kAhead], next_val[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
        const uint32_t j = min(beg + a, end - 1);
        next_key[a] = P.keys[j];
        next_val[a] = P.vals[j];
    }
    for (uint32_t j0 = beg; j0 < end; j0 += kAhead) {
        uint32_t key[kAhead];
        Unit<T, VB> w[kAhead][R];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            key[a] = next_key[a];
            const bool named = key[a] < P.rows && j0 + a < end;
            const char *src = P.grad + size_t(next_val[a]) * P.grad_bytes;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t u = u0 + r * lanes;
                w[a][r].word = W{};
                if (named && u < P.units) w[a][r].word = __ldcs(reinterpret_cast<const W *>(src + size_t(u) * VB));
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t j = min(j0 + kAhead + a, end - 1);
            next_key[a] = P.keys[j];
            next_val[a] = P.vals[j];
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
// follow while they continue the segment.  A warp looks at one chunk and adds
// a segment of few chunks itself; segments of many (hot ids) are shared by
// the block's threads, each taking a contiguous run of the parts, and the
// runs' sums are added in order.
template <typename T, int VB>
__global__ void __launch_bounds__(kJoinThreads) join_parts_kernel(const SumParams P) {
    if (blockIdx.x >= P.join_blocks) {
        zero_rows<VB>(P, blockIdx.x - P.join_blocks, gridDim.x - P.join_blocks);
        return;
    }
    constexpr uint32_t kCols = kJoinThreads / kJoinSlices;  // columns of a slice's threads
    __shared__ float partial[kJoinSlices][kCols];
    __shared__ uint32_t long_key[kJoinWarps], long_count[kJoinWarps];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t c = blockIdx.x * kJoinWarps + warp;
    if (lane == 0) long_count[warp] = 0;
    if (c + 1 < P.chunks) {
        const uint32_t end = (c + 1) * P.chunk, beg = end - P.chunk;
        const uint32_t key = P.keys[end - 1];
        // a segment of a row crosses this end, and starts in this chunk
        if (key < P.rows && P.keys[end] == key && (beg == 0 || P.keys[beg] != key || P.keys[beg - 1] != key)) {
            // first parts of chunks c + 1 .. c + count: the chunks that the
            // segment fills, and the one it ends in
            uint32_t count = 1;
            const uint64_t far = uint64_t(end) + uint64_t(lane + 1) * P.chunk;  // end of chunk c + 1 + lane
            const bool on = far < P.n && P.keys[far] == key;
            const uint32_t filled = __ballot_sync(0xffffffffu, !on);
            if (filled) {
                count += __ffs(filled) - 1;
            } else {
                // chunks c + 1 .. c + lo are filled; the first that is not by
                // 32 places at a time
                uint32_t lo = 32, hi = P.chunks - 1 - c;  // c + hi: at most the last chunk
                while (hi - lo > 1) {
                    const uint32_t step = (hi - lo + 31) / 32;
                    const uint64_t k = uint64_t(lo) + uint64_t(lane + 1) * step;
                    const uint64_t at = uint64_t(end) + k * P.chunk;
                    const bool past = k >= hi || at >= P.n || P.keys[at] != key;
                    const uint32_t f = __ffs(__ballot_sync(0xffffffffu, past));  // 1 + the first lane past
                    hi = f ? min(uint64_t(hi), uint64_t(lo) + uint64_t(f) * step) : hi;
                    lo = f ? lo + (f - 1) * step : lo + 32 * step;
                }
                count = lo + 1;
            }
            if (count <= kJoinLong) {
                for (uint32_t col = lane; col < P.columns; col += 32) {
                    float s = P.parts[size_t(2 * c + 1) * P.columns + col];
#pragma unroll 4
                    for (uint32_t k = 1; k <= count; ++k) s += P.parts[size_t(2) * (c + k) * P.columns + col];
                    reinterpret_cast<T *>(P.out)[size_t(key) * P.columns + col] = from_f<T>(P.scale * s);
                }
            } else if (lane == 0) {
                long_key[warp] = key;
                long_count[warp] = count;
            }
        }
    }
    __syncthreads();
    const uint32_t slice = threadIdx.x / kCols, tc = threadIdx.x % kCols;
    for (uint32_t w = 0; w < uint32_t(kJoinWarps); ++w) {
        const uint32_t count = long_count[w], key = long_key[w], from = blockIdx.x * kJoinWarps + w;
        if (count == 0) continue;  // the same for every thread
        const uint32_t per = (count + kJoinSlices - 1) / kJoinSlices;
        const uint32_t k0 = 1 + slice * per, k1 = min(count + 1, k0 + per);
        for (uint32_t col0 = 0; col0 < P.columns; col0 += kCols) {
            const uint32_t col = col0 + tc;
            float s = 0.0f;
            if (col < P.columns) {
#pragma unroll 8
                for (uint32_t k = k0; k < k1; ++k) s += P.parts[size_t(2) * (from + k) * P.columns + col];
            }
            partial[slice][tc] = s;
            __syncthreads();
            if (slice == 0 && col < P.columns) {
                float t = P.parts[size_t(2 * from + 1) * P.columns + col];
                for (uint32_t q = 0; q < kJoinSlices; ++q) t += partial[q][tc];
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
// less; 148 SMs x 128), and no more parts than needed.
uint32_t chunk_of(uint32_t n) {
    uint32_t c = 4;
    while (c < 64 && uint64_t(c) * 148 * 128 < n) c *= 2;
    return c;
}

struct RowGradLayout {
    size_t keys[2], vals[2], counts, totals, touched, parts, total;
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
    l.counts = take(size_t(kMaxBins) * sort_tiles(n) * 4 * (sort_tiles(n) <= kFewTiles ? kMaxPasses : 1));
    l.totals = take(kMaxBins * 4);
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
    const uint32_t step_row = kLookupThreads / units, step_col = kLookupThreads % units;
    // few units: more blocks of fewer items.  1M rows of 49 floats at skewed
    // ids with 4, 8, 16 items: 102, 106, 111 us, and 97 us with 8 and streaming
    // stores (the output does not push the table's hot rows out of L2); a
    // warp per 8 rows, lanes along the row, takes 165.
    if (total < 148ull * 2048 * 4) {
        lookup_kernel<T, I, VB, 2><<<unsigned((total + 511) / 512), kLookupThreads, 0, stream>>>(
            static_cast<const char *>(table), rows, row_bytes, static_cast<const I *>(ids), total, units, step_row, step_col, scale,
            static_cast<char *>(out));
    } else {
        lookup_kernel<T, I, VB, 8><<<unsigned((total + 2047) / 2048), kLookupThreads, 0, stream>>>(
            static_cast<const char *>(table), rows, row_bytes, static_cast<const I *>(ids), total, units, step_row, step_col, scale,
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
    const dim3 grid((P.chunks + groups - 1) / groups, (P.units + P.lane_units - 1) / P.lane_units);
    if (R == 4) sum_rows_kernel<T, VB, (VB < 16 ? 4 : 2)><<<grid, kSumThreads, 0, stream>>>(P);
    else if (R == 2) sum_rows_kernel<T, VB, 2><<<grid, kSumThreads, 0, stream>>>(P);
    else sum_rows_kernel<T, VB, 1><<<grid, kSumThreads, 0, stream>>>(P);
    P.join_blocks = (P.chunks + kJoinWarps - 1) / kJoinWarps;
    const uint64_t zero_units = uint64_t(P.rows) * P.units;
    const uint32_t zero_blocks = uint32_t(std::min<uint64_t>((zero_units + 4095) / 4096, 148 * 16));
    join_parts_kernel<T, VB><<<P.join_blocks + zero_blocks, kJoinThreads, 0, stream>>>(P);
    return cudaGetLastError();
}

template <typename I, int ITEMS>
cudaError_t sort_in_block(const SortPass &P, int bits, cudaStream_t stream) {
    constexpr size_t kSmem = block_sort_smem(ITEMS);
    cudaError_t e = cudaFuncSetAttribute(sort_block_kernel<I, ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmem));
    if (e != cudaSuccess) return e;
    const unsigned clear = unsigned(std::min<uint64_t>((uint64_t(P.rows) + 16383) / 16384, 147));
    sort_block_kernel<I, ITEMS><<<1 + clear, kBlockSortThreads, kSmem, stream>>>(P, bits);
    return cudaGetLastError();
}

template <typename I>
cudaError_t sort_ids(SortPass &P, uint32_t *const keys[2], uint32_t *const vals[2], int &cur, cudaStream_t stream) {
    int bits = 0;  // of the largest key, `rows`
    while (bits < 32 && (uint64_t(P.rows) >> bits) != 0) ++bits;
    if (P.n <= kBlockSort) {
        cur = 0;
        P.keys_out = keys[0];
        P.vals_out = vals[0];
        return P.n <= 2 * kBlockSortThreads ? sort_in_block<I, 2>(P, bits, stream)
                                            : sort_in_block<I, kBlockSort / kBlockSortThreads>(P, bits, stream);
    }
    const int passes = (bits + 8) / 9, width = (bits + passes - 1) / passes;
    P.tiles = sort_tiles(P.n);
    P.bins = 1 << width;
    const bool few = P.tiles <= kFewTiles;
    const uint32_t words = P.tiles * P.bins;
    uint32_t *const counts = P.counts;
    cur = 0;
    for (int p = 0; p < passes; ++p) {
        P.shift = p * width;
        P.keys_in = keys[cur ^ 1];
        P.vals_in = vals[cur ^ 1];
        P.keys_out = keys[cur];
        P.vals_out = vals[cur];
        if (few) {
            P.clear_counts = (passes - 1) * words;
            if (p == 0) digit_counts_kernel<I, true, true><<<P.tiles, kSortThreads, 0, stream>>>(P);
            P.counts = counts + p * words;
            P.next_counts = p + 1 < passes ? P.counts + words : nullptr;
            if (p == 0) scatter_digits_kernel<I, true, true><<<P.tiles, kSortThreads, 0, stream>>>(P);
            else scatter_digits_kernel<I, false, true><<<P.tiles, kSortThreads, 0, stream>>>(P);
        } else {
            if (p == 0) digit_counts_kernel<I, true, false><<<P.tiles, kSortThreads, 0, stream>>>(P);
            else digit_counts_kernel<I, false, false><<<P.tiles, kSortThreads, 0, stream>>>(P);
            scan_counts_kernel<<<(P.bins + 7) / 8, 256, 0, stream>>>(P);
            if (p == 0) scatter_digits_kernel<I, true, false><<<P.tiles, kSortThreads, 0, stream>>>(P);
            else scatter_digits_kernel<I, false, false><<<P.tiles, kSortThreads, 0, stream>>>(P);
        }
        if (p + 1 < passes) cur ^= 1;
    }
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
    rows = nameable_rows(rows, itype);
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
    SortPass S{};
    S.ids = ids;
    S.counts = reinterpret_cast<uint32_t *>(ws + l.counts);
    S.totals = reinterpret_cast<uint32_t *>(ws + l.totals);
    S.n = n;
    S.rows = rows;
    S.named = nameable_rows(rows, itype);
    S.touched = touched;
    int cur = 0;
    const cudaError_t e = itype == SDFOAM_I64 ? sort_ids<long long>(S, keys, vals, cur, stream)
                                              : sort_ids<uint32_t>(S, keys, vals, cur, stream);
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

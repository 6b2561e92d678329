#pragma once
// Rows in the order of the group that they belong to: a stable counting sort by one or more digits of the group's number.
//
// The sort reads an index per row and writes a place per row: what bounds it is the latency of its launches and of their steps, not
// its bytes (2^20 rows: 8 MB). So a digit has as many values as the LDS has counters for, which makes one pass of up to 4399
// groups, and a batch that fits the registers of a workgroup is sorted by one workgroup in one launch.
//
// Measured: 64 rows, 8 groups 4.5 us; 2^20 rows, 4096 groups 28 us: count 6.0, scan 5.2, scatter 17 (2^20 places of 4 bytes, of which a
// tile of 4096 rows has one in a line: the writes); 65536 rows, 65536 groups: two passes of 4.5 + 6.8, without a scan.
//
// The place of a row among those of its digit is found by ballots: of the lanes of a wavefront with the same digit, those
// with lower numbers come first; wavefronts and tiles follow in the order of their rows. No atomic decides an order.

#include <qmlp/kernels/token_types.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

constexpr int GROUP_SMALL_THREADS = 1024, GROUP_SMALL_ITEMS = 8, GROUP_SMALL_BITS = 8;
constexpr int GROUP_SMALL_ROWS = GROUP_SMALL_THREADS * GROUP_SMALL_ITEMS;
constexpr int GROUP_THREADS = 1024;   // tiles of as many rows, or ITEMS times as many
constexpr int GROUP_MOST_DIGITS = 4400;   // 36 bytes of LDS each
constexpr int GROUP_SCAN_DIGITS = 64, GROUP_SCAN_SLICES = 16;
constexpr int GROUP_FEW_TILES = 64;   // that many, the workgroups of the last kernel add up the tiles before theirs themselves

/** The group of a row; 'groups' for rows whose index names none. */
template <typename I>
__device__ __forceinline__ unsigned groupOf(const I* __restrict__ index, long long stride, long long row, unsigned groups)
{
    const I g = index[row * stride];
    return g >= 0 && g < static_cast<I>(groups) ? static_cast<unsigned>(g) : groups;
}

/** The lanes of the wavefront, among those of 'active', whose 'bits' lowest bits of d are this lane's. */
__device__ __forceinline__ unsigned long long lanesLike(unsigned d, int bits, unsigned long long active)
{
    unsigned long long same = active;
    for (int b = 0; b < bits; ++b) {
        const bool set = (d >> b) & 1;
        const unsigned long long votes = __ballot(set);
        same &= set ? votes : ~votes;
    }
    return same;
}

__device__ __forceinline__ int lanesBelow(unsigned long long lanes)
{
    return __popcll(lanes & ((1ull << (threadIdx.x % 64)) - 1));
}

/**
 * Exclusive scan of n values in LDS by the whole workgroup of THREADS; 'sums' holds a value per wavefront.
 * Every thread takes n / THREADS consecutive values.
 */
template <int THREADS>
__device__ __forceinline__ void scanInLds(unsigned* values, int n, unsigned* sums)
{
    constexpr int WAVES = THREADS / 64;
    const int each = (n + THREADS - 1) / THREADS;
    const int from = min(static_cast<int>(threadIdx.x) * each, n), to = min(from + each, n);
    unsigned own = 0;
    for (int i = from; i < to; ++i) own += values[i];
    unsigned before = own;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const unsigned other = __shfl_up(before, m);
        if (static_cast<int>(threadIdx.x) % 64 >= m) before += other;
    }
    if (threadIdx.x % 64 == 63) sums[threadIdx.x / 64] = before;
    before -= own;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < WAVES; ++k)
        if (k < static_cast<int>(threadIdx.x) / 64) before += sums[k];
    for (int i = from; i < to; ++i) {
        const unsigned v = values[i];
        values[i] = before;
        before += v;
    }
    __syncthreads();
}

/** The first of n sorted keys that is not below g. */
__device__ __forceinline__ unsigned lowerBound(const unsigned* keys, unsigned n, unsigned g)
{
    unsigned from = 0;
    while (n > 0) {
        const unsigned half = n / 2;
        if (keys[from + half] < g) {
            from += half + 1;
            n -= half + 1;
        } else
            n = half;
    }
    return from;
}

/**
 * Where the entries of a group among the sorted keys begin and end: spans[group] and spans[groups + group], from the entry at i. Groups
 * without entries have no spans: whatever lies there, a reader finds that no key at the beginning it names is the group's.
 */
__device__ __forceinline__ void markSpans(const unsigned* keys, long long i, long long rows, unsigned groups, unsigned* __restrict__ spans)
{
    const unsigned key = keys[i];
    if (key >= groups) return;
    if (i == 0 || keys[i - 1] != key) spans[key] = static_cast<unsigned>(i);
    if (i == rows - 1 || keys[i + 1] != key) spans[groups + key] = static_cast<unsigned>(i + 1);
}

/**
 * What is kept of a row's place in the order: the place itself; -1 - place of rows that belong to no group. Its store goes to a line of its own where rows
 * next to each other in the order lie apart: us of all kernels without | with places 4.8 | 4.9 for 48 rows, 13.1 | 15.2 for 8192 of 64 groups, 16.2 | 16.5
 * for 2^19 of 128, 28 | 29 for 2^20 of 4096, 58 | 72 for 2^20 of 70000, whose second pass takes rows in the order of the first.
 */
__device__ __forceinline__ int placeOf(unsigned key, unsigned groups, unsigned place)
{
    return static_cast<int>(key < groups ? place : ~place);
}

/**
 * All of up to GROUP_SMALL_ROWS rows by one workgroup. bits: of the number 'groups'. keys (the groups in order), offsets (groups + 1
 * of them), spans (see markSpans()) and places (see placeOf()) may be null. LDS: GROUP_SMALL_ROWS keys and rows, the counters of the wavefronts.
 */
template <typename I>
__global__ void __launch_bounds__(GROUP_SMALL_THREADS)
GroupSmallKernel(const I* __restrict__ index, long long stride, int rows, unsigned groups, int bits, int* __restrict__ order,
                 unsigned* __restrict__ keys, int* __restrict__ offsets, unsigned* __restrict__ spans, int* __restrict__ places)
{
    constexpr int WAVES = GROUP_SMALL_THREADS / 64;
    extern __shared__ unsigned groupLds[];
    unsigned* const keysLds = groupLds;
    unsigned* const counters = groupLds + rows;   // [digit][wavefront]
    unsigned* const sums = counters + (WAVES << (bits < GROUP_SMALL_BITS ? bits : GROUP_SMALL_BITS));
    unsigned short* const rowsLds = reinterpret_cast<unsigned short*>(sums + WAVES);
    const int wave = threadIdx.x / 64;
    // a wavefront takes consecutive rows, 64 at a time
    const int items = (rows + GROUP_SMALL_THREADS - 1) / GROUP_SMALL_THREADS;
    unsigned key[GROUP_SMALL_ITEMS];
    int row[GROUP_SMALL_ITEMS];
#pragma unroll
    for (int i = 0; i < GROUP_SMALL_ITEMS; ++i) {
        row[i] = (wave * items + i) * 64 + threadIdx.x % 64;
        if (i < items && row[i] < rows) key[i] = groupOf(index, stride, row[i], groups);
    }
    for (int shift = 0; shift < bits; shift += GROUP_SMALL_BITS) {
        const int digitBits = min(GROUP_SMALL_BITS, bits - shift);
        const int digits = 1 << digitBits;
        for (int i = threadIdx.x; i < digits * WAVES; i += GROUP_SMALL_THREADS) counters[i] = 0;
        __syncthreads();
        unsigned place[GROUP_SMALL_ITEMS];
#pragma unroll
        for (int i = 0; i < GROUP_SMALL_ITEMS; ++i) {
            if (i >= items) break;
            const bool has = (wave * items + i) * 64 + static_cast<int>(threadIdx.x) % 64 < rows;
            const unsigned d = has ? (key[i] >> shift) & (digits - 1) : 0;
            const unsigned long long same = lanesLike(d, digitBits, __ballot(has));
            unsigned* const counter = counters + d * WAVES + wave;
            const unsigned before = has ? *counter : 0;
            place[i] = before + lanesBelow(same);
            waveLdsSync();
            if (has && lanesBelow(same) == 0) *counter = before + __popcll(same);
            waveLdsSync();
        }
        __syncthreads();
        scanInLds<GROUP_SMALL_THREADS>(counters, digits * WAVES, sums);
#pragma unroll
        for (int i = 0; i < GROUP_SMALL_ITEMS; ++i) {
            if (i >= items) break;
            if ((wave * items + i) * 64 + static_cast<int>(threadIdx.x) % 64 >= rows) continue;
            const unsigned d = (key[i] >> shift) & (digits - 1);
            const unsigned p = counters[d * WAVES + wave] + place[i];
            keysLds[p] = key[i];
            rowsLds[p] = static_cast<unsigned short>(row[i]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < GROUP_SMALL_ITEMS; ++i) {
            const int p = (wave * items + i) * 64 + threadIdx.x % 64;
            if (i < items && p < rows) {
                key[i] = keysLds[p];
                row[i] = rowsLds[p];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < GROUP_SMALL_ITEMS; ++i) {
        const int p = (wave * items + i) * 64 + threadIdx.x % 64;
        if (i < items && p < rows) {
            order[p] = row[i];
            if (keys) keys[p] = key[i];
            if (places) places[row[i]] = placeOf(key[i], groups, p);
            if (spans) markSpans(keysLds, p, rows, groups, spans);
        }
    }
    if (offsets)   // (keysLds: as the last pass left them)
        for (unsigned g = threadIdx.x; g <= groups; g += GROUP_SMALL_THREADS) offsets[g] = static_cast<int>(lowerBound(keysLds, rows, g));
}

/** What a pass of the sort of many rows reads: the index itself (first pass) or the keys and rows of the pass before. */
template <typename I>
struct GroupSource
{
    const I* index;
    long long stride;
    const unsigned* keys;
    const int* order;
    unsigned groups;
    __device__ __forceinline__ unsigned key(long long i) const { return keys ? keys[i] : groupOf(index, stride, i, groups); }
    __device__ __forceinline__ int row(long long i) const { return order ? order[i] : static_cast<int>(i); }
};

/** Rows per digit of every tile: counts[tile][digit]; digits: as many as there are, their bits in 'mask'. LDS: a counter per digit. */
template <typename I, int ITEMS>
__global__ void __launch_bounds__(GROUP_THREADS)
GroupCountKernel(GroupSource<I> source, long long rows, int shift, unsigned mask, int digits, unsigned* __restrict__ counts)
{
    extern __shared__ unsigned groupLds[];
    for (int d = threadIdx.x; d < digits; d += GROUP_THREADS) groupLds[d] = 0;
    __syncthreads();
    const long long first = static_cast<long long>(blockIdx.x) * (GROUP_THREADS * ITEMS);
    unsigned key[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const long long r = first + i * GROUP_THREADS + threadIdx.x;
        if (r < rows) key[i] = source.key(r);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (first + i * GROUP_THREADS + threadIdx.x < rows) atomicAdd(groupLds + ((key[i] >> shift) & mask), 1u);
    __syncthreads();
    unsigned* out = counts + static_cast<long long>(blockIdx.x) * digits;
    for (int d = threadIdx.x; d < digits; d += GROUP_THREADS) out[d] = groupLds[d];
}

/** counts[tile][digit] becomes the rows of the digit in the tiles before; totals[digit]: in all tiles. */
__global__ void __launch_bounds__(GROUP_SCAN_DIGITS* GROUP_SCAN_SLICES)
GroupScanKernel(unsigned* __restrict__ counts, int tiles, int digits, unsigned* __restrict__ totals)
{
    __shared__ unsigned sums[GROUP_SCAN_SLICES][GROUP_SCAN_DIGITS];
    const int column = threadIdx.x % GROUP_SCAN_DIGITS, slice = threadIdx.x / GROUP_SCAN_DIGITS;
    const int d = blockIdx.x * GROUP_SCAN_DIGITS + column;
    const int each = (tiles + GROUP_SCAN_SLICES - 1) / GROUP_SCAN_SLICES;
    const int from = min(slice * each, tiles), to = d < digits ? min(from + each, tiles) : from;
    unsigned sum = 0;
    constexpr int KEPT = 16;   // that many per slice are read once
    unsigned kept[KEPT];
    unsigned* const own = counts + static_cast<long long>(from) * digits + d;
#pragma unroll
    for (int n = 0; n < KEPT; ++n) kept[n] = from + n < to ? own[static_cast<long long>(n) * digits] : 0;
#pragma unroll
    for (int n = 0; n < KEPT; ++n) sum += kept[n];
#pragma unroll 8
    for (int t = from + KEPT; t < to; ++t) sum += counts[static_cast<long long>(t) * digits + d];
    sums[slice][column] = sum;
    __syncthreads();
    unsigned before = 0;
    for (int s = 0; s < slice; ++s) before += sums[s][column];
    if (d < digits && slice == GROUP_SCAN_SLICES - 1) totals[d] = before + sum;
#pragma unroll
    for (int n = 0; n < KEPT; ++n) {
        if (from + n < to) own[static_cast<long long>(n) * digits] = before;
        before += kept[n];
    }
#pragma unroll 8
    for (int t = from + KEPT; t < to; ++t) {
        unsigned* const at = counts + static_cast<long long>(t) * digits + d;
        const unsigned v = *at;
        *at = before;
        before += v;
    }
}

/**
 * Writes the rows of a tile to their places. counts: as GroupScanKernel leaves them, with totals; without totals (up to
 * GROUP_FEW_TILES tiles) as GroupCountKernel does. keysOut, offsets, places (of the last pass): may be null; offsets for a sort of one pass
 * only, whose digits are the groups. LDS: a start per digit, the counters of the wavefronts.
 */
template <typename I, int ITEMS>
__global__ void __launch_bounds__(GROUP_THREADS)
GroupScatterKernel(GroupSource<I> source, long long rows, int shift, int digitBits, int digits, const unsigned* __restrict__ counts,
                   const unsigned* __restrict__ totals, int* __restrict__ orderOut, unsigned* __restrict__ keysOut, int* __restrict__ offsets,
                   int* __restrict__ places)
{
    constexpr int WAVES = GROUP_THREADS / 64;
    const unsigned mask = (1u << digitBits) - 1;
    extern __shared__ unsigned groupLds[];
    unsigned* const starts = groupLds;
    unsigned short* const counters = reinterpret_cast<unsigned short*>(groupLds + digits);   // [wavefront][digit]
    __shared__ unsigned sums[WAVES];
    const int wave = threadIdx.x / 64;
    // Workgroups go to the dies in turn; a die takes consecutive tiles, whose rows of a group come one after the other, so that the lines it
    // writes parts of are its own for the most part.
    const unsigned die = blockIdx.x % DIES;
    const int tile = static_cast<int>(die * (gridDim.x / DIES) + min(die, gridDim.x % DIES) + blockIdx.x / DIES);
    constexpr int OWN = (GROUP_MOST_DIGITS + GROUP_THREADS - 1) / GROUP_THREADS;
    unsigned before[OWN];   // rows of the thread's digits in the tiles before
#pragma unroll
    for (int n = 0; n < OWN; ++n) {
        const int d = n * GROUP_THREADS + threadIdx.x;
        if (d >= digits) break;
        if (totals) {
            starts[d] = totals[d];
            before[n] = counts[static_cast<long long>(tile) * digits + d];
        } else {
            unsigned all = 0, those = 0;
            const int tiles = gridDim.x;
#pragma unroll 16
            for (int t = 0; t < tiles; ++t) {
                const unsigned here = counts[t * digits + d];
                all += here;
                those += t < tile ? here : 0;
            }
            starts[d] = all;
            before[n] = those;
        }
    }
    for (int i = threadIdx.x; i < (digits * WAVES + 1) / 2; i += GROUP_THREADS) reinterpret_cast<unsigned*>(counters)[i] = 0;
    // a wavefront takes consecutive rows, 64 at a time
    const long long first = static_cast<long long>(tile) * (GROUP_THREADS * ITEMS) + wave * (64 * ITEMS) + threadIdx.x % 64;
    unsigned key[ITEMS];
    int row[ITEMS];
    unsigned short place[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
        if (first + i * 64 < rows) {
            key[i] = source.key(first + i * 64);
            row[i] = source.row(first + i * 64);
        }
    __syncthreads();
    scanInLds<GROUP_THREADS>(starts, digits, sums);
    if (offsets && tile == 0)
        for (unsigned g = threadIdx.x; g <= source.groups; g += GROUP_THREADS) offsets[g] = static_cast<int>(starts[g]);   // (nothing is before the first tile)
#pragma unroll
    for (int n = 0; n < OWN; ++n) {
        const int d = n * GROUP_THREADS + threadIdx.x;
        if (d < digits) starts[d] += before[n];
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const bool has = first + i * 64 < rows;
        const unsigned d = has ? (key[i] >> shift) & mask : 0;
        const unsigned long long same = lanesLike(d, digitBits, __ballot(has));
        unsigned short* const counter = counters + wave * digits + d;
        const unsigned own = has ? *counter : 0;
        place[i] = static_cast<unsigned short>(own + lanesBelow(same));
        waveLdsSync();
        if (has && lanesBelow(same) == 0) *counter = static_cast<unsigned short>(own + __popcll(same));
        waveLdsSync();
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (first + i * 64 >= rows) continue;
        const unsigned d = (key[i] >> shift) & mask;
        unsigned p = starts[d] + place[i];
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w)
            if (w < wave) p += counters[w * digits + d];
        orderOut[p] = row[i];
        if (keysOut) keysOut[p] = key[i];
        if (places) places[row[i]] = placeOf(key[i], source.groups, p);
    }
}

/** Where every group begins among sorted keys. */
__global__ void __launch_bounds__(256) GroupOffsetsKernel(const unsigned* __restrict__ keys, long long rows, unsigned groups, int* __restrict__ offsets)
{
    const long long g = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (g <= groups) offsets[g] = static_cast<int>(lowerBound(keys, static_cast<unsigned>(rows), static_cast<unsigned>(g)));
}

QUICKMLP_KERNEL_NAMESPACE_END

#pragma once
// Rows of a table by token, times a scale, and the gradient of the table.
//
//   y[i] = scale table[index[i]],  zero where index[i] names no row;   dtable[v] = scale sum over i with index[i] = v of dy[i]
//
// Both are bound by memory. The gradient is written row by row, each element once and also where no token names the row: the
// tokens are sorted first (row_groups.h), so that a row's terms are consecutive, and no float is added by an atomic. The terms
// of frequent tokens are shared out: blocks of consecutive places of the sorted order that hold one token only are summed in
// advance, blocks of such blocks likewise, so that no row has more than a few blocks of each size left to add.
//
// Measured, 65536 tokens, most of them rare, of a vocabulary of 65536 x 1024 bfloat16: lookup 39 us, of which 134 MB are writes; gradient
// 17 + 4 us for the blocks (22 us of sorting before) and 60 us for the table, 134 MB again and the rare tokens' rows. 20011 codes of
// 1000 x 64 floats: 3.4 us, and 8 + 4 + 15 us.

#include <qmlp/kernels/row_groups.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

constexpr int EMBEDDING_THREADS = 256;
constexpr int EMBEDDING_BLOCK_BITS = 6;   // 64 places per block, 64 blocks per block of the next size

/** G lanes per row, AT_ONCE consecutive rows at a time: their indices and then their pieces are in flight together. */
template <typename T, typename I, int VEC, int G, int AT_ONCE>
__global__ void __launch_bounds__(EMBEDDING_THREADS)
EmbeddingKernel(const I* __restrict__ index, long long strideIndex, const T* __restrict__ table, long long strideTable, float scale,
                T* __restrict__ y, long long strideY, long long rows, long long vocabulary, int C)
{
    constexpr int ROWS = EMBEDDING_THREADS / G * AT_ONCE;
    const int lane = threadIdx.x % G;
    for (long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G * AT_ONCE; row < rows; row += static_cast<long long>(gridDim.x) * ROWS) {
        long long v[AT_ONCE];
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) v[n] = index[min(row + n, rows - 1) * strideIndex];
        for (int c = lane * VEC; c < C; c += G * VEC) {
            const int at = VEC == 1 ? c : min(c, C - VEC);   // the last piece ends with the row
            Raw<T, VEC> raw[AT_ONCE];
#pragma unroll
            for (int n = 0; n < AT_ONCE; ++n)
                if (v[n] >= 0 && v[n] < vocabulary) raw[n].load(table + v[n] * strideTable + at);
#pragma unroll
            for (int n = 0; n < AT_ONCE; ++n) {
                const bool valid = v[n] >= 0 && v[n] < vocabulary;
                float values[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) values[k] = valid ? static_cast<float>(raw[n].v[k]) * scale : 0;
                if (row + n < rows) streamFloats(y + (row + n) * strideY + at, values);
            }
        }
    }
}

/** Adds COUNT terms of T; at(n) is where the n-th one is. All of them are asked for before the first is added. */
template <typename T, int VEC, int COUNT, typename At>
__device__ __forceinline__ void addTerms(float (&sum)[VEC], At at)
{
    Raw<T, VEC> terms[COUNT];
#pragma unroll
    for (int n = 0; n < COUNT; ++n) terms[n].load(at(n));
#pragma unroll
    for (int n = 0; n < COUNT; ++n)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += static_cast<float>(terms[n].v[k]);
}
/** Adds 'count' consecutive terms, as many of them in flight as go into REGISTERS. */
template <typename T, int VEC, int REGISTERS, typename At>
__device__ __forceinline__ void addRange(float (&sum)[VEC], int count, At at)
{
    constexpr int MOST = REGISTERS * 4 / (VEC * static_cast<int>(sizeof(T))), BATCH = MOST < 16 ? MOST : 16;
    static_assert(BATCH >= 4, "batches, batches of 4, and single terms");
    int n = 0;
    for (; n + BATCH <= count; n += BATCH) addTerms<T, VEC, BATCH>(sum, [&](int k) { return at(n + k); });
    if constexpr (BATCH > 4)
        for (; n + 4 <= count; n += 4) addTerms<T, VEC, 4>(sum, [&](int k) { return at(n + k); });
    for (; n < count; ++n) addTerms<T, VEC, 1>(sum, [&](int k) { return at(n + k); });
}

/**
 * Adds the rows of dy at 'count' consecutive places of the order, which are looked up 64 at a time. WAVE: all lanes of the wavefront call it with
 * the same place and count; a place is a lane's register then, which the others read.
 */
template <typename T, int VEC, int REGISTERS, bool WAVE>
__device__ __forceinline__ void addPlaces(float (&sum)[VEC], const int* __restrict__ order, int count, const T* __restrict__ adjY, long long stride)
{
    if constexpr (WAVE)
        for (int n = 0; n < count; n += 64) {
            const int own = order[n + min(static_cast<int>(threadIdx.x % 64), count - n - 1)];
            addRange<T, VEC, REGISTERS>(sum, min(64, count - n), [&](int k) { return adjY + __builtin_amdgcn_readlane(own, k) * stride; });
        }
    else
        addRange<T, VEC, REGISTERS>(sum, count, [&](int n) { return adjY + order[n] * stride; });
}

/**
 * The sums of the blocks of one size that hold one token only: sums[block][C], G lanes per block. FIRST: blocks of places, whose
 * terms are rows of dy through the order, and the spans of all tokens (null: they are known); otherwise blocks of blocks, whose terms
 * are the sums of those. 1 << bits places per block.
 */
template <typename T, int VEC, int G, bool FIRST>
__global__ void __launch_bounds__(EMBEDDING_THREADS)
EmbeddingBlocksKernel(const unsigned* __restrict__ keys, const int* __restrict__ order, long long rows, unsigned vocabulary, int bits,
                      const T* __restrict__ adjY, long long strideAdjY, const float* __restrict__ smaller, float* __restrict__ sums, int C,
                      unsigned* __restrict__ spans)
{
    const long long block = static_cast<long long>(blockIdx.x) * (EMBEDDING_THREADS / G) + threadIdx.x / G;
    const long long from = block << bits, to = (block + 1) << bits;
    if (FIRST && spans)
        for (long long i = from + threadIdx.x % G; i < min(to, rows); i += G) markSpans(keys, i, rows, vocabulary, spans);
    if (to > rows || keys[from] != keys[to - 1] || keys[from] >= vocabulary) return;
    // (all lanes go through the loop, those behind the last column with its address)
    for (int column = 0; column < C; column += G * VEC) {
        const int c = column + threadIdx.x % G * VEC, at = min(c, C - VEC);
        float sum[VEC] = {};
        if constexpr (FIRST) addPlaces<T, VEC, 64, (G >= 64)>(sum, order + from, 1 << EMBEDDING_BLOCK_BITS, adjY + at, strideAdjY);
        else addRange<float, VEC, 64>(sum, 1 << EMBEDDING_BLOCK_BITS, [&](int i) { return smaller + ((block << EMBEDDING_BLOCK_BITS) + i) * C + at; });
        if (c < C) storeFloats(sums + block * C + at, sum);
    }
}

/** The sums of blocks of every size: sums[s] of blocks of 1 << (EMBEDDING_BLOCK_BITS (s + 1)) places. */
struct EmbeddingBlocks
{
    static constexpr int SIZES = 6;
    int sizes;
    const float* sums[SIZES];
};

constexpr int EMBEDDING_MOST_ROWS = EMBEDDING_THREADS;   // a thread looks up each
/**
 * The gradient of up to 'each' (EMBEDDING_MOST_ROWS at most) rows of the table per workgroup, G lanes per row. Their spans are
 * looked up together first, with the only term of those that have one. The rows of a workgroup are those of its number and as many as
 * there are workgroups apart: frequent tokens often have neighbouring numbers (65536 tokens of a vocabulary of 65536 x 1024 bfloat16 in the
 * order of their frequency: 54 us, 236 with consecutive rows), and workgroups that write consecutive rows write all channels of the
 * memory at a time (tokens that name no row: 25 us, 42 with consecutive rows per workgroup).
 */
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(EMBEDDING_THREADS)
EmbeddingAdjointKernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ spans, const int* __restrict__ order, long long rows,
                       EmbeddingBlocks blocks, const T* __restrict__ adjY, long long strideAdjY, float scale, T* __restrict__ adjTable,
                       long long strideTable, long long vocabulary, int C)
{
    __shared__ unsigned begin[EMBEDDING_MOST_ROWS], end[EMBEDDING_MOST_ROWS];
    __shared__ int only[EMBEDDING_MOST_ROWS];
    const int count = static_cast<int>((vocabulary - blockIdx.x + gridDim.x - 1) / gridDim.x);
    if (static_cast<int>(threadIdx.x) < count) {
        const long long v = blockIdx.x + static_cast<long long>(threadIdx.x) * gridDim.x;
        const unsigned from = spans[v], to = spans[vocabulary + v];
        const bool any = from < rows && keys[from] == v;   // otherwise no token names the row, and nothing was written there
        begin[threadIdx.x] = any ? from : 0;
        end[threadIdx.x] = any ? to : 0;
        only[threadIdx.x] = any ? order[from] : 0;
    }
    __syncthreads();
    const int lane = threadIdx.x % G;
    for (int r = threadIdx.x / G; r < count; r += EMBEDDING_THREADS / G) {
        unsigned span[2] = {begin[r], end[r]};
        int single = only[r];
        if constexpr (G >= 64) {   // one row for the whole wavefront
            span[0] = __builtin_amdgcn_readfirstlane(span[0]);
            span[1] = __builtin_amdgcn_readfirstlane(span[1]);
            single = __builtin_amdgcn_readfirstlane(single);
        }
        const long long from = span[0], to = span[1];
        for (int column = 0; column < C; column += G * VEC) {   // (all lanes, as above)
            const int c = column + lane * VEC, at = min(c, C - VEC);
            float sum[VEC] = {};
            if (to - from == 1) addTerms<T, VEC, 1>(sum, [&](int) { return adjY + single * strideAdjY + at; });
            else if (to > from) {
                // places up to the first block, blocks up to the first larger block, ..., and down again
                long long i = from;
                auto add = [&](int size, long long last) {
                    const int bits = EMBEDDING_BLOCK_BITS * size;
                    const long long first = i >> bits;
                    const int terms = static_cast<int>((last - i) >> bits);
                    if (size == 0) addPlaces<T, VEC, 32, (G >= 64)>(sum, order + first, terms, adjY + at, strideAdjY);
                    else {
                        const float* p = blocks.sums[size - 1] + first * C + at;
                        addRange<float, VEC, 32>(sum, terms, [&](int n) { return p + static_cast<long long>(n) * C; });
                    }
                    i = last;
                };
                int size = 0;
                for (; size < blocks.sizes; ++size) {
                    const long long places = 1ll << (EMBEDDING_BLOCK_BITS * (size + 1)), next = (i + places - 1) & -places;
                    if (next + places > to) break;   // no larger block in here
                    add(size, next);
                }
                for (; size >= 0; --size) add(size, to >> (EMBEDDING_BLOCK_BITS * size) << (EMBEDDING_BLOCK_BITS * size));
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] *= scale;
            if (c < C) streamFloats(adjTable + (blockIdx.x + static_cast<long long>(r) * gridDim.x) * strideTable + at, sum);
        }
    }
}

QUICKMLP_KERNEL_NAMESPACE_END

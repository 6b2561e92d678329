#pragma once
// Rows of a table by token, times a scale, and the gradient of the table.
//
//   y[i] = scale table[index[i]],  zero where index[i] names no row;   dtable[v] = scale sum over i with index[i] = v of dy[i]
//
// Both are bound by memory. The gradient is written row by row, each element once and also where no token names the row: the
// tokens are sorted first (row_groups.h), so that a row's terms are consecutive, and no float is added by an atomic. The terms
// of frequent tokens are shared out: blocks of consecutive places of the sorted order that hold one token only are summed in
// advance, blocks of such blocks likewise, so that no row has more than a few blocks of each size left to add.

#include <qmlp/kernels/row_groups.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

constexpr int EMBEDDING_THREADS = 256;
constexpr int EMBEDDING_BLOCK_BITS = 5;   // 32 places per block, 32 blocks per block of the next size

/** G lanes per row, PIECES of VEC entries each at a time. */
template <typename T, typename I, int VEC, int G>
__global__ void __launch_bounds__(EMBEDDING_THREADS)
EmbeddingKernel(const I* __restrict__ index, long long strideIndex, const T* __restrict__ table, long long strideTable, float scale,
                T* __restrict__ y, long long strideY, long long rows, long long vocabulary, int C)
{
    constexpr int ROWS = EMBEDDING_THREADS / G;
    const int lane = threadIdx.x % G;
    for (long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G; row < rows; row += static_cast<long long>(gridDim.x) * ROWS) {
        const long long v = index[row * strideIndex];
        const bool valid = v >= 0 && v < vocabulary;
        const T* from = table + (valid ? v : 0) * strideTable;
        T* to = y + row * strideY;
#pragma unroll 4
        for (int c = lane * VEC; c < C; c += G * VEC) {
            const int at = VEC == 1 ? c : min(c, C - VEC);   // the last piece ends with the row
            float values[VEC] = {};
            if (valid) loadFloats(from + at, values);
#pragma unroll
            for (int k = 0; k < VEC; ++k) values[k] = valid ? values[k] * scale : 0;
            storeFloats(to + at, values);
        }
    }
}

/** Entries of the sorted order that begin (end) a token's terms: spans[token] and spans[vocabulary + token]. */
__global__ void __launch_bounds__(EMBEDDING_THREADS)
EmbeddingSpansKernel(const unsigned* __restrict__ keys, long long rows, unsigned vocabulary, unsigned* __restrict__ spans)
{
    const long long i = static_cast<long long>(blockIdx.x) * EMBEDDING_THREADS + threadIdx.x;
    if (i >= rows) return;
    const unsigned key = keys[i];
    if (key >= vocabulary) return;
    if (i == 0 || keys[i - 1] != key) spans[key] = static_cast<unsigned>(i);
    if (i == rows - 1 || keys[i + 1] != key) spans[vocabulary + key] = static_cast<unsigned>(i + 1);
}

/**
 * The sums of the blocks of one size that hold one token only: sums[block][C], G lanes per block. FIRST: blocks of places, whose
 * terms are rows of dy through the order; otherwise blocks of blocks, whose terms are the sums of those. 1 << bits places per block.
 */
template <typename T, int VEC, int G, bool FIRST>
__global__ void __launch_bounds__(EMBEDDING_THREADS)
EmbeddingBlocksKernel(const unsigned* __restrict__ keys, const int* __restrict__ order, long long rows, unsigned vocabulary, int bits,
                      const T* __restrict__ adjY, long long strideAdjY, const float* __restrict__ smaller, float* __restrict__ sums, int C)
{
    const long long block = static_cast<long long>(blockIdx.x) * (EMBEDDING_THREADS / G) + threadIdx.x / G;
    const long long from = block << bits, to = (block + 1) << bits;
    if (to > rows || keys[from] != keys[to - 1] || keys[from] >= vocabulary) return;
    for (int c = threadIdx.x % G * VEC; c < C; c += G * VEC) {
        const int at = VEC == 1 ? c : min(c, C - VEC);
        float sum[VEC] = {};
#pragma unroll 8
        for (int i = 0; i < (1 << EMBEDDING_BLOCK_BITS); ++i) {
            float term[VEC];
            if constexpr (FIRST) loadFloats(adjY + order[from + i] * strideAdjY + at, term);
            else loadFloats(smaller + ((block << EMBEDDING_BLOCK_BITS) + i) * C + at, term);
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += term[k];
        }
        storeFloats(sums + block * C + at, sum);
    }
}

/** The sums of blocks of every size: sums[s] of blocks of 1 << (EMBEDDING_BLOCK_BITS (s + 1)) places. */
struct EmbeddingBlocks
{
    static constexpr int SIZES = 6;
    int sizes;
    const float* sums[SIZES];
};

/** G lanes per row of the table. */
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(EMBEDDING_THREADS)
EmbeddingAdjointKernel(const unsigned* __restrict__ spans, const int* __restrict__ order, EmbeddingBlocks blocks, const T* __restrict__ adjY,
                       long long strideAdjY, float scale, T* __restrict__ adjTable, long long strideTable, long long vocabulary, int C)
{
    constexpr int ROWS = EMBEDDING_THREADS / G;
    const int lane = threadIdx.x % G;
    for (long long v = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G; v < vocabulary; v += static_cast<long long>(gridDim.x) * ROWS) {
        const long long from = spans[v], to = spans[vocabulary + v];
        for (int c = lane * VEC; c < C; c += G * VEC) {
            const int at = VEC == 1 ? c : min(c, C - VEC);
            float sum[VEC] = {};
            auto add = [&](auto* p) {
                float term[VEC];
                loadFloats(p + at, term);
#pragma unroll
                for (int k = 0; k < VEC; ++k) sum[k] += term[k];
            };
            // the largest whole block that begins here, one after the other
            long long i = from;
            while (i < to) {
                int size = 0;
                while (size < blocks.sizes) {
                    const long long places = 1ll << (EMBEDDING_BLOCK_BITS * (size + 1));
                    if ((i & (places - 1)) != 0 || i + places > to) break;
                    ++size;
                }
                if (size == 0) {
                    add(adjY + order[i] * strideAdjY);
                    ++i;
                } else {
                    const int bits = EMBEDDING_BLOCK_BITS * size;
                    add(blocks.sums[size - 1] + (i >> bits) * C);
                    i += 1ll << bits;
                }
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] *= scale;
            storeFloats(adjTable + v * strideTable + at, sum);
        }
    }
}

QUICKMLP_KERNEL_NAMESPACE_END

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
constexpr int EMBEDDING_BLOCK_BITS = 6;   // 64 places per block, 64 blocks per block of the next size

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

/** Adds COUNT terms; term(n, values) has the n-th one. */
template <int VEC, int COUNT, typename Term>
__device__ __forceinline__ void addTerms(float (&sum)[VEC], Term term)
{
    float terms[COUNT][VEC];   // all of them asked for before the first is added
#pragma unroll
    for (int n = 0; n < COUNT; ++n) term(n, terms[n]);
#pragma unroll
    for (int n = 0; n < COUNT; ++n)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += terms[n][k];
}
/** Adds 'count' consecutive terms, eight of them in flight. */
template <int VEC, typename Term>
__device__ __forceinline__ void addRange(float (&sum)[VEC], int count, Term term)
{
    int n = 0;
    for (; n + 8 <= count; n += 8) addTerms<VEC, 8>(sum, [&](int k, float (&v)[VEC]) { term(n + k, v); });
    if (n + 4 <= count) {
        addTerms<VEC, 4>(sum, [&](int k, float (&v)[VEC]) { term(n + k, v); });
        n += 4;
    }
    for (; n < count; ++n) addTerms<VEC, 1>(sum, [&](int k, float (&v)[VEC]) { term(n + k, v); });
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
    for (int c = threadIdx.x % G * VEC; c < C; c += G * VEC) {
        const int at = VEC == 1 ? c : min(c, C - VEC);
        float sum[VEC] = {};
        addRange(sum, 1 << EMBEDDING_BLOCK_BITS, [&](int i, float (&v)[VEC]) {
            if constexpr (FIRST) loadFloats(adjY + order[from + i] * strideAdjY + at, v);
            else loadFloats(smaller + ((block << EMBEDDING_BLOCK_BITS) + i) * C + at, v);
        });
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
EmbeddingAdjointKernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ spans, const int* __restrict__ order, long long rows,
                       EmbeddingBlocks blocks, const T* __restrict__ adjY, long long strideAdjY, float scale, T* __restrict__ adjTable,
                       long long strideTable, long long vocabulary, int C)
{
    constexpr int ROWS = EMBEDDING_THREADS / G;
    const int lane = threadIdx.x % G;
    for (long long v = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G; v < vocabulary; v += static_cast<long long>(gridDim.x) * ROWS) {
        unsigned span[2] = {spans[v], spans[vocabulary + v]};
        if constexpr (G >= 64) {   // one row for the whole wavefront
            span[0] = __builtin_amdgcn_readfirstlane(span[0]);
            span[1] = __builtin_amdgcn_readfirstlane(span[1]);
        }
        const long long from = span[0];
        const bool any = from < rows && keys[from] == v;   // otherwise no token names the row, and nothing was written there
        const long long to = any ? static_cast<long long>(span[1]) : from;
        for (int c = lane * VEC; c < C; c += G * VEC) {
            const int at = VEC == 1 ? c : min(c, C - VEC);
            float sum[VEC] = {};
            // places up to the first block, blocks up to the first larger block, ..., and down again
            long long i = from;
            auto add = [&](int size, long long end) {
                const int bits = EMBEDDING_BLOCK_BITS * size;
                const long long first = i >> bits;
                const int count = static_cast<int>((end - i) >> bits);
                if (size == 0) addRange(sum, count, [&](int n, float (&term)[VEC]) { loadFloats(adjY + order[first + n] * strideAdjY + at, term); });
                else {
                    const float* p = blocks.sums[size - 1] + first * C + at;
                    addRange(sum, count, [&](int n, float (&term)[VEC]) { loadFloats(p + static_cast<long long>(n) * C, term); });
                }
                i = end;
            };
            int size = 0;
            for (; size < blocks.sizes; ++size) {
                const long long places = 1ll << (EMBEDDING_BLOCK_BITS * (size + 1)), next = (i + places - 1) & -places;
                if (next + places > to) break;   // no larger block in here
                add(size, next);
            }
            for (; size >= 0; --size) add(size, to >> (EMBEDDING_BLOCK_BITS * size) << (EMBEDDING_BLOCK_BITS * size));
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] *= scale;
            storeFloats(adjTable + v * strideTable + at, sum);
        }
    }
}

QUICKMLP_KERNEL_NAMESPACE_END

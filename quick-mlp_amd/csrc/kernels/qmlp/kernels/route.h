#pragma once
// The router of a layer with experts: for every row of logits the experts with the largest ones and their weights.
//
//   p = softmax(l),  index = the 'chosen' largest of l, the first of equals,  w[j] = p[index[j]]
//   normalised: w = softmax over the chosen ones alone.  An expert whose logit is -inf is taken by no row: index -1 and w 0 in its place.
//   dl = p (G - sum over j of g[j] w[j]),  G the g[j] at their experts;  normalised: the same with p = 0 at experts that were not chosen
//
// A row lies in the registers of 8 to 64 lanes, so that reading it is one access each. What bounds it is the choice, one after the other: the
// largest key of the row by operations between neighbouring lanes, the lowest lane that has it, its first entry.

#include <qmlp/kernels/token_types.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

constexpr int ROUTE_THREADS = 256;

/** Numbers in the order of the logits: NaN above all, both zeros the same. 0: none. */
__device__ __forceinline__ unsigned routeKey(float v)
{
    const int bits = __builtin_bit_cast(int, v + 0.0f);
    const unsigned key = static_cast<unsigned>(bits) ^ (static_cast<unsigned>(bits >> 31) | 0x80000000u);
    return v != v ? 0xffffffffu : key;
}
constexpr unsigned ROUTE_KEY_NONE = 0x007fffffu;   // of -inf, which is not chosen
__device__ __forceinline__ float routeValue(unsigned key)
{
    return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

/** The value of another lane of the row of 16 that a lane belongs to. */
template <int CONTROL, typename V>
__device__ __forceinline__ V movedLanes(V v)
{
    return __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}
/** op over the G (8 to 64) consecutive lanes that a lane belongs to, in all of them. All lanes of the wavefront call it. */
template <int G, typename V, typename Op>
__device__ __forceinline__ V overLanes(V v, Op op)
{
    v = op(v, movedLanes<0xb1>(v));    // lanes 1 0 3 2 of every four
    v = op(v, movedLanes<0x4e>(v));    // lanes 2 3 0 1
    v = op(v, movedLanes<0x141>(v));   // the other way round in every eight
    if constexpr (G >= 16) v = op(v, movedLanes<0x140>(v));   // and in every sixteen
    if constexpr (G >= 32) v = op(v, __shfl_xor(v, 16));
    if constexpr (G >= 64) v = op(v, __shfl_xor(v, 32));
    return v;
}
template <int G>
__device__ __forceinline__ unsigned largestOfLanes(unsigned v)
{
    return overLanes<G>(v, [](unsigned a, unsigned b) { return max(a, b); });
}
template <int G>
__device__ __forceinline__ float totalOfLanes(float v)
{
    return overLanes<G>(v, [](float a, float b) { return a + b; });
}

/** The lane's entries of a row of 'experts' logits; -inf behind the last. */
template <typename T, int ENTRIES>
__device__ __forceinline__ void loadLogits(const T* __restrict__ row, int first, int experts, float (&v)[ENTRIES])
{
    if (first + ENTRIES <= experts) loadFloats(row + first, v);
    else
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) v[i] = first + i < experts ? static_cast<float>(row[first + i]) : -__builtin_inff();
}

/** G lanes per row, ENTRIES logits each. LDS: 8 bytes for every chosen expert of the workgroup's rows. */
template <typename T, int G, int ENTRIES>
__global__ void __launch_bounds__(ROUTE_THREADS)
RouteKernel(const T* __restrict__ logits, long long strideLogits, T* __restrict__ weights, long long strideWeights, int* __restrict__ index,
            long long strideIndex, long long rows, int experts, int chosen, int normalised)
{
    constexpr int ROWS = ROUTE_THREADS / G;
    extern __shared__ unsigned routeLds[];
    const int lane = threadIdx.x % G;
    unsigned* const keys = routeLds + threadIdx.x / G * (2 * chosen);
    int* const indices = reinterpret_cast<int*>(keys + chosen);
    for (long long first = static_cast<long long>(blockIdx.x) * ROWS; first < rows; first += static_cast<long long>(gridDim.x) * ROWS) {
        const long long row = min(first + threadIdx.x / G, rows - 1);   // (lanes behind the last row do its work once more)
        float v[ENTRIES];
        loadLogits(logits + row * strideLogits, lane * ENTRIES, experts, v);
        unsigned key[ENTRIES];
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) key[i] = routeKey(v[i]);
        unsigned top = 0;
        for (int j = 0; j < chosen; ++j) {
            unsigned own = key[0];
#pragma unroll
            for (int i = 1; i < ENTRIES; ++i) own = max(own, key[i]);
            const unsigned best = largestOfLanes<G>(own);
            if (j == 0) top = best;
            // (the lowest lane has the first of equals)
            const unsigned long long have = __ballot(own == best) >> (threadIdx.x % 64 / G * G);
            if (lane == __ffsll(have) - 1) {
                int at = 0;
#pragma unroll
                for (int i = ENTRIES - 1; i >= 0; --i) at = key[i] == best ? i : at;
#pragma unroll
                for (int i = 0; i < ENTRIES; ++i) key[i] = i == at ? 0 : key[i];
                keys[j] = best;
                indices[j] = best > ROUTE_KEY_NONE ? lane * ENTRIES + at : -1;
            }
        }
        waveLdsSync();
        const bool any = top > ROUTE_KEY_NONE;
        const float largest = routeValue(top);
        float total = 0;
        if (normalised) {
            for (int j = lane; j < chosen; j += G) total += indices[j] >= 0 ? expf(routeValue(keys[j]) - largest) : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < ENTRIES; ++i) total += any ? expf(v[i] - largest) : 0.0f;
        }
        total = totalOfLanes<G>(total);
        if (first + threadIdx.x / G < rows)
            for (int j = lane; j < chosen; j += G) {
                const int e = indices[j];
                index[row * strideIndex + j] = e;
                weights[row * strideWeights + j] = static_cast<T>(e >= 0 ? expf(routeValue(keys[j]) - largest) / total : 0.0f);
            }
        waveLdsSync();
    }
}

/** What stands for no gradient in LDS: a NaN that arithmetic does not make. */
constexpr unsigned ROUTE_NOT_CHOSEN = 0x7fffdeadu;

/** Gradient of the logits, written as a whole. index: as RouteKernel left it; others than 0 .. experts - 1 are no experts. */
template <typename T, int G, int ENTRIES>
__global__ void __launch_bounds__(ROUTE_THREADS)
RouteAdjointKernel(const T* __restrict__ logits, long long strideLogits, const int* __restrict__ index, long long strideIndex,
                   const T* __restrict__ adjWeights, long long strideAdjWeights, T* __restrict__ adjLogits, long long strideAdjLogits, long long rows,
                   int experts, int chosen, int normalised)
{
    constexpr int ROWS = ROUTE_THREADS / G;
    __shared__ __attribute__((aligned(16))) float routeRows[ROWS][G * ENTRIES];
    const int lane = threadIdx.x % G, from = lane * ENTRIES;
    float* const own = routeRows[threadIdx.x / G];
    for (long long first = static_cast<long long>(blockIdx.x) * ROWS; first < rows; first += static_cast<long long>(gridDim.x) * ROWS) {
        const long long row = min(first + threadIdx.x / G, rows - 1);
        float v[ENTRIES];
        loadLogits(logits + row * strideLogits, from, experts, v);
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) top = max(top, routeKey(v[i]));
        top = largestOfLanes<G>(top);
        const float largest = routeValue(top);
        float total = 0;
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) {
            v[i] = top > ROUTE_KEY_NONE ? expf(v[i] - largest) : 0.0f;
            total += v[i];
            own[from + i] = v[i];
        }
        waveLdsSync();
        float taken = 0, inner = 0;
        const int* const indices = index + row * strideIndex;
        const T* const gradients = adjWeights + row * strideAdjWeights;
        for (int j = lane; j < chosen; j += G) {
            const int e = indices[j];
            if (e < 0 || e >= experts) continue;
            taken += own[e];
            inner += own[e] * static_cast<float>(gradients[j]);
        }
        total = totalOfLanes<G>(normalised ? taken : total);
        inner = totalOfLanes<G>(inner) / total;
        waveLdsSync();
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) own[from + i] = __builtin_bit_cast(float, ROUTE_NOT_CHOSEN);
        waveLdsSync();
        for (int j = lane; j < chosen; j += G) {
            const int e = indices[j];
            const float g = static_cast<float>(gradients[j]);
            if (e >= 0 && e < experts) own[e] = g != g ? __builtin_nanf("") : g;
        }
        waveLdsSync();
        float out[ENTRIES];
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) {
            const unsigned bits = __builtin_bit_cast(unsigned, own[from + i]);
            const bool held = bits != ROUTE_NOT_CHOSEN;
            const float g = held ? __builtin_bit_cast(float, bits) : 0.0f;
            // (rows without experts have no total)
            out[i] = top > ROUTE_KEY_NONE && (held || !normalised) ? v[i] / total * (g - inner) : 0.0f;
        }
        if (first + threadIdx.x / G < rows) {
            T* const to = adjLogits + row * strideAdjLogits + from;
            if (from + ENTRIES <= experts) storeFloats(to, out);
            else
#pragma unroll
                for (int i = 0; i < ENTRIES; ++i)
                    if (from + i < experts) to[i] = static_cast<T>(out[i]);
        }
        waveLdsSync();
    }
}

// ------------------------------------------------------------------------------------------------ more experts than registers
/** The largest of the workgroup's values, in all threads. */
__device__ __forceinline__ unsigned long long largestOfGroup(unsigned long long v, unsigned long long* lds)
{
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v = max(v, static_cast<unsigned long long>(__shfl_xor(static_cast<long long>(v), m)));
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ROUTE_THREADS / 64; ++w) v = max(v, lds[w]);
    return v;
}
__device__ __forceinline__ float totalOfGroup(float v, float* lds)
{
    v = sumOfLanes<64>(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < ROUTE_THREADS / 64; ++w) v += lds[w];
    return v;
}

/** A key and, below it, the expert: of equal keys the first is the largest. */
__device__ __forceinline__ unsigned long long routePair(float v, int expert)
{
    return static_cast<unsigned long long>(routeKey(v)) << 32 | (0xffffffffu - static_cast<unsigned>(expert));
}

/** A workgroup per row, which is read once more for every chosen expert: the largest pair below the one before. */
template <typename T>
__global__ void __launch_bounds__(ROUTE_THREADS)
RouteLongKernel(const T* __restrict__ logits, long long strideLogits, T* __restrict__ weights, long long strideWeights, int* __restrict__ index,
                long long strideIndex, long long rows, int experts, int chosen, int normalised)
{
    __shared__ unsigned long long pairs[ROUTE_THREADS / 64];
    __shared__ float sums[ROUTE_THREADS / 64];
    extern __shared__ unsigned routeLds[];
    int* const indices = reinterpret_cast<int*>(routeLds + chosen);
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* const own = logits + row * strideLogits;
        unsigned long long last = ~0ull;   // (above every pair: the last expert's number is not 2^32 - 1)
        float largest = 0;
        bool any = false;
        for (int j = 0; j < chosen; ++j) {
            unsigned long long best = 0;
            for (int e = threadIdx.x; e < experts; e += ROUTE_THREADS) {
                const unsigned long long pair = routePair(static_cast<float>(own[e]), e);
                if (pair < last && pair > best) best = pair;
            }
            last = largestOfGroup(best, pairs);
            const unsigned key = static_cast<unsigned>(last >> 32);
            if (j == 0) {
                any = key > ROUTE_KEY_NONE;
                largest = routeValue(key);
            }
            if (threadIdx.x == 0) {
                routeLds[j] = key;
                indices[j] = key > ROUTE_KEY_NONE ? static_cast<int>(0xffffffffu - static_cast<unsigned>(last)) : -1;
            }
        }
        float total = 0;
        __syncthreads();
        if (normalised) {
            for (int j = threadIdx.x; j < chosen; j += ROUTE_THREADS) total += indices[j] >= 0 ? expf(routeValue(routeLds[j]) - largest) : 0.0f;
        } else if (any)
            for (int e = threadIdx.x; e < experts; e += ROUTE_THREADS) total += expf(static_cast<float>(own[e]) - largest);
        total = totalOfGroup(total, sums);
        for (int j = threadIdx.x; j < chosen; j += ROUTE_THREADS) {
            index[row * strideIndex + j] = indices[j];
            weights[row * strideWeights + j] = static_cast<T>(indices[j] >= 0 ? expf(routeValue(routeLds[j]) - largest) / total : 0.0f);
        }
        __syncthreads();
    }
}

/** A workgroup per row: gradients as of experts that were not chosen first, those of the chosen ones over them. */
template <typename T>
__global__ void __launch_bounds__(ROUTE_THREADS)
RouteLongAdjointKernel(const T* __restrict__ logits, long long strideLogits, const int* __restrict__ index, long long strideIndex,
                       const T* __restrict__ adjWeights, long long strideAdjWeights, T* __restrict__ adjLogits, long long strideAdjLogits, long long rows,
                       int experts, int chosen, int normalised)
{
    __shared__ unsigned long long pairs[ROUTE_THREADS / 64];
    __shared__ float sums[ROUTE_THREADS / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* const own = logits + row * strideLogits;
        const int* const indices = index + row * strideIndex;
        const T* const gradients = adjWeights + row * strideAdjWeights;
        T* const to = adjLogits + row * strideAdjLogits;
        unsigned long long best = 0;
        for (int e = threadIdx.x; e < experts; e += ROUTE_THREADS) best = max(best, routePair(static_cast<float>(own[e]), e));
        const unsigned top = static_cast<unsigned>(largestOfGroup(best, pairs) >> 32);
        const bool any = top > ROUTE_KEY_NONE;
        const float largest = routeValue(top);
        float total = 0, inner = 0;
        if (any && !normalised)
            for (int e = threadIdx.x; e < experts; e += ROUTE_THREADS) total += expf(static_cast<float>(own[e]) - largest);
        if (any)
            for (int j = threadIdx.x; j < chosen; j += ROUTE_THREADS) {
                const int e = indices[j];
                if (e < 0 || e >= experts) continue;
                const float p = expf(static_cast<float>(own[e]) - largest);
                if (normalised) total += p;
                inner += p * static_cast<float>(gradients[j]);
            }
        total = totalOfGroup(total, sums);
        inner = totalOfGroup(inner, sums) / total;
        for (int e = threadIdx.x; e < experts; e += ROUTE_THREADS)
            to[e] = static_cast<T>(any && !normalised ? expf(static_cast<float>(own[e]) - largest) / total * (0.0f - inner) : 0.0f);
        __syncthreads();   // (waits for these stores as well)
        if (any)
            for (int j = threadIdx.x; j < chosen; j += ROUTE_THREADS) {
                const int e = indices[j];
                if (e < 0 || e >= experts) continue;
                to[e] = static_cast<T>(expf(static_cast<float>(own[e]) - largest) / total * (static_cast<float>(gradients[j]) - inner));
            }
        __syncthreads();
    }
}

QUICKMLP_KERNEL_NAMESPACE_END

#pragma once
// The router of a layer with experts: for every row of logits the experts with the largest ones and their weights.
//
//   p = softmax(l),  index = the 'chosen' largest of l, the first of equals,  w[j] = p[index[j]]
//   normalised: w = softmax over the chosen ones alone.  An expert whose logit is -inf is taken by no row: index -1 and w 0 in its place.
//   dl = p (G - sum over j of g[j] w[j]),  G the g[j] at their experts;  normalised: the same with p = 0 at experts that were not chosen
//
// A row lies in the registers of 8 to 64 lanes, so that reading it is one access each, and every lane sorts what it has. A choice then is the largest
// of the lanes' first keys by operations between neighbouring lanes, and a step of the list it came from.
//
// What bounds the forward pass is what a row takes besides its bytes and choices: 65536 rows of 128 floats with 1, 2, 4, 8 chosen take 11.9, 12.1, 13.3,
// 15.9 us, 0.6 a choice and 11 without any, of which the bytes would be 7; of bfloat16, half the bytes, 10.3 and 13.2 with 1 and 8. Keys, sort and
// exponentials of a row follow each other, and a wavefront has no other row under way. The gradient is bound by memory: 14.9 (72 MB, 4.8 TB/s).
// Others, single precision, us forward and gradient: 65536 of 16, 2 chosen 5.6 and 5.6; 8192 of 1024, 8 chosen 18.3 and 19.0; 500 of 2000, which no
// wavefront holds and which is read again for every choice, with two barriers, 17.1 (1 chosen 6.1) and 9.1; bfloat16, 24 rows of 64 2.6. By a search for
// the largest key and its entry in every step 65536 of 128, 8 chosen, took 20.4, its gradient with a division for every logit 17.2.

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

/**
 * exp(d) for d <= 0, to 2 units of the last place: what the product with log2(e) loses comes back as the first term of its exponential. The instruction
 * keeps no result below 2^-126 (d = -87.3). SMALL: those are made 2^64 times as large and are off by half of the smallest number besides; otherwise they
 * are 0, which is nothing beside a total of at least 1, and 2^-126 of the largest gradient in gradients (with SMALL these took 3 to 6 % longer).
 */
template <bool SMALL>
__device__ __forceinline__ float routeExp(float d)
{
    constexpr float LOG2E = 1.44269502f, REST = 1.92596303e-8f, LN2 = 0.693147182f;   // log2(e) = LOG2E + REST
    d = fmaxf(d, -200.0f);
    const float t = d * LOG2E;
    const float lost = __builtin_fmaf(d, REST, __builtin_fmaf(d, LOG2E, -t));
    const bool small = SMALL && t < -126.0f;
    const float e = __builtin_amdgcn_exp2f(small ? t + 64.0f : t);
    return __builtin_fmaf(e, lost * LN2, e) * (small ? 0x1p-64f : 1.0f);
}
/** A row with a NaN or +inf has no weights. */
__device__ __forceinline__ float routeTotal(float total, unsigned top) { return top < 0xff800000u ? total : __builtin_nanf(""); }

/** Sorted with the largest first: Batcher's merge exchange, by instructions for the smaller and the larger of two. */
template <int N>
struct RouteSort
{
    template <int I, int J>
    static __device__ __forceinline__ void exchange(unsigned (&k)[N])
    {
        const unsigned larger = max(k[I], k[J]);
        k[J] = min(k[I], k[J]);
        k[I] = larger;
    }
    /** Entries I, I + 2 R, ... before END, each with the one R behind it. */
    template <int I, int R, int END>
    static __device__ __forceinline__ void exchanges(unsigned (&k)[N])
    {
        if constexpr (I + R < END) {
            exchange<I, I + R>(k);
            exchanges<I + 2 * R, R, END>(k);
        }
    }
    /** Entries FROM, FROM + R, ..., COUNT / R of them, whose halves are sorted. */
    template <int FROM, int COUNT, int R>
    static __device__ __forceinline__ void merge(unsigned (&k)[N])
    {
        if constexpr (2 * R < COUNT) {
            merge<FROM, COUNT, 2 * R>(k);
            merge<FROM + R, COUNT, 2 * R>(k);
            exchanges<FROM + R, R, FROM + COUNT>(k);
        } else
            exchange<FROM, FROM + R>(k);
    }
    template <int FROM, int COUNT>
    static __device__ __forceinline__ void sort(unsigned (&k)[N])
    {
        if constexpr (COUNT > 1) {
            sort<FROM, COUNT / 2>(k);
            sort<FROM + COUNT / 2, COUNT / 2>(k);
            merge<FROM, COUNT, 1>(k);
        }
    }
};

/** The chosen experts of a row and their keys, by keys as they are: the lowest lane with the largest one has the first of equals. All lanes call it. */
template <int G, int ENTRIES>
__device__ __forceinline__ void chooseExactly(const float (&v)[ENTRIES], int chosen, unsigned* keys, int* indices)
{
    const int lane = threadIdx.x % G;
    unsigned key[ENTRIES];
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i) key[i] = routeKey(v[i]);
    for (int j = 0; j < chosen; ++j) {
        unsigned own = key[0];
#pragma unroll
        for (int i = 1; i < ENTRIES; ++i) own = max(own, key[i]);
        const unsigned best = largestOfLanes<G>(own);
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
}

/**
 * G lanes per row, ENTRIES logits each. The expert's number takes the place of the last bits of a key, so that a key is all that a lane has to sort and
 * to pass on, and equal logits come in the order of their experts. Of 16-bit logits these bits are all the same; in single precision rows of which
 * two that count differ in them alone are chosen from once more, by whole keys. LDS: 8 bytes for every chosen expert of the workgroup's rows.
 */
template <typename T, int G, int ENTRIES>
__global__ void __launch_bounds__(ROUTE_THREADS)
RouteKernel(const T* __restrict__ logits, long long strideLogits, T* __restrict__ weights, long long strideWeights, int* __restrict__ index,
            long long strideIndex, long long rows, int experts, int chosen, int normalised)
{
    constexpr int ROWS = ROUTE_THREADS / G;
    constexpr unsigned LAST = G * ENTRIES - 1;   // bits of an expert's number
    static_assert(LAST < 1u << 13, "bits that are free in a key of a half");
    extern __shared__ unsigned routeLds[];
    const int lane = threadIdx.x % G;
    unsigned* const keys = routeLds + threadIdx.x / G * (2 * chosen);
    int* const indices = reinterpret_cast<int*>(keys + chosen);
    for (long long first = static_cast<long long>(blockIdx.x) * ROWS; first < rows; first += static_cast<long long>(gridDim.x) * ROWS) {
        const long long row = min(first + threadIdx.x / G, rows - 1);   // (lanes behind the last row do its work once more)
        const T* const own = logits + row * strideLogits;
        float v[ENTRIES];
        loadLogits(own, lane * ENTRIES, experts, v);
        unsigned key[ENTRIES], top = 0;
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) {
            key[i] = routeKey(v[i]);
            top = max(top, key[i]);
            key[i] = (key[i] & ~LAST) | (LAST - (lane * ENTRIES + i));
        }
        top = largestOfLanes<G>(top);
        const bool any = top > ROUTE_KEY_NONE;
        const float largest = any ? routeValue(top) : 0.0f;
        RouteSort<ENTRIES>::template sort<0, ENTRIES>(key);
        unsigned before = 0;
        bool close = false;
        for (int j = 0; j < chosen; ++j) {
            const unsigned best = largestOfLanes<G>(key[0]);
            // (by bits: of a choice between entries the compiler makes one between their numbers)
            const unsigned mine = key[0] == best ? ~0u : 0u;
#pragma unroll
            for (int i = 0; i + 1 < ENTRIES; ++i) key[i] = (mine & key[i + 1]) | (~mine & key[i]);
            key[ENTRIES - 1] &= ~mine;
            if (lane == 0) keys[j] = best;
            if (sizeof(T) == 4) close |= (best ^ before) <= LAST && best > ROUTE_KEY_NONE;
            before = best;
        }
        if (sizeof(T) == 4) close |= (largestOfLanes<G>(key[0]) ^ before) <= LAST && before > ROUTE_KEY_NONE;
        waveLdsSync();
        if (sizeof(T) == 4 && __ballot(close) != 0) chooseExactly<G>(v, chosen, keys, indices);
        else
            for (int j = lane; j < chosen; j += G) {
                const unsigned k = keys[j];
                const int e = k > ROUTE_KEY_NONE ? static_cast<int>(LAST - (k & LAST)) : -1;
                indices[j] = e;
                // (the logit itself, or the bits of it that there are)
                if (sizeof(T) == 4) keys[j] = e >= 0 ? routeKey(static_cast<float>(own[e])) : k;
                else keys[j] = k & 0x80000000u ? k & ~LAST : k | LAST;
            }
        float total = 0;
        if (normalised) {
            for (int j = lane; j < chosen; j += G) total += indices[j] >= 0 ? routeExp<false>(routeValue(keys[j]) - largest) : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < ENTRIES; ++i) total += routeExp<false>(v[i] - largest);
        }
        total = routeTotal(totalOfLanes<G>(total), top);
        if (first + threadIdx.x / G < rows)
            for (int j = lane; j < chosen; j += G) {
                const int e = indices[j];
                index[row * strideIndex + j] = e;
                weights[row * strideWeights + j] = static_cast<T>(e >= 0 ? routeExp<true>(routeValue(keys[j]) - largest) / total : 0.0f);
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
        const bool any = top > ROUTE_KEY_NONE;
        const float largest = any ? routeValue(top) : 0.0f;
        float total = 0;
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) {
            v[i] = routeExp<false>(v[i] - largest);
            total += v[i];
        }
        __builtin_memcpy(__builtin_assume_aligned(own + from, 16), v, sizeof(v));
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
        const float share = 1.0f / routeTotal(totalOfLanes<G>(normalised ? taken : total), top);
        inner = totalOfLanes<G>(inner) * share;
        waveLdsSync();
        unsigned none[ENTRIES];
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) none[i] = ROUTE_NOT_CHOSEN;
        __builtin_memcpy(__builtin_assume_aligned(own + from, 16), none, sizeof(none));
        waveLdsSync();
        for (int j = lane; j < chosen; j += G) {
            const int e = indices[j];
            const float g = static_cast<float>(gradients[j]);
            if (e >= 0 && e < experts) own[e] = g != g ? __builtin_nanf("") : g;
        }
        waveLdsSync();
        float out[ENTRIES];
        unsigned gradient[ENTRIES];
        __builtin_memcpy(gradient, __builtin_assume_aligned(own + from, 16), sizeof(gradient));
#pragma unroll
        for (int i = 0; i < ENTRIES; ++i) {
            const unsigned bits = gradient[i];
            const bool held = bits != ROUTE_NOT_CHOSEN;
            const float g = held ? __builtin_bit_cast(float, bits) : 0.0f;
            // (rows without experts have no total)
            out[i] = any && (held || !normalised) ? v[i] * share * (g - inner) : 0.0f;
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

/** A key and, below it, the expert: of equal keys the first is the largest. Less than 2^64 - 1. */
__device__ __forceinline__ unsigned long long routePair(float v, int expert)
{
    return static_cast<unsigned long long>(routeKey(v)) << 32 | (0xfffffffeu - static_cast<unsigned>(expert));
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
        unsigned long long last = ~0ull;   // (above every pair)
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
                indices[j] = key > ROUTE_KEY_NONE ? static_cast<int>(0xfffffffeu - static_cast<unsigned>(last)) : -1;
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

#pragma once
// Rows of tokens to the places of their experts' rows, and back.
//
//   dispatch: rows[places[t][j]] = x[t];  dx[t] = sum over j of drows[places[t][j]]
//   combine:  y[t] = residual[t] + sum over j of w[t][j] rows[places[t][j]]
//             drows[places[t][j]] = w[t][j] dy[t],  dw[t][j] = <dy[t], rows[places[t][j]]>,  dresidual = dy
//
// A place p < 0 is that of row -1 - p, which belongs to no expert: it gets zeros and is not read. Places are those of a permutation, so that
// every row is written once; others than those of a row there is are left out.
//
// All of them are bound by memory, and go by token: what a token has of its own (x, dy) is read once, however many experts it has.

#include <qmlp/kernels/token_types.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

constexpr int EXPERT_ROWS_THREADS = 256;

/** Which row a place means, and whether it belongs to an expert. */
struct Place
{
    long long row;
    bool expert, there;
    __device__ __forceinline__ Place(int p, long long rows) : row(p >= 0 ? p : ~p), expert(p >= 0), there(row < rows) {}
};

/** Weights of T or of floats; null: ones. */
template <typename T>
__device__ __forceinline__ float weightAt(const void* weights, int single, long long at)
{
    if (!weights) return 1.0f;
    return single ? static_cast<const float*>(weights)[at] : static_cast<float>(static_cast<const T*>(weights)[at]);
}

/** G lanes per token; T is any type of its size. */
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(EXPERT_ROWS_THREADS)
DispatchKernel(const T* __restrict__ x, long long strideX, const int* __restrict__ places, long long stridePlaces, int chosen, T* __restrict__ rows,
               long long strideRows, long long tokens, int C)
{
    constexpr int TOKENS = EXPERT_ROWS_THREADS / G;
    const long long total = tokens * chosen;
    for (long long t = static_cast<long long>(blockIdx.x) * TOKENS + threadIdx.x / G; t < tokens; t += static_cast<long long>(gridDim.x) * TOKENS) {
        const int* const own = places + t * stridePlaces;
        for (int c = threadIdx.x % G * VEC; c < C; c += G * VEC) {
            const int at = VEC == 1 ? c : min(c, C - VEC);   // the last piece ends with the row
            Raw<T, VEC> raw;
            raw.load(x + t * strideX + at);
            for (int j = 0; j < chosen; ++j) {
                const Place place(own[j], total);
                if (!place.there) continue;
                Raw<T, VEC> out;
#pragma unroll
                for (int k = 0; k < VEC; ++k) out.v[k] = place.expert ? raw.v[k] : 0;
                if constexpr (VEC * sizeof(T) == 16) streamPiece(rows + place.row * strideRows + at, __builtin_bit_cast(u32x4, out));
                else __builtin_memcpy(rows + place.row * strideRows + at, &out, sizeof(out));
            }
        }
    }
}

/** G lanes per token. weights, residual: may be null. */
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(EXPERT_ROWS_THREADS)
CombineKernel(const T* __restrict__ rows, long long strideRows, const int* __restrict__ places, long long stridePlaces, int chosen,
              const void* __restrict__ weights, long long strideWeights, int single, const T* __restrict__ residual, long long strideResidual,
              T* __restrict__ y, long long strideY, long long tokens, int C)
{
    constexpr int TOKENS = EXPERT_ROWS_THREADS / G;
    const long long total = tokens * chosen;
    for (long long t = static_cast<long long>(blockIdx.x) * TOKENS + threadIdx.x / G; t < tokens; t += static_cast<long long>(gridDim.x) * TOKENS) {
        const int* const own = places + t * stridePlaces;
        for (int c = threadIdx.x % G * VEC; c < C; c += G * VEC) {
            const int at = VEC == 1 ? c : min(c, C - VEC);
            float sum[VEC] = {};
            if (residual) loadFloats(residual + t * strideResidual + at, sum);
            for (int j = 0; j < chosen; ++j) {
                const Place place(own[j], total);
                if (!place.there || !place.expert) continue;
                float v[VEC];
                loadFloats(rows + place.row * strideRows + at, v);
                const float w = weightAt<T>(weights, single, t * strideWeights + j);
#pragma unroll
                for (int k = 0; k < VEC; ++k) sum[k] += w * v[k];
            }
            streamFloats(y + t * strideY + at, sum);
        }
    }
}

/** G (up to 64) lanes per token. adjRows, adjWeights: may be null. */
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(EXPERT_ROWS_THREADS)
CombineAdjointKernel(const T* __restrict__ rows, long long strideRows, const int* __restrict__ places, long long stridePlaces, int chosen,
                     const void* __restrict__ weights, long long strideWeights, int single, const T* __restrict__ adjY, long long strideAdjY,
                     T* __restrict__ adjRows, long long strideAdjRows, void* __restrict__ adjWeights, long long strideAdjWeights, long long tokens, int C)
{
    constexpr int TOKENS = EXPERT_ROWS_THREADS / G;
    const int lane = threadIdx.x % G;
    const long long total = tokens * chosen;
    for (long long first = static_cast<long long>(blockIdx.x) * TOKENS; first < tokens; first += static_cast<long long>(gridDim.x) * TOKENS) {
        const long long t = first + threadIdx.x / G;
        for (int j = 0; j < chosen; ++j) {
            float inner = 0;
            if (t < tokens) {
                const Place place(places[t * stridePlaces + j], total);
                const float w = weightAt<T>(weights, single, t * strideWeights + j);
                if (place.there)
                    for (int c = lane * VEC; c < C; c += G * VEC) {
                        const int at = VEC == 1 ? c : min(c, C - VEC);
                        float g[VEC], v[VEC] = {};
                        loadFloats(adjY + t * strideAdjY + at, g);
                        if (place.expert && adjWeights) loadFloats(rows + place.row * strideRows + at, v);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            if (place.expert && k >= c - at) inner += g[k] * v[k];
                            g[k] = place.expert ? w * g[k] : 0.0f;
                        }
                        if (adjRows) streamFloats(adjRows + place.row * strideAdjRows + at, g);
                    }
            }
            if (!adjWeights) continue;
            inner = sumOfLanes<G>(inner);
            if (lane == 0 && t < tokens) {
                if (single) static_cast<float*>(adjWeights)[t * strideAdjWeights + j] = inner;
                else static_cast<T*>(adjWeights)[t * strideAdjWeights + j] = static_cast<T>(inner);
            }
        }
    }
}

QUICKMLP_KERNEL_NAMESPACE_END

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
// All of them are bound by memory, and go by token: what a token has of its own (x, dy) is read once, however many experts it has. Results are stored
// past the L2. Where there are few tokens, workgroups share out their columns, wavefronts of the adjoint kernel their rows. Measured, us: 32768 tokens
// of 2 experts, 2048 channels, bfloat16 70 (dispatch, 403 MB, 5.8 TB/s), 72 (its gradient), 91 (combine with residual, 537 MB, 5.9 TB/s), 121 (its
// gradients, 671 MB, 5.5 TB/s); 5003 tokens of 3, 333 floats 8.1 (combine), 10.8 (gradients); 24 tokens of 2, 1024 channels, bfloat16 2.8 and 3.2.

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

/** The columns of a workgroup: those of its number among 'parts', where there are few tokens, a step of its lanes each. */
template <int VEC, int G>
struct Columns
{
    int first, step;
    long long block;   // of tokens
    __device__ __forceinline__ explicit Columns(int parts)
        : first((static_cast<int>(blockIdx.x % parts) * G + static_cast<int>(threadIdx.x) % G) * VEC), step(parts * G * VEC), block(blockIdx.x / parts)
    {
    }
    /** The last piece ends with the row. */
    static __device__ __forceinline__ int at(int c, int C) { return VEC == 1 ? c : min(c, C - VEC); }
};

/** G lanes per token; T is any type of its size. */
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(EXPERT_ROWS_THREADS)
DispatchKernel(const T* __restrict__ x, long long strideX, const int* __restrict__ places, long long stridePlaces, int chosen, T* __restrict__ rows,
               long long strideRows, long long tokens, int C, int parts)
{
    constexpr int TOKENS = EXPERT_ROWS_THREADS / G;
    const long long total = tokens * chosen, blocks = gridDim.x / parts;
    const Columns<VEC, G> columns(parts);
    for (long long t = columns.block * TOKENS + threadIdx.x / G; t < tokens; t += blocks * TOKENS) {
        const int* const own = places + t * stridePlaces;
        for (int c = columns.first; c < C; c += columns.step) {
            const int at = columns.at(c, C);
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
              T* __restrict__ y, long long strideY, long long tokens, int C, int parts)
{
    constexpr int TOKENS = EXPERT_ROWS_THREADS / G;
    const long long total = tokens * chosen, blocks = gridDim.x / parts;
    const Columns<VEC, G> columns(parts);
    for (long long t = columns.block * TOKENS + threadIdx.x / G; t < tokens; t += blocks * TOKENS) {
        const int* const own = places + t * stridePlaces;
        for (int c = columns.first; c < C; c += columns.step) {
            const int at = columns.at(c, C);
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

/**
 * G (up to 64) lanes per token, or for each of 'split' parts of its rows, BATCH pieces of a row a lane at a time. adjRows, adjWeights: may be null.
 * What they hold of dy at a time stays for all rows of a token, where it is all of it.
 */
template <typename T, int VEC, int G, int BATCH>
__global__ void __launch_bounds__(EXPERT_ROWS_THREADS)
CombineAdjointKernel(const T* __restrict__ rows, long long strideRows, const int* __restrict__ places, long long stridePlaces, int chosen,
                     const void* __restrict__ weights, long long strideWeights, int single, const T* __restrict__ adjY, long long strideAdjY,
                     T* __restrict__ adjRows, long long strideAdjRows, void* __restrict__ adjWeights, long long strideAdjWeights, long long tokens, int C,
                     int split)
{
    constexpr int UNITS = EXPERT_ROWS_THREADS / G, STEP = G * VEC;
    const int lane = threadIdx.x % G;
    const long long total = tokens * chosen, units = tokens * split;   // (less than 2^31)
    const bool once = C <= BATCH * STEP;
    for (long long first = static_cast<long long>(blockIdx.x) * UNITS; first < units; first += static_cast<long long>(gridDim.x) * UNITS) {
        const long long unit = min(first + threadIdx.x / G, units - 1);   // (lanes behind the last one do its work once more)
        const long long t = split == 1 ? unit : static_cast<unsigned>(unit) / static_cast<unsigned>(split);
        Raw<T, VEC> g[BATCH];
        auto load = [&](int c) {
#pragma unroll
            for (int n = 0; n < BATCH; ++n)
                if (c + n * STEP < C) g[n].load(adjY + t * strideAdjY + Columns<VEC, G>::at(c + n * STEP, C));
        };
        if (once) load(lane * VEC);
        for (int j = static_cast<int>(unit - t * split); j < chosen; j += split) {
            const Place place(places[t * stridePlaces + j], total);
            const bool read = place.expert && place.there;
            const float w = read ? weightAt<T>(weights, single, t * strideWeights + j) : 0.0f;
            float inner = 0;
            if (place.there)
                for (int c = lane * VEC; c < C; c += BATCH * STEP) {
                    Raw<T, VEC> v[BATCH];
                    if (!once) load(c);
                    if (read && adjWeights)
#pragma unroll
                        for (int n = 0; n < BATCH; ++n)
                            if (c + n * STEP < C) v[n].load(rows + place.row * strideRows + Columns<VEC, G>::at(c + n * STEP, C));
#pragma unroll
                    for (int n = 0; n < BATCH; ++n) {
                        if (c + n * STEP >= C) continue;
                        const int at = Columns<VEC, G>::at(c + n * STEP, C);
                        float out[VEC];
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            const float d = static_cast<float>(g[n].v[k]);
                            // (entries that the piece before has, too, are left out)
                            if (adjWeights && read && k >= c + n * STEP - at) inner += d * static_cast<float>(v[n].v[k]);
                            out[k] = read ? w * d : 0.0f;
                        }
                        if (adjRows) streamFloats(adjRows + place.row * strideAdjRows + at, out);
                    }
                }
            if (!adjWeights) continue;
            inner = sumOfLanes<G>(inner);
            if (lane != 0) continue;
            if (single) static_cast<float*>(adjWeights)[t * strideAdjWeights + j] = inner;
            else static_cast<T*>(adjWeights)[t * strideAdjWeights + j] = static_cast<T>(inner);
        }
    }
}

QUICKMLP_KERNEL_NAMESPACE_END

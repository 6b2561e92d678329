#pragma once
// Layer norm over the channels of every row, and its adjoint.
//
//   y = n w + b,  n = (x - mean) r,  r = 1 / sqrt(variance + eps)
//   dx = r (h - avg(h) - n avg(h n)),  h = dy w;   dw = sum over rows of dy n,  db = sum over rows of dy
//
// Both are bound by memory: a row is read once, stays in the registers of the G lanes that share it, and mean and variance
// are two sums over them (the variance of what is left after the mean is taken off, so that a large mean costs no digits).
// Workgroups stay for many rows, with the weights in registers; the adjoint's sums over rows are kept there as well and
// leave a workgroup once, as a row of 'partial', which a second kernel sums in a fixed order.
//
// Measured: 32768 x 4096 bfloat16 105 us forward and 143 + 5 us adjoint, 5.1 and 5.6 TB/s of what has to be moved (a large copy: 5.1 to
// 5.5); 4099 x 777 float 6.6 and 11.7 + 4.0 us; one row of 1024 halves 2.8 us.

#include <qmlp/kernels/token_types.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

constexpr int layerNormThreads(int G) { return G < 256 ? 256 : G; }

/** Sums of N values over the G lanes of a row, in all of them. 'slots': LDS of wavefronts x N floats, for rows of several wavefronts. */
template <int G, int N>
__device__ __forceinline__ void sumOfRow(float (&v)[N], float* slots)
{
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sumOfLanes<(G < 64 ? G : 64)>(v[i]);
    if constexpr (G > 64) {
        constexpr int WAVES = G / 64;
        const int wave = threadIdx.x / 64;
        __syncthreads();   // the slots' readers of before are done
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) slots[i * WAVES + wave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0;
#pragma unroll
            for (int k = 0; k < WAVES; ++k) v[i] += slots[i * WAVES + k];
        }
    }
}

/** Entries of a lane's pieces of a vector of C entries; 'otherwise' without a vector. */
template <typename T, int VEC, int G, int CHUNKS>
__device__ __forceinline__ void loadPieces(const RowPieces<VEC, G>& at, const T* __restrict__ p, float otherwise, float (&v)[CHUNKS][VEC])
{
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j][k] = otherwise;
        if (p && at.has(j)) loadFloats(p + at.start(j), v[j]);
    }
}

/** A lane's pieces of a row, as they are in memory. */
template <typename T, int VEC, int G, int CHUNKS>
struct RawPieces
{
    Raw<T, VEC> raw[CHUNKS];
    __device__ __forceinline__ void load(const RowPieces<VEC, G>& at, const T* __restrict__ p)
    {
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j)
            if (at.has(j)) raw[j].load(p + at.start(j));
    }
    /** As floats; 0 where the lane has none. */
    __device__ __forceinline__ void floats(const RowPieces<VEC, G>& at, float (&v)[CHUNKS][VEC]) const
    {
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[j][k] = at.has(j) ? static_cast<float>(raw[j].v[k]) : 0;
    }
};

/**
 * One row per G lanes. weight, bias: may be null (1 and 0); mean, rstd: may be null (not kept for an adjoint).
 * G * VEC * CHUNKS >= C >= VEC.
 */
template <typename T, typename W, int VEC, int G, int CHUNKS>
__global__ void __launch_bounds__(layerNormThreads(G))
LayerNormKernel(const T* __restrict__ x, long long strideX, const W* __restrict__ weight, const W* __restrict__ bias, float eps,
                T* __restrict__ y, long long strideY, float* __restrict__ mean, float* __restrict__ rstd, long long rows, int C)
{
    constexpr int ROWS = layerNormThreads(G) / G;
    __shared__ float slots[G > 64 ? G / 64 : 1];
    const RowPieces<VEC, G> at{C, static_cast<int>(threadIdx.x) % G};
    float w[CHUNKS][VEC], b[CHUNKS][VEC];
    loadPieces(at, weight, 1.0f, w);
    loadPieces(at, bias, 0.0f, b);
    const long long step = static_cast<long long>(gridDim.x) * ROWS;
    long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G;
    RawPieces<T, VEC, G, CHUNKS> coming;   // the next row is asked for before the present one is worked on
    if (row < rows) coming.load(at, x + row * strideX);
    for (; row < rows; row += step) {
        float v[CHUNKS][VEC];
        coming.floats(at, v);
        if (row + step < rows) coming.load(at, x + (row + step) * strideX);
        float sum[1] = {0};
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[0] += k >= at.first(j) ? v[j][k] : 0;
        sumOfRow<G>(sum, slots);
        const float m = sum[0] / C;   // (a division: the mean of equal values is exact)
        sum[0] = 0;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                v[j][k] -= m;
                sum[0] += at.has(j) && k >= at.first(j) ? v[j][k] * v[j][k] : 0;
            }
        sumOfRow<G>(sum, slots);
        const float r = 1.0f / sqrtf(sum[0] / C + eps);
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[j][k] = v[j][k] * r * w[j][k] + b[j][k];
            if (at.has(j)) streamFloats(y + row * strideY + at.start(j), v[j]);
        }
        if (at.lane == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
    }
}

/**
 * The adjoint of one row per G lanes. adjX: may be null; partial: a row of 2 C floats per workgroup, its sums for the weight and
 * for the bias, or null.
 */
template <typename T, typename W, int VEC, int G, int CHUNKS>
__global__ void __launch_bounds__(layerNormThreads(G))
LayerNormAdjointKernel(const T* __restrict__ x, long long strideX, const W* __restrict__ weight, const float* __restrict__ mean,
                       const float* __restrict__ rstd, const T* __restrict__ adjY, long long strideAdjY, T* __restrict__ adjX, long long strideAdjX,
                       float* __restrict__ partial, long long rows, int C)
{
    constexpr int ROWS = layerNormThreads(G) / G;
    __shared__ float slots[G > 64 ? 2 * (G / 64) : 1];
    const RowPieces<VEC, G> at{C, static_cast<int>(threadIdx.x) % G};
    float w[CHUNKS][VEC], sumW[CHUNKS][VEC] = {}, sumB[CHUNKS][VEC] = {};
    loadPieces(at, weight, 1.0f, w);
    const float scale = 1.0f / C;
    const long long step = static_cast<long long>(gridDim.x) * ROWS;
    long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / G;
    RawPieces<T, VEC, G, CHUNKS> comingX, comingD;   // of the next row
    float comingMean = 0, comingRstd = 0;
    auto ask = [&](long long r) {
        comingX.load(at, x + r * strideX);
        comingD.load(at, adjY + r * strideAdjY);
        comingMean = mean[r];
        comingRstd = rstd[r];
    };
    if (row < rows) ask(row);
    for (; row < rows; row += step) {
        const float m = comingMean, r = comingRstd;
        float n[CHUNKS][VEC], d[CHUNKS][VEC];
        comingX.floats(at, n);
        comingD.floats(at, d);
        if (row + step < rows) ask(row + step);
        float sums[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                n[j][k] = at.has(j) ? (n[j][k] - m) * r : 0;
                sumW[j][k] += d[j][k] * n[j][k];
                sumB[j][k] += d[j][k];
                d[j][k] *= w[j][k];
                const float h = k >= at.first(j) ? d[j][k] : 0;
                sums[0] += h;
                sums[1] += k >= at.first(j) ? h * n[j][k] : 0;
            }
        sumOfRow<G>(sums, slots);
        const float a = sums[0] * scale, c = sums[1] * scale;
        if (adjX) {
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) d[j][k] = r * (d[j][k] - a - n[j][k] * c);
                if (at.has(j)) streamFloats(adjX + row * strideAdjX + at.start(j), d[j]);
            }
        }
    }
    if (!partial) return;
    float* out = partial + static_cast<long long>(blockIdx.x) * 2 * C;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j)
            if (at.has(j)) {   // (entries of two pieces have the same sums)
                storeFloats(out + at.start(j), sumW[j]);
                storeFloats(out + C + at.start(j), sumB[j]);
            }
    } else {
        // the rows that the workgroup had at a time, one after the other
        __shared__ float total[2][G * VEC * CHUNKS];
        for (int turn = 0; turn < ROWS; ++turn) {
            if (static_cast<int>(threadIdx.x) / G == turn) {
#pragma unroll
                for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        if (at.has(j) && k >= at.first(j)) {
                            const int c = at.start(j) + k;
                            total[0][c] = (turn ? total[0][c] : 0.0f) + sumW[j][k];
                            total[1][c] = (turn ? total[1][c] : 0.0f) + sumB[j][k];
                        }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < C; c += layerNormThreads(G)) {
            out[c] = total[0][c];
            out[C + c] = total[1][c];
        }
    }
}

constexpr int LAYER_NORM_SUM_COLUMNS = 32, LAYER_NORM_SUM_THREADS = 1024;

/** Sums the rows of 'partial' (count x 2 C): the first C columns into adjWeight, the others into adjBias; either may be null. */
template <typename W>
__global__ void __launch_bounds__(LAYER_NORM_SUM_THREADS)
LayerNormSumKernel(const float* __restrict__ partial, int count, int C, W* __restrict__ adjWeight, W* __restrict__ adjBias)
{
    constexpr int COLUMNS = LAYER_NORM_SUM_COLUMNS, SLICES = LAYER_NORM_SUM_THREADS / COLUMNS;
    __shared__ float sums[SLICES][COLUMNS + 1];
    const int column = threadIdx.x % COLUMNS, slice = threadIdx.x / COLUMNS;
    for (long long first = static_cast<long long>(blockIdx.x) * COLUMNS; first < 2ll * C; first += static_cast<long long>(gridDim.x) * COLUMNS) {
        const long long c = first + column;
        float sum = 0;
        if (c < 2ll * C)
#pragma unroll 8
            for (int p = slice; p < count; p += SLICES) sum += partial[static_cast<long long>(p) * 2 * C + c];
        sums[slice][column] = sum;
        __syncthreads();
#pragma unroll
        for (int half = SLICES / 2; half > 0; half /= 2) {
            if (slice < half) sums[slice][column] += sums[slice + half][column];
            __syncthreads();
        }
        if (slice == 0 && c < 2ll * C) {   // (the total's reader is the one who writes there next)
            W* out = c < C ? adjWeight : adjBias;
            if (out) out[c < C ? c : c - C] = static_cast<W>(sums[0][column]);
        }
    }
}

constexpr int LAYER_NORM_LONG_THREADS = 1024;

/** LayerNormKernel for rows that no workgroup keeps in its registers: they are read three times, the last two from the L2. */
template <typename T, typename W>
__global__ void __launch_bounds__(LAYER_NORM_LONG_THREADS)
LayerNormLongKernel(const T* __restrict__ x, long long strideX, const W* __restrict__ weight, const W* __restrict__ bias, float eps,
                    T* __restrict__ y, long long strideY, float* __restrict__ mean, float* __restrict__ rstd, long long rows, int C)
{
    __shared__ float slots[LAYER_NORM_LONG_THREADS / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = x + row * strideX;
        float sum[1] = {0};
        for (int c = threadIdx.x; c < C; c += LAYER_NORM_LONG_THREADS) sum[0] += static_cast<float>(in[c]);
        sumOfRow<LAYER_NORM_LONG_THREADS>(sum, slots);
        const float m = sum[0] / C;
        sum[0] = 0;
        for (int c = threadIdx.x; c < C; c += LAYER_NORM_LONG_THREADS) {
            const float v = static_cast<float>(in[c]) - m;
            sum[0] += v * v;
        }
        sumOfRow<LAYER_NORM_LONG_THREADS>(sum, slots);
        const float r = 1.0f / sqrtf(sum[0] / C + eps);
        for (int c = threadIdx.x; c < C; c += LAYER_NORM_LONG_THREADS)
            y[row * strideY + c] = static_cast<T>((static_cast<float>(in[c]) - m) * r * (weight ? static_cast<float>(weight[c]) : 1.0f)
                                                  + (bias ? static_cast<float>(bias[c]) : 0.0f));
        if (threadIdx.x == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
    }
}

/** adjX of such rows; the sums over rows are LayerNormLongSumsKernel's. */
template <typename T, typename W>
__global__ void __launch_bounds__(LAYER_NORM_LONG_THREADS)
LayerNormLongAdjointKernel(const T* __restrict__ x, long long strideX, const W* __restrict__ weight, const float* __restrict__ mean,
                           const float* __restrict__ rstd, const T* __restrict__ adjY, long long strideAdjY, T* __restrict__ adjX,
                           long long strideAdjX, long long rows, int C)
{
    __shared__ float slots[2 * LAYER_NORM_LONG_THREADS / 64];
    const float scale = 1.0f / C;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const float m = mean[row], r = rstd[row];
        auto normal = [&](int c) { return (static_cast<float>(x[row * strideX + c]) - m) * r; };
        auto inner = [&](int c) { return static_cast<float>(adjY[row * strideAdjY + c]) * (weight ? static_cast<float>(weight[c]) : 1.0f); };
        float sums[2] = {0, 0};
        for (int c = threadIdx.x; c < C; c += LAYER_NORM_LONG_THREADS) {
            const float h = inner(c);
            sums[0] += h;
            sums[1] += h * normal(c);
        }
        sumOfRow<LAYER_NORM_LONG_THREADS>(sums, slots);
        for (int c = threadIdx.x; c < C; c += LAYER_NORM_LONG_THREADS)
            adjX[row * strideAdjX + c] = static_cast<T>(r * (inner(c) - sums[0] * scale - normal(c) * (sums[1] * scale)));
    }
}

/** Sums over a slice of the rows, one column per lane: a row of 'partial' per slice. Workgroups: slices x columns / 256. */
template <typename T>
__global__ void __launch_bounds__(256)
LayerNormLongSumsKernel(const T* __restrict__ x, long long strideX, const float* __restrict__ mean, const float* __restrict__ rstd,
                        const T* __restrict__ adjY, long long strideAdjY, float* __restrict__ partial, long long rows, int C, int slices)
{
    const int slice = blockIdx.x % slices;
    const int c = blockIdx.x / slices * 256 + threadIdx.x;
    if (c >= C) return;
    float sumW = 0, sumB = 0;
    for (long long row = slice; row < rows; row += slices) {
        const float d = static_cast<float>(adjY[row * strideAdjY + c]);
        sumW += d * ((static_cast<float>(x[row * strideX + c]) - mean[row]) * rstd[row]);
        sumB += d;
    }
    partial[static_cast<long long>(slice) * 2 * C + c] = sumW;
    partial[static_cast<long long>(slice) * 2 * C + C + c] = sumB;
}

QUICKMLP_KERNEL_NAMESPACE_END

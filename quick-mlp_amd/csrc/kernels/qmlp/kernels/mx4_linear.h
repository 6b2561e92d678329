#pragma once
// The linear layer of every expert on its own rows, with rows and weights of 4 bits (mx4.h):
//
//   y[r] = W[e] x[r] + b[e]  for the rows r of expert e: offsets[e] <= r < offsets[e + 1];  zero for rows behind the last expert's
//
// The matrix cores multiply blocks of 32 codes with their scales: an operand of 16 rows by 128 entries has a block of a row in each lane,
// 16 bytes and a byte of scale, as they lie in memory. Sums are held in floats.

#include <qmlp/kernels/grouped_linear.h>
#include <qmlp/kernels/mx4.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

typedef int i32x8 __attribute__((ext_vector_type(8)));

/** Codes and scales of a matrix, or of one per expert: rows of 'blocks' blocks. */
struct Mx4Matrix
{
    const unsigned char *codes, *scales;
    long long codesExpert, scalesExpert;   // strides between experts
    long long codesRow, scalesRow;         // and between rows
};

/** offsets: null where there is one expert. */
__device__ __forceinline__ ExpertTile mx4Tile(const int* __restrict__ offsets, int experts, int rows, int tileRows, int place)
{
    if (offsets) return expertTile(offsets, experts, rows, tileRows, place);
    ExpertTile t;
    t.expert = 0;
    t.index = place;
    t.from = static_cast<int>(min(static_cast<long long>(place) * tileRows, static_cast<long long>(rows)));
    t.to = static_cast<int>(min((static_cast<long long>(place) + 1) * tileRows, static_cast<long long>(rows)));
    t.expertRows = rows;
    return t;
}

constexpr int MX4_FEW_WAVES = 4;
/**
 * 16 rows by 16 outputs per wavefront, operands straight from memory: lane l has block l / 16 of every four of row l % 16. Results: lane l has
 * outputs 4 (l / 16) .. + 3 of row l % 16.
 */
template <typename T>
__global__ void __launch_bounds__(64 * MX4_FEW_WAVES)
Mx4FewKernel(const unsigned char* __restrict__ x, const unsigned char* __restrict__ scalesX, long long strideX, long long strideScalesX, Mx4Matrix weights,
             const T* __restrict__ bias, long long strideBias, const int* __restrict__ offsets, int experts, T* __restrict__ y, long long strideY, int rows,
             int J, int blocks, int places, int tilesJ)
{
    const int place = static_cast<int>(blockIdx.x % places), tile = static_cast<int>(blockIdx.x / places);
    const ExpertTile at = mx4Tile(offsets, experts, rows, 16, place);
    if (at.to <= at.from) return;
    const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
    const int j0 = (tile * MX4_FEW_WAVES + static_cast<int>(threadIdx.x) / 64) * 16;
    if (j0 >= J) return;
    const bool none = at.expert >= experts;
    f32x4 sum = {};
    if (!none) {
        const long long row = min(at.from + i, at.to - 1), output = min(j0 + i, J - 1);   // (rows and outputs behind the last: any, not written)
        const unsigned char* const ownX = x + row * strideX;
        const unsigned char* const ownScalesX = scalesX + row * strideScalesX;
        const unsigned char* const own = weights.codes + at.expert * weights.codesExpert + output * weights.codesRow;
        const unsigned char* const ownScales = weights.scales + at.expert * weights.scalesExpert + output * weights.scalesRow;
        for (int b = g; b < (blocks + 3) / 4 * 4; b += 4) {
            i32x8 codesW = {}, codesX = {};
            unsigned scaleW = 127, scaleX = 127;
            if (b < blocks) {
                __builtin_memcpy(&codesW, own + b * 16ll, 16);
                __builtin_memcpy(&codesX, ownX + b * 16ll, 16);
                scaleW = ownScales[b];
                scaleX = ownScalesX[b];
            }
            sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codesW, codesX, sum, 4, 4, 0, scaleW, 0, scaleX);
        }
    }
    if (at.from + i >= at.to) return;
    const int j = j0 + 4 * g;
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = sum[k] + (bias && !none && j + k < J ? static_cast<float>(bias[at.expert * strideBias + j + k]) : 0.0f);
    storeUpToFour(y + (at.from + i) * strideY + j, v, J - j);
}

QUICKMLP_KERNEL_NAMESPACE_END

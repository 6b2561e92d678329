#pragma once
// Numbers of 4 bits in blocks of 32 with a common scale: MXFP4 as the OCP Microscaling Formats specification 1.0 has it.
//
//   block: 32 consecutive entries of a row;  scale 2^e, e = floor(log2(largest magnitude)) - 2, between -127 and 127, kept as e + 127
//   code: sign, two bits of exponent and one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6;  nearest to x / 2^e, halfway to the even code, 6 beyond
//   a block with an infinity or a NaN has the scale 255, which makes all of its entries NaN
//
// A row of n entries has ceil(n / 32) blocks: 16 bytes of codes each, the first entry in the low bits, zeros behind the last, and a byte of scale.
// The hardware's conversions take the exponent bits of a float as the scale, also those of 0 (2^-127).
//
// Bound by memory. Four lanes share a block that is quantised, 8 entries each, so that a wavefront writes consecutive bytes of codes; where values are
// written a lane has 16 bytes of them. Measured: 65536 rows of 2048, bfloat16, 64 us to codes (340 MB, 5.3 TB/s) and 49 us back (6.9 TB/s; 63 without
// stores past the L2); 4099 rows of 777 floats 4.2 and 4.9 us (4 entries a lane to codes: 4.9; 8 back: 6.1).

#include <qmlp/kernels/token_types.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

constexpr int MX4_THREADS = 256, MX4_BLOCK = 32;
constexpr int MX4_ENTRIES = 8, MX4_LANES = MX4_BLOCK / MX4_ENTRIES;   // of a block that is quantised

/** The scale (biased exponent) of a block whose largest magnitude has these bits. */
__device__ __forceinline__ unsigned mx4Scale(unsigned largest)
{
    const int exponent = static_cast<int>(largest >> 23);
    return exponent == 255 ? 255 : max(exponent - 2, 0);
}
__device__ __forceinline__ float mx4ScaleBits(unsigned scale) { return __builtin_bit_cast(float, scale << 23); }

/** The codes of values that are finite. */
__device__ __forceinline__ unsigned mx4Codes(const float (&v)[MX4_ENTRIES], float scale)
{
    unsigned codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], scale, 3);
}

/** The lane's entries of a row of C, zeros behind the last. */
template <typename T>
__device__ __forceinline__ void mx4Load(const T* __restrict__ row, int at, int C, float (&v)[MX4_ENTRIES])
{
    if (at + MX4_ENTRIES <= C) loadFloats(row + at, v);
    else
#pragma unroll
        for (int k = 0; k < MX4_ENTRIES; ++k) v[k] = at + k < C ? static_cast<float>(row[at + k]) : 0.0f;
}
/** The codes of the lane's entries and the scale of the block, which four lanes share: all of them call it. */
__device__ __forceinline__ unsigned mx4Pack(const float (&v)[MX4_ENTRIES], unsigned& scale)
{
    unsigned largest = 0;
#pragma unroll
    for (int k = 0; k < MX4_ENTRIES; ++k) largest = max(largest, __builtin_bit_cast(unsigned, v[k]) & 0x7fffffffu);
    // (lanes 1 0 3 2 and 2 3 0 1 of every four)
    largest = max(largest, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(largest), 0xb1, 0xf, 0xf, true)));
    largest = max(largest, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(largest), 0x4e, 0xf, 0xf, true)));
    scale = mx4Scale(largest);
    return scale == 255 ? 0 : mx4Codes(v, mx4ScaleBits(scale));
}

/** A block of a row. (A division of 32 bits where that is enough.) */
struct Mx4Unit
{
    long long row;
    int block;
    __device__ __forceinline__ Mx4Unit(long long unit, int blocks)
    {
        if (unit >> 32 == 0) row = static_cast<unsigned>(unit) / static_cast<unsigned>(blocks);
        else row = unit / blocks;
        block = static_cast<int>(unit - row * blocks);
    }
};

/** x (rows, C), rows of any stride; codes (rows, blocks, 16) and scales (rows, blocks), rows of any stride. */
template <typename T>
__global__ void __launch_bounds__(MX4_THREADS)
Mx4QuantiseKernel(const T* __restrict__ x, long long strideX, unsigned char* __restrict__ codes, long long strideCodes, unsigned char* __restrict__ scales,
                  long long strideScales, long long units, int blocks, int C)
{
    const int lane = threadIdx.x % MX4_LANES;
    for (long long first = static_cast<long long>(blockIdx.x) * MX4_THREADS; first < units * MX4_LANES; first += static_cast<long long>(gridDim.x) * MX4_THREADS) {
        const Mx4Unit at(min((first + threadIdx.x) / MX4_LANES, units - 1), blocks);   // (the last ones are written more than once)
        float v[MX4_ENTRIES];
        mx4Load(x + at.row * strideX, at.block * MX4_BLOCK + lane * MX4_ENTRIES, C, v);
        unsigned scale;
        const unsigned packed = mx4Pack(v, scale);
        __builtin_memcpy(codes + at.row * strideCodes + at.block * 16 + lane * 4, &packed, 4);
        if (lane == 0) scales[at.row * strideScales + at.block] = static_cast<unsigned char>(scale);
    }
}

/** What codes and scales stand for: y (rows, C). */
template <typename T>
__global__ void __launch_bounds__(MX4_THREADS)
Mx4ValuesKernel(const unsigned char* __restrict__ codes, long long strideCodes, const unsigned char* __restrict__ scales, long long strideScales,
                T* __restrict__ y, long long strideY, long long units, int blocks, int C)
{
    constexpr int N = WIDE<T>, LANES = MX4_BLOCK / N;
    const int lane = threadIdx.x % LANES;
    for (long long i = static_cast<long long>(blockIdx.x) * MX4_THREADS + threadIdx.x; i < units * LANES; i += static_cast<long long>(gridDim.x) * MX4_THREADS) {
        const Mx4Unit at(i / LANES, blocks);
        unsigned packed = 0;
        __builtin_memcpy(&packed, codes + at.row * strideCodes + at.block * 16 + lane * (N / 2), N / 2);
        const unsigned scale = scales[at.row * strideScales + at.block];
        const float s = mx4ScaleBits(scale);
        f32x2 pairs[N / 2];
        pairs[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, s, 0);
        pairs[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, s, 1);
        if constexpr (N == 8) {
            pairs[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, s, 2);
            pairs[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, s, 3);
        }
        float v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = scale == 255 ? __builtin_nanf("") : pairs[k / 2][k % 2];
        const int column = at.block * MX4_BLOCK + lane * N;
        T* const to = y + at.row * strideY + column;
        if (column + N <= C) streamFloats(to, v);
        else
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (column + k < C) to[k] = static_cast<T>(v[k]);
    }
}

QUICKMLP_KERNEL_NAMESPACE_END

#pragma once
// Element types and vector accesses shared by the operators on rows of tokens (layer_norm.h, embedding.h, row_groups.h,
// grouped_linear.h). Values are read and written in float, half or bfloat16 and computed in float.

#include <qmlp/kernels/common.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

typedef __bf16 bf16;

/** Entries of T in an access of 16 bytes. */
template <typename T>
constexpr int WIDE = 16 / static_cast<int>(sizeof(T));

/** N consecutive entries as they are in memory, for values that wait in registers: half of the registers of floats. */
template <typename T, int N>
struct Raw
{
    T v[N];
    __device__ __forceinline__ void load(const T* __restrict__ p) { __builtin_memcpy(v, p, sizeof(v)); }
};

/**
 * N consecutive entries as floats. The address needs the alignment of one entry only: the hardware takes wide accesses at any
 * address, so rows of odd lengths are moved 16 bytes at a time as well.
 */
template <int N, typename T>
__device__ __forceinline__ void loadFloats(const T* __restrict__ p, float (&v)[N])
{
    T raw[N];
    __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(raw[i]);
}

/** N consecutive entries from floats, each rounded once to nearest even. */
template <int N, typename T>
__device__ __forceinline__ void storeFloats(T* __restrict__ p, const float (&v)[N])
{
    if constexpr (N == 1) {
        *p = static_cast<T>(v[0]);
    } else {
        typedef T Pair __attribute__((ext_vector_type(2)));
        Pair raw[N / 2];
#pragma unroll
        for (int i = 0; i < N; i += 2) raw[i / 2] = __builtin_convertvector(f32x2{v[i], v[i + 1]}, Pair);
        __builtin_memcpy(p, raw, sizeof(raw));
    }
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
/**
 * 16 bytes of a result, at any address that T may have. They are marked as not to be kept: the kernel that reads them comes later, and lines that
 * the L2 would hold until then are in the way of this one's reads and are still to be written when it ends. us without | with the mark, one
 * operator alone, half: lookup of 65536 x 2048 88 | 78, layer norm of them 112 | 92; layer of 2^17 rows of 512 experts, 64 -> 64, 10.8 | 9.2; of
 * 16384 rows of 16, 256 -> 512, 14.7 | 12.5; of 99480 rows of 44, 16 -> 2096, 182 | 135; three products of 32768 rows of 16, 2048 -> 4096,
 * bfloat16, 1648 | 1645. With its readers right behind (lookup, layer norm, layer, activation, layer), rows x channels -> hidden: 64 x 256 -> 512
 * 16.8 | 17.4; 2048 x 256 -> 512 22.0 | 22.8; 16384 x 256 -> 512 62 | 60; 2^17 x 64 -> 64 55.6 | 57.7; 32768 x 1024 -> 2048 513 | 502; 65536 x
 * 2048 -> 2048 1526 | 1534.
 */
template <typename T>
__device__ __forceinline__ void streamPiece(T* __restrict__ p, u32x4 piece)
{
    typedef u32x4 Loose __attribute__((aligned(2)));   // of the smallest T
    __builtin_nontemporal_store(piece, reinterpret_cast<Loose*>(p));
}
/** As storeFloats(), for results. */
template <int N, typename T>
__device__ __forceinline__ void streamFloats(T* __restrict__ p, const float (&v)[N])
{
    if constexpr (N * sizeof(T) == 16) {
        u32x4 piece;
        storeFloats(reinterpret_cast<T*>(&piece), v);
        streamPiece(p, piece);
    } else
        storeFloats(p, v);
}

/** Sum over the G (a power of two up to 64) consecutive lanes that a lane belongs to, in all of them. */
template <int G>
__device__ __forceinline__ float sumOfLanes(float v)
{
#pragma unroll
    for (int m = 1; m < G; m *= 2) v += __shfl_xor(v, m);
    return v;
}

/**
 * The places of a row of C entries that one of the G lanes of the row holds: CHUNKS pieces of VEC entries. The last piece of
 * a row whose length is no multiple of VEC starts earlier, so that it ends with the row: its first entries are the piece's before
 * too, read and written twice with the same values, and 'first' tells how many to leave out of sums. C >= VEC.
 */
template <int VEC, int G>
struct RowPieces
{
    int C, lane;
    __device__ __forceinline__ bool has(int j) const { return (j * G + lane) * VEC < C; }
    __device__ __forceinline__ int start(int j) const
    {
        const int c = (j * G + lane) * VEC;
        return VEC == 1 ? c : min(c, C - VEC);
    }
    __device__ __forceinline__ int first(int j) const { return (j * G + lane) * VEC - start(j); }
};

QUICKMLP_KERNEL_NAMESPACE_END

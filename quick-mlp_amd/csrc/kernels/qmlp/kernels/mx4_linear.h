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

// ------------------------------------------------------------------------------------------------ many rows
/** Bytes of codes in the tiles of grouped_linear.h. */
template <>
struct Matrix<unsigned char>
{
    typedef u32x4 Operand;
};

/** Of two operands of 32 x 64 codes: a lane has block l / 32 of row l % 32, and its scale in byte S. */
template <int S>
__device__ __forceinline__ f32x16 mx4Multiply(u32x4 a, u32x4 b, f32x16 c, unsigned scaleA, unsigned scaleB)
{
    const i32x8 wideA = __builtin_bit_cast(i32x8, __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1));
    const i32x8 wideB = __builtin_bit_cast(i32x8, __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1));
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wideA, wideB, c, 4, 4, S, scaleA, S, scaleB);
}

/**
 * The scales of a matrix' rows for two tiles of 8 blocks each: a thread takes the 16 bytes of a row at a time, its half of every tile side by side
 * for the lanes that read them.
 */
template <int TI, int TJ, int THREADS>
struct Mx4Scales
{
    static constexpr int ROWS = TI + TJ, EACH = (ROWS + THREADS - 1) / THREADS, BYTES = ROWS * 16;
    const unsigned char* p[EACH];
    u32x4 raw[EACH];
    __device__ __forceinline__ void begin(const unsigned char* a, long long strideA, int ni, const unsigned char* b, long long strideB, int nj)
    {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int row = n * THREADS + threadIdx.x;
            p[n] = row < TI ? a + min(row, ni - 1) * strideA : b + min(row - TI, nj - 1) * strideB;
        }
    }
    /** Asks for the next 16 blocks, of which 'left' are there; the others' scales are 1. */
    __device__ __forceinline__ void load(int left)
    {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            if (left >= 16) __builtin_memcpy(&raw[n], p[n], 16);
            else
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    unsigned v = 0x7f7f7f7fu;
                    if (left >= 4 * d + 4) __builtin_memcpy(&v, p[n] + 4 * d, 4);
                    else
#pragma unroll
                        for (int k = 0; k < 3; ++k)
                            if (4 * d + k < left) v = (v & ~(0xffu << (8 * k))) | static_cast<unsigned>(p[n][4 * d + k]) << (8 * k);
                    raw[n][d] = v;
                }
            p[n] += 16;
        }
    }
    __device__ __forceinline__ void write(char* lds) const
    {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int row = n * THREADS + threadIdx.x;
            const u32x4 ordered = {raw[n][0], raw[n][2], raw[n][1], raw[n][3]};
            if (row < ROWS) __builtin_memcpy(__builtin_assume_aligned(lds + row * 16, 16), &ordered, 16);
        }
    }
    /** Of the lane's row among the 32 from 'row' on: its half of two tiles. */
    static __device__ __forceinline__ u32x2 read(const char* lds, int row)
    {
        u32x2 v;
        __builtin_memcpy(&v, __builtin_assume_aligned(lds + (row + threadIdx.x % 32) * 16 + threadIdx.x % 64 / 32 * 8, 8), 8);
        return v;
    }
};

/**
 * The sums of a tile of TI x TJ by WI x WJ wavefronts, laid out as in TileProduct; tiles of 128 bytes of every row go straight to LDS, two ahead of
 * the matrix cores. Half h of the lanes takes blocks 4 h .. 4 h + 3 of a tile, one a step, so that their scales are one register.
 */
template <int TI, int TJ, int WI, int WJ>
struct Mx4Product
{
    static constexpr int THREADS = 64 * WI * WJ, NI = TI / WI / 32, NJ = TJ / WJ / 32, STEPS = 4;
    typedef unsigned char Byte;
    typedef Tile<Byte, true, TI, THREADS> TileA;
    typedef Tile<Byte, true, TJ, THREADS> TileB;
    typedef DirectTile<Byte, true, TI, THREADS> LoadsA;
    typedef DirectTile<Byte, true, TJ, THREADS> LoadsB;
    typedef Mx4Scales<TI, TJ, THREADS> Scales;
    static constexpr unsigned BYTES_A = TileA::BYTES, BYTES = BYTES_A + TileB::BYTES;

    f32x16 sums[NI][NJ];

    static __device__ __forceinline__ int firstI() { return threadIdx.x / 64 / WJ * (NI * 32); }
    static __device__ __forceinline__ int firstJ() { return threadIdx.x / 64 % WJ * (NJ * 32); }

    struct Operands
    {
        u32x4 a[NI], b[NJ];
    };
    template <int SIZE>
    static __device__ __forceinline__ u32x4 operand(const char* lds, int i, int step)
    {
        const int lane = threadIdx.x % 64;
        u32x4 v;
        __builtin_memcpy(&v, __builtin_assume_aligned(lds + Tile<Byte, true, SIZE, THREADS>::place(i + lane % 32, (lane / 32 * 4 + step) * 16), 16), 16);
        return v;
    }
    static __device__ __forceinline__ void readStep(Operands& o, const char* lds, int step)
    {
#pragma unroll
        for (int j = 0; j < NJ; ++j) o.b[j] = operand<TJ>(lds + BYTES_A, firstJ() + j * 32, step);
#pragma unroll
        for (int i = 0; i < NI; ++i) o.a[i] = operand<TI>(lds, firstI() + i * 32, step);
        __builtin_amdgcn_sched_barrier(0);   // the compiler would move the reads to where they are used
    }
    template <int S, typename Between>
    __device__ __forceinline__ void multiplyStep(const Operands& o, const unsigned (&scalesA)[NI], const unsigned (&scalesB)[NJ], Between between)
    {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                sums[i][j] = mx4Multiply<S>(o.b[j], o.a[i], sums[i][j], scalesB[j], scalesA[i]);
                between(i * NJ + j);
            }
    }

    /** LDS: two tiles of each operand, two pairs of tiles' scales. */
    __device__ __forceinline__ void run(char* lds, const Source<Byte>& a, const Source<Byte>& b, Scales& scales, int blocks)
    {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) sums[i][j] = f32x16{};
        if (blocks <= 0) return;
        LoadsA tileA;
        LoadsB tileB;
        constexpr int LOADS = LoadsA::EACH + LoadsB::EACH, PRODUCTS = NI * NJ;
        const unsigned at = static_cast<unsigned>(reinterpret_cast<unsigned long long>((__attribute__((address_space(3))) char*)lds));
        char* const scalesLds = lds + 2 * BYTES;
        int ahead = blocks, scalesAhead = blocks;   // blocks that have not been asked for
        auto askScales = [&] {
            if (scalesAhead > 0) scales.load(scalesAhead);
            scalesAhead -= 16;
        };
        askScales();
        tileA.begin(a);
        tileB.begin(b);
        auto ask = [&](unsigned buffer) {
            const int ks = min(ahead, 8);
            ahead -= ks;
            tileA.next(at + buffer, ks * 16);
            tileB.next(at + buffer + BYTES_A, ks * 16);
        };
        auto load = [&](int from, int to) {
#pragma unroll
            for (int n = from; n < to; ++n) {
                if (n < LoadsA::EACH) tileA.load(n);
                else tileB.load(n - LoadsA::EACH);
            }
        };
        ask(0);
        load(0, LOADS);
        scales.write(scalesLds);
        askScales();
        if (ahead > 0) {
            ask(BYTES);
            load(0, LOADS);
        }
        waitForTiles<0>();
        Operands operands[2];   // of a step and of the one behind it
        u32x2 pairsA[NI], pairsB[NJ];
        auto readScales = [&](unsigned from) {
#pragma unroll
            for (int i = 0; i < NI; ++i) pairsA[i] = Scales::read(scalesLds + from, firstI() + i * 32);
#pragma unroll
            for (int j = 0; j < NJ; ++j) pairsB[j] = Scales::read(scalesLds + from, TI + firstJ() + j * 32);
        };
        readScales(0);
        readStep(operands[0], lds, 0);
        const auto nothing = [](int) {};
        unsigned buffer = 0, pair = 0;   // (where the tile and the scales of its pair lie)
        bool second = false;             // of a pair
        for (int k = 0; k < blocks; k += 8) {
            unsigned scalesA[NI], scalesB[NJ];
#pragma unroll
            for (int i = 0; i < NI; ++i) scalesA[i] = second ? pairsA[i][1] : pairsA[i][0];
#pragma unroll
            for (int j = 0; j < NJ; ++j) scalesB[j] = second ? pairsB[j][1] : pairsB[j][0];
            readStep(operands[1], lds + buffer, 1);
            multiplyStep<0>(operands[0], scalesA, scalesB, nothing);
            __builtin_amdgcn_sched_barrier(0);
            readStep(operands[0], lds + buffer, 2);
            multiplyStep<1>(operands[1], scalesA, scalesB, nothing);
            __builtin_amdgcn_sched_barrier(0);
            readStep(operands[1], lds + buffer, 3);
            multiplyStep<2>(operands[0], scalesA, scalesB, nothing);
            __builtin_amdgcn_sched_barrier(0);
            const bool more = ahead > 0, last = k + 8 >= blocks;
            if (!last) {
                if (more) ask(buffer);
                buffer ^= BYTES;
                waitForTiles<0>();
            }
            // Behind the barrier the matrix cores go on at once; what else there is to do stands between the products. The scales of a pair are
            // asked for two barriers before it begins, written to LDS behind the first of them and read behind the second. (The compiler, which
            // does not know of the loads to LDS, waits for all loads when it waits for these: none are under way where they are written.)
            multiplyStep<3>(operands[1], scalesA, scalesB, [&](int n) {
                if (n == 0 && !last) {
                    readStep(operands[0], lds + buffer, 0);
                    if (second) {
                        pair ^= Scales::BYTES;
                        readScales(pair);
                        askScales();
                    } else if (k + 16 < blocks)
                        scales.write(scalesLds + (pair ^ Scales::BYTES));
                }
                if (more) load(n * LOADS / PRODUCTS, (n + 1) * LOADS / PRODUCTS);
                __builtin_amdgcn_sched_barrier(0);
            });
            second = !second;
        }
    }
};

/** Workgroups: places of tiles x tiles of J. */
template <typename T, int TI, int TJ, int WI, int WJ>
__global__ void __launch_bounds__(64 * WI * WJ)
Mx4TilesKernel(const unsigned char* __restrict__ x, const unsigned char* __restrict__ scalesX, long long strideX, long long strideScalesX, Mx4Matrix weights,
               const T* __restrict__ bias, long long strideBias, const int* __restrict__ offsets, int experts, T* __restrict__ y, long long strideY, int rows,
               int J, int blocks, int places, int tilesJ)
{
    typedef Mx4Product<TI, TJ, WI, WJ> Product;
    extern __shared__ __attribute__((aligned(16))) char groupedLds[];
    const Work work = workOf(blockIdx.x, places, tilesJ);
    const ExpertTile at = mx4Tile(offsets, experts, rows, TI, work.place);
    if (at.to <= at.from) return;
    const int j0 = work.tile * TJ;
    const int ni = at.to - at.from, nj = min(J - j0, TJ);
    const bool none = at.expert >= experts;
    const long long expert = none ? 0 : at.expert;
    Product product;
    const Source<unsigned char> a = {x + at.from * strideX, strideX, ni, rows - at.from};
    const Source<unsigned char> b = {weights.codes + expert * weights.codesExpert + j0 * weights.codesRow, weights.codesRow, nj, J - j0};
    typename Product::Scales scales;
    scales.begin(scalesX + at.from * strideScalesX, strideScalesX, ni, weights.scales + expert * weights.scalesExpert + j0 * weights.scalesRow,
                 weights.scalesRow, nj);
    product.run(groupedLds, a, b, scales, none ? 0 : blocks);
    storeTile(product, groupedLds, bias && !none ? bias + expert * strideBias + j0 : nullptr, y + at.from * strideY + j0, strideY, ni, nj);
}

// ------------------------------------------------------------------------------------------------ few rows
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

#pragma once
// The linear layer of every expert on its own rows, with rows and weights of 4 bits (mx4.h):
//
//   y[r] = W[e] x[r] + b[e]  for the rows r of expert e: offsets[e] <= r < offsets[e + 1];  zero for rows behind the last expert's
//
// The matrix cores multiply blocks of 32 codes with their scales: an operand has a block of a row in each lane, 16 bytes and a byte of scale, as
// they lie in memory. Sums are held in floats.
//
// What bounds them. Few rows: the weights that are read, 2.2 MB for every expert that has rows of 1024 -> 4096, bfloat16: 3.8 us for one expert, 6.6 for
// 8, 11.4 for 17, 14.7 for 23 (4.6 TB/s behind the 3.3 that a launch, the offsets and the first loads take). Many rows: what the
// matrix cores take from LDS, and their own rate at the clock that the power allows. 32768 rows of 16 experts, 2048 -> 4096, bfloat16: 199 us, 2.8
// PFLOP/s, behind 28 us that quantise the rows; 159 without the stores. The same tiles with 8192 inputs take 680 us, without the loads to LDS 519,
// without the reads from it 626, with the products alone, without barriers too, 448 (4.9 PFLOP/s; operands that stay the same reach 7.6), with a third
// more reads, by wavefronts of 64 x 64, 964. Tiles of K that were in the L2 already save nothing with 2048 inputs.

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
 * Moves tiles of SIZE rows of 128 bytes straight to LDS, laid out as by Tile; address and strides are multiples of 16 bytes, and rows do not
 * overlap. What is not there is zero: rows behind the last lie behind the buffer.
 */
template <int SIZE, int THREADS>
struct Mx4Loads
{
    static constexpr int TURN = THREADS / 8, EACH = SIZE / TURN;   // rows of a turn, turns
    static_assert(SIZE % TURN == 0 && TURN % 16 == 0, "a thread's pieces lie in one column, which the order of pieces in LDS does not change");
    const unsigned char* p;
    int indices;
    unsigned stride, first, turn;
    u32x4 buffer;
    unsigned to, from;

    static __device__ __forceinline__ int column()
    {
        const int row = threadIdx.x / 8;
        return (static_cast<int>(threadIdx.x) % 8 ^ (row >> 1 & 7)) * 16;
    }
    __device__ __forceinline__ void begin(const Source<unsigned char>& s)
    {
        p = s.p;
        stride = static_cast<unsigned>(s.stride);
        indices = s.indices;
        first = threadIdx.x / 8 * stride + column();
        turn = TURN * stride;
    }
    /** Turns to the tile of the next 'ks' bytes of every row, which goes to LDS from 'lds' on with the calls of load(0) to load(EACH - 1). */
    __device__ __forceinline__ void next(unsigned lds, int ks)
    {
        buffer = bufferAt(p, (indices - 1) * stride + ks);
        to = __builtin_amdgcn_readfirstlane(lds + threadIdx.x / 64 * 1024);
        from = column() < ks ? first : 0x80000000u;
        p += 128;
    }
    __device__ __forceinline__ void load(int n) const { loadToLds(buffer, from + n * turn, to + n * THREADS * 16); }
};

/**
 * The scales of a matrix' rows for two tiles of 8 blocks each: a thread takes the 16 bytes of a row at a time, its half of every tile side by side
 * for the lanes that read them. Scales behind the last block are 1.
 */
template <int TI, int TJ, int THREADS>
struct Mx4Scales
{
    static constexpr int ROWS = TI + TJ, EACH = (ROWS + THREADS - 1) / THREADS, BYTES = ROWS * 16;
    static constexpr unsigned ONES = 0x7f7f7f7fu;
    const unsigned char* p[EACH];
    u32x4 raw[EACH];
    int blocks, next, away;   // the first block that has not been asked for; bytes before the first one asked for
    /** Asks for the first pair. */
    __device__ __forceinline__ void begin(const unsigned char* a, long long strideA, int ni, const unsigned char* b, long long strideB, int nj, int blocks_)
    {
        blocks = blocks_;
        next = away = 0;
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int row = n * THREADS + threadIdx.x;
            p[n] = row < TI ? a + min(row, ni - 1) * strideA : b + min(row - TI, nj - 1) * strideB;
        }
        if (blocks >= 16) {
            ask();
            return;
        }
        next = 16;
#pragma unroll
        for (int n = 0; n < EACH; ++n)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                unsigned v = ONES;
                if (blocks >= 4 * d + 4) __builtin_memcpy(&v, p[n] + 4 * d, 4);
                else
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        if (4 * d + k < blocks) v = (v & ~(0xffu << (8 * k))) | static_cast<unsigned>(p[n][4 * d + k]) << (8 * k);
                raw[n][d] = v;
            }
    }
    /** Asks for the next pair, if there is one; for the last one with blocks before it. */
    __device__ __forceinline__ void ask()
    {
        if (next >= blocks) return;
        const int from = min(next, blocks - 16);
        away = next - from;
        next += 16;
#pragma unroll
        for (int n = 0; n < EACH; ++n) __builtin_memcpy(&raw[n], p[n] + from, 16);
    }
    __device__ __forceinline__ void write(char* lds) const
    {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int row = n * THREADS + threadIdx.x;
            unsigned v[4] = {raw[n][0], raw[n][1], raw[n][2], raw[n][3]};
#pragma unroll
            for (int d = 0; d < 4; ++d) v[d] = away & 8 ? (d < 2 ? v[d + 2] : ONES) : v[d];
#pragma unroll
            for (int d = 0; d < 4; ++d) v[d] = away & 4 ? (d < 3 ? v[d + 1] : ONES) : v[d];
#pragma unroll
            for (int d = 0; d < 4; ++d) v[d] = __builtin_amdgcn_alignbyte(d < 3 ? v[d + 1] : ONES, v[d], away & 3);
            const u32x4 ordered = {v[0], v[2], v[1], v[3]};
            if (ROWS >= (n + 1) * THREADS || row < ROWS) __builtin_memcpy(__builtin_assume_aligned(lds + row * 16, 16), &ordered, 16);
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

/** Which tile of a pair. */
template <int W>
struct Mx4Which
{
    static constexpr int value = W;
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
    typedef Mx4Loads<TI, THREADS> LoadsA;
    typedef Mx4Loads<TJ, THREADS> LoadsB;
    typedef Mx4Scales<TI, TJ, THREADS> Scales;
    static constexpr unsigned BYTES_A = TileA::BYTES, BYTES = BYTES_A + TileB::BYTES;

    f32x16 sums[NI][NJ];

    static __device__ __forceinline__ int firstI() { return threadIdx.x / 64 / WJ * (NI * 32); }
    static __device__ __forceinline__ int firstJ() { return threadIdx.x / 64 % WJ * (NJ * 32); }

    struct Operands
    {
        u32x4 a[NI], b[NJ];
    };
    /**
     * Where in LDS the lane finds its pieces of every step of a tile, for the first 32 rows of each operand; those of the next 32 lie 4096 bytes
     * behind (Tile::place() orders pieces by 16 rows), which needs no register.
     */
    struct Places
    {
        unsigned a[STEPS], b[STEPS];
        __device__ __forceinline__ void begin(unsigned lds)
        {
            const int lane = threadIdx.x % 64;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const unsigned piece = TileA::place(lane % 32, (lane / 32 * 4 + s) * 16);
                a[s] = lds + firstI() * 128 + piece;
                b[s] = lds + BYTES_A + firstJ() * 128 + piece;
            }
        }
        /** To the other tile. */
        __device__ __forceinline__ void turn(unsigned by)
        {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                a[s] += by;
                b[s] += by;
                // (otherwise the compiler keeps a register for each of their reads)
                asm volatile("" : "+v"(a[s]), "+v"(b[s]));
            }
        }
    };
    static __device__ __forceinline__ u32x4 pieceAt(unsigned place) { return *(const __attribute__((address_space(3))) u32x4*)(place); }
    static __device__ __forceinline__ void readStep(Operands& o, const Places& places, int step)
    {
#pragma unroll
        for (int j = 0; j < NJ; ++j) o.b[j] = pieceAt(places.b[step] + j * 4096);
#pragma unroll
        for (int i = 0; i < NI; ++i) o.a[i] = pieceAt(places.a[step] + i * 4096);
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
                asm volatile("" : "+v"(sums[i][j]));   // here and not behind the next barrier
                between(i * NJ + j);
            }
    }

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) sums[i][j] = f32x16{};
    }
    /** LDS: two tiles of each operand, two pairs of tiles' scales. blocks > 0. */
    __device__ __forceinline__ void run(char* lds, const Source<Byte>& a, const Source<Byte>& b, Scales& scales, int blocks)
    {
        LoadsA tileA;
        LoadsB tileB;
        constexpr int LOADS = LoadsA::EACH + LoadsB::EACH, PRODUCTS = NI * NJ;
        const unsigned at = static_cast<unsigned>(reinterpret_cast<unsigned long long>((__attribute__((address_space(3))) char*)lds));
        char* const scalesLds = lds + 2 * BYTES;
        int ahead = blocks;   // blocks that have not been asked for
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
        scales.ask();
        ask(BYTES);
        load(0, LOADS);
        waitForTiles<0>();
        Operands operands[2];   // of a step and of the one behind it
        u32x2 pairsA[NI], pairsB[NJ];
        auto readScales = [&](unsigned from) {
#pragma unroll
            for (int i = 0; i < NI; ++i) pairsA[i] = Scales::read(scalesLds + from, firstI() + i * 32);
#pragma unroll
            for (int j = 0; j < NJ; ++j) pairsB[j] = Scales::read(scalesLds + from, TI + firstJ() + j * 32);
        };
        clear();
        readScales(0);
        Places places;
        places.begin(at);
        readStep(operands[0], places, 0);
        const auto nothing = [](int) {};
        unsigned pair = 0;   // (where the scales lie)
        // All tiles go through the same code, without a branch that products would wait for: behind the last one lie tiles of zeros, which are not
        // read from memory.
        auto tile = [&](auto which) {
            constexpr int W = decltype(which)::value;
            unsigned scalesA[NI], scalesB[NJ];
#pragma unroll
            for (int i = 0; i < NI; ++i) scalesA[i] = pairsA[i][W];
#pragma unroll
            for (int j = 0; j < NJ; ++j) scalesB[j] = pairsB[j][W];
            readStep(operands[1], places, 1);
            multiplyStep<0>(operands[0], scalesA, scalesB, nothing);
            __builtin_amdgcn_sched_barrier(0);
            readStep(operands[0], places, 2);
            multiplyStep<1>(operands[1], scalesA, scalesB, nothing);
            __builtin_amdgcn_sched_barrier(0);
            readStep(operands[1], places, 3);
            multiplyStep<2>(operands[0], scalesA, scalesB, nothing);
            __builtin_amdgcn_sched_barrier(0);
            ask(W == 0 ? 0 : BYTES);
            places.turn(W == 0 ? BYTES : 0u - BYTES);
            waitForTiles<0>();
            // Behind the barrier the matrix cores go on at once; what else there is to do stands between the products. The scales of a pair are
            // asked for two barriers before it begins, written to LDS behind the first of them and read behind the second. (The compiler, which
            // does not know of the loads to LDS, waits for all loads when it waits for these: none are under way where they are written.)
            multiplyStep<3>(operands[1], scalesA, scalesB, [&](int n) {
                if (n == 0) {
                    readStep(operands[0], places, 0);
                    if constexpr (W == 0) scales.write(scalesLds + (pair ^ Scales::BYTES));
                }
                load(n * LOADS / PRODUCTS, (n + 1) * LOADS / PRODUCTS);
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (W == 1) {
                pair ^= Scales::BYTES;
                readScales(pair);
                scales.ask();
            }
        };
        for (int k = 0;;) {
            tile(Mx4Which<0>{});
            if ((k += 8) >= blocks) break;
            tile(Mx4Which<1>{});
            if ((k += 8) >= blocks) break;
        }
        waitForTiles<0>();
    }
};

/**
 * As storeTile(), for few steps of K behind which there is little else to do: of a whole tile eight pieces a lane are on their way at a time.
 */
template <typename Product, typename T>
__device__ __forceinline__ void mx4Store(const Product& product, char* lds, const T* __restrict__ bias, T* __restrict__ to, long long stride, int ni, int nj)
{
    constexpr int NI = Product::NI, NJ = Product::NJ, ROW = NJ * 32, PIECE = WIDE<T>, PIECES = ROW / PIECE, MASK = PIECES < 8 ? PIECES - 1 : 7;
    constexpr int TURNS = NI * 32 * PIECES / 64, BATCH = TURNS < 8 ? TURNS : 8, TURN = 64 / PIECES;   // rows of a turn
    const int lane = threadIdx.x % 64;
    const int fromI = Product::firstI(), fromJ = Product::firstJ();
    T* const part = reinterpret_cast<T*>(lds) + threadIdx.x / 64 * (NI * 32 * ROW);
    __syncthreads();   // the last tiles have been read
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        float b[16] = {};
        if (bias)
#pragma unroll
            for (int n = 0; n < 16; ++n) b[n] = static_cast<float>(bias[min(fromJ + j * 32 + n / 4 * 8 + lane / 32 * 4 + n % 4, nj - 1)]);   // (columns behind: any)
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int n = 0; n < 16; n += 4) {
                const int row = i * 32 + lane % 32, column = j * 32 + n * 2 + lane / 32 * 4;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = product.sums[i][j][n + k] + b[n + k];
                // (a row's pieces in an order that depends on the row, for the banks)
                T* at = part + row * ROW + ((column / PIECE ^ (row & MASK)) * PIECE + column % PIECE);
                storeFloats(static_cast<T*>(__builtin_assume_aligned(at, 4 * sizeof(T))), v);
            }
    }
    waveLdsSync();
    const int row = lane / PIECES, piece = lane % PIECES, j = fromJ + piece * PIECE;
    T* out = to + (fromI + row) * stride + j;
    const bool whole = ni - fromI >= NI * 32 && nj - fromJ >= ROW;   // (of the wavefront's part)
#pragma unroll 1
    for (int n = 0; n < TURNS; n += BATCH) {
        u32x4 raw[BATCH];
#pragma unroll
        for (int m = 0; m < BATCH; ++m) {
            const int r = (n + m) * TURN + row;
            __builtin_memcpy(&raw[m], __builtin_assume_aligned(part + r * ROW + (piece ^ (r & MASK)) * PIECE, 16), 16);
        }
        if (whole) {
#pragma unroll
            for (int m = 0; m < BATCH; ++m) streamPiece(out + m * TURN * stride, raw[m]);
        } else
#pragma unroll
            for (int m = 0; m < BATCH; ++m) {
                if (fromI + (n + m) * TURN + row >= ni || j >= nj) continue;
                T* const at = out + m * TURN * stride;
                if (j + PIECE <= nj) streamPiece(at, raw[m]);
                else {
                    T entries[PIECE];
                    __builtin_memcpy(entries, &raw[m], 16);
#pragma unroll
                    for (int k = 0; k < PIECE - 1; ++k)
                        if (j + k < nj) at[k] = entries[k];
                }
            }
        out += BATCH * TURN * stride;
    }
}

/** Workgroups: places of tiles x tiles of J. (Two wavefronts per SIMD at least: with all of its registers the compiler would keep the sums where each
 *  product has to fetch them from.) */
template <typename T, int TI, int TJ, int WI, int WJ>
__global__ void __launch_bounds__(64 * WI * WJ, 2)
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
    const bool none = at.expert >= experts;   // (then there may be no weights at all)
    const long long expert = none ? 0 : at.expert;
    Product product;
    if (none) product.clear();
    else {
        const Source<unsigned char> a = {x + at.from * strideX, strideX, ni, rows - at.from};
        const Source<unsigned char> b = {weights.codes + expert * weights.codesExpert + j0 * weights.codesRow, weights.codesRow, nj, J - j0};
        typename Product::Scales scales;
        scales.begin(scalesX + at.from * strideScalesX, strideScalesX, ni, weights.scales + expert * weights.scalesExpert + j0 * weights.scalesRow,
                     weights.scalesRow, nj, blocks);
        product.run(groupedLds, a, b, scales, blocks);
    }
    mx4Store(product, groupedLds, bias && !none ? bias + expert * strideBias + j0 : nullptr, y + at.from * strideY + j0, strideY, ni, nj);
}

// ------------------------------------------------------------------------------------------------ few rows
constexpr int MX4_FEW_WAVES = 4;
/** Where experts have few rows: blocks of K at a time, their steps of 4 blocks, and what a row of them takes in LDS (no two of 16 in one bank). */
constexpr int MX4_FEW_BLOCKS = 32, MX4_FEW_STEPS = MX4_FEW_BLOCKS / 4, MX4_FEW_CODES = MX4_FEW_BLOCKS * 16 + 16, MX4_FEW_SCALES = MX4_FEW_BLOCKS + 16;

/** Rows of a chunk of MX4_FEW_BLOCKS blocks from block 'first' on, in LDS: quantised, or as they are where X holds codes. Blocks behind the last: zeros. */
template <typename X>
__device__ __forceinline__ void mx4Stage(const X* __restrict__ x, const unsigned char* __restrict__ scalesX, long long strideX, long long strideScalesX, int count,
                                         int first, int blocks, int inputs, char* codesLds, char* scalesLds)
{
    constexpr bool CODES = sizeof(X) == 1;
    constexpr int LANES = CODES ? 1 : MX4_LANES;
    for (int unit = threadIdx.x / LANES; unit < count * MX4_FEW_BLOCKS; unit += 64 * MX4_FEW_WAVES / LANES) {
        const int row = unit / MX4_FEW_BLOCKS, block = unit % MX4_FEW_BLOCKS, b = first + block;
        char* const toCodes = codesLds + row * MX4_FEW_CODES + block * 16;
        char* const toScale = scalesLds + row * MX4_FEW_SCALES + block;
        if constexpr (CODES) {
            u32x4 codes = {};
            unsigned char scale = 127;
            if (b < blocks) {
                __builtin_memcpy(&codes, x + row * strideX + b * 16ll, 16);
                scale = scalesX[row * strideScalesX + b];
            }
            __builtin_memcpy(__builtin_assume_aligned(toCodes, 16), &codes, 16);
            *toScale = static_cast<char>(scale);
        } else {
            const int lane = threadIdx.x % LANES;
            float v[MX4_ENTRIES];
            mx4Load(x + row * strideX, b * MX4_BLOCK + lane * MX4_ENTRIES, inputs, v);
            unsigned scale;
            const unsigned packed = mx4Pack(v, scale);
            __builtin_memcpy(__builtin_assume_aligned(toCodes + lane * 4, 4), &packed, 4);
            if (lane == 0) *toScale = static_cast<char>(scale);
        }
    }
}

/**
 * The tile of 16 rows that begins at the given row; to <= from: there is none. So there are no more places of tiles than rows, however many experts
 * have none.
 */
__device__ __forceinline__ ExpertTile mx4TileAt(const int* __restrict__ offsets, int experts, int rows, int row)
{
    int from = 0, begin = 0, end = rows;   // of the last expert that begins at the row or before it, as in expertTile()
    const int lane = threadIdx.x % 64;
    for (int count = offsets ? experts : 0; count > 0;) {
        const int step = (count + 63) / 64, ahead = (lane + 1) * step, e = from + min(ahead, count);
        const int begins = expertBegin(offsets, e, rows);
        const int reached = __popcll(__ballot(ahead <= count && begins <= row));
        if (reached > 0) begin = __builtin_amdgcn_readlane(begins, reached - 1);
        if (reached < 64 && (reached + 1) * step <= count) end = __builtin_amdgcn_readlane(begins, reached);
        from += reached * step;
        count = min(step - 1, count - reached * step);
    }
    ExpertTile t;
    t.expert = from;
    t.index = (row - begin) / 16;
    t.from = row;
    t.to = (row - begin) % 16 == 0 ? min(end, static_cast<int>(min(row + 16ll, static_cast<long long>(rows)))) : row;
    t.expertRows = max(0, end - begin);
    return t;
}

/**
 * 16 rows by 16 outputs per wavefront, the weights straight from memory: lane l has block l / 16 of every four of output l % 16, a chunk ahead of the
 * matrix cores. WJ wavefronts take outputs of their own, WK share the chunk's steps and add up what they have. Results: lane l has outputs
 * 4 (l / 16) .. + 3 of row l % 16. X: T, or bytes of codes. byRow: places are rows, of which those work that a tile begins at.
 */
template <typename T, typename X, int WJ, int WK>
__global__ void __launch_bounds__(64 * MX4_FEW_WAVES)
Mx4FewKernel(const X* __restrict__ x, const unsigned char* __restrict__ scalesX, long long strideX, long long strideScalesX, Mx4Matrix weights,
             const T* __restrict__ bias, long long strideBias, const int* __restrict__ offsets, int experts, T* __restrict__ y, long long strideY, int rows,
             int J, int blocks, int inputs, int byRow, int tilesJ)
{
    static_assert(WJ * WK == MX4_FEW_WAVES, "wavefronts of a workgroup");
    constexpr int STEPS = MX4_FEW_STEPS / WK, ROWS = 16;
    __shared__ __attribute__((aligned(16))) char codesLds[2][ROWS * MX4_FEW_CODES];
    __shared__ __attribute__((aligned(16))) char scalesLds[2][ROWS * MX4_FEW_SCALES];
    const int place = static_cast<int>(blockIdx.x / tilesJ), tile = static_cast<int>(blockIdx.x % tilesJ);
    const ExpertTile at = byRow ? mx4TileAt(offsets, experts, rows, place) : mx4Tile(offsets, experts, rows, ROWS, place);
    if (at.to <= at.from) return;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, i = lane % 16, g = lane / 16;
    const int j0 = (tile * WJ + wave / WK) * 16, step0 = wave % WK * STEPS;
    const int count = at.to - at.from;
    f32x4 sum = {};
    if (at.expert < experts) {
        const long long output = min(j0 + i, J - 1);   // (outputs behind the last: any, not written)
        const unsigned char* const own = weights.codes + at.expert * weights.codesExpert + output * weights.codesRow;
        const unsigned char* const ownScales = weights.scales + at.expert * weights.scalesExpert + output * weights.scalesRow;
        u32x4 codes[2][STEPS];
        unsigned scales[2][STEPS];   // in the lane's byte g
        auto load = [&](int first, u32x4 (&c)[STEPS], unsigned (&s)[STEPS]) {
            const int b = first + step0 * 4;
            if (b + STEPS * 4 <= blocks) {
#pragma unroll
                for (int n = 0; n < STEPS; ++n) __builtin_memcpy(&c[n], own + (b + n * 4 + g) * 16ll, 16);
                __builtin_memcpy(s, ownScales + b, sizeof(s));
            } else
#pragma unroll
                for (int n = 0; n < STEPS; ++n) {
                    const int block = b + n * 4 + g;
                    c[n] = u32x4{};
                    s[n] = 127u << (8 * g);
                    if (block >= blocks) continue;
                    __builtin_memcpy(&c[n], own + block * 16ll, 16);
                    s[n] = static_cast<unsigned>(ownScales[block]) << (8 * g);
                }
        };
        auto stage = [&](int first, int buffer) {
            mx4Stage(x + at.from * strideX, scalesX + at.from * strideScalesX, strideX, strideScalesX, count, first, blocks, inputs, codesLds[buffer], scalesLds[buffer]);
        };
        auto multiply = [&](int buffer, const u32x4 (&c)[STEPS], const unsigned (&s)[STEPS]) {
            // (rows behind the last of the tile hold anything, and so do their results)
            const char* const rowCodes = codesLds[buffer] + i * MX4_FEW_CODES;
            const char* const rowScales = scalesLds[buffer] + i * MX4_FEW_SCALES;
#pragma unroll
            for (int n = 0; n < STEPS; ++n) {
                u32x4 other;
                unsigned otherScale;
                __builtin_memcpy(&other, __builtin_assume_aligned(rowCodes + ((step0 + n) * 4 + g) * 16, 16), 16);
                __builtin_memcpy(&otherScale, __builtin_assume_aligned(rowScales + (step0 + n) * 4, 4), 4);
                const i32x8 wideW = __builtin_bit_cast(i32x8, __builtin_shufflevector(c[n], c[n], 0, 1, 2, 3, -1, -1, -1, -1));
                const i32x8 wideX = __builtin_bit_cast(i32x8, __builtin_shufflevector(other, other, 0, 1, 2, 3, -1, -1, -1, -1));
                sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wideW, wideX, sum, 4, 4, 0, s[n] >> (8 * g), 0, otherScale >> (8 * g));
            }
        };
        load(0, codes[0], scales[0]);
        stage(0, 0);
        __syncthreads();
        for (int first = 0;; first += 2 * MX4_FEW_BLOCKS) {
            const bool second = first + MX4_FEW_BLOCKS < blocks, third = first + 2 * MX4_FEW_BLOCKS < blocks;
            if (second) load(first + MX4_FEW_BLOCKS, codes[1], scales[1]);
            multiply(0, codes[0], scales[0]);
            if (!second) break;
            stage(first + MX4_FEW_BLOCKS, 1);
            __syncthreads();
            if (third) load(first + 2 * MX4_FEW_BLOCKS, codes[0], scales[0]);
            multiply(1, codes[1], scales[1]);
            if (!third) break;
            stage(first + 2 * MX4_FEW_BLOCKS, 0);
            __syncthreads();
        }
    }
    if constexpr (WK > 1) {
        __shared__ f32x4 others[WJ][WK - 1][64];
        if (wave % WK > 0) others[wave / WK][wave % WK - 1][lane] = sum;
        __syncthreads();
        if (wave % WK > 0) return;
#pragma unroll
        for (int k = 0; k < WK - 1; ++k) sum += others[wave / WK][k][lane];
    }
    const int j = j0 + 4 * g;
    if (j >= J || i >= count) return;
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        v[k] = sum[k] + (bias && at.expert < experts ? static_cast<float>(bias[at.expert * strideBias + min(j + k, J - 1)]) : 0.0f);
    storeUpToFour(y + (at.from + i) * strideY + j, v, J - j);
}

QUICKMLP_KERNEL_NAMESPACE_END

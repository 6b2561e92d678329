#pragma once
// The linear layer of every expert on its own rows, and its adjoint.
//
//   y[r] = W[e] x[r] + b[e]  for the rows r of expert e: offsets[e] <= r < offsets[e + 1];  zero for rows behind the last expert's
//   dx[r] = W[e]^T dy[r],    dW[e] = sum over the rows of e of dy[r] x[r]^T,    db[e] = sum over the rows of e of dy[r]
//
// All three are matrix products C(i, j) = sum over k of A(i, k) B(j, k) in tiles of TI x TJ, with j the index along which the
// result is consecutive in memory. An operand is consecutive along k (x and W of the first, dy of the second) or along its own
// index (W of the second, dy and x of the third).
//
// How many rows an expert has is known on the device only. The rows of the experts are cut into tiles that begin where the
// expert does, and the places of the tiles follow without a scan: expert e has the places from e + floor(offsets[e] / TI) on,
// of which it has always enough, as floor(b / T) - floor(a / T) + 1 >= ceil((b - a) / T). A workgroup finds the expert of its
// place among the offsets, 64 at a time, and has nothing to do where the expert has fewer tiles than places.
//
// Offsets are limited to the rows there are wherever they are read: no access depends on their values.
//
// What bounds them: where experts have many rows, the bytes that a product takes from LDS (the matrix cores are busy 58 % of the cycles also
// without any loads from memory); the weights' bytes where experts have few rows; the latency of a tile's first bytes in between. Measured, us for
// y, dx and dW + db: 32768 rows of 16 experts, 2048 -> 4096, bfloat16 566, 567, 535 one after the other, each by itself (970 to 1030 TFLOP/s;
// a library's products of these sizes, every row with one matrix, in turn with them 392, 430, 508); 2^17 rows of 512 experts, 64 -> 64, half
// 11.8, 10.3, 12.2; 5003 rows of 12 experts, 333 -> 200, float 21, 21, 22 + 5; y of 24 rows of 64 experts, 1024 -> 4096, bfloat16 33 (the
// weights: 4.8 TB/s).

#include <qmlp/kernels/token_types.h>

QUICKMLP_KERNEL_NAMESPACE_BEGIN

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------------------------------------ matrix cores
typedef short s16x4 __attribute__((ext_vector_type(4)));
/** 16 lanes name 4 consecutive entries each of 4 rows of 16 entries, row by row; each gets the 4 entries of one of the columns. */
__device__ __forceinline__ s16x4 readTransposed16(const void* p)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

/** Operands of 32 x 32 matrix products: STEP consecutive values of k for two halves of the lanes, 32 rows each. */
template <typename T>
struct Matrix;
template <>
struct Matrix<f16>
{
    typedef f16x8 Operand;
    typedef f16x4 Quad;
    static __device__ __forceinline__ f32x16 multiply(Operand a, Operand b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Quad readTransposed(const f16* p)
    {
        return __builtin_bit_cast(Quad, readTransposed16(p));
    }
};
template <>
struct Matrix<bf16>
{
    typedef bf16x8 Operand;
    typedef bf16x4 Quad;
    static __device__ __forceinline__ f32x16 multiply(Operand a, Operand b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Quad readTransposed(const bf16* p)
    {
        return __builtin_bit_cast(Quad, readTransposed16(p));
    }
};
template <>
struct Matrix<float>
{
    typedef f32x4 Operand;
    // the instruction takes one k of each half of the lanes: the operands' k-th ones together
    static __device__ __forceinline__ f32x16 multiply(Operand a, Operand b, f32x16 c)
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[k], b[k], c, 0, 0, 0);
        return c;
    }
};

// ------------------------------------------------------------------------------------------------ tiles in LDS
/** Values of k in a tile: 128 bytes of a row. */
template <typename T>
constexpr int TILE_K = 128 / static_cast<int>(sizeof(T));
/** Values of k that an operand of the matrix cores takes of a tile. */
template <typename T>
constexpr int STEP_K = 2 * WIDE<T>;

/**
 * A tile of an operand in LDS: SIZE of its indices by TILE_K. ALONG_K: rows of 128 bytes, one for each index; otherwise one row for
 * each k. THREADS move it 16 bytes at a time, in EACH turns. Pieces of a row lie in an order that depends on the row, so that the
 * lanes that read the same piece of different rows find them in different banks.
 */
template <typename T, bool ALONG_K, int SIZE, int THREADS>
struct Tile
{
    static constexpr int PIECE = WIDE<T>;                                  // entries per access
    static constexpr int ROW = ALONG_K ? TILE_K<T> : SIZE;                 // entries of a row
    static constexpr int PIECES = ROW / PIECE;                             // of a row
    static constexpr int EACH = SIZE * 8 / THREADS;                        // pieces per thread
    static constexpr int BYTES = SIZE * 128;
    static_assert(SIZE * 8 % THREADS == 0, "every thread moves the same number of pieces");

    /** Place of an entry of the tile. */
    static __device__ __forceinline__ int place(int row, int column)
    {
        if constexpr (ALONG_K) return row * ROW + ((column / PIECE ^ (row >> 1 & 7)) * PIECE + column % PIECE);   // 16 rows of a piece: all 64 banks
        else if constexpr (sizeof(T) == 2) {
            // 32 entries (64 bytes) are read of each of four consecutive rows
            constexpr int UNITS = ROW / 32;
            return row * ROW + (((column / 32) ^ (row & (UNITS < 4 ? UNITS - 1 : 3))) * 32 + column % 32);
        } else
            return row * ROW + column;
    }

    /** The operand of the matrix cores for 32 indices from i on and the given step of the tile's k. */
    static __device__ __forceinline__ typename Matrix<T>::Operand operand(const T* lds, int i, int step)
    {
        const int lane = threadIdx.x % 64;
        if constexpr (ALONG_K) {
            typename Matrix<T>::Operand v;
            __builtin_memcpy(&v, __builtin_assume_aligned(lds + place(i + lane % 32, step * STEP_K<T> + lane / 32 * PIECE), 16), 16);
            return v;
        } else if constexpr (sizeof(T) == 2) {
            // of 4 rows by 16 columns that 16 lanes read, each lane gets a column
            const int row = step * STEP_K<T> + lane / 32 * PIECE + lane % 16 / 4, column = i + lane / 16 % 2 * 16 + lane % 4 * 4;
            const auto low = Matrix<T>::readTransposed(lds + place(row, column)), high = Matrix<T>::readTransposed(lds + place(row + 4, column));
            return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            typename Matrix<T>::Operand v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = lds[place(step * STEP_K<T> + lane / 32 * 4 + k, i + lane % 32)];
            return v;
        }
    }
};

/** An operand of a tile of results: at its first index and k = 0. */
template <typename T>
struct Source
{
    const T* p;
    long long stride;   // between rows
    int indices;        // that the tile of results has of it
    int rows;           // of the matrix from p on
};

/**
 * Moves the tiles of an operand of any address and size through registers; its rows are less than 2^21 entries apart. Indices that are not there hold anything, which no result
 * depends on; k that are not there are zero.
 */
template <typename T, bool ALONG_K, int SIZE, int THREADS>
struct RegisterTile
{
    typedef Tile<T, ALONG_K, SIZE, THREADS> Layout;
    static constexpr int PIECE = Layout::PIECE, PIECES = Layout::PIECES, EACH = Layout::EACH;
    // A thread's pieces lie in one column of pieces, 'TURN' rows apart.
    static constexpr int TURN = THREADS / PIECES;
    static_assert(THREADS % PIECES == 0, "a column of pieces per thread");
    const T* p;    // the next tile
    const T* at;   // the tile that is being read
    long long stride;
    unsigned first, turn;   // bytes from a tile to the thread's first piece, and from one to its next
    int indices, ks, safe, nextSafe;
    u32x4 raw[EACH];

    static __device__ __forceinline__ int row() { return threadIdx.x / PIECES; }
    static __device__ __forceinline__ int column() { return threadIdx.x % PIECES * PIECE; }
    __device__ __forceinline__ void begin(const Source<T>& s)
    {
        stride = s.stride;
        indices = s.indices;
        p = s.p;
        first = static_cast<unsigned>((row() * stride + column()) * sizeof(T));
        turn = static_cast<unsigned>(TURN * stride * sizeof(T));
        // rows whose last piece may be read as a whole: behind it begins the next row
        nextSafe = s.stride >= PIECE ? s.rows - 1 : 0;
    }
    /** Turns to the tile of the 'ks' next values of k, which the calls of load(0) to load(EACH - 1) read. */
    __device__ __forceinline__ void next(unsigned, int ks_)
    {
        ks = ks_;
        at = p;
        safe = nextSafe;
        p += ALONG_K ? TILE_K<T> : TILE_K<T> * stride;
        if (!ALONG_K) nextSafe -= TILE_K<T>;
    }
    /** (One load or none into registers that are zero before: anything more would make the compiler wait for it here.) */
    __device__ __forceinline__ void load(int n)
    {
        const int rows = ALONG_K ? indices : ks, columns = ALONG_K ? ks : indices;
        // pieces that end with their row or before it, and others that something lies behind
        const int upTo = column() + PIECE <= columns ? rows : column() < columns ? min(rows, safe) : 0;
        raw[n] = u32x4{0, 0, 0, 0};
        if (row() < upTo - n * TURN) __builtin_memcpy(&raw[n], piece(n), 16);
    }
    __device__ __forceinline__ const T* piece(int n) const
    {
        return reinterpret_cast<const T*>(reinterpret_cast<const char*>(at) + (first + n * turn));
    }
    /** Writes the tile, with what load() left to do: pieces that end behind the last column. */
    __device__ __forceinline__ void write(T* lds)
    {
        const int rows = ALONG_K ? indices : ks, columns = ALONG_K ? ks : indices;
        if (columns < Layout::ROW && column() < columns && column() + PIECE > columns) {
            constexpr int WORD = 4 / static_cast<int>(sizeof(T));   // entries of 32 bits
#pragma unroll
            for (int n = 0; n < EACH; ++n) {
                if (row() + n * TURN >= rows) continue;
                if (row() + n * TURN >= safe) {
                    const T* from = piece(n);
#pragma unroll
                    for (int k = 0; k < PIECE; ++k)
                        if (column() + k < columns) {
                            if constexpr (sizeof(T) == 2) raw[n][k / 2] |= static_cast<unsigned>(__builtin_bit_cast(unsigned short, from[k])) << (k % 2 * 16);
                            else raw[n][k] = __builtin_bit_cast(unsigned, from[k]);
                        }
                } else
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int left = columns - column() - k * WORD;
                        raw[n][k] = left >= WORD ? raw[n][k] : left > 0 ? raw[n][k] & 0xffffu : 0u;
                    }
            }
        }
#pragma unroll
        for (int n = 0; n < EACH; ++n)
            __builtin_memcpy(__builtin_assume_aligned(lds + Layout::place(row() + n * TURN, column()), 16), &raw[n], 16);
    }
};

/** A buffer descriptor for raw accesses of 'bytes' bytes at p; reads behind them give zeros. */
__device__ __forceinline__ u32x4 bufferAt(const void* p, unsigned bytes)
{
    const unsigned long long a = reinterpret_cast<unsigned long long>(p);
    return u32x4{static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(a))),
                 static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32))) & 0xffffu,
                 static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(bytes))), 0x00020000u};
}
/**
 * Every lane moves 16 bytes from its offset into the buffer to LDS, those of the wavefront side by side from 'lds' on. As a builtin the
 * compiler would wait for it in front of every later read of LDS; this way it is waited for by waitForTiles() alone. (The wait states: a
 * descriptor in scalar registers that vector instructions wrote may be read five later.)
 */
__device__ __forceinline__ void loadToLds(u32x4 buffer, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory", "m0");
}
/** The wavefront's writes to and reads of LDS are done, and so are those of the others. */
__device__ __forceinline__ void waitForLds()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
/** All but the last 'pending' of the wavefront's loads to LDS have arrived, its reads of LDS are done, and so are those of the others. */
template <int PENDING>
__device__ __forceinline__ void waitForTiles()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PENDING) : "memory");
}

/**
 * Moves the tiles of an operand straight from global memory to LDS. The address, the strides and the operand's sizes are
 * multiples of 16 bytes, and rows do not overlap. Indices that are not there hold others' values, which no result depends on;
 * k that are not there are zero.
 */
template <typename T, bool ALONG_K, int SIZE, int THREADS>
struct DirectTile
{
    typedef Tile<T, ALONG_K, SIZE, THREADS> Layout;
    static constexpr int PIECES = Layout::PIECES, EACH = Layout::EACH;
    const T* p;
    long long stride;
    int indices;
    unsigned offsets[EACH];
    int columns[EACH];   // along k: the first k of a piece

    __device__ __forceinline__ void begin(const Source<T>& s)
    {
        p = s.p;
        stride = s.stride;
        indices = s.indices;
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int piece = n * THREADS + threadIdx.x;
            const int row = piece / PIECES;
            // which piece belongs here is what Layout::place() says of the piece there: exchanging is its own inverse
            const int column = Layout::place(row, piece % PIECES * WIDE<T>) - row * Layout::ROW;
            columns[n] = column;
            // (rows behind the last index are read from the last one; columns behind it lie in the next row, or behind the buffer)
            offsets[n] = static_cast<unsigned>(((ALONG_K ? min(row, indices - 1) : row) * stride + column) * sizeof(T));
        }
    }
    u32x4 buffer;
    unsigned to;
    int ks;
    /** Turns to the tile of the 'ks' next values of k, which goes to LDS from 'lds' on with the calls of load(0) to load(EACH - 1). */
    __device__ __forceinline__ void next(unsigned lds, int ks_)
    {
        ks = ks_;
        buffer = bufferAt(p, static_cast<unsigned>(((ALONG_K ? indices - 1 : ks - 1) * stride + (ALONG_K ? ks : indices)) * sizeof(T)));
        to = __builtin_amdgcn_readfirstlane(lds + threadIdx.x / 64 * 1024);
        p += ALONG_K ? TILE_K<T> : TILE_K<T> * stride;
    }
    __device__ __forceinline__ void load(int n) const
    {
        loadToLds(buffer, !ALONG_K || columns[n] < ks ? offsets[n] : 0x80000000u, to + n * THREADS * 16);
    }
};

/** How tiles are moved. */
template <bool DIRECT, typename T, bool ALONG_K, int SIZE, int THREADS>
struct Loads
{
    typedef RegisterTile<T, ALONG_K, SIZE, THREADS> Type;
};
template <typename T, bool ALONG_K, int SIZE, int THREADS>
struct Loads<true, T, ALONG_K, SIZE, THREADS>
{
    typedef DirectTile<T, ALONG_K, SIZE, THREADS> Type;
};

/**
 * The sums of a tile of TI x TJ by WI x WJ wavefronts. In an accumulator, lane l holds C(i, j) of i = l % 32 and
 * j = 8 (n / 4) + 4 (l / 32) + n % 4 for n = 0 .. 15: four consecutive j at a time.
 *
 * Tiles are asked for two ahead of the matrix cores, DIRECT ones straight to LDS. Operands are read from LDS a step ahead, also from
 * one tile to the next: the barrier between two tiles stands before the last step of the first, whose operands every wavefront has by
 * then.
 */
template <bool DIRECT, typename T, bool A_ALONG_K, bool B_ALONG_K, int TI, int TJ, int WI, int WJ>
struct TileProduct
{
    static constexpr int THREADS = 64 * WI * WJ;
    static constexpr int NI = TI / WI / 32, NJ = TJ / WJ / 32;
    typedef Tile<T, A_ALONG_K, TI, THREADS> TileA;
    typedef Tile<T, B_ALONG_K, TJ, THREADS> TileB;

    f32x16 sums[NI][NJ];
    float sumsOfA[NI];   // over k alone, of index l % 32; lanes l and l ^ 32 have half of the k each

    static __device__ __forceinline__ int firstI() { return threadIdx.x / 64 / WJ * (NI * 32); }
    static __device__ __forceinline__ int firstJ() { return threadIdx.x / 64 % WJ * (NJ * 32); }

    /** What a wavefront multiplies in one step of a tile's k. */
    struct Operands
    {
        typename Matrix<T>::Operand a[NI], b[NJ];
    };
    static constexpr int STEPS = TILE_K<T> / STEP_K<T>;
    static __device__ __forceinline__ void readStep(Operands& o, const T* ldsA, const T* ldsB, int step)
    {
#pragma unroll
        for (int j = 0; j < NJ; ++j) o.b[j] = TileB::operand(ldsB, firstJ() + j * 32, step);
#pragma unroll
        for (int i = 0; i < NI; ++i) o.a[i] = TileA::operand(ldsA, firstI() + i * 32, step);
    }
    /** between(n): what is to be done beside the n-th product. */
    template <typename Between>
    __device__ __forceinline__ void multiplyStep(const Operands& o, bool sumA, Between between)
    {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                sums[i][j] = Matrix<T>::multiply(o.b[j], o.a[i], sums[i][j]);
                between(i * NJ + j);
            }
        if (sumA)
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int n = 0; n < WIDE<T>; ++n) sumsOfA[i] += static_cast<float>(o.a[i][n]);
    }

    /** sumA: also sums A over k. */
    __device__ __forceinline__ void run(char* lds, const Source<T>& a, const Source<T>& b, int K, bool sumA)
    {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            sumsOfA[i] = 0;
#pragma unroll
            for (int j = 0; j < NJ; ++j) sums[i][j] = f32x16{};
        }
        if (K <= 0) return;
        typedef typename Loads<DIRECT, T, A_ALONG_K, TI, THREADS>::Type LoadsA;
        typedef typename Loads<DIRECT, T, B_ALONG_K, TJ, THREADS>::Type LoadsB;
        LoadsA tileA;
        LoadsB tileB;
        tileA.begin(a);
        tileB.begin(b);
        constexpr unsigned BYTES_A = TileA::BYTES, BYTES = BYTES_A + TileB::BYTES;
        constexpr int LOADS = LoadsA::EACH + LoadsB::EACH, PRODUCTS = NI * NJ;
        const unsigned at = static_cast<unsigned>(reinterpret_cast<unsigned long long>((__attribute__((address_space(3))) char*)lds));
        int ahead = K;   // values of k that have not been asked for
        auto ask = [&](unsigned buffer) {
            const int ks = min(ahead, TILE_K<T>);   // (none left: 0)
            ahead -= ks;
            tileA.next(at + buffer, ks);
            tileB.next(at + buffer + BYTES_A, ks);
        };
        auto load = [&](int from, int to) {
#pragma unroll
            for (int n = from; n < to; ++n) {
                if (n < LoadsA::EACH) tileA.load(n);
                else tileB.load(n - LoadsA::EACH);
            }
        };
        auto write = [&](unsigned buffer) {
            if constexpr (!DIRECT) {
                tileA.write(reinterpret_cast<T*>(lds + buffer));
                tileB.write(reinterpret_cast<T*>(lds + buffer + BYTES_A));
            }
        };
        static_assert(STEPS % 2 == 0, "the operands of a tile's first step are the first ones");
        Operands operands[2];   // of a step and of the one behind it
        auto read = [&](Operands& o, unsigned buffer, int step) {
            readStep(o, reinterpret_cast<const T*>(lds + buffer), reinterpret_cast<const T*>(lds + buffer + BYTES_A), step);
            __builtin_amdgcn_sched_barrier(0);   // the compiler would move the reads to where they are used
        };
        ask(0);
        load(0, LOADS);
        write(0);
        if constexpr (DIRECT) {
            if (ahead > 0) {
                ask(BYTES);
                load(0, LOADS);
                waitForTiles<LOADS>();
            } else
                waitForTiles<0>();
        } else {
            ask(BYTES);
            load(0, LOADS);
            waitForLds();
        }
        read(operands[0], 0, 0);
        unsigned buffer = 0;
        for (int k = 0; k < K; k += TILE_K<T>) {
#pragma unroll
            for (int step = 0; step + 1 < STEPS; ++step) {
                read(operands[(step + 1) % 2], buffer, step + 1);
                multiplyStep(operands[step % 2], sumA, [](int) {});
                __builtin_amdgcn_sched_barrier(0);
            }
            // Through registers a tile of no k is asked for and written where there is none: with branches around the loads the compiler
            // would wait for each before the next.
            const bool more = !DIRECT || ahead > 0, last = k + TILE_K<T> >= K;
            if (!DIRECT || !last) {
                write(buffer ^ BYTES);   // (the next tile; the barrier before saw the last readers of the one there)
                if (more) ask(buffer);
                buffer ^= BYTES;
                if constexpr (DIRECT) waitForTiles<0>();
                else waitForLds();
            }
            // Behind the barrier the matrix cores go on at once; what else there is to do stands between the products.
            multiplyStep(operands[1], sumA, [&](int n) {
                if (n == 0 && !last) read(operands[0], buffer, 0);
                if (more) load(n * LOADS / PRODUCTS, (n + 1) * LOADS / PRODUCTS);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    }

    /** Hands every four consecutive results to put(i, j, values), with i and j counted from the tile's first ones. */
    template <typename Put>
    __device__ __forceinline__ void results(Put put) const
    {
        const int lane = threadIdx.x % 64;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int n = 0; n < 16; n += 4) {
                    float v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = sums[i][j][n + k];
                    put(firstI() + i * 32 + lane % 32, firstJ() + j * 32 + n * 2 + lane / 32 * 4, v);
                }
    }
};

/**
 * Writes a tile of results, converted to T, as whole rows: through LDS, which by then holds no operands any more. From registers a
 * lane would write 8 bytes of a row each time. bias: of the tile's first j, or null. All threads take part.
 */
template <typename Product, typename T>
__device__ __forceinline__ void storeTile(const Product& product, char* lds, const T* __restrict__ bias, T* __restrict__ to, long long stride, int ni, int nj)
{
    constexpr int NI = Product::NI, NJ = Product::NJ, ROW = NJ * 32, PIECE = WIDE<T>, PIECES = ROW / PIECE;   // of a wavefront's own part
    const int lane = threadIdx.x % 64;
    const int fromI = Product::firstI(), fromJ = Product::firstJ();
    T* const part = reinterpret_cast<T*>(lds) + threadIdx.x / 64 * (NI * 32 * ROW);
    float b[NJ][16] = {};
    if (bias)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                const int at = fromJ + j * 32 + n / 4 * 8 + lane / 32 * 4 + n % 4;
                b[j][n] = static_cast<float>(bias[min(at, nj - 1)]);   // (the columns behind are not written)
            }
    __syncthreads();   // the last tiles have been read
    // (a row's pieces in an order that depends on the row, for the banks)
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int n = 0; n < 16; n += 4) {
                const int row = i * 32 + lane % 32, column = j * 32 + n * 2 + lane / 32 * 4;
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = product.sums[i][j][n + k] + b[j][n + k];
                T* at = part + row * ROW + ((column / PIECE ^ (row & (PIECES < 8 ? PIECES - 1 : 7))) * PIECE + column % PIECE);
                storeFloats(static_cast<T*>(__builtin_assume_aligned(at, 4 * sizeof(T))), v);
            }
    waveLdsSync();
#pragma unroll 4
    for (int n = 0; n < NI * 32 * PIECES / 64; ++n) {
        const int row = (n * 64 + lane) / PIECES, piece = (n * 64 + lane) % PIECES;
        u32x4 raw;
        __builtin_memcpy(&raw, __builtin_assume_aligned(part + row * ROW + (piece ^ (row & (PIECES < 8 ? PIECES - 1 : 7))) * PIECE, 16), 16);
        const int i = fromI + row, j = fromJ + piece * PIECE;
        if (i >= ni || j >= nj) continue;
        T* out = to + i * stride + j;
        if (j + PIECE <= nj) streamPiece(out, raw);
        else {
            T entries[PIECE];
            __builtin_memcpy(entries, &raw, 16);
#pragma unroll
            for (int k = 0; k < PIECE; ++k)
                if (j + k < nj) out[k] = entries[k];
        }
    }
}

/** Up to four consecutive values, as many as are left before 'end'. */
template <typename T>
__device__ __forceinline__ void storeUpToFour(T* __restrict__ p, const float (&v)[4], int left)
{
    if (left >= 4) storeFloats(p, v);
    else
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < left) p[k] = static_cast<T>(v[k]);
}

// ------------------------------------------------------------------------------------------------ experts
/** offsets[e], never outside of the rows there are; the first expert begins at row 0. */
__device__ __forceinline__ int expertBegin(const int* __restrict__ offsets, int e, int rows)
{
    return e == 0 ? 0 : min(max(offsets[e], 0), rows);
}

struct ExpertTile
{
    int expert;       // the number of experts: rows behind the last one's
    int index;        // of the tile among the expert's
    int from, to;     // rows
    int expertRows;
};

/** What the given place has; to <= from: nothing. */
__device__ __forceinline__ ExpertTile expertTile(const int* __restrict__ offsets, int experts, int rows, int tileRows, int place)
{
    // the last e of 0 .. experts with e + floor(begin / tileRows) <= place, which the first one has: 64 of those behind it at a time
    const int lane = threadIdx.x % 64;
    int from = 0, begin = 0, end = rows;   // of expert 'from'; the end while it is the last one
    for (int count = experts; count > 0;) {
        const int step = (count + 63) / 64, ahead = (lane + 1) * step, e = from + min(ahead, count);
        const int begins = expertBegin(offsets, e, rows);
        const int reached = __popcll(__ballot(ahead <= count && e + static_cast<int>(static_cast<unsigned>(begins) / tileRows) <= place));
        if (reached > 0) begin = __builtin_amdgcn_readlane(begins, reached - 1);
        if (reached < 64 && (reached + 1) * step <= count) end = __builtin_amdgcn_readlane(begins, reached);
        from += reached * step;
        count = min(step - 1, count - reached * step);
    }
    ExpertTile t;
    t.expert = from;
    t.index = place - (from + begin / tileRows);
    const long long first = begin + static_cast<long long>(max(t.index, 0)) * tileRows;
    t.from = static_cast<int>(min(first, static_cast<long long>(rows)));
    t.to = min(end, static_cast<int>(min(first + tileRows, static_cast<long long>(rows))));
    if (t.index < 0) t.to = t.from;   // (offsets out of order)
    t.expertRows = max(0, end - begin);
    return t;
}

/**
 * Which of 'places' x 'tiles' a workgroup takes. Workgroups go to the dies in turn, each with an L2 of its own. In an order that goes
 * through the tiles for GROUP_PLACES places at a time, 32 consecutive ones are the work of one die (a workgroup for each of its
 * compute units), so that they share both operands; the next 32 are the next die's, so that all have as much to do.
 */
constexpr unsigned GROUP_PLACES = 4, DIE_UNITS = 32;
struct Work
{
    int place, tile;
};
__device__ __forceinline__ Work workOf(unsigned id, unsigned places, unsigned tiles)
{
    const unsigned total = places * tiles, round = DIES * DIE_UNITS;
    const unsigned n = id < total / round * round ? id / round * round + id % DIES * DIE_UNITS + id % round / DIES : id;
    const unsigned group = n / (GROUP_PLACES * tiles), within = n - group * (GROUP_PLACES * tiles);
    const unsigned count = min(GROUP_PLACES, places - group * GROUP_PLACES);
    return {static_cast<int>(group * GROUP_PLACES + within % count), static_cast<int>(within / count)};
}

// ------------------------------------------------------------------------------------------------ kernels
/**
 * Rows times the experts' matrices: y[r][j] = sum over k of x[r][k] B(j, k) + bias[e][j]. B_ALONG_K: weights[e][j][k] (the layer),
 * otherwise weights[e][k][j] (its adjoint). Workgroups: places of tiles x tiles of J, times slices of 'slice' of the K where those are too
 * few: then every slice leaves its floats in partial[slice][r][j], for GroupedJoinKernel.
 */
template <typename T, bool DIRECT, bool B_ALONG_K, int TI, int TJ, int WI, int WJ>
__global__ void __launch_bounds__(64 * WI * WJ)
GroupedRowsKernel(const T* __restrict__ x, long long strideX, const T* __restrict__ weights, long long strideExpert, long long strideWeights,
                  const T* __restrict__ bias, long long strideBias, const int* __restrict__ offsets, int experts, T* __restrict__ y, long long strideY,
                  int rows, int J, int K, int places, int tilesJ, int slices, int slice, float* __restrict__ partial)
{
    typedef TileProduct<DIRECT, T, true, B_ALONG_K, TI, TJ, WI, WJ> Product;
    extern __shared__ __attribute__((aligned(16))) char groupedLds[];
    const Work work = workOf(blockIdx.x / slices, places, tilesJ);
    const int s = blockIdx.x % slices, k0 = s * slice;
    const ExpertTile at = expertTile(offsets, experts, rows, TI, work.place);
    if (at.to <= at.from) return;
    const int j0 = work.tile * TJ;
    const int ni = at.to - at.from, nj = min(J - j0, TJ);
    Product product;
    const bool none = at.expert >= experts;
    const T* w = weights + (none ? 0 : at.expert) * strideExpert;
    const Source<T> a = {x + at.from * strideX + k0, strideX, ni, rows - at.from};
    const Source<T> b = {w + (B_ALONG_K ? j0 * strideWeights + k0 : k0 * strideWeights + j0), strideWeights, nj, B_ALONG_K ? J - j0 : K - k0};
    product.run(groupedLds, a, b, none ? 0 : min(slice, K - k0), false);
    const T* const biases = bias && !none && s == 0 ? bias + at.expert * strideBias + j0 : nullptr;
    if (!partial) {
        storeTile(product, groupedLds, biases, y + at.from * strideY + j0, strideY, ni, nj);
        return;
    }
    float* const out = partial + (static_cast<long long>(s) * rows + at.from) * J + j0;
    product.results([&](int i, int j, float (&v)[4]) {
        if (i >= ni || j >= nj) return;
        if (biases)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += static_cast<float>(biases[min(j + k, nj - 1)]);
        storeUpToFour(out + static_cast<long long>(i) * J + j, v, nj - j);
    });
}

/**
 * The adjoint of the weights: adjWeights[e][i][j] = sum over the rows r of e of adjY[r][i] x[r][j], and of the biases, the sums of
 * adjY (null: not wanted). Workgroups: places of 'chunk' rows x tiles of I x tiles of J. An expert with more rows than a chunk has
 * its sums per chunk in partial[place], I x J and I floats, for GroupedSumKernel.
 */
template <typename T, bool DIRECT, int TI, int TJ, int WI, int WJ>
__global__ void __launch_bounds__(64 * WI * WJ)
GroupedWeightsKernel(const T* __restrict__ adjY, long long strideAdjY, const T* __restrict__ x, long long strideX, const int* __restrict__ offsets,
                     int experts, T* __restrict__ adjWeights, T* __restrict__ adjBias, float* __restrict__ partial, int rows, int I, int J, int places,
                     int tilesI, int tilesJ, int chunk)
{
    typedef TileProduct<DIRECT, T, false, false, TI, TJ, WI, WJ> Product;
    extern __shared__ __attribute__((aligned(16))) char groupedLds[];
    const Work work = workOf(blockIdx.x % (tilesI * tilesJ), tilesI, tilesJ);   // (tiles of one place: rows of tiles for its places)
    const int place = blockIdx.x / (tilesI * tilesJ);
    const ExpertTile at = expertTile(offsets, experts, rows, chunk, place);
    if (at.expert >= experts || (at.to <= at.from && at.index != 0)) return;   // (the first place of an expert without rows writes zeros)
    const int i0 = work.place * TI, j0 = work.tile * TJ;
    const int ni = min(I - i0, TI), nj = min(J - j0, TJ);
    const bool whole = at.expertRows <= chunk;
    const bool sumA = adjBias && j0 == 0 && Product::firstJ() == 0;   // the wavefronts of the first columns
    Product product;
    const Source<T> a = {adjY + at.from * strideAdjY + i0, strideAdjY, ni, rows - at.from}, b = {x + at.from * strideX + j0, strideX, nj, rows - at.from};
    product.run(groupedLds, a, b, max(0, at.to - at.from), sumA);
    const long long size = static_cast<long long>(I) * J;
    float* sums = whole ? nullptr : partial + place * (size + I);
    if (!whole)
        product.results([&](int i, int j, float (&v)[4]) {
            if (i < ni && j < nj) storeUpToFour(sums + static_cast<long long>(i0 + i) * J + j0 + j, v, nj - j);
        });
    else if (adjWeights)
        storeTile(product, groupedLds, static_cast<const T*>(nullptr), adjWeights + at.expert * size + static_cast<long long>(i0) * J + j0, J, ni, nj);
    if (sumA)
#pragma unroll
        for (int n = 0; n < Product::NI; ++n) {
            const int i = Product::firstI() + n * 32 + threadIdx.x % 32;
            const float sum = product.sumsOfA[n] + __shfl_xor(product.sumsOfA[n], 32);
            if (threadIdx.x % 64 >= 32 || i >= ni) continue;
            if (whole) adjBias[static_cast<long long>(at.expert) * I + i0 + i] = static_cast<T>(sum);
            else sums[size + i0 + i] = sum;
        }
}

/** y = the sum over the slices of GroupedRowsKernel. */
template <typename T>
__global__ void __launch_bounds__(256)
GroupedJoinKernel(const float* __restrict__ partial, int slices, T* __restrict__ y, long long strideY, int rows, int J)
{
    const long long size = static_cast<long long>(rows) * J;
    for (long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; at < size; at += static_cast<long long>(gridDim.x) * 256) {
        float sum = 0;
#pragma unroll 4
        for (int s = 0; s < slices; ++s) sum += partial[s * size + at];
        y[at / J * strideY + at % J] = static_cast<T>(sum);
    }
}

/** Adds up the sums per chunk of the experts that have several. Workgroups: experts x pieces of 256 of their size + I sums. */
template <typename T>
__global__ void __launch_bounds__(256)
GroupedSumKernel(const float* __restrict__ partial, const int* __restrict__ offsets, T* __restrict__ adjWeights, T* __restrict__ adjBias, int rows,
                 long long size, int I, int chunk, int pieces)
{
    const int e = blockIdx.x / pieces;
    const int begin = expertBegin(offsets, e, rows), end = expertBegin(offsets, e + 1, rows);
    if (end - begin <= chunk) return;
    const long long at = static_cast<long long>(blockIdx.x % pieces) * 256 + threadIdx.x;
    if (at >= size + (adjBias ? I : 0)) return;
    const float* p = partial + static_cast<long long>(e + begin / chunk) * (size + I) + at;
    const int chunks = (end - begin + chunk - 1) / chunk;
    float sum = 0;
#pragma unroll 4
    for (int n = 0; n < chunks; ++n) sum += p[n * (size + I)];
    if (at >= size) adjBias[static_cast<long long>(e) * I + at - size] = static_cast<T>(sum);
    else if (adjWeights) adjWeights[e * size + at] = static_cast<T>(sum);
}

QUICKMLP_KERNEL_NAMESPACE_END

#include "token_calls.h"

#include <array>

QUICKMLP_NAMESPACE_BEGIN

using namespace token;

namespace {

// ------------------------------------------------------------------------------------------------ groups
// as in kernels/row_groups.h
constexpr int GROUP_SMALL_THREADS = 1024, GROUP_SMALL_ROWS = 8192, GROUP_SMALL_BITS = 8, GROUP_THREADS = 1024, GROUP_FEW_TILES = 64, GROUP_MOST_DIGITS = 4400, GROUP_PASS_BITS = 12,
              GROUP_SCAN_DIGITS = 64, GROUP_SCAN_THREADS = 1024;
/** GroupSource of kernels/row_groups.h */
struct GroupSource
{
    const void* index;
    long long stride;
    const unsigned* keys;
    const int* order;
    unsigned groups;
};

int bitsOf(unsigned v)
{
    int bits = 1;
    while (v >> bits && bits < 32) ++bits;
    return bits;
}

/** How many rows are sorted, and where what lies between the passes. */
struct GroupPlan
{
    int64_t rows;
    unsigned groups;
    int passes, digitBits, maxDigits, items;
    int64_t tiles;
    unsigned *counts = nullptr, *totals = nullptr, *keys[2] = {};
    int* order[2] = {};

    /** \param keysKept whether the caller has a place for the keys in order */
    GroupPlan(int64_t rows_, unsigned groups_, bool keysKept, Workspace& memory) : rows(rows_), groups(groups_)
    {
        const int bits = bitsOf(groups);
        const bool small = rows <= GROUP_SMALL_ROWS;
        passes = groups < GROUP_MOST_DIGITS ? 1 : divUp(bits, GROUP_PASS_BITS);
        digitBits = divUp(bits, passes);
        maxDigits = static_cast<int>(std::min<int64_t>(1ll << digitBits, static_cast<int64_t>(groups) + 1));
        // a workgroup for every compute unit: tiles of one row per thread, of four where there are as many anyway
        items = rows <= 256 * GROUP_THREADS ? 1 : 4;
        tiles = divUp<int64_t>(rows, GROUP_THREADS * items);
        if (small) return;
        counts = memory.take<unsigned>(tiles * maxDigits);
        totals = memory.take<unsigned>(maxDigits);
        // a pass writes where the one before did not; the last one where the caller wants it
        for (int i = 0; i < std::min(passes - 1, 2); ++i) {
            keys[i] = memory.take<unsigned>(rows);
            order[i] = memory.take<int>(rows);
        }
        if (passes == 2 && !keysKept) keys[1] = memory.take<unsigned>(rows);
    }
};

/** Sorts; keysOut (the groups in order), offsets and places may be null. spans, if not null, are written for small batches: true. */
bool sortByGroup(const Tensor& index, GroupPlan& plan, int* order, unsigned* keysOut, int* offsets, unsigned* spans, int* places, stream_t stream)
{
    const Tensor::Precision type = index.precision();
    const long long stride = strideOf(index, 0);
    const int bits = bitsOf(plan.groups);
    if (plan.rows <= GROUP_SMALL_ROWS) {
        const size_t lds = plan.rows * 6 + 64 + (static_cast<size_t>(GROUP_SMALL_THREADS / 64 * 4) << std::min(bits, GROUP_SMALL_BITS)) + 4;
        tokenKernel("row_groups.h", kernelKey(GROUP_SMALL, type), [&] { return str("GroupSmallKernel<", scalarName(type), ">"); })
            .call(1, GROUP_SMALL_THREADS, static_cast<unsigned>(lds), stream, index.rawPtr(), stride, static_cast<int>(plan.rows), plan.groups, bits, order,
                  keysOut, offsets, spans, places);
        return spans != nullptr;
    }
    auto arguments = [&] { return str("<", scalarName(type), ", ", plan.items, ">"); };
    GroupSource source{index.rawPtr(), stride, nullptr, nullptr, plan.groups};
    long long rows = plan.rows;
    for (int pass = 0; pass < plan.passes; ++pass) {
        const bool last = pass == plan.passes - 1;
        const int shift = pass * plan.digitBits;
        const int digitBits = std::min(plan.digitBits, bits - shift);
        const int digits = static_cast<int>(std::min<int64_t>(1ll << digitBits, static_cast<int64_t>(plan.groups >> shift) + 1));
        const unsigned mask = (1u << digitBits) - 1;
        const unsigned tiles = static_cast<unsigned>(plan.tiles);
        tokenKernel("row_groups.h", kernelKey(GROUP_COUNT, type, plan.items), [&] { return "GroupCountKernel" + arguments(); })
            .call(tiles, GROUP_THREADS, digits * 4, stream, source, rows, shift, mask, digits, plan.counts);
        const bool few = tiles <= GROUP_FEW_TILES;
        if (!few)
            tokenKernel("row_groups.h", kernelKey(GROUP_SCAN), [] { return "GroupScanKernel"; })
                .call(static_cast<unsigned>(divUp(digits, GROUP_SCAN_DIGITS)), GROUP_SCAN_THREADS, 0, stream, plan.counts, static_cast<int>(tiles), digits,
                      plan.totals);
        int* to = last ? order : plan.order[pass % 2];
        unsigned* toKeys = last ? (keysOut ? keysOut : plan.passes > 1 ? plan.keys[pass % 2] : nullptr) : plan.keys[pass % 2];
        const unsigned lds = digits * 4 + digits * 2 * (GROUP_THREADS / 64);
        tokenKernel("row_groups.h", kernelKey(GROUP_SCATTER, type, plan.items), [&] { return "GroupScatterKernel" + arguments(); })
            .call(tiles, GROUP_THREADS, lds, stream, source, rows, shift, digitBits, digits, static_cast<const unsigned*>(plan.counts),
                  few ? nullptr : static_cast<const unsigned*>(plan.totals), to, toKeys, plan.passes == 1 ? offsets : nullptr,
                  last ? places : nullptr);
        source.keys = toKeys;
        source.order = to;
    }
    if (offsets && plan.passes > 1)
        tokenKernel("row_groups.h", kernelKey(GROUP_OFFSETS), [] { return "GroupOffsetsKernel"; })
            .call(static_cast<unsigned>(divUp<int64_t>(static_cast<int64_t>(plan.groups) + 1, 256)), 256, 0, stream, source.keys, rows, plan.groups, offsets);
    return false;
}

// ------------------------------------------------------------------------------------------------ embeddings
// as in kernels/embedding.h
constexpr int EMBEDDING_THREADS = 256, EMBEDDING_BLOCK_BITS = 6, EMBEDDING_MOST_ROWS = 256;
struct EmbeddingBlocks
{
    static constexpr int SIZES = 6;
    int sizes;
    const float* sums[SIZES];
};

/** Four rows at a time where that leaves four workgroups for every compute unit. */
int embeddingRowsAtOnce(int64_t rows, int lanes) { return rows >= 4 * 4 * 256 * (EMBEDDING_THREADS / lanes) ? 4 : 1; }
/**
 * Rows of the table per workgroup of the adjoint kernel: as many as its lanes take at a time, and more where there are many workgroups, up to
 * 64; all that a workgroup can have where a launch would not take the threads otherwise.
 */
int embeddingAdjointRows(int64_t vocabulary, int lanes)
{
    const int64_t atATime = EMBEDDING_THREADS / lanes, most = isLaunch(divUp<int64_t>(vocabulary, 64), EMBEDDING_THREADS) ? 64 : EMBEDDING_MOST_ROWS;
    return static_cast<int>(std::min<int64_t>(most, roundUp(std::max<int64_t>(1, vocabulary / 2048), atATime)));
}

struct EmbeddingPlan
{
    Workspace memory;
    unsigned *keys, *spans;
    int* order;
    EmbeddingBlocks blocks = {};
    GroupPlan sort;
    EmbeddingPlan(int64_t rows, int64_t vocabulary, int channels, void* base)
        : memory{static_cast<char*>(base)}, keys(memory.take<unsigned>(rows)), spans(memory.take<unsigned>(2 * vocabulary)), order(memory.take<int>(rows)),
          sort(rows, static_cast<unsigned>(vocabulary), true, memory)
    {
        // (blocks of places whenever there is one, larger blocks where a row could have many of the smaller ones to add)
        for (int s = 0; s < EmbeddingBlocks::SIZES && rows >> (EMBEDDING_BLOCK_BITS * (s + 1)) >= (s == 0 ? 1 : 4); ++s) {
            blocks.sums[s] = memory.take<float>((rows >> (EMBEDDING_BLOCK_BITS * (s + 1))) * channels);
            blocks.sizes = s + 1;
        }
    }
};

// ------------------------------------------------------------------------------------------------ layer norm
// as in kernels/layer_norm.h
constexpr int LAYER_NORM_SUM_COLUMNS = 32, LAYER_NORM_SUM_THREADS = 1024, LAYER_NORM_LONG_THREADS = 1024;

/** Lanes that share a row, and how many entries each of them holds. */
struct LayerNormShape
{
    int lanes, entries, vec;   // lanes = 0: no workgroup holds a row
    int threads() const { return std::max(lanes, 256); }
    int rows() const { return threads() / lanes; }   // of a workgroup at a time
    std::string arguments() const { return std::to_string(vec) + ", " + std::to_string(lanes) + ", " + std::to_string(entries / vec); }
};
// 8 entries a lane for short rows, so that many lanes ask for memory; 64 lanes at first, whose sums need no LDS.
// (32 entries a lane do not fit the registers: the adjoint kernel holds seven values for each, two of them of the next row)
constexpr std::array<std::array<int, 2>, 9> LAYER_NORM_SHAPES = {
    {{8, 8}, {16, 8}, {32, 8}, {64, 8}, {64, 16}, {256, 8}, {256, 16}, {512, 16}, {1024, 16}}};

LayerNormShape layerNormShape(int channels, Tensor::Precision p)
{
    if (channels < wide(p)) return {8, 1, 1};
    for (const auto& s : LAYER_NORM_SHAPES)
        if (s[0] * s[1] >= channels) return {s[0], s[1], wide(p)};
    return {0, 0, 0};
}
std::string valueTypes(Tensor::Precision p, Tensor::Precision weights) { return std::string(scalarName(p)) + ", " + scalarName(weights); }

/** Workgroups of the adjoint kernel: each leaves a row of sums. Two per compute unit, one where a row takes all of its threads. */
unsigned layerNormAdjointWorkgroups(int64_t rows, int channels, const LayerNormShape& s)
{
    // slices of the rows, and no more of them than a launch takes with a thread for each of their sums
    if (s.lanes == 0) return workgroups(rows, std::min<int64_t>(256, ((1ll << 32) - 1) / roundUp<int64_t>(channels, 256)));
    return workgroups(divUp<int64_t>(rows, s.rows()), s.lanes == 1024 ? 256 : 512);
}

// ------------------------------------------------------------------------------------------------ grouped linear layers
struct GroupedTiles
{
    int i, j, wavesI, wavesJ;
    int threads() const { return 64 * wavesI * wavesJ; }
    /** Two tiles of each operand (one, where that is all there is of K; through registers a second one is written all the same), later the results. */
    unsigned lds(int64_t K, int entry, bool direct) const
    {
        return static_cast<unsigned>(std::max((direct && K * entry <= 128 ? 1 : 2) * 128 * (i + j), i * j * entry));
    }
    std::string arguments() const { return str(i, ", ", j, ", ", wavesI, ", ", wavesJ); }
};
constexpr GroupedTiles HUGE_TILES = {256, 256, 2, 4}, LARGE_TILES = {128, 128, 2, 2}, SMALL_TILES = {64, 64, 2, 2}, FEW_TILES = {32, 64, 1, 2};
const std::array<GroupedTiles, 4> GROUPED_TILES = {HUGE_TILES, LARGE_TILES, SMALL_TILES, FEW_TILES};

/**
 * The tiles for 'rows' of 'each' rows per expert and J results of K terms each, for values of 16 bits. A huge tile takes a compute unit
 * for itself, so that its first loads and its last stores stand alone: it pays where sums are long or where there are many of them, and
 * small ones pay where larger ones would leave compute units without work. us, huge | large | small, bfloat16, 16 or 17 experts (all of them
 * before results were stored past the L2, see streamPiece()):
 * 32768 rows, K 2048, J 4096: 610 | 670 | 958; 54272, 2240, 256: 79 | 94 | 140; 54272, 256, 2240: 142 | 139 | 192; 16384, 1024, 1024: 65 | 51 | 64;
 * 4096, 1024, 1024: 34 | 22 | 25; 16384, 4096, 64: 91 | 47 | 38; through registers 32768, 2047, 4095: 840 | 996 | 1467.
 * Single precision is bound by the matrix cores with small tiles as well (16384 rows, 4 experts, 1024, 1024: - | 365 | 343).
 * Where an expert has few rows, the weights are what is read, and half of a small tile would be empty. small | few, y and dx of 64 experts,
 * 1024 -> 4096, behind a training step's writes: 24 rows 69, 71 | 64, 48; 768 rows 141, 127 | 140, 115; 1536 rows 144, 123 | 140, 107; 2048 rows
 * 140, 133 | 161, 162.
 */
GroupedTiles rowsTiles(Tensor::Precision p, int64_t rows, int64_t experts, int64_t J, int64_t K)
{
    const int64_t each = rows / std::max<int64_t>(experts, 1);
    if (each <= 24) return FEW_TILES;
    if (p == Tensor::FLOAT) return SMALL_TILES;
    auto count = [&](const GroupedTiles& t) { return (rows / t.i + experts) * divUp<int64_t>(J, t.j); };
    if (each > 128 && J > 128 && ((K >= 1536 && count(HUGE_TILES) >= 192) || (K >= 512 && count(HUGE_TILES) >= 768))) return HUGE_TILES;
    return each > 64 && J > 64 && count(LARGE_TILES) >= 256 ? LARGE_TILES : SMALL_TILES;
}
/**
 * The tiles of the weights' gradients, experts x (I, J), whose terms, an expert's rows, may be shared out in chunks. us, huge | large | small, as above:
 * 32768 rows, I 4096, J 2048: 542 | 641 | 1001; 16384, 1024, 1024: 127 | 48 | 65; through registers, where the huge tile's registers do not
 * suffice, 32768, 4095, 2047: 1095 | 982 | 1488; float, 16384 rows of 4 experts, 1024, 1024: - | 302 | 337 (through
 * registers - | 317 | 324); 32768 of 16, 512, 2048: - | 554 | 615; 20000 of 12, 192, 320: - | 46 | 40; 16384 of 16, 64, 1024: - | 44 | 28.
 */
GroupedTiles weightsTiles(Tensor::Precision p, int64_t rows, int64_t experts, int64_t I, int64_t J, bool direct)
{
    const int64_t each = divUp(rows, experts);
    auto count = [&](const GroupedTiles& t, int64_t chunk) { return experts * divUp<int64_t>(I, t.i) * divUp<int64_t>(J, t.j) * std::max<int64_t>(1, each / chunk); };
    if (p == Tensor::FLOAT) return direct && I > 64 && J > 64 && count(LARGE_TILES, 2048) >= 256 ? LARGE_TILES : SMALL_TILES;
    if (direct && I > 128 && J > 128 && each >= 512 && count(HUGE_TILES, 2048) >= 512) return HUGE_TILES;
    return I > 64 && J > 64 && count(LARGE_TILES, 256) >= 256 ? LARGE_TILES : SMALL_TILES;
}

/** Whether tiles of the operand can go straight from global memory to LDS (DirectTile). */
bool isDirect(const Tensor& t)
{
    if (reinterpret_cast<uintptr_t>(t.rawPtr()) % 16 != 0) return false;
    const int n = t.ndim(), piece = 16 / static_cast<int>(t.bytesPerEntry());
    if (t.size(n - 1) % piece != 0) return false;
    for (int d = 0; d + 1 < n; ++d)
        if (t.size(d) > 1 && t.stride(d) % piece != 0) return false;
    // rows that do not overlap, 256 of which have 32-bit offsets
    return t.size(n - 2) <= 1 || (t.stride(n - 2) >= t.size(n - 1) && t.stride(n - 2) < (1 << 21));
}
const char* boolName(bool b) { return b ? "true" : "false"; }

/** Places of tiles (kernels/grouped_linear.h): one more than rows / tileRows for each expert and for the rows behind them. */
int64_t tilePlaces(int64_t rows, int64_t experts, int64_t tileRows) { return rows / tileRows + experts + 1; }

/**
 * Rows of a chunk of GroupedWeightsKernel: several chunks per expert where the tiles of all experts are less than two per compute unit. The rule goes by
 * their number alone, and experts just short of it pay for the second kernel and the memory between: us for dW of 2^17 rows, 64 -> 64, half, of 255,
 * 256, 511 | 512, 513, 1024 experts with as many rows each: 18, 16, 23 | 6.4, 8.3, 6.8. From there on an expert has one workgroup per tile,
 * however many rows it has: half of the rows in one of 511 | 512 experts 36 | 417.
 */
int64_t weightsChunk(int64_t rows, int64_t experts, int64_t tiles, int tile)
{
    const int64_t chunks = divUp<int64_t>(512, std::max<int64_t>(1, experts * tiles));   // per expert
    if (chunks <= 1) return std::max<int64_t>(rows, 1);
    return std::max<int64_t>(2 * tile, roundUp<int64_t>(divUp<int64_t>(rows, experts * chunks), 64));
}

struct GroupedAdjointPlan
{
    GroupedTiles tiles;
    int64_t tilesI, tilesJ, chunk, places;
    Workspace memory;
    float* partial = nullptr;
    GroupedAdjointPlan(Tensor::Precision p, int64_t rows, int64_t experts, int64_t inputs, int64_t outputs, bool direct, void* base) : memory{static_cast<char*>(base)}
    {
        tiles = weightsTiles(p, rows, experts, outputs, inputs, direct);
        tilesI = divUp<int64_t>(outputs, tiles.i);
        tilesJ = divUp<int64_t>(inputs, tiles.j);
        chunk = weightsChunk(rows, experts, tilesI * tilesJ, tiles.i);
        places = rows / chunk + experts;
        if (chunk < rows) partial = memory.take<float>(places * (outputs * inputs + outputs));
    }
};

/** Rows of an operand of the experts' products have 32-bit offsets within a tile. */
void checkRows(const Tensor& t, const char* what)
{
    const int d = t.ndim() - 2;
    CHECK_ERROR(t.size(d) <= 1 || t.stride(d) < (1 << 21), "rows of ", what, " must be less than 2^21 entries apart");
}

struct GroupedSizes
{
    int rows, experts, inputs, outputs;
};
GroupedSizes checkGrouped(const Tensor& input, const Tensor& weight, const Tensor& offsets)
{
    checkValues(input, "input", 2);
    checkValues(weight, "weight", 3);
    checkType(weight, "weight", input.precision());
    checkRows(input, "input");
    checkRows(weight, "weight");
    CHECK_ERROR(offsets.defined() && offsets.ndim() == 1, "offsets must be a tensor with 1 dimension");
    checkType(offsets, "offsets", Tensor::INT32);
    CHECK_ERROR(offsets.size(0) <= 1 || offsets.stride(0) == 1, "offsets must be contiguous");
    const GroupedSizes s{input.size(0), weight.size(0), input.size(1), weight.size(1)};
    CHECK_ERROR(s.inputs > 0 && s.outputs > 0, "experts must have inputs and outputs");
    checkSizes(weight, "weight", {s.experts, s.outputs, s.inputs});
    checkSizes(offsets, "offsets", {s.experts + 1ll});
    checkSteps("rows", s.rows);
    checkSteps("inputs", s.inputs);
    checkSteps("outputs", s.outputs);
    return s;
}

/** How GroupedRowsKernel makes (rows, J) of sums of K terms. */
struct RowsPlan
{
    GroupedTiles tiles;
    int64_t tilesJ, places;
    int slices = 1, slice;
    size_t bytes = 0;   // of memory for the slices
    RowsPlan(Tensor::Precision p, int64_t rows, int64_t experts, int64_t J, int64_t K)
        : tiles(rowsTiles(p, rows, experts, J, K)), tilesJ(divUp<int64_t>(J, tiles.j)), places(tilePlaces(rows, experts, tiles.i)), slice(static_cast<int>(K))
    {
        // Few tiles of long sums: a tile goes through 16 tiles of K or more (about 1 us each) alone on its compute unit, or, where there are few
        // rows, too little of the weights is on its way. Slices of four at least, and a second launch that adds them up.
        const bool few = tiles.i == FEW_TILES.i;
        const int64_t tileK = 128 / Tensor::BytesPerEntry[p], steps = divUp(K, tileK);
        const int64_t count = (rows / tiles.i + std::min(experts, rows)) * tilesJ;
        if (steps < 16 || count >= (few ? 768 : 256) || count == 0) return;
        const int64_t wanted = std::min<int64_t>({divUp<int64_t>(few ? 1536 : 512, count), steps / 4, 32});
        slice = static_cast<int>(divUp(steps, wanted) * tileK);
        slices = static_cast<int>(divUp<int64_t>(K, slice));
        if (slices > 1) bytes = roundUp<size_t>(sizeof(float) * slices * rows * J, ALIGNMENT);
    }
};
/** Memory for any type. */
size_t rowsMemory(int64_t rows, int64_t experts, int64_t J, int64_t K)
{
    return std::max(RowsPlan(Tensor::FLOAT, rows, experts, J, K).bytes, RowsPlan(Tensor::HALF, rows, experts, J, K).bytes);
}

/** y (rows, J) from x (rows, K) and the weights along K (the layer) or across it (its adjoint). */
void launchRows(bool alongK, const Tensor& x, const Tensor& weight, const Tensor& offsets, const Tensor& bias, const Tensor& y, const GroupedSizes& s,
                int J, int K, void* memory, stream_t stream)
{
    const Tensor::Precision p = x.precision();
    const bool direct = isDirect(x) && isDirect(weight);
    const RowsPlan plan(p, s.rows, s.experts, J, K);
    const GroupedTiles& t = plan.tiles;
    const int64_t groups = plan.places * plan.tilesJ * plan.slices;
    checkLaunch(groups, t.threads());
    float* partial = plan.slices > 1 ? static_cast<float*>(memory) : nullptr;
    tokenKernel("grouped_linear.h", kernelKey(GROUPED_ROWS, p * 4 + direct * 2 + alongK, t.i, t.j, t.wavesI, t.wavesJ),
                [&] { return str("GroupedRowsKernel<", scalarName(p), ", ", boolName(direct), ", ", boolName(alongK), ", ", t.arguments(), ">"); })
        .call(static_cast<unsigned>(groups), t.threads(), t.lds(plan.slice, x.bytesPerEntry(), direct), stream, x.rawPtr(), strideOf(x, 0),
              static_cast<const void*>(ptr<void>(weight)), strideOf(weight, 0), strideOf(weight, 1), static_cast<const void*>(ptr<void>(bias)),
              bias.defined() ? strideOf(bias, 0) : 0ll, static_cast<const int*>(ptr<int>(offsets)), s.experts, static_cast<void*>(ptr<void>(y)),
              strideOf(y, 0), s.rows, J, K, static_cast<int>(plan.places), static_cast<int>(plan.tilesJ), plan.slices, plan.slice, partial);
    if (partial)
        tokenKernel("grouped_linear.h", kernelKey(GROUPED_JOIN, p), [&] { return str("GroupedJoinKernel<", scalarName(p), ">"); })
            .call(workgroups(divUp<int64_t>(static_cast<int64_t>(s.rows) * J, 256), 4096), 256, 0, stream, static_cast<const float*>(partial), plan.slices,
                  static_cast<void*>(ptr<void>(y)), strideOf(y, 0), s.rows, J);
}

} // namespace

// ------------------------------------------------------------------------------------------------ entry points
size_t Tokens::groupMemory(int64_t rows, int groups)
{
    CHECK_ERROR(rows >= 0 && rows < (1ll << 31) && groups >= 0, "rows and groups must not be negative and fit into 32 bits");
    Workspace memory{nullptr};
    GroupPlan plan(rows, static_cast<unsigned>(groups), false, memory);
    return memory.bytes;
}

void Tokens::group(const Tensor& index, int groups, Tensor& order, Tensor& offsets, void* memory, stream_t stream)
{
    Tensor places;
    group(index, groups, order, offsets, places, memory, stream);
}

void Tokens::group(const Tensor& index, int groups, Tensor& order, Tensor& offsets, Tensor& places, void* memory, stream_t stream)
{
    checkIndex(index, "index");
    CHECK_ERROR(groups >= 0, "the number of groups must not be negative");
    for (const auto& [t, what, size] : {std::tuple<const Tensor&, const char*, int64_t>{order, "order", index.size(0)}, {offsets, "offsets", groups + 1ll},
                                        {places, "places", index.size(0)}}) {
        if (&t == &places && !t.defined()) continue;
        CHECK_ERROR(t.defined() && t.ndim() == 1, what, " must be a tensor with 1 dimension");
        checkType(t, what, Tensor::INT32);
        checkSizes(t, what, {size});
        checkContiguous(t, what);
    }
    checkMemory(memory, groupMemory(index.size(0), groups));
    Workspace workspace{static_cast<char*>(memory)};
    GroupPlan plan(index.size(0), static_cast<unsigned>(groups), false, workspace);
    sortByGroup(index, plan, ptr<int>(order), nullptr, ptr<int>(offsets), nullptr, ptr<int>(places), stream);
}

void Tokens::embedding(const Tensor& index, const Tensor& table, float scale, Tensor& output, stream_t stream)
{
    checkIndex(index, "index");
    checkValues(table, "table", 2);
    checkValues(output, "output", 2);
    checkType(output, "output", table.precision());
    checkSizes(output, "output", {index.size(0), table.size(1)});
    checkOutput(output, "output");
    checkSteps("channels", table.size(1));
    if (output.numel() == 0) return;
    const int C = table.size(1), vec = C < wide(table.precision()) ? 1 : wide(table.precision()), lanes = lanesPerRow(C, vec);
    const long long rows = index.size(0), vocabulary = table.size(0);
    const int atOnce = embeddingRowsAtOnce(rows, lanes), each = EMBEDDING_THREADS / lanes * atOnce;
    const Tensor::Precision p = table.precision(), i = index.precision();
    tokenKernel("embedding.h", kernelKey(EMBEDDING, p, i, vec, lanes, atOnce),
                [&] { return str("EmbeddingKernel<", scalarName(p), ", ", scalarName(i), ", ", vec, ", ", lanes, ", ", atOnce, ">"); })
        .call(workgroups(divUp<int64_t>(rows, each), 1 << 20), EMBEDDING_THREADS, 0, stream, index.rawPtr(), strideOf(index, 0),
              static_cast<const void*>(ptr<void>(table)), strideOf(table, 0), scale, output.rawPtr(), strideOf(output, 0), rows, vocabulary, C);
}

size_t Tokens::embeddingAdjointMemory(int64_t rows, int64_t vocabulary, int channels)
{
    CHECK_ERROR(rows >= 0 && rows < (1ll << 31) && vocabulary >= 0 && vocabulary < (1ll << 31) && channels >= 0,
                "rows, vocabulary and channels must not be negative and fit into 32 bits");
    return EmbeddingPlan(rows, vocabulary, channels, nullptr).memory.bytes;
}

void Tokens::embeddingAdjoint(const Tensor& index, const Tensor& adjOutput, float scale, Tensor& adjTable, void* memory, stream_t stream)
{
    checkIndex(index, "index");
    checkValues(adjTable, "adjTable", 2);
    checkOutput(adjTable, "adjTable");
    checkValues(adjOutput, "adjOutput", 2);
    checkType(adjOutput, "adjOutput", adjTable.precision());
    checkSizes(adjOutput, "adjOutput", {index.size(0), adjTable.size(1)});
    checkSteps("channels", adjTable.size(1));
    const long long rows = index.size(0), vocabulary = adjTable.size(0);
    const int C = adjTable.size(1);
    checkMemory(memory, embeddingAdjointMemory(rows, vocabulary, C));
    if (adjTable.numel() == 0) return;
    const Tensor::Precision p = adjTable.precision();
    const int vec = C < wide(p) ? 1 : wide(p), lanes = lanesPerRow(C, vec);
    checkLaunch(divUp<int64_t>(divUp<int64_t>(rows, 1 << EMBEDDING_BLOCK_BITS), EMBEDDING_THREADS / lanes), EMBEDDING_THREADS);   // (the first blocks)
    auto arguments = [&] { return str("<", scalarName(p), ", ", vec, ", ", lanes); };
    EmbeddingPlan plan(rows, vocabulary, C, memory);
    const void* dy = ptr<void>(adjOutput);
    if (rows > 0) {
        const bool marked = sortByGroup(index, plan.sort, plan.order, plan.keys, nullptr, plan.spans, nullptr, stream);
        for (int s = 0; s < plan.blocks.sizes; ++s) {
            // (the first kernel looks at every place for the spans)
            const int64_t blocks = s == 0 && !marked ? divUp<int64_t>(rows, 1 << EMBEDDING_BLOCK_BITS) : rows >> (EMBEDDING_BLOCK_BITS * (s + 1));
            tokenKernel("embedding.h", kernelKey(EMBEDDING_BLOCKS, p, vec, lanes, s == 0),
                        [&] { return "EmbeddingBlocksKernel" + arguments() + (s == 0 ? ", true>" : ", false>"); })
                .call(static_cast<unsigned>(divUp<int64_t>(blocks, EMBEDDING_THREADS / lanes)), EMBEDDING_THREADS, 0, stream,
                      static_cast<const unsigned*>(plan.keys), static_cast<const int*>(plan.order), rows, static_cast<unsigned>(vocabulary),
                      EMBEDDING_BLOCK_BITS * (s + 1), dy, strideOf(adjOutput, 0), s == 0 ? nullptr : plan.blocks.sums[s - 1],
                      const_cast<float*>(plan.blocks.sums[s]), C, marked ? nullptr : plan.spans);
        }
    }
    const int each = embeddingAdjointRows(vocabulary, lanes);
    tokenKernel("embedding.h", kernelKey(EMBEDDING_ADJOINT, p, vec, lanes), [&] { return "EmbeddingAdjointKernel" + arguments() + ">"; })
        .call(static_cast<unsigned>(divUp<int64_t>(vocabulary, each)), EMBEDDING_THREADS, 0, stream, static_cast<const unsigned*>(plan.keys), static_cast<const unsigned*>(plan.spans), static_cast<const int*>(plan.order), rows, plan.blocks, dy, strideOf(adjOutput, 0), scale,
              adjTable.rawPtr(), strideOf(adjTable, 0), vocabulary, C);
}

void Tokens::layerNorm(const Tensor& input, const Tensor& weight, const Tensor& bias, float epsilon, Tensor& output, Tensor& mean, Tensor& rstd,
                       stream_t stream)
{
    checkValues(input, "input", 2);
    const long long rows = input.size(0);
    const int C = input.size(1);
    checkSteps("channels", C);
    const Tensor::Precision p = input.precision(), weights = weight.defined() ? weight.precision() : bias.defined() ? bias.precision() : p;
    for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{weight, "weight"}, {bias, "bias"}}) {
        if (!t.defined()) continue;
        checkValues(t, what, 1);
        checkSizes(t, what, {C});
        CHECK_ERROR(t.precision() == p || t.precision() == Tensor::FLOAT, what, " must be of the input's type or FLOAT");
        CHECK_ERROR(t.precision() == weights, "weight and bias must be of one type");
    }
    checkValues(output, "output", 2);
    checkType(output, "output", p);
    checkSizes(output, "output", {rows, C});
    checkOutput(output, "output");
    for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{mean, "mean"}, {rstd, "rstd"}}) {
        if (!t.defined()) continue;
        checkValues(t, what, 1);
        checkType(t, what, Tensor::FLOAT);
        checkSizes(t, what, {rows});
    }
    if (input.numel() == 0) return;
    const LayerNormShape s = layerNormShape(C, p);
    auto types = [&] { return "<" + valueTypes(p, weights); };
    const void *x = input.rawPtr(), *w = ptr<void>(weight), *b = ptr<void>(bias);
    const long long strideX = strideOf(input, 0), strideY = strideOf(output, 0);
    const bool isLong = s.lanes == 0;
    tokenKernel("layer_norm.h", isLong ? kernelKey(LAYER_NORM_LONG, p, weights) : kernelKey(LAYER_NORM, p, weights, s.vec, s.lanes, s.entries),
                [&] { return isLong ? "LayerNormLongKernel" + types() + ">" : "LayerNormKernel" + types() + ", " + s.arguments() + ">"; })
        .call(isLong ? workgroups(rows, 512) : workgroups(divUp<int64_t>(rows, s.rows()), s.lanes == 1024 ? 512 : 2048),
              isLong ? LAYER_NORM_LONG_THREADS : s.threads(), 0, stream, x, strideX, w, b, epsilon, output.rawPtr(), strideY, ptr<float>(mean),
              ptr<float>(rstd), rows, C);
}

size_t Tokens::layerNormAdjointMemory(int64_t rows, int channels)
{
    CHECK_ERROR(rows >= 0 && channels >= 0, "rows and channels must not be negative");
    if (rows == 0) return 0;
    // (for any precision)
    size_t bytes = 0;
    for (const Tensor::Precision p : {Tensor::FLOAT, Tensor::HALF})
        bytes = std::max(bytes, sizeof(float) * 2 * channels * layerNormAdjointWorkgroups(rows, channels, layerNormShape(channels, p)));
    return roundUp(bytes, ALIGNMENT);
}

void Tokens::layerNormAdjoint(const Tensor& input, const Tensor& weight, const Tensor& mean, const Tensor& rstd, const Tensor& adjOutput, Tensor& adjInput,
                              Tensor& adjWeight, Tensor& adjBias, void* memory, stream_t stream)
{
    checkValues(input, "input", 2);
    const long long rows = input.size(0);
    const int C = input.size(1);
    checkSteps("channels", C);
    const Tensor::Precision p = input.precision();
    if (weight.defined()) {
        checkValues(weight, "weight", 1);
        checkSizes(weight, "weight", {C});
        CHECK_ERROR(weight.precision() == p || weight.precision() == Tensor::FLOAT, "weight must be of the input's type or FLOAT");
    }
    for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{mean, "mean"}, {rstd, "rstd"}}) {
        checkValues(t, what, 1);
        checkType(t, what, Tensor::FLOAT);
        checkSizes(t, what, {rows});
    }
    checkValues(adjOutput, "adjOutput", 2);
    checkType(adjOutput, "adjOutput", p);
    checkSizes(adjOutput, "adjOutput", {rows, C});
    if (adjInput.defined()) {
        checkValues(adjInput, "adjInput", 2);
        checkType(adjInput, "adjInput", p);
        checkSizes(adjInput, "adjInput", {rows, C});
        checkOutput(adjInput, "adjInput");
    }
    Tensor::Precision weights = weight.defined() ? weight.precision() : p;
    for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{adjWeight, "adjWeight"}, {adjBias, "adjBias"}}) {
        if (!t.defined()) continue;
        checkValues(t, what, 1);
        checkSizes(t, what, {C});
        CHECK_ERROR(t.precision() == p || t.precision() == Tensor::FLOAT, what, " must be of the input's type or FLOAT");
        if (!weight.defined()) weights = t.precision();
    }
    for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{adjWeight, "adjWeight"}, {adjBias, "adjBias"}})
        if (t.defined()) checkType(t, what, weights);
    const bool sums = adjWeight.defined() || adjBias.defined();
    if (C == 0 || (!sums && !adjInput.defined())) return;
    const size_t bytes = sums ? layerNormAdjointMemory(rows, C) : 0;
    checkMemory(memory, bytes);
    float* partial = sums ? static_cast<float*>(memory) : nullptr;
    const LayerNormShape s = layerNormShape(C, p);
    auto types = [&] { return "<" + valueTypes(p, weights); };
    int count = 0;
    if (rows > 0) {
        const unsigned groups = layerNormAdjointWorkgroups(rows, C, s);
        count = static_cast<int>(groups);
        const void *x = input.rawPtr(), *w = ptr<void>(weight), *dy = adjOutput.rawPtr();
        const float *m = ptr<float>(mean), *r = ptr<float>(rstd);
        const long long strideX = strideOf(input, 0), strideDy = strideOf(adjOutput, 0), strideDx = adjInput.defined() ? strideOf(adjInput, 0) : 0;
        void* dx = ptr<void>(adjInput);
        if (s.lanes > 0) {
            tokenKernel("layer_norm.h", kernelKey(LAYER_NORM_ADJOINT, p, weights, s.vec, s.lanes, s.entries),
                        [&] { return "LayerNormAdjointKernel" + types() + ", " + s.arguments() + ">"; })
                .call(groups, s.threads(), 0, stream, x, strideX, w, m, r, dy, strideDy, dx, strideDx, partial, rows, C);
        } else {
            if (dx)
                tokenKernel("layer_norm.h", kernelKey(LAYER_NORM_LONG_ADJOINT, p, weights), [&] { return "LayerNormLongAdjointKernel" + types() + ">"; })
                    .call(workgroups(rows, 512), LAYER_NORM_LONG_THREADS, 0, stream, x, strideX, w, m, r, dy, strideDy, dx, strideDx, rows, C);
            if (sums)
                tokenKernel("layer_norm.h", kernelKey(LAYER_NORM_LONG_SUMS, p), [&] { return str("LayerNormLongSumsKernel<", scalarName(p), ">"); })
                    .call(groups * static_cast<unsigned>(divUp(C, 256)), 256, 0, stream, x, strideX, m, r, dy, strideDy, partial, rows, C, count);
        }
    }
    if (sums)
        tokenKernel("layer_norm.h", kernelKey(LAYER_NORM_SUM, weights), [&] { return str("LayerNormSumKernel<", scalarName(weights), ">"); })
            .call(workgroups(divUp<int64_t>(2ll * C, LAYER_NORM_SUM_COLUMNS), 1 << 20), LAYER_NORM_SUM_THREADS, 0, stream, static_cast<const float*>(partial), count, C,
                  ptr<void>(adjWeight), ptr<void>(adjBias));
}

size_t Tokens::groupedLinearMemory(int64_t rows, int experts, int inputs, int outputs)
{
    CHECK_ERROR(rows >= 0 && experts >= 0 && inputs >= 0 && outputs >= 0, "sizes must not be negative");
    return rowsMemory(rows, experts, outputs, inputs);
}

void Tokens::groupedLinear(const Tensor& input, const Tensor& weight, const Tensor& offsets, const Tensor& bias, Tensor& output, void* memory,
                           stream_t stream)
{
    const GroupedSizes s = checkGrouped(input, weight, offsets);
    const Tensor::Precision p = input.precision();
    if (bias.defined()) {
        checkValues(bias, "bias", 2);
        checkType(bias, "bias", p);
        checkSizes(bias, "bias", {s.experts, s.outputs});
    }
    checkValues(output, "output", 2);
    checkType(output, "output", p);
    checkSizes(output, "output", {s.rows, s.outputs});
    checkOutput(output, "output");
    if (s.rows == 0) return;
    checkMemory(memory, groupedLinearMemory(s.rows, s.experts, s.inputs, s.outputs));
    launchRows(true, input, weight, offsets, bias, output, s, s.outputs, s.inputs, memory, stream);
}

size_t Tokens::groupedLinearAdjointMemory(int64_t rows, int experts, int inputs, int outputs)
{
    CHECK_ERROR(rows >= 0 && experts >= 0 && inputs >= 0 && outputs >= 0, "sizes must not be negative");
    // (for any type and alignment; the input's gradients are done before the weights' begin)
    size_t bytes = rowsMemory(rows, experts, inputs, outputs);
    if (experts == 0) return bytes;
    for (const Tensor::Precision p : {Tensor::FLOAT, Tensor::HALF})
        for (const bool direct : {false, true}) bytes = std::max(bytes, GroupedAdjointPlan(p, rows, experts, inputs, outputs, direct, nullptr).memory.bytes);
    return bytes;
}

void Tokens::groupedLinearAdjoint(const Tensor& input, const Tensor& weight, const Tensor& offsets, const Tensor& adjOutput, Tensor& adjInput,
                                  Tensor& adjWeight, Tensor& adjBias, void* memory, stream_t stream)
{
    const GroupedSizes s = checkGrouped(input, weight, offsets);
    const Tensor::Precision p = input.precision();
    checkValues(adjOutput, "adjOutput", 2);
    checkType(adjOutput, "adjOutput", p);
    checkSizes(adjOutput, "adjOutput", {s.rows, s.outputs});
    checkRows(adjOutput, "adjOutput");
    if (adjInput.defined()) {
        checkValues(adjInput, "adjInput", 2);
        checkType(adjInput, "adjInput", p);
        checkSizes(adjInput, "adjInput", {s.rows, s.inputs});
        checkOutput(adjInput, "adjInput");
    }
    if (adjWeight.defined()) {
        checkValues(adjWeight, "adjWeight", 3);
        checkType(adjWeight, "adjWeight", p);
        checkSizes(adjWeight, "adjWeight", {s.experts, s.outputs, s.inputs});
        checkContiguous(adjWeight, "adjWeight");
    }
    if (adjBias.defined()) {
        checkValues(adjBias, "adjBias", 2);
        checkType(adjBias, "adjBias", p);
        checkSizes(adjBias, "adjBias", {s.experts, s.outputs});
        checkContiguous(adjBias, "adjBias");
    }
    const int* off = ptr<int>(offsets);
    const void *x = ptr<void>(input), *dy = ptr<void>(adjOutput);
    const bool inputs = adjInput.defined() && s.rows > 0, weights = s.experts > 0 && (adjWeight.defined() || adjBias.defined());
    if (!inputs && !weights) return;
    checkMemory(memory, groupedLinearAdjointMemory(s.rows, s.experts, s.inputs, s.outputs));
    const bool direct = isDirect(input) && isDirect(adjOutput);
    GroupedAdjointPlan plan(p, s.rows, weights ? s.experts : 1, s.inputs, s.outputs, direct, memory);
    const int64_t groups = plan.places * plan.tilesI * plan.tilesJ;
    const long long size = static_cast<long long>(s.inputs) * s.outputs;
    const int64_t pieces = divUp<int64_t>(size + s.outputs, 256);
    if (weights) {   // (before the input's gradients are launched)
        checkLaunch(groups, plan.tiles.threads());
        checkLaunch(plan.partial ? pieces * s.experts : 0, 256);
    }
    if (inputs) launchRows(false, adjOutput, weight, offsets, {}, adjInput, s, s.inputs, s.outputs, memory, stream);
    if (!weights) return;
    const int chunk = static_cast<int>(plan.chunk);
    tokenKernel("grouped_linear.h", kernelKey(GROUPED_WEIGHTS, p * 2 + direct, plan.tiles.i, plan.tiles.j, plan.tiles.wavesI, plan.tiles.wavesJ),
                [&] { return str("GroupedWeightsKernel<", scalarName(p), ", ", boolName(direct), ", ", plan.tiles.arguments(), ">"); })
        .call(static_cast<unsigned>(groups), plan.tiles.threads(), plan.tiles.lds(s.rows, input.bytesPerEntry(), direct), stream, dy, strideOf(adjOutput, 0), x, strideOf(input, 0), off, s.experts,
              ptr<void>(adjWeight), ptr<void>(adjBias), plan.partial, s.rows, s.outputs, s.inputs,
              static_cast<int>(plan.places), static_cast<int>(plan.tilesI), static_cast<int>(plan.tilesJ), chunk);
    if (plan.partial)
        tokenKernel("grouped_linear.h", kernelKey(GROUPED_SUM, p), [&] { return str("GroupedSumKernel<", scalarName(p), ">"); })
            .call(static_cast<unsigned>(pieces * s.experts), 256, 0, stream, static_cast<const float*>(plan.partial), off, ptr<void>(adjWeight),
                  ptr<void>(adjBias), s.rows, size, s.outputs, chunk, static_cast<int>(pieces));
}

void Tokens::precompile(Tensor::Precision p)
{
    CHECK_ERROR(isValue(p), "precision must be float, half or bfloat16");
    const std::string t = scalarName(p);
    const std::vector<std::string> indices = {"int", "long long"};
    for (const auto& i : indices)
    {
        precompileKernel("row_groups.h", str("GroupSmallKernel<", i, ">"));
        for (const int items : {1, 4})
            for (const char* kernel : {"GroupCountKernel", "GroupScatterKernel"}) precompileKernel("row_groups.h", str(kernel, "<", i, ", ", items, ">"));
    }
    for (const char* kernel : {"GroupScanKernel", "GroupOffsetsKernel"}) precompileKernel("row_groups.h", kernel);
    for (const int vec : {1, wide(p)})
        for (const int lanes : {8, 16, 32, 64, 128, 256}) {
            if (vec == 1 && lanes > 8) continue;
            const std::string shape = str(t, ", ", vec, ", ", lanes);
            for (const auto& i : indices)
                for (const int atOnce : {1, 4}) precompileKernel("embedding.h", str("EmbeddingKernel<", t, ", ", i, ", ", vec, ", ", lanes, ", ", atOnce, ">"));
            precompileKernel("embedding.h", str("EmbeddingBlocksKernel<", shape, ", true>"));
            precompileKernel("embedding.h", str("EmbeddingBlocksKernel<", shape, ", false>"));
            precompileKernel("embedding.h", str("EmbeddingAdjointKernel<", shape, ">"));
        }
    std::vector<LayerNormShape> shapes = {{8, 1, 1}};
    for (const auto& s : LAYER_NORM_SHAPES) shapes.push_back({s[0], s[1], wide(p)});
    std::vector<Tensor::Precision> weights = {p};   // of a layer norm
    if (p != Tensor::FLOAT) weights.push_back(Tensor::FLOAT);
    for (const Tensor::Precision w : weights) {
        const std::string types = valueTypes(p, w);
        for (const LayerNormShape& s : shapes)
            for (const char* kernel : {"LayerNormKernel", "LayerNormAdjointKernel"}) precompileKernel("layer_norm.h", str(kernel, "<", types, ", ", s.arguments(), ">"));
        for (const char* kernel : {"LayerNormLongKernel", "LayerNormLongAdjointKernel"}) precompileKernel("layer_norm.h", str(kernel, "<", types, ">"));
        precompileKernel("layer_norm.h", str("LayerNormSumKernel<", scalarName(w), ">"));
    }
    precompileKernel("layer_norm.h", str("LayerNormLongSumsKernel<", t, ">"));
    for (const bool direct : {false, true})
        for (const GroupedTiles& tiles : GROUPED_TILES) {
            const bool few = tiles.i == FEW_TILES.i, huge = tiles.i == HUGE_TILES.i, single = p == Tensor::FLOAT;
            if (single && (huge || (tiles.i == LARGE_TILES.i && !direct))) continue;
            const std::string types = str(t, ", ", boolName(direct));
            for (const char* along : {", true, ", ", false, "})
                if (!single || tiles.i <= SMALL_TILES.i) precompileKernel("grouped_linear.h", str("GroupedRowsKernel<", types, along, tiles.arguments(), ">"));
            if (!few && (direct || !huge)) precompileKernel("grouped_linear.h", str("GroupedWeightsKernel<", types, ", ", tiles.arguments(), ">"));
        }
    for (const char* kernel : {"GroupedSumKernel", "GroupedJoinKernel"}) precompileKernel("grouped_linear.h", str(kernel, "<", t, ">"));
    precompileExperts(p);
}

QUICKMLP_NAMESPACE_END

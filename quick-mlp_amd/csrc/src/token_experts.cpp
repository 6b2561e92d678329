#include "token_calls.h"

QUICKMLP_NAMESPACE_BEGIN

using namespace token;

namespace {

// ------------------------------------------------------------------------------------------------ router
// as in kernels/route.h
constexpr int ROUTE_THREADS = 256, ROUTE_MOST_CHOSEN = 64;

/** Lanes that share a row, and how many logits each of them holds; none of them: more than a wavefront holds. */
struct RouteShape
{
    int lanes, entries;
    int rows() const { return ROUTE_THREADS / lanes; }
    std::string arguments(Tensor::Precision p) const { return str("<", scalarName(p), ", ", lanes, ", ", entries, ">"); }
};
constexpr RouteShape ROUTE_SHAPES[] = {{8, 4}, {8, 8}, {16, 8}, {32, 8}, {64, 8}, {64, 16}};
RouteShape routeShape(int experts)
{
    for (const RouteShape& s : ROUTE_SHAPES)
        if (s.lanes * s.entries >= experts) return s;
    return {0, 0};
}

struct RouteSizes
{
    long long rows;
    int experts, chosen;
};
RouteSizes checkRoute(const Tensor& logits, const Tensor& weights, const char* what, const Tensor& index)
{
    checkValues(logits, "logits", 2);
    checkValues(weights, what, 2);
    checkType(weights, what, logits.precision());
    CHECK_ERROR(index.defined() && index.ndim() == 2, "index must be a tensor with 2 dimensions");
    checkType(index, "index", Tensor::INT32);
    checkStrides(index, "index");
    CHECK_ERROR(index.size(1) <= 1 || index.numel() == 0 || index.stride(1) == 1, "index must be consecutive along its last dimension");
    const RouteSizes s{logits.size(0), logits.size(1), index.size(1)};
    CHECK_ERROR(s.chosen >= 1 && s.chosen <= s.experts && s.chosen <= ROUTE_MOST_CHOSEN, "between 1 and ", ROUTE_MOST_CHOSEN,
                " experts can be chosen, and no more than there are, but they are ", s.chosen, " of ", s.experts);
    checkSizes(weights, what, {s.rows, s.chosen});
    checkSizes(index, "index", {s.rows, s.chosen});
    checkSteps("experts", s.experts);
    return s;
}

// ------------------------------------------------------------------------------------------------ rows to experts and back
// as in kernels/expert_rows.h
constexpr int EXPERT_ROWS_THREADS = 256;

struct ExpertRowsSizes
{
    long long tokens;
    int chosen, channels;
    /** Entries of an access and lanes of a token. */
    int vec(Tensor::Precision p) const { return channels < wide(p) ? 1 : wide(p); }
    int lanes(Tensor::Precision p, int most) const { return lanesPerRow(channels, vec(p), most); }
    /**
     * Workgroups that share the columns of their tokens: as many as have some, where there are few tokens. us of dispatch() by one | by several, 4096
     * channels, bfloat16: 24 tokens of 8 experts 6.1 | 4.1, 256 of 4 4.6 | 3.7, 1024 of 4 7.8 | 7.4, 4096 of 4 25.5 | 25.8.
     */
    int parts(Tensor::Precision p, int lanes) const
    {
        const int64_t all = divUp<int64_t>(channels, lanes * vec(p)), blocks = divUp<int64_t>(tokens, EXPERT_ROWS_THREADS / lanes);
        return static_cast<int>(blocks * all <= 2048 ? all : 1);
    }
};
ExpertRowsSizes checkExpertRows(const Tensor& rows, const Tensor& places)
{
    checkValues(rows, "rows", 2);
    CHECK_ERROR(places.defined() && places.ndim() == 2, "places must be a tensor with 2 dimensions");
    checkType(places, "places", Tensor::INT32);
    checkStrides(places, "places");
    CHECK_ERROR(places.size(1) <= 1 || places.numel() == 0 || places.stride(1) == 1, "places must be consecutive along its last dimension");
    const ExpertRowsSizes s{places.size(0), places.size(1), rows.size(1)};
    CHECK_ERROR(places.numel() < (1ll << 31), "tokens times chosen experts must fit into 32 bits");
    checkSizes(rows, "rows", {places.numel(), s.channels});
    checkSteps("channels", s.channels);
    return s;
}
void checkTokens(const Tensor& t, const char* what, const Tensor& rows, const ExpertRowsSizes& s)
{
    checkValues(t, what, 2);
    checkType(t, what, rows.precision());
    checkSizes(t, what, {s.tokens, s.channels});
}
/** Weights or their gradients. */
void checkExpertWeights(const Tensor& t, const char* what, const Tensor& rows, const ExpertRowsSizes& s)
{
    if (!t.defined()) return;
    checkValues(t, what, 2);
    CHECK_ERROR(t.precision() == rows.precision() || t.precision() == Tensor::FLOAT, what, " must be of the rows' type or FLOAT");
    checkSizes(t, what, {s.tokens, s.chosen});
}
long long strideOrNone(const Tensor& t) { return t.defined() ? strideOf(t, 0) : 0; }

/**
 * Pieces of a row that a lane of the adjoint kernel has at a time, and the wavefronts that share the rows of a token (all of them or one). us of one
 * and one piece | one, 4 | all, 1 | all, 4: bfloat16, 24 tokens of 8 experts, 4096 channels 31 | 27 | 6.5 | 5.8; 2048, 8, 512 11.4 | 12.3 | 8.7 |
 * 12.7; 4096, 8, 512 14.7 | 15.8 | 15.6 | 22; 16384, 8, 512 45 | 55 | 53 | 79; 16384, 4, 768 39 | 41 | 38 | 54; 4096, 8, 1024 23.9 | 24.2 | 24.6 |
 * 30; 16384, 8, 1024 110 | 122 | 98 | 159; 32768, 2, 2048 134 | 130 | 122 | 143; 8192, 4, 4096 133 | 130 | 109 | 107. Single precision, 1024, 4,
 * 1024 13.8 | 10.0 | 6.8 | 6.9; 4096, 4, 1024 29 | 23.7 | 25 | 23.8; 5003, 3, 333 11.7 | 10.5 | 11.9 | 11.8; 8192, 8, 1024 121 | 106 | 107 | 105;
 * 16384, 8, 512 114 | 103 | 105 | 116.
 */
int expertRowsBatch(Tensor::Precision p, int channels, int vec, int lanes) { return p == Tensor::FLOAT && channels > vec * lanes ? 4 : 1; }
int expertRowsSplit(Tensor::Precision p, const ExpertRowsSizes& s, int vec, int lanes)
{
    return s.tokens <= 2048 || (p != Tensor::FLOAT && s.channels >= 2 * vec * lanes) ? s.chosen : 1;
}

/** Values are moved as they are: a name of a type of their size. */
const char* bitsName(Tensor::Precision p) { return p == Tensor::FLOAT ? "unsigned" : "unsigned short"; }

// ------------------------------------------------------------------------------------------------ numbers of 4 bits
// as in kernels/mx4.h and kernels/mx4_linear.h
constexpr int MX4_THREADS = 256, MX4_BLOCK = 32, MX4_LANES = 4, MX4_FEW_WAVES = 4;
struct Mx4Matrix
{
    const unsigned char *codes, *scales;
    long long codesExpert, scalesExpert, codesRow, scalesRow;
};

/** Codes and scales of 'dims' dimensions; returns the blocks of a row. */
int checkMx4(const Tensor& codes, const char* whatCodes, const Tensor& scales, const char* whatScales, int dims)
{
    for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{codes, whatCodes}, {scales, whatScales}}) {
        CHECK_ERROR(t.defined() && t.ndim() == dims, what, " must be a tensor with ", dims, " dimensions");
        checkType(t, what, Tensor::UINT8);
        checkStrides(t, what);
        CHECK_ERROR(t.size(dims - 1) <= 1 || t.numel() == 0 || t.stride(dims - 1) == 1, what, " must be consecutive along its last dimension");
    }
    const int blocks = scales.size(dims - 1);
    for (int d = 0; d + 1 < dims; ++d)
        CHECK_ERROR(codes.size(d) == scales.size(d), whatCodes, " and ", whatScales, " must be of one size, but have ", codes.size(d), " and ",
                    scales.size(d), " entries at dimension ", d);
    CHECK_ERROR(codes.size(dims - 1) == 16ll * blocks, whatCodes, " must have 16 bytes for each of the ", blocks, " blocks of a row, but has ",
                codes.size(dims - 1));
    return blocks;
}
struct Mx4Tiles
{
    int i, j, wavesI, wavesJ;
    int wavesK = 0;   // few rows: wavefronts that share a chunk of K; otherwise 0
    int threads() const { return wavesK ? 64 * MX4_FEW_WAVES : 64 * wavesI * wavesJ; }
    /** Two tiles of each operand and two pairs of tiles' scales, later the results. */
    unsigned lds(int entry) const { return wavesK ? 0 : static_cast<unsigned>(std::max((2 * 128 + 2 * 16) * (i + j), i * j * entry)); }
    std::string arguments() const { return str(i, ", ", j, ", ", wavesI, ", ", wavesJ); }
};
constexpr Mx4Tiles MX4_HUGE = {256, 256, 2, 4}, MX4_LARGE = {128, 128, 2, 2}, MX4_SMALL = {64, 64, 2, 2};
constexpr Mx4Tiles MX4_TILES[] = {MX4_HUGE, MX4_LARGE, MX4_SMALL};
/** 16 rows at a time, as many outputs for each of the wavefronts that do not share K. */
constexpr Mx4Tiles mx4Few(int wavesK) { return {16, 16 * MX4_FEW_WAVES / wavesK, 1, MX4_FEW_WAVES / wavesK, wavesK}; }
constexpr int MX4_FEW_SHARES[] = {1, 4};

struct Mx4Plan
{
    Mx4Tiles tiles;
    bool inPlace = false;   // the product's workgroups quantise the rows, each for its own outputs
};
/**
 * How the product of 'rows' rows, 'blocks' blocks each, with J outputs of every expert is made. us of the call in a captured graph, bfloat16; rows,
 * experts, inputs, outputs; rows spread evenly at random (23 of 64 experts have some of 24, all of 256, 87 of 100 of 200):
 * Few rows or tiles: the weights straight from memory, one wavefront for a chunk of K; four of them; tiles of 64. Each with rows that are codes | with
 * values, quantised in place, before. 24, 64, 1024, 4096: 14.4 | 14.7, 16.9; 14.9 | 15.6, 17.7; 19.3 | 22.1. 8 of them: 5.4 | 5.6, 7.4; 6.3 | 6.6, 8.4;
 * 10.4 | 12.9. One: 4.3 | 4.5, 6.2; 3.6 | 3.8, 5.5; 6.8 | 8.9. 256, 64, 1024, 4096: 32.8 | 38.0, 36.3; 37.0 | 45.8, 39.4; 32.1 | 34.7. 1, 1, 1024, 1024:
 * 4.3 | 4.5, 6.2; 3.8 | 3.8, 5.5; 5.0 | 7.2. 1, 1, 4096, 4096: 8.8 | 9.4, 11.0; 5.4 | 6.2, 7.7; 12.4 | 14.4. 8, 1, 4096, 4096: 8.9 | 12.7, 11.3; 5.8 |
 * 9.6, 8.1; 12.2 | 14.4. 16, 1, 4096, 4096: 9.6 | 17.2, 12.7; 6.4 | 14.0, 9.5; 12.1 | 14.9. 16, 1, 1024, 1024: 4.6 | 6.5, 7.0; 3.9 | 5.7, 6.3; 5.1 | 7.8.
 * 32, 1, 1024, 1024: 4.6 | 6.5, 6.9; 4.0 | 5.7, 6.3; 5.1 | 7.8. 60, 4, 2048, 2048: 6.3 | 10.1, 9.0; 5.8 | 9.9, 8.2; 6.6 | 10.0. 200, 100, 200, 300:
 * 5.1 | 6.1, 7.6; 6.6 | 8.1, 9.3; 6.0 | 8.6.
 * The rule takes the slower side of 8, 64, 1024, 4096 (four wavefronts, 6.6 with values for 5.6), 200, 100, 200, 300 with codes (tiles, 6.0 for 5.1) and
 * 32, 1, 1024, 1024 with values (before, 6.3 for 5.7).
 * Tiles of 64, 128 and 256, codes: 5003, 12, 333, 200: 6.3, 7.2, 10.7; 256, 1, 4096, 4096: 10.5, 17.9, 28.4; 6400, 64, 512, 512: 9.0, 7.6, 10.0; 3200,
 * 64, 2048, 2048: 34, 37, 52; 6400, 64, 2048, 2048: 52, 46, 53; 16384, 16, 1024, 1024: 29.5, 24.0, 26.5; 8192, 16, 2048, 4096: 87, 62, 62; 32768, 16,
 * 2048, 4096: 306, 204, 183. Single precision, whose results take too much LDS for tiles of 256: 32768, 16, 2048, 4096: 329, 237; 5003, 12, 333,
 * 200: 6.6, 8.0.
 */
Mx4Plan mx4Plan(Tensor::Precision p, int64_t rows, int64_t experts, int64_t J, int64_t blocks, bool values, bool direct)
{
    const int64_t each = rows / std::max<int64_t>(experts, 1);
    auto count = [&](const Mx4Tiles& t) { return (rows / t.i + std::min(experts, rows)) * divUp<int64_t>(J, t.j); };
    auto whole = [&](const Mx4Tiles& t) { return rows / t.i * divUp<int64_t>(J, t.j); };
    const Mx4Tiles few = mx4Few(blocks >= 16 && count(mx4Few(1)) < 700 ? 4 : 1);
    // (what a workgroup and what all of them have to quantise)
    const bool inPlace = values && rows <= 256 && each <= 16 && each * blocks <= 512 && rows * blocks * divUp<int64_t>(J, few.j) <= 1 << 18;
    if (inPlace || !direct || each <= 1 || (each <= 64 && count(MX4_SMALL) <= 128)) return {few, inPlace};
    if (p != Tensor::FLOAT && each > 128 && J > 128 && whole(MX4_HUGE) >= 512) return {MX4_HUGE};
    return {each > 64 && J > 64 && whole(MX4_LARGE) >= 128 ? MX4_LARGE : MX4_SMALL};
}

int mx4Blocks(int64_t columns) { return static_cast<int>(divUp<int64_t>(columns, MX4_BLOCK)); }
unsigned mx4Workgroups(long long units, int lanes) { return workgroups(divUp<int64_t>(units * lanes, MX4_THREADS), 1 << 16); }

void launchQuantise(const Tensor& input, unsigned char* codes, long long strideCodes, unsigned char* scales, long long strideScales, stream_t stream)
{
    const int blocks = mx4Blocks(input.size(1));
    const long long units = static_cast<long long>(input.size(0)) * blocks;
    if (units == 0) return;
    const Tensor::Precision p = input.precision();
    tokenKernel("mx4.h", kernelKey(MX4_QUANTISE, p), [&] { return str("Mx4QuantiseKernel<", scalarName(p), ">"); })
        .call(mx4Workgroups(units, MX4_LANES), MX4_THREADS, 0, stream, input.rawPtr(), strideOf(input, 0), codes, strideCodes, scales, strideScales, units, blocks,
              static_cast<int>(input.size(1)));
}

std::string mx4FewName(Tensor::Precision p, bool inPlace, const Mx4Tiles& t)
{
    return str("Mx4FewKernel<", scalarName(p), ", ", inPlace ? scalarName(p) : "unsigned char", ", ", t.wavesJ, ", ", t.wavesK, ">");
}

/** Rows of the 4-bit operand as a call makes them in its memory. */
struct Mx4Rows
{
    Workspace memory;
    unsigned char *codes, *scales;
    Mx4Rows(int64_t rows, int blocks, void* base)
        : memory{static_cast<char*>(base)}, codes(memory.take<unsigned char>(rows * blocks * 16)), scales(memory.take<unsigned char>(rows * blocks))
    {
    }
};

} // namespace

// ------------------------------------------------------------------------------------------------ entry points
void Tokens::route(const Tensor& logits, bool normalised, Tensor& weights, Tensor& index, stream_t stream)
{
    const RouteSizes s = checkRoute(logits, weights, "weights", index);
    checkOutput(weights, "weights");
    checkOutput(index, "index");
    if (s.rows == 0) return;
    const Tensor::Precision p = logits.precision();
    const RouteShape shape = routeShape(s.experts);
    const bool isLong = shape.lanes == 0;
    tokenKernel("route.h", isLong ? kernelKey(ROUTE_LONG, p) : kernelKey(ROUTE, p, shape.lanes, shape.entries),
                [&] { return isLong ? str("RouteLongKernel<", scalarName(p), ">") : "RouteKernel" + shape.arguments(p); })
        .call(isLong ? workgroups(s.rows, 4096) : workgroups(divUp<int64_t>(s.rows, shape.rows()), 1 << 16), ROUTE_THREADS,
              8 * s.chosen * (isLong ? 1 : shape.rows()), stream, logits.rawPtr(), strideOf(logits, 0), weights.rawPtr(), strideOf(weights, 0),
              ptr<int>(index), strideOf(index, 0), s.rows, s.experts, s.chosen, static_cast<int>(normalised));
}

void Tokens::routeAdjoint(const Tensor& logits, const Tensor& index, const Tensor& adjWeights, bool normalised, Tensor& adjLogits, stream_t stream)
{
    const RouteSizes s = checkRoute(logits, adjWeights, "adjWeights", index);
    checkValues(adjLogits, "adjLogits", 2);
    checkType(adjLogits, "adjLogits", logits.precision());
    checkSizes(adjLogits, "adjLogits", {s.rows, s.experts});
    checkOutput(adjLogits, "adjLogits");
    if (s.rows == 0) return;
    const Tensor::Precision p = logits.precision();
    const RouteShape shape = routeShape(s.experts);
    const bool isLong = shape.lanes == 0;
    tokenKernel("route.h", isLong ? kernelKey(ROUTE_LONG_ADJOINT, p) : kernelKey(ROUTE_ADJOINT, p, shape.lanes, shape.entries),
                [&] { return isLong ? str("RouteLongAdjointKernel<", scalarName(p), ">") : "RouteAdjointKernel" + shape.arguments(p); })
        .call(isLong ? workgroups(s.rows, 4096) : workgroups(divUp<int64_t>(s.rows, shape.rows()), 1 << 16), ROUTE_THREADS, 0, stream, logits.rawPtr(),
              strideOf(logits, 0), static_cast<const int*>(ptr<int>(index)), strideOf(index, 0), adjWeights.rawPtr(), strideOf(adjWeights, 0),
              adjLogits.rawPtr(), strideOf(adjLogits, 0), s.rows, s.experts, s.chosen, static_cast<int>(normalised));
}

void Tokens::dispatch(const Tensor& input, const Tensor& places, Tensor& rows, stream_t stream)
{
    const ExpertRowsSizes s = checkExpertRows(rows, places);
    checkTokens(input, "input", rows, s);
    checkOutput(rows, "rows");
    if (rows.numel() == 0) return;
    const Tensor::Precision p = rows.precision();
    const int vec = s.vec(p), lanes = s.lanes(p, EXPERT_ROWS_THREADS), parts = s.parts(p, lanes);
    tokenKernel("expert_rows.h", kernelKey(DISPATCH, rows.bytesPerEntry(), vec, lanes),
                [&] { return str("DispatchKernel<", bitsName(p), ", ", vec, ", ", lanes, ">"); })
        .call(workgroups(divUp<int64_t>(s.tokens, EXPERT_ROWS_THREADS / lanes), 1 << 20) * parts, EXPERT_ROWS_THREADS, 0, stream, input.rawPtr(),
              strideOf(input, 0), static_cast<const int*>(ptr<int>(places)), strideOf(places, 0), s.chosen, rows.rawPtr(), strideOf(rows, 0), s.tokens, s.channels,
              parts);
}

void Tokens::combine(const Tensor& rows, const Tensor& places, const Tensor& weights, const Tensor& residual, Tensor& output, stream_t stream)
{
    const ExpertRowsSizes s = checkExpertRows(rows, places);
    checkExpertWeights(weights, "weights", rows, s);
    if (residual.defined()) checkTokens(residual, "residual", rows, s);
    checkTokens(output, "output", rows, s);
    checkOutput(output, "output");
    if (output.numel() == 0) return;
    const Tensor::Precision p = rows.precision();
    const int vec = s.vec(p), lanes = s.lanes(p, EXPERT_ROWS_THREADS), parts = s.parts(p, lanes);
    tokenKernel("expert_rows.h", kernelKey(COMBINE, p, vec, lanes), [&] { return str("CombineKernel<", scalarName(p), ", ", vec, ", ", lanes, ">"); })
        .call(workgroups(divUp<int64_t>(s.tokens, EXPERT_ROWS_THREADS / lanes), 1 << 20) * parts, EXPERT_ROWS_THREADS, 0, stream, rows.rawPtr(),
              strideOf(rows, 0), static_cast<const int*>(ptr<int>(places)), strideOf(places, 0), s.chosen, static_cast<const void*>(ptr<void>(weights)),
              strideOrNone(weights), static_cast<int>(weights.defined() && weights.precision() == Tensor::FLOAT),
              static_cast<const void*>(ptr<void>(residual)), strideOrNone(residual), output.rawPtr(), strideOf(output, 0), s.tokens, s.channels, parts);
}

void Tokens::combineAdjoint(const Tensor& rows, const Tensor& places, const Tensor& weights, const Tensor& adjOutput, Tensor& adjRows, Tensor& adjWeights,
                            stream_t stream)
{
    const Tensor& like = rows.defined() || adjWeights.defined() ? rows : adjRows;   // (only the weights' gradient reads the rows)
    const ExpertRowsSizes s = checkExpertRows(like, places);
    checkExpertWeights(weights, "weights", like, s);
    checkExpertWeights(adjWeights, "adjWeights", like, s);
    if (weights.defined() && adjWeights.defined()) checkType(adjWeights, "adjWeights", weights.precision());
    checkTokens(adjOutput, "adjOutput", like, s);
    if (adjRows.defined()) {
        checkValues(adjRows, "adjRows", 2);
        checkType(adjRows, "adjRows", like.precision());
        checkSizes(adjRows, "adjRows", {like.size(0), s.channels});
        checkOutput(adjRows, "adjRows");
    }
    if (adjWeights.defined()) checkOutput(adjWeights, "adjWeights");
    if (places.numel() == 0 || (!adjRows.defined() && !adjWeights.defined())) return;
    const Tensor::Precision p = like.precision();
    const int vec = s.vec(p), lanes = s.lanes(p, 64);
    const Tensor& typed = weights.defined() ? weights : adjWeights;
    const int batch = expertRowsBatch(p, s.channels, vec, lanes), split = expertRowsSplit(p, s, vec, lanes);
    tokenKernel("expert_rows.h", kernelKey(COMBINE_ADJOINT, p, vec, lanes, batch),
                [&] { return str("CombineAdjointKernel<", scalarName(p), ", ", vec, ", ", lanes, ", ", batch, ">"); })
        .call(workgroups(divUp<int64_t>(s.tokens * split, EXPERT_ROWS_THREADS / lanes), 1 << 20), EXPERT_ROWS_THREADS, 0, stream,
              static_cast<const void*>(ptr<void>(rows)), strideOrNone(rows), static_cast<const int*>(ptr<int>(places)), strideOf(places, 0), s.chosen,
              static_cast<const void*>(ptr<void>(weights)), strideOrNone(weights),
              static_cast<int>(typed.defined() && typed.precision() == Tensor::FLOAT), adjOutput.rawPtr(), strideOf(adjOutput, 0), ptr<void>(adjRows),
              strideOrNone(adjRows), ptr<void>(adjWeights), strideOrNone(adjWeights), s.tokens, s.channels, split);
}

void Tokens::quantiseMx4(const Tensor& input, Tensor& codes, Tensor& scales, stream_t stream)
{
    checkValues(input, "input", 2);
    checkSteps("columns", input.size(1));
    const int blocks = checkMx4(codes, "codes", scales, "scales", 2);
    CHECK_ERROR(blocks == mx4Blocks(input.size(1)), "scales must have ", mx4Blocks(input.size(1)), " entries at dimension 1, but has ", blocks);
    checkSizes(scales, "scales", {input.size(0), blocks});
    checkOutput(codes, "codes");
    checkOutput(scales, "scales");
    launchQuantise(input, ptr<unsigned char>(codes), strideOf(codes, 0), ptr<unsigned char>(scales), strideOf(scales, 0), stream);
}

void Tokens::valuesMx4(const Tensor& codes, const Tensor& scales, Tensor& output, stream_t stream)
{
    checkValues(output, "output", 2);
    checkOutput(output, "output");
    checkSteps("columns", output.size(1));
    const int blocks = checkMx4(codes, "codes", scales, "scales", 2);
    CHECK_ERROR(blocks == mx4Blocks(output.size(1)), "scales must have ", mx4Blocks(output.size(1)), " entries at dimension 1, but has ", blocks);
    checkSizes(scales, "scales", {output.size(0), blocks});
    const long long units = static_cast<long long>(output.size(0)) * blocks;
    if (units == 0) return;
    const Tensor::Precision p = output.precision();
    tokenKernel("mx4.h", kernelKey(MX4_VALUES, p), [&] { return str("Mx4ValuesKernel<", scalarName(p), ">"); })
        .call(mx4Workgroups(units, MX4_BLOCK / wide(p)), MX4_THREADS, 0, stream, static_cast<const unsigned char*>(ptr<unsigned char>(codes)), strideOf(codes, 0),
              static_cast<const unsigned char*>(ptr<unsigned char>(scales)), strideOf(scales, 0), output.rawPtr(), strideOf(output, 0), units, blocks,
              static_cast<int>(output.size(1)));
}

size_t Tokens::mx4LinearMemory(int64_t rows, int experts, int inputs, int outputs)
{
    CHECK_ERROR(rows >= 0 && experts >= 0 && inputs >= 0 && outputs >= 0, "sizes must not be negative");
    const int blocks = mx4Blocks(inputs);
    return mx4Plan(Tensor::FLOAT, rows, experts, outputs, blocks, true, true).inPlace ? 0 : Mx4Rows(rows, blocks, nullptr).memory.bytes;
}

void Tokens::mx4Linear(const Tensor& input, const Tensor& inputScales, const Tensor& weight, const Tensor& scales, const Tensor& offsets, const Tensor& bias,
                       Tensor& output, void* memory, stream_t stream)
{
    const int blocks = checkMx4(weight, "weight", scales, "scales", 3);
    const bool quantised = inputScales.defined();
    if (quantised) {
        const int of = checkMx4(input, "input", inputScales, "inputScales", 2);
        CHECK_ERROR(of == blocks, "input must have the weights' ", blocks, " blocks in a row, but has ", of);
    } else {
        checkValues(input, "input", 2);
        CHECK_ERROR(mx4Blocks(input.size(1)) == blocks, "input must have the weights' ", blocks, " blocks in a row, but has ", mx4Blocks(input.size(1)));
    }
    const int rows = input.size(0), experts = weight.size(0), outputs = weight.size(1);
    CHECK_ERROR(blocks > 0 && outputs > 0, "experts must have inputs and outputs");
    if (offsets.defined()) {
        CHECK_ERROR(offsets.ndim() == 1, "offsets must be a tensor with 1 dimension");
        checkType(offsets, "offsets", Tensor::INT32);
        CHECK_ERROR(offsets.size(0) <= 1 || offsets.stride(0) == 1, "offsets must be contiguous");
        checkSizes(offsets, "offsets", {experts + 1ll});
    } else
        CHECK_ERROR(experts == 1, "without offsets there must be one expert, but there are ", experts);
    checkValues(output, "output", 2);
    if (!quantised) checkType(output, "output", input.precision());
    checkSizes(output, "output", {rows, outputs});
    checkOutput(output, "output");
    if (bias.defined()) {
        checkValues(bias, "bias", 2);
        checkType(bias, "bias", output.precision());
        checkSizes(bias, "bias", {experts, outputs});
    }
    checkSteps("rows", rows);
    checkSteps("inputs", static_cast<int64_t>(blocks) * MX4_BLOCK);
    checkSteps("outputs", outputs);
    if (rows == 0) return;
    const Tensor::Precision p = output.precision();
    // pieces of 16 bytes, rows that do not overlap and whose tiles have 32-bit offsets: straight to LDS
    const auto direct = [](const Tensor& t) {
        const int n = t.ndim();
        for (int d = 0; d + 1 < n; ++d)
            if (t.size(d) > 1 && t.stride(d) % 16 != 0) return false;
        return reinterpret_cast<uintptr_t>(t.rawPtr()) % 16 == 0 && (t.size(n - 2) <= 1 || (t.stride(n - 2) >= t.size(n - 1) && t.stride(n - 2) < 1 << 22));
    };
    const bool isDirect = direct(weight) && (!quantised || direct(input)) && blocks < 1 << 17;
    const Mx4Plan plan = mx4Plan(p, rows, experts, outputs, blocks, !quantised, isDirect);
    const Mx4Tiles& tiles = plan.tiles;
    const bool few = tiles.wavesK > 0;
    const int64_t all = static_cast<int64_t>(rows) / tiles.i + experts + 1, places = few ? std::min<int64_t>(all, rows) : all, tilesJ = divUp<int64_t>(outputs, tiles.j);
    checkLaunch(places * tilesJ, tiles.threads());
    const Mx4Matrix w{ptr<unsigned char>(weight), ptr<unsigned char>(scales), strideOf(weight, 0), strideOf(scales, 0), strideOf(weight, 1), strideOf(scales, 1)};
    const void* const b = ptr<void>(bias);
    const int* const off = ptr<int>(offsets);
    const int count = static_cast<int>(places), countJ = static_cast<int>(tilesJ), byRow = places < all;
    const unsigned groups = static_cast<unsigned>(places * tilesJ);
    const void* x = input.rawPtr();
    const unsigned char* scalesX = ptr<unsigned char>(inputScales);
    long long strideX = strideOf(input, 0), strideScalesX = strideOrNone(inputScales);
    if (!quantised && !plan.inPlace) {
        const Mx4Rows codes(rows, blocks, memory);
        checkMemory(memory, codes.memory.bytes);
        strideX = blocks * 16ll;
        strideScalesX = blocks;
        launchQuantise(input, codes.codes, strideX, codes.scales, strideScalesX, stream);
        x = codes.codes;
        scalesX = codes.scales;
    }
    if (few)
        tokenKernel("mx4_linear.h", kernelKey(MX4_FEW, p, plan.inPlace, tiles.wavesK), [&] { return mx4FewName(p, plan.inPlace, tiles); })
            .call(groups, tiles.threads(), 0, stream, x, scalesX, strideX, strideScalesX, w, b, strideOrNone(bias), off, experts, output.rawPtr(),
                  strideOf(output, 0), rows, outputs, blocks, plan.inPlace ? static_cast<int>(input.size(1)) : 0, byRow, countJ);
    else
        tokenKernel("mx4_linear.h", kernelKey(MX4_TILES_OF, p, tiles.i, tiles.j, tiles.wavesI, tiles.wavesJ),
                    [&] { return str("Mx4TilesKernel<", scalarName(p), ", ", tiles.arguments(), ">"); })
            .call(groups, tiles.threads(), tiles.lds(output.bytesPerEntry()), stream, x, scalesX, strideX, strideScalesX, w, b, strideOrNone(bias), off,
                  experts, output.rawPtr(), strideOf(output, 0), rows, outputs, blocks, count, countJ);
}

void token::precompileExperts(Tensor::Precision p)
{
    const std::string t = scalarName(p);
    for (const RouteShape& s : ROUTE_SHAPES)
        for (const char* kernel : {"RouteKernel", "RouteAdjointKernel"}) precompileKernel("route.h", kernel + s.arguments(p));
    for (const char* kernel : {"RouteLongKernel", "RouteLongAdjointKernel"}) precompileKernel("route.h", str(kernel, "<", t, ">"));
    for (const int vec : {1, wide(p)})
        for (const int lanes : {8, 16, 32, 64, 128, 256}) {
            if (vec == 1 && lanes > 8) continue;
            const std::string shape = str(", ", vec, ", ", lanes, ">");
            precompileKernel("expert_rows.h", str("DispatchKernel<", bitsName(p), shape));
            precompileKernel("expert_rows.h", str("CombineKernel<", t, shape));
            for (const int batch : {1, 4})
                if (batch == 1 ? lanes <= 64 : lanes == 64 && p == Tensor::FLOAT)
                    precompileKernel("expert_rows.h", str("CombineAdjointKernel<", t, ", ", vec, ", ", lanes, ", ", batch, ">"));
        }
    for (const char* kernel : {"Mx4QuantiseKernel", "Mx4ValuesKernel"}) precompileKernel("mx4.h", str(kernel, "<", t, ">"));
    for (const bool inPlace : {false, true})
        for (const int share : MX4_FEW_SHARES) precompileKernel("mx4_linear.h", mx4FewName(p, inPlace, mx4Few(share)));
    for (const Mx4Tiles& tiles : MX4_TILES)
        if (p != Tensor::FLOAT || tiles.i < MX4_HUGE.i) precompileKernel("mx4_linear.h", str("Mx4TilesKernel<", t, ", ", tiles.arguments(), ">"));
}

QUICKMLP_NAMESPACE_END

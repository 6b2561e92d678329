// The operators around experts by the C++ class qmlp::Tokens: a layer of experts from the logits to the sum of its rows, with numbers that have
// exact results, its gradients, and refusals. Usage: test_tokens_api [--host]. With --host only the part that needs no GPU runs. Exit code 0 = all
// checks passed.
#include <qmlp/qmlp.h>
#include <qmlp/tmp_memory.h>
#include <qmlp/tokens.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

using namespace qmlp;

static int failures = 0;
#define CHECK(cond)                                                            \
    do {                                                                       \
        if (!(cond)) {                                                         \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);      \
            ++failures;                                                        \
        }                                                                      \
    } while (0)

template <typename Call>
static bool refuses(Call call, const char* what)
{
    try {
        call();
    } catch (const std::exception& e) {
        return std::strstr(e.what(), what) != nullptr;
    }
    return false;
}

static Tensor described(Tensor::Precision p, const std::vector<int32_t>& sizes)
{
    std::vector<int32_t> strides(sizes.size(), 1);
    for (size_t d = sizes.size() - 1; d > 0; --d) strides[d - 1] = strides[d] * sizes[d];
    return Tensor(reinterpret_cast<void*>(256), p, sizes, strides);
}

static void hostPart()
{
    const Tensor logits = described(Tensor::FLOAT, {4, 6}), none;
    Tensor weights = described(Tensor::FLOAT, {4, 7}), index = described(Tensor::INT32, {4, 7});
    CHECK(refuses([&] { Tokens::route(logits, false, weights, index, nullptr); }, "no more than there are"));
    Tensor rows = described(Tensor::FLOAT, {7, 6});
    const Tensor places = described(Tensor::INT32, {4, 2});
    CHECK(refuses([&] { Tokens::dispatch(logits, places, rows, nullptr); }, "must have 8 entries"));
    Tensor output = described(Tensor::HALF, {4, 6});
    CHECK(refuses([&] { Tokens::combine(described(Tensor::FLOAT, {8, 6}), places, none, none, output, nullptr); }, "must be of type FLOAT"));
    Tensor noRows, adjWeights = described(Tensor::FLOAT, {4, 2});
    CHECK(refuses([&] { Tokens::combineAdjoint(none, places, none, logits, noRows, adjWeights, nullptr); }, "rows is undefined"));
    Tensor codes = described(Tensor::UINT8, {4, 16}), scales = described(Tensor::FLOAT, {4, 1});
    CHECK(refuses([&] { Tokens::quantiseMx4(logits, codes, scales, nullptr); }, "must be of type UINT8"));
    // codes and scales of 400 rows of 2 blocks, each to a multiple of 256 bytes; few rows are quantised where they are multiplied
    CHECK(Tokens::mx4LinearMemory(400, 3, 40, 5) == 400 * 32 + 1024 && Tokens::mx4LinearMemory(4, 3, 40, 5) == 0);
}

template <typename T>
static Tensor onDevice(Tensor::Precision p, const std::vector<int32_t>& sizes, const std::vector<T>& values)
{
    Tensor t(p, sizes);
    t.copyFromHost(values.data(), sizeof(T) * values.size());
    return t;
}
template <typename T>
static std::vector<T> onHost(const Tensor& t)
{
    std::vector<T> values(t.numel());
    t.copyToHost(values.data(), sizeof(T) * values.size());
    return values;
}

static void gpuPart()
{
    const int TOKENS = 3, EXPERTS = 4, CHOSEN = 2, C = 32;
    const float no = -INFINITY;
    // the last token takes one expert only; the two experts of the first have equal logits, so that its weights are halves
    const Tensor logits = onDevice<float>(Tensor::FLOAT, {TOKENS, EXPERTS}, {1, 3, 3, 0, /**/ 5, 1, 5, 5, /**/ no, no, 2, no});
    Tensor weights(Tensor::FLOAT, {TOKENS, CHOSEN}), index(Tensor::INT32, {TOKENS, CHOSEN});
    Tokens::route(logits, true, weights, index, nullptr);
    CHECK((onHost<int32_t>(index) == std::vector<int32_t>{1, 2, 0, 2, 2, -1}));
    CHECK((onHost<float>(weights) == std::vector<float>{0.5f, 0.5f, 0.5f, 0.5f, 1, 0}));

    Tensor order(Tensor::INT32, {TOKENS * CHOSEN}), offsets(Tensor::INT32, {EXPERTS + 1}), places(Tensor::INT32, {TOKENS * CHOSEN});
    TmpMemory sort(Tokens::groupMemory(TOKENS * CHOSEN, EXPERTS));
    const Tensor flat(index.rawPtr(), Tensor::INT32, {TOKENS * CHOSEN}, {1});
    Tokens::group(flat, EXPERTS, order, offsets, places, sort.get(), nullptr);
    CHECK((onHost<int32_t>(order) == std::vector<int32_t>{2, 0, 1, 3, 4, 5}));
    CHECK((onHost<int32_t>(offsets) == std::vector<int32_t>{0, 1, 2, 5, 5}));
    CHECK((onHost<int32_t>(places) == std::vector<int32_t>{1, 2, 0, 3, 4, -6}));

    std::vector<float> x(TOKENS * C);
    const float numbers[] = {0, 0.5f, 1, 1.5f, 2, 3, 4, 6};
    for (int i = 0; i < TOKENS * C; ++i) x[i] = (i % 3 == 1 ? -1 : 1) * numbers[(i + 7) % 8];   // (the first of every block is 6: scale 1)
    const Tensor input = onDevice(Tensor::FLOAT, {TOKENS, C}, x), at(places.rawPtr(), Tensor::INT32, {TOKENS, CHOSEN}, {CHOSEN, 1});
    Tensor rows(Tensor::FLOAT, {TOKENS * CHOSEN, C});
    Tokens::dispatch(input, at, rows, nullptr);
    const int tokenOf[] = {1, 0, 0, 1, 2, -1};   // of the rows
    std::vector<float> expected(TOKENS * CHOSEN * C, 0.f);
    for (int r = 0; r < 5; ++r)
        for (int c = 0; c < C; ++c) expected[r * C + c] = x[tokenOf[r] * C + c];
    CHECK(onHost<float>(rows) == expected);

    // expert e multiplies by 2^e; a bias of 1 for all
    std::vector<float> w(EXPERTS * C * C, 0.f), ones(EXPERTS * C, 1.f);
    for (int e = 0; e < EXPERTS; ++e)
        for (int c = 0; c < C; ++c) w[(e * C + c) * C + c] = std::ldexp(1.f, e);
    Tensor codes(Tensor::UINT8, {EXPERTS * C, 16}), scales(Tensor::UINT8, {EXPERTS * C, 1}), values(Tensor::FLOAT, {EXPERTS * C, C});
    Tokens::quantiseMx4(onDevice(Tensor::FLOAT, {EXPERTS * C, C}, w), codes, scales, nullptr);
    Tokens::valuesMx4(codes, scales, values, nullptr);
    CHECK(onHost<float>(values) == w);
    const Tensor bias = onDevice(Tensor::FLOAT, {EXPERTS, C}, ones), none;
    const Tensor codes3(codes.rawPtr(), Tensor::UINT8, {EXPERTS, C, 16}, {C * 16, 16, 1}), scales3(scales.rawPtr(), Tensor::UINT8, {EXPERTS, C, 1}, {C, 1, 1});
    Tensor hidden(Tensor::FLOAT, {TOKENS * CHOSEN, C});
    TmpMemory memory(std::max<size_t>(1, Tokens::mx4LinearMemory(TOKENS * CHOSEN, EXPERTS, C, C)));
    Tokens::mx4Linear(rows, none, codes3, scales3, offsets, bias, hidden, memory.get(), nullptr);
    const float factor[] = {1, 2, 4, 4, 4};   // of the rows' experts
    for (int r = 0; r < 5; ++r)
        for (int c = 0; c < C; ++c) expected[r * C + c] = factor[r] * expected[r * C + c] + 1;
    CHECK(onHost<float>(hidden) == expected);

    Tensor output(Tensor::FLOAT, {TOKENS, C});
    Tokens::combine(hidden, at, weights, input, output, nullptr);
    const std::vector<float> y = onHost<float>(output);
    const float sum[] = {4, 3.5f, 5};   // x (1 + the sum of weight times factor) + the sum of the weights
    int bad = 0;
    for (int i = 0; i < TOKENS * C; ++i) bad += y[i] != sum[i / C] * x[i] + 1;
    CHECK(bad == 0);

    // gradients: of the rows without the rows themselves, of the weights with them, of the logits
    Tensor adjRows(Tensor::FLOAT, {TOKENS * CHOSEN, C}), adjWeights(Tensor::FLOAT, {TOKENS, CHOSEN}), noTensor, adjLogits(Tensor::FLOAT, {TOKENS, EXPERTS});
    Tokens::combineAdjoint(none, at, weights, input, adjRows, noTensor, nullptr);
    const float weightOf[] = {0.5f, 0.5f, 0.5f, 0.5f, 1, 0};   // of the rows
    const std::vector<float> dr = onHost<float>(adjRows);
    bad = 0;
    for (int i = 0; i < TOKENS * CHOSEN * C; ++i) bad += dr[i] != (tokenOf[i / C] < 0 ? 0 : weightOf[i / C] * x[tokenOf[i / C] * C + i % C]);
    CHECK(bad == 0);
    Tokens::combineAdjoint(hidden, at, weights, input, noTensor, adjWeights, nullptr);
    std::vector<float> dw(TOKENS * CHOSEN, 0.f);
    const int rowOf[] = {1, 2, 0, 3, 4, -1};
    for (int i = 0; i < TOKENS * CHOSEN; ++i)
        for (int c = 0; rowOf[i] >= 0 && c < C; ++c) dw[i] += x[i / CHOSEN * C + c] * expected[rowOf[i] * C + c];   // (halves and quarters: exact)
    CHECK(onHost<float>(adjWeights) == dw);
    Tokens::routeAdjoint(logits, index, adjWeights, true, adjLogits, nullptr);
    const std::vector<float> dl = onHost<float>(adjLogits);
    const float a = 0.25f * (dw[0] - dw[1]), b = 0.25f * (dw[2] - dw[3]);   // p (g - p g - q h) with p = q = 1/2
    CHECK((dl == std::vector<float>{0, a, -a, 0, b, 0, -b, 0, 0, 0, 0, 0}));
}

int main(int argc, char** argv)
{
    const bool hostOnly = argc > 1 && std::strcmp(argv[1], "--host") == 0;
    try {
        QuickMLP::Instance().setLogLevel("error");
        hostPart();
        if (!hostOnly) {
            QuickMLP::Instance().checkHipAvailable();
            gpuPart();
        }
    } catch (const std::exception& e) {
        std::printf("FAILED with exception: %s\n", e.what());
        return 2;
    }
    std::printf(failures ? "%d check(s) failed\n" : "all checks passed\n", failures);
    return failures ? 1 : 0;
}

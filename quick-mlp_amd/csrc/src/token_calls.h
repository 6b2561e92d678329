#pragma once
// What the operators on rows of tokens (tokens.cpp, token_experts.cpp) have in common: their kernels, memory and checks.

#include <qmlp/tokens.h>

#include <qmlp/errors.h>
#include <qmlp/qmlp.h>

#include "qmlp_hip.h"

#include <algorithm>
#include <mutex>
#include <unordered_map>

QUICKMLP_NAMESPACE_BEGIN

namespace token {

constexpr size_t ALIGNMENT = 256;

// ------------------------------------------------------------------------------------------------ kernels
inline const char* scalarName(Tensor::Precision p)
{
    switch (p) {
        case Tensor::FLOAT: return "float";
        case Tensor::HALF: return "_Float16";
        case Tensor::BFLOAT16: return "__bf16";
        case Tensor::INT32: return "int";
        case Tensor::INT64: return "long long";
        default: throw std::runtime_error("values must be float, half or bfloat16, indices 32- or 64-bit integers");
    }
}

/** Entries of a 16-byte access. */
inline int wide(Tensor::Precision p) { return 16 / Tensor::BytesPerEntry[p]; }

enum KernelId { GROUP_SMALL = 1, GROUP_COUNT, GROUP_SCAN, GROUP_SCATTER, GROUP_OFFSETS, EMBEDDING, EMBEDDING_BLOCKS, EMBEDDING_ADJOINT, LAYER_NORM,
                LAYER_NORM_ADJOINT, LAYER_NORM_SUM, LAYER_NORM_LONG, LAYER_NORM_LONG_ADJOINT, LAYER_NORM_LONG_SUMS, GROUPED_ROWS, GROUPED_WEIGHTS,
                GROUPED_SUM, GROUPED_JOIN, ROUTE, ROUTE_ADJOINT, ROUTE_LONG, ROUTE_LONG_ADJOINT, DISPATCH, COMBINE, COMBINE_ADJOINT, MX4_QUANTISE, MX4_VALUES, MX4_FEW, MX4_TILES_OF,
                KERNEL_IDS };
/**
 * One number for a kernel and its template arguments, each below 2^11: to build its name takes as long as to launch it. No id is 0, so that
 * kernels with n arguments have numbers from 2^(11 n) up to less than 2^(11 (n + 1)).
 */
template <typename... Args>
constexpr uint64_t kernelKey(KernelId id, Args... args)
{
    static_assert(sizeof...(args) <= 5 && KERNEL_IDS <= 1 << (64 - 5 * 11), "64 bits");
    uint64_t key = id;
    ((key = key << 11 | static_cast<uint64_t>(args)), ...);
    return key;
}
static_assert(kernelKey(GROUP_SMALL, 0) > kernelKey(KERNEL_IDS), "the smallest number with an argument is above all without");
/** The kernels in use, which stay loaded for the life of the process. */
struct TokenKernels
{
    std::mutex mutex;
    std::unordered_map<uint64_t, KernelFunction> loaded;
};
inline TokenKernels& tokenKernels()
{
    static TokenKernels kernels;
    return kernels;
}
/** File: below kernels/qmlp/kernels; name(): with its template arguments. */
template <typename Name>
KernelFunction& tokenKernel(const char* file, uint64_t key, Name name)
{
    TokenKernels& kernels = tokenKernels();
    std::lock_guard<std::mutex> lock(kernels.mutex);
    auto it = kernels.loaded.find(key);
    if (it == kernels.loaded.end()) {
        auto loaded = QuickMLP::Instance().kernelLoader()->getKernel("qmlp::kernel::" + std::string(name()),
                                                                     KernelLoader::MainFile(std::string("qmlp/kernels/") + file),
                                                                     QuickMLP::Instance().getCompileFlags() | KernelLoader::CompileThrowOnError);
        it = kernels.loaded.emplace(key, std::move(*loaded)).first;
    }
    return it->second;
}
inline void precompileKernel(const char* file, const std::string& name)
{
    QuickMLP::Instance().kernelLoader()->getKernel("qmlp::kernel::" + name, KernelLoader::MainFile(std::string("qmlp/kernels/") + file),
                                                   QuickMLP::Instance().getCompileFlags() | KernelLoader::CompileThrowOnError | KernelLoader::CompileOnly);
}

/** Hands out a workspace piece by piece; without a base only its size is wanted. */
struct Workspace
{
    char* base;
    size_t bytes = 0;
    template <typename T>
    T* take(int64_t count)
    {
        T* p = base ? reinterpret_cast<T*>(base + bytes) : nullptr;
        bytes += roundUp(static_cast<size_t>(std::max<int64_t>(count, 0)) * sizeof(T), ALIGNMENT);
        return p;
    }
};

// ------------------------------------------------------------------------------------------------ checks
inline bool isValue(Tensor::Precision p) { return p == Tensor::FLOAT || p == Tensor::HALF || p == Tensor::BFLOAT16; }

inline void checkStrides(const Tensor& t, const char* what)
{
    for (int d = 0; d < t.ndim(); ++d) {
        CHECK_ERROR(t.size(d) >= 0, what, " has a negative size");
        if (t.size(d) <= 1) continue;   // its stride is not used
        CHECK_ERROR(t.stride(d) >= 0, what, " has a negative stride");
    }
}
/** Values, whose last dimension is consecutive. */
inline void checkValues(const Tensor& t, const char* what, int dims)
{
    CHECK_ERROR(t.defined(), what, " is undefined");
    CHECK_ERROR(t.ndim() == dims, what, " must be a tensor with ", dims, " dimensions, but has ", t.ndim());
    CHECK_ERROR(isValue(t.precision()), what, " must be of type float, half or bfloat16, but is ", Tensor::NamePerEntry[t.precision()]);
    checkStrides(t, what);
    CHECK_ERROR(t.size(dims - 1) <= 1 || t.numel() == 0 || t.stride(dims - 1) == 1, what, " must be consecutive along its last dimension");
}
inline void checkSizes(const Tensor& t, const char* what, std::initializer_list<int64_t> sizes)
{
    int d = 0;
    for (const int64_t s : sizes) {
        CHECK_ERROR(t.size(d) == s, what, " must have ", s, " entries at dimension ", d, ", but has ", t.size(d));
        ++d;
    }
}
inline void checkType(const Tensor& t, const char* what, Tensor::Precision p)
{
    CHECK_ERROR(t.precision() == p, what, " must be of type ", Tensor::NamePerEntry[p], ", but is ", Tensor::NamePerEntry[t.precision()]);
}
/** Something is written: no two entries may be one. */
inline void checkOutput(const Tensor& t, const char* what)
{
    for (int d = 0; d + 1 < t.ndim(); ++d) {
        int64_t inner = 1;
        for (int k = d + 1; k < t.ndim(); ++k) inner += static_cast<int64_t>(t.size(k) - 1) * t.stride(k);
        CHECK_ERROR(t.numel() == 0 || t.size(d) <= 1 || t.stride(d) >= inner, what, " has entries that share memory");
    }
}
inline void checkContiguous(const Tensor& t, const char* what)
{
    int64_t stride = 1;
    for (int d = t.ndim() - 1; d >= 0; --d) {
        CHECK_ERROR(t.size(d) <= 1 || t.stride(d) == stride, what, " must be contiguous");
        stride *= t.size(d);
    }
}
/** The kernels go along some sizes in steps of up to 2048 entries, counted in 32 bits: the step behind the last entry has a number too. */
inline void checkSteps(const char* what, int64_t size)
{
    constexpr int64_t most = (1ll << 31) - (1ll << 12);
    CHECK_ERROR(size <= most, what, " must not be more than ", most, ", but are ", size);
}
inline void checkIndex(const Tensor& t, const char* what)
{
    CHECK_ERROR(t.defined() && t.ndim() == 1, what, " must be a tensor with 1 dimension");
    CHECK_ERROR(t.precision() == Tensor::INT32 || t.precision() == Tensor::INT64, what, " must hold 32- or 64-bit integers, but is ",
                Tensor::NamePerEntry[t.precision()]);
    checkStrides(t, what);
}
inline void checkMemory(const void* memory, size_t bytes)
{
    CHECK_ERROR(bytes == 0 || memory != nullptr, "the call needs ", bytes, " bytes of memory");
    CHECK_ERROR(reinterpret_cast<uintptr_t>(memory) % ALIGNMENT == 0, "memory must be aligned to ", ALIGNMENT, " bytes");
}

template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(const_cast<void*>(t.rawPtr())) : nullptr; }
/** The stride of a dimension; of one with a single entry it may be anything and is taken to be that of rows side by side. */
inline long long strideOf(const Tensor& t, int d) { return t.size(d) <= 1 ? t.size(t.ndim() - 1) : t.stride(d); }

/** A launch counts its threads in 32 bits. */
inline bool isLaunch(int64_t groups, int threads) { return groups * threads < (1ll << 32); }
inline void checkLaunch(int64_t groups, int threads) { CHECK_ERROR(isLaunch(groups, threads), "the call is too large for one launch"); }
/** Workgroups for so many pieces of work of their own, no more than 'most' (the kernels go on in steps of the grid). */
inline unsigned workgroups(int64_t pieces, int64_t most) { return static_cast<unsigned>(std::max<int64_t>(1, std::min(pieces, most))); }

/** Lanes of a workgroup of 256, or of as many as 'most', that share a row of C entries. */
inline int lanesPerRow(int C, int vec, int most = 256)
{
    int lanes = 8;
    while (lanes < most && lanes * vec < C) lanes *= 2;
    return lanes;
}

/** Kernels of token_experts.cpp. */
void precompileExperts(Tensor::Precision p);

} // namespace token

QUICKMLP_NAMESPACE_END

#pragma once

#include "common.h"
#include "tensor.h"

QUICKMLP_NAMESPACE_BEGIN

/**
 * Operators on rows of tokens: what a model of tokens with experts needs beside networks and encodings. They have no
 * counterpart in the reference.
 *
 * Values are float, half or bfloat16, sums are held in float and rounded once. Rows are the first dimension; the last one has
 * to be consecutive in memory (stride 1), the others may have any stride that is not negative. Indices are 32- or 64-bit integers.
 * Channels, inputs, outputs and the rows of experts are no more than 2^31 - 2^12.
 *
 * Every call only enqueues kernels on the stream: it allocates nothing, does not wait and can be captured into a graph once its kernels are
 * loaded. 'memory' is device memory of the caller, aligned to 256 bytes, of the size that the function beside tells,
 * and the call's own until its kernels have run.
 */
class Tokens
{
public:
    /** Bytes of 'memory' for group(). */
    static size_t groupMemory(int64_t rows, int groups);
    /**
     * Rows in the order of their groups, rows of one group in their own order.
     * \param index (rows) the group of a row; a row whose index is not in 0 .. groups - 1 belongs to none
     * \param groups number of groups
     * \param order (rows) INT32, the rows by group; those of no group come last
     * \param offsets (groups + 1) INT32: group g has the entries offsets[g] to offsets[g + 1] - 1 of 'order'
     */
    static void group(const Tensor& index, int groups, Tensor& order, Tensor& offsets, void* memory, stream_t stream);

    /**
     * output[i] = scale * table[index[i]]; a row of zeros where the index names no row of the table.
     * \param index (rows) \param table (vocabulary, channels) \param output (rows, channels)
     */
    static void embedding(const Tensor& index, const Tensor& table, float scale, Tensor& output, stream_t stream);
    /** Bytes of 'memory' for embeddingAdjoint(). */
    static size_t embeddingAdjointMemory(int64_t rows, int64_t vocabulary, int channels);
    /**
     * Gradient of the table, written as a whole: adjTable[v] = scale * sum of the adjOutput[i] with index[i] = v. The same inputs give
     * the same bits.
     */
    static void embeddingAdjoint(const Tensor& index, const Tensor& adjOutput, float scale, Tensor& adjTable, void* memory, stream_t stream);

    /**
     * output = (input - mean) / sqrt(variance + epsilon) * weight + bias, mean and variance of every row over its channels.
     * \param input (rows, channels) \param weight (channels), of the input's type or FLOAT, or undefined: 1
     * \param bias as weight, or undefined: 0 \param output (rows, channels)
     * \param mean (rows) FLOAT, or undefined: not kept for the adjoint \param rstd (rows) FLOAT, 1 / sqrt(variance + epsilon), or undefined
     */
    static void layerNorm(const Tensor& input, const Tensor& weight, const Tensor& bias, float epsilon, Tensor& output, Tensor& mean,
                          Tensor& rstd, stream_t stream);
    /** Bytes of 'memory' for layerNormAdjoint(). */
    static size_t layerNormAdjointMemory(int64_t rows, int channels);
    /**
     * Gradients, written as a whole, each of them may be undefined: not wanted. input, mean, rstd: as the forward pass saw and left them.
     */
    static void layerNormAdjoint(const Tensor& input, const Tensor& weight, const Tensor& mean, const Tensor& rstd, const Tensor& adjOutput,
                                 Tensor& adjInput, Tensor& adjWeight, Tensor& adjBias, void* memory, stream_t stream);

    /** Bytes of 'memory' for groupedLinear(). */
    static size_t groupedLinearMemory(int64_t rows, int experts, int inputs, int outputs);
    /**
     * The linear layer of every expert on its rows: output[r] = weight[e] input[r] + bias[e] for offsets[e] <= r < offsets[e + 1].
     * \param input (rows, inputs) \param weight (experts, outputs, inputs), of the input's type \param offsets (experts + 1) INT32, in device
     * memory, not decreasing, from 0 on; rows behind the last expert's get zeros \param bias (experts, outputs) or undefined
     * \param output (rows, outputs)
     */
    static void groupedLinear(const Tensor& input, const Tensor& weight, const Tensor& offsets, const Tensor& bias, Tensor& output, void* memory,
                              stream_t stream);
    /** Bytes of 'memory' for groupedLinearAdjoint(). */
    static size_t groupedLinearAdjointMemory(int64_t rows, int experts, int inputs, int outputs);
    /**
     * Gradients, written as a whole, each of them may be undefined: not wanted. adjWeight and adjBias are contiguous. The same inputs
     * give the same bits.
     */
    static void groupedLinearAdjoint(const Tensor& input, const Tensor& weight, const Tensor& offsets, const Tensor& adjOutput, Tensor& adjInput,
                                     Tensor& adjWeight, Tensor& adjBias, void* memory, stream_t stream);

    /** Compiles the kernels for values of one precision into the kernel cache; needs no GPU. */
    static void precompile(Tensor::Precision precision);
};

QUICKMLP_NAMESPACE_END

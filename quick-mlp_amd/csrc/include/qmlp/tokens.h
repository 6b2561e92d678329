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
 * Results share no memory with arguments.
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
    /** \param places (rows) INT32, the place of every row in 'order', -1 - place of the rows that belong to no group; or undefined */
    static void group(const Tensor& index, int groups, Tensor& order, Tensor& offsets, Tensor& places, void* memory, stream_t stream);

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

    /**
     * The router's choice: index[r] are the experts with the largest logits of row r, the first of equals, and weights[r] their shares of the softmax
     * over all experts, or, 'normalised', over the chosen ones. No row takes an expert whose logit is -inf: -1 and a weight of 0 stand in its place. A
     * NaN counts as the largest; weights of rows with a NaN or +inf are NaN.
     * \param logits (rows, experts) \param weights (rows, chosen), of the logits' type \param index (rows, chosen) INT32. 1 <= chosen <= experts, <= 64
     */
    static void route(const Tensor& logits, bool normalised, Tensor& weights, Tensor& index, stream_t stream);
    /** Gradient of the logits, written as a whole. index: as the forward pass left it. */
    static void routeAdjoint(const Tensor& logits, const Tensor& index, const Tensor& adjWeights, bool normalised, Tensor& adjLogits, stream_t stream);

    /**
     * Rows of tokens to the places of their experts' rows: rows[places[t][j]] = input[t]; rows of zeros at the places of no expert.
     * \param input (tokens, channels) \param places (tokens, chosen) INT32, as group() returns them for the chosen experts of every token: those of a
     * permutation, -1 - place where there is no expert \param rows (tokens * chosen, channels)
     */
    static void dispatch(const Tensor& input, const Tensor& places, Tensor& rows, stream_t stream);
    /**
     * And back: output[t] = residual[t] + sum over j of weights[t][j] rows[places[t][j]], without the terms of no expert. It is the gradient of dispatch(),
     * too, with neither weights nor residual.
     * \param weights (tokens, chosen), of the rows' type or FLOAT, or undefined: 1 \param residual (tokens, channels), or undefined: 0
     */
    static void combine(const Tensor& rows, const Tensor& places, const Tensor& weights, const Tensor& residual, Tensor& output, stream_t stream);
    /**
     * Gradients, written as a whole, each of them may be undefined: not wanted. That of the residual is adjOutput. adjWeights: of the weights' type.
     * \param rows may be undefined where adjWeights is \param weights only adjRows depends on them
     */
    static void combineAdjoint(const Tensor& rows, const Tensor& places, const Tensor& weights, const Tensor& adjOutput, Tensor& adjRows,
                               Tensor& adjWeights, stream_t stream);

    /**
     * Numbers of 4 bits in blocks of 32 consecutive entries of a row with a common power of two (MXFP4 of the OCP Microscaling Formats specification
     * 1.0): sign, two bits of exponent and one of mantissa, to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale, halfway to the even code.
     * A block with an infinity or a NaN becomes NaN.
     * \param input (rows, columns) \param codes (rows, 16 * ceil(columns / 32)) UINT8, two codes a byte, the first in the low bits, zeros behind the last
     * \param scales (rows, ceil(columns / 32)) UINT8, the exponents plus 127; 255: NaN
     */
    static void quantiseMx4(const Tensor& input, Tensor& codes, Tensor& scales, stream_t stream);
    /** The values that codes and scales stand for, in the output's type (rows, columns). */
    static void valuesMx4(const Tensor& codes, const Tensor& scales, Tensor& output, stream_t stream);

    /** Bytes of 'memory' for mx4Linear() where input holds values; codes need none. */
    static size_t mx4LinearMemory(int64_t rows, int experts, int inputs, int outputs);
    /**
     * groupedLinear() with weights of 4 bits, on rows that are quantised by the call or have been before.
     * \param input (rows, inputs), or codes as of quantiseMx4() with inputScales \param inputScales undefined where input holds values
     * \param weight (experts, outputs, 16 * blocks) UINT8, codes of rows along the inputs \param scales (experts, outputs, blocks) UINT8
     * \param offsets as of groupedLinear(), or undefined: one expert has all rows \param bias (experts, outputs) of the output's type, or undefined
     * \param output (rows, outputs), of the input's type where that holds values
     */
    static void mx4Linear(const Tensor& input, const Tensor& inputScales, const Tensor& weight, const Tensor& scales, const Tensor& offsets,
                          const Tensor& bias, Tensor& output, void* memory, stream_t stream);

    /** Compiles the kernels for values of one precision into the kernel cache; needs no GPU. */
    static void precompile(Tensor::Precision precision);
};

QUICKMLP_NAMESPACE_END

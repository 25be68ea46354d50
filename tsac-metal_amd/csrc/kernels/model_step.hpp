// Launchers of a model's step around the attention over a paged cache: products of 8-bit integers
// with a scale for each token and each channel, the norms before and after a block, rotated
// positions on the way into the cache, and the rules on logits before drafts are verified.
#pragma once

#include "paged.hpp"

namespace tsac_hip
{
// Element types of rows.
enum class Type
{
    bf16,
    half,
    single
};

// ---- products of 8-bit integers (channel_linear.hip) ---------------------------
constexpr std::size_t channel_linear_max_inputs = 131071; // 128 x 128 x these stay below 2^31
constexpr std::size_t channel_linear_max_outputs = std::size_t(1) << 24;

// Weights in operand tiles: 32 outputs x 32 inputs, 16 bytes of row l % 32 from input 16 (l / 32) on
// for lane l; tiles [outputs / 32][inputs / 32], padded with zeros to whole tiles and to 128 inputs.
struct ChannelWeights
{
    const int8_t* values = nullptr;
    const float* scales = nullptr; // [outputs]
    const float* bias = nullptr;   // [outputs], or null
    int inputs = 0, outputs = 0;
};
std::size_t channel_tiles_bytes(std::size_t inputs, std::size_t outputs);
void channel_tiles(const int8_t* canonical, std::size_t inputs, std::size_t outputs, int8_t* tiled, hipStream_t stream);

struct ChannelRows
{
    const int8_t* q = nullptr;
    std::size_t q_stride = 0;
    const float* scales = nullptr; // [rows]
    void* out = nullptr;
    std::size_t out_stride = 0; // elements
    int rows = 0;
    Type type = Type::bf16;
};
void channel_linear(const ChannelWeights& weights, const ChannelRows& rows, hipStream_t stream);

// ---- norms around a block, tokens to 8 bits (block_norm.hip) -------------------
enum class Norm
{
    none,
    rms,
    layer
};
struct NormRule
{
    Norm norm = Norm::none;
    const void* gain = nullptr; // [width], or null: 1
    const void* bias = nullptr; // [width], or null: 0
};
constexpr std::size_t max_norm_width = 65536;
struct BlockRows
{
    int rows = 0, width = 0;
    Type type = Type::bf16;
    const void* input = nullptr;
    std::size_t input_stride = 0;
    NormRule post;
    const void* gate = nullptr;
    std::size_t gate_stride = 0; // 0: one row for all
    float scale = 1;
    Type residual_type = Type::bf16;
    const void* residual = nullptr;
    std::size_t residual_stride = 0;
    void* sum = nullptr; // of residual_type
    std::size_t sum_stride = 0;
    NormRule norm;
    float epsilon = 0;
    void* out = nullptr; // of type, or int8 where there are out_scales
    std::size_t out_stride = 0;
    float* out_scales = nullptr;
};
void block_norm(const BlockRows& rows, hipStream_t stream);

// ---- rotated positions on the way into the cache (rotary_append.hip) -----------
struct RotaryRows
{
    const uint16_t* query = nullptr; // [rows][heads][head_width]
    std::size_t query_stride = 0;
    uint16_t* out = nullptr; // rotated queries
    std::size_t out_stride = 0;
    int heads = 0;
    const uint16_t* keys = nullptr; // [rows][cache heads][head_width]
    const uint16_t* values = nullptr;
    std::size_t row_stride = 0;
    int rows = 0, max_rows = 0;
    const int* starts = nullptr;
    const int* positions = nullptr; // [rows], or null
    const uint64_t* mask = nullptr; // [rows][words], or null
    std::size_t words = 0;
    const double* frequencies = nullptr; // [rotary / 2], radians a position
    int rotary = 0;
    bool interleaved = false;
    float amplitude = 1;
};
void pages_append(const PagedCache& cache, int layer, const RotaryRows& rows, int* status, hipStream_t stream);

// ---- rules on logits (logits.hip) ----------------------------------------------
constexpr std::size_t max_alphabet_tokens = std::size_t(1) << 20;
struct LogitRules
{
    const int* starts = nullptr;
    int sequences = 0;
    const int* history = nullptr;
    std::size_t history_stride = 0;
    const int* history_lengths = nullptr;
    const int* prompt_lengths = nullptr;
    const int* tokens = nullptr;
    const uint64_t* mask = nullptr;
    std::size_t words = 0;
    const float* repetition = nullptr;
    const float* presence = nullptr;
    const float* frequency = nullptr;
    const int* bias_starts = nullptr;
    const int* bias_tokens = nullptr;
    const float* bias_values = nullptr;
    int biases = 0;
    const uint32_t* allowed = nullptr;
    std::size_t allowed_stride = 0;
    const float* temperature = nullptr;
};
struct LogitRows
{
    const void* logits = nullptr;
    std::size_t stride = 0;
    Type type = Type::bf16;
    int rows = 0, alphabet = 0;
    void* out = nullptr;
    std::size_t out_stride = 0;
    Type out_type = Type::bf16;
    bool probabilities = false;
};
std::size_t logits_workspace(const LogitRows& rows);
void adjust_logits(const LogitRows& rows, const LogitRules& rules, void* workspace, std::size_t bytes,
                   hipStream_t stream);
} // namespace tsac_hip

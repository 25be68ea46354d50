// Products of 8-bit integers with a scale for each token and for each output channel:
//
//   y[m][n] = (sum_k q[m][k] w[n][k]) * (s[m] c[n]) + b[n]
//
// The sum is exact in 32 bits, in any order and however it is divided, so that no variant, split or batch
// size changes a result: what is rounded is the sum as it becomes a float, the product of the two scales,
// theirs, the addition and the store.
//
// Weights lie in operand tiles, laid out once: 32 outputs x 32 inputs as the matrix instruction takes them,
// 16 bytes a lane, so that a wave's load is 1 KiB in one piece. Inputs are padded with zeros to 128 and outputs to
// 32, which is what makes odd sizes ordinary: whatever stands in an activation row behind its last input is
// multiplied with 0. Rows of activations are read as they lie; past the last row, or past the last piece of
// 16 bytes that has an input, the last one is read again.
//
// The first operand is the weights and the second the activations: lane l, register r of a 32 x 32 result
// holds output 8 (r / 4) + 4 (l / 32) + r % 4 of row l % 32.
#include "model_step.hpp"
#include "values.hpp"

#include <algorithm>

namespace tsac_hip
{
namespace
{
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int lanes = 64;
constexpr int tile = 32;         // outputs, inputs and rows of one instruction
constexpr int step = 128;        // inputs of one step
constexpr int slices = step / tile;
constexpr int tile_bytes = tile * tile;

struct Launch
{
    const int8_t* weights;
    const float* channel_scales;
    const float* bias;
    const int8_t* q;
    std::size_t q_stride;
    const float* token_scales;
    void* out;
    std::size_t out_stride;
    int rows, outputs, steps;
    int last_piece; // the last 16 bytes of a row that have an input
};

template <Type T> __device__ __forceinline__ value_t<T> finished(int sum, float token, float channel, float bias)
{
    return narrow<T>(float(sum) * (token * channel) + bias);
}

// ------------------------------------------------------------------ few rows
//
// What costs is reading the weights. A workgroup takes 32 outputs and up to Groups x 32 rows, each of its waves every
// Waves-th step of 128 inputs, from memory to registers; the waves' sums meet in LDS.
constexpr int narrow_waves = 8;

template <Type T, int Groups>
__global__ __launch_bounds__(narrow_waves * lanes) void narrow_kernel(Launch l)
{
    __shared__ int sums[narrow_waves * tile * (tile + 1)];
    const int lane = threadIdx.x % lanes, warp = threadIdx.x / lanes;
    const int n0 = blockIdx.x * tile, m0 = blockIdx.y * Groups * tile;
    v16i acc[Groups] = {};
    const int8_t* weights = l.weights + std::size_t(blockIdx.x) * l.steps * (slices * tile_bytes) + lane * 16;
    const int8_t* rows[Groups];
#pragma unroll
    for (int g = 0; g < Groups; ++g)
    {
        rows[g] = l.q + std::size_t(min(m0 + g * tile + lane % tile, l.rows - 1)) * l.q_stride;
    }
    for (int s = warp; s < l.steps; s += narrow_waves)
    {
        v4i w[slices], x[Groups][slices];
#pragma unroll
        for (int i = 0; i < slices; ++i)
        {
            w[i] = __builtin_nontemporal_load(
                reinterpret_cast<const v4i*>(weights + (std::size_t(s) * slices + i) * tile_bytes));
            const int at = min(s * step + i * tile + lane / tile * 16, l.last_piece);
#pragma unroll
            for (int g = 0; g < Groups; ++g)
            {
                x[g][i] = *reinterpret_cast<const v4i*>(rows[g] + at);
            }
        }
#pragma unroll
        for (int i = 0; i < slices; ++i)
        {
#pragma unroll
            for (int g = 0; g < Groups; ++g)
            {
                acc[g] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[i], x[g][i], acc[g], 0, 0, 0);
            }
        }
    }
    auto* out = static_cast<value_t<T>*>(l.out);
#pragma unroll
    for (int g = 0; g < Groups; ++g)
    {
        __syncthreads();
        int* mine = sums + (warp * tile + lane % tile) * (tile + 1) + 4 * (lane / tile);
#pragma unroll
        for (int r = 0; r < 16; ++r)
        {
            mine[8 * (r / 4) + r % 4] = acc[g][r];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < tile * tile; i += narrow_waves * lanes)
        {
            const int m = m0 + g * tile + i / tile, n = n0 + i % tile;
            if (m >= l.rows || n >= l.outputs)
            {
                continue;
            }
            int sum = 0;
#pragma unroll
            for (int w = 0; w < narrow_waves; ++w)
            {
                sum += sums[(w * tile + i / tile) * (tile + 1) + i % tile];
            }
            out[std::size_t(m) * l.out_stride + n] =
                finished<T>(sum, l.token_scales[m], l.channel_scales[n], l.bias ? l.bias[n] : 0.0f);
        }
    }
}

// 16 bytes a thread of the operand tiles.
__global__ void tiles_kernel(const int8_t* __restrict__ canonical, int inputs, int outputs, int steps,
                             int8_t* __restrict__ tiled, std::size_t pieces)
{
    const std::size_t piece = std::size_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (piece >= pieces)
    {
        return;
    }
    const int lane = piece % lanes;
    const std::size_t t = piece / lanes, across = std::size_t(steps) * slices;
    const std::size_t n = t / across * tile + lane % tile;
    const int k = int(t % across) * tile + lane / tile * 16;
    int8_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        v[i] = n < std::size_t(outputs) && k + i < inputs ? canonical[n * inputs + k + i] : int8_t(0);
    }
    __builtin_memcpy(tiled + 16 * piece, v, 16);
}

int steps_of(std::size_t inputs)
{
    return int((inputs + step - 1) / step);
}

template <Type T> void launch(const Launch& l, hipStream_t stream)
{
    const unsigned across = unsigned((l.outputs + tile - 1) / tile), groups = unsigned((l.rows + tile - 1) / tile);
    const auto go = [&](auto kernel, unsigned each)
    { kernel<<<dim3(across, (groups + each - 1) / each), narrow_waves * lanes, 0, stream>>>(l); };
    groups <= 1 ? go(narrow_kernel<T, 1>, 1) : groups <= 2 ? go(narrow_kernel<T, 2>, 2) : go(narrow_kernel<T, 4>, 4);
    check_hip(hipGetLastError(), "channel linear launch");
}
} // namespace

std::size_t channel_tiles_bytes(std::size_t inputs, std::size_t outputs)
{
    return (outputs + tile - 1) / tile * tile * std::size_t(steps_of(inputs)) * step;
}

void channel_tiles(const int8_t* canonical, std::size_t inputs, std::size_t outputs, int8_t* tiled, hipStream_t stream)
{
    const std::size_t pieces = channel_tiles_bytes(inputs, outputs) / 16;
    tiles_kernel<<<unsigned((pieces + 255) / 256), 256, 0, stream>>>(canonical, int(inputs), int(outputs),
                                                                     steps_of(inputs), tiled, pieces);
    check_hip(hipGetLastError(), "channel linear tiles launch");
}

std::size_t channel_linear_workspace(const ChannelWeights&, std::size_t)
{
    return 0;
}

void channel_linear(const ChannelWeights& weights, const ChannelRows& rows, void* workspace, std::size_t bytes,
                    hipStream_t stream)
{
    const std::size_t need = channel_linear_workspace(weights, std::size_t(rows.rows));
    require(bytes >= need && (workspace || !need), "channel linear: workspace too small");
    if (!rows.rows)
    {
        return;
    }
    const Launch l = {weights.values,
                      weights.scales,
                      weights.bias,
                      rows.q,
                      rows.q_stride,
                      rows.scales,
                      rows.out,
                      rows.out_stride,
                      rows.rows,
                      weights.outputs,
                      steps_of(std::size_t(weights.inputs)),
                      (weights.inputs - 1) / 16 * 16};
    switch (rows.type)
    {
    case Type::bf16: return launch<Type::bf16>(l, stream);
    case Type::half: return launch<Type::half>(l, stream);
    default: return launch<Type::single>(l, stream);
    }
}
} // namespace tsac_hip

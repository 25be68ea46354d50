// What a program does to a model's logits before it samples or verifies drafts: penalties for tokens that a
// sequence has had already, biases, a grammar's mask, and the softmax at a temperature.
//
//   x = logit; where the token was had: x / r if x > 0, else x r        (repetition r)
//   x = x - f count - (count > 0 ? g : 0)                                (frequency f, presence g)
//   x = x + bias;  -infinity where the grammar has no bit
//   p = e^((x - m) / t) / sum e^((x - m) / t),  m = max x;   t = 0: 1 at the lowest of the largest
//
// A drafted node has had its sequence's history and the tokens of the nodes on its line. No table of counts
// over the alphabet is kept or read: a workgroup counts the history's tokens of its own part of the alphabet in
// LDS, with integer additions, whose order does not matter, and the history lies in the caches for all of
// a sequence's rows. Biases are found by their place in the list, so that the last of a token's counts.
//
// A row of up to 32,768 tokens is one workgroup's, held in registers between its maximum, its sum and its
// store. Longer ones are divided: one launch leaves each part's maximum and sum, another joins them in
// ascending order and computes the part again.
#include "model_step.hpp"
#include "paged_device.hpp"
#include "values.hpp"

#include <algorithm>

namespace tsac_hip
{
namespace
{
constexpr int lanes = 64;
constexpr int most_threads = 512;
constexpr float minus_infinity = -__builtin_inff();
constexpr float log2e = 1.44269504f;

struct Part // of a row: what its softmax needs of it
{
    float top, sum;
    int first;  // the lowest place of the largest
    int broken; // one is not a number
};

struct Launch
{
    LogitRows rows;
    LogitRules rules;
    Part* parts;  // [rows][splits], or null
    int splits;   // of a row
    int width;    // tokens of a split
    bool aligned; // logits and outputs in whole vectors
};

// What a workgroup works on.
struct Place
{
    int row, sequence, node; // node: the row's place in its sequence
    int first, count;        // the sequence's rows
    int from, to;            // tokens
};

__device__ __forceinline__ bool place_of(const Launch& l, Place& p)
{
    p.row = blockIdx.x / l.splits;
    p.sequence = sequence_of(l.rules.starts, l.rules.sequences, p.row);
    p.count = rows_of(l.rules.starts, p.sequence, l.rows.rows, p.first);
    p.node = p.row - p.first;
    p.from = int(blockIdx.x % l.splits) * l.width;
    p.to = min(p.from + l.width, l.rows.alphabet);
    return p.node >= 0 && p.node < p.count;
}

// Counts of a chunk's tokens: twice the number of times they were said, and 1 more if the prompt had them.
struct Counts
{
    unsigned* said; // [chunk]
    unsigned* bias; // [chunk]: place in the list of biases and 1, or 0; null without biases
};

__device__ void count_chunk(const Launch& l, const Place& p, int base, int chunk, const Counts& counts)
{
    const LogitRules& r = l.rules;
    for (int i = threadIdx.x; i < chunk; i += blockDim.x)
    {
        counts.said[i] = 0;
        if (counts.bias)
        {
            counts.bias[i] = 0;
        }
    }
    __syncthreads();
    if (r.history)
    {
        const int held = int(min(r.history_stride, std::size_t(1) << 30));
        const int length = max(0, min(r.history_lengths[p.sequence], held));
        const int prompt = r.prompt_lengths ? max(0, min(r.prompt_lengths[p.sequence], length)) : 0;
        const int* history = r.history + p.sequence * r.history_stride;
        for (int i = threadIdx.x; i < length; i += blockDim.x)
        {
            const unsigned t = unsigned(history[i]) - unsigned(base);
            if (t < unsigned(chunk))
            {
                i < prompt ? (void)atomicOr(&counts.said[t], 1u) : (void)atomicAdd(&counts.said[t], 2u);
            }
        }
    }
    if (r.tokens)
    {
        const uint64_t* line = r.mask ? r.mask + std::size_t(p.row) * r.words : nullptr;
        const int nodes = r.mask ? int(min(std::size_t(p.count), 64 * r.words)) : p.node + 1;
        for (int j = threadIdx.x; j < nodes; j += blockDim.x)
        {
            const unsigned t = unsigned(r.tokens[p.first + j]) - unsigned(base);
            if (t < unsigned(chunk) && (!line || (line[j / 64] >> j % 64 & 1)))
            {
                atomicAdd(&counts.said[t], 2u);
            }
        }
    }
    if (counts.bias)
    {
        const int begin = max(0, min(r.bias_starts[p.sequence], r.biases));
        const int end = min(r.bias_starts[p.sequence + 1], r.biases);
        for (int i = begin + int(threadIdx.x); i < end; i += blockDim.x)
        {
            const unsigned t = unsigned(r.bias_tokens[i]) - unsigned(base);
            if (t < unsigned(chunk))
            {
                atomicMax(&counts.bias[t], unsigned(i) + 1);
            }
        }
    }
    __syncthreads();
}

struct Penalties
{
    float repetition, presence, frequency;
};

// Eight tokens from `token` on, `at` from the chunk's first.
template <Type T>
__device__ __forceinline__ void adjusted(const Launch& l, const Place& p, const Penalties& k, const Counts& counts, int token,
                                         int at, float (&x)[8])
{
    const auto* logits = static_cast<const value_t<T>*>(l.rows.logits) + std::size_t(p.row) * l.rows.stride;
    const int count = p.to - token;
    load8<T>(logits + token, count, l.aligned, minus_infinity, x);
    const uint4 low = *reinterpret_cast<const uint4*>(counts.said + at), high = *reinterpret_cast<const uint4*>(counts.said + at + 4);
    const unsigned said[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        if (said[e] && e < count)
        {
            const float times = float(said[e] >> 1);
            x[e] = x[e] > 0.0f ? x[e] / k.repetition : x[e] * k.repetition;
            x[e] -= k.frequency * times;
            x[e] -= times > 0.0f ? k.presence : 0.0f;
        }
    }
    if (counts.bias)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            if (const unsigned i = counts.bias[at + e]; i && e < count)
            {
                x[e] += l.rules.bias_values[i - 1];
            }
        }
    }
    if (l.rules.allowed && count > 0)
    {
        // Tokens come in eights, so that their bits are in one word.
        const uint32_t word = l.rules.allowed[p.row * l.rules.allowed_stride + token / 32] >> token % 32;
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            x[e] = word >> e & 1 ? x[e] : minus_infinity;
        }
    }
}

template <class Join, class V> __device__ __forceinline__ V joined(V value, V* shared, Join join)
{
#pragma unroll
    for (int step = 1; step < lanes; step *= 2)
    {
        value = join(value, __shfl_xor(value, step));
    }
    const int waves = int(blockDim.x) / lanes;
    if (waves > 1)
    {
        __syncthreads(); // the last one's values have been read
        if (threadIdx.x % lanes == 0)
        {
            shared[threadIdx.x / lanes] = value;
        }
        __syncthreads();
        value = shared[0];
        for (int i = 1; i < waves; ++i)
        {
            value = join(value, shared[i]);
        }
    }
    return value;
}

struct Exchange
{
    float f[most_threads / lanes];
    int i[most_threads / lanes];
};

// e^((x - top) / t) as a power of two. -infinity gives 0, what is not a number and +infinity no number.
__device__ __forceinline__ float weight(float x, float top, float per_log2)
{
    return x == minus_infinity ? 0.0f : __builtin_amdgcn_exp2f((x - top) * per_log2);
}

// A temperature's factor; so small that it overflows, it is the largest number: 0 times it is still 0.
__device__ __forceinline__ float factor_of(float temperature)
{
    return __builtin_fminf(log2e / temperature, 3.402823466e38f);
}

// What is known of values held in registers: the largest and its lowest place, the sum of weights.
template <int Vectors>
__device__ __forceinline__ Part part_of(const float (&x)[Vectors][8], int from, float temperature, Exchange& shared)
{
    Part part;
    float top = minus_infinity;
#pragma unroll
    for (int i = 0; i < Vectors; ++i)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            top = __builtin_fmaxf(top, x[i][e]); // the number, of a number and none
        }
    }
    part.top = top = joined(top, shared.f, [](float a, float b) { return __builtin_fmaxf(a, b); });
    part.sum = 0.0f;
    part.first = 1 << 30;
    part.broken = 0;
    if (temperature > 0.0f)
    {
        const float factor = factor_of(temperature);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                sum += weight(x[i][e], top, factor);
            }
        }
        part.sum = joined(sum, shared.f, [](float a, float b) { return a + b; });
    }
    else
    {
        int first = 1 << 30, broken = 0;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                const int token = from + 8 * (i * int(blockDim.x) + int(threadIdx.x)) + e;
                first = x[i][e] == top && top > minus_infinity ? min(first, token) : first;
                broken |= x[i][e] != x[i][e];
            }
        }
        part.first = joined(first, shared.i, [](int a, int b) { return min(a, b); });
        part.broken = joined(broken, shared.i, [](int a, int b) { return a | b; });
    }
    return part;
}

// A later part joined to what is in front of it.
__device__ __forceinline__ Part join(const Part& a, const Part& b, float temperature)
{
    Part r;
    r.top = __builtin_fmaxf(a.top, b.top);
    r.first = a.top >= b.top ? a.first : b.first;
    r.broken = a.broken | b.broken;
    r.sum = 0.0f;
    if (temperature > 0.0f)
    {
        const float factor = factor_of(temperature);
        // A part without a number above -infinity has a sum of 0, or none that is a number.
        const float wa = a.top == r.top ? 1.0f : weight(a.top, r.top, factor);
        const float wb = b.top == r.top ? 1.0f : weight(b.top, r.top, factor);
        r.sum = (a.top == minus_infinity ? a.sum : a.sum * wa) + (b.top == minus_infinity ? b.sum : b.sum * wb);
    }
    return r;
}

enum class Step
{
    adjust, // x as it is
    whole,  // the softmax of a row in one part
    parts,  // each part's maximum and sum
    finish  // the softmax from these
};

template <Type T, Type O, Step S, int Vectors>
__global__ __launch_bounds__(most_threads) void logits_kernel(Launch l)
{
    extern __shared__ unsigned memory[]; // the counts of a chunk, and its biases
    __shared__ Exchange shared;
    Place p;
    if (!place_of(l, p))
    {
        return;
    }
    const int chunk = 8 * blockDim.x;
    const Counts counts = {memory, l.rules.bias_starts ? memory + chunk : nullptr};
    const LogitRules& r = l.rules;
    const Penalties k = {r.repetition ? r.repetition[p.sequence] : 1.0f, r.presence ? r.presence[p.sequence] : 0.0f,
                         r.frequency ? r.frequency[p.sequence] : 0.0f};
    float x[Vectors][8];
#pragma unroll
    for (int i = 0; i < Vectors; ++i)
    {
        const int base = p.from + i * chunk;
        if (i)
        {
            __syncthreads(); // the last chunk's counts have been read
        }
        count_chunk(l, p, base, chunk, counts);
        adjusted<T>(l, p, k, counts, base + 8 * int(threadIdx.x), 8 * int(threadIdx.x), x[i]);
    }
    float scale = 1.0f, top = 0.0f, factor = 0.0f;
    Part part = {};
    bool soft = false;
    if constexpr (S != Step::adjust)
    {
        const float temperature = r.temperature ? r.temperature[p.sequence] : 1.0f;
        soft = temperature > 0.0f;
        if constexpr (S == Step::finish)
        {
            const Part* parts = l.parts + std::size_t(p.row) * l.splits;
            part = parts[0];
            for (int i = 1; i < l.splits; ++i)
            {
                part = join(part, parts[i], temperature);
            }
        }
        else
        {
            part = part_of<Vectors>(x, p.from, temperature, shared);
        }
        if constexpr (S == Step::parts)
        {
            if (threadIdx.x == 0)
            {
                l.parts[blockIdx.x] = part;
            }
            return;
        }
        top = part.top;
        factor = factor_of(temperature);
        scale = part.sum == 0.0f ? 0.0f : 1.0f / part.sum;
    }
    auto* out = static_cast<value_t<O>*>(l.rows.out) + std::size_t(p.row) * l.rows.out_stride;
#pragma unroll
    for (int i = 0; i < Vectors; ++i)
    {
        const int token = p.from + i * chunk + 8 * int(threadIdx.x);
        if (token >= p.to)
        {
            break;
        }
        if constexpr (S != Step::adjust)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                x[i][e] = soft          ? weight(x[i][e], top, factor) * scale
                          : part.broken ? __uint_as_float(0x7fc00000u)
                                        : (token + e == part.first ? 1.0f : 0.0f);
            }
        }
        store8<O>(out + token, p.to - token, l.aligned, x[i]);
    }
}

// Threads and eights a thread, of a row or a part of one.
struct Shape
{
    int threads, vectors, splits, width;
};
Shape shape_of(int alphabet)
{
    const int eights = (alphabet + 7) / 8;
    Shape s;
    s.threads = std::min(most_threads, (eights + lanes - 1) / lanes * lanes);
    const int rounds = (eights + s.threads - 1) / s.threads;
    s.vectors = rounds <= 1 ? 1 : rounds <= 2 ? 2 : rounds <= 4 ? 4 : 8;
    s.width = 8 * s.threads * s.vectors;
    s.splits = (alphabet + s.width - 1) / s.width;
    return s;
}

template <Type T, Type O, Step S> void launch(const Launch& l, const Shape& s, hipStream_t stream)
{
    const unsigned grid = unsigned(l.rows.rows) * unsigned(l.splits);
    const std::size_t bytes = std::size_t(8 * s.threads) * 4 * (l.rules.bias_starts ? 2 : 1);
    const auto go = [&](auto kernel) { kernel<<<grid, unsigned(s.threads), bytes, stream>>>(l); };
    s.vectors == 1   ? go(logits_kernel<T, O, S, 1>)
    : s.vectors == 2 ? go(logits_kernel<T, O, S, 2>)
    : s.vectors == 4 ? go(logits_kernel<T, O, S, 4>)
                     : go(logits_kernel<T, O, S, 8>);
    check_hip(hipGetLastError(), "logits launch");
}

template <Type T, Type O> void steps(const Launch& l, const Shape& s, hipStream_t stream)
{
    if (!l.rows.probabilities)
    {
        launch<T, O, Step::adjust>(l, s, stream);
    }
    else if (s.splits == 1)
    {
        launch<T, O, Step::whole>(l, s, stream);
    }
    else
    {
        launch<T, O, Step::parts>(l, s, stream);
        launch<T, O, Step::finish>(l, s, stream);
    }
}
} // namespace

std::size_t logits_workspace(const LogitRows& rows)
{
    const Shape s = shape_of(rows.alphabet);
    return rows.probabilities && s.splits > 1 ? std::size_t(rows.rows) * s.splits * sizeof(Part) : 0;
}

void adjust_logits(const LogitRows& rows, const LogitRules& rules, void* workspace, std::size_t bytes,
                   hipStream_t stream)
{
    if (!rows.rows || !rules.sequences)
    {
        return;
    }
    const Shape s = shape_of(rows.alphabet);
    require(std::size_t(rows.rows) * s.splits < (std::size_t(1) << 31), "logits: too many rows");
    require(bytes >= logits_workspace(rows) && (workspace || !logits_workspace(rows)), "logits: workspace too small");
    const auto whole = [](const void* pointer, std::size_t stride, Type type)
    { return reinterpret_cast<std::uintptr_t>(pointer) % 16 == 0 && stride * (type == Type::single ? 4 : 2) % 16 == 0; };
    const Launch l = {rows, rules, static_cast<Part*>(workspace), s.splits, s.width,
                      whole(rows.logits, rows.stride, rows.type) && whole(rows.out, rows.out_stride, rows.out_type)};
    const auto to = [&](auto in)
    {
        constexpr Type T = decltype(in)::value;
        switch (rows.out_type)
        {
        case Type::bf16: return steps<T, Type::bf16>(l, s, stream);
        case Type::half: return steps<T, Type::half>(l, s, stream);
        default: return steps<T, Type::single>(l, s, stream);
        }
    };
    switch (rows.type)
    {
    case Type::bf16: return to(std::integral_constant<Type, Type::bf16>{});
    case Type::half: return to(std::integral_constant<Type, Type::half>{});
    default: return to(std::integral_constant<Type, Type::single>{});
    }
}
} // namespace tsac_hip

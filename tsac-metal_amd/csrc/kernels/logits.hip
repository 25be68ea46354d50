// What a program does to a model's logits before it samples or verifies drafts: penalties for tokens that a
// sequence has had already, biases, a grammar's mask, and the softmax at a temperature.
//
//   x = logit; where the token was had: x / r if x > 0, else x r (repetition r)
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
// ascending order and computes the part again. Logits are asked for before anything is counted.
//
// 902 rows of 32,000 with a history of 4,093, BF16 to half, six batches in turn: 62 us, where a copy of their bytes
// takes 25; without rules 40, adjusted without a softmax 48 (32 without rules). What is left is some 30 instructions a
// token and the waits between the phases of two workgroups a unit. Rows in 1,024 threads left one workgroup a unit or
// spilled (100 us); spilled registers alone cost 5 us, penalties by branches 25, since most waves have a token of the
// history in each place.
// For results of 32 bits, quotients are products with factors of two floats, each rounded once (24 rows of 128,001: 1 us of 27; with
// factors of one float, probabilities far below the largest were off by twice as much).
#include "lanes.hpp"
#include "model_step.hpp"
#include "paged_device.hpp"
#include "values.hpp"

#include <algorithm>
#include <type_traits>

namespace tsac_hip
{
namespace
{
constexpr int lanes = 64;
constexpr int units = 256; // of the card: a workspace is asked for where there is none, too
constexpr int most_threads = 512;
constexpr int most_vectors = 8; // eights of a thread
// Tokens of the history that a thread has in flight.
constexpr int asked_for(int vectors)
{
    return vectors <= 2 ? 16 : vectors <= 4 ? 8 : 4;
}
constexpr float minus_infinity = -__builtin_inff();
constexpr float log2e = 0x1.715476p0f, log2e_rest = 0x1.4ae0cp-26f;
constexpr float little = 0x1p-126f;

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
    bool counted; // there is a history, or there are drafted tokens
};

// What a token has had, in a word of LDS or two: twice the times it was said and 1 more if the prompt has it; and the
// place in its sequence's list of biases and 1, or 0. One word has 16 bits of each, where no count reaches 2^15 and no
// place 2^16.
template <bool Narrow> struct Words
{
    static constexpr int each = Narrow ? 1 : 2;
    unsigned* memory; // counts (and biases), then the biases of wide words
    int chunk;

    __device__ __forceinline__ void clear(int at) const
    {
#pragma unroll
        for (int i = 0; i < each; ++i)
        {
            *reinterpret_cast<uint4*>(memory + i * chunk + at) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(memory + i * chunk + at + 4) = make_uint4(0, 0, 0, 0);
        }
    }
    // Before counts are added to the same words.
    __device__ __forceinline__ void bias(unsigned token, unsigned place) const
    {
        atomicMax(memory + (Narrow ? 0 : chunk) + token, Narrow ? place << 16 : place);
    }
    __device__ __forceinline__ void count(unsigned token, bool said) const
    {
        said ? (void)atomicAdd(memory + token, 2u) : (void)atomicOr(memory + token, 1u);
    }
    __device__ __forceinline__ void read(int at, unsigned (&said)[8], unsigned (&bias)[8]) const
    {
        eight(memory + at, said);
        if constexpr (!Narrow)
        {
            eight(memory + chunk + at, bias);
        }
        else
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                bias[e] = said[e];
                said[e] &= 0xffffu;
            }
        }
    }
    // Whether one of eight has a bias, and its place.
    static __device__ __forceinline__ bool biased(const unsigned (&bias)[8])
    {
        const unsigned any = bias[0] | bias[1] | bias[2] | bias[3] | bias[4] | bias[5] | bias[6] | bias[7];
        return Narrow ? any > 0xffffu : any != 0;
    }
    static __device__ __forceinline__ unsigned place(unsigned bias)
    {
        return Narrow ? bias >> 16 : bias;
    }
    static __device__ __forceinline__ void eight(const unsigned* from, unsigned (&to)[8])
    {
        const uint4 a = *reinterpret_cast<const uint4*>(from), b = *reinterpret_cast<const uint4*>(from + 4);
        to[0] = a.x, to[1] = a.y, to[2] = a.z, to[3] = a.w;
        to[4] = b.x, to[5] = b.y, to[6] = b.z, to[7] = b.w;
    }
};

template <class V, class Join> __device__ __forceinline__ V joined(V value, V* shared, Join join)
{
    value = over_lanes(value, join);
    const int waves = int(blockDim.x) / lanes;
    if (waves > 1)
    {
        lds_barrier(); // the last one's values have been read
        if (threadIdx.x % lanes == 0)
        {
            shared[threadIdx.x / lanes] = value;
        }
        lds_barrier();
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

// A factor as the sum of two floats, so that a product with it is rounded once: a rounded factor would be off in one direction
// for all tokens of a row. Results of 16 bits, whose own rounding is at least 2^7 times what that makes of them, take the first
// float alone.
struct Factor
{
    float high, low;
};
template <bool Fine> __device__ __forceinline__ float times(float x, const Factor& by)
{
    return Fine ? __builtin_fmaf(x, by.high, x * by.low) : x * by.high;
}

// (a + rest) / b of numbers above 0, from a / b. Both parts are above 0, so that infinities stay what they are; where a / b is far
// out there is no second one to speak of.
template <bool Fine> __device__ __forceinline__ Factor divided(float quotient, float a, float rest, float b)
{
    const bool near = Fine && quotient > 0x1p-100f && quotient < 0x1p100f;
    const float high = near ? __uint_as_float(__float_as_uint(quotient) - 1) : quotient;
    const float low = (__builtin_fmaf(-high, b, a) + rest) * __builtin_amdgcn_rcpf(b);
    return {high, near ? __builtin_fmaxf(low, little) : little};
}

// e^((x - top) / t) as a power of two, of a finite top. -infinity gives 0, what is not a number and +infinity no number.
template <bool Fine> __device__ __forceinline__ float weight(float x, float top, const Factor& per_log2)
{
    return __builtin_amdgcn_exp2f(times<Fine>(x - top, per_log2));
}

// What stands for the largest of a row in which nothing is above -infinity: its weights are 0, or no numbers.
__device__ __forceinline__ float reference(float top)
{
    return top == minus_infinity ? 0.0f : top;
}

// A temperature's factor; where that would be infinite the largest number, which times 0 is still 0, where it would be 0 a
// small one, which times -infinity is still that.
template <bool Fine> __device__ __forceinline__ Factor factor_of(float temperature)
{
    const float quotient = __builtin_fmaxf(__builtin_fminf(log2e / temperature, 0x1.fffffep127f), 0x1p-126f);
    return divided<Fine>(quotient, log2e, log2e_rest, temperature);
}

// What is known of values held in registers: the largest and its lowest place, the sum of weights, which stand in the
// values' place afterwards.
template <bool Fine, int Vectors>
__device__ __forceinline__ Part part_of(float (&x)[Vectors][8], int from, bool soft, const Factor& factor, Exchange& shared)
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
    if (soft)
    {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                x[i][e] = weight<Fine>(x[i][e], reference(top), factor);
                sum += x[i][e];
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
template <bool Fine> __device__ __forceinline__ Part join(const Part& a, const Part& b, bool soft, const Factor& factor)
{
    Part r;
    r.top = __builtin_fmaxf(a.top, b.top);
    r.first = a.top >= b.top ? a.first : b.first;
    r.broken = a.broken | b.broken;
    r.sum = 0.0f;
    if (soft)
    {
        // A part without a number above -infinity has a sum of 0, or none that is a number.
        const float wa = a.top == r.top ? 1.0f : weight<Fine>(a.top, r.top, factor);
        const float wb = b.top == r.top ? 1.0f : weight<Fine>(b.top, r.top, factor);
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

// Eight logits as they are asked for.
template <bool Wide> struct Raw
{
    uint4 v[Wide ? 2 : 1];
};

// Rounds: how often LDS holds the words of a part of the workgroup's tokens. Wide: logits of 32 bits; Fine: results of 32 bits.
template <Step S, bool Wide, int Vectors, int Rounds, bool Narrow, bool Fine>
__global__ __launch_bounds__(most_threads, 4) void logits_kernel(Launch l)
{
    constexpr int held = Vectors / Rounds; // eights of a thread in a round
    constexpr int asked = asked_for(Vectors);
    extern __shared__ __attribute__((aligned(16))) unsigned memory[];
    __shared__ Exchange shared;
    const int thread = threadIdx.x, threads = blockDim.x;
    const int row = blockIdx.x / l.splits, from = int(blockIdx.x - row * l.splits) * l.width;
    const int to = min(from + l.width, l.rows.alphabet);
    const LogitRules& r = l.rules;
    const int s = __builtin_amdgcn_readfirstlane(sequence_of(r.starts, r.sequences, row));
    int first;
    const int count = rows_of(r.starts, s, l.rows.rows, first), node = row - first;
    if (node < 0 || node >= count)
    {
        return;
    }

    // Everything that is read is asked for at once, in the order of its use, in which loads complete: the first biases,
    // what of the history and of the line's nodes a thread can hold, the logits, the grammar's bits.
    const int bias_begin = r.bias_starts ? max(0, min(r.bias_starts[s], r.biases)) : 0;
    const int bias_end = r.bias_starts ? min(r.bias_starts[s + 1], r.biases) : 0;
    const int bias_token = bias_begin + thread < bias_end ? r.bias_tokens[bias_begin + thread] : -1;
    int length = 0, prompt = 0;
    int past[asked];
    const int* const history = r.history + std::size_t(s) * r.history_stride;
    if (r.history)
    {
        const int room = int(min(r.history_stride, std::size_t(1) << 30));
        length = max(0, min(r.history_lengths[s], room));
        prompt = r.prompt_lengths ? max(0, min(r.prompt_lengths[s], length)) : 0;
#pragma unroll
        for (int i = 0; i < asked; ++i)
        {
            const int at = thread + i * threads;
            past[i] = at < length ? history[at] : -1;
        }
    }
    const uint64_t* const line = r.mask ? r.mask + std::size_t(row) * r.words : nullptr;
    const int nodes = !r.tokens ? 0 : r.mask ? int(min(std::size_t(count), 64 * r.words)) : node + 1;
    int drafted = -1;
    uint64_t lined = ~uint64_t(0);
    if (thread < nodes)
    {
        drafted = r.tokens[first + thread];
        lined = line ? line[thread / 64] : lined;
    }
    const std::size_t begin = std::size_t(row) * l.rows.stride;
    Raw<Wide> raw[Vectors];
    // Tokens come in eights, so that their bits are a byte. Of eight eights they are read where they are used: there is no
    // register left.
    constexpr bool early = Vectors < most_vectors;
    const auto* const bits = reinterpret_cast<const uint8_t*>(r.allowed + std::size_t(row) * r.allowed_stride);
    uint8_t grammar[Vectors];
#pragma unroll
    for (int i = 0; i < Vectors; ++i)
    {
        const int token = from + 8 * (i * threads + thread);
        if (l.aligned && token + 8 <= to)
        {
            raw[i] = *reinterpret_cast<const Raw<Wide>*>(static_cast<const char*>(l.rows.logits) +
                                                         (begin + token) * (Wide ? 4 : 2));
        }
        if (early && r.allowed && token < to)
        {
            grammar[i] = bits[token / 8];
        }
    }

    const float repetition = r.repetition ? r.repetition[s] : 1.0f, presence = r.presence ? r.presence[s] : 0.0f;
    const float frequency = r.frequency ? r.frequency[s] : 0.0f;
    const float temperature = S != Step::adjust && r.temperature ? r.temperature[s] : 1.0f;
    const bool soft = temperature > 0.0f;
    const Factor factor = factor_of<Fine>(temperature);
    const Factor inverse = divided<Fine>(1.0f / __builtin_fabsf(repetition), 1.0f, 0.0f, __builtin_fabsf(repetition));
    const float reciprocal = __builtin_copysignf(inverse.high, repetition);
    const float reciprocal_rest = __builtin_copysignf(inverse.low, repetition);
    const bool edited = l.counted || bias_begin < bias_end;
    const Words<Narrow> words = {memory, 8 * threads * held};
    float x[Vectors][8];
#pragma unroll
    for (int round = 0; round < Rounds; ++round)
    {
        const int base = from + round * words.chunk;
        const unsigned inside = unsigned(max(0, min(words.chunk, to - base))); // tokens of the alphabet among its words
        if (edited)
        {
#pragma unroll
            for (int i = 0; i < held; ++i)
            {
                words.clear(8 * (i * threads + thread)); // the words that this thread reads
            }
            lds_barrier();
            if (bias_begin < bias_end)
            {
                const auto add = [&](int token, int i)
                {
                    const unsigned t = unsigned(token) - unsigned(base);
                    if (t < inside)
                    {
                        words.bias(t, unsigned(i - bias_begin) + 1);
                    }
                };
                if (const int i = bias_begin + thread; i < bias_end)
                {
                    add(bias_token, i);
                }
                for (int i = bias_begin + threads + thread; i < bias_end; i += threads)
                {
                    add(r.bias_tokens[i], i);
                }
                lds_barrier();
            }
            const auto had = [&](int token, bool said)
            {
                const unsigned t = unsigned(token) - unsigned(base);
                if (t < inside)
                {
                    words.count(t, said);
                }
            };
            if (r.history)
            {
#pragma unroll
                for (int i = 0; i < asked; ++i)
                {
                    if (const int at = thread + i * threads; at < length)
                    {
                        had(past[i], at >= prompt);
                    }
                }
                for (int later = asked * threads; later < length; later += asked * threads)
                {
                    int more[asked];
#pragma unroll
                    for (int i = 0; i < asked; ++i)
                    {
                        const int at = later + thread + i * threads;
                        more[i] = at < length ? history[at] : -1;
                    }
#pragma unroll
                    for (int i = 0; i < asked; ++i)
                    {
                        if (const int at = later + thread + i * threads; at < length)
                        {
                            had(more[i], at >= prompt);
                        }
                    }
                }
            }
            if (thread < nodes && (lined >> thread % 64 & 1))
            {
                had(drafted, true);
            }
            for (int j = thread + threads; j < nodes; j += threads)
            {
                if (!line || (line[j / 64] >> j % 64 & 1))
                {
                    had(r.tokens[first + j], true);
                }
            }
            lds_barrier();
        }
#pragma unroll
        for (int h = 0; h < held; ++h)
        {
            const int i = round * held + h, token = from + 8 * (i * threads + thread), there = to - token;
            const auto widened = [&](auto type)
            {
                constexpr Type T = decltype(type)::value;
                if (l.aligned && there >= 8)
                {
                    const Eight<T> eight = __builtin_bit_cast(Eight<T>, raw[i]);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                    {
                        x[i][e] = widen<T>(eight.v[e]);
                    }
                }
                else
                {
                    load8<T>(static_cast<const value_t<T>*>(l.rows.logits) + begin + token, there, false, minus_infinity, x[i]);
                }
            };
            if constexpr (Wide)
            {
                widened(std::integral_constant<Type, Type::single>{});
            }
            else
            {
                l.rows.type == Type::bf16 ? widened(std::integral_constant<Type, Type::bf16>{})
                                          : widened(std::integral_constant<Type, Type::half>{});
            }
            if (edited)
            {
                unsigned said[8], bias[8];
                words.read(8 * (h * threads + thread), said, bias);
                // Without branches: with a long history most waves have a token of it in each place. Past the last token
                // nothing is counted, and -infinity stays what it is.
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    const float count = float(said[e] >> 1);
                    const bool above = x[i][e] > 0.0f;
                    const float rest = Fine && said[e] && above ? x[i][e] * reciprocal_rest : 0.0f;
                    const float by = said[e] ? (above ? reciprocal : repetition) : 1.0f;
                    x[i][e] = Fine ? __builtin_fmaf(x[i][e], by, rest) : x[i][e] * by;
                    x[i][e] = __builtin_fmaf(-frequency, count, x[i][e]);
                    x[i][e] = __builtin_fmaf(-presence, __builtin_fminf(count, 1.0f), x[i][e]);
                }
                if (words.biased(bias))
                {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                    {
                        if (const unsigned place = words.place(bias[e]); place)
                        {
                            x[i][e] += r.bias_values[bias_begin + int(place) - 1];
                        }
                    }
                }
            }
            if (r.allowed && there > 0)
            {
                const unsigned byte = early ? grammar[i] : bits[token / 8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    const int keep = int(byte << (31 - e)) >> 31; // all bits or none
                    x[i][e] = __uint_as_float((__float_as_uint(x[i][e]) & keep) | (0xff800000u & ~keep));
                }
            }
        }
    }

    Factor scale = {};
    float top = 0.0f;
    Part part = {};
    if constexpr (S != Step::adjust)
    {
        if constexpr (S == Step::finish)
        {
            const Part* const parts = l.parts + std::size_t(row) * l.splits;
            part = parts[0];
            for (int i = 1; i < l.splits; ++i)
            {
                part = join<Fine>(part, parts[i], soft, factor);
            }
        }
        else
        {
            part = part_of<Fine>(x, from, soft, factor, shared);
        }
        if constexpr (S == Step::parts)
        {
            if (thread == 0)
            {
                l.parts[blockIdx.x] = part;
            }
            return;
        }
        top = reference(part.top);
        if (part.sum != 0.0f)
        {
            scale.high = 1.0f / part.sum;
            scale.low = __builtin_fmaf(-scale.high, part.sum, 1.0f) * scale.high;
        }
    }
    const std::size_t at = std::size_t(row) * l.rows.out_stride;
#pragma unroll
    for (int i = 0; i < Vectors; ++i)
    {
        const int token = from + 8 * (i * threads + thread);
        if (token >= to)
        {
            break;
        }
        if constexpr (S != Step::adjust)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                if (soft)
                {
                    x[i][e] = times<Fine>(S == Step::whole ? x[i][e] : weight<Fine>(x[i][e], top, factor), scale);
                }
                else
                {
                    x[i][e] = part.broken ? __uint_as_float(0x7fc00000u) : token + e == part.first ? 1.0f : 0.0f;
                }
            }
        }
        const auto store = [&](auto type)
        {
            constexpr Type T = decltype(type)::value;
            store8<T>(static_cast<value_t<T>*>(l.rows.out) + at + token, to - token, l.aligned, x[i]);
        };
        if constexpr (Fine)
        {
            store(std::integral_constant<Type, Type::single>{});
        }
        else
        {
            l.rows.out_type == Type::bf16 ? store(std::integral_constant<Type, Type::bf16>{})
                                          : store(std::integral_constant<Type, Type::half>{});
        }
    }
}

// Threads, eights of a thread, parts of a row.
struct Shape
{
    int threads, vectors, splits, width;
};
Shape shape_of(const LogitRows& rows, std::size_t history)
{
    const int eights = (rows.alphabet + 7) / 8;
    Shape s;
    // Threads for the tokens or, where these are few and the history is long, for that.
    const std::size_t wanted = std::max(std::size_t(eights), std::min<std::size_t>(history / asked_for(1), most_threads));
    s.threads = int(std::min<std::size_t>(most_threads, (wanted + lanes - 1) / lanes * lanes));
    const int rounds = (eights + s.threads - 1) / s.threads;
    s.vectors = rounds <= 1 ? 1 : rounds <= 2 ? 2 : rounds <= 4 ? 4 : most_vectors;
    if (rounds > most_vectors || !rows.probabilities)
    {
        // Parts, then: of four eights a thread (902 rows of 32,000, adjusted alone, one batch again and again: 40 us, of eight
        // 51, of two 49), of fewer where rows are few, for a workgroup a unit at least, if there are as many (24 rows of
        // 128,001 in parts of 16,384, 8,192 and 4,096 tokens: 27.4, 26.9 and 43 us).
        s.vectors = std::min(s.vectors, 4);
        while (s.vectors > 1 && std::size_t(rows.rows) * ((rounds + s.vectors - 1) / s.vectors) < std::size_t(units))
        {
            s.vectors /= 2;
        }
    }
    s.width = 8 * s.threads * s.vectors;
    s.splits = (rows.alphabet + s.width - 1) / s.width;
    return s;
}

template <Step S> void launch(const Launch& l, const Shape& s, bool narrow, hipStream_t stream)
{
    const unsigned grid = unsigned(l.rows.rows) * unsigned(l.splits);
    const auto go = [&](auto kernel, int held, int each)
    {
        const std::size_t bytes = std::size_t(8 * s.threads) * held * each * 4;
        kernel<<<grid, unsigned(s.threads), bytes, stream>>>(l);
    };
    const auto of = [&](auto wide, auto few, auto fine)
    {
        constexpr bool W = decltype(wide)::value, N = decltype(few)::value, F = decltype(fine)::value;
        constexpr int each = Words<N>::each;
        // Words of at most 64 KiB at a time, so that a unit has two workgroups.
        constexpr int most = N ? 4 : 2;
        if constexpr (S == Step::whole)
        {
            if (s.vectors == most_vectors)
            {
                return go(logits_kernel<S, W, most_vectors, most_vectors / most, N, F>, most, each);
            }
        }
        s.vectors == 1   ? go(logits_kernel<S, W, 1, 1, N, F>, 1, each)
        : s.vectors == 2 ? go(logits_kernel<S, W, 2, 1, N, F>, 2, each)
                         : go(logits_kernel<S, W, 4, 4 / most, N, F>, most, each);
    };
    const auto chosen = [](bool yes, auto next) { yes ? next(std::true_type{}) : next(std::false_type{}); };
    chosen(l.rows.type == Type::single,
           [&](auto wide)
           {
               chosen(narrow,
                      [&](auto few)
                      { chosen(l.rows.out_type == Type::single, [&](auto fine) { of(wide, few, fine); }); });
           });
    check_hip(hipGetLastError(), "logits launch");
}
} // namespace

// Of the narrowest parts: how many parts a row has falls where there are more rows, and a workspace that a program keeps for
// its largest batch has to do for smaller ones.
std::size_t logits_workspace(const LogitRows& rows)
{
    if (!rows.probabilities || shape_of(rows, 0).splits == 1) // a history changes the threads of rows in one part alone
    {
        return 0;
    }
    constexpr std::size_t narrowest = 8 * most_threads;
    return std::size_t(rows.rows) * ((rows.alphabet + narrowest - 1) / narrowest) * sizeof(Part);
}

void adjust_logits(const LogitRows& rows, const LogitRules& rules, void* workspace, std::size_t bytes,
                   hipStream_t stream)
{
    if (!rows.rows || !rules.sequences)
    {
        return;
    }
    const std::size_t history = rules.history ? rules.history_stride : 0;
    const Shape s = shape_of(rows, history);
    // 2^32 work-items are a launch's limit.
    require(std::size_t(rows.rows) * s.splits < (std::size_t(1) << 32) / s.threads, "logits: too many rows");
    require(bytes >= logits_workspace(rows) && (workspace || !logits_workspace(rows)), "logits: workspace too small");
    const auto whole = [](const void* pointer, std::size_t stride, Type type)
    { return reinterpret_cast<std::uintptr_t>(pointer) % 16 == 0 && stride * (type == Type::single ? 4 : 2) % 16 == 0; };
    const Launch l = {rows,
                      rules,
                      static_cast<Part*>(workspace),
                      s.splits,
                      s.width,
                      whole(rows.logits, rows.stride, rows.type) && whole(rows.out, rows.out_stride, rows.out_type),
                      rules.history || rules.tokens};
    const std::size_t nodes = !rules.tokens ? 0 : rules.mask ? 64 * rules.words : std::size_t(rows.rows);
    const bool narrow = history + nodes < (1u << 15) && std::size_t(rules.biases) < (1u << 16);
    if (!rows.probabilities)
    {
        launch<Step::adjust>(l, s, narrow, stream);
    }
    else if (s.splits == 1)
    {
        launch<Step::whole>(l, s, narrow, stream);
    }
    else
    {
        launch<Step::parts>(l, s, narrow, stream);
        launch<Step::finish>(l, s, narrow, stream);
    }
}
} // namespace tsac_hip

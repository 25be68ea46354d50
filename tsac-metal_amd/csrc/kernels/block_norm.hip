// The rows between two blocks of a model, in one pass over them:
//
//   u = scale * gate * post(x)      s = residual + u      h = norm(s)
//
//   rms(x)   = x / sqrt(mean x^2 + epsilon) * gain + bias
//   layer(x) = (x - m) / sqrt(mean (x - m)^2 + epsilon) * gain + bias,   m = mean x
//
// s leaves in the residual's type, h in 16 bits or, for a product of 8-bit integers, as whole numbers
// q of 8 bits and a scale a row: scale = max |h| * fl(1 / 127), q = h / scale to the nearest, ties to even.
// Nothing is rounded in between: h is the norm of the sum before it is rounded for its store.
//
// Up to 16,384 values a row's stay in the registers of its threads, so that the mean, the squares around it and
// the largest value each are a pass over registers, in 32 bits and in an order that depends on the
// width alone; a row of up to 1,024 values is one wave's, or a part of one's, which needs no barrier. What bounds it is
// memory: 8190 rows of 8192, BF16, with a residual of 32 bits in 164 us, where a copy of their bytes takes 169; rows to 8 bits
// in 46 (42), and with a norm in front of that 75.
//
// Longer rows do not fit a lane's 128 registers: 112 to 825 of a lane's values go through scratch memory, and rows are read as
// those of any alignment. Odd widths past 8,192 leave 1 to 41 there, and in FP32 odd ones of 513 to 1,024 and from 4,097 on 1 to 6.
// A norm of 67 M values, BF16, 57 us as a copy: 55 at width 16384, 98 at 12289, 370 at 16385, 217 at 32768, 610 at 65536.
#include "lanes.hpp"
#include "model_step.hpp"
#include "values.hpp"

#include <algorithm>
#include <type_traits>

namespace tsac_hip
{
namespace
{
constexpr int lanes = 64;

template <int Threads, class Join> __device__ __forceinline__ float joined(float value, float* shared, Join join)
{
    value = over_lanes<(Threads < lanes ? Threads : lanes)>(value, join);
    if constexpr (Threads > lanes)
    {
        lds_barrier(); // the last one's values have been read
        if (threadIdx.x % lanes == 0)
        {
            shared[threadIdx.x / lanes] = value;
        }
        lds_barrier();
        value = shared[0];
#pragma unroll
        for (int i = 1; i < Threads / lanes; ++i)
        {
            value = join(value, shared[i]);
        }
    }
    return value;
}

template <int Threads> __device__ __forceinline__ float row_sum(float value, float* shared)
{
    return joined<Threads>(value, shared, [](float a, float b) { return a + b; });
}

// Of bit patterns without their signs, which order numbers, then infinities, then what is no number.
template <int Threads> __device__ __forceinline__ unsigned row_max_bits(unsigned value, float* shared)
{
    return __float_as_uint(joined<Threads>(__uint_as_float(value), shared,
                                           [](float a, float b)
                                           {
                                               const unsigned x = __float_as_uint(a), y = __float_as_uint(b);
                                               return __uint_as_float(x > y ? x : y);
                                           }));
}

// What is known of rows: all of their eights are whole and at multiples of 16 bytes; all but the last of a row; nothing.
enum class Rows
{
    whole,
    ragged,
    any
};

// Eight values from `at` on, of which `count` there are, as they lie in memory; 0 behind them. The last ones of a ragged row
// are read in pieces of 16 bytes that have one of them, so that no element of its own is asked for.
template <Rows M, Type T>
__device__ __forceinline__ Eight<T> fetch8(const value_t<T>* at, int count, bool aligned)
{
    Eight<T> eight = {};
    if constexpr (M == Rows::any)
    {
        if (!aligned || count < 8)
        {
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                if (i < count)
                {
                    eight.v[i] = at[i];
                }
            }
            return eight;
        }
    }
    constexpr int piece = 16 / int(sizeof(value_t<T>));
#pragma unroll
    for (int i = 0; i < 8; i += piece)
    {
        if (i < count)
        {
            __builtin_memcpy(eight.v + i, __builtin_assume_aligned(at + i, 16), 16);
        }
    }
    if constexpr (M == Rows::ragged)
    {
#pragma unroll
        for (int i = 1; i < 8; ++i)
        {
            eight.v[i] = i < count ? eight.v[i] : value_t<T>(0);
        }
    }
    return eight;
}

template <Rows M, Type T>
__device__ __forceinline__ void put8(value_t<T>* at, int count, bool aligned, const float (&in)[8])
{
    if (count > 0)
    {
        store8<T>(at, M == Rows::whole ? 8 : count, M != Rows::any || aligned, in);
    }
}

template <Rows M, Type T, int Vectors, int Threads>
__device__ __forceinline__ void normalise(float (&v)[Vectors][8], const NormRule& rule, bool aligned, int width,
                                          float epsilon, int thread, float* shared)
{
    if (rule.norm == Norm::none)
    {
        return;
    }
    float mean = 0.0f;
    if (rule.norm == Norm::layer)
    {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                sum += v[i][e]; // 0 past the width
            }
        }
        mean = row_sum<Threads>(sum, shared) / float(width);
    }
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < Vectors; ++i)
    {
        const int count = width - 8 * (i * Threads + thread);
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            v[i][e] = (M == Rows::whole ? 0 : e) < count ? v[i][e] - mean : 0.0f;
            squares = __builtin_fmaf(v[i][e], v[i][e], squares);
        }
    }
    const float factor = 1.0f / __builtin_sqrtf(row_sum<Threads>(squares, shared) / float(width) + epsilon);
#pragma unroll
    for (int i = 0; i < Vectors; ++i)
    {
        const int at = 8 * (i * Threads + thread), count = width - at;
        Eight<T> gain = {}, bias = {};
        if (rule.gain)
        {
            gain = fetch8<M, T>(static_cast<const value_t<T>*>(rule.gain) + at, count, aligned);
        }
        if (rule.bias)
        {
            bias = fetch8<M, T>(static_cast<const value_t<T>*>(rule.bias) + at, count, aligned);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            float x = v[i][e] * factor;
            x = rule.gain ? x * widen<T>(gain.v[e]) : x;
            x = rule.bias ? x + widen<T>(bias.v[e]) : x;
            v[i][e] = (M == Rows::whole ? 0 : e) < count ? x : 0.0f;
        }
    }
}

// x / scale to the nearest whole number, a tie to the even one. The product with the reciprocal is off by
// less than half a step, and x - r scale, which 24 bits hold, tells on which side of a border x is.
__device__ __forceinline__ int nearest(float x, float scale, float reciprocal)
{
    float r = __builtin_rintf(x * reciprocal);
    const float rest = __builtin_fmaf(-r, scale, x), half = 0.5f * scale;
    const bool odd = int(r) & 1;
    if (__builtin_fabsf(rest) > half || (__builtin_fabsf(rest) == half && odd))
    {
        r += __builtin_copysignf(1.0f, rest);
    }
    return int(__builtin_fminf(__builtin_fmaxf(r, -127.0f), 127.0f));
}

// Eight of them, a byte each. x / scale + 1.5 2^23 has the whole number in its lowest bits; where the rest of one is half a
// step or more, which takes a border within 2^-15 of a step, all are done with care.
__device__ __forceinline__ uint2 nearest8(const float (&x)[8], float scale, float reciprocal)
{
    constexpr float whole = 0x1.8p23f;
    float worst = 0.0f;
    unsigned bits[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
    {
        const float shifted = __builtin_fmaf(x[e], reciprocal, whole);
        bits[e] = __float_as_uint(shifted);
        worst = __builtin_fmaxf(worst, __builtin_fabsf(__builtin_fmaf(whole - shifted, scale, x[e])));
    }
    if (worst >= 0.5f * scale)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            bits[e] = unsigned(nearest(x[e], scale, reciprocal));
        }
    }
    const auto four = [](const unsigned* b)
    { return __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu); };
    return make_uint2(four(bits), four(bits + 4));
}

// Which pointers of a row's are at multiples of 16 bytes, with their strides.
enum Aligned
{
    input_aligned = 1,
    gate_aligned = 2,
    residual_aligned = 4,
    sum_aligned = 8,
    out_aligned = 16,
    post_aligned = 32,
    norm_aligned = 64
};

// T: the values; R: the residual. A row is taken by Threads threads, each Vectors times eight values. Unless they are
// `any`, a workgroup takes rows one after the other, and the next one's are on their way while one is worked on: they pass
// barriers, which are for LDS alone. 8190 rows of 8192 with a residual of 32 bits: a row a workgroup, without that, 204 us for 167.
template <Type T, Type R, int Vectors, int Threads, Rows M>
__global__ __launch_bounds__(Threads > 256 ? Threads : 256, 4) void block_norm_kernel(BlockRows p, int aligned)
{
    constexpr bool Ahead = M != Rows::any;
    constexpr int together = Threads < 256 ? 256 / Threads : 1; // rows of a workgroup
    __shared__ float shared[Threads > lanes ? Threads / lanes : 1];
    const int thread = threadIdx.x % Threads, stride = gridDim.x * together;
    int row = blockIdx.x * together + threadIdx.x / Threads;
    Eight<T> inputs[Vectors];
    Eight<R> residuals[Vectors];
    const auto ask_input = [&](int from)
    {
        const auto* x = static_cast<const value_t<T>*>(p.input) + std::size_t(from) * p.input_stride;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
            const int at = 8 * (i * Threads + thread);
            inputs[i] = fetch8<M, T>(x + at, p.width - at, aligned & input_aligned);
        }
    };
    const auto ask_residual = [&](int from)
    {
        const auto* x = static_cast<const value_t<R>*>(p.residual) + std::size_t(from) * p.residual_stride;
#pragma unroll
        for (int i = 0; p.residual && i < Vectors; ++i)
        {
            const int at = 8 * (i * Threads + thread);
            residuals[i] = fetch8<M, R>(x + at, p.width - at, aligned & residual_aligned);
        }
    };
    // A row's lanes end together, and where it has several waves these are the workgroup.
    if (Ahead && row < p.rows)
    {
        ask_input(row);
        ask_residual(row);
    }
    for (; row < p.rows; row += stride)
    {
        if constexpr (!Ahead)
        {
            ask_input(row);
        }
        float v[Vectors][8], before[Ahead ? Vectors : 1][8];
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                v[i][e] = widen<T>(inputs[i].v[e]);
                if (Ahead && p.residual)
                {
                    before[Ahead ? i : 0][e] = widen<R>(residuals[i].v[e]);
                }
            }
        }
        // Hidden from the compiler, which otherwise holds gains, biases and gates of all rows in registers and spills others
        // for it (8190 rows of 8192: 176 us for 166); read again, they come from the caches.
        asm volatile("" : "+s"(p.gate), "+s"(p.post.gain), "+s"(p.post.bias), "+s"(p.norm.gain), "+s"(p.norm.bias));
        if constexpr (Ahead)
        {
            if (row + stride < p.rows)
            {
                ask_input(row + stride);
                ask_residual(row + stride);
            }
        }
        normalise<M, T, Vectors, Threads>(v, p.post, aligned & post_aligned, p.width, p.epsilon, thread, shared);
        if constexpr (!Ahead)
        {
            ask_residual(row);
        }
        const auto* gate = static_cast<const value_t<T>*>(p.gate) + std::size_t(row) * p.gate_stride;
        auto* sum = static_cast<value_t<R>*>(p.sum) + std::size_t(row) * p.sum_stride;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
            const int at = 8 * (i * Threads + thread), count = p.width - at;
            Eight<T> gates = {};
            if (p.gate)
            {
                gates = fetch8<M, T>(gate + at, count, aligned & gate_aligned);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                float u = p.gate ? v[i][e] * widen<T>(gates.v[e]) : v[i][e];
                u *= p.scale;
                u = !p.residual ? u : (Ahead ? before[Ahead ? i : 0][e] : widen<R>(residuals[i].v[e])) + u;
                v[i][e] = (M == Rows::whole ? 0 : e) < count ? u : 0.0f;
            }
            if (p.sum)
            {
                put8<M, R>(sum + at, count, aligned & sum_aligned, v[i]);
            }
        }
        if (!p.out)
        {
            continue;
        }
        normalise<M, T, Vectors, Threads>(v, p.norm, aligned & norm_aligned, p.width, p.epsilon, thread, shared);
        if (!p.out_scales)
        {
            auto* out = static_cast<value_t<T>*>(p.out) + std::size_t(row) * p.out_stride;
#pragma unroll
            for (int i = 0; i < Vectors; ++i)
            {
                const int at = 8 * (i * Threads + thread), count = p.width - at;
                put8<M, T>(out + at, count, aligned & out_aligned, v[i]);
            }
            continue;
        }
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                const unsigned bits = __float_as_uint(v[i][e]) & 0x7fffffffu;
                top = bits > top ? bits : top;
            }
        }
        top = row_max_bits<Threads>(top, shared);
        const bool finite = top < 0x7f800000u;
        const float most = __uint_as_float(top), scale = most * (1.0f / 127.0f);
        if (thread == 0)
        {
            p.out_scales[row] = finite ? scale : __uint_as_float(0x7fc00000u);
        }
        // Small rows are taken times 2^64, which changes no quotient, so that the reciprocal is finite and half
        // the scale exact.
        const bool small = most < 0x1p-60f, zero = !finite || scale == 0.0f;
        const float lifted = small ? scale * 0x1p64f : scale, reciprocal = 1.0f / lifted;
        auto* q = static_cast<int8_t*>(p.out) + std::size_t(row) * p.out_stride;
#pragma unroll
        for (int i = 0; i < Vectors; ++i)
        {
            const int at = 8 * (i * Threads + thread), count = p.width - at;
            uint2 packed = {};
            if (!zero && small)
            {
                // A scale of few bits may leave quotients past 127.
                uint64_t bytes = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    bytes |= uint64_t(uint8_t(nearest(v[i][e] * 0x1p64f, lifted, reciprocal))) << 8 * e;
                }
                packed = make_uint2(unsigned(bytes), unsigned(bytes >> 32));
            }
            else if (!zero)
            {
                packed = nearest8(v[i], lifted, reciprocal);
            }
            if (M == Rows::whole ? count > 0 : count >= 8) // rows of 8-bit integers begin at multiples of 16 bytes
            {
                *reinterpret_cast<uint2*>(q + at) = packed;
            }
            else if constexpr (M != Rows::whole)
            {
                for (int e = 0; e < count; ++e)
                {
                    q[at + e] = int8_t((e < 4 ? packed.x : packed.y) >> e % 4 * 8);
                }
            }
        }
    }
}

template <Type T, Type R> void launch(const BlockRows& p, int aligned, hipStream_t stream)
{
    // A workgroup takes several rows where there are more than are worked on at a time, or than a launch has room for.
    constexpr int most_groups = 1 << 13; // a unit's
    const auto go = [&](auto kernel, int threads, int a_unit)
    {
        const int together = threads < 256 ? 256 / threads : 1;
        const int groups = std::min({(p.rows + together - 1) / together, compute_units() * a_unit, 1 << 21});
        kernel<<<unsigned(groups), threads * together, 0, stream>>>(p, aligned);
    };
    const auto of = [&](auto rows)
    {
        constexpr Rows W = decltype(rows)::value;
        const auto a_unit = [](int groups) { return W != Rows::any ? groups : most_groups; };
        // By the width alone, so that a row's result does not depend on how many there are.
        const int w = p.width;
        w <= 128      ? go(block_norm_kernel<T, R, 1, 16, W>, 16, a_unit(8))
        : w <= 256    ? go(block_norm_kernel<T, R, 1, 32, W>, 32, a_unit(8))
        : w <= 512    ? go(block_norm_kernel<T, R, 1, 64, W>, 64, a_unit(8))
        : w <= 1024   ? go(block_norm_kernel<T, R, 2, 64, W>, 64, a_unit(4))
        : w <= 2048   ? go(block_norm_kernel<T, R, 1, 256, W>, 256, a_unit(8))
        : w <= 4096   ? go(block_norm_kernel<T, R, 2, 256, W>, 256, a_unit(4))
        : w <= 8192   ? go(block_norm_kernel<T, R, 2, 512, W>, 512, a_unit(2))
        : w <= 16384  ? go(block_norm_kernel<T, R, 2, 1024, W>, 1024, a_unit(1))
        : w <= 32768  ? go(block_norm_kernel<T, R, 4, 1024, Rows::any>, 1024, most_groups)
                      : go(block_norm_kernel<T, R, 8, 1024, Rows::any>, 1024, most_groups);
    };
    constexpr int every =
        input_aligned | gate_aligned | residual_aligned | sum_aligned | out_aligned | post_aligned | norm_aligned;
    aligned != every     ? of(std::integral_constant<Rows, Rows::any>{})
    : p.width % 8 != 0   ? of(std::integral_constant<Rows, Rows::ragged>{})
                         : of(std::integral_constant<Rows, Rows::whole>{});
    check_hip(hipGetLastError(), "block norm launch");
}
} // namespace

void block_norm(const BlockRows& p, hipStream_t stream)
{
    require(p.width > 0 && std::size_t(p.width) <= max_norm_width, "block norm: width out of range");
    if (!p.rows)
    {
        return;
    }
    const auto whole = [](const void* pointer, std::size_t stride, std::size_t size)
    { return reinterpret_cast<std::uintptr_t>(pointer) % 16 == 0 && stride * size % 16 == 0; };
    const std::size_t size = p.type == Type::single ? 4 : 2, wide = p.residual_type == Type::single ? 4 : 2;
    int aligned = 0;
    aligned |= whole(p.input, p.input_stride, size) ? input_aligned : 0;
    aligned |= whole(p.gate, p.gate_stride, size) ? gate_aligned : 0;
    aligned |= whole(p.residual, p.residual_stride, wide) ? residual_aligned : 0;
    aligned |= whole(p.sum, p.sum_stride, wide) ? sum_aligned : 0;
    aligned |= whole(p.out, p.out_stride, p.out_scales ? 1 : size) ? out_aligned : 0;
    aligned |= whole(p.post.gain, 0, size) && whole(p.post.bias, 0, size) ? post_aligned : 0;
    aligned |= whole(p.norm.gain, 0, size) && whole(p.norm.bias, 0, size) ? norm_aligned : 0;
    const bool wider = p.residual_type == Type::single;
    switch (p.type)
    {
    case Type::bf16:
        return wider ? launch<Type::bf16, Type::single>(p, aligned, stream)
                     : launch<Type::bf16, Type::bf16>(p, aligned, stream);
    case Type::half:
        return wider ? launch<Type::half, Type::single>(p, aligned, stream)
                     : launch<Type::half, Type::half>(p, aligned, stream);
    default: return launch<Type::single, Type::single>(p, aligned, stream);
    }
}
} // namespace tsac_hip

// Rows of 16-bit or 32-bit numbers, computed with in 32 bits: loads and stores of single values
// and of eight at a time. Rounding is to nearest even, once, as a value is stored.
#pragma once

#include "model_step.hpp"

namespace tsac_hip
{
template <Type T> struct Value
{
    using type = uint16_t;
};
template <> struct Value<Type::single>
{
    using type = float;
};
template <Type T> using value_t = typename Value<T>::type;

template <Type T> __device__ __forceinline__ float widen(value_t<T> bits)
{
    if constexpr (T == Type::bf16)
    {
        return __uint_as_float(unsigned(bits) << 16);
    }
    else if constexpr (T == Type::half)
    {
        return float(__builtin_bit_cast(_Float16, bits));
    }
    else
    {
        return bits;
    }
}

template <Type T> __device__ __forceinline__ value_t<T> narrow(float x)
{
    if constexpr (T == Type::bf16)
    {
        return __builtin_bit_cast(uint16_t, __bf16(x));
    }
    else if constexpr (T == Type::half)
    {
        return __builtin_bit_cast(uint16_t, _Float16(x));
    }
    else
    {
        return x;
    }
}

// Eight values as they lie in memory.
template <Type T> struct alignas(16) Eight
{
    value_t<T> v[8];
};

// Eight values from `at` on, of which `count` there are: at once where all are there and the place is
// `aligned` to 16 bytes, one by one otherwise; `rest` stands for those that are not.
template <Type T> __device__ __forceinline__ void load8(const value_t<T>* at, int count, bool aligned, float rest, float (&out)[8])
{
    if (aligned && count >= 8)
    {
        const Eight<T> e = *reinterpret_cast<const Eight<T>*>(at);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            out[i] = widen<T>(e.v[i]);
        }
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            out[i] = i < count ? widen<T>(at[i]) : rest;
        }
    }
}

template <Type T> __device__ __forceinline__ void store8(value_t<T>* at, int count, bool aligned, const float (&in)[8])
{
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        e.v[i] = narrow<T>(in[i]);
    }
    if (aligned && count >= 8)
    {
        *reinterpret_cast<Eight<T>*>(at) = e;
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            if (i < count)
            {
                at[i] = e.v[i];
            }
        }
    }
}
} // namespace tsac_hip

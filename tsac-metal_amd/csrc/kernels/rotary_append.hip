// New rows of queries, keys and values on their way into a paged cache: queries and keys are rotated by
// their positions, keys and values go to their places in the pages.
//
//   (a, b) -> amplitude * (a cos t - b sin t, a sin t + b cos t),   t = position * frequency[pair]
//
// for the pairs (i, i + rotary / 2) of a head or (2 i, 2 i + 1); what lies behind `rotary` stays. A far
// position times a frequency has more whole turns than 32 bits hold beside the angle: turns are counted in
// 64 bits and only what is left of the last one is narrowed. A row's angles are computed once, by as many
// lanes as there are pairs, for all of its heads; no table of them is read.
//
// Bytes are what it moves: a row is read once and written once, in 16-byte pieces. 8191 rows of 32 query and 8 key heads of
// 128, BF16: 41 us, a large copy's rate; a few rows 4 us, a chain of dependent loads.
#include "model_step.hpp"
#include "paged_device.hpp"
#include "values.hpp"

#include <algorithm>

namespace tsac_hip
{
namespace
{
constexpr int row_threads = 256;
constexpr double turns_a_radian = 0.15915494309189533577; // 1 / (2 pi)

enum class Pairs
{
    halves,     // (i, i + rotary / 2), rotary a multiple of 16
    neighbours, // (2 i, 2 i + 1)
    uneven      // halves of any length, value by value
};

struct Angles
{
    float cos[64], sin[64];
};

template <bool Half> constexpr Type type_of = Half ? Type::half : Type::bf16;

// Unit `unit` of a head: what a thread reads, turns and writes.
template <Type T, Pairs P>
__device__ __forceinline__ void turn(const uint16_t* from, uint16_t* to, int unit, int rotary, const Angles& angles)
{
    if constexpr (P == Pairs::halves)
    {
        const int half = rotary / 2;
        if (unit < half / 8)
        {
            float a[8], b[8], x[8], y[8];
            load8<T>(from + 8 * unit, 8, true, 0.0f, a);
            load8<T>(from + half + 8 * unit, 8, true, 0.0f, b);
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                const float c = angles.cos[8 * unit + e], s = angles.sin[8 * unit + e];
                x[e] = __builtin_fmaf(a[e], c, -(b[e] * s));
                y[e] = __builtin_fmaf(a[e], s, b[e] * c);
            }
            store8<T>(to + 8 * unit, 8, true, x);
            store8<T>(to + half + 8 * unit, 8, true, y);
        }
        else
        {
            const int at = rotary + 8 * (unit - half / 8);
            *reinterpret_cast<uint4*>(to + at) = *reinterpret_cast<const uint4*>(from + at);
        }
    }
    else if constexpr (P == Pairs::neighbours)
    {
        const int at = 8 * unit;
        if (at >= rotary)
        {
            *reinterpret_cast<uint4*>(to + at) = *reinterpret_cast<const uint4*>(from + at);
            return;
        }
        const Eight<T> raw = *reinterpret_cast<const Eight<T>*>(from + at);
        Eight<T> out = raw;
#pragma unroll
        for (int e = 0; e < 8; e += 2)
        {
            if (at + e < rotary)
            {
                const float a = widen<T>(raw.v[e]), b = widen<T>(raw.v[e + 1]);
                const float c = angles.cos[at / 2 + e / 2], s = angles.sin[at / 2 + e / 2];
                out.v[e] = narrow<T>(__builtin_fmaf(a, c, -(b * s)));
                out.v[e + 1] = narrow<T>(__builtin_fmaf(a, s, b * c));
            }
        }
        *reinterpret_cast<Eight<T>*>(to + at) = out;
    }
    else
    {
        const int half = rotary / 2;
        if (unit < half)
        {
            const float a = widen<T>(from[unit]), b = widen<T>(from[unit + half]);
            const float c = angles.cos[unit], s = angles.sin[unit];
            to[unit] = narrow<T>(__builtin_fmaf(a, c, -(b * s)));
            to[unit + half] = narrow<T>(__builtin_fmaf(a, s, b * c));
        }
        else
        {
            to[unit + half] = from[unit + half];
        }
    }
}

// Units of a head.
template <Pairs P> __device__ __forceinline__ int units_of(int rotary, int width)
{
    return P == Pairs::halves ? rotary / 16 + (width - rotary) / 8 : P == Pairs::neighbours ? width / 8 : width - rotary / 2;
}

// blockIdx: a row's place in its sequence, the sequence; or (`Find`) a row of all.
template <bool Half, Pairs P, bool Find>
__global__ __launch_bounds__(row_threads) void append_kernel(PagedCache cache, int layer, RotaryRows rows, int* status)
{
    __shared__ Angles angles;
    int row = blockIdx.x, s = blockIdx.y, first;
    if constexpr (Find)
    {
        s = sequence_of(rows.starts, cache.sequences, row);
    }
    const int count = rows_of(rows.starts, s, rows.rows, first);
    if constexpr (Find)
    {
        row -= first;
    }
    if (row < 0 || row >= rows.max_rows || row >= count)
    {
        return;
    }
    const std::size_t at = std::size_t(first) + row;
    const int length = cache.lengths[s];
    long long position = (long long)length + row;
    const int page = writable_page(cache, s, position);
    if (threadIdx.x < unsigned(rows.rotary / 2))
    {
        long long turned = position;
        if (rows.positions)
        {
            turned = rows.positions[at];
        }
        else if (rows.mask)
        {
            int depth = 0;
            for (std::size_t w = 0; w < rows.words; ++w)
            {
                depth += __popcll(rows.mask[at * rows.words + w]);
            }
            turned = (long long)length + (depth > 0 ? depth - 1 : 0);
        }
        const double turns = double(turned) * (rows.frequencies[threadIdx.x] * turns_a_radian);
        float sine, cosine;
        sincospif(2.0f * float(turns - __builtin_rint(turns)), &sine, &cosine);
        angles.cos[threadIdx.x] = rows.amplitude * cosine;
        angles.sin[threadIdx.x] = rows.amplitude * sine;
    }
    __syncthreads();
    if (page < 0 && threadIdx.x == 0)
    {
        report(status, status_invalid);
    }
    constexpr Type T = type_of<Half>;
    const int width = cache.head_width, units = units_of<P>(rows.rotary, width);
    const int queries = rows.heads * units, keys = page < 0 ? 0 : cache.heads * units;
    const std::size_t place = page < 0 ? 0 : layer * cache.layer_stride + page * cache.page_stride +
                                                 position % cache.page_rows * cache.row_stride;
    for (int i = threadIdx.x; i < queries + keys; i += row_threads)
    {
        const bool key = i >= queries;
        const int unit = key ? i - queries : i, head = unit / units;
        const uint16_t* from = key ? rows.keys + at * rows.row_stride : rows.query + at * rows.query_stride;
        uint16_t* to = key ? cache.keys + place : rows.out + at * rows.out_stride;
        turn<T, P>(from + head * width, to + head * width, unit - head * units, rows.rotary, angles);
    }
    const int vectors = page < 0 ? 0 : cache.heads * width / 8;
    for (int i = threadIdx.x; i < vectors; i += row_threads)
    {
        *reinterpret_cast<uint4*>(cache.values + place + 8 * i) =
            *reinterpret_cast<const uint4*>(rows.values + at * rows.row_stride + 8 * i);
    }
}

template <bool Half, Pairs P> void launch(const PagedCache& cache, int layer, const RotaryRows& rows, int* status,
                                          hipStream_t stream)
{
    const bool find = std::size_t(rows.max_rows) * cache.sequences >= 2 * std::size_t(rows.rows);
    const dim3 grid(unsigned(find ? rows.rows : rows.max_rows), unsigned(find ? 1 : cache.sequences));
    find ? append_kernel<Half, P, true><<<grid, row_threads, 0, stream>>>(cache, layer, rows, status)
         : append_kernel<Half, P, false><<<grid, row_threads, 0, stream>>>(cache, layer, rows, status);
    check_hip(hipGetLastError(), "pages append launch");
}
} // namespace

void pages_append(const PagedCache& cache, int layer, const RotaryRows& rows, int* status, hipStream_t stream)
{
    if (!rows.rows || !rows.max_rows || !cache.sequences)
    {
        return;
    }
    const auto go = [&](auto half)
    {
        constexpr bool H = decltype(half)::value;
        rows.interleaved           ? launch<H, Pairs::neighbours>(cache, layer, rows, status, stream)
        : rows.rotary % 16 == 0    ? launch<H, Pairs::halves>(cache, layer, rows, status, stream)
                                   : launch<H, Pairs::uneven>(cache, layer, rows, status, stream);
    };
    cache.half ? go(std::true_type{}) : go(std::false_type{});
}
} // namespace tsac_hip

// Attention of new rows over a paged cache of keys and values: a token a sequence, a chain
// of them, or the nodes of a tree of drafted tokens, whose own keys and values lie in the
// cache behind the sequence's length.
//
//   score(row, t) = scale * q . k_t        out(row) = sum_t e^(score - m) v_t / sum_t e^(score - m)
//
// One pass over the keys with a running reference m and sum. Unlike the coder's attention, whose
// sums have one fixed order, this runs on matrix cores with 32-bit sums.
//
// A wave takes 16, 32 or 64 query rows (the heads that share a key/value head, times the
// sequence's new rows) and every fourth block of 32 keys of its workgroup's chunk. Scores are
// computed transposed (keys x queries), so that a lane holds eight keys of one query; the
// weights then are the second product's operand as they lie, with keys in the order of the
// registers. Its other operand needs eight keys of one coordinate per lane: a lane loads 8
// (or 4) coordinates of eight keys and pairs halves with one byte permute a register, so neither
// keys nor values pass through LDS, and a row of the cache is read in whole lines. The waves'
// sums are joined in LDS, the chunks' in a second kernel, in ascending order.
#include "paged.hpp"

#include <algorithm>

namespace tsac_hip
{
namespace
{
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_ __attribute__((ext_vector_type(2)));

constexpr int waves = 4;
constexpr int block = 32; // keys of one step of a wave
constexpr float minus_infinity = -__builtin_inff();

template <bool Half> __device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (Half)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0,
                                                      0, 0);
    }
    else
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
}

// Two values rounded to nearest even, the first in the low half.
template <bool Half> __device__ __forceinline__ unsigned pack(float low, float high)
{
    if constexpr (Half)
    {
        const half2_ v = {_Float16(low), _Float16(high)};
        return __builtin_bit_cast(unsigned, v);
    }
    else
    {
        const bf16x2 v = {__bf16(low), __bf16(high)};
        return __builtin_bit_cast(unsigned, v);
    }
}

template <bool Half> __device__ __forceinline__ bool nonfinite(uint16_t bits)
{
    constexpr unsigned exponent = Half ? 0x7c00 : 0x7f80;
    return (bits & exponent) == exponent;
}

template <bool Half> __device__ __forceinline__ float widen(uint16_t bits)
{
    if constexpr (Half)
    {
        return float(__builtin_bit_cast(_Float16, bits));
    }
    else
    {
        return __uint_as_float(unsigned(bits) << 16);
    }
}

// Largest over the four lanes that hold a query.
__device__ __forceinline__ float query_max(float value)
{
    value = fmaxf(value, __shfl_xor(value, 16));
    return fmaxf(value, __shfl_xor(value, 32));
}

__device__ __forceinline__ float query_sum(float value)
{
    value += __shfl_xor(value, 16);
    return value + __shfl_xor(value, 32);
}

struct Launch
{
    PagedCache cache; // keys and values of the layer
    PagedRows rows;
    int group;      // query heads of a key/value head
    int page_shift; // log2 of page_rows
    int tiles, splits, chunk; // query tiles of a sequence and head, chunks, keys of a chunk
    int units;                // sequences x chunks x key/value heads
    float scale_log2;
    float* partial;
};

// What a workgroup or a merge works on: sequence, key/value head, query tile, chunk.
struct Place
{
    int sequence, head, tile, split;
    int first, nodes; // the sequence's rows
    int length;       // cached keys in front of them
    int total;        // keys that any row of the tile sees
};

template <int Queries> __device__ __forceinline__ bool place_of(const Launch& l, int unit, int tile, Place& p)
{
    p.head = unit % l.cache.heads;
    p.split = unit / l.cache.heads % l.splits;
    p.sequence = unit / l.cache.heads / l.splits;
    p.tile = tile;
    p.first = l.rows.starts[p.sequence];
    const int end = min(l.rows.starts[p.sequence + 1], l.rows.rows);
    p.nodes = p.first < 0 ? 0 : min(end - p.first, l.rows.max_rows);
    p.length = min(max(l.cache.lengths[p.sequence], 0), 1 << 30);
    if (p.nodes * l.group <= tile * Queries)
    {
        return false;
    }
    // Without a mask a row sees the rows up to its own.
    const int last = min((tile * Queries + Queries - 1) / l.group, p.nodes - 1);
    p.total = p.length + (l.rows.mask ? p.nodes : last + 1);
    return true;
}

// Keys of a chunk: the last one takes what there is.
__device__ __forceinline__ int chunk_end(const Launch& l, const Place& p)
{
    return p.split == l.splits - 1 ? p.total : min(p.total, (p.split + 1) * l.chunk);
}

// Chunks of a tile that hold keys (one, empty, for a tile without any).
__device__ __forceinline__ int chunks_of(const Launch& l, const Place& p)
{
    return max(1, min(l.splits, (p.total + l.chunk - 1) / l.chunk));
}

// A lane's share of a tile: row `query` = lane % 16 of each 16, and of its output the
// coordinates (4 * (lane / 16) + i) * step + j.
template <int HW, int Tiles> struct Sums
{
    static constexpr int step = HW / 16;
    f32x4 out[Tiles][step]; // [j][i]
    float reference[Tiles], total[Tiles];

    static constexpr int words = Tiles * (4 * step + 2);

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int t = 0; t < Tiles; ++t)
        {
            reference[t] = minus_infinity;
            total[t] = 0;
#pragma unroll
            for (int j = 0; j < step; ++j)
            {
                out[t][j] = f32x4{0, 0, 0, 0};
            }
        }
    }
    __device__ __forceinline__ void scale(int t, float factor)
    {
        total[t] *= factor;
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            out[t][j] *= factor;
        }
    }
    // [word][lane]
    __device__ __forceinline__ void store(float* to, int lane) const
    {
#pragma unroll
        for (int t = 0; t < Tiles; ++t)
        {
#pragma unroll
            for (int j = 0; j < step; ++j)
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    to[(((t * 4 + i) * step + j)) * 64 + lane] = out[t][j][i];
                }
            }
            to[(Tiles * 4 * step + 2 * t) * 64 + lane] = reference[t];
            to[(Tiles * 4 * step + 2 * t + 1) * 64 + lane] = total[t];
        }
    }
    __device__ __forceinline__ void join(const float* from, int lane)
    {
#pragma unroll
        for (int t = 0; t < Tiles; ++t)
        {
            const float other = from[(Tiles * 4 * step + 2 * t) * 64 + lane];
            const float most = fmaxf(reference[t], other);
            const float mine = reference[t] == most ? 1.0f : __builtin_amdgcn_exp2f(reference[t] - most);
            const float theirs = other == most ? 1.0f : __builtin_amdgcn_exp2f(other - most);
            reference[t] = most;
            total[t] = total[t] * mine + from[(Tiles * 4 * step + 2 * t + 1) * 64 + lane] * theirs;
#pragma unroll
            for (int j = 0; j < step; ++j)
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    out[t][j][i] = out[t][j][i] * mine + from[((t * 4 + i) * step + j) * 64 + lane] * theirs;
                }
            }
        }
    }
};

// Four times `step` coordinates of one row, a lane's part, divided by the row's sum. A row that no
// key reached is 0.
template <int HW, bool Half>
__device__ __forceinline__ void write_part(const Launch& l, const Place& p, int row, int lane, int i, const float* values,
                                           float total)
{
    constexpr int step = HW / 16;
    const int node = row / l.group, head = p.head * l.group + row % l.group;
    const float inverse = total == 0 ? 0.0f : 1.0f / total;
    unsigned word[step / 2];
#pragma unroll
    for (int j = 0; j < step / 2; ++j)
    {
        word[j] = pack<Half>(total == 0 ? 0.0f : values[2 * j] * inverse, total == 0 ? 0.0f : values[2 * j + 1] * inverse);
    }
    uint16_t* const to = l.rows.out + std::size_t(p.first + node) * l.rows.out_stride + std::size_t(head) * HW +
                         (4 * (lane / 16) + i) * step;
    __builtin_memcpy(__builtin_assume_aligned(to, 2 * step), word, 2 * step);
}

// The keys and values of one block in a wave's registers.
template <int HW> struct Tile
{
    static constexpr int depth = HW / 32;        // products over a key's coordinates
    static constexpr int step = HW / 16;         // coordinates of a value row a lane loads
    u32x4 key[2][depth];
    unsigned value[8][step / 2]; // of key 16 * (slot / 4) + 4 * (lane / 16) + slot % 4
    bool there[2];               // pages of the block's halves that exist
};

template <int HW, bool Half, int Tiles>
__global__ __launch_bounds__(64 * waves, Tiles == 4 ? 1 : 2) void paged_kernel(Launch l)
{
    constexpr int queries = 16 * Tiles, depth = HW / 32, step = HW / 16;
    extern __shared__ float joined[];
    const int lane = threadIdx.x % 64, warp = __builtin_amdgcn_readfirstlane(int(threadIdx.x / 64));
    const int column = lane % 16, quarter = lane / 16;
    // Workgroups go round the eight dies: a unit's tiles, which read the same keys, follow one
    // another on one die.
    const int unit = blockIdx.x / (8 * l.tiles) * 8 + blockIdx.x % 8, tile = blockIdx.x / 8 % l.tiles;
    Place p;
    if (unit >= l.units || !place_of<queries>(l, unit, tile, p) || p.split >= chunks_of(l, p))
    {
        return;
    }
    const int begin = p.split * l.chunk, end = chunk_end(l, p);
    const int limit = min(l.cache.held[p.sequence], int(l.cache.table_stride));
    const int* const table = l.cache.table + std::size_t(p.sequence) * l.cache.table_stride;

    // Queries, and where their mask lies.
    u32x4 query[Tiles][depth];
    int node[Tiles];
#pragma unroll
    for (int t = 0; t < Tiles; ++t)
    {
        const int row = p.tile * queries + 16 * t + column;
        node[t] = row / l.group;
        const bool live = node[t] < p.nodes;
        node[t] = live ? node[t] : -1;
        const uint16_t* const from = l.rows.query + std::size_t(p.first + (live ? node[t] : 0)) * l.rows.query_stride +
                                     std::size_t(p.head * l.group + row % l.group) * HW + quarter * 8;
#pragma unroll
        for (int d = 0; d < depth; ++d)
        {
            query[t][d] = live ? *reinterpret_cast<const u32x4*>(from + 32 * d) : u32x4{0, 0, 0, 0};
        }
    }

    const unsigned stride = unsigned(l.cache.row_stride);
    const uint16_t* const keys = l.cache.keys + p.head * HW;
    const uint16_t* const values = l.cache.values + p.head * HW;
    const unsigned key_lane = column * stride + quarter * 8, value_lane = 4 * quarter * stride + column * step;

    const auto load = [&](Tile<HW>& x, int at)
    {
#pragma unroll
        for (int half = 0; half < 2; ++half)
        {
            const int position = at + 16 * half, index = position >> l.page_shift;
            int page = index < limit ? table[index] : -1;
            x.there[half] = page >= 0 && page < l.cache.pages;
            page = x.there[half] ? page : 0; // masked below
            const std::size_t base =
                page * l.cache.page_stride + std::size_t(position & (l.cache.page_rows - 1)) * l.cache.row_stride;
#pragma unroll
            for (int d = 0; d < depth; ++d)
            {
                x.key[half][d] = *reinterpret_cast<const u32x4*>(keys + base + key_lane + 32 * d);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const uint16_t* const from = values + base + value_lane + i * stride;
                if constexpr (step == 8)
                {
                    *reinterpret_cast<u32x4*>(x.value[4 * half + i]) = *reinterpret_cast<const u32x4*>(from);
                }
                else
                {
                    *reinterpret_cast<u32x2*>(x.value[4 * half + i]) = *reinterpret_cast<const u32x2*>(from);
                }
            }
        }
    };

    Sums<HW, Tiles> sums;
    sums.clear();

    const auto compute = [&](Tile<HW>& x, int at)
    {
        // Every row of the tile sees the whole block if it lies in front of what masks cover.
        const int open = l.rows.mask ? p.length : p.length + p.tile * queries / l.group + 1;
        const bool whole = at + block <= open && at + block <= end && x.there[0] && x.there[1];
        unsigned live[Tiles]; // bit k: key at + k counts for this lane's query
        unsigned poisoned = 0; // keys of new rows with a value that is not finite
#pragma unroll
        for (int t = 0; t < Tiles; ++t)
        {
            live[t] = ~0u;
        }
        if (!whole)
        {
            unsigned exist = (x.there[0] ? 0xffffu : 0u) | (x.there[1] ? 0xffff0000u : 0u);
            exist &= end - at >= block ? ~0u : (1u << (end - at)) - 1;
            const int cached = p.length - at; // keys of the block in front of the new rows
            const unsigned before = cached >= block ? ~0u : cached <= 0 ? 0u : (1u << cached) - 1;
#pragma unroll
            for (int t = 0; t < Tiles; ++t)
            {
                unsigned drafted = 0; // of new rows, bits as in `live`
                if (node[t] >= 0 && cached < block)
                {
                    if (l.rows.mask)
                    {
                        const uint64_t* const words = l.rows.mask + std::size_t(p.first + node[t]) * l.rows.words;
                        const int from = cached > 0 ? 0 : -cached; // first new row of the block
                        const std::size_t word = from / 64;
                        uint64_t bits = word < l.rows.words ? words[word] >> from % 64 : 0;
                        if (from % 64 && word + 1 < l.rows.words)
                        {
                            bits |= words[word + 1] << (64 - from % 64);
                        }
                        drafted = cached > 0 ? unsigned(bits) << cached : unsigned(bits);
                    }
                    else
                    {
                        const int seen = cached + node[t] + 1; // keys of the block up to the row's own
                        drafted = (seen >= block ? ~0u : seen <= 0 ? 0u : (1u << seen) - 1) & ~before;
                    }
                }
                live[t] = node[t] < 0 ? 0u : exist & (before | drafted);
            }
            // Values of keys that no row may see are dropped here: a weight of zero does not
            // drop one that is not finite. New rows that only some rows see follow below.
#pragma unroll
            for (int slot = 0; slot < 8; ++slot)
            {
                const int key = 16 * (slot / 4) + 4 * quarter + slot % 4;
                bool wrong = false;
#pragma unroll
                for (int w = 0; w < step / 2; ++w)
                {
                    x.value[slot][w] = exist >> key & 1 ? x.value[slot][w] : 0u;
                    wrong |= nonfinite<Half>(uint16_t(x.value[slot][w])) || nonfinite<Half>(uint16_t(x.value[slot][w] >> 16));
                }
                const uint64_t lanes = __ballot(wrong && !(before >> key & 1));
#pragma unroll
                for (int q = 0; q < 4; ++q)
                {
                    poisoned |= (lanes >> 16 * q & 0xffff ? 1u : 0u) << (16 * (slot / 4) + 4 * q + slot % 4);
                }
            }
            if (poisoned)
            {
#pragma unroll
                for (int slot = 0; slot < 8; ++slot)
                {
                    const int key = 16 * (slot / 4) + 4 * quarter + slot % 4;
#pragma unroll
                    for (int w = 0; w < step / 2; ++w)
                    {
                        unsigned& v = x.value[slot][w];
                        const unsigned keep = (nonfinite<Half>(uint16_t(v)) ? 0u : 0xffffu) |
                                              (nonfinite<Half>(uint16_t(v >> 16)) ? 0u : 0xffff0000u);
                        v = poisoned >> key & 1 ? v & keep : v;
                    }
                }
            }
        }

        u32x4 weight[Tiles];
#pragma unroll
        for (int t = 0; t < Tiles; ++t)
        {
            float score[8];
#pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                f32x4 s = {0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < depth; ++d)
                {
                    s = product<Half>(x.key[half][d], query[t][d], s);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    score[4 * half + i] = s[i] * l.scale_log2;
                }
            }
            if (!whole)
            {
#pragma unroll
                for (int slot = 0; slot < 8; ++slot)
                {
                    const int key = 16 * (slot / 4) + 4 * quarter + slot % 4;
                    score[slot] = live[t] >> key & 1 ? score[slot] : minus_infinity;
                }
            }
            float most = score[0];
#pragma unroll
            for (int slot = 1; slot < 8; ++slot)
            {
                most = fmaxf(most, score[slot]);
            }
            // The reference moves only when a score passes it by 2^8: weights stay in range
            // without it, and most blocks need neither the exchange nor the scaling.
            if (__any(most > sums.reference[t] + 8.0f))
            {
                most = fmaxf(query_max(most), sums.reference[t]);
                const float factor =
                    most == sums.reference[t] ? 1.0f : __builtin_amdgcn_exp2f(sums.reference[t] - most);
                sums.scale(t, factor);
                sums.reference[t] = most;
            }
            const float reference = sums.reference[t] == minus_infinity ? 0.0f : sums.reference[t];
            float e[8];
#pragma unroll
            for (int slot = 0; slot < 8; ++slot)
            {
                e[slot] = __builtin_amdgcn_exp2f(score[slot] - reference);
                sums.total[t] += e[slot];
            }
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                weight[t][w] = pack<Half>(e[2 * w], e[2 * w + 1]);
            }
            if (poisoned)
            {
                for (unsigned left = poisoned; left; left &= left - 1)
                {
                    const int key = __builtin_ctz(left);
                    float mine = e[0];
#pragma unroll
                    for (int slot = 1; slot < 8; ++slot)
                    {
                        mine = 4 * (key / 16) + key % 4 == slot ? e[slot] : mine;
                    }
                    mine = __shfl(mine, key % 16 / 4 * 16 + column);
                    const int position = at + key, page = table[position >> l.page_shift];
                    const uint16_t* const from =
                        values + page * l.cache.page_stride +
                        std::size_t(position & (l.cache.page_rows - 1)) * l.cache.row_stride + 4 * quarter * step;
                    if (live[t] >> key & 1)
                    {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                        {
#pragma unroll
                            for (int j = 0; j < step; ++j)
                            {
                                const uint16_t bits = from[i * step + j];
                                sums.out[t][j][i] += nonfinite<Half>(bits) ? mine * widen<Half>(bits) : 0.0f;
                            }
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            u32x4 operand; // coordinate column * step + j of the block's keys, in the order of the weights
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                operand[w] = __builtin_amdgcn_perm(x.value[2 * w + 1][j / 2], x.value[2 * w][j / 2],
                                                   j % 2 ? 0x07060302u : 0x05040100u);
            }
#pragma unroll
            for (int t = 0; t < Tiles; ++t)
            {
                sums.out[t][j] = product<Half>(operand, weight[t], sums.out[t][j]);
            }
        }
    };

    // Two blocks in registers: one is loaded while the other is used.
    Tile<HW> a, b;
    int at = begin + block * warp;
    constexpr int stride_keys = block * waves;
    if (at < end)
    {
        load(a, at);
    }
    while (at < end)
    {
        if (at + stride_keys < end)
        {
            load(b, at + stride_keys);
        }
        compute(a, at);
        at += stride_keys;
        if (at >= end)
        {
            break;
        }
        if (at + stride_keys < end)
        {
            load(a, at + stride_keys);
        }
        compute(b, at);
        at += stride_keys;
    }

#pragma unroll
    for (int t = 0; t < Tiles; ++t)
    {
        sums.total[t] = query_sum(sums.total[t]);
    }
    // Waves 2 and 3 to 0 and 1, then 1 to 0.
    constexpr int record = Sums<HW, Tiles>::words * 64;
#pragma unroll
    for (int half = 2; half >= 1; half /= 2)
    {
        if (warp >= half && warp < 2 * half)
        {
            sums.store(joined + (warp - half) * record, lane);
        }
        __syncthreads();
        if (warp < half)
        {
            sums.join(joined + warp * record, lane);
        }
        __syncthreads();
    }
    if (warp)
    {
        return;
    }
    if (chunks_of(l, p) > 1)
    {
        sums.store(l.partial + (std::size_t(unit) * l.tiles + tile) * record, lane);
        return;
    }
#pragma unroll
    for (int t = 0; t < Tiles; ++t)
    {
        if (node[t] >= 0)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                float part[step];
#pragma unroll
                for (int j = 0; j < step; ++j)
                {
                    part[j] = sums.out[t][j][i];
                }
                write_part<HW, Half>(l, p, p.tile * queries + 16 * t + column, lane, i, part, sums.total[t]);
            }
        }
    }
}

// Joins the chunks of a (sequence, head, tile): wave i of workgroup t takes coordinates i of
// the t-th 16 rows.
template <int HW, bool Half, int Tiles> __global__ __launch_bounds__(256) void paged_join_kernel(Launch l)
{
    constexpr int queries = 16 * Tiles, step = HW / 16, record = Sums<HW, Tiles>::words * 64;
    const int lane = threadIdx.x % 64, i = threadIdx.x / 64;
    const int t = blockIdx.x % Tiles, tile = blockIdx.x / Tiles % l.tiles, pair = blockIdx.x / Tiles / l.tiles;
    const int head = pair % l.cache.heads, sequence = pair / l.cache.heads;
    const auto unit = [&](int split) { return (sequence * l.splits + split) * l.cache.heads + head; };
    Place p;
    if (!place_of<queries>(l, unit(0), tile, p))
    {
        return;
    }
    const int chunks = chunks_of(l, p), row = tile * queries + 16 * t + lane % 16;
    if (chunks == 1 || row / l.group >= p.nodes)
    {
        return;
    }
    float reference = minus_infinity, total = 0, out[step] = {};
    for (int split = 0; split < chunks; ++split)
    {
        const float* const from = l.partial + (std::size_t(unit(split)) * l.tiles + tile) * record + lane;
        const float other = from[(Tiles * 4 * step + 2 * t) * 64], part = from[(Tiles * 4 * step + 2 * t + 1) * 64];
        const float most = fmaxf(reference, other);
        const float mine = reference == most ? 1.0f : __builtin_amdgcn_exp2f(reference - most);
        const float theirs = other == most ? 1.0f : __builtin_amdgcn_exp2f(other - most);
        reference = most;
        total = total * mine + part * theirs;
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            out[j] = out[j] * mine + from[((t * 4 + i) * step + j) * 64] * theirs;
        }
    }
    write_part<HW, Half>(l, p, row, lane, i, out, total);
}

// The launch's shape: it depends on what the host knows, sizes and not lengths.
struct Shape
{
    int rows_a_tile; // 16-row tiles of a wave
    int tiles, splits, chunk;
    std::size_t units, record;
};

Shape shape_of(const PagedCache& cache, const PagedRows& rows)
{
    Shape s;
    const std::size_t group = std::size_t(rows.heads / cache.heads), queries = std::size_t(rows.max_rows) * group;
    s.rows_a_tile = queries <= 16 ? 1 : queries <= 32 ? 2 : 4;
    s.tiles = int((queries + 16 * s.rows_a_tile - 1) / (16 * s.rows_a_tile));
    const std::size_t pairs = std::size_t(cache.sequences) * cache.heads;
    // Two workgroups a compute unit, of at least 256 keys each.
    const std::size_t wanted = std::max<std::size_t>(1, 2 * std::size_t(compute_units()) / (pairs * s.tiles));
    const std::size_t most = std::max<std::size_t>(1, (rows.max_length + 255) / 256);
    s.splits = int(std::min(wanted, most));
    constexpr std::size_t keys = block * waves;
    s.chunk = int(((rows.max_length + s.splits - 1) / s.splits + keys - 1) / keys * keys);
    s.chunk = std::max<int>(s.chunk, keys);
    s.units = pairs * s.splits;
    s.record = 64 * std::size_t(s.rows_a_tile) * (cache.head_width / 4 + 2);
    return s;
}

template <int HW, bool Half, int Tiles> void launch(const Launch& l, std::size_t pairs, hipStream_t stream)
{
    const std::size_t lds = 2 * Sums<HW, Tiles>::words * 64 * 4;
    const auto kernel = paged_kernel<HW, Half, Tiles>;
    if (lds > 65536)
    {
        check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)),
                  "paged attention LDS");
    }
    const std::size_t grid = (std::size_t(l.units) + 7) / 8 * 8 * l.tiles;
    kernel<<<unsigned(grid), 64 * waves, lds, stream>>>(l);
    check_hip(hipGetLastError(), "paged attention launch");
    if (l.splits > 1)
    {
        paged_join_kernel<HW, Half, Tiles><<<unsigned(pairs * l.tiles * Tiles), 256, 0, stream>>>(l);
        check_hip(hipGetLastError(), "paged attention launch");
    }
}
} // namespace

std::size_t attention_paged_workspace(const PagedCache& cache, const PagedRows& rows)
{
    if (!rows.rows || !rows.max_rows || !cache.sequences)
    {
        return 0;
    }
    const Shape s = shape_of(cache, rows);
    return s.splits > 1 ? s.units * s.tiles * s.record * 4 : 0;
}

void attention_paged(const PagedCache& cache, int layer, const PagedRows& rows, void* workspace, std::size_t bytes,
                     hipStream_t stream)
{
    if (!rows.rows || !rows.max_rows || !cache.sequences)
    {
        return;
    }
    const Shape s = shape_of(cache, rows);
    // 2^32 work-items along x are a grid's limit.
    require((s.units + 8) * s.tiles < (std::size_t(1) << 22), "paged attention: too many workgroups for one launch");
    require(s.splits == 1 || (workspace && bytes >= s.units * s.tiles * s.record * 4),
            "paged attention: the workspace is too small");
    Launch l{};
    l.cache = cache;
    l.cache.keys += layer * cache.layer_stride;
    l.cache.values += layer * cache.layer_stride;
    l.rows = rows;
    l.group = rows.heads / cache.heads;
    l.page_shift = __builtin_ctz(unsigned(cache.page_rows));
    l.tiles = s.tiles;
    l.splits = s.splits;
    l.chunk = s.chunk;
    l.units = int(s.units);
    l.scale_log2 = rows.scale * 1.44269504088896340736f;
    l.partial = static_cast<float*>(workspace);
    const std::size_t pairs = std::size_t(cache.sequences) * cache.heads;
    const auto by_tiles = [&](auto width, auto half)
    {
        constexpr int HW = decltype(width)::value;
        constexpr bool Half = decltype(half)::value;
        switch (s.rows_a_tile)
        {
        case 1: launch<HW, Half, 1>(l, pairs, stream); break;
        case 2: launch<HW, Half, 2>(l, pairs, stream); break;
        default: launch<HW, Half, 4>(l, pairs, stream); break;
        }
    };
    const auto by_type = [&](auto width)
    { cache.half ? by_tiles(width, std::true_type{}) : by_tiles(width, std::false_type{}); };
    cache.head_width == 64 ? by_type(std::integral_constant<int, 64>{}) : by_type(std::integral_constant<int, 128>{});
}
} // namespace tsac_hip

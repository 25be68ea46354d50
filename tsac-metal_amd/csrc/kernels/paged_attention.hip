// Attention of new rows over a paged cache of keys and values: a token a sequence, a chain
// of them, or the nodes of a tree of drafted tokens, whose own keys and values lie in the
// cache behind the sequence's length.
//
//   score(row, t) = scale * q . k_t        out(row) = sum_t e^(score - m) v_t / sum_t e^(score - m)
//
// One pass over the keys with a running reference m and sum. Unlike the coder's attention, whose
// sums have one fixed order, this runs on matrix cores with 32-bit sums.
//
// The query rows of a (sequence, key/value head), its new rows times the heads that share the
// keys, are taken 16 at a time, the keys 32 at a time (a block). Scores are computed transposed
// (keys x queries), so that a lane holds eight keys of one query; the weights then are the
// second product's operand as they lie, with keys in the order of the registers. Its other
// operand needs eight keys of one coordinate per lane: a lane loads 8 (or 4) coordinates of
// eight keys and pairs halves with one byte permute a register, so that a row of the cache is
// read in whole lines and nothing is transposed through memory.
//
// Up to 32 query rows (direct_kernel) the cache's bytes are what costs: a wave takes all rows
// and every fourth block of its workgroup's chunk of keys, straight from memory into operand
// registers. More rows (staged_kernel) cost products and exponentials: a wave takes 32 rows, and
// the four of a workgroup share blocks that they stage in LDS in operand order. Chunks are
// joined in ascending order by join_kernel.
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

constexpr int waves = 4;  // of a workgroup
constexpr int block = 32; // keys of one step
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

// Bits 0 .. count-1, for any count.
__device__ __forceinline__ unsigned low_bits(int count)
{
    return count >= 32 ? ~0u : count <= 0 ? 0u : (1u << count) - 1;
}

struct Launch
{
    const uint16_t* keys; // of the layer
    const uint16_t* values;
    std::size_t page_stride;
    const int* table;
    std::size_t table_stride;
    const int* held;
    const int* lengths;
    const int* starts;
    const uint16_t* query;
    std::size_t query_stride;
    uint16_t* out;
    std::size_t out_stride;
    const uint64_t* mask;
    float* partial;
    unsigned row_stride;
    int pages, page_shift; // log2 of a page's rows
    int heads, group;      // key/value heads, and query heads of each
    int rows, max_rows, words;
    int tiles;  // query tiles of a workgroup's kind, of a sequence and head
    int parts;  // 16 rows each, of a sequence and head
    int splits, chunk; // chunks, keys of a chunk
    int units;         // sequences x chunks x key/value heads
    float scale_log2;  // above or at 0
    bool negative;     // scale is below: queries are taken negative
};

// What a workgroup or a join works on: sequence, key/value head, chunk, and from which of its
// query rows on.
struct Place
{
    int sequence, head, split, row;
    int first, nodes; // the sequence's rows
    int length;       // cached keys in front of them
    int total;        // keys that any of the rows sees
    int limit;        // entries of the table
};

// False if there is no such row.
__device__ __forceinline__ bool place_of(const Launch& l, int unit, int row, int count, Place& p)
{
    p.head = unit % l.heads;
    p.split = unit / l.heads % l.splits;
    p.sequence = unit / l.heads / l.splits;
    p.row = row;
    p.first = l.starts[p.sequence];
    const int end = min(l.starts[p.sequence + 1], l.rows);
    p.nodes = p.first < 0 ? 0 : min(end - p.first, l.max_rows);
    p.length = min(max(l.lengths[p.sequence], 0), 1 << 30);
    p.limit = min(l.held[p.sequence], int(l.table_stride));
    if (p.nodes * l.group <= row)
    {
        return false;
    }
    // Without a mask a row sees the rows up to its own.
    p.total = p.length + (l.mask ? p.nodes : min((row + count - 1) / l.group, p.nodes - 1) + 1);
    return true;
}

__device__ __forceinline__ int chunks_of(const Launch& l, const Place& p)
{
    return max(1, min(l.splits, (p.total + l.chunk - 1) / l.chunk));
}

// The last chunk takes what there is.
__device__ __forceinline__ int chunk_end(const Launch& l, const Place& p)
{
    return p.split == l.splits - 1 ? p.total : min(p.total, (p.split + 1) * l.chunk);
}

// Where 16 keys from a position start, as an offset into keys and values; `there` if they lie in
// a page of the pool, otherwise the offset is some page's.
__device__ __forceinline__ std::size_t locate(const Launch& l, const Place& p, int position, bool& there)
{
    const int index = position >> l.page_shift;
    const int page = index < p.limit ? l.table[p.sequence * l.table_stride + index] : -1;
    there = page >= 0 && page < l.pages;
    return (there ? page : 0) * l.page_stride +
           std::size_t(position & ((1 << l.page_shift) - 1)) * l.row_stride;
}

// One 16-row part's running sums. A lane has row lane % 16 and of its output the coordinates
// (4 * (lane / 16) + i) * step + j.
template <int HW> struct Sums
{
    static constexpr int step = HW / 16;
    static constexpr int words = 4 * step + 2; // of a record, [word][lane]
    f32x4 out[step];                           // [j][i]
    f32x4 total;                               // four times the same
    float reference;

    __device__ __forceinline__ void clear()
    {
        reference = minus_infinity;
        total = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            out[j] = f32x4{0, 0, 0, 0};
        }
    }
    // To a reference not below the present one.
    __device__ __forceinline__ void move(float to)
    {
        const float factor = to == reference ? 1.0f : __builtin_amdgcn_exp2f(reference - to);
        reference = to;
        total *= factor;
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            out[j] *= factor;
        }
    }
    __device__ __forceinline__ void store(float* to, int lane) const
    {
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                to[(i * step + j) * 64 + lane] = out[j][i];
            }
        }
        to[(4 * step) * 64 + lane] = reference;
        to[(4 * step + 1) * 64 + lane] = total[0];
    }
    __device__ __forceinline__ void join(const float* from, int lane)
    {
        const float other = from[(4 * step) * 64 + lane], most = fmaxf(reference, other);
        move(most);
        const float theirs = other == most ? 1.0f : __builtin_amdgcn_exp2f(other - most);
        total += from[(4 * step + 1) * 64 + lane] * theirs;
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                out[j][i] += from[(i * step + j) * 64 + lane] * theirs;
            }
        }
    }
};

// A lane's part i of one row, divided by the row's sum. A row that no key reached is 0.
template <int HW, bool Half>
__device__ __forceinline__ void write_part(const Launch& l, const Place& p, int row, int lane, int i, const float* values,
                                           float total)
{
    constexpr int step = HW / 16;
    const int node = row / l.group, head = p.head * l.group + row % l.group;
    const float inverse = 1.0f / total;
    unsigned word[step / 2];
#pragma unroll
    for (int j = 0; j < step / 2; ++j)
    {
        word[j] = total == 0 ? 0u : pack<Half>(values[2 * j] * inverse, values[2 * j + 1] * inverse);
    }
    uint16_t* const to = l.out + std::size_t(p.first + node) * l.out_stride + std::size_t(head) * HW +
                         (4 * (lane / 16) + i) * step;
    __builtin_memcpy(__builtin_assume_aligned(to, 2 * step), word, 2 * step);
}

// A part's sums: to the output, or as the chunk's record.
template <int HW, bool Half>
__device__ __forceinline__ void finish(const Launch& l, const Place& p, int unit, int row, int lane, const Sums<HW>& sums)
{
    if (chunks_of(l, p) > 1)
    {
        sums.store(l.partial + (std::size_t(unit) * l.parts + row / 16) * (Sums<HW>::words * 64), lane);
        return;
    }
    const int mine = row + lane % 16;
    if (mine / l.group >= p.nodes)
    {
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        float part[Sums<HW>::step];
#pragma unroll
        for (int j = 0; j < Sums<HW>::step; ++j)
        {
            part[j] = sums.out[j][i];
        }
        write_part<HW, Half>(l, p, mine, lane, i, part, sums.total[0]);
    }
}

// 16 rows' queries as operands, from row `row`; `node` is the lane's row's, -1 past the last.
template <int HW>
__device__ __forceinline__ void load_query(const Launch& l, const Place& p, int row, int lane, u32x4 (&query)[HW / 32],
                                           int& node)
{
    const int mine = row + lane % 16;
    const bool live = mine / l.group < p.nodes;
    node = live ? mine / l.group : -1;
    const uint16_t* const from = l.query + std::size_t(p.first + (live ? node : 0)) * l.query_stride +
                                 std::size_t(p.head * l.group + (live ? mine % l.group : 0)) * HW + lane / 16 * 8;
    const unsigned sign = l.negative ? 0x80008000u : 0u;
#pragma unroll
    for (int d = 0; d < HW / 32; ++d)
    {
        query[d] = live ? *reinterpret_cast<const u32x4*>(from + 32 * d) ^ sign : u32x4{0, 0, 0, 0};
    }
}

// Which keys of the block at `at` count for a lane's query: those of `exist` that are cached, or
// new rows that its node sees.
__device__ __forceinline__ unsigned seen(const Launch& l, const Place& p, int at, unsigned exist, int node)
{
    const int cached = p.length - at; // keys of the block in front of the new rows
    if (node < 0)
    {
        return 0;
    }
    if (!l.mask)
    {
        return exist & low_bits(cached + node + 1);
    }
    unsigned fresh = 0;
    if (cached < block)
    {
        const uint64_t* const words = l.mask + std::size_t(p.first + node) * l.words;
        const int from = max(-cached, 0), word = from / 64; // the block's first new row
        uint64_t bits = word < l.words ? words[word] >> from % 64 : 0;
        if (from % 64 && word + 1 < l.words)
        {
            bits |= words[word + 1] << (64 - from % 64);
        }
        fresh = cached > 0 ? unsigned(bits) << cached : unsigned(bits);
    }
    return exist & (low_bits(cached) | fresh);
}

// A value row that is not finite, of new row `key` of the block, for the rows that see it.
template <int HW, bool Half>
__device__ __forceinline__ void add_poisoned(const Launch& l, const Place& p, int at, int key, float weight, bool live,
                                             int lane, Sums<HW>& sums)
{
    constexpr int step = HW / 16;
    bool there;
    const std::size_t base = locate(l, p, at + key / 16 * 16, there) + std::size_t(p.head) * HW;
    const uint16_t* const from = l.values + base + std::size_t(key % 16) * l.row_stride + lane / 16 * 4 * step;
    if (live && there)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
#pragma unroll
            for (int j = 0; j < step; ++j)
            {
                const uint16_t bits = from[i * step + j];
                sums.out[j][i] += nonfinite<Half>(bits) ? weight * widen<Half>(bits) : 0.0f;
            }
        }
    }
}

// Drops from half a block's values, slots 4 * half .. of the lane, those of keys that do not exist
// (a weight of zero would not drop one that is not finite), and those not finite of new rows,
// which only some queries see. Returns the bits of the latter's keys.
template <int HW, bool Half>
__device__ __forceinline__ unsigned clean(unsigned (&value)[4][HW / 32], int half, unsigned exist, unsigned cached, int lane)
{
    unsigned poisoned = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const int key = 16 * half + 4 * (lane / 16) + i;
        const bool there = exist >> key & 1, fresh = !(cached >> key & 1);
        bool wrong = false;
#pragma unroll
        for (int w = 0; w < HW / 32; ++w)
        {
            unsigned& v = value[i][w];
            const unsigned keep = (nonfinite<Half>(uint16_t(v)) ? 0u : 0xffffu) |
                                  (nonfinite<Half>(uint16_t(v >> 16)) ? 0u : 0xffff0000u);
            wrong = wrong || keep != ~0u;
            v = !there ? 0u : fresh ? v & keep : v;
        }
        const uint64_t lanes = __ballot(wrong && there && fresh);
#pragma unroll
        for (int q = 0; q < 4; ++q)
        {
            poisoned |= (lanes >> 16 * q & 0xffff ? 1u : 0u) << (16 * half + 4 * q + i);
        }
    }
    return poisoned;
}

// Adds a block's keys to `Parts` parts of 16 rows. key(half, d) and value(j) give the operands;
// next() runs once the keys are used up.
// Masks are looked at where the block is not `whole`: not all of it exists, or it reaches into
// what some row does not see.
template <int HW, bool Half, int Parts, class Key, class Values, class Next>
__device__ __forceinline__ void attend(const Launch& l, const Place& p, int at, bool whole, unsigned exist,
                                       unsigned poisoned, int lane, const u32x4 (&query)[Parts][HW / 32],
                                       const int (&node)[Parts], Sums<HW> (&sums)[Parts], Key key, Values value, Next next)
{
    constexpr int depth = HW / 32, step = HW / 16;
    f32x4 score[Parts][2];
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            score[t][half] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int d = 0; d < depth; ++d)
        {
            const u32x4 k = key(half, d);
#pragma unroll
            for (int t = 0; t < Parts; ++t)
            {
                score[t][half] = product<Half>(k, query[t][d], score[t][half]);
            }
        }
    }
    next();
    unsigned live[Parts];
    if (!whole)
    {
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            live[t] = seen(l, p, at, exist, node[t]) >> 4 * (lane / 16);
#pragma unroll
            for (int slot = 0; slot < 8; ++slot)
            {
                f32x4& s = score[t][slot / 4];
                s[slot % 4] = live[t] >> (16 * (slot / 4) + slot % 4) & 1 ? s[slot % 4] : minus_infinity;
            }
        }
    }
    // The reference moves only when a score passes it by 2^8: weights stay in range without it,
    // and most blocks need neither the exchange nor the scaling.
    float most[Parts];
    bool move = false;
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        const f32x4 a = score[t][0], b = score[t][1];
        most[t] = fmaxf(fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(b[0], b[1])), fmaxf(b[2], b[3]));
        // Not a product with -infinity, which a scale of 0 would make no number.
        most[t] = most[t] == minus_infinity ? most[t] : most[t] * l.scale_log2;
        move = move || most[t] > sums[t].reference + 8.0f;
    }
    if (__any(move))
    {
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            sums[t].move(fmaxf(query_max(most[t]), sums[t].reference));
        }
    }
    u32x4 weight[Parts];
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        const float reference = sums[t].reference == minus_infinity ? 0.0f : sums[t].reference;
        float e[8];
#pragma unroll
        for (int slot = 0; slot < 8; ++slot)
        {
            e[slot] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[t][slot / 4][slot % 4], l.scale_log2, -reference));
        }
        if (!whole)
        {
#pragma unroll
            for (int slot = 0; slot < 8; ++slot)
            {
                e[slot] = live[t] >> (16 * (slot / 4) + slot % 4) & 1 ? e[slot] : 0.0f;
            }
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
        {
            weight[t][w] = pack<Half>(e[2 * w], e[2 * w + 1]);
        }
        if (poisoned)
        {
            const unsigned mine = seen(l, p, at, exist, node[t]);
            for (unsigned left = poisoned; left; left &= left - 1)
            {
                const int k = __builtin_ctz(left);
                float x = e[0];
#pragma unroll
                for (int slot = 1; slot < 8; ++slot)
                {
                    x = 4 * (k / 16) + k % 4 == slot ? e[slot] : x;
                }
                x = __shfl(x, k % 16 / 4 * 16 + lane % 16);
                add_poisoned<HW, Half>(l, p, at, k, x, mine >> k & 1, lane, sums[t]);
            }
        }
    }
    // The sum of a row's weights, as they are rounded, is one more product.
    constexpr unsigned one = Half ? 0x3c003c00u : 0x3f803f80u;
    const u32x4 ones = {one, one, one, one};
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        sums[t].total = product<Half>(ones, weight[t], sums[t].total);
    }
#pragma unroll
    for (int j = 0; j < step; ++j)
    {
        const u32x4 v = value(j);
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            sums[t].out[j] = product<Half>(v, weight[t], sums[t].out[j]);
        }
    }
}

// Half a block's values as a lane loads them, 16 keys: `step` coordinates of four keys.
template <int HW>
__device__ __forceinline__ void load_values(const uint16_t* from, unsigned row_stride, int lane, unsigned (&value)[4][HW / 32])
{
    constexpr int step = HW / 16;
    const uint16_t* const mine = from + 4 * (lane / 16) * row_stride + lane % 16 * step;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        if constexpr (step == 8)
        {
            *reinterpret_cast<u32x4*>(value[i]) = *reinterpret_cast<const u32x4*>(mine + i * row_stride);
        }
        else
        {
            *reinterpret_cast<u32x2*>(value[i]) = *reinterpret_cast<const u32x2*>(mine + i * row_stride);
        }
    }
}

// Coordinate j of keys i and i + 1, out of a lane's values.
template <int HW> __device__ __forceinline__ unsigned pair(const unsigned (&value)[4][HW / 32], int i, int j)
{
    return __builtin_amdgcn_perm(value[i + 1][j / 2], value[i][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
}

// Workgroups go round the eight dies: a unit's tiles, which read the same keys, follow one
// another on one die.
__device__ __forceinline__ void unit_of(const Launch& l, int& unit, int& tile)
{
    unit = blockIdx.x / (8 * l.tiles) * 8 + blockIdx.x % 8;
    tile = blockIdx.x / 8 % l.tiles;
}

// A tile is `Parts` x 16 rows; a wave takes every fourth block of the chunk.
template <int HW, bool Half, int Parts> __global__ __launch_bounds__(64 * waves, Parts == 1 ? 3 : 2) void direct_kernel(Launch l)
{
    constexpr int depth = HW / 32, record = Sums<HW>::words * 64;
    extern __shared__ float joined[];
    const int lane = threadIdx.x % 64, warp = __builtin_amdgcn_readfirstlane(int(threadIdx.x / 64));
    int unit, tile;
    unit_of(l, unit, tile);
    Place p;
    if (unit >= l.units || !place_of(l, unit, tile * 16 * Parts, 16 * Parts, p) || p.split >= chunks_of(l, p))
    {
        return;
    }
    const int begin = p.split * l.chunk, end = chunk_end(l, p);
    // Every row sees what lies in front of this.
    const int open = l.mask ? p.length : p.length + p.row / l.group + 1;
    u32x4 query[Parts][depth];
    int node[Parts];
    Sums<HW> sums[Parts];
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        load_query<HW>(l, p, p.row + 16 * t, lane, query[t], node[t]);
        sums[t].clear();
    }

    // A block's keys are asked for as soon as the last one's are used up, and so are its values:
    // one set of registers each, and either is under way while the other is worked on.
    u32x4 key[2][depth];
    unsigned value[2][4][HW / 32];
    std::size_t base[2];
    bool there[2];
    const auto find = [&](int at)
    {
#pragma unroll
        for (int half = 0; half < 2; ++half)
        {
            base[half] = locate(l, p, at + 16 * half, there[half]) + std::size_t(p.head) * HW;
        }
    };
    const auto load_keys = [&]
    {
#pragma unroll
        for (int half = 0; half < 2; ++half)
        {
#pragma unroll
            for (int d = 0; d < depth; ++d)
            {
                key[half][d] = *reinterpret_cast<const u32x4*>(l.keys + base[half] + lane % 16 * l.row_stride +
                                                               lane / 16 * 8 + 32 * d);
            }
        }
    };
    const auto load_both_values = [&]
    {
#pragma unroll
        for (int half = 0; half < 2; ++half)
        {
            load_values<HW>(l.values + base[half], l.row_stride, lane, value[half]);
        }
    };
    constexpr int stride = block * waves;
    int at = begin + block * warp;
    if (at < end)
    {
        find(at);
        load_keys();
        load_both_values();
    }
    for (; at < end; at += stride)
    {
        unsigned exist = ~0u, poisoned = 0;
        const bool whole = at + block <= min(open, end) && there[0] && there[1];
        if (!whole)
        {
            exist = low_bits(end - at) & ((there[0] ? 0xffffu : 0u) | (there[1] ? 0xffff0000u : 0u));
            const unsigned cached = low_bits(p.length - at);
            poisoned = clean<HW, Half>(value[0], 0, exist, cached, lane) | clean<HW, Half>(value[1], 1, exist, cached, lane);
        }
        attend<HW, Half, Parts>(
            l, p, at, whole, exist, poisoned, lane, query, node, sums, [&](int half, int d) { return key[half][d]; },
            [&](int j)
            {
                return u32x4{pair<HW>(value[0], 0, j), pair<HW>(value[0], 2, j), pair<HW>(value[1], 0, j),
                             pair<HW>(value[1], 2, j)};
            },
            [&]
            {
                if (at + stride < end)
                {
                    find(at + stride);
                    load_keys();
                }
            });
        if (at + stride < end)
        {
            load_both_values();
        }
    }

    // Waves 2 and 3 to 0 and 1, then 1 to 0.
#pragma unroll
    for (int half = 2; half >= 1; half /= 2)
    {
        if (warp >= half && warp < 2 * half)
        {
#pragma unroll
            for (int t = 0; t < Parts; ++t)
            {
                sums[t].store(joined + ((warp - half) * Parts + t) * record, lane);
            }
        }
        __syncthreads();
        if (warp < half)
        {
#pragma unroll
            for (int t = 0; t < Parts; ++t)
            {
                sums[t].join(joined + (warp * Parts + t) * record, lane);
            }
        }
        __syncthreads();
    }
    if (warp == 0)
    {
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            if (p.row + 16 * t < p.nodes * l.group)
            {
                finish<HW, Half>(l, p, unit, p.row + 16 * t, lane, sums[t]);
            }
        }
    }
}

// A tile is 128 rows, 32 a wave. Two blocks lie in LDS in operand order while the next two are
// under way to registers, a quarter a wave: 16 keys, and 16 keys' values paired.
template <int HW, bool Half> __global__ __launch_bounds__(64 * waves, 2) void staged_kernel(Launch l)
{
    constexpr int depth = HW / 32, step = HW / 16, parts = 2, rows = 16 * parts * waves, keys = 2 * block;
    // [buffer][block][half, d or j][lane] 16 bytes each.
    __shared__ u32x4 key_tile[2][2][2 * depth][64];
    __shared__ u32x4 value_tile[2][2][step][64];
    __shared__ unsigned exists[2][2][2], poison[2][2][2]; // [buffer][block][half]
    const int lane = threadIdx.x % 64, warp = __builtin_amdgcn_readfirstlane(int(threadIdx.x / 64));
    int unit, tile;
    unit_of(l, unit, tile);
    Place p;
    if (unit >= l.units || !place_of(l, unit, tile * rows, rows, p) || p.split >= chunks_of(l, p))
    {
        return;
    }
    const int begin = p.split * l.chunk, end = chunk_end(l, p);
    const int row = p.row + 16 * parts * warp;
    const bool idle = row >= p.nodes * l.group;
    const int open = l.mask ? p.length : p.length + row / l.group + 1;
    u32x4 query[parts][depth];
    int node[parts];
    Sums<HW> sums[parts];
#pragma unroll
    for (int t = 0; t < parts; ++t)
    {
        load_query<HW>(l, p, row + 16 * t, lane, query[t], node[t]);
        sums[t].clear();
    }

    // A wave's quarter: half `half` of block `which`.
    const int which = warp / 2, half = warp % 2;
    u32x4 key[depth];
    unsigned value[4][HW / 32];
    bool there = false;
    const auto load = [&](int at)
    {
        const std::size_t base =
            locate(l, p, at + block * which + 16 * half, there) + std::size_t(p.head) * HW;
#pragma unroll
        for (int d = 0; d < depth; ++d)
        {
            key[d] = *reinterpret_cast<const u32x4*>(l.keys + base + lane % 16 * l.row_stride + lane / 16 * 8 + 32 * d);
        }
        load_values<HW>(l.values + base, l.row_stride, lane, value);
    };
    const auto stage = [&](int at, int buffer)
    {
        const int mine = at + block * which;
        const unsigned here = half ? 0xffff0000u : 0xffffu;
        unsigned exist = here, poisoned = 0;
        if (mine + block > min(p.length, end) || !there)
        {
            exist = there ? low_bits(end - mine) & here : 0u;
            poisoned = clean<HW, Half>(value, half, exist, low_bits(p.length - mine), lane);
        }
        if (lane == 0)
        {
            exists[buffer][which][half] = exist;
            poison[buffer][which][half] = poisoned;
        }
#pragma unroll
        for (int d = 0; d < depth; ++d)
        {
            key_tile[buffer][which][half * depth + d][lane] = key[d];
        }
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            const u32x2 v = {pair<HW>(value, 0, j), pair<HW>(value, 2, j)};
            reinterpret_cast<u32x2*>(&value_tile[buffer][which][j][lane])[half] = v;
        }
    };
    int buffer = 0;
    if (begin < end)
    {
        load(begin);
        stage(begin, 0);
    }
    __syncthreads();
    for (int at = begin; at < end; at += keys, buffer ^= 1)
    {
        const bool more = at + keys < end;
        if (more)
        {
            load(at + keys);
        }
        if (!idle)
        {
#pragma unroll
            for (int b = 0; b < 2; ++b)
            {
                const unsigned exist =
                    __builtin_amdgcn_readfirstlane(exists[buffer][b][0] | exists[buffer][b][1]);
                const unsigned poisoned =
                    __builtin_amdgcn_readfirstlane(poison[buffer][b][0] | poison[buffer][b][1]);
                if (exist)
                {
                    attend<HW, Half, parts>(
                        l, p, at + block * b, exist == ~0u && at + block * (b + 1) <= open, exist, poisoned, lane, query,
                        node, sums, [&](int h, int d) { return key_tile[buffer][b][h * depth + d][lane]; },
                        [&](int j) { return value_tile[buffer][b][j][lane]; }, [] {});
                }
            }
        }
        if (more)
        {
            stage(at + keys, buffer ^ 1);
        }
        __syncthreads();
    }
    if (!idle)
    {
#pragma unroll
        for (int t = 0; t < parts; ++t)
        {
            if (row + 16 * t < p.nodes * l.group)
            {
                finish<HW, Half>(l, p, unit, row + 16 * t, lane, sums[t]);
            }
        }
    }
}

// Joins the chunks of 16 rows of a (sequence, head), in ascending order: a wave takes
// coordinates i of a lane's four.
template <int HW, bool Half> __global__ __launch_bounds__(256) void join_kernel(Launch l, int tile_rows)
{
    constexpr int step = HW / 16, record = Sums<HW>::words * 64;
    const int lane = threadIdx.x % 64, i = threadIdx.x / 64;
    const int part = blockIdx.x % l.parts, pair = blockIdx.x / l.parts;
    const int head = pair % l.heads, sequence = pair / l.heads;
    const auto unit = [&](int split) { return (sequence * l.splits + split) * l.heads + head; };
    Place p;
    // The chunks are those of the tile that the rows were in.
    if (!place_of(l, unit(0), 16 * part / tile_rows * tile_rows, tile_rows, p))
    {
        return;
    }
    const int chunks = chunks_of(l, p), row = 16 * part + lane % 16;
    if (chunks == 1 || row / l.group >= p.nodes)
    {
        return;
    }
    const float* const first = l.partial + (std::size_t(unit(0)) * l.parts + part) * record + lane;
    const std::size_t apart = std::size_t(l.heads) * l.parts * record;
    float reference = minus_infinity;
    for (int split = 0; split < chunks; ++split)
    {
        reference = fmaxf(reference, first[split * apart + 4 * step * 64]);
    }
    float total = 0, out[step] = {};
#pragma unroll 4
    for (int split = 0; split < chunks; ++split)
    {
        const float* const from = first + split * apart;
        const float other = from[4 * step * 64];
        const float factor = other == reference ? 1.0f : __builtin_amdgcn_exp2f(other - reference);
        total += from[(4 * step + 1) * 64] * factor;
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            out[j] += from[(i * step + j) * 64] * factor;
        }
    }
    write_part<HW, Half>(l, p, row, lane, i, out, total);
}

// The launch's shape: it depends on what the host knows, sizes and not lengths.
struct Shape
{
    int parts_a_tile; // 16-row parts of a workgroup's tile: 1 or 2 (direct), 8 (staged)
    int tiles, parts, splits, chunk;
    std::size_t units, record;
};

Shape shape_of(const PagedCache& cache, const PagedRows& rows)
{
    Shape s;
    const std::size_t group = std::size_t(rows.heads / cache.heads), queries = std::size_t(rows.max_rows) * group;
    s.parts = int((queries + 15) / 16);
    s.parts_a_tile = s.parts <= 2 ? s.parts : 8;
    s.tiles = (s.parts + s.parts_a_tile - 1) / s.parts_a_tile;
    const std::size_t pairs = std::size_t(cache.sequences) * cache.heads;
    const std::size_t slots = (s.parts_a_tile == 1 ? 3 : 2) * std::size_t(compute_units());
    const std::size_t wanted = std::max<std::size_t>(1, slots / (pairs * s.tiles));
    const std::size_t most = std::max<std::size_t>(1, (rows.max_length + 255) / 256);
    s.splits = int(std::min(wanted, most));
    constexpr std::size_t keys = block * waves;
    s.chunk = int(((rows.max_length + s.splits - 1) / s.splits + keys - 1) / keys * keys);
    s.chunk = std::max<int>(s.chunk, keys);
    s.units = pairs * s.splits;
    s.record = 64 * std::size_t(cache.head_width / 4 + 2);
    return s;
}

template <int HW, bool Half> void launch(const Launch& l, const Shape& s, std::size_t pairs, hipStream_t stream)
{
    const unsigned grid = unsigned((s.units + 7) / 8 * 8 * std::size_t(s.tiles));
    const std::size_t lds = 2 * Sums<HW>::words * 64 * 4;
    switch (s.parts_a_tile)
    {
    case 1: direct_kernel<HW, Half, 1><<<grid, 64 * waves, lds, stream>>>(l); break;
    case 2: direct_kernel<HW, Half, 2><<<grid, 64 * waves, 2 * lds, stream>>>(l); break;
    default: staged_kernel<HW, Half><<<grid, 64 * waves, 0, stream>>>(l); break;
    }
    check_hip(hipGetLastError(), "paged attention launch");
    if (s.splits > 1)
    {
        join_kernel<HW, Half><<<unsigned(pairs * s.parts), 256, 0, stream>>>(l, 16 * s.parts_a_tile);
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
    return s.splits > 1 ? s.units * s.parts * s.record * 4 : 0;
}

void attention_paged(const PagedCache& cache, int layer, const PagedRows& rows, void* workspace, std::size_t bytes,
                     hipStream_t stream)
{
    if (!rows.rows || !rows.max_rows || !cache.sequences)
    {
        return;
    }
    const Shape s = shape_of(cache, rows);
    const std::size_t pairs = std::size_t(cache.sequences) * cache.heads;
    // 2^32 work-items along x are a grid's limit.
    require((s.units + 8) * s.tiles < (std::size_t(1) << 23) && pairs * s.parts < (std::size_t(1) << 23),
            "paged attention: too many workgroups for one launch");
    require(s.splits == 1 || (workspace && bytes >= s.units * s.parts * s.record * 4),
            "paged attention: the workspace is too small");
    Launch l{};
    l.keys = cache.keys + layer * cache.layer_stride;
    l.values = cache.values + layer * cache.layer_stride;
    l.page_stride = cache.page_stride;
    l.table = cache.table;
    l.table_stride = cache.table_stride;
    l.held = cache.held;
    l.lengths = cache.lengths;
    l.starts = rows.starts;
    l.query = rows.query;
    l.query_stride = rows.query_stride;
    l.out = rows.out;
    l.out_stride = rows.out_stride;
    l.mask = rows.mask;
    l.partial = static_cast<float*>(workspace);
    l.row_stride = unsigned(cache.row_stride);
    l.pages = cache.pages;
    l.page_shift = __builtin_ctz(unsigned(cache.page_rows));
    l.heads = cache.heads;
    l.group = rows.heads / cache.heads;
    l.rows = rows.rows;
    l.max_rows = rows.max_rows;
    l.words = int(rows.words);
    l.tiles = s.tiles;
    l.parts = s.parts;
    l.splits = s.splits;
    l.chunk = s.chunk;
    l.units = int(s.units);
    l.negative = rows.scale < 0;
    l.scale_log2 = (l.negative ? -rows.scale : rows.scale) * 1.44269504088896340736f;
    const auto by_type = [&](auto width)
    {
        constexpr int HW = decltype(width)::value;
        cache.half ? launch<HW, true>(l, s, pairs, stream) : launch<HW, false>(l, s, pairs, stream);
    };
    cache.head_width == 64 ? by_type(std::integral_constant<int, 64>{}) : by_type(std::integral_constant<int, 128>{});
}
} // namespace tsac_hip

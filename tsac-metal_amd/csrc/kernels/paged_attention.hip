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
// operand needs eight keys of one coordinate per lane: LDS transposes values as they are read.
//
// Rows of the cache go from memory straight into LDS, in whole lines. Up to 32 query rows
// (narrow_kernel) the cache's bytes are what costs: a wave takes all rows and every eighth block
// of its workgroup's chunk of keys, through LDS of its own. More rows (staged_kernel) cost
// products and exponentials: a wave takes 32 rows, and all eight of a workgroup read the same
// stages of keys. Chunks are joined in ascending order by join_kernel.
#include "paged.hpp"

#include <algorithm>
#include <type_traits>

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

constexpr int waves = 8;     // of a workgroup
constexpr int few_waves = 2; // where there are many, of short sequences
constexpr int block = 32;    // keys of one step
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

__device__ __forceinline__ float maximum(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
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
    int together;      // of them that one die takes
    unsigned first;    // workgroup of the launch
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
    // What no page holds nobody sees, however long a sequence says it is.
    p.total = min(p.total, max(p.limit, 0) << l.page_shift);
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

// A number that no kernel writes meanwhile, through the scalar cache: as a vector load, which the
// compiler makes it beside assembly that touches memory, its wait would be one for all loads
// of keys and values in flight (64 nodes over 131,001 positions: 187 us so).
__device__ __forceinline__ int scalar_load(const int* from)
{
    return *(const __attribute__((address_space(4))) int*)reinterpret_cast<std::uintptr_t>(from);
}

// Where 16 keys from a position start, as an offset into keys and values; `there` if they lie in
// a page of the pool, otherwise the offset is some page's.
__device__ __forceinline__ std::size_t locate(const Launch& l, const Place& p, int position, bool& there)
{
    const int index = position >> l.page_shift;
    const int read = scalar_load(l.table + p.sequence * l.table_stride + max(min(index, p.limit - 1), 0));
    there = index < p.limit && read >= 0 && read < l.pages;
    return (there ? read : 0) * l.page_stride + std::size_t(position & ((1 << l.page_shift) - 1)) * l.row_stride;
}

// One 16-row part's running sums. A lane has row lane % 16 and its coordinates
// 16 * j + 4 * (lane / 16) + i.
template <int HW> struct Sums
{
    static constexpr int step = HW / 16;
    static constexpr int words = 4 * step + 2; // a lane's, joined within a workgroup
    static constexpr int record = 16 * HW + 32; // floats of a chunk's record: [row][HW], references, sums
    f32x4 out[step]; // [j][i]
    f32x4 total;     // four times the same
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
    // [word][lane]
    __device__ __forceinline__ void hand_over(float* to, int lane) const
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
    __device__ __forceinline__ void store(float* to, int lane) const
    {
        const int row = lane % 16;
#pragma unroll
        for (int j = 0; j < step; ++j)
        {
            *reinterpret_cast<f32x4*>(to + row * HW + 16 * j + 4 * (lane / 16)) = out[j];
        }
        if (lane < 16)
        {
            to[16 * HW + row] = reference;
            to[16 * HW + 16 + row] = total[0];
        }
    }
};

// Coordinates of one row from `first` on, divided by the row's sum. A row that no key reached is 0.
template <int HW, bool Half, int Count>
__device__ __forceinline__ void write_row(const Launch& l, const Place& p, int row, int first, const float (&values)[Count],
                                          float total)
{
    const int node = row / l.group, head = p.head * l.group + row % l.group;
    const float inverse = 1.0f / total;
    unsigned word[Count / 2];
#pragma unroll
    for (int k = 0; k < Count / 2; ++k)
    {
        word[k] = total == 0 ? 0u : pack<Half>(values[2 * k] * inverse, values[2 * k + 1] * inverse);
    }
    uint16_t* const to = l.out + std::size_t(p.first + node) * l.out_stride + std::size_t(head) * HW + first;
    __builtin_memcpy(__builtin_assume_aligned(to, sizeof word), word, sizeof word);
}

// A part's sums: to the output, or as the chunk's record.
template <int HW, bool Half>
__device__ __forceinline__ void finish(const Launch& l, const Place& p, int unit, int row, int lane,
                                       const Sums<HW>& sums)
{
    if (chunks_of(l, p) > 1)
    {
        sums.store(l.partial + (std::size_t(unit) * l.parts + row / 16) * Sums<HW>::record, lane);
        return;
    }
    const int mine = row + lane % 16;
    if (mine / l.group < p.nodes)
    {
#pragma unroll
        for (int j = 0; j < Sums<HW>::step; ++j)
        {
            const float values[4] = {sums.out[j][0], sums.out[j][1], sums.out[j][2], sums.out[j][3]};
            write_row<HW, Half>(l, p, mine, 16 * j + 4 * (lane / 16), values, sums.total[0]);
        }
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
    const uint16_t* const from = l.values + base + std::size_t(key % 16) * l.row_stride;
    if (live && there)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
#pragma unroll
            for (int j = 0; j < step; ++j)
            {
                const uint16_t bits = from[16 * j + 4 * (lane / 16) + i];
                sums.out[j][i] += nonfinite<Half>(bits) ? weight * widen<Half>(bits) : 0.0f;
            }
        }
    }
}

// What masks ask of a block: which keys exist, and which new ones have values that are not finite.
struct Marks
{
    unsigned exist, poisoned;
};

// A block's scores for `Parts` parts of 16 rows, unscaled: keys 16 * half + 4 * (lane / 16) + i.
template <int HW, bool Half, int Parts>
__device__ __forceinline__ void score_block(const u32x4 (&key)[2][HW / 32], const u32x4 (&query)[Parts][HW / 32],
                                            f32x4 (&score)[Parts][2])
{
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            score[t][half] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int d = 0; d < HW / 32; ++d)
        {
#pragma unroll
            for (int t = 0; t < Parts; ++t)
            {
                score[t][half] = product<Half>(key[half][d], query[t][d], score[t][half]);
            }
        }
    }
}

// The weight of a score that a reference is moved to, as a power of two: weights and their sums have it as a
// factor, which leaves their quotient. Weights in half are subnormal below 2^-14 and nothing below
// 2^-25, and a long context can have most of its sum in such ones: with 2^7, of the 2^16 there is, they are
// lost below 2^-32 of the largest. BF16 has the range of 32 bits.
template <bool Half> constexpr float weight_log2 = Half ? 7.0f : 0.0f;

// Moves the running references, if need be, before a block's scores are weighed: only when a
// score passes what one was moved to by 2^8. Weights stay in range without it, and most blocks need neither the
// exchange nor the scaling. By how much it passes one is computed as its weight is: where scores are so large that
// neighbouring numbers lie far apart, a rounded bound would let weights in half past their range.
template <int HW, bool Half, int Parts>
__device__ __forceinline__ void settle(const Launch& l, const f32x4 (&score)[Parts][2], Sums<HW> (&sums)[Parts])
{
    float most[Parts];
    bool move = false;
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        const f32x4 a = score[t][0], b = score[t][1];
        // Of scores that are not numbers it is none either, and so is the row.
        most[t] = maximum(maximum(maximum(a[0], a[1], a[2]), a[3], b[0]), maximum(b[1], b[2], b[3]), b[3]);
        // Of -infinity alone it is no number, or less.
        move = move || __builtin_fmaf(most[t], l.scale_log2, -sums[t].reference) > 8.0f + weight_log2<Half>;
    }
    if (__any(move))
    {
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            const float score = query_max(most[t]);
            // Not a product with -infinity, which a scale of 0 would make no number.
            const float to = score == minus_infinity ? score : score * l.scale_log2 - weight_log2<Half>;
            sums[t].move(fmaxf(to, sums[t].reference));
        }
    }
}

// Weights of a block's scores against the references.
template <int HW, bool Half, int Parts>
__device__ __forceinline__ void weigh(const Launch& l, const f32x4 (&score)[Parts][2],
                                      const Sums<HW> (&sums)[Parts], u32x4 (&weight)[Parts])
{
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        // Where no key had a score the reference is -infinity, and so are the scores.
        const float reference = sums[t].reference == minus_infinity ? 0.0f : sums[t].reference;
        float e[8];
#pragma unroll
        for (int slot = 0; slot < 8; ++slot)
        {
            e[slot] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[t][slot / 4][slot % 4], l.scale_log2, -reference));
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
        {
            weight[t][w] = pack<Half>(e[2 * w], e[2 * w + 1]);
        }
    }
}

// Adds a block's weighted values; value[j]: coordinate 16 * j + lane % 16 of its keys. The
// sum of a row's weights, as they are rounded, is one more product.
template <int HW, bool Half, int Parts>
__device__ __forceinline__ void add_block(const u32x4 (&weight)[Parts], Sums<HW> (&sums)[Parts], const u32x4 (&value)[HW / 16])
{
    constexpr unsigned one = Half ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        sums[t].total = product<Half>(u32x4{one, one, one, one}, weight[t], sums[t].total);
    }
#pragma unroll
    for (int j = 0; j < HW / 16; ++j)
    {
        const u32x4 v = value[j];
#pragma unroll
        for (int t = 0; t < Parts; ++t)
        {
            sums[t].out[j] = product<Half>(v, weight[t], sums[t].out[j]);
        }
    }
}

// A block with masks: the keys that a row does not see weigh nothing, whatever they are.
template <int HW, bool Half, int Parts>
__device__ __forceinline__ void attend_masked(const Launch& l, const Place& p, int at, Marks marks, int lane,
                                              const u32x4 (&key)[2][HW / 32], const u32x4 (&query)[Parts][HW / 32],
                                              const int (&node)[Parts], Sums<HW> (&sums)[Parts], const u32x4 (&value)[HW / 16])
{
    f32x4 score[Parts][2];
    score_block<HW, Half>(key, query, score);
    unsigned live[Parts];
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        live[t] = seen(l, p, at, marks.exist, node[t]);
#pragma unroll
        for (int slot = 0; slot < 8; ++slot)
        {
            f32x4& x = score[t][slot / 4];
            x[slot % 4] = live[t] >> (16 * (slot / 4) + 4 * (lane / 16) + slot % 4) & 1 ? x[slot % 4] : minus_infinity;
        }
    }
    settle<HW, Half>(l, score, sums);
    u32x4 weight[Parts];
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        const float reference = sums[t].reference == minus_infinity ? 0.0f : sums[t].reference;
        float e[8];
#pragma unroll
        for (int slot = 0; slot < 8; ++slot)
        {
            // Chosen once more: a scale of 0 makes no number of -infinity.
            const float x =
                __builtin_amdgcn_exp2f(__builtin_fmaf(score[t][slot / 4][slot % 4], l.scale_log2, -reference));
            e[slot] = live[t] >> (16 * (slot / 4) + 4 * (lane / 16) + slot % 4) & 1 ? x : 0.0f;
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
        {
            weight[t][w] = pack<Half>(e[2 * w], e[2 * w + 1]);
        }
        for (unsigned left = marks.poisoned; left; left &= left - 1)
        {
            const int k = __builtin_ctz(left);
            float x = e[0];
#pragma unroll
            for (int slot = 1; slot < 8; ++slot)
            {
                x = 4 * (k / 16) + k % 4 == slot ? e[slot] : x;
            }
            x = __shfl(x, k % 16 / 4 * 16 + lane % 16);
            add_poisoned<HW, Half>(l, p, at, k, x, live[t] >> k & 1, lane, sums[t]);
        }
    }
    add_block<HW, Half>(weight, sums, value);
}

// 16 bytes a lane, from `offset` bytes behind `from`, to `to`, lane after lane; the wave waits for it
// with its other loads (s_waitcnt vmcnt). Written out because the compiler would wait for it
// before any other read of LDS. A load to LDS needs a wait state behind a write of M0, which the
// compiler does not put into assembly. M0 is reserved, so that clang warns where it is named; nothing
// else uses it. `Once`: past the caches.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <bool Once> __device__ __forceinline__ void load_to_lds(const void* from, unsigned offset, void* to)
{
    const unsigned address = __builtin_amdgcn_readfirstlane(
        unsigned(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) const void*)to)));
    if constexpr (Once)
    {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(offset), "s"(from),
                     "s"(address)
                     : "memory", "m0");
    }
    else
    {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(from),
                     "s"(address)
                     : "memory", "m0");
    }
}
#pragma clang diagnostic pop

// Four keys of coordinate lane % 16 of the 16 that start at each four lanes' rows: lanes 4 r .. 4 r + 3
// of 16 name row r.
__device__ __forceinline__ u32x2 read_transposed(const char* from)
{
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from));
}

// Drops from `Pieces` KiB of values in LDS, whole rows, those of keys that do not exist (a weight of
// zero would not drop one that is not finite), and those not finite of new rows, which only some
// queries see. Returns the bits of the latter's keys.
template <int HW, bool Half, int Pieces>
__device__ __forceinline__ unsigned clean(char* values, unsigned exist, unsigned cached, int lane)
{
    constexpr int lanes = HW / 8, rows_a_piece = 64 / lanes; // lanes of a row
    unsigned poisoned = 0;
#pragma unroll 1
    for (int i = 0; i < Pieces; ++i)
    {
        const int key = i * rows_a_piece + lane / lanes;
        u32x4& v = *reinterpret_cast<u32x4*>(values + i * 1024 + lane * 16);
        u32x4 x = v;
        const bool here = exist >> key & 1, fresh = !(cached >> key & 1);
        bool wrong = false;
#pragma unroll
        for (int w = 0; w < 4; ++w)
        {
            const unsigned keep = (nonfinite<Half>(uint16_t(x[w])) ? 0u : 0xffffu) |
                                  (nonfinite<Half>(uint16_t(x[w] >> 16)) ? 0u : 0xffff0000u);
            wrong = wrong || keep != ~0u;
            x[w] = !here ? 0u : fresh ? x[w] & keep : x[w];
        }
        v = x;
        const uint64_t bad = __ballot(wrong && here && fresh);
#pragma unroll
        for (int k = 0; k < rows_a_piece; ++k)
        {
            poisoned |= (bad >> k * lanes & ((1ull << lanes) - 1) ? 1u : 0u) << (i * rows_a_piece + k);
        }
    }
    return poisoned;
}

// clean() for a stage, eight keys a wave, for the whole workgroup.
template <int HW, bool Half>
__device__ __forceinline__ void clean_stage(const Launch& l, const Place& p, int at, int end, int warp, int lane,
                                            char* values, Marks* marked)
{
    const int first = at + 8 * warp; // of the wave's keys
    bool there;
    locate(l, p, first / 16 * 16, there);
    const unsigned exist = there ? low_bits(end - first) & 0xff : 0u;
    const unsigned poisoned =
        clean<HW, Half, HW / 64>(values + warp * (HW / 64) * 1024, exist, low_bits(p.length - first), lane);
    if (lane == 0)
    {
        marked[warp] = Marks{exist, poisoned};
    }
    __syncthreads();
}

// Whether every page from one position to another is there, for the whole workgroup.
template <int Threads>
__device__ __forceinline__ bool all_there(const Launch& l, const Place& p, int from, int to, int& flag)
{
    const int first = from >> l.page_shift, last = (to - 1) >> l.page_shift;
    bool good = true;
    for (int i = first + int(threadIdx.x); i <= last; i += Threads)
    {
        const int page = i < p.limit ? l.table[p.sequence * l.table_stride + i] : -1;
        good = good && page >= 0 && page < l.pages;
    }
    if (threadIdx.x == 0)
    {
        flag = 1;
    }
    __syncthreads();
    if (!good)
    {
        flag = 0;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(flag);
}

// Workgroups go round the eight dies. A unit's tiles, which read the same keys, follow one another
// on one die, and so do `together` heads of a chunk, which read the rows of the same positions:
// where a die reads one head alone, its requests meet in two of its cache's sixteen channels.
__device__ __forceinline__ void unit_of(const Launch& l, int& unit, int& tile)
{
    const unsigned index = l.first + blockIdx.x;
    const int die = index % 8, i = index / 8, j = i / l.tiles;
    tile = i % l.tiles;
    unit = (j / l.together * 8 + die) * l.together + j % l.together;
}

// How far the 16-byte pieces of a key row and the 32-byte pieces of a value row are shifted in LDS (by
// exclusive or), so that a piece of 16 rows meets every bank: 16 keys' pieces are read at a time,
// and 16 value rows' transposed.
template <int HW> __device__ __forceinline__ int key_shift(int row)
{
    return HW == 128 ? row & 15 : row >> 1 & 7;
}
template <int HW> __device__ __forceinline__ int value_shift(int row)
{
    return HW == 128 ? row & 7 : row >> 1 & 3;
}

// At most `count` of the wave's memory operations still under way (they complete in order).
template <int Count> __device__ __forceinline__ void wait_memory()
{
    static_assert(Count < 16);
    __builtin_amdgcn_s_waitcnt(Count | 7 << 4 | 15 << 8);
    asm volatile("" ::: "memory"); // no read of LDS moves in front
}

__device__ __forceinline__ void wait_lds()
{
    __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);
    asm volatile("" ::: "memory");
}

// Reads a block's operands from where its rows lie in LDS.
template <int HW> struct Reading
{
    static constexpr int row_bytes = 2 * HW;
    int key_lane, key_shifted, value_lane, value_shifted;

    __device__ explicit Reading(int lane)
    {
        const int key_row = lane % 16, value_row = lane % 16 / 4 + 4 * (lane / 16); // of a half, by the lane's address
        key_lane = key_row * row_bytes;
        key_shifted = 16 * (lane / 16 ^ key_shift<HW>(key_row));
        value_lane = value_row * row_bytes + lane % 4 * 8;
        value_shifted = 32 * value_shift<HW>(value_row);
    }
    __device__ __forceinline__ void keys(const char* rows, u32x4 (&key)[2][HW / 32]) const
    {
        const char* const from = rows + key_lane;
#pragma unroll
        for (int d = 0; d < HW / 32; ++d)
        {
            const char* const piece = from + (64 * d ^ key_shifted);
            key[0][d] = *reinterpret_cast<const u32x4*>(piece);
            key[1][d] = *reinterpret_cast<const u32x4*>(piece + 16 * row_bytes);
        }
        asm volatile("" ::: "memory"); // here, not where they are used
    }
    __device__ __forceinline__ void values(const char* rows, u32x4 (&value)[HW / 16]) const
    {
        const char* const from = rows + value_lane;
#pragma unroll
        for (int j = 0; j < HW / 16; ++j)
        {
            const char* const piece = from + (32 * j ^ value_shifted);
            const u32x2 low = read_transposed(piece), high = read_transposed(piece + 16 * row_bytes);
            value[j] = u32x4{low[0], low[1], high[0], high[1]};
        }
        asm volatile("" ::: "memory");
    }
};

// A tile is `Parts` x 16 rows, and a wave takes every eighth (or, of two, second) block of the chunk. A block's keys and
// values come into the wave's own 16 KiB of LDS in whole rows, and the next ones are asked for
// once these are in registers: eight waves have up to 128 KiB under way, and its waves wait for nothing
// but their own loads. A token of each of 8 sequences, 264 MB of keys and values: 47 us, 5.6 TB/s,
// and 5 us for the join. Before loads went past the caches it was 52 us so, and 58 with operands
// loaded from memory into registers, 64 bytes of a row at a time.
template <int HW, bool Half, int Parts, int Waves, bool Once>
__global__ __launch_bounds__(64 * Waves, 2) void narrow_kernel(Launch l)
{
    constexpr int depth = HW / 32, step = HW / 16, row_bytes = 2 * HW, lanes = HW / 8, rows_a_piece = 64 / lanes;
    constexpr int half_pieces = 16 / rows_a_piece, pieces = 2 * half_pieces; // loads of a block's keys, or values
    constexpr int words = Sums<HW>::words * 64;
    extern __shared__ __attribute__((aligned(128))) char memory[]; // [wave]: keys [key][HW], values [key][HW]
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
    const int open = min(end, l.mask ? p.length : p.length + p.row / l.group + 1);

    char* const own = memory + warp * (2 * block * row_bytes);
    char* const own_values = own + block * row_bytes;
    unsigned key_offset[half_pieces], value_offset[half_pieces]; // bytes, of a lane, from a half's start
#pragma unroll
    for (int i = 0; i < half_pieces; ++i)
    {
        const int r = i * rows_a_piece + lane / lanes, place = lane % lanes;
        key_offset[i] = 2 * (r * l.row_stride) + 16 * (place ^ key_shift<HW>(r));
        value_offset[i] = 2 * (r * l.row_stride) + 16 * (place ^ 2 * value_shift<HW>(r));
    }
    std::size_t base[2]; // where the halves of the next block to load lie
    bool there[2];
    const auto find = [&](int at)
    {
#pragma unroll
        for (int half = 0; half < 2; ++half)
        {
            base[half] = locate(l, p, at + 16 * half, there[half]) + std::size_t(p.head) * HW;
        }
    };
    const auto load = [&](const uint16_t* rows, const unsigned (&offset)[half_pieces], char* to)
    {
#pragma unroll
        for (int half = 0; half < 2; ++half)
        {
#pragma unroll
            for (int i = 0; i < half_pieces; ++i)
            {
                load_to_lds<Once>(rows + base[half], offset[i], to + (half * half_pieces + i) * 1024);
            }
        }
    };
    int at = begin + block * warp;
    constexpr int stride = block * Waves;
    bool here[2] = {}; // `there` of the block that is worked on
    if (at < end)
    {
        find(at);
        load(l.keys, key_offset, own);
        load(l.values, value_offset, own_values);
        here[0] = there[0];
        here[1] = there[1];
        find(at + stride);
    }
    u32x4 query[Parts][depth];
    int node[Parts];
    Sums<HW> sums[Parts];
#pragma unroll
    for (int t = 0; t < Parts; ++t)
    {
        load_query<HW>(l, p, p.row + 16 * t, lane, query[t], node[t]);
        sums[t].clear();
    }
    u32x4 key[2][depth], value[step];
    const Reading<HW> reading(lane);
    // The block at `at` into registers, and the next one asked for.
    const auto take = [&](auto clean_values)
    {
        const bool more = at + stride < end;
        wait_memory<pieces>(); // the keys
        reading.keys(own, key);
        wait_lds();
        if (more)
        {
            load(l.keys, key_offset, own);
            wait_memory<pieces>(); // the values
        }
        else
        {
            wait_memory<0>();
        }
        clean_values();
        reading.values(own_values, value);
        wait_lds();
        if (more)
        {
            load(l.values, value_offset, own_values);
            here[0] = there[0];
            here[1] = there[1];
            find(at + 2 * stride);
        }
    };
    for (; at + block <= open && here[0] && here[1]; at += stride)
    {
        take([] {});
        f32x4 score[Parts][2];
        score_block<HW, Half>(key, query, score);
        settle<HW, Half>(l, score, sums);
        u32x4 weight[Parts];
        weigh<HW, Half>(l, score, sums, weight);
        add_block<HW, Half>(weight, sums, value);
    }
    // From the first block on that asks for masks.
#pragma unroll 1
    for (; at < end; at += stride)
    {
        Marks marks = {low_bits(end - at) & ((here[0] ? 0xffffu : 0u) | (here[1] ? 0xffff0000u : 0u)), 0};
        take(
            [&]
            {
                marks.poisoned = clean<HW, Half, pieces>(own_values, marks.exist, low_bits(p.length - at), lane);
                wait_lds();
            });
        attend_masked<HW, Half>(l, p, at, marks, lane, key, query, node, sums, value);
    }

    // Half the waves to the other half, down to one.
    float* const joined = reinterpret_cast<float*>(memory);
    __syncthreads();
#pragma unroll 1
    for (int half = Waves / 2; half >= 1; half /= 2)
    {
        if (warp >= half && warp < 2 * half)
        {
#pragma unroll
            for (int t = 0; t < Parts; ++t)
            {
                sums[t].hand_over(joined + ((warp - half) * Parts + t) * words, lane);
            }
        }
        __syncthreads();
        if (warp < half)
        {
#pragma unroll
            for (int t = 0; t < Parts; ++t)
            {
                sums[t].join(joined + (warp * Parts + t) * words, lane);
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

constexpr int staged_keys = 2 * block; // of a stage
constexpr int stages = 4;              // in LDS

// A tile is 256 / Teams rows, 32 a wave; a team of waves takes all stages, or every second
// block. Stages of 64 keys go from memory straight into a ring of four in LDS, eight rows a wave, in
// whole rows (4 TB/s where a load took 64 bytes of 16 rows, 5.5 so). 32 trees of 32 nodes over 4,093
// positions, 497 MB: 95 us, 5.2 TB/s; 64 nodes over 131,001, 137 GFLOP and 538 MB: 155 us and 11 for
// the join, 885 TFLOP/s with the matrix units busy 45% of the time.
template <int HW, bool Half, int Teams, bool Once>
__global__ __launch_bounds__(64 * waves, 2) void staged_kernel(Launch l)
{
    constexpr int depth = HW / 32, step = HW / 16, parts = 2, team = waves / Teams, rows = 16 * parts * team;
    constexpr int keys = staged_keys, row_bytes = 2 * HW, key_bytes = keys * row_bytes;
    constexpr int stage_bytes = 2 * key_bytes;
    constexpr int pieces = HW / 64; // 1 KiB each, of keys and of values, that a wave loads of a stage
    extern __shared__ __attribute__((aligned(128))) char ring[]; // [stage]: keys [key][HW], values [key][HW]
    __shared__ Marks marked[waves]; // of eight keys each
    __shared__ int flag;
    const int lane = threadIdx.x % 64, warp = __builtin_amdgcn_readfirstlane(int(threadIdx.x / 64));
    int unit, tile;
    unit_of(l, unit, tile);
    Place p;
    if (unit >= l.units || !place_of(l, unit, tile * rows, rows, p) || p.split >= chunks_of(l, p))
    {
        return;
    }
    const int begin = p.split * l.chunk, end = chunk_end(l, p), count = (max(end - begin, 0) + keys - 1) / keys;
    const int row = p.row + 16 * parts * (warp % team);
    const bool idle = row >= p.nodes * l.group;
    // Up to here stages are whole for every row of the tile, if the chunk's pages are all there.
    const int open = min(end, l.mask ? p.length : p.length + p.row / l.group + 1);
    const int whole =
        all_there<64 * waves>(l, p, begin, open, flag) ? max(open - begin, 0) / keys : 0; // stages

    u32x4 query[parts][depth];
    int node[parts];
    Sums<HW> sums[parts];
#pragma unroll
    for (int t = 0; t < parts; ++t)
    {
        load_query<HW>(l, p, row + 16 * t, lane, query[t], node[t]);
        sums[t].clear();
    }

    // A wave's eighth: eight rows of keys and of values, of 16-key half `half`. A row's 16-byte
    // pieces of keys and 32-byte pieces of values are shifted by its number.
    const int half = warp / 2;
    constexpr int lanes = HW / 8, rows_a_piece = 64 / lanes; // lanes of a row; rows that one load takes
    unsigned key_offset[pieces], value_offset[pieces];       // bytes, of a lane
#pragma unroll
    for (int i = 0; i < pieces; ++i)
    {
        const int r = 8 * (warp % 2) + i * rows_a_piece + lane / lanes, place = lane % lanes;
        key_offset[i] = 2 * (r * l.row_stride) + 16 * (place ^ key_shift<HW>(r));
        value_offset[i] = 2 * (r * l.row_stride) + 16 * (place ^ 2 * value_shift<HW>(r));
    }
    bool there;
    std::size_t base = 0; // where the wave's half of the next stage to load lies
    const auto find = [&](int stage)
    { base = locate(l, p, begin + keys * stage + 16 * half, there) + std::size_t(p.head) * HW; };
    const auto load = [&](int stage)
    {
        char* const to = ring + stage % stages * stage_bytes + warp * pieces * 1024;
        const char* const from_keys = reinterpret_cast<const char*>(l.keys + base);
        const char* const from_values = reinterpret_cast<const char*>(l.values + base);
#pragma unroll
        for (int i = 0; i < pieces; ++i)
        {
            load_to_lds<Once>(from_keys, key_offset[i], to + i * 1024);
            load_to_lds<Once>(from_values, value_offset[i], to + key_bytes + i * 1024);
        }
        find(stage + 1);
    };
    int issued = 0; // stages asked for
    const auto load_up_to = [&](int last)
    {
        for (; issued <= min(last, count - 1); ++issued)
        {
            load(issued);
        }
    };
    // Stage `next` is in LDS, as are those in front of it, for all waves, and what they have read
    // of LDS is in registers.
    const auto arrive = [&](int next)
    {
        switch (issued - 1 - next)
        {
        case 3: wait_memory<3 * 2 * pieces>(); break;
        case 2: wait_memory<2 * 2 * pieces>(); break;
        case 1: wait_memory<2 * pieces>(); break;
        default: wait_memory<0>(); break;
        }
        __syncthreads();
    };
    find(0);
    // One team works on block 0 of a stage while the stage in front of it is still read for block 1
    // by others; of two teams each is done with a stage once it has its values.
    constexpr int ahead = Teams == 1 ? 2 : 3;
    load_up_to(ahead);
    arrive(Teams - 1);

    u32x4 key[2][depth], value[step];
    const Reading<HW> reading(lane);
    const auto read_keys = [&](int stage, int b)
    { reading.keys(ring + stage % stages * stage_bytes + b * block * row_bytes, key); };
    const auto read_values = [&](int stage, int b)
    { reading.values(ring + stage % stages * stage_bytes + key_bytes + b * block * row_bytes, value); };
    const int mine = Teams == 1 ? 0 : warp / team; // the first block of a stage that the wave takes
    int stage = 0;
    if (idle)
    {
        for (; stage < whole; ++stage)
        {
            arrive(stage + Teams);
            load_up_to(stage + ahead + 1);
        }
    }
    else if (whole)
    {
        // The next block's scores are products while this block's weights are exponentials: a wave
        // has work for both units at any time. Keys and values are read from LDS a phase before
        // they are used.
        f32x4 score[parts][2], next[parts][2];
        u32x4 weight[parts];
        read_keys(0, mine);
        score_block<HW, Half>(key, query, score);
        read_keys(Teams == 1 ? 0 : 1, Teams == 1 ? 1 : mine);
        settle<HW, Half>(l, score, sums);
        const auto turn = [&](f32x4(&now)[parts][2], f32x4(&then)[parts][2], int block_stage, int b, int key_stage, int key_b,
                              bool last, auto between)
        {
            read_values(block_stage, b);
            score_block<HW, Half>(key, query, then);
            weigh<HW, Half>(l, now, sums, weight);
            between();
            read_keys(key_stage, key_b);
            add_block<HW, Half>(weight, sums, value);
            if (!last)
            {
                settle<HW, Half>(l, then, sums);
            }
        };
        // While there are stages to ask for, nothing of a turn depends on their number.
        const auto steady = [&]
        {
            wait_memory<2 * pieces>();
            __syncthreads();
            load(issued);
            ++issued;
        };
        const auto drain = [&]
        {
            arrive(stage + Teams);
            load_up_to(stage + ahead + 1);
        };
        const int enough = min(whole - 1, count - ahead - 1); // up to here a stage is asked for in each
        if constexpr (Teams == 1)
        {
            for (; stage < enough; ++stage)
            {
                turn(score, next, stage, 0, stage + 1, 0, false, steady);
                turn(next, score, stage, 1, stage + 1, 1, false, [] {});
            }
#pragma unroll 1
            for (; stage < whole; ++stage)
            {
                turn(score, next, stage, 0, stage + 1, 0, false, drain);
                turn(next, score, stage, 1, stage + 1, 1, stage + 1 == whole, [] {});
            }
        }
        else
        {
            for (; stage + 1 < enough; stage += 2)
            {
                turn(score, next, stage, mine, stage + 2, mine, false, steady);
                turn(next, score, stage + 1, mine, stage + 3, mine, false, steady);
            }
#pragma unroll 1
            for (; stage < whole; ++stage)
            {
                turn(score, next, stage, mine, stage + 2, mine, stage + 1 == whole, drain);
#pragma unroll
                for (int t = 0; t < parts; ++t)
                {
                    score[t][0] = next[t][0];
                    score[t][1] = next[t][1];
                }
            }
        }
    }
    for (; stage < count; ++stage)
    {
        const int at = begin + keys * stage;
        arrive(stage);
        load_up_to(stage + stages - 1);
        clean_stage<HW, Half>(l, p, at, end, warp, lane, ring + stage % stages * stage_bytes + key_bytes, marked);
#pragma unroll 1
        for (int b = mine; b < 2 && !idle; b += Teams)
        {
            Marks marks = {0, 0};
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                marks.exist |= marked[4 * b + w].exist << 8 * w;
                marks.poisoned |= marked[4 * b + w].poisoned << 8 * w;
            }
            marks.exist = __builtin_amdgcn_readfirstlane(marks.exist);
            marks.poisoned = __builtin_amdgcn_readfirstlane(marks.poisoned);
            if (marks.exist)
            {
                read_keys(stage, b);
                read_values(stage, b);
                attend_masked<HW, Half>(l, p, at + block * b, marks, lane, key, query, node, sums, value);
            }
        }
    }
    __syncthreads();
    if constexpr (Teams == 2)
    {
        constexpr int words = Sums<HW>::words * 64;
        float* const joined = reinterpret_cast<float*>(ring) + warp % team * parts * words;
        if (warp >= team && !idle)
        {
#pragma unroll
            for (int t = 0; t < parts; ++t)
            {
                sums[t].hand_over(joined + t * words, lane);
            }
        }
        __syncthreads();
        if (warp < team && !idle)
        {
#pragma unroll
            for (int t = 0; t < parts; ++t)
            {
                sums[t].join(joined + t * words, lane);
            }
        }
    }
    if (warp < team)
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

// Joins the chunks of 16 rows of a (sequence, head), in ascending order.
template <int HW, bool Half> __global__ __launch_bounds__(256) void join_kernel(Launch l, int tile_rows)
{
    constexpr int step = HW / 16, record = Sums<HW>::record; // coordinates of a thread
    const int mine = threadIdx.x / 16, first = threadIdx.x % 16 * step;
    const int part = blockIdx.x % l.parts, pair = blockIdx.x / l.parts;
    const int head = pair % l.heads, sequence = pair / l.heads;
    const int unit = sequence * l.splits * l.heads + head; // of the first chunk
    Place p;
    // The chunks are those of the tile that the rows were in.
    if (!place_of(l, unit, 16 * part / tile_rows * tile_rows, tile_rows, p))
    {
        return;
    }
    const int chunks = chunks_of(l, p), row = 16 * part + mine;
    if (chunks == 1 || row / l.group >= p.nodes)
    {
        return;
    }
    const float* const records = l.partial + (std::size_t(unit) * l.parts + part) * record;
    const std::size_t apart = std::size_t(l.heads) * l.parts * record;
    // Eight chunks are read at a time, the last one again past the end, where it counts nothing.
    constexpr int together = 8;
    float reference = minus_infinity, total = 0, out[step] = {};
    for (int base = 0; base < chunks; base += together)
    {
        float other[together], part_total[together], part_out[together][step];
#pragma unroll
        for (int c = 0; c < together; ++c)
        {
            const float* const from = records + min(base + c, chunks - 1) * apart;
            other[c] = from[16 * HW + mine];
            part_total[c] = from[16 * HW + 16 + mine];
            __builtin_memcpy(part_out[c], __builtin_assume_aligned(from + mine * HW + first, 16), sizeof part_out[c]);
        }
        float most = reference;
#pragma unroll
        for (int c = 0; c < together; ++c)
        {
            most = fmaxf(most, other[c]);
        }
        const float ours = reference == most ? 1.0f : __builtin_amdgcn_exp2f(reference - most);
        reference = most;
        total *= ours;
#pragma unroll
        for (int k = 0; k < step; ++k)
        {
            out[k] *= ours;
        }
#pragma unroll
        for (int c = 0; c < together; ++c)
        {
            const float factor = other[c] == most ? 1.0f : __builtin_amdgcn_exp2f(other[c] - most);
            if (base + c < chunks)
            {
                total += part_total[c] * factor;
#pragma unroll
                for (int k = 0; k < step; ++k)
                {
                    out[k] += part_out[c][k] * factor;
                }
            }
        }
    }
    write_row<HW, Half>(l, p, row, first, out, total);
}

// The launch's shape: it depends on what the host knows, sizes and not lengths.
struct Shape
{
    int parts_a_tile; // 16-row parts of a workgroup's tile: 1 or 2 (narrow), 8 or 16 (staged)
    int tiles, parts, splits, chunk;
    std::size_t units, record;
    int narrow_waves; // of a workgroup
    bool once;        // keys and values go past the caches
};

Shape shape_of(const PagedCache& cache, const PagedRows& rows)
{
    Shape s;
    const std::size_t group = std::size_t(rows.heads / cache.heads), queries = std::size_t(rows.max_rows) * group;
    s.parts = int((queries + 15) / 16);
    const std::size_t pairs = std::size_t(cache.sequences) * cache.heads;
    // A wave of the narrow kernel has registers for 32 rows: 64 us, call and join included, for 32
    // over 8,190 positions of 8 sequences, 8 heads, where the staged kernel takes 65; 11 for 18 with
    // 12 rows over 1,021 of 3, 16 heads. Above that tiles of 128 rows, of which more start at once (2
    // prompts of 500 rows over 2,580 positions, 16 heads: 34 us for 40, with the join; 2 trees of 64
    // nodes over 16,381, four query heads to each of 8: 59 for 65), or of 256, which read a chunk's
    // keys half as often, where these give each unit 2,048 keys (4 prompts of 500 rows over 6,001:
    // 228 us for 246; 64 nodes over 131,001: 192 for 206).
    const std::size_t tall_tiles = pairs * ((s.parts + 15) / 16);
    const bool tall =
        s.parts > 8 && tall_tiles * std::max<std::size_t>(1, rows.max_length / 2048) >= std::size_t(compute_units());
    // Where there are more (sequence, head) pairs than units, and short ones, workgroups of two waves
    // with a quarter of the LDS start and end apart, and take two tiles of 32 rows too. 256 sequences, 8
    // heads of 128, a token each: over 100 positions 27 us for 67, over 500 81 for 111; 128 over 2,000
    // 152 for 156, but 256 over 4,000 589 for 570. 256 of 48 rows over 100: 64 for 91 staged (but 128
    // rows 118 for 117). 16 heads of 64: 256 over 100 24 for 51, over 500 83 for 83, but 128 over 1,000
    // 90 for 76. With fewer pairs (16 sequences, 8 heads of 128, 2,000 positions): 34 for 33.
    const bool many = pairs > std::size_t(compute_units()) &&
                      rows.max_length <= std::size_t(cache.head_width == 128 ? 2048 : 512);
    s.narrow_waves = many ? few_waves : waves;
    s.parts_a_tile = s.parts == 1 ? 1 : s.parts <= (many ? 4 : 2) ? 2 : tall ? 16 : 8;
    s.tiles = (s.parts + s.parts_a_tile - 1) / s.parts_a_tile;
    // One workgroup a compute unit. Two a unit, with half the keys each, joins included: 55 us for 52 (8
    // sequences of one token over 8,190 positions, 8 heads), 121 for 98 (32 trees of 32 nodes over 4,093),
    // 175 for 162 (64 nodes over 131,001, 256-row tiles), 42 for 33 (2 prompts of 500 rows over 2,580).
    const std::size_t wanted = std::max<std::size_t>(1, std::size_t(compute_units()) / (pairs * s.tiles));
    // With fewer, a chunk has 256 keys or more: 64 nodes of 8 heads to one over 3,000 positions 23 us, with
    // chunks of 512 27, of 1,024 37; 500 rows over 1,000, 16 heads of 64: 23, 24, 25. In the narrow
    // kernel it has 512, two blocks a wave, and there is a chunk less, for what the join costs: a
    // token over 3,000 positions, 4 heads of 128, 15 us, with chunks of 1,024 19; but 3 trees of 12
    // nodes over 1,021, 16 heads of 64, 11.6 in one chunk, 11.9 in two, 12.9 in four.
    const std::size_t most = std::max<std::size_t>(
        1, s.parts_a_tile > 2 ? rows.max_length / 256 : std::max<std::size_t>(2, rows.max_length / 512) - 1);
    s.splits = int(std::min(wanted, most));
    constexpr std::size_t keys = block * waves;
    s.chunk = int(((rows.max_length + s.splits - 1) / s.splits + keys - 1) / keys * keys);
    s.chunk = std::max<int>(s.chunk, keys);
    s.units = pairs * s.splits;
    s.record = 16 * std::size_t(cache.head_width) + 32;
    // One tile reads a unit's keys and values, and they are more than the dies' caches of 4 MiB hold:
    // 8 sequences of one token over 8,190 positions, 8 heads: 47 us for 52, 32 trees of 32 nodes over
    // 4,093: 93 for 106. With another tile to come, 2 prompts of 500 rows: 31 for 29; of 12 MB 11.6
    // for 11.0.
    s.once = s.tiles == 1 && pairs * rows.max_length * cache.head_width * 4 > (std::size_t(8) << 22);
    return s;
}

// Workgroups of one launch, of which 2^32 work-items along x are the limit, and of one call. Those without rows
// end at once: 8.6 million take 16 ms.
constexpr std::size_t launch_limit = (std::size_t(1) << 23) - 8, call_limit = std::size_t(1) << 30;

template <int HW, bool Half> void launch(Launch l, const Shape& s, std::size_t pairs, hipStream_t stream)
{
    const std::size_t groups = s.units / l.together;
    const std::size_t grid = (groups + 7) / 8 * 8 * l.together * s.tiles;
    const auto run = [&](auto kernel, int threads, std::size_t lds)
    {
        if (lds > 65536)
        {
            check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)),
                      "paged attention LDS");
        }
        for (std::size_t first = 0; first < grid; first += launch_limit)
        {
            l.first = unsigned(first);
            kernel<<<unsigned(std::min(grid - first, launch_limit)), threads, lds, stream>>>(l);
            check_hip(hipGetLastError(), "paged attention launch");
        }
    };
    constexpr std::size_t narrow_wave = 2 * block * HW * 2, staged = stages * staged_keys * HW * 4;
    const auto run_either = [&](auto read_once)
    {
        constexpr bool once = decltype(read_once)::value;
        switch (s.parts_a_tile)
        {
        case 1:
            s.narrow_waves == waves
                ? run(narrow_kernel<HW, Half, 1, waves, once>, 64 * waves, waves * narrow_wave)
                : run(narrow_kernel<HW, Half, 1, few_waves, once>, 64 * few_waves, few_waves * narrow_wave);
            break;
        case 2:
            s.narrow_waves == waves
                ? run(narrow_kernel<HW, Half, 2, waves, once>, 64 * waves, waves * narrow_wave)
                : run(narrow_kernel<HW, Half, 2, few_waves, once>, 64 * few_waves, few_waves * narrow_wave);
            break;
        case 8: run(staged_kernel<HW, Half, 2, once>, 64 * waves, staged); break;
        default: run(staged_kernel<HW, Half, 1, once>, 64 * waves, staged); break;
        }
    };
    s.once ? run_either(std::true_type{}) : run_either(std::false_type{});
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
    require((s.units + 8 * cache.heads) * s.tiles < call_limit, "paged attention: too many rows, sequences and heads");
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
    // As many heads as leave each die eight groups.
    l.together = cache.heads;
    while (cache.heads % l.together || (l.together > 1 && s.units / l.together < 64))
    {
        --l.together;
    }
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

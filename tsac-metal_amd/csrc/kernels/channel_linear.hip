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
#include <cmath>
#include <iterator>
#include <type_traits>

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
    bool aligned;   // outputs in whole 16 bytes
};

template <Type T> __device__ __forceinline__ value_t<T> finished(int sum, float token, float channel, float bias)
{
    return narrow<T>(__builtin_fmaf(float(sum), token * channel, bias));
}

// 16 (or 4) bytes a lane, from `offset` bytes behind `from`, to `to`, lane after lane; the wave waits for it with
// its other loads (s_waitcnt vmcnt). `Once`: past the caches. Written out because the compiler would wait for it before
// any other read of LDS. A load to LDS needs a wait state behind a write of M0, which the compiler does not put into
// assembly. M0 is reserved, so that clang warns where it is named; nothing else uses it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ unsigned lds_address(const void* p)
{
    return __builtin_amdgcn_readfirstlane(
        unsigned(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) const void*)p)));
}
template <bool Once> __device__ __forceinline__ void load16_to_lds(const void* from, unsigned offset, const void* to)
{
    if constexpr (Once)
    {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(offset), "s"(from),
                     "s"(lds_address(to))
                     : "memory", "m0");
    }
    else
    {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(from),
                     "s"(lds_address(to))
                     : "memory", "m0");
    }
}
__device__ __forceinline__ void load4_to_lds(const void* from, unsigned offset, const void* to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(from),
                 "s"(lds_address(to))
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// At most N of the wave's vector memory operations outstanding (they complete in the order of issue).
template <int N> __device__ __forceinline__ void wait_loads()
{
    constexpr int n = N < 63 ? N : 63;
    __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 7 << 4 | 15 << 8);
}

// A workgroup's barrier behind its LDS reads, which leaves loads in flight.
__device__ __forceinline__ void ring_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4); // lgkmcnt(0) alone
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ------------------------------------------------------------------ few rows
//
// What costs is reading the weights. A workgroup takes 32 outputs and up to 8 Pieces rows, each of its waves every fourth
// step of 128 inputs, through a ring of Ring steps in LDS of its own: it asks for a step as soon as it has read the one
// whose place that takes, and waits for nobody until the waves' sums meet. Rows of activations come in whole lines of 128 bytes,
// which straight into registers, 32 bytes of each of 32 rows at a time, they would not (48 rows, 8192 x 8192: 26 us
// for 17 now, where reading the weights takes 10), their pieces exchanged by row so that eight rows' meet different banks.
// More steps in flight, or eight waves, gain nothing (rings of 3 and 4: 17 us) and keep a unit from a second workgroup.
namespace narrow
{
constexpr int waves = 4;

template <int Pieces, int Ring> struct Shape
{
    static constexpr int groups = (Pieces + 3) / 4; // 32 rows of an instruction each
    static constexpr int rows = 8 * Pieces;
    static constexpr int weight_bytes = slices * tile_bytes, step_bytes = weight_bytes + Pieces * 1024;
    static constexpr int loads = slices + Pieces; // of a wave and step
    // Rows of an instruction that no piece fills are read from what lies behind: for the last step that is this much more.
    static constexpr int ring_bytes = waves * Ring * step_bytes + (groups * 4 - Pieces) * 1024;
    static constexpr int sum_bytes = waves * tile * (tile + 1) * 4;
    static constexpr int lds_bytes = ring_bytes > sum_bytes ? ring_bytes : sum_bytes;
    static_assert(lds_bytes <= 160 * 1024);
};
} // namespace narrow

template <Type T, int Pieces, int Ring>
__global__ __launch_bounds__(narrow::waves * lanes) void narrow_kernel(Launch l)
{
    using namespace narrow;
    using S = Shape<Pieces, Ring>;
    extern __shared__ __attribute__((aligned(1024))) int8_t lds[];
    const int lane = threadIdx.x % lanes, warp = __builtin_amdgcn_readfirstlane(threadIdx.x / lanes);
    const int n0 = blockIdx.x * tile;
    const int8_t* const weights = l.weights + std::size_t(blockIdx.x) * l.steps * S::weight_bytes;
    int8_t* const mine = lds + warp * Ring * S::step_bytes;
    unsigned row_offset[Pieces];
#pragma unroll
    for (int j = 0; j < Pieces; ++j)
    {
        row_offset[j] = unsigned(min(8 * j + lane / 8, l.rows - 1)) * unsigned(l.q_stride);
    }
    const auto ask = [&](int s, int slot)
    {
        s = min(s, l.steps - 1); // past the end the last one again, which nobody reads
        int8_t* const to = mine + slot * S::step_bytes;
#pragma unroll
        for (int i = 0; i < slices; ++i)
        {
            load16_to_lds<true>(weights, unsigned(s * slices + i) * tile_bytes + lane * 16, to + i * tile_bytes);
        }
#pragma unroll
        for (int j = 0; j < Pieces; ++j)
        {
            // The lane's row is 8 j + lane / 8; the piece of 16 bytes that belongs into place lane % 8 of it.
            const int piece = (lane % 8 ^ lane / 8 ^ j % 2) * 16;
            load16_to_lds<false>(l.q, row_offset[j] + unsigned(min(s * step + piece, l.last_piece)),
                                 to + S::weight_bytes + j * 1024);
        }
    };
#pragma unroll
    for (int d = 0; d < Ring; ++d)
    {
        ask(warp + d * waves, d);
    }
    v16i acc[S::groups] = {};
    int slot = 0;
    for (int s = warp; s < l.steps; s += waves)
    {
        wait_loads<(Ring - 1) * S::loads>();
        asm volatile("" ::: "memory");
        const int8_t* const from = mine + slot * S::step_bytes;
        v4i w[slices], x[S::groups][slices];
#pragma unroll
        for (int i = 0; i < slices; ++i)
        {
            w[i] = *reinterpret_cast<const v4i*>(from + i * tile_bytes + lane * 16);
#pragma unroll
            for (int g = 0; g < S::groups; ++g)
            {
                const int row = lane % tile;
                x[g][i] = *reinterpret_cast<const v4i*>(from + S::weight_bytes + (g * tile + row) * step +
                                                        ((2 * i + lane / tile) ^ row % 8 ^ row / 8 % 2) * 16);
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4); // they have been read: lgkmcnt(0) alone
        asm volatile("" ::: "memory");
        ask(s + Ring * waves, slot);
#pragma unroll
        for (int i = 0; i < slices; ++i)
        {
#pragma unroll
            for (int g = 0; g < S::groups; ++g)
            {
                acc[g] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[i], x[g][i], acc[g], 0, 0, 0);
            }
        }
        slot = slot + 1 < Ring ? slot + 1 : 0;
    }
    wait_loads<0>(); // before the rings' memory takes the sums
    auto* out = static_cast<value_t<T>*>(l.out);
    int* const sums = reinterpret_cast<int*>(lds);
#pragma unroll
    for (int g = 0; g < S::groups; ++g)
    {
        __syncthreads();
        int* const to = sums + (warp * tile + lane % tile) * (tile + 1) + 4 * (lane / tile);
#pragma unroll
        for (int r = 0; r < 16; ++r)
        {
            to[8 * (r / 4) + r % 4] = acc[g][r];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < tile * tile; i += waves * lanes)
        {
            const int m = g * tile + i / tile, n = n0 + i % tile;
            if (m >= l.rows || n >= l.outputs)
            {
                continue;
            }
            int sum = 0;
#pragma unroll
            for (int w = 0; w < waves; ++w)
            {
                sum += sums[(w * tile + i / tile) * (tile + 1) + i % tile];
            }
            out[std::size_t(m) * l.out_stride + n] =
                finished<T>(sum, l.token_scales[m], l.channel_scales[n], l.bias ? l.bias[n] : 0.0f);
        }
    }
}

// ------------------------------------------------------------------ many rows
//
// Workgroups of four waves, 2 x 2, take tiles of 64 JN outputs x 64 JM rows one after the other, each wave JN x JM
// results of 32 x 32. A stage is 64 or 128 inputs of a tile's operands. Stages pass from memory straight into a ring in
// LDS, across the tiles' borders: while a tile is stored the next one's first stages are on their way. At a stage's
// barrier the next one has landed, so that its first operands are read from LDS under the stage's last products.
//
// Activation rows lie in LDS with their 16-byte pieces exchanged by row, so that lanes that read one piece of
// consecutive rows meet different banks; weights lie as they are read.
//
// 8192 x 8192 x 8192: 480 us, 2,290 TOP/s, matrix units busy 56%, the clock held down to about 1.9 GHz. With weights of
// zero, which cost no power, 352 us; without the loads, in a copy, 354, without the barriers too 343; with all loads from
// one tile 475, so that it is their way into LDS that costs, not memory. Results by way of LDS, in whole lines, were
// slower (525 us).
//
// A die's workgroups take neighbouring tiles, four of rows by as many of outputs as there are, which share what they
// read in its cache.
namespace tiled
{
constexpr int threads = 256;
constexpr int dies = 8;
constexpr int together = 4; // row tiles that are walked side by side

template <int JN, int JM, int Depth, int Ring> struct Shape
{
    static_assert(Depth == 64 || Depth == 128);
    static constexpr int n = 64 * JN, m = 64 * JM, ring = Ring;
    static constexpr int cuts = Depth / tile;                        // slices of 32 inputs
    static constexpr int weight_bytes = n * Depth, stage_bytes = (n + m) * Depth;
    static constexpr int weight_loads = JN * Depth / 64, row_loads = JM * Depth / 64; // of a wave and stage
    static constexpr int loads = weight_loads + row_loads;
    static constexpr int constants = 2 * n + m;                     // scales and bias of a tile
    static constexpr int constant_loads = (constants / 64 + 3) / 4; // of a wave and tile
    // With the fewest stages a tile, two of 64 or one of 128, the scales of the tile Ring / 2, or Ring - 1, further on
    // arrive before this one is stored.
    static constexpr int constant_slots = Depth == 64 ? Ring / 2 + 1 : Ring;
    static constexpr int lds_bytes = ring * stage_bytes + 4 * constant_slots * constants;
    static constexpr int row_pieces = Depth / 16;
    static_assert(lds_bytes <= 160 * 1024 && Ring >= 3);
};
} // namespace tiled

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// A 32 x 32 block of results: the lane's row has `four` + 8 (r / 4) + r % 4 of its 32 outputs.
template <Type T>
__device__ __forceinline__ void store_block(const v16i& sums, float token, const float (&scale)[16], const float (&bias)[16],
                                            value_t<T>* to, bool there, int columns, int four, bool whole)
{
    value_t<T> v[16];
#pragma unroll
    for (int r = 0; r < 16; ++r)
    {
        v[r] = finished<T>(sums[r], token, scale[r], bias[r]);
    }
    if (whole)
    {
        if constexpr (T == Type::single)
        {
            if (there)
            {
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                {
                    *reinterpret_cast<float4*>(to + 2 * r + four) = make_float4(v[r], v[r + 1], v[r + 2], v[r + 3]);
                }
            }
        }
        else
        {
            // Halves of the wave exchange pairs of four, so that a lane has eight neighbours; all lanes take part.
            u32x4 eight[2];
#pragma unroll
            for (int r = 0; r < 16; r += 8)
            {
                const auto pair = [&](int a) { return unsigned(v[a]) | unsigned(v[a + 1]) << 16; };
                const auto p = __builtin_amdgcn_permlane32_swap(pair(r), pair(r + 4), false, false);
                const auto q = __builtin_amdgcn_permlane32_swap(pair(r + 2), pair(r + 6), false, false);
                eight[r / 8] = u32x4{unsigned(p[0]), unsigned(q[0]), unsigned(p[1]), unsigned(q[1])};
            }
            if (there)
            {
                *reinterpret_cast<u32x4*>(to + 2 * four) = eight[0];
                *reinterpret_cast<u32x4*>(to + 16 + 2 * four) = eight[1];
            }
        }
    }
    else if (there)
    {
#pragma unroll
        for (int r = 0; r < 16; ++r)
        {
            const int n = 8 * (r / 4) + r % 4;
            if (n < columns - four)
            {
                to[four + n] = v[r];
            }
        }
    }
}

// Once: all rows are in one row tile, so that each weight is read once and need not stay in a cache, where the results and
// the rows then do. With six layers' weights in turn, 190 x 2043 x 32003 to FP32 in 28.7 us for 30.8, to BF16 26.2 for
// 28.2, 256 x 4096 x 14336 26.8 for 26.6; one layer's again and again, 65 MB, as before.
template <Type T, int JN, int JM, int Depth, int Ring, int PerUnit, bool Once>
__global__ __launch_bounds__(tiled::threads, PerUnit) void tiled_kernel(Launch l, int row_tiles, int column_tiles)
{
    using namespace tiled;
    using S = Shape<JN, JM, Depth, Ring>;
    extern __shared__ __attribute__((aligned(1024))) int8_t lds[];
    float* const constants = reinterpret_cast<float*>(lds + Ring * S::stage_bytes); // [slot]: scales and bias [n], tokens [m]
    const int lane = threadIdx.x % lanes, warp = __builtin_amdgcn_readfirstlane(threadIdx.x / lanes);
    const int wn = warp % 2, wm = warp / 2;
    const int total = row_tiles * column_tiles;
    const int die = blockIdx.x % dies, mates = gridDim.x / dies;
    const int begin = int((long long)total * die / dies), end = int((long long)total * (die + 1) / dies);
    const int mine = begin + int(blockIdx.x / dies);
    const int tiles = mine < end ? (end - mine + mates - 1) / mates : 0;
    const int stages = l.steps * (step / Depth); // of a tile
    const int groups = (l.outputs + tile - 1) / tile;
    struct Spot
    {
        int n, m; // first output and row
    };
    const auto spot = [&](int k)
    {
        const int t = mine + k * mates, block = t / (together * column_tiles), rest = t - block * together * column_tiles;
        const int high = min(together, row_tiles - block * together);
        return Spot{rest / high * S::n, (block * together + rest % high) * S::m};
    };
    // Where piece `c` of 16 bytes of a row lies in LDS: so that one piece of consecutive rows is in different banks.
    const auto place = [](int row, int c)
    { return Depth == 64 ? c ^ (row / 2 & 3) ^ (row / 8 & 1) : c ^ (row & 7) ^ (row / 8 & 1); };
    if (tiles == 0)
    {
        return;
    }
    // Tile and stage that are asked for next; past the last tile its stages once more, which nobody reads, so that as many
    // loads are behind a stage wherever it is.
    int loading = 0, loading_stage = 0;
    Spot from = spot(0);
    const int8_t* weights[S::weight_loads];
    const int8_t* rows_base;
    unsigned row_offset[S::row_loads];
    const auto start_tile = [&]
    {
#pragma unroll
        for (int j = 0; j < S::weight_loads; ++j)
        {
            const int copy = warp * S::weight_loads + j, group = min(from.n / tile + copy / S::cuts, groups - 1);
            weights[j] = l.weights + (std::size_t(group) * l.steps * slices + copy % S::cuts) * tile_bytes;
        }
        rows_base = l.q + std::size_t(from.m) * l.q_stride;
#pragma unroll
        for (int j = 0; j < S::row_loads; ++j)
        {
            const int row = (warp * S::row_loads + j) * (64 / S::row_pieces) + lane / S::row_pieces;
            row_offset[j] = unsigned(min(row, l.rows - 1 - from.m)) * unsigned(l.q_stride);
        }
    };
    const auto ask_weights = [&](int slot, int j)
    {
        load16_to_lds<Once>(weights[j], unsigned(loading_stage) * (S::cuts * tile_bytes) + lane * 16,
                            lds + slot * S::stage_bytes + (warp * S::weight_loads + j) * tile_bytes);
    };
    const auto ask_rows = [&](int slot, int j)
    {
        const int row = (warp * S::row_loads + j) * (64 / S::row_pieces) + lane / S::row_pieces;
        const int piece = place(row, lane % S::row_pieces) * 16;
        load16_to_lds<false>(rows_base, row_offset[j] + unsigned(min(loading_stage * Depth + piece, l.last_piece)),
                             lds + slot * S::stage_bytes + S::weight_bytes + (warp * S::row_loads + j) * 1024);
    };
    const auto asked = [&]
    {
        if (loading_stage == 0)
        {
            float* const c = constants + loading % S::constant_slots * S::constants;
#pragma unroll
            for (int j = 0; j < S::constant_loads; ++j)
            {
                const int part = min(warp * S::constant_loads + j, S::constants / 64 - 1), at = part * 64 + lane;
                const int n = min(from.n + at % S::n, l.outputs - 1), m = min(from.m + at - 2 * S::n, l.rows - 1);
                const float* const source = part >= 2 * JN ? l.token_scales : part >= JN && l.bias ? l.bias : l.channel_scales;
                load4_to_lds(source, unsigned(part >= 2 * JN ? m : n) * 4, c + part * 64);
            }
        }
        if (++loading_stage == stages)
        {
            loading_stage = 0;
            ++loading;
            from = spot(min(loading, tiles - 1));
            start_tile();
        }
    };
    start_tile();
#pragma unroll
    for (int slot = 0; slot < Ring - 1; ++slot)
    {
#pragma unroll
        for (int j = 0; j < S::weight_loads; ++j)
        {
            ask_weights(slot, j);
        }
#pragma unroll
        for (int j = 0; j < S::row_loads; ++j)
        {
            ask_rows(slot, j);
        }
        asked();
    }
    wait_loads<(Ring - 2) * S::loads>();
    ring_barrier();

    v16i acc[JN][JM];
    v4i w[2][JN], x[2][JM];
    const auto read = [&](int slot, int slice, v4i (&a)[JN], v4i (&b)[JM])
    {
        const int8_t* const at = lds + slot * S::stage_bytes;
#pragma unroll
        for (int j = 0; j < JN; ++j)
        {
            a[j] = *reinterpret_cast<const v4i*>(at + ((wn * JN + j) * S::cuts + slice) * tile_bytes + lane * 16);
        }
        const int row = lane % 32, swapped = place(row, 2 * slice + lane / 32) * 16;
#pragma unroll
        for (int j = 0; j < JM; ++j)
        {
            b[j] = *reinterpret_cast<const v4i*>(at + S::weight_bytes + ((wm * JM + j) * 32 + row) * Depth + swapped);
        }
    };
    read(0, 0, w[0], x[0]);
    constexpr int stores = T == Type::single ? 4 * JN * JM : 2 * JN * JM;
    int slot = 0;        // of the stage
    bool stored = false; // a whole tile's stores are behind the loads that are waited for next
    const auto stage = [&](auto first, int since)
    {
        // The next stage has landed: what may be outstanding is what was asked for behind it.
        if (stored && since < Ring - 2)
        {
            wait_loads<(Ring - 3) * S::loads + stores>();
        }
        else
        {
            wait_loads<(Ring - 3) * S::loads>();
        }
        ring_barrier();
        const v16i zero = {};
        const int behind = slot ? slot - 1 : Ring - 1, next = slot + 1 < Ring ? slot + 1 : 0;
#pragma unroll
        for (int cut = 0; cut < S::cuts; ++cut)
        {
            if (cut == S::cuts - 1)
            {
                asked();
                read(next, 0, w[0], x[0]);
            }
            else
            {
                read(slot, cut + 1, w[(cut + 1) % 2], x[(cut + 1) % 2]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < JN; ++j)
            {
#pragma unroll
                for (int i = 0; i < JM; ++i)
                {
                    acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
                        w[cut % 2][j], x[cut % 2][i], decltype(first)::value && cut == 0 ? zero : acc[j][i], 0, 0, 0);
                }
                if (cut == 0)
                {
                    // The loads of the stage that takes the last one's place, among the products, which leave the time for it.
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int a = j; a < (S::loads + 1) / 2; a += JN)
                    {
                        if (a < S::weight_loads)
                        {
                            ask_weights(behind, a);
                        }
                        if (a < S::row_loads)
                        {
                            ask_rows(behind, a);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (cut == 0)
            {
#pragma unroll
                for (int a = (S::loads + 1) / 2; a < (S::weight_loads > S::row_loads ? S::weight_loads : S::row_loads); ++a)
                {
                    if (a < S::weight_loads)
                    {
                        ask_weights(behind, a);
                    }
                    if (a < S::row_loads)
                    {
                        ask_rows(behind, a);
                    }
                }
            }
        }
        slot = next;
    };
    for (int k = 0; k < tiles; ++k)
    {
        stage(std::true_type{}, 0);
        for (int s = 1; s < stages; ++s)
        {
            stage(std::false_type{}, s);
        }
        const Spot to = spot(k);
        // Stores are counted where every lane has one.
        stored = l.aligned && to.n + S::n <= l.outputs && to.m + S::m <= l.rows;
        // The lane's row and first of four outputs. Hidden from the compiler, which otherwise holds what follows from them
        // for all blocks in registers throughout the tiles.
        int row = lane % 32, four = 4 * (lane / 32);
        asm volatile("" : "+v"(row), "+v"(four));
        const float* const c = constants + k % S::constant_slots * S::constants;
        const int rows_left = l.rows - to.m - wm * 32 * JM - row;
        auto* out = static_cast<value_t<T>*>(l.out) + std::size_t(to.m + wm * 32 * JM + row) * l.out_stride + to.n + wn * 32 * JN;
        int columns_left = l.outputs - to.n - wn * 32 * JN;
#pragma unroll
        for (int j = 0; j < JN; ++j)
        {
            float scale[16], bias[16];
#pragma unroll
            for (int r = 0; r < 16; r += 4)
            {
                const float* const at = c + (wn * JN + j) * 32 + 2 * r + four;
                const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + S::n);
                scale[r] = a.x, scale[r + 1] = a.y, scale[r + 2] = a.z, scale[r + 3] = a.w;
                bias[r] = l.bias ? b.x : 0.0f, bias[r + 1] = l.bias ? b.y : 0.0f;
                bias[r + 2] = l.bias ? b.z : 0.0f, bias[r + 3] = l.bias ? b.w : 0.0f;
            }
            const bool whole = l.aligned && 32 <= columns_left;
#pragma unroll
            for (int i = 0; i < JM; ++i)
            {
                __builtin_amdgcn_sched_barrier(0); // one block's values in registers at a time
                store_block<T>(acc[j][i], c[2 * S::n + (wm * JM + i) * 32 + row], scale, bias,
                               out + std::size_t(32 * i) * l.out_stride, 32 * i < rows_left, columns_left, four, whole);
            }
            out += 32;
            columns_left -= 32;
            asm volatile("" : "+v"(four));
        }
    }
    wait_loads<0>(); // before its LDS is another workgroup's
}

// 16 bytes a thread of the operand tiles.
__global__ void tiles_kernel(const int8_t* __restrict__ canonical, int inputs, int outputs, int steps,
                             int8_t* __restrict__ tiled, std::size_t pieces)
{
    const std::size_t across = std::size_t(steps) * slices, threads = std::size_t(gridDim.x) * blockDim.x;
    for (std::size_t piece = std::size_t(blockIdx.x) * blockDim.x + threadIdx.x; piece < pieces; piece += threads)
    {
        const int lane = piece % lanes;
        const std::size_t t = piece / lanes, n = t / across * tile + lane % tile;
        const int k = int(t % across) * tile + lane / tile * 16;
        int8_t v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            v[i] = n < std::size_t(outputs) && k + i < inputs ? canonical[n * inputs + k + i] : int8_t(0);
        }
        __builtin_memcpy(tiled + 16 * piece, v, 16);
    }
}

int steps_of(std::size_t inputs)
{
    return int((inputs + step - 1) / step);
}

template <class Kernel> void allow_lds(Kernel kernel, int bytes)
{
    if (bytes > 65536)
    {
        check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      bytes),
                  "channel linear LDS");
    }
}

template <Type T, int JN, int JM, int Depth, int Ring, int PerUnit> void launch_tiled(const Launch& l, hipStream_t stream)
{
    using S = tiled::Shape<JN, JM, Depth, Ring>;
    static_assert(S::lds_bytes * PerUnit <= 160 * 1024);
    const int row_tiles = (l.rows + S::m - 1) / S::m, column_tiles = (l.outputs + S::n - 1) / S::n;
    auto kernel = tiled_kernel<T, JN, JM, Depth, Ring, PerUnit, false>;
    if constexpr (S::m > 64) // fewer rows than 65 do not come here
    {
        if (row_tiles == 1)
        {
            kernel = tiled_kernel<T, JN, JM, Depth, Ring, PerUnit, true>;
        }
    }
    allow_lds(kernel, S::lds_bytes);
    const std::size_t total = std::size_t(row_tiles) * column_tiles;
    require(total < (std::size_t(1) << 30), "channel linear: too many tiles");
    const std::size_t most = std::size_t(compute_units()) * PerUnit / tiled::dies * tiled::dies;
    const std::size_t grid = std::min(most, (total + tiled::dies - 1) / tiled::dies * tiled::dies);
    kernel<<<unsigned(std::max<std::size_t>(grid, tiled::dies)), tiled::threads, S::lds_bytes, stream>>>(l, row_tiles,
                                                                                                         column_tiles);
    check_hip(hipGetLastError(), "channel linear launch");
}

template <Type T, int Pieces, int Ring> void launch_narrow(const Launch& l, hipStream_t stream)
{
    using S = narrow::Shape<Pieces, Ring>;
    const auto kernel = narrow_kernel<T, Pieces, Ring>;
    allow_lds(kernel, S::lds_bytes);
    kernel<<<unsigned((l.outputs + tile - 1) / tile), narrow::waves * lanes, S::lds_bytes, stream>>>(l);
    check_hip(hipGetLastError(), "channel linear launch");
}

// Tiles of many rows, and what one costs a compute unit: microseconds for 64 inputs, and to begin and store it.
struct Tiles
{
    int n, m;
    double inputs, each;
};
constexpr Tiles tiles[] = {{256, 256, 0.85, 6.5}, {128, 256, 0.50, 3.7}, {128, 128, 0.29, 2.0}, {64, 64, 0.115, 0.8}};

// Which of them: the least time by what one costs and how many of them the fullest compute unit has. Large tiles share
// more of what they read, small ones are more of a few rows' work at once. Measured with eight layers' weights in turn, us
// (256 x 256, 128 x 256, 128 x 128, 64 x 64): 128 rows x 4096 x 4096 49, 30, 19, 10.8; 1024 x 1024 x 4096 20, 13.7, 10.6, 11.8;
// 512 x 8192 x 8192 101, 73, 44, 70; 1024 x 8192 x 8192 103, 79, 83, 131; 4096 x 4096 x 4096 68, 75, 84, 113; 30960 x 1024 x
// 4096 165, 178, 198, 255. By this rule: 10.8, 10.6, 44, 79, 68, 165.
int tiles_for(const Launch& l)
{
    int best = 0;
    double least = 0;
    for (int c = 0; c < int(std::size(tiles)); ++c)
    {
        const Tiles& t = tiles[c];
        const double count = double((l.rows + t.m - 1) / t.m) * ((l.outputs + t.n - 1) / t.n);
        const double time = std::ceil(count / compute_units()) * (t.inputs * 2 * l.steps + t.each);
        if (c == 0 || time < least)
        {
            best = c;
            least = time;
        }
    }
    return best;
}

template <Type T> void launch(const Launch& l, hipStream_t stream)
{
    if (l.rows <= 64)
    {
        l.rows <= 8    ? launch_narrow<T, 1, 2>(l, stream)
        : l.rows <= 16 ? launch_narrow<T, 2, 2>(l, stream)
        : l.rows <= 32 ? launch_narrow<T, 4, 2>(l, stream)
        : l.rows <= 48 ? launch_narrow<T, 6, 2>(l, stream)
                       : launch_narrow<T, 8, 2>(l, stream);
        return;
    }
    switch (tiles_for(l))
    {
    case 0: return launch_tiled<T, 4, 4, 64, 4, 1>(l, stream);
    case 1: return launch_tiled<T, 2, 4, 128, 3, 1>(l, stream);
    case 2: return launch_tiled<T, 2, 2, 128, 4, 1>(l, stream);
    default: return launch_tiled<T, 1, 1, 128, 4, 2>(l, stream);
    }
}
} // namespace

std::size_t channel_tiles_bytes(std::size_t inputs, std::size_t outputs)
{
    return (outputs + tile - 1) / tile * tile * std::size_t(steps_of(inputs)) * step;
}

void channel_tiles(const int8_t* canonical, std::size_t inputs, std::size_t outputs, int8_t* tiled, hipStream_t stream)
{
    const std::size_t pieces = channel_tiles_bytes(inputs, outputs) / 16;
    const std::size_t groups = std::min<std::size_t>((pieces + 255) / 256, 1 << 20);
    tiles_kernel<<<unsigned(groups), 256, 0, stream>>>(canonical, int(inputs), int(outputs), steps_of(inputs), tiled, pieces);
    check_hip(hipGetLastError(), "channel linear tiles launch");
}

void channel_linear(const ChannelWeights& weights, const ChannelRows& rows, hipStream_t stream)
{
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
                      (weights.inputs - 1) / 16 * 16,
                      reinterpret_cast<std::uintptr_t>(rows.out) % 16 == 0 &&
                          rows.out_stride * (rows.type == Type::single ? 4 : 2) % 16 == 0};
    switch (rows.type)
    {
    case Type::bf16: return launch<Type::bf16>(l, stream);
    case Type::half: return launch<Type::half>(l, stream);
    default: return launch<Type::single>(l, stream);
    }
}
} // namespace tsac_hip

// Verification of drafted tokens: which of them the target model's probabilities keep, with
// random numbers given, and the token that follows.
//
// At a node with children c_1 < c_2 < ... the k-th is accepted with probability
// min(1, r(x)/q(x)), r the target's distribution less what the refused ones took of it:
// r <- norm(max(0, r - q)) after each refusal. With r = max(0, p - s q) / W that is
//   s <- s + W,  W <- sum_t max(0, p_t - s q_t),   s = 0 and W = 1 at first,
// so a trial is u q(x) W < max(0, p(x) - s q(x)): two values of the row, and one pass over it for
// each refused child that has a sibling behind it. Drafts without a distribution are certain
// of their token: the trial is u W < p(x), and a refused token is struck out of p.
// The token that follows is drawn from max(0, p - s q) (or p without those struck out) at the
// node where no child was accepted.
//
// Results are whole numbers that decide what a model goes on with, so everything is held in 64
// bits, and a sum's order depends on the alphabet alone.
#include "paged.hpp"

#include <algorithm>
#include <type_traits>

namespace tsac_hip
{
namespace
{
constexpr int vector_width = 8;            // values a lane reads at a time
constexpr int segment = 64 * vector_width; // values of one wave's step
constexpr int max_alphabet = 1 << 20;
constexpr int max_segments = max_alphabet / segment;
enum class Type
{
    bf16,
    half,
    single
};

template <Type T> struct Value
{
    using type = uint16_t;
};
template <> struct Value<Type::single>
{
    using type = float;
};

// A probability: what is negative or not finite counts as 0.
template <Type T> __device__ __forceinline__ double probability(typename Value<T>::type bits)
{
    if constexpr (T == Type::bf16)
    {
        return double(__uint_as_float(bits < 0x7f80 ? unsigned(bits) << 16 : 0u));
    }
    else if constexpr (T == Type::half)
    {
        return double(float(__builtin_bit_cast(_Float16, uint16_t(bits < 0x7c00 ? bits : 0))));
    }
    else
    {
        const unsigned whole = __builtin_bit_cast(unsigned, bits);
        return double(__uint_as_float(whole < 0x7f800000u ? whole : 0u));
    }
}

// One level of a butterfly over lanes, started from stride 1: every group of `stride` lanes holds
// one value, so that any lane of the neighbouring group will do.
template <int stride> __device__ __forceinline__ double add_neighbours(double value)
{
    const uint64_t bits = __builtin_bit_cast(uint64_t, value);
    const int low = int(bits), high = int(bits >> 32);
    const auto whole = [](unsigned l, unsigned h) { return __builtin_bit_cast(double, uint64_t(h) << 32 | l); };
    if constexpr (stride < 16)
    {
        // quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror
        constexpr int control = stride == 1 ? 0xb1 : stride == 2 ? 0x4e : stride == 4 ? 0x141 : 0x140;
        return value + whole(__builtin_amdgcn_mov_dpp(low, control, 0xf, 0xf, false),
                             __builtin_amdgcn_mov_dpp(high, control, 0xf, 0xf, false));
    }
    else if constexpr (stride == 16)
    {
        const auto l = __builtin_amdgcn_permlane16_swap(low, low, false, false);
        const auto h = __builtin_amdgcn_permlane16_swap(high, high, false, false);
        return whole(l[0], h[0]) + whole(l[1], h[1]);
    }
    else
    {
        const auto l = __builtin_amdgcn_permlane32_swap(low, low, false, false);
        const auto h = __builtin_amdgcn_permlane32_swap(high, high, false, false);
        return whole(l[0], h[0]) + whole(l[1], h[1]);
    }
}

__device__ __forceinline__ double wave_sum(double value)
{
    value = add_neighbours<2>(add_neighbours<1>(value));
    value = add_neighbours<8>(add_neighbours<4>(value));
    return add_neighbours<32>(add_neighbours<16>(value));
}

// One step of a scan over lanes: adds the value that DPP `control` names to the lanes of `rows`.
template <int control, int rows> __device__ __forceinline__ double add_from(double value)
{
    const uint64_t bits = __builtin_bit_cast(uint64_t, value);
    const unsigned low = __builtin_amdgcn_update_dpp(0, int(bits), control, rows, 0xf, true);
    const unsigned high = __builtin_amdgcn_update_dpp(0, int(bits >> 32), control, rows, 0xf, true);
    return value + __builtin_bit_cast(double, uint64_t(high) << 32 | low);
}

// Inclusive sums over the lanes: row_shr 1, 2, 4, 8, then the rows' last lanes to the rows behind.
__device__ __forceinline__ double wave_scan(double value)
{
    value = add_from<0x112, 0xf>(add_from<0x111, 0xf>(value));
    value = add_from<0x118, 0xf>(add_from<0x114, 0xf>(value));
    return add_from<0x143, 0xc>(add_from<0x142, 0xa>(value));
}

struct Shared
{
    int parents[max_draft_nodes], tokens[max_draft_nodes];
    float uniforms[max_draft_nodes];
    double target[max_draft_nodes], draft[max_draft_nodes]; // p and q of a node's token in its parent's row
    int struck[max_draft_nodes];
    double sums[max_segments];
};

// A node's row of each distribution.
template <Type T, bool Draft> struct Rows
{
    using V = typename Value<T>::type;
    const V* target;
    const V* draft;
    int alphabet;

    static constexpr int words = vector_width * sizeof(V) / 4;
    struct Raw
    {
        unsigned target[words], draft[Draft ? words : 1];
    };
    // Eight values from `at`, zeros past the alphabet.
    __device__ __forceinline__ void read(const V* row, int at, unsigned* to) const
    {
        if (at + vector_width <= alphabet)
        {
            __builtin_memcpy(to, row + at, sizeof(unsigned) * words); // at any alignment
            return;
        }
#pragma unroll
        for (int w = 0; w < words; ++w)
        {
            to[w] = 0;
#pragma unroll
            for (int j = 0; j < int(4 / sizeof(V)); ++j)
            {
                const int i = at + w * int(4 / sizeof(V)) + j;
                using Bits = std::conditional_t<sizeof(V) == 4, unsigned, uint16_t>;
                to[w] |= i < alphabet ? unsigned(__builtin_bit_cast(Bits, row[i])) << (16 * j) : 0u;
            }
        }
    }
    __device__ __forceinline__ void read(int at, Raw& raw) const
    {
        read(target, at, raw.target);
        if constexpr (Draft)
        {
            read(draft, at, raw.draft);
        }
    }
    __device__ static __forceinline__ double value(const unsigned* raw, int j)
    {
        if constexpr (sizeof(V) == 4)
        {
            return probability<T>(__uint_as_float(raw[j]));
        }
        else
        {
            return probability<T>(V(raw[j / 2] >> 16 * (j % 2)));
        }
    }
};

// What refused children take of a row.
struct Taken
{
    double shift;      // times the draft's row, or
    const int* struck; // tokens without the draft's
    int count;
};

// What is left of eight values from `at`.
template <Type T, bool Draft>
__device__ __forceinline__ void left_of(const typename Rows<T, Draft>::Raw& raw, int at, const Taken& taken,
                                        double (&to)[vector_width])
{
#pragma unroll
    for (int j = 0; j < vector_width; ++j)
    {
        to[j] = Rows<T, Draft>::value(raw.target, j);
        if constexpr (Draft)
        {
            to[j] = __builtin_fmax(__builtin_fma(-taken.shift, Rows<T, Draft>::value(raw.draft, j), to[j]), 0.0);
        }
    }
    if constexpr (!Draft)
    {
        for (int k = 0; k < taken.count; ++k)
        {
            const int j = taken.struck[k] - at;
#pragma unroll
            for (int i = 0; i < vector_width; ++i)
            {
                to[i] = i == j ? 0.0 : to[i];
            }
        }
    }
}

// A lane's eight.
template <Type T, bool Draft>
__device__ __forceinline__ double lane_sum(const typename Rows<T, Draft>::Raw& raw, int at, const Taken& taken)
{
    double value[vector_width];
    left_of<T, Draft>(raw, at, taken, value);
    return ((value[0] + value[1]) + (value[2] + value[3])) + ((value[4] + value[5]) + (value[6] + value[7]));
}

// The token in a segment that the goal falls to, given the sum in front of it: the lowest whose
// inclusive sum passes it, or the last one with anything left if rounding passes over all.
template <Type T, bool Draft>
__device__ __forceinline__ int find_in(const typename Rows<T, Draft>::Raw& raw, int at, const Taken& taken, double before,
                                       double goal)
{
    double value[vector_width];
    left_of<T, Draft>(raw, at, taken, value);
    double sum = 0;
#pragma unroll
    for (int j = 0; j < vector_width; ++j)
    {
        sum += value[j];
    }
    double inclusive = before + (wave_scan(sum) - sum);
    int token = -1, some = -1;
#pragma unroll
    for (int j = 0; j < vector_width; ++j)
    {
        inclusive += value[j];
        token = token < 0 && value[j] > 0.0 && inclusive > goal ? at + j : token;
        some = value[j] > 0.0 ? at + j : some;
    }
    const uint64_t past = __ballot(token >= 0), any = __ballot(some >= 0);
    return past  ? __shfl(token, __builtin_ctzll(past))
           : any ? __shfl(some, 63 - __builtin_clzll(any))
                 : -1;
}

// The whole sum, from the segments'; every wave for itself.
__device__ __forceinline__ double total_of(const double* sums, int segments)
{
    const int lane = threadIdx.x % 64;
    double total = 0;
    for (int base = 0; base < segments; base += 64)
    {
        total += wave_sum(base + lane < segments ? sums[base + lane] : 0.0);
    }
    return total;
}

// The segment that a goal falls to, as find_in(), and the sum in front of it.
__device__ __forceinline__ int find_segment(const double* sums, int segments, double goal, double& before)
{
    const int lane = threadIdx.x % 64;
    double front = 0; // sum of the segments in front
    int last = 0;
    before = 0;
    for (int base = 0; base < segments; base += 64)
    {
        const double mine = base + lane < segments ? sums[base + lane] : 0.0;
        const double inclusive = front + wave_scan(mine);
        const uint64_t past = __ballot(inclusive > goal && mine > 0.0), some = __ballot(mine > 0.0);
        const int at = past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : -1;
        if (at >= 0)
        {
            last = base + at;
            before = __shfl(inclusive - mine, at);
        }
        if (past)
        {
            break;
        }
        front = __shfl(inclusive, 63);
    }
    return last;
}

// A row of the alphabet as a workgroup sums it and draws from it. One that its waves can hold in
// registers, at_a_time segments each, is read once however often it is summed.
template <Type T, bool Draft> struct Summed
{
    using Raw = typename Rows<T, Draft>::Raw;
    // Segments a wave reads before it uses them, in at most 32 registers.
    static constexpr int at_a_time = sizeof(typename Rows<T, Draft>::V) == 4 ? 2 : 4;
    Rows<T, Draft> rows{};
    Raw held[at_a_time];
    const int lane = threadIdx.x % 64, warp = threadIdx.x / 64, waves = blockDim.x / 64;
    int segments = 0;
    bool holds = false;

    __device__ __forceinline__ void open(const Rows<T, Draft>& of)
    {
        rows = of;
        segments = (rows.alphabet + segment - 1) / segment;
        holds = segments <= waves * at_a_time;
        if (holds)
        {
            read(0, segments);
        }
    }
    __device__ __forceinline__ int place(int s) const
    {
        return s * segment + lane * vector_width;
    }
    __device__ __forceinline__ void read(int first, int last)
    {
#pragma unroll
        for (int i = 0; i < at_a_time; ++i)
        {
            const int s = first + warp + i * waves;
            if (s < last)
            {
                rows.read(place(s), held[i]);
            }
        }
    }
    __device__ __forceinline__ void sum_up(int first, int last, const Taken& taken, double* sums) const
    {
#pragma unroll
        for (int i = 0; i < at_a_time; ++i)
        {
            const int s = first + warp + i * waves;
            if (s < last)
            {
                const double sum = wave_sum(lane_sum<T, Draft>(held[i], place(s), taken));
                if (lane == 0)
                {
                    sums[s] = sum;
                }
            }
            __builtin_amdgcn_sched_barrier(0); // one segment's sums in registers at a time
        }
    }
    // The sums of segments first .. last - 1, of a row that is not held.
    __device__ __forceinline__ void sum_range(int first, int last, const Taken& taken, double* sums)
    {
        for (; first < last; first += waves * at_a_time)
        {
            read(first, last);
            sum_up(first, last, taken, sums);
        }
    }
    // The whole sum, for every thread; the segments' stay in `sums`, in LDS.
    __device__ __forceinline__ double sum(const Taken& taken, double* sums)
    {
        __syncthreads(); // the sums in front of these are read
        if (holds)
        {
            sum_up(0, segments, taken, sums);
        }
        else
        {
            sum_range(0, segments, taken, sums);
        }
        __syncthreads();
        return total_of(sums, segments);
    }
    // The whole sum alone, for every thread: over the lanes once.
    __device__ __forceinline__ double weigh(const Taken& taken, double* sums)
    {
        double mine = 0;
        for (int first = 0; first < segments; first += waves * at_a_time)
        {
            if (!holds)
            {
                read(first, segments);
            }
#pragma unroll
            for (int i = 0; i < at_a_time; ++i)
            {
                const int s = first + warp + i * waves;
                if (s < segments)
                {
                    mine += lane_sum<T, Draft>(held[i], place(s), taken);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        mine = wave_sum(mine);
        __syncthreads(); // the sums in front of these are read
        if (lane == 0)
        {
            sums[warp] = mine;
        }
        __syncthreads();
        return total_of(sums, waves);
    }
    // Writes the token that the goal falls to, from the segments' sums: on the wave that has it.
    __device__ __forceinline__ void draw(const Taken& taken, double goal, const double* sums, int* to) const
    {
        double before;
        const int s = find_segment(sums, segments, goal, before);
        if (s % waves != warp)
        {
            return;
        }
        Raw raw{};
        if (holds)
        {
#pragma unroll
            for (int i = 0; i < at_a_time; ++i)
            {
                if (s / waves == i)
                {
                    raw = held[i];
                }
            }
        }
        else
        {
            rows.read(place(s), raw);
        }
        const int token = find_in<T, Draft>(raw, place(s), taken, before, goal);
        if (lane == 0)
        {
            *to = token;
        }
    }
};

// What draw_kernel needs of a sequence's walk, in front of its segments' sums.
struct Walk
{
    double shift;
    int node, struck; // node -1: a sequence without nodes
};

template <Type T, bool Draft> struct Sequence
{
    using V = typename Value<T>::type;
    const Drafts& d;
    int first, nodes;

    __device__ Sequence(const Drafts& drafts, int s) : d(drafts)
    {
        first = d.starts[s];
        const int end = min(d.starts[s + 1], d.rows);
        nodes = first < 0 ? 0 : min(max(end - first, 0), d.max_nodes);
    }
    __device__ __forceinline__ Rows<T, Draft> rows(int node) const
    {
        return {static_cast<const V*>(d.target) + std::size_t(first + node) * d.target_stride,
                Draft ? static_cast<const V*>(d.draft) + std::size_t(first + node) * d.draft_stride : nullptr, d.alphabet};
    }
};

// A sequence's tree, and a wave's first 64 nodes of it in its lanes: parents, and whether a node is
// accepted if it is the first child that is tried.
struct Tree
{
    const Shared& shared;
    int nodes, parent;
    uint64_t first_accepted;

    template <bool Draft> __device__ __forceinline__ void read()
    {
        const int lane = threadIdx.x % 64;
        const bool here = lane < nodes;
        parent = here ? shared.parents[lane] : -1;
        first_accepted = __ballot(here && shared.uniforms[lane] * (Draft ? shared.draft[lane] : 1.0) < shared.target[lane]);
    }
    // The next child of `node` behind `after`, -1 if there is none.
    __device__ __forceinline__ int next_child(int node, int after) const
    {
        const int lane = threadIdx.x % 64;
        if (after < 63)
        {
            const uint64_t children = __ballot(lane > after && parent == node);
            if (children)
            {
                return __builtin_ctzll(children);
            }
        }
        for (int base = max((after + 1) / 64, 1) * 64; base < nodes; base += 64)
        {
            const int i = base + lane;
            const uint64_t children = __ballot(i > after && i < nodes && shared.parents[i] == node);
            if (children)
            {
                return base + __builtin_ctzll(children);
            }
        }
        return -1;
    }
};

// What a node's children came to: the one accepted, -1 if none, and what those refused took.
struct Outcome
{
    double shift;
    int child, struck;
};

// Reads a sequence's tree into LDS, and what decides over its nodes.
template <Type T, bool Draft>
__device__ __forceinline__ void read_tree(const Sequence<T, Draft>& sequence, Shared& shared)
{
    using V = typename Value<T>::type;
    const Drafts& d = sequence.d;
    const int first = sequence.first;
    for (int i = threadIdx.x; i < sequence.nodes; i += blockDim.x)
    {
        const int parent = i ? d.parents[first + i] : -1;
        const bool known = parent >= 0 && parent < i; // anything else is never reached
        shared.parents[i] = known ? parent : -1;
        const int token = d.tokens[first + i];
        const bool valid = known && token >= 0 && token < d.alphabet;
        shared.tokens[i] = token;
        shared.uniforms[i] = d.uniforms[first + i];
        const std::size_t row = first + (known ? parent : 0);
        shared.target[i] =
            valid ? probability<T>(static_cast<const V*>(d.target)[row * d.target_stride + token]) : 0.0;
        if constexpr (Draft)
        {
            shared.draft[i] =
                valid ? probability<T>(static_cast<const V*>(d.draft)[row * d.draft_stride + token]) : 0.0;
        }
    }
    __syncthreads();
}

// Tries a node's children in order, the same in every wave. The node's row is opened where it has to
// be summed.
template <Type T, bool Draft>
__device__ __forceinline__ Outcome try_children(const Sequence<T, Draft>& sequence, const Tree& tree, int node,
                                                Shared& shared, Summed<T, Draft>& row, bool& opened)
{
    const int lane = threadIdx.x % 64;
    int child = tree.next_child(node, node);
    opened = false;
    if (child >= 0 && child < 64 && tree.first_accepted >> child & 1)
    {
        return {0, child, 0};
    }
    Taken taken{0, shared.struck, 0};
    double weight = 1;
    while (child >= 0)
    {
        const double u = shared.uniforms[child], p = shared.target[child];
        if constexpr (Draft)
        {
            const double q = shared.draft[child], left = __builtin_fma(-taken.shift, q, p);
            if (u * q * weight < (left > 0.0 ? left : 0.0))
            {
                return {taken.shift, child, 0};
            }
            taken.shift += weight;
            child = tree.next_child(node, child);
            if (child >= 0)
            {
                if (!opened)
                {
                    row.open(sequence.rows(node));
                    opened = true;
                }
                weight = row.weigh(taken, shared.sums);
            }
        }
        else
        {
            const int token = shared.tokens[child];
            bool gone = false; // refused before, as another child
            for (int base = 0; base < taken.count && !gone; base += 64)
            {
                gone = __any(base + lane < taken.count && shared.struck[base + lane] == token);
            }
            const double left = gone ? 0.0 : p;
            if (u * weight < left)
            {
                return {0, child, 0};
            }
            __syncthreads();
            if (threadIdx.x == 0)
            {
                shared.struck[taken.count] = token;
            }
            __syncthreads();
            ++taken.count;
            weight -= left;
            child = tree.next_child(node, child);
        }
    }
    return {taken.shift, -1, taken.count};
}

// Workgroups stand for (sequence, chunk of the alphabet): every one follows the sequence's path for
// itself, each of its waves too, and sums its chunk of the row where the path ends. With one
// chunk it draws the token as well; otherwise draw_kernel does.
template <Type T, bool Draft>
__global__ __launch_bounds__(1024) void verify_kernel(Drafts d, int chunks, Walk* walks, double* chunk_sums)
{
    extern __shared__ char memory[];
    auto& shared = *reinterpret_cast<Shared*>(memory);
    const int s = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const Sequence<T, Draft> sequence(d, s);
    const int nodes = sequence.nodes;
    int* const path = d.path + std::size_t(s) * d.max_nodes;
    const bool writes = threadIdx.x == 0 && chunk == 0;
    const double goal = d.draws[s];
    Tree tree{shared, nodes, -1, 0};
    read_tree(sequence, shared);
    tree.template read<Draft>();
    // Node 0, then the accepted ones.
    int node = nodes ? 0 : -1, kept = 0;
    Summed<T, Draft> row;
    while (node >= 0)
    {
        if (writes)
        {
            path[kept] = node;
        }
        ++kept;
        bool opened = false;
        const Outcome outcome = try_children(sequence, tree, node, shared, row, opened);
        if (outcome.child >= 0)
        {
            node = outcome.child;
            continue;
        }
        // The path ends here: what is left of the row is drawn from.
        Taken taken{outcome.shift, shared.struck, outcome.struck};
        if (chunks > 1)
        {
            if (writes)
            {
                walks[s] = {outcome.shift, node, outcome.struck};
            }
            row.rows = sequence.rows(node);
            row.segments = (d.alphabet + segment - 1) / segment;
            const int each = (row.segments + chunks - 1) / chunks;
            row.sum_range(min(chunk * each, row.segments), min((chunk + 1) * each, row.segments), taken,
                          chunk_sums + std::size_t(s) * row.segments);
            break;
        }
        if (!opened)
        {
            row.open(sequence.rows(node));
        }
        double total = row.sum(taken, shared.sums);
        if (!(total > 0.0))
        {
            taken = {0, shared.struck, 0};
            total = row.sum(taken, shared.sums);
        }
        if (total > 0.0)
        {
            row.draw(taken, goal * total, shared.sums, d.next + s);
        }
        else if (writes)
        {
            d.next[s] = -1;
        }
        break;
    }
    if (chunk == 0)
    {
        for (int i = kept + threadIdx.x; i < d.max_nodes; i += blockDim.x)
        {
            path[i] = -1;
        }
    }
    if (writes)
    {
        d.accepted[s] = kept;
        if (!nodes)
        {
            d.next[s] = -1;
            if (chunks > 1)
            {
                walks[s] = {0, -1, 0};
            }
        }
    }
}

// The token that follows, from the chunks' sums. Where the path ended every child was refused, so
// that those struck out are the node's children.
template <Type T, bool Draft>
__global__ __launch_bounds__(256) void draw_kernel(Drafts d, const Walk* __restrict__ walks,
                                                   const double* __restrict__ chunk_sums)
{
    __shared__ double sums[max_segments];
    __shared__ int struck[max_draft_nodes];
    __shared__ int count;
    const int s = blockIdx.x;
    const Walk walk = walks[s];
    if (walk.node < 0)
    {
        return;
    }
    const double goal = d.draws[s];
    const int segments = (d.alphabet + segment - 1) / segment;
    for (int i = threadIdx.x; i < segments; i += blockDim.x)
    {
        sums[i] = chunk_sums[std::size_t(s) * segments + i];
    }
    const Sequence<T, Draft> sequence(d, s);
    if (!Draft && walk.struck)
    {
        if (threadIdx.x == 0)
        {
            count = 0;
        }
        __syncthreads();
        for (int i = walk.node + 1 + int(threadIdx.x); i < sequence.nodes; i += blockDim.x)
        {
            if (d.parents[sequence.first + i] == walk.node)
            {
                struck[atomicAdd(&count, 1)] = d.tokens[sequence.first + i]; // in any order
            }
        }
    }
    __syncthreads();
    Taken taken{walk.shift, struck, walk.struck};
    Summed<T, Draft> row;
    row.rows = sequence.rows(walk.node);
    row.segments = segments;
    double total = total_of(sums, segments);
    if (!(total > 0.0))
    {
        taken = {0, struck, 0};
        total = row.sum(taken, sums);
    }
    if (total > 0.0)
    {
        row.draw(taken, goal * total, sums, d.next + s);
    }
    else if (threadIdx.x == 0)
    {
        d.next[s] = -1;
    }
}

// Chunks of the alphabet of one sequence, a workgroup each; what follows is drawn by a second launch
// then, 4 to 5 us. Every one follows the path for itself and with drafts sums whole rows for it, so that
// they gain where all run at once: a workgroup a unit with drafts, two without, and none below four chunks. Over
// 128,001 values in BF16, several chunks and one: with drafts, trees of 16 nodes of up to four children, 4
// sequences 56 us and 66, 32 of them 67 and 73 (15 chunks each: 81), 64 72 and 75 (144); without, 4 sequences 12
// and 28, 64 19 and 33 (15 chunks: 24), 128 26 and 33 (8: 29), 256 42 and 35. Over 50,257 with drafts 128
// sequences are 44 in two chunks, 42 in one.
int chunks_of(int sequences, int alphabet, bool draft)
{
    const int room = (draft ? 1 : 2) * compute_units() / std::max(1, sequences);
    const int chunks = std::min(alphabet / 8192, room);
    return chunks < 4 ? 1 : chunks;
}

struct Workspace
{
    std::size_t walks = 0, sums = 0, bytes = 0; // offsets, and the whole

    explicit Workspace(const Drafts& d)
    {
        const auto room = [&](std::size_t size)
        {
            const std::size_t at = bytes;
            bytes += (size + 255) / 256 * 256;
            return at;
        };
        if (!d.sequences)
        {
            return;
        }
        if (chunks_of(d.sequences, d.alphabet, false) > 1) // with drafts there are no more
        {
            walks = room(d.sequences * sizeof(Walk));
            sums = room(std::size_t(d.sequences) * ((d.alphabet + segment - 1) / segment) * 8);
        }
    }
};
} // namespace

std::size_t verify_drafts_workspace(const Drafts& drafts)
{
    return Workspace(drafts).bytes;
}

void verify_drafts(const Drafts& drafts, void* workspace, std::size_t bytes, hipStream_t stream)
{
    if (!drafts.sequences)
    {
        return;
    }
    const Workspace space(drafts);
    require(!space.bytes || (workspace && bytes >= space.bytes), "verify: the workspace is too small");
    const int chunks = chunks_of(drafts.sequences, drafts.alphabet, drafts.draft != nullptr);
    char* const memory = static_cast<char*>(workspace);
    auto* const walks = reinterpret_cast<Walk*>(memory + space.walks);
    auto* const sums = reinterpret_cast<double*>(memory + space.sums);
    // Four waves where each has a segment or two (3 sequences over 1,024 values: 7.6 us, with eight 8.1,
    // with sixteen 9.7), eight where a walk sums no rows, only the chunk it ends with (64 sequences
    // over 128,001, 15 chunks: 20 us, with sixteen 30), sixteen otherwise (32 over 32,000: 25 us, with eight 28).
    const unsigned threads = drafts.alphabet <= 8 * segment ? 256 : chunks > 1 && !drafts.draft ? 512 : 1024;
    const auto launch = [&](auto type, auto draft)
    {
        constexpr Type T = decltype(type)::value;
        constexpr bool Draft = decltype(draft)::value;
        verify_kernel<T, Draft><<<unsigned(drafts.sequences) * chunks, threads, sizeof(Shared), stream>>>(
            drafts, chunks, walks, sums);
        check_hip(hipGetLastError(), "verify launch");
        if (chunks > 1)
        {
            draw_kernel<T, Draft><<<unsigned(drafts.sequences), 256, 0, stream>>>(drafts, walks, sums);
            check_hip(hipGetLastError(), "verify launch");
        }
    };
    const auto by_draft = [&](auto type)
    { drafts.draft ? launch(type, std::true_type{}) : launch(type, std::false_type{}); };
    switch (drafts.type)
    {
    case 0: by_draft(std::integral_constant<Type, Type::bf16>{}); break;
    case 1: by_draft(std::integral_constant<Type, Type::half>{}); break;
    default: by_draft(std::integral_constant<Type, Type::single>{}); break;
    }
}
} // namespace tsac_hip

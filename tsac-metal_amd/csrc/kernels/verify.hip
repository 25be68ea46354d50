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

namespace tsac_hip
{
namespace
{
constexpr int threads = 1024;
constexpr int waves = threads / 64;
constexpr int vector_width = 8;             // values a lane reads at a time
constexpr int segment = 64 * vector_width;  // values of one wave's step
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
    float v;
    if constexpr (T == Type::bf16)
    {
        v = __uint_as_float(unsigned(bits) << 16);
    }
    else if constexpr (T == Type::half)
    {
        v = float(__builtin_bit_cast(_Float16, bits));
    }
    else
    {
        v = bits;
    }
    return v > 0.0f && v < __builtin_inff() ? double(v) : 0.0;
}

// The eight values from `at`, zeros past the alphabet.
template <Type T>
__device__ __forceinline__ void load(const typename Value<T>::type* row, int at, int alphabet, double (&to)[vector_width])
{
    using V = typename Value<T>::type;
    V raw[vector_width];
    if (at + vector_width <= alphabet)
    {
        __builtin_memcpy(raw, row + at, sizeof raw); // at any alignment
    }
    else
    {
        for (int j = 0; j < vector_width; ++j)
        {
            raw[j] = at + j < alphabet ? row[at + j] : V(0);
        }
    }
#pragma unroll
    for (int j = 0; j < vector_width; ++j)
    {
        to[j] = probability<T>(raw[j]);
    }
}

__device__ __forceinline__ double wave_sum(double value)
{
#pragma unroll
    for (int step = 1; step < 64; step *= 2)
    {
        value += __shfl_xor(value, step);
    }
    return value;
}

__device__ __forceinline__ double wave_scan(double value, int lane)
{
#pragma unroll
    for (int step = 1; step < 64; step *= 2)
    {
        const double below = __shfl_up(value, step);
        value += lane >= step ? below : 0.0;
    }
    return value;
}

struct Shared
{
    int parents[max_draft_nodes], tokens[max_draft_nodes];
    float uniforms[max_draft_nodes];
    double target[max_draft_nodes], draft[max_draft_nodes]; // p and q of a node's token in its parent's row
    int struck[max_draft_nodes];
    double sums[max_segments];
    double total;
};

template <Type T, bool Draft> struct Rows
{
    using V = typename Value<T>::type;
    const V* target;
    const V* draft;
    int alphabet;

    // What is left of the eight values from `at`.
    __device__ __forceinline__ void left(int at, double shift, const int* struck, int count,
                                         double (&to)[vector_width]) const
    {
        load<T>(target, at, alphabet, to);
        if constexpr (Draft)
        {
            if (shift != 0.0)
            {
                double q[vector_width];
                load<T>(draft, at, alphabet, q);
#pragma unroll
                for (int j = 0; j < vector_width; ++j)
                {
                    const double w = to[j] - shift * q[j];
                    to[j] = w > 0.0 ? w : 0.0;
                }
            }
        }
        else
        {
            for (int k = 0; k < count; ++k)
            {
                const int j = struck[k] - at;
#pragma unroll
                for (int i = 0; i < vector_width; ++i)
                {
                    to[i] = i == j ? 0.0 : to[i];
                }
            }
        }
    }
};

// The sum of each segment of what is left, and of all of them, for every thread.
template <Type T, bool Draft>
__device__ double sum_left(const Rows<T, Draft>& rows, double shift, int struck, Shared& shared)
{
    const int lane = threadIdx.x % 64, warp = threadIdx.x / 64;
    const int segments = (rows.alphabet + segment - 1) / segment;
    for (int s = warp; s < segments; s += waves)
    {
        double value[vector_width];
        rows.left(s * segment + lane * vector_width, shift, shared.struck, struck, value);
        double sum = 0;
#pragma unroll
        for (int j = 0; j < vector_width; ++j)
        {
            sum += value[j];
        }
        sum = wave_sum(sum);
        if (lane == 0)
        {
            shared.sums[s] = sum;
        }
    }
    __syncthreads();
    if (warp == 0)
    {
        double total = 0;
        for (int base = 0; base < segments; base += 64)
        {
            total += wave_sum(base + lane < segments ? shared.sums[base + lane] : 0.0);
        }
        if (lane == 0)
        {
            shared.total = total;
        }
    }
    __syncthreads();
    const double total = shared.total;
    __syncthreads();
    return total;
}

// The lowest token whose inclusive sum passes `goal`, by the first wave, from the segments' sums;
// the last one with anything left if rounding passes over all.
template <Type T, bool Draft>
__device__ int find(const Rows<T, Draft>& rows, double shift, int struck, double goal, const Shared& shared)
{
    const int lane = threadIdx.x % 64;
    const int segments = (rows.alphabet + segment - 1) / segment;
    double front = 0; // sum of the segments in front
    int found = -1, last = 0;
    double before = 0;
    for (int base = 0; base < segments && found < 0; base += 64)
    {
        const double mine = base + lane < segments ? shared.sums[base + lane] : 0.0;
        const double inclusive = front + wave_scan(mine, lane);
        const uint64_t past = __ballot(inclusive > goal && mine > 0.0), some = __ballot(mine > 0.0);
        const int at = past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : -1;
        if (at >= 0)
        {
            last = base + at;
            before = __shfl(inclusive - mine, at);
            found = past ? last : -1;
        }
        front = __shfl(inclusive, 63);
    }
    double value[vector_width];
    const int first = last * segment + lane * vector_width;
    rows.left(first, shift, shared.struck, struck, value);
    double sum = 0;
#pragma unroll
    for (int j = 0; j < vector_width; ++j)
    {
        sum += value[j];
    }
    double inclusive = before + (wave_scan(sum, lane) - sum);
    int token = -1, some = -1;
#pragma unroll
    for (int j = 0; j < vector_width; ++j)
    {
        inclusive += value[j];
        token = token < 0 && value[j] > 0.0 && inclusive > goal ? first + j : token;
        some = value[j] > 0.0 ? first + j : some;
    }
    const uint64_t past = __ballot(token >= 0), any = __ballot(some >= 0);
    return past  ? __shfl(token, __builtin_ctzll(past))
           : any ? __shfl(some, 63 - __builtin_clzll(any))
                 : -1;
}

// The next child of `node` behind `after`, -1 if there is none; the same in every wave.
__device__ __forceinline__ int next_child(const Shared& shared, int nodes, int node, int after)
{
    const int lane = threadIdx.x % 64;
    for (int base = (after + 1) / 64 * 64; base < nodes; base += 64)
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

// A workgroup a sequence; every wave follows the same path through the tree, and the
// workgroup shares the sums over a row.
template <Type T, bool Draft> __global__ __launch_bounds__(threads) void verify_kernel(Drafts d)
{
    using V = typename Value<T>::type;
    extern __shared__ char memory[];
    auto& shared = *reinterpret_cast<Shared*>(memory);
    const int s = blockIdx.x, first = d.starts[s];
    const int end = d.starts[s + 1] < d.rows ? d.starts[s + 1] : d.rows;
    int nodes = first < 0 || end < first ? 0 : end - first;
    nodes = nodes < d.max_nodes ? nodes : d.max_nodes;
    int* const path = d.path + std::size_t(s) * d.max_nodes;
    const auto target_row = [&](int node)
    { return static_cast<const V*>(d.target) + std::size_t(first + node) * d.target_stride; };
    const auto draft_row = [&](int node)
    { return static_cast<const V*>(d.draft) + std::size_t(first + node) * d.draft_stride; };
    for (int i = threadIdx.x; i < nodes; i += threads)
    {
        const int parent = i ? d.parents[first + i] : -1, token = d.tokens[first + i];
        const bool known = parent >= 0 && parent < i; // anything else is never reached
        const bool valid = known && token >= 0 && token < d.alphabet;
        shared.parents[i] = known ? parent : -1;
        shared.tokens[i] = token;
        shared.uniforms[i] = d.uniforms[first + i];
        shared.target[i] = valid ? probability<T>(target_row(parent)[token]) : 0.0;
        if constexpr (Draft)
        {
            shared.draft[i] = valid ? probability<T>(draft_row(parent)[token]) : 0.0;
        }
    }
    __syncthreads();
    if (!nodes)
    {
        for (int i = threadIdx.x; i < d.max_nodes; i += threads)
        {
            path[i] = -1;
        }
        if (threadIdx.x == 0)
        {
            d.accepted[s] = 0;
            d.next[s] = -1;
        }
        return;
    }
    int node = 0, kept = 1, struck = 0;
    double shift = 0;
    if (threadIdx.x == 0)
    {
        path[0] = 0;
    }
    for (;;)
    {
        double weight = 1;
        int taken = -1;
        shift = 0;
        struck = 0;
        for (int child = next_child(shared, nodes, node, node); child >= 0;)
        {
            const double u = shared.uniforms[child], p = shared.target[child];
            if constexpr (Draft)
            {
                const double q = shared.draft[child], left = p - shift * q;
                if (u * q * weight < (left > 0.0 ? left : 0.0))
                {
                    taken = child;
                    break;
                }
                shift += weight;
                child = next_child(shared, nodes, node, child);
                if (child >= 0)
                {
                    weight = sum_left(Rows<T, Draft>{target_row(node), draft_row(node), d.alphabet}, shift, 0, shared);
                }
            }
            else
            {
                const int lane = threadIdx.x % 64, token = shared.tokens[child];
                bool gone = false; // refused before, as another child
                for (int base = 0; base < struck && !gone; base += 64)
                {
                    gone = __any(base + lane < struck && shared.struck[base + lane] == token);
                }
                const double left = gone ? 0.0 : p;
                if (u * weight < left)
                {
                    taken = child;
                    break;
                }
                __syncthreads();
                if (threadIdx.x == 0)
                {
                    shared.struck[struck] = token;
                }
                __syncthreads();
                ++struck;
                weight -= left;
                child = next_child(shared, nodes, node, child);
            }
        }
        if (taken < 0)
        {
            break;
        }
        node = taken;
        if (threadIdx.x == 0)
        {
            path[kept] = node;
        }
        ++kept;
    }
    const Rows<T, Draft> rows{target_row(node), Draft ? draft_row(node) : nullptr, d.alphabet};
    double total = sum_left(rows, shift, struck, shared);
    if (!(total > 0.0))
    {
        shift = 0;
        struck = 0;
        total = sum_left(rows, shift, struck, shared);
    }
    if (threadIdx.x < 64)
    {
        const int token = total > 0.0 ? find(rows, shift, struck, double(d.draws[s]) * total, shared) : -1;
        if (threadIdx.x == 0)
        {
            d.accepted[s] = kept;
            d.next[s] = token;
        }
    }
    for (int i = kept + threadIdx.x; i < d.max_nodes; i += threads)
    {
        path[i] = -1;
    }
}
} // namespace

std::size_t verify_drafts_workspace(const Drafts&)
{
    return 0;
}

void verify_drafts(const Drafts& drafts, void*, std::size_t, hipStream_t stream)
{
    if (!drafts.sequences)
    {
        return;
    }
    require(drafts.alphabet > 0 && drafts.alphabet <= max_alphabet, "verify: alphabets of 1 to 2^20 tokens");
    const auto launch = [&](auto kernel)
    {
        kernel<<<unsigned(drafts.sequences), threads, sizeof(Shared), stream>>>(drafts);
        check_hip(hipGetLastError(), "verify launch");
    };
    const bool draft = drafts.draft != nullptr;
    switch (drafts.type)
    {
    case 0: draft ? launch(verify_kernel<Type::bf16, true>) : launch(verify_kernel<Type::bf16, false>); break;
    case 1: draft ? launch(verify_kernel<Type::half, true>) : launch(verify_kernel<Type::half, false>); break;
    default: draft ? launch(verify_kernel<Type::single, true>) : launch(verify_kernel<Type::single, false>); break;
    }
}
} // namespace tsac_hip

// The pages of a key/value cache: taking, sharing, writing, compacting and giving them back.
//
// A page is free while its reference count is 0. Calls that take pages take the lowest free
// ones, in the order of their list, from one workgroup that scans the counts: what a
// sequence gets depends on the counts and the list alone, on no order of atomics and no
// history of calls.
#include "paged.hpp"

#include <algorithm>

namespace tsac_hip
{
namespace
{
constexpr int taking_threads = 1024;
constexpr int taking_waves = taking_threads / 64;
constexpr int scanned = 4; // reference counts a thread reads at a time

__device__ __forceinline__ void report(int* status, int what)
{
    if (status)
    {
        *status = what;
    }
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ long long wave_scan(long long value, int lane)
{
#pragma unroll
    for (int step = 1; step < 64; step *= 2)
    {
        const long long below = __shfl_up(value, step);
        value += lane >= step ? below : 0;
    }
    return value;
}

struct TakingShared
{
    int before[max_listed_sequences + 1]; // pages taken by the entries in front of each one
    unsigned seen[max_sequences / 32 + 1];
    long long sums[taking_waves];
    int bad, stopped;
};

// Exclusive sums of each entry's need into `before`, for the whole workgroup; returns the total.
template <class Need> __device__ long long sum_needs(TakingShared& shared, int count, Need need)
{
    const int lane = threadIdx.x % 64, warp = threadIdx.x / 64;
    long long total = 0;
    for (int base = 0; base < count; base += taking_threads)
    {
        const int i = base + threadIdx.x;
        const long long mine = i < count ? need(i) : 0;
        const long long inclusive = wave_scan(mine, lane);
        if (lane == 63)
        {
            shared.sums[warp] = inclusive;
        }
        __syncthreads();
        long long front = total, all = 0;
        for (int w = 0; w < taking_waves; ++w)
        {
            front += w < warp ? shared.sums[w] : 0;
            all += shared.sums[w];
        }
        if (i < count)
        {
            // Beyond 2^31 the call fails: there are fewer pages.
            shared.before[i] = int(front + inclusive - mine);
        }
        total += all;
        __syncthreads();
    }
    if (threadIdx.x == 0)
    {
        shared.before[count] = int(total);
    }
    __syncthreads();
    return total;
}

// Hands the `total` lowest free pages to take(entry, index within the entry's need, page), in
// order, and counts them once; false, with what was handed out given to undo(), if there are
// too few. The counts are read four a thread; the scan ends as soon as enough are found.
template <class Take, class Undo>
__device__ bool take_pages(TakingShared& shared, int count, int total, int* references, int pages, Take take, Undo undo)
{
    const int lane = threadIdx.x % 64, warp = threadIdx.x / 64;
    int found = 0;
    const auto entry = [&](int rank)
    {
        int low = 0, high = count; // the last entry with before <= rank
        while (high - low > 1)
        {
            const int middle = (low + high) / 2;
            (shared.before[middle] <= rank ? low : high) = middle;
        }
        return low;
    };
    for (long long base = 0; base < pages && found < total; base += taking_threads * scanned)
    {
        const long long first = base + threadIdx.x * scanned;
        unsigned free = 0;
#pragma unroll
        for (int j = 0; j < scanned; ++j)
        {
            free |= (first + j < pages && references[first + j] == 0 ? 1u : 0u) << j;
        }
        const long long inclusive = wave_scan(__popc(free), lane);
        if (lane == 63)
        {
            shared.sums[warp] = inclusive;
        }
        __syncthreads();
        int rank = found + int(inclusive) - __popc(free), all = 0;
        for (int w = 0; w < taking_waves; ++w)
        {
            rank += w < warp ? int(shared.sums[w]) : 0;
            all += int(shared.sums[w]);
        }
#pragma unroll
        for (int j = 0; j < scanned; ++j)
        {
            if (free >> j & 1)
            {
                if (rank < total)
                {
                    const int i = entry(rank), page = int(first + j);
                    take(i, rank - shared.before[i], page);
                    references[page] = 1;
                }
                ++rank;
            }
        }
        found += all;
        __syncthreads();
    }
    if (found >= total)
    {
        return true;
    }
    for (int rank = threadIdx.x; rank < found; rank += taking_threads)
    {
        const int i = entry(rank);
        references[undo(i, rank - shared.before[i])] = 0;
    }
    return false;
}

__device__ __forceinline__ void clear_seen(TakingShared& shared)
{
    for (int i = threadIdx.x; i < max_sequences / 32 + 1; i += taking_threads)
    {
        shared.seen[i] = 0;
    }
    if (threadIdx.x == 0)
    {
        shared.bad = 0;
    }
    __syncthreads();
}

__global__ __launch_bounds__(taking_threads) void reserve_kernel(PagedCache cache, const int* __restrict__ sequences,
                                                                 const int* __restrict__ rows, int count, int* status)
{
    extern __shared__ char memory[];
    auto& shared = *reinterpret_cast<TakingShared*>(memory);
    clear_seen(shared);
    const auto sequence = [&](int i) { return sequences ? sequences[i] : i; };
    // Checked below before it is used.
    const auto need = [&](int i) -> long long
    {
        const int s = sequence(i);
        const long long last = (long long)cache.lengths[s] + rows[i];
        const long long pages = (last + cache.page_rows - 1) / cache.page_rows - cache.held[s];
        return pages > 0 ? pages : 0;
    };
    for (int i = threadIdx.x; i < count; i += taking_threads)
    {
        const int s = sequence(i);
        bool ok = s >= 0 && s < cache.sequences;
        if (ok)
        {
            ok = !(atomicOr(&shared.seen[s / 32], 1u << s % 32) >> s % 32 & 1) && rows[i] >= 0 && cache.lengths[s] >= 0 &&
                 cache.held[s] >= 0 && std::size_t(cache.held[s]) <= cache.table_stride &&
                 std::size_t((cache.lengths[s] + (long long)rows[i] + cache.page_rows - 1) / cache.page_rows) <=
                     cache.table_stride;
        }
        if (!ok)
        {
            shared.bad = 1;
        }
    }
    __syncthreads();
    if (shared.bad)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_invalid);
        }
        return;
    }
    const long long total = sum_needs(shared, count, need);
    const auto slot = [&](int i, int j) -> int&
    {
        const int s = sequence(i);
        return cache.table[s * cache.table_stride + cache.held[s] + j];
    };
    const bool enough =
        total <= cache.pages && take_pages(
                                    shared, count, int(total), cache.references, cache.pages,
                                    [&](int i, int j, int page) { slot(i, j) = page; },
                                    [&](int i, int j)
                                    {
                                        const int page = slot(i, j);
                                        slot(i, j) = -1;
                                        return page;
                                    });
    if (!enough)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_exhausted);
        }
        return;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += taking_threads)
    {
        cache.held[sequence(i)] += shared.before[i + 1] - shared.before[i];
    }
}

// While a fork runs, a target's `held` says so: what it will hold, `forking`, and above it how
// many workgroups of fork_copy_kernel are done with the target; the last one leaves the
// number alone. A refused call sets no such mark, so that the second kernel does nothing.
constexpr int forking = 1 << 30, arrival = 1 << 21;
static_assert(max_table_pages < arrival && 2 * max_layers + 1 < forking / arrival);

// Checks the list, takes a page for each source's last partial one and makes the targets
// hold their pages; what is shared and copied follows in fork_copy_kernel.
__global__ __launch_bounds__(taking_threads) void fork_kernel(PagedCache cache, const int* __restrict__ sources,
                                                              const int* __restrict__ targets, int count, int* status)
{
    extern __shared__ char memory[];
    auto& shared = *reinterpret_cast<TakingShared*>(memory);
    clear_seen(shared);
    for (int i = threadIdx.x; i < count; i += taking_threads)
    {
        const int t = targets[i];
        if (t < 0 || t >= cache.sequences || (atomicOr(&shared.seen[t / 32], 1u << t % 32) >> t % 32 & 1) ||
            cache.held[t] != 0)
        {
            shared.bad = 1;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += taking_threads)
    {
        const int s = sources[i];
        bool ok = s >= 0 && s < cache.sequences && !(shared.seen[s / 32] >> s % 32 & 1);
        if (ok)
        {
            ok = cache.lengths[s] >= 0 && cache.held[s] >= 0 && std::size_t(cache.held[s]) <= cache.table_stride &&
                 (cache.lengths[s] + (long long)cache.page_rows - 1) / cache.page_rows <= cache.held[s];
        }
        if (!ok)
        {
            shared.bad = 1;
        }
    }
    __syncthreads();
    if (shared.bad)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_invalid);
        }
        return;
    }
    const auto partial = [&](int i) -> long long { return cache.lengths[sources[i]] % cache.page_rows != 0; };
    const long long total = sum_needs(shared, count, partial);
    const auto slot = [&](int i) -> int&
    { return cache.table[targets[i] * cache.table_stride + cache.lengths[sources[i]] / cache.page_rows]; };
    const bool enough = take_pages(
        shared, count, int(total), cache.references, cache.pages, [&](int i, int, int page) { slot(i) = page; },
        [&](int i, int)
        {
            const int page = slot(i);
            slot(i) = -1;
            return page;
        });
    if (!enough)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_exhausted);
        }
        return;
    }
    for (int i = threadIdx.x; i < count; i += taking_threads)
    {
        const int length = cache.lengths[sources[i]];
        cache.lengths[targets[i]] = length;
        cache.held[targets[i]] = forking | int((length + (long long)cache.page_rows - 1) / cache.page_rows);
    }
}

constexpr int copying_threads = 256;

// Shares the full pages.
__device__ __forceinline__ void share_pages(const PagedCache& cache, const int* from, int* to, int full, int* status)
{
    for (int j = threadIdx.x; j < full; j += copying_threads)
    {
        int page = from[j];
        if (page < 0 || page >= cache.pages)
        {
            report(status, status_invalid);
            page = -1;
        }
        else
        {
            atomicAdd(&cache.references[page], 1);
        }
        to[j] = page;
    }
}

// Copies the rows of the last page, of one layer's keys or values.
__device__ __forceinline__ void copy_rows(const PagedCache& cache, int part, int old, int fresh, int rest, int* status)
{
    if (old < 0 || old >= cache.pages || fresh < 0 || fresh >= cache.pages)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_invalid);
        }
        return;
    }
    uint16_t* const memory = (part % 2 ? cache.values : cache.keys) + part / 2 * cache.layer_stride;
    const int vectors = cache.heads * cache.head_width / 8;
    for (int i = threadIdx.x; i < rest * vectors; i += copying_threads)
    {
        const std::size_t at = i / vectors * cache.row_stride + i % vectors * 8;
        const uint4 value = *reinterpret_cast<const uint4*>(memory + old * cache.page_stride + at);
        *reinterpret_cast<uint4*>(memory + fresh * cache.page_stride + at) = value;
    }
}

// blockIdx: the entry of the list, then (layer, keys or values), past the last of them the
// sharing.
__global__ __launch_bounds__(copying_threads) void fork_copy_kernel(PagedCache cache, const int* __restrict__ sources,
                                                                    const int* __restrict__ targets, int* status)
{
    __shared__ int mark;
    const int target = targets[blockIdx.x], source = sources[blockIdx.x];
    if (target < 0 || target >= cache.sequences || source < 0 || source >= cache.sequences)
    {
        return; // refused
    }
    if (threadIdx.x == 0)
    {
        mark = __hip_atomic_load(&cache.held[target], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (mark < forking)
    {
        return; // refused
    }
    const int length = cache.lengths[target];
    const int full = length / cache.page_rows, rest = length % cache.page_rows;
    const int* const from = cache.table + source * cache.table_stride;
    int* const to = cache.table + target * cache.table_stride;
    if (int(blockIdx.y) == 2 * cache.layers)
    {
        share_pages(cache, from, to, full, status);
    }
    else if (rest)
    {
        copy_rows(cache, blockIdx.y, from[full], to[full], rest, status);
    }
    if (threadIdx.x == 0)
    {
        const int before = atomicAdd(&cache.held[target], arrival);
        if ((before & (forking - 1)) / arrival == 2 * cache.layers)
        {
            __hip_atomic_store(&cache.held[target], before & (arrival - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// A workgroup a listed sequence. The first to take what it holds gives it back: a sequence
// listed twice is freed once.
__global__ __launch_bounds__(copying_threads) void free_kernel(PagedCache cache, const int* __restrict__ sequences,
                                                               int* status)
{
    __shared__ int held;
    const int s = sequences ? sequences[blockIdx.x] : int(blockIdx.x);
    if (s < 0 || s >= cache.sequences)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_invalid);
        }
        return;
    }
    if (threadIdx.x == 0)
    {
        held = atomicExch(&cache.held[s], 0);
        if (held)
        {
            cache.lengths[s] = 0;
        }
    }
    __syncthreads();
    int* const table = cache.table + s * cache.table_stride;
    const int count = held < 0 ? 0 : std::size_t(held) < cache.table_stride ? held : int(cache.table_stride);
    for (int j = threadIdx.x; j < count; j += copying_threads)
    {
        const int page = table[j];
        table[j] = -1;
        if (page < 0 || page >= cache.pages || atomicSub(&cache.references[page], 1) <= 0)
        {
            if (page >= 0 && page < cache.pages)
            {
                atomicAdd(&cache.references[page], 1); // it was not counted
            }
            report(status, status_invalid);
        }
    }
}

// The page of a position that its sequence may write, -1 if there is none: covered by what the
// sequence holds, and held by it alone.
__device__ __forceinline__ int writable_page(const PagedCache& cache, int s, long long position)
{
    const long long index = position / cache.page_rows;
    if (position < 0 || index >= cache.held[s] || std::size_t(index) >= cache.table_stride)
    {
        return -1;
    }
    const int page = cache.table[s * cache.table_stride + index];
    return page >= 0 && page < cache.pages && cache.references[page] == 1 ? page : -1;
}

// A sequence's rows among `rows`, from the ascending starts.
__device__ __forceinline__ int rows_of(const int* starts, int s, int rows, int& first)
{
    first = starts[s];
    const int end = starts[s + 1] < rows ? starts[s + 1] : rows;
    return first < 0 || end < first ? 0 : end - first;
}

// blockIdx: a row's place in its sequence, the sequence, the layer.
__global__ __launch_bounds__(copying_threads) void write_kernel(PagedCache cache, int layer, NewRows fresh,
                                                                const int* __restrict__ starts, int* status)
{
    const int row = blockIdx.x, s = blockIdx.y;
    int first;
    if (row >= rows_of(starts, s, fresh.rows, first))
    {
        return;
    }
    const long long position = (long long)cache.lengths[s] + row;
    const int page = writable_page(cache, s, position);
    if (page < 0)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_invalid);
        }
        return;
    }
    const std::size_t to = (layer + blockIdx.z) * cache.layer_stride + page * cache.page_stride +
                           position % cache.page_rows * cache.row_stride;
    const std::size_t from = blockIdx.z * fresh.layer_stride + std::size_t(first + row) * fresh.row_stride;
    const int vectors = cache.heads * cache.head_width / 8;
    for (int i = threadIdx.x; i < 2 * vectors; i += copying_threads)
    {
        const bool value = i >= vectors;
        const std::size_t at = 8 * std::size_t(value ? i - vectors : i);
        *reinterpret_cast<uint4*>((value ? cache.values : cache.keys) + to + at) =
            *reinterpret_cast<const uint4*>((value ? fresh.values : fresh.keys) + from + at);
    }
}

// How many rows a sequence keeps, -1 if its path is none: ascending nodes of its own.
__device__ __forceinline__ int kept_rows(const int* path, int accepted, int nodes, std::size_t path_stride, int* bad)
{
    if (threadIdx.x == 0)
    {
        *bad = accepted < 0 || accepted > nodes || std::size_t(accepted < 0 ? 0 : accepted) > path_stride;
    }
    __syncthreads();
    if (!*bad)
    {
        for (int k = threadIdx.x; k < accepted; k += blockDim.x)
        {
            if (path[k] < (k ? path[k - 1] + 1 : 0) || path[k] >= nodes)
            {
                *bad = 1;
            }
        }
    }
    __syncthreads();
    return *bad ? -1 : accepted;
}

constexpr int moved = 8; // rows a thread moves at a time

// blockIdx: 256 vectors of a row, the sequence, (layer, keys or values). A thread moves one
// vector of every kept row, in ascending order: row k comes from node path[k] >= k, so that
// reading `moved` rows before writing them never meets a row that was written already.
__global__ __launch_bounds__(copying_threads) void keep_kernel(PagedCache cache, const int* __restrict__ starts,
                                                               const int* __restrict__ path, std::size_t path_stride,
                                                               const int* __restrict__ accepted, int* lengths,
                                                               int* status)
{
    __shared__ int bad;
    const int s = blockIdx.y;
    const int length = cache.lengths[s];
    const int nodes = starts[s + 1] - starts[s];
    path += s * path_stride;
    const int kept = kept_rows(path, accepted[s], nodes, path_stride, &bad);
    const bool reporter = threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.z == 0;
    if (lengths && reporter)
    {
        lengths[s] = length + (kept > 0 ? kept : 0);
    }
    if (kept < 0 || length < 0)
    {
        if (reporter)
        {
            report(status, status_invalid);
        }
        return;
    }
    const int vector = blockIdx.x * copying_threads + threadIdx.x;
    if (vector >= cache.heads * cache.head_width / 8)
    {
        return;
    }
    uint16_t* const memory =
        (blockIdx.z % 2 ? cache.values : cache.keys) + blockIdx.z / 2 * cache.layer_stride + 8 * std::size_t(vector);
    const auto at = [&](int row) -> uint16_t*
    {
        const int page = writable_page(cache, s, (long long)length + row);
        return page < 0 ? nullptr
                        : memory + page * cache.page_stride + (length + (long long)row) % cache.page_rows * cache.row_stride;
    };
    int k = 0;
    while (k < kept && path[k] == k)
    {
        ++k;
    }
    for (; k < kept; k += moved)
    {
        uint4 value[moved];
        uint16_t* to[moved];
#pragma unroll
        for (int j = 0; j < moved; ++j)
        {
            const uint16_t* const from = k + j < kept ? at(path[k + j]) : nullptr;
            to[j] = from ? at(k + j) : nullptr;
            if (to[j])
            {
                value[j] = *reinterpret_cast<const uint4*>(from);
            }
            else if (k + j < kept)
            {
                report(status, status_invalid);
            }
        }
#pragma unroll
        for (int j = 0; j < moved; ++j)
        {
            if (to[j])
            {
                *reinterpret_cast<uint4*>(to[j]) = value[j];
            }
        }
    }
}

// The lengths in place, once every workgroup of keep_kernel has read them.
__global__ __launch_bounds__(64) void keep_lengths_kernel(const int* __restrict__ starts,
                                                          const int* __restrict__ path, std::size_t path_stride,
                                                          const int* __restrict__ accepted, int* lengths)
{
    __shared__ int bad;
    const int s = blockIdx.x;
    const int kept =
        kept_rows(path + s * path_stride, accepted[s], starts[s + 1] - starts[s], path_stride, &bad);
    if (threadIdx.x == 0 && kept > 0)
    {
        lengths[s] += kept;
    }
}

// A workgroup a sequence, a thread a node: the words from the node's own down, along its line.
__global__ __launch_bounds__(256) void tree_mask_kernel(const int* __restrict__ parents, int rows,
                                                        const int* __restrict__ starts, int max_nodes,
                                                        unsigned long long* __restrict__ mask, int words)
{
    __shared__ int above[max_draft_nodes];
    int first;
    int nodes = rows_of(starts, blockIdx.x, rows, first);
    nodes = nodes < max_nodes ? nodes : max_nodes;
    for (int i = threadIdx.x; i < nodes; i += blockDim.x)
    {
        const int parent = parents[first + i];
        above[i] = parent >= 0 && parent < i ? parent : -1; // anything else makes a root, so that every line ends
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nodes; i += blockDim.x)
    {
        int node = i;
        for (int w = words - 1; w >= 0; --w)
        {
            unsigned long long bits = 0;
            while (node >= 0 && node / 64 == w)
            {
                bits |= 1ull << node % 64;
                node = above[node];
            }
            mask[std::size_t(first + i) * words + w] = bits;
        }
    }
}
} // namespace

void pages_reserve(const PagedCache& cache, const int* sequences, const int* rows, std::size_t count, int* status,
                   hipStream_t stream)
{
    if (!count)
    {
        return;
    }
    reserve_kernel<<<1, taking_threads, sizeof(TakingShared), stream>>>(cache, sequences, rows, int(count), status);
    check_hip(hipGetLastError(), "pages reserve launch");
}

void pages_fork(const PagedCache& cache, const int* sources, const int* targets, std::size_t count, int* status,
                hipStream_t stream)
{
    if (!count)
    {
        return;
    }
    fork_kernel<<<1, taking_threads, sizeof(TakingShared), stream>>>(cache, sources, targets, int(count), status);
    check_hip(hipGetLastError(), "pages fork launch");
    const dim3 grid{unsigned(count), unsigned(2 * cache.layers + 1)};
    fork_copy_kernel<<<grid, copying_threads, 0, stream>>>(cache, sources, targets, status);
    check_hip(hipGetLastError(), "pages fork launch");
}

void pages_free(const PagedCache& cache, const int* sequences, std::size_t count, int* status, hipStream_t stream)
{
    if (!count)
    {
        return;
    }
    free_kernel<<<unsigned(count), copying_threads, 0, stream>>>(cache, sequences, status);
    check_hip(hipGetLastError(), "pages free launch");
}

void pages_write(const PagedCache& cache, int layer, int layers, const NewRows& fresh, const int* starts, int max_rows,
                 int* status, hipStream_t stream)
{
    if (!max_rows || !layers || !cache.sequences)
    {
        return;
    }
    const dim3 grid(static_cast<unsigned>(max_rows), static_cast<unsigned>(cache.sequences),
                    static_cast<unsigned>(layers));
    write_kernel<<<grid, copying_threads, 0, stream>>>(cache, layer, fresh, starts, status);
    check_hip(hipGetLastError(), "pages write launch");
}

void pages_keep(const PagedCache& cache, const int* starts, const int* path, std::size_t path_stride,
                const int* accepted, int* lengths, int* status, hipStream_t stream)
{
    if (!cache.sequences)
    {
        return;
    }
    const unsigned vectors = unsigned(cache.heads * cache.head_width / 8);
    const bool in_place = lengths == cache.lengths;
    const dim3 grid((vectors + copying_threads - 1) / copying_threads, unsigned(cache.sequences),
                    unsigned(2 * cache.layers));
    keep_kernel<<<grid, copying_threads, 0, stream>>>(cache, starts, path, path_stride, accepted,
                                                      in_place ? nullptr : lengths, status);
    check_hip(hipGetLastError(), "pages keep launch");
    if (in_place)
    {
        keep_lengths_kernel<<<unsigned(cache.sequences), 64, 0, stream>>>(starts, path, path_stride, accepted,
                                                                          lengths);
        check_hip(hipGetLastError(), "pages keep launch");
    }
}

void tree_mask(const int* parents, int rows, const int* starts, int sequences, int max_nodes, uint64_t* mask,
               std::size_t words, hipStream_t stream)
{
    if (!rows || !sequences)
    {
        return;
    }
    tree_mask_kernel<<<unsigned(sequences), 256, 0, stream>>>(
        parents, rows, starts, max_nodes, reinterpret_cast<unsigned long long*>(mask), int(words));
    check_hip(hipGetLastError(), "tree mask launch");
}
} // namespace tsac_hip

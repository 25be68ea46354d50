// The pages of a key/value cache: taking, sharing, writing, compacting and giving them back.
//
// A page is free while its reference count is 0. Calls that take pages take the lowest free
// ones, in the order of their list, from one workgroup that scans the counts: what a
// sequence gets depends on the counts and the list alone, on no order of atomics and no
// history of calls.
#include "paged_device.hpp"

#include <algorithm>

namespace tsac_hip
{
namespace
{
constexpr int most_threads = 1024; // of a workgroup that takes pages
constexpr int scanned = 4;         // reference counts a thread reads at a time

// Lanes below this one whose bit is set.
__device__ __forceinline__ int lanes_below(uint64_t bits)
{
    return __builtin_amdgcn_mbcnt_hi(unsigned(bits >> 32), __builtin_amdgcn_mbcnt_lo(unsigned(bits), 0));
}

struct TakingShared
{
    int before[max_listed_sequences + 1]; // pages taken by the entries in front of each one
    unsigned seen[max_sequences / 32 + 1];
    int sums[2][most_threads / 64];
    int bad;
};

// A list of sequences is checked and worked on by one workgroup of `Threads`, an entry a thread
// and round. The first round's reference counts are asked for at the start: they need nothing
// else, and each wait for memory here is a fifth of a small call.
template <int Threads> struct Taking
{
    static constexpr int waves = Threads / 64;
    TakingShared& shared;
    const PagedCache& cache;
    int count;
    int first_counts[scanned];
    const int lane = threadIdx.x % 64, warp = threadIdx.x / 64;

    __device__ Taking(TakingShared& s, const PagedCache& c, int n) : shared(s), cache(c), count(n)
    {
        read_counts(0, first_counts);
    }
    // Counts from `base` on, of the thread's pages; not 0 past the last page.
    __device__ __forceinline__ void read_counts(long long base, int (&counts)[scanned]) const
    {
        const long long first = base + threadIdx.x * scanned;
#pragma unroll
        for (int j = 0; j < scanned; ++j)
        {
            counts[j] = first + j < cache.pages ? cache.references[first + j] : 1;
        }
    }
    // Whether every entry passes, and names a sequence that no other one does.
    template <class Sequence, class Check> __device__ bool check(Sequence sequence, Check check_entry)
    {
        for (int i = threadIdx.x; i < count; i += Threads)
        {
            const int s = sequence(i);
            if (s >= 0 && s < cache.sequences)
            {
                shared.seen[s / 32] = 0;
            }
        }
        if (threadIdx.x == 0)
        {
            shared.bad = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += Threads)
        {
            const int s = sequence(i);
            if (s < 0 || s >= cache.sequences || (atomicOr(&shared.seen[s / 32], 1u << s % 32) >> s % 32 & 1) ||
                !check_entry(i, s))
            {
                shared.bad = 1;
            }
        }
        __syncthreads();
        return !shared.bad;
    }
    // Exclusive sums of each entry's need (below 2^21) into `before`; returns the total.
    template <class Need> __device__ long long sum_needs(Need need)
    {
        long long total = 0;
        for (int base = 0, round = 0; base < count; base += Threads, round ^= 1)
        {
            const int i = base + int(threadIdx.x), mine = i < count ? need(i) : 0;
            int inclusive = mine;
#pragma unroll
            for (int step = 1; step < 64; step *= 2)
            {
                const int below = __shfl_up(inclusive, step);
                inclusive += lane >= step ? below : 0;
            }
            if (lane == 63)
            {
                shared.sums[round][warp] = inclusive;
            }
            __syncthreads();
            int front = 0, all = 0;
#pragma unroll
            for (int w = 0; w < waves; ++w)
            {
                front += w < warp ? shared.sums[round][w] : 0;
                all += shared.sums[round][w];
            }
            if (i < count)
            {
                // Past 2^31 the call fails: there are fewer pages.
                shared.before[i] = int(total + front + inclusive - mine);
            }
            total += all;
        }
        if (threadIdx.x == 0)
        {
            shared.before[count] = int(total);
        }
        __syncthreads();
        return total;
    }
    // The last entry with before <= rank.
    __device__ __forceinline__ int entry(int rank) const
    {
        int low = 0, high = count;
        while (high - low > 1)
        {
            const int middle = (low + high) / 2;
            (shared.before[middle] <= rank ? low : high) = middle;
        }
        return low;
    }
    // Hands the `total` lowest free pages to take(entry, index within the entry's need, page), in
    // order, and counts them once; false, with what was handed out given to undo(), if there are
    // too few. The scan ends as soon as enough are found.
    template <class Take, class Undo> __device__ bool take_pages(long long total, Take take, Undo undo)
    {
        if (total > cache.pages)
        {
            return false;
        }
        int found = 0;
        int counts[scanned];
#pragma unroll
        for (int j = 0; j < scanned; ++j)
        {
            counts[j] = first_counts[j];
        }
        for (long long base = 0; base < cache.pages && found < total;)
        {
            // Free pages of the lanes below, and of the thread's in front.
            int rank = 0, mine = 0;
#pragma unroll
            for (int j = 0; j < scanned; ++j)
            {
                rank += lanes_below(__ballot(counts[j] == 0));
                mine += __popcll(__ballot(counts[j] == 0));
            }
            const int round = base / (Threads * scanned) % 2;
            if (lane == 0)
            {
                shared.sums[round][warp] = mine;
            }
            __syncthreads();
            int all = 0;
            rank += found;
#pragma unroll
            for (int w = 0; w < waves; ++w)
            {
                rank += w < warp ? shared.sums[round][w] : 0;
                all += shared.sums[round][w];
            }
#pragma unroll
            for (int j = 0; j < scanned; ++j)
            {
                if (counts[j] == 0)
                {
                    if (rank < total)
                    {
                        const int i = entry(rank), page = int(base + threadIdx.x * scanned + j);
                        take(i, rank - shared.before[i], page);
                        cache.references[page] = 1;
                    }
                    ++rank;
                }
            }
            found += all;
            base += Threads * scanned;
            if (base < cache.pages && found < total)
            {
                read_counts(base, counts);
            }
        }
        if (found >= total)
        {
            return true;
        }
        __syncthreads();
        for (int rank = threadIdx.x; rank < found; rank += Threads)
        {
            const int i = entry(rank);
            cache.references[undo(i, rank - shared.before[i])] = 0;
        }
        return false;
    }
};

template <int Threads>
__global__ __launch_bounds__(Threads) void reserve_kernel(PagedCache cache, const int* __restrict__ sequences,
                                                          const int* __restrict__ rows, int count, int* status)
{
    extern __shared__ char memory[];
    Taking<Threads> taking(*reinterpret_cast<TakingShared*>(memory), cache, count);
    const auto sequence = [&](int i) { return sequences ? sequences[i] : i; };
    // Pages that positions up to length + rows take.
    const auto pages = [&](int i, int s) -> long long
    { return ((long long)cache.lengths[s] + rows[i] + cache.page_rows - 1) / cache.page_rows; };
    const bool good = taking.check(sequence,
                                   [&](int i, int s)
                                   {
                                       return rows[i] >= 0 && cache.lengths[s] >= 0 && cache.held[s] >= 0 &&
                                              std::size_t(cache.held[s]) <= cache.table_stride &&
                                              std::size_t(pages(i, s)) <= cache.table_stride;
                                   });
    if (!good)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_invalid);
        }
        return;
    }
    const long long total = taking.sum_needs(
        [&](int i)
        {
            const int s = sequence(i);
            const int more = int(pages(i, s)) - cache.held[s];
            return more > 0 ? more : 0;
        });
    const auto slot = [&](int i, int j) -> int&
    {
        const int s = sequence(i);
        return cache.table[s * cache.table_stride + cache.held[s] + j];
    };
    const bool enough = taking.take_pages(
        total, [&](int i, int j, int page) { slot(i, j) = page; },
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
    for (int i = threadIdx.x; i < count; i += Threads)
    {
        cache.held[sequence(i)] += taking.shared.before[i + 1] - taking.shared.before[i];
    }
}

// While a fork runs, a target's `held` says so: what it will hold, `forking`, and above it how
// many workgroups of fork_copy_kernel are done with the target; the last one leaves the
// number alone. A refused call sets no such mark, so that the second kernel does nothing.
constexpr int forking = 1 << 30, arrival = 1 << 21;
static_assert(max_table_pages < arrival && 2 * max_layers + 1 < forking / arrival);

// Checks the list, takes a page for each source's last partial one and makes the targets
// hold their pages; what is shared and copied follows in fork_copy_kernel.
template <int Threads>
__global__ __launch_bounds__(Threads) void fork_kernel(PagedCache cache, const int* __restrict__ sources,
                                                       const int* __restrict__ targets, int count, int* status)
{
    extern __shared__ char memory[];
    auto& shared = *reinterpret_cast<TakingShared*>(memory);
    Taking<Threads> taking(shared, cache, count);
    // The words that sources are looked for in, too.
    for (int i = threadIdx.x; i < count; i += Threads)
    {
        const int s = sources[i];
        if (s >= 0 && s < cache.sequences)
        {
            shared.seen[s / 32] = 0;
        }
    }
    bool good = taking.check([&](int i) { return targets[i]; }, [&](int, int t) { return cache.held[t] == 0; });
    for (int i = threadIdx.x; i < count; i += Threads)
    {
        const int s = sources[i];
        if (s < 0 || s >= cache.sequences || (shared.seen[s / 32] >> s % 32 & 1) || cache.lengths[s] < 0 ||
            cache.held[s] < 0 || std::size_t(cache.held[s]) > cache.table_stride ||
            (cache.lengths[s] + (long long)cache.page_rows - 1) / cache.page_rows > cache.held[s])
        {
            shared.bad = 1;
        }
    }
    __syncthreads();
    good = good && !shared.bad;
    if (!good)
    {
        if (threadIdx.x == 0)
        {
            report(status, status_invalid);
        }
        return;
    }
    const long long total = taking.sum_needs([&](int i) { return cache.lengths[sources[i]] % cache.page_rows != 0; });
    const auto slot = [&](int i) -> int&
    { return cache.table[targets[i] * cache.table_stride + cache.lengths[sources[i]] / cache.page_rows]; };
    const bool enough = taking.take_pages(
        total, [&](int i, int, int page) { slot(i) = page; },
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
    for (int i = threadIdx.x; i < count; i += Threads)
    {
        const int length = cache.lengths[sources[i]];
        cache.lengths[targets[i]] = length;
        cache.held[targets[i]] = forking | int((length + (long long)cache.page_rows - 1) / cache.page_rows);
    }
}

constexpr int copying_threads = 256;

// Shares the full pages. A last one that is out of range has nothing to copy: the page that was taken for
// the copy, and has another sequence's old rows, is given back.
__device__ __forceinline__ void share_pages(const PagedCache& cache, const int* from, int* to, int full, int rest,
                                            int* status)
{
    if (threadIdx.x == 0 && rest && (from[full] < 0 || from[full] >= cache.pages))
    {
        const int fresh = to[full];
        if (fresh >= 0 && fresh < cache.pages)
        {
            cache.references[fresh] = 0;
        }
        to[full] = -1;
        report(status, status_invalid);
    }
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

typedef unsigned Vector __attribute__((ext_vector_type(4)));

// Copies the rows of the last page, of one layer's keys or values. Stores go past the caches, which
// keep the source for its other targets: 64 targets of 8 sources 28 us, with plain stores 49 (and with
// loads past them too, 50).
__device__ __forceinline__ void copy_rows(const PagedCache& cache, int part, int old, int fresh, int rest)
{
    if (old < 0 || old >= cache.pages || fresh < 0 || fresh >= cache.pages)
    {
        return; // reported by share_pages
    }
    uint16_t* const memory = (part % 2 ? cache.values : cache.keys) + part / 2 * cache.layer_stride;
    const int vectors = cache.heads * cache.head_width / 8;
    for (int i = threadIdx.x; i < rest * vectors; i += copying_threads)
    {
        const std::size_t at = i / vectors * cache.row_stride + i % vectors * 8;
        const auto value = *reinterpret_cast<const Vector*>(memory + old * cache.page_stride + at);
        __builtin_nontemporal_store(value, reinterpret_cast<Vector*>(memory + fresh * cache.page_stride + at));
    }
}

// blockIdx: the entry of the list, then (layer, keys or values), past the last of them the
// sharing. 64 targets of pages of 64 rows, 12 layers of 8 x 128: 105 MB are written in 28 us, 3.8 TB/s.
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
    // A refused call leaves `held` as it was, and that may look like a mark: what it has to agree with
    // where it is one keeps the table's bounds.
    const int length = cache.lengths[target];
    const long long pages = (length + (long long)cache.page_rows - 1) / cache.page_rows;
    if (length < 0 || length != cache.lengths[source] || pages != (mark & (arrival - 1)) ||
        std::size_t(pages) > cache.table_stride || pages > cache.held[source])
    {
        return;
    }
    const int full = length / cache.page_rows, rest = length % cache.page_rows;
    const int* const from = cache.table + source * cache.table_stride;
    int* const to = cache.table + target * cache.table_stride;
    if (int(blockIdx.y) == 2 * cache.layers)
    {
        share_pages(cache, from, to, full, rest, status);
    }
    else if (rest)
    {
        copy_rows(cache, blockIdx.y, from[full], to[full], rest);
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
        cache.lengths[s] = 0;
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

// blockIdx: a row's place in its sequence, the sequence, the layer; or (`Find`) a row of all, 0, the layer. 64
// sequences of up to 32 rows, 12 layers of 8 x 128: 177 MB read and written in 36 us, the rate of a large copy.
template <bool Find>
__global__ __launch_bounds__(copying_threads) void write_kernel(PagedCache cache, int layer, NewRows fresh, int max_rows,
                                                                const int* __restrict__ starts, int* status)
{
    int row = blockIdx.x, s = blockIdx.y, first;
    if constexpr (Find)
    {
        s = sequence_of(starts, cache.sequences, row);
    }
    const int rows = rows_of(starts, s, fresh.rows, first);
    if constexpr (Find)
    {
        row -= first;
        if (row < 0 || row >= max_rows)
        {
            return;
        }
    }
    if (row >= rows)
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

constexpr int moved = 4;       // rows a thread moves at a time
constexpr int placed = 256;    // rows whose places are looked up at a time

// blockIdx: vectors of a row, the sequence, (layer, keys or values). Threads stand side by side for
// up to 256 vectors of a row, and rows apart for the rest; rows are moved in ascending order, as
// many at a time as there are threads for, all read before any is written: row k comes from node
// path[k] >= k, so that no row is read that was written.
__global__ __launch_bounds__(copying_threads) void keep_kernel(PagedCache cache, const int* __restrict__ starts,
                                                               const int* __restrict__ path, std::size_t path_stride,
                                                               const int* __restrict__ accepted, int* lengths,
                                                               int* status)
{
    __shared__ int bad;
    __shared__ long long from[placed], to[placed]; // offsets of rows, -1: not moved
    const int s = blockIdx.y;
    const int length = cache.lengths[s], count = accepted[s];
    const int nodes = starts[s + 1] - starts[s];
    path += s * path_stride;
    const int kept = kept_rows(path, count, nodes, path_stride, &bad);
    const bool reporter = threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.z == 0;
    if (lengths && reporter)
    {
        lengths[s] = length + (kept > 0 && length >= 0 ? kept : 0);
    }
    if (kept < 0 || length < 0)
    {
        if (reporter)
        {
            report(status, status_invalid);
        }
        return;
    }
    const int vectors = cache.heads * cache.head_width / 8, first = int(blockIdx.x) * copying_threads;
    const int wide = min(vectors - first, copying_threads), apart = copying_threads / wide;
    const int vector = first + int(threadIdx.x) % wide, row = int(threadIdx.x) / wide;
    uint16_t* const memory =
        (blockIdx.z % 2 ? cache.values : cache.keys) + blockIdx.z / 2 * cache.layer_stride + 8 * std::size_t(vector);
    const auto place = [&](int node) -> long long
    {
        const long long position = (long long)length + node;
        const int page = writable_page(cache, s, position);
        return page < 0 ? -1
                        : (long long)(page * cache.page_stride + position % cache.page_rows * cache.row_stride);
    };
    for (int base = 0; base < kept; base += placed)
    {
        const int rows = min(kept - base, placed);
        __syncthreads();
        for (int k = threadIdx.x; k < rows; k += copying_threads)
        {
            const int node = path[base + k];
            // Rows that are in place already stay.
            const long long source = node == base + k ? -1 : place(node), target = node == base + k ? -1 : place(base + k);
            from[k] = source;
            to[k] = source < 0 ? -1 : target;
            if (node != base + k && (source < 0 || target < 0))
            {
                report(status, status_invalid);
            }
        }
        __syncthreads();
        for (int k = 0; k < rows; k += moved * apart)
        {
            uint4 value[moved];
#pragma unroll
            for (int j = 0; j < moved; ++j)
            {
                const int mine = k + j * apart + row;
                if (row < apart && mine < rows && to[mine] >= 0)
                {
                    value[j] = *reinterpret_cast<const uint4*>(memory + from[mine]);
                }
            }
            __syncthreads(); // one thread's row is another one's source
#pragma unroll
            for (int j = 0; j < moved; ++j)
            {
                const int mine = k + j * apart + row;
                if (row < apart && mine < rows && to[mine] >= 0)
                {
                    *reinterpret_cast<uint4*>(memory + to[mine]) = value[j];
                }
            }
            __syncthreads();
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
    if (threadIdx.x == 0 && kept > 0 && lengths[s] >= 0)
    {
        lengths[s] += kept;
    }
}

// A workgroup a sequence, a thread a node: the words from the node's own down, along its line, one read of
// LDS after another: 10 us for three trees of 1,024 nodes ten levels deep, 168 for chains of as many.
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
    // Four waves for lists that fit them: their barriers are short (3 sequences: 6.2 us, with sixteen
    // waves 8.0).
    (count <= 256 ? reserve_kernel<256><<<1, 256, sizeof(TakingShared), stream>>>(cache, sequences, rows, int(count), status)
                  : reserve_kernel<most_threads><<<1, most_threads, sizeof(TakingShared), stream>>>(
                        cache, sequences, rows, int(count), status));
    check_hip(hipGetLastError(), "pages reserve launch");
}

void pages_fork(const PagedCache& cache, const int* sources, const int* targets, std::size_t count, int* status,
                hipStream_t stream)
{
    if (!count)
    {
        return;
    }
    (count <= 256 ? fork_kernel<256><<<1, 256, sizeof(TakingShared), stream>>>(cache, sources, targets, int(count), status)
                  : fork_kernel<most_threads><<<1, most_threads, sizeof(TakingShared), stream>>>(cache, sources, targets,
                                                                                                 int(count), status));
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
    // A workgroup for every row that a sequence may have where most have one: a batch of single rows and one of
    // 8,192, 256 sequences, 12 layers of 8 x 128, takes 208 us with a look for the sequence, 5.4 ms without; 64
    // of 8 rows announced as 16 20 and 25; but 64 of 32 rows 44 and 41, 2,000 of one 53 and 45.
    const bool find = std::size_t(max_rows) * cache.sequences >= 2 * std::size_t(fresh.rows);
    const dim3 grid(unsigned(find ? fresh.rows : max_rows), unsigned(find ? 1 : cache.sequences), unsigned(layers));
    (find ? write_kernel<true><<<grid, copying_threads, 0, stream>>>(cache, layer, fresh, max_rows, starts, status)
          : write_kernel<false><<<grid, copying_threads, 0, stream>>>(cache, layer, fresh, max_rows, starts, status));
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

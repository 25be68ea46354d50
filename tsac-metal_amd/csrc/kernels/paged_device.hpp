// What kernels over a paged cache share: the rows of a batch, and the pages they may write.
#pragma once

#include "paged.hpp"

namespace tsac_hip
{
__device__ __forceinline__ void report(int* status, int what)
{
    if (status)
    {
        *status = what;
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

// The last sequence that starts at or in front of a row, by a wave: 64 starts at a time.
__device__ __forceinline__ int sequence_of(const int* starts, int sequences, int row)
{
    const int lane = threadIdx.x % 64;
    int low = 0, high = sequences;
    while (high - low > 1)
    {
        const int step = (high - low + 63) / 64, i = low + lane * step;
        const uint64_t bits = __ballot(i < high && starts[i] <= row);
        low += bits ? (63 - __builtin_clzll(bits)) * step : 0;
        high = min(low + step, high);
    }
    return low;
}
} // namespace tsac_hip

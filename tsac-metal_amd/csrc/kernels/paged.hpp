// Launchers of drafted decoding: a cache of keys and values in pages, attention of
// drafted rows over it, and the verification of drafted tokens.
#pragma once

#include "kernels.hpp"

namespace tsac_hip
{
// What kernels write to a call's status word (include/tsac_hip.h); plain stores.
constexpr int status_invalid = 1;   // a number, length or page out of range
constexpr int status_exhausted = 2; // too few free pages

// A cache's device memory, as the kernels take it. keys and values: 16-bit elements
// [layers][pages][page_rows][heads][head_width] at the given strides (in elements).
struct PagedCache
{
    uint16_t* keys = nullptr;
    uint16_t* values = nullptr;
    std::size_t layer_stride = 0, page_stride = 0, row_stride = 0;
    int layers = 0, pages = 0, page_rows = 0, heads = 0, head_width = 0;
    bool half = false; // IEEE half precision, otherwise BF16
    int* table = nullptr; // [sequences][table_stride]
    std::size_t table_stride = 0;
    int* held = nullptr;
    int* lengths = nullptr;
    int* references = nullptr;
    int sequences = 0;
};

constexpr int max_listed_sequences = 8192; // of one reserve or fork
constexpr int max_sequences = 65535;
constexpr int max_layers = 255;
constexpr int max_table_pages = 1 << 20; // of one sequence
constexpr int max_draft_nodes = 1024; // of one sequence's tree

void pages_reserve(const PagedCache& cache, const int* sequences, const int* rows, std::size_t count, int* status,
                   hipStream_t stream);
void pages_fork(const PagedCache& cache, const int* sources, const int* targets, std::size_t count, int* status,
                hipStream_t stream);
void pages_free(const PagedCache& cache, const int* sequences, std::size_t count, int* status, hipStream_t stream);

// Rows of keys and values [layers][rows][heads][head_width] at their strides into layers
// layer .. layer + layers - 1.
struct NewRows
{
    const uint16_t* keys = nullptr;
    const uint16_t* values = nullptr;
    std::size_t layer_stride = 0, row_stride = 0;
    int rows = 0;
};
void pages_write(const PagedCache& cache, int layer, int layers, const NewRows& fresh, const int* starts, int max_rows,
                 int* status, hipStream_t stream);
void pages_keep(const PagedCache& cache, const int* starts, const int* path, std::size_t path_stride,
                const int* accepted, int* lengths, int* status, hipStream_t stream);

void tree_mask(const int* parents, int rows, const int* starts, int sequences, int max_nodes, uint64_t* mask,
               std::size_t words, hipStream_t stream);

struct PagedRows
{
    const uint16_t* query = nullptr; // [rows][heads][head_width]
    std::size_t query_stride = 0;    // elements from row to row
    uint16_t* out = nullptr;
    std::size_t out_stride = 0;
    int rows = 0, heads = 0;
    const int* starts = nullptr;
    int max_rows = 0;               // of one sequence
    std::size_t max_length = 0;     // cached and new rows of one sequence; shapes the launch only
    const uint64_t* mask = nullptr; // [rows][words]
    std::size_t words = 0;
    float scale = 0;
};
std::size_t attention_paged_workspace(const PagedCache& cache, const PagedRows& rows);
void attention_paged(const PagedCache& cache, int layer, const PagedRows& rows, void* workspace, std::size_t bytes,
                     hipStream_t stream);

struct Drafts
{
    const void* target = nullptr; // [rows][alphabet] probabilities
    std::size_t target_stride = 0;
    const void* draft = nullptr; // null: each drafted token was certain
    std::size_t draft_stride = 0;
    int type = 0; // 0 BF16, 1 half, 2 float
    int alphabet = 0, rows = 0;
    const int* tokens = nullptr;
    const int* parents = nullptr;
    const int* starts = nullptr;
    int sequences = 0, max_nodes = 0;
    const float* uniforms = nullptr;
    const float* draws = nullptr;
    int* path = nullptr; // [sequences][max_nodes]
    int* accepted = nullptr;
    int* next = nullptr;
};
std::size_t verify_drafts_workspace(const Drafts& drafts);
void verify_drafts(const Drafts& drafts, void* workspace, std::size_t bytes, hipStream_t stream);
} // namespace tsac_hip

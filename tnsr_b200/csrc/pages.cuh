// Operators on the pages of caches and on states of sequences (pages.cu).
#pragma once

#include "paged.cuh"

namespace tb {

struct PageBook {
    uint32_t *table, *lengths, *holders;
    int* d_status;
    uint32_t sequences, table_ld, page_rows, pool_pages;
    void* workspace;
    uint32_t* refused;              // what became of the last reserve, or null
};
struct PagePools {
    void* const* tensors;
    const uint64_t* page_bytes;
    uint32_t count;
};

uint64_t pages_workspace_bytes(uint32_t sequences, uint32_t pool_pages);
int launch_pages_fork(const PageBook& b, const uint32_t* parents, cudaStream_t stream);
int launch_pages_reserve(const PageBook& b, const PagePools& pools, const uint32_t* rows, uint32_t rows_each, cudaStream_t stream);
int launch_pages_release(const PageBook& b, const uint8_t* gone, cudaStream_t stream);
int launch_pages_compact(const PageBook& b, const PagePools& pools, uint32_t* live_pages, cudaStream_t stream);
int launch_pages_copy(const PagePools& pools, const uint32_t* from, const uint32_t* to, uint32_t pairs, uint32_t pool_pages, int* d_status,
                      cudaStream_t stream);
int launch_reorder_states(void* const* tensors, const uint64_t* row_bytes, const uint64_t* pitches, uint32_t count, const uint32_t* parents,
                          uint32_t groups, uint32_t beams, int* d_status, cudaStream_t stream);

struct PagedAppend {
    const void *k, *v;
    void *k_pool, *v_pool;
    const uint32_t *table, *lengths, *row_starts;
    int* d_status;
    uint64_t k_page, k_row, k_head, v_page, v_row, v_head;
    uint32_t sequences, chunk, rows, k_ld, v_ld, kv_heads, dim, vdim, table_ld, page_rows, pool_pages;
    const uint32_t* refused;
};
int launch_paged_append(const PagedAppend& a, int dtype, cudaStream_t stream);

constexpr uint32_t PAGES_MAX_SEQUENCES = 12288;   // what fork stages a column of
constexpr uint32_t REORDER_MAX_BEAMS = 32;

}  // namespace tb

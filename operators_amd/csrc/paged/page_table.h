// What PageTableUpdate and PageTableCompact check alike, and the device pieces
// they share: pages in words of 64 (one ballot), words in chunks of 16 (one
// workgroup's turn), counts of chunks added up by whoever needs them.
#ifndef INFINIOP_AMD_PAGE_TABLE_H
#define INFINIOP_AMD_PAGE_TABLE_H

#include "paged_cache.h"

constexpr uint32_t kChunkWords = 16, kChunkPages = 64 * kChunkWords;
constexpr uint64_t kMostPages = 1ull << 24;// every workgroup adds up the counts of all chunks
constexpr uint64_t kMostTableRows = 8192;  // the growth of all rows lies in LDS

namespace amd {

// A table before and after, and the counts of pages before and after.
struct TableSizes {
    PagedRows old_rows, new_rows;
    uint32_t pages, page;
};

inline infiniopStatus_t page_tables(infiniopTensorDescriptor_t new_table, infiniopTensorDescriptor_t new_refcount, infiniopTensorDescriptor_t table,
                                    infiniopTensorDescriptor_t refcount, uint64_t page_size, TableSizes *out) {
    if (page_size == 0 || page_size >= (1ull << 20)) return STATUS_BAD_PARAM;
    infiniopStatus_t st = paged_table(table, page_size, &out->old_rows);
    if (st == STATUS_SUCCESS) st = paged_table(new_table, page_size, &out->new_rows);
    if (st != STATUS_SUCCESS) return st;
    if (out->new_rows.rows != out->old_rows.rows || out->new_rows.cols != out->old_rows.cols) return STATUS_BAD_TENSOR_SHAPE;
    if (refcount->ndim != 1) return STATUS_BAD_TENSOR_SHAPE;
    const uint64_t pages = refcount->shape[0];
    if (pages == 0 || pages >= kMostPages || out->old_rows.rows > kMostTableRows) return STATUS_BAD_TENSOR_SHAPE;
    if (static_cast<uint64_t>(out->old_rows.rows) * out->old_rows.cols >= (1ull << 31)) return STATUS_BAD_TENSOR_SHAPE;
    out->pages = static_cast<uint32_t>(pages);
    out->page = static_cast<uint32_t>(page_size);
    st = paged_vector(refcount, pages);
    return st != STATUS_SUCCESS ? st : paged_vector(new_refcount, pages);
}

inline uint64_t chunks_of(uint32_t pages) { return ceil_div(pages, kChunkPages); }

}// namespace amd

#endif

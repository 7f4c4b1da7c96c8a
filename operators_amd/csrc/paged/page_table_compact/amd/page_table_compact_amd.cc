// Create-time validation for PageTableCompact on the amd-gpu device.
#include "page_table_compact_amd.h"
#include <new>

infiniopStatus_t amdCreatePageTableCompactDescriptor(AmdHandle_t handle, PageTableCompactAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t new_table,
                                                     infiniopTensorDescriptor_t new_refcount, infiniopTensorDescriptor_t pairs,
                                                     infiniopTensorDescriptor_t result, infiniopTensorDescriptor_t table,
                                                     infiniopTensorDescriptor_t lengths, infiniopTensorDescriptor_t refcount, uint64_t page_size) {
    if (desc_ptr == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    amd::TableSizes sizes;
    infiniopStatus_t st = amd::page_tables(new_table, new_refcount, table, refcount, page_size, &sizes);
    if (st == STATUS_SUCCESS) st = amd::paged_vector(lengths, sizes.old_rows.rows);
    if (st == STATUS_SUCCESS) st = amd::paged_pairs(pairs);
    if (st == STATUS_SUCCESS) st = amd::paged_vector(result, 2);
    if (st != STATUS_SUCCESS) {
        return st;
    }
    if (pairs->shape[0] < sizes.pages / 2) {
        return STATUS_BAD_TENSOR_SHAPE;
    }
    // the bits of the used pages, their count by chunk, the used pages before each word, {used, below}
    const uint64_t chunks = amd::chunks_of(sizes.pages);
    const uint64_t bytes = chunks * kChunkWords * 12 + chunks * 4;
    auto *desc = new (std::nothrow) PageTableCompactAmdDescriptor{DevAmdGpu, handle->device_id, sizes, static_cast<uint32_t>(pairs->shape[0]), bytes};
    if (desc == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    *desc_ptr = desc;
    return STATUS_SUCCESS;
}

infiniopStatus_t amdDestroyPageTableCompactDescriptor(PageTableCompactAmdDescriptor_t desc) {
    delete desc;
    return STATUS_SUCCESS;
}

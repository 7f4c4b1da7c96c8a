// Create-time validation for PageTableUpdate on the amd-gpu device.
#include "page_table_update_amd.h"
#include <new>

infiniopStatus_t amdCreatePageTableUpdateDescriptor(AmdHandle_t handle, PageTableUpdateAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t new_table,
                                                    infiniopTensorDescriptor_t new_lengths, infiniopTensorDescriptor_t new_refcount,
                                                    infiniopTensorDescriptor_t pairs, infiniopTensorDescriptor_t result,
                                                    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t lengths,
                                                    infiniopTensorDescriptor_t refcount, infiniopTensorDescriptor_t source,
                                                    infiniopTensorDescriptor_t grow, uint64_t page_size) {
    if (desc_ptr == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    amd::TableSizes sizes;
    infiniopStatus_t st = amd::page_tables(new_table, new_refcount, table, refcount, page_size, &sizes);
    const uint64_t rows = sizes.old_rows.rows;
    for (infiniopTensorDescriptor_t t : {lengths, new_lengths, source, grow}) {
        if (st == STATUS_SUCCESS) st = amd::paged_vector(t, rows);
    }
    if (st == STATUS_SUCCESS) st = amd::paged_pairs(pairs);
    if (st == STATUS_SUCCESS) st = amd::paged_vector(result, 2);
    if (st != STATUS_SUCCESS) {
        return st;
    }
    if (pairs->shape[0] != rows) {
        return STATUS_BAD_TENSOR_SHAPE;
    }
    // the bits of the free pages and their count by chunk; a row's length before it grows and its growth; the rows that change
    const uint64_t chunks = amd::chunks_of(sizes.pages);
    const uint64_t bytes = chunks * kChunkWords * 8 + chunks * 4 + rows * 8 + rows * sizes.old_rows.cols * 4;
    auto *desc = new (std::nothrow) PageTableUpdateAmdDescriptor{DevAmdGpu, handle->device_id, sizes, bytes};
    if (desc == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    *desc_ptr = desc;
    return STATUS_SUCCESS;
}

infiniopStatus_t amdDestroyPageTableUpdateDescriptor(PageTableUpdateAmdDescriptor_t desc) {
    delete desc;
    return STATUS_SUCCESS;
}

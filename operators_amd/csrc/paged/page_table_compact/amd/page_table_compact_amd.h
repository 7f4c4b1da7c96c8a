// amd-gpu back end of PageTableCompact.
#ifndef INFINIOP_AMD_PAGE_TABLE_COMPACT_H
#define INFINIOP_AMD_PAGE_TABLE_COMPACT_H

#include "../../page_table.h"

struct PageTableCompactAmdDescriptor {
    Device device;
    int device_id;
    amd::TableSizes sizes;
    uint32_t pairs;
    uint64_t workspace;
};
typedef PageTableCompactAmdDescriptor *PageTableCompactAmdDescriptor_t;

infiniopStatus_t amdCreatePageTableCompactDescriptor(AmdHandle_t handle, PageTableCompactAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t new_table,
                                                     infiniopTensorDescriptor_t new_refcount, infiniopTensorDescriptor_t pairs,
                                                     infiniopTensorDescriptor_t result, infiniopTensorDescriptor_t table,
                                                     infiniopTensorDescriptor_t lengths, infiniopTensorDescriptor_t refcount, uint64_t page_size);
infiniopStatus_t amdPageTableCompact(PageTableCompactAmdDescriptor_t desc, void *workspace, uint64_t workspace_size, void *new_table, void *new_refcount,
                                     void *pairs, void *result, void const *table, void const *lengths, void const *refcount, void *stream);
infiniopStatus_t amdDestroyPageTableCompactDescriptor(PageTableCompactAmdDescriptor_t desc);

#endif

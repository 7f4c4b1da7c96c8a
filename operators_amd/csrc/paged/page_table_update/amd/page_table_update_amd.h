// amd-gpu back end of PageTableUpdate.
#ifndef INFINIOP_AMD_PAGE_TABLE_UPDATE_H
#define INFINIOP_AMD_PAGE_TABLE_UPDATE_H

#include "../../page_table.h"

struct PageTableUpdateAmdDescriptor {
    Device device;
    int device_id;
    amd::TableSizes sizes;
    uint64_t workspace;
};
typedef PageTableUpdateAmdDescriptor *PageTableUpdateAmdDescriptor_t;

infiniopStatus_t amdCreatePageTableUpdateDescriptor(AmdHandle_t handle, PageTableUpdateAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t new_table,
                                                    infiniopTensorDescriptor_t new_lengths, infiniopTensorDescriptor_t new_refcount,
                                                    infiniopTensorDescriptor_t pairs, infiniopTensorDescriptor_t result,
                                                    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t lengths,
                                                    infiniopTensorDescriptor_t refcount, infiniopTensorDescriptor_t source,
                                                    infiniopTensorDescriptor_t grow, uint64_t page_size);
infiniopStatus_t amdPageTableUpdate(PageTableUpdateAmdDescriptor_t desc, void *workspace, uint64_t workspace_size, void *new_table, void *new_lengths,
                                    void *new_refcount, void *pairs, void *result, void const *table, void const *lengths, void const *refcount,
                                    void const *source, void const *grow, void *stream);
infiniopStatus_t amdDestroyPageTableUpdateDescriptor(PageTableUpdateAmdDescriptor_t desc);

#endif

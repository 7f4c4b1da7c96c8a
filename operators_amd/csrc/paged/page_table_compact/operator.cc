// Public entry points of PageTableCompact: argument checks that need no device, and the way to the device's back end.
#include "amd/page_table_compact_amd.h"

INFINIOP_C infiniopStatus_t infiniopCreatePageTableCompactDescriptor(
    infiniopHandle_t handle, infiniopPageTableCompactDescriptor_t *desc_ptr, infiniopTensorDescriptor_t new_table,
    infiniopTensorDescriptor_t new_refcount, infiniopTensorDescriptor_t pairs, infiniopTensorDescriptor_t result, infiniopTensorDescriptor_t table,
    infiniopTensorDescriptor_t lengths, infiniopTensorDescriptor_t refcount,
    uint64_t page_size) {
    if (handle == nullptr) {
        return STATUS_BAD_PARAM;
    }
    for (infiniopTensorDescriptor_t t : {new_table, new_refcount, pairs, result, table, lengths, refcount}) {
        if (t == nullptr) return STATUS_BAD_PARAM;
    }
    switch (handle->device) {
        case DevAmdGpu:
            return amdCreatePageTableCompactDescriptor(reinterpret_cast<AmdHandle_t>(handle),
                                                      reinterpret_cast<PageTableCompactAmdDescriptor_t *>(desc_ptr), new_table, new_refcount,
                                                      pairs, result, table, lengths, refcount, page_size);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopGetPageTableCompactWorkspaceSize(infiniopPageTableCompactDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || size == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            *size = reinterpret_cast<PageTableCompactAmdDescriptor_t>(desc)->workspace;
            return STATUS_SUCCESS;
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopPageTableCompact(infiniopPageTableCompactDescriptor_t desc, void *workspace, uint64_t workspace_size, void *new_table,
                                                    void *new_refcount, void *pairs, void *result, void const *table,
                                                    void const *lengths, void const *refcount, void *stream) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdPageTableCompact(reinterpret_cast<PageTableCompactAmdDescriptor_t>(desc), workspace, workspace_size, new_table,
                                      new_refcount, pairs, result, table, lengths, refcount, stream);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopDestroyPageTableCompactDescriptor(infiniopPageTableCompactDescriptor_t desc) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdDestroyPageTableCompactDescriptor(reinterpret_cast<PageTableCompactAmdDescriptor_t>(desc));
        default:
            return STATUS_BAD_DEVICE;
    }
}

// Public entry points of PageTableUpdate: argument checks that need no device, and the way to the device's back end.
#include "amd/page_table_update_amd.h"

INFINIOP_C infiniopStatus_t infiniopCreatePageTableUpdateDescriptor(
    infiniopHandle_t handle, infiniopPageTableUpdateDescriptor_t *desc_ptr, infiniopTensorDescriptor_t new_table, infiniopTensorDescriptor_t new_lengths,
    infiniopTensorDescriptor_t new_refcount, infiniopTensorDescriptor_t pairs, infiniopTensorDescriptor_t result, infiniopTensorDescriptor_t table,
    infiniopTensorDescriptor_t lengths, infiniopTensorDescriptor_t refcount, infiniopTensorDescriptor_t source, infiniopTensorDescriptor_t grow,
    uint64_t page_size) {
    if (handle == nullptr) {
        return STATUS_BAD_PARAM;
    }
    for (infiniopTensorDescriptor_t t : {new_table, new_lengths, new_refcount, pairs, result, table, lengths, refcount, source, grow}) {
        if (t == nullptr) return STATUS_BAD_PARAM;
    }
    switch (handle->device) {
        case DevAmdGpu:
            return amdCreatePageTableUpdateDescriptor(reinterpret_cast<AmdHandle_t>(handle),
                                                      reinterpret_cast<PageTableUpdateAmdDescriptor_t *>(desc_ptr), new_table, new_lengths, new_refcount,
                                                      pairs, result, table, lengths, refcount, source, grow, page_size);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopGetPageTableUpdateWorkspaceSize(infiniopPageTableUpdateDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || size == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            *size = reinterpret_cast<PageTableUpdateAmdDescriptor_t>(desc)->workspace;
            return STATUS_SUCCESS;
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopPageTableUpdate(infiniopPageTableUpdateDescriptor_t desc, void *workspace, uint64_t workspace_size, void *new_table,
                                                    void *new_lengths, void *new_refcount, void *pairs, void *result, void const *table,
                                                    void const *lengths, void const *refcount, void const *source, void const *grow, void *stream) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdPageTableUpdate(reinterpret_cast<PageTableUpdateAmdDescriptor_t>(desc), workspace, workspace_size, new_table, new_lengths,
                                      new_refcount, pairs, result, table, lengths, refcount, source, grow, stream);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopDestroyPageTableUpdateDescriptor(infiniopPageTableUpdateDescriptor_t desc) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdDestroyPageTableUpdateDescriptor(reinterpret_cast<PageTableUpdateAmdDescriptor_t>(desc));
        default:
            return STATUS_BAD_DEVICE;
    }
}

// Public entry points of PagedAttention: argument checks that need no device, and the way to the device's back end.
#include "amd/paged_attention_amd.h"

INFINIOP_C infiniopStatus_t infiniopCreatePagedAttentionDescriptor(
    infiniopHandle_t handle, infiniopPagedAttentionDescriptor_t *desc_ptr, infiniopTensorDescriptor_t out, infiniopTensorDescriptor_t q,
    infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache, infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale,
    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets, infiniopTensorDescriptor_t lengths, uint64_t max_tokens, float scale) {
    if (handle == nullptr) {
        return STATUS_BAD_PARAM;
    }
    for (infiniopTensorDescriptor_t t : {out, q, k_cache, v_cache, k_scale, v_scale, table, offsets, lengths}) {
        if (t == nullptr) return STATUS_BAD_PARAM;
    }
    switch (handle->device) {
        case DevAmdGpu:
            return amdCreatePagedAttentionDescriptor(reinterpret_cast<AmdHandle_t>(handle), reinterpret_cast<PagedAttentionAmdDescriptor_t *>(desc_ptr),
                                                     out, q, k_cache, v_cache, k_scale, v_scale, table, offsets, lengths, max_tokens, scale);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopGetPagedAttentionWorkspaceSize(infiniopPagedAttentionDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || size == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            *size = reinterpret_cast<PagedAttentionAmdDescriptor_t>(desc)->workspace;
            return STATUS_SUCCESS;
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopPagedAttention(infiniopPagedAttentionDescriptor_t desc, void *workspace, uint64_t workspace_size, void *out,
                                                   void const *q, void const *k_cache, void const *v_cache, void const *k_scale, void const *v_scale,
                                                   void const *table, void const *offsets, void const *lengths, void *stream) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdPagedAttention(reinterpret_cast<PagedAttentionAmdDescriptor_t>(desc), workspace, workspace_size, out, q, k_cache, v_cache, k_scale,
                                     v_scale, table, offsets, lengths, stream);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopDestroyPagedAttentionDescriptor(infiniopPagedAttentionDescriptor_t desc) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdDestroyPagedAttentionDescriptor(reinterpret_cast<PagedAttentionAmdDescriptor_t>(desc));
        default:
            return STATUS_BAD_DEVICE;
    }
}

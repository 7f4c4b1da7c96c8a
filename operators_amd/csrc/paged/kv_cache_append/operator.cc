// Public entry points of KVCacheAppend: argument checks that need no device, and the way to the device's back end.
#include "amd/kv_cache_append_amd.h"

INFINIOP_C infiniopStatus_t infiniopCreateKVCacheAppendDescriptor(
    infiniopHandle_t handle, infiniopKVCacheAppendDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
    infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale, infiniopTensorDescriptor_t k, infiniopTensorDescriptor_t v,
    infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets, infiniopTensorDescriptor_t lengths) {
    if (handle == nullptr) {
        return STATUS_BAD_PARAM;
    }
    for (infiniopTensorDescriptor_t t : {k_cache, v_cache, k_scale, v_scale, k, v, table, offsets, lengths}) {
        if (t == nullptr) return STATUS_BAD_PARAM;
    }
    switch (handle->device) {
        case DevAmdGpu:
            return amdCreateKVCacheAppendDescriptor(reinterpret_cast<AmdHandle_t>(handle), reinterpret_cast<KVCacheAppendAmdDescriptor_t *>(desc_ptr),
                                                    k_cache, v_cache, k_scale, v_scale, k, v, table, offsets, lengths);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopGetKVCacheAppendWorkspaceSize(infiniopKVCacheAppendDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || size == nullptr) {
        return STATUS_BAD_PARAM;
    }
    *size = 0;
    return STATUS_SUCCESS;
}

INFINIOP_C infiniopStatus_t infiniopKVCacheAppend(infiniopKVCacheAppendDescriptor_t desc, void *, uint64_t, void *k_cache, void *v_cache, void *k_scale,
                                                  void *v_scale, void const *k, void const *v, void const *table, void const *offsets,
                                                  void const *lengths, void *stream) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdKVCacheAppend(reinterpret_cast<KVCacheAppendAmdDescriptor_t>(desc), k_cache, v_cache, k_scale, v_scale, k, v, table, offsets, lengths,
                                    stream);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopDestroyKVCacheAppendDescriptor(infiniopKVCacheAppendDescriptor_t desc) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdDestroyKVCacheAppendDescriptor(reinterpret_cast<KVCacheAppendAmdDescriptor_t>(desc));
        default:
            return STATUS_BAD_DEVICE;
    }
}

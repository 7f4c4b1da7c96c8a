// Public entry points of KVCacheCopy: argument checks that need no device, and the way to the device's back end.
#include "amd/kv_cache_copy_amd.h"

INFINIOP_C infiniopStatus_t infiniopCreateKVCacheCopyDescriptor(infiniopHandle_t handle, infiniopKVCacheCopyDescriptor_t *desc_ptr,
                                                                infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
                                                                infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale,
                                                                infiniopTensorDescriptor_t pairs) {
    if (handle == nullptr) {
        return STATUS_BAD_PARAM;
    }
    for (infiniopTensorDescriptor_t t : {k_cache, v_cache, k_scale, v_scale, pairs}) {
        if (t == nullptr) return STATUS_BAD_PARAM;
    }
    switch (handle->device) {
        case DevAmdGpu:
            return amdCreateKVCacheCopyDescriptor(reinterpret_cast<AmdHandle_t>(handle), reinterpret_cast<KVCacheCopyAmdDescriptor_t *>(desc_ptr), k_cache,
                                                  v_cache, k_scale, v_scale, pairs);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopKVCacheCopy(infiniopKVCacheCopyDescriptor_t desc, void *k_cache, void *v_cache, void *k_scale, void *v_scale,
                                                void const *pairs, void *stream) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdKVCacheCopy(reinterpret_cast<KVCacheCopyAmdDescriptor_t>(desc), k_cache, v_cache, k_scale, v_scale, pairs, stream);
        default:
            return STATUS_BAD_DEVICE;
    }
}

INFINIOP_C infiniopStatus_t infiniopDestroyKVCacheCopyDescriptor(infiniopKVCacheCopyDescriptor_t desc) {
    if (desc == nullptr) {
        return STATUS_BAD_PARAM;
    }
    switch (desc->device) {
        case DevAmdGpu:
            return amdDestroyKVCacheCopyDescriptor(reinterpret_cast<KVCacheCopyAmdDescriptor_t>(desc));
        default:
            return STATUS_BAD_DEVICE;
    }
}

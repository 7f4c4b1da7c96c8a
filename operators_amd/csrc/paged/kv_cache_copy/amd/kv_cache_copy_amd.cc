// Create-time validation for KVCacheCopy on the amd-gpu device.
#include "kv_cache_copy_amd.h"
#include <new>

infiniopStatus_t amdCreateKVCacheCopyDescriptor(AmdHandle_t handle, KVCacheCopyAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_cache,
                                                infiniopTensorDescriptor_t v_cache, infiniopTensorDescriptor_t k_scale,
                                                infiniopTensorDescriptor_t v_scale, infiniopTensorDescriptor_t pairs) {
    if (desc_ptr == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    amd::PagedCache cache;
    infiniopStatus_t st = amd::paged_cache(k_cache, v_cache, k_scale, v_scale, &cache);
    if (st == STATUS_SUCCESS) st = amd::paged_pairs(pairs);
    if (st != STATUS_SUCCESS) {
        return st;
    }
    auto *desc = new (std::nothrow) KVCacheCopyAmdDescriptor{DevAmdGpu, handle->device_id, cache, static_cast<uint32_t>(pairs->shape[0])};
    if (desc == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    *desc_ptr = desc;
    return STATUS_SUCCESS;
}

infiniopStatus_t amdDestroyKVCacheCopyDescriptor(KVCacheCopyAmdDescriptor_t desc) {
    delete desc;
    return STATUS_SUCCESS;
}

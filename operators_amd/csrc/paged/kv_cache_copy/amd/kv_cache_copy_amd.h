// amd-gpu back end of KVCacheCopy.
#ifndef INFINIOP_AMD_KV_CACHE_COPY_H
#define INFINIOP_AMD_KV_CACHE_COPY_H

#include "../../paged_cache.h"

struct KVCacheCopyAmdDescriptor {
    Device device;
    int device_id;
    amd::PagedCache cache;
    uint32_t pairs;
};
typedef KVCacheCopyAmdDescriptor *KVCacheCopyAmdDescriptor_t;

infiniopStatus_t amdCreateKVCacheCopyDescriptor(AmdHandle_t handle, KVCacheCopyAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_cache,
                                                infiniopTensorDescriptor_t v_cache, infiniopTensorDescriptor_t k_scale,
                                                infiniopTensorDescriptor_t v_scale, infiniopTensorDescriptor_t pairs);
infiniopStatus_t amdKVCacheCopy(KVCacheCopyAmdDescriptor_t desc, void *k_cache, void *v_cache, void *k_scale, void *v_scale, void const *pairs,
                                void *stream);
infiniopStatus_t amdDestroyKVCacheCopyDescriptor(KVCacheCopyAmdDescriptor_t desc);

#endif

// amd-gpu back end of KVCacheAppend.
#ifndef INFINIOP_AMD_KV_CACHE_APPEND_H
#define INFINIOP_AMD_KV_CACHE_APPEND_H

#include "../../paged_cache.h"

struct KVCacheAppendAmdDescriptor {
    Device device;
    int device_id;
    amd::Elem elem;// of k and v
    amd::PagedCache cache;
    amd::PagedRows rows;
    uint32_t tokens;
    int64_t k_token, k_head, v_token, v_head;// strides of k and v, elements
};
typedef KVCacheAppendAmdDescriptor *KVCacheAppendAmdDescriptor_t;

infiniopStatus_t amdCreateKVCacheAppendDescriptor(AmdHandle_t handle, KVCacheAppendAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_cache,
                                                  infiniopTensorDescriptor_t v_cache, infiniopTensorDescriptor_t k_scale,
                                                  infiniopTensorDescriptor_t v_scale, infiniopTensorDescriptor_t k, infiniopTensorDescriptor_t v,
                                                  infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets,
                                                  infiniopTensorDescriptor_t lengths);
infiniopStatus_t amdKVCacheAppend(KVCacheAppendAmdDescriptor_t desc, void *k_cache, void *v_cache, void *k_scale, void *v_scale, void const *k,
                                  void const *v, void const *table, void const *offsets, void const *lengths, void *stream);
infiniopStatus_t amdDestroyKVCacheAppendDescriptor(KVCacheAppendAmdDescriptor_t desc);

#endif

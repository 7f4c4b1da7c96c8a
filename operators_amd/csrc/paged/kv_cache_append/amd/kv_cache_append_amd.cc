// Create-time validation for KVCacheAppend on the amd-gpu device.
#include "kv_cache_append_amd.h"
#include <new>

infiniopStatus_t amdCreateKVCacheAppendDescriptor(AmdHandle_t handle, KVCacheAppendAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_cache,
                                                  infiniopTensorDescriptor_t v_cache, infiniopTensorDescriptor_t k_scale,
                                                  infiniopTensorDescriptor_t v_scale, infiniopTensorDescriptor_t k, infiniopTensorDescriptor_t v,
                                                  infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets,
                                                  infiniopTensorDescriptor_t lengths) {
    if (desc_ptr == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    amd::PagedCache cache;
    amd::PagedRows rows;
    infiniopStatus_t st = amd::paged_cache(k_cache, v_cache, k_scale, v_scale, &cache);
    if (st == STATUS_SUCCESS) st = amd::paged_table(table, cache.page, &rows);
    if (st == STATUS_SUCCESS) st = amd::paged_vector(offsets, static_cast<uint64_t>(rows.rows) + 1);
    if (st == STATUS_SUCCESS) st = amd::paged_vector(lengths, rows.rows);
    if (st == STATUS_SUCCESS) st = amd::paged_tokens(k);
    if (st == STATUS_SUCCESS) st = amd::paged_tokens(v);
    if (st != STATUS_SUCCESS) {
        return st;
    }
    if (!amd::same_dt(k->dt, v->dt)) {
        return STATUS_BAD_TENSOR_DTYPE;
    }
    for (infiniopTensorDescriptor_t t : {k, v}) {
        if (t->shape[0] != k->shape[0] || t->shape[1] != cache.kv_heads || t->shape[2] != cache.dim) return STATUS_BAD_TENSOR_SHAPE;
    }
    auto *desc = new (std::nothrow) KVCacheAppendAmdDescriptor{
        DevAmdGpu, handle->device_id, amd::elem_of(k->dt), cache, rows, static_cast<uint32_t>(k->shape[0]),
        k->strides[0], k->strides[1], v->strides[0], v->strides[1]};
    if (desc == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    *desc_ptr = desc;
    return STATUS_SUCCESS;
}

infiniopStatus_t amdDestroyKVCacheAppendDescriptor(KVCacheAppendAmdDescriptor_t desc) {
    delete desc;
    return STATUS_SUCCESS;
}

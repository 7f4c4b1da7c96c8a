// Create-time validation for PagedAttention on the amd-gpu device, and how its work is cut up.
#include "paged_attention_amd.h"
#include <cmath>
#include <new>

namespace {

uint32_t padded(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 && dim % 48 == 0 ? 192 : 256; }

}// namespace

infiniopStatus_t amdCreatePagedAttentionDescriptor(AmdHandle_t handle, PagedAttentionAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t out,
                                                   infiniopTensorDescriptor_t q, infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
                                                   infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale,
                                                   infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets,
                                                   infiniopTensorDescriptor_t lengths, uint64_t max_tokens, float scale) {
    if (desc_ptr == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    amd::PagedCache cache;
    amd::PagedRows rows;
    infiniopStatus_t st = amd::paged_cache(k_cache, v_cache, k_scale, v_scale, &cache);
    if (st == STATUS_SUCCESS) st = amd::paged_table(table, cache.page, &rows);
    if (st == STATUS_SUCCESS) st = amd::paged_vector(offsets, static_cast<uint64_t>(rows.rows) + 1);
    if (st == STATUS_SUCCESS) st = amd::paged_vector(lengths, rows.rows);
    if (st == STATUS_SUCCESS) st = amd::paged_tokens(q);
    if (st == STATUS_SUCCESS) st = amd::paged_tokens(out);
    if (st != STATUS_SUCCESS) {
        return st;
    }
    if (!amd::same_dt(q->dt, out->dt)) {
        return STATUS_BAD_TENSOR_DTYPE;
    }
    const uint64_t tokens = q->shape[0], heads = q->shape[1];
    if (out->shape[0] != tokens || out->shape[1] != heads || out->shape[2] != cache.dim || q->shape[2] != cache.dim) {
        return STATUS_BAD_TENSOR_SHAPE;
    }
    const uint64_t group = heads / cache.kv_heads;
    if (heads % cache.kv_heads != 0 || tokens * group >= (1ull << 31)) {
        return STATUS_BAD_TENSOR_SHAPE;// the query heads split evenly over the K/V heads
    }
    if (max_tokens == 0 || !std::isfinite(scale)) {
        return STATUS_BAD_PARAM;
    }
    if (max_tokens > tokens) max_tokens = tokens;

    PagedAttentionShape shape;
    // (two sets of 16 rows share what they read; heads wider than 128 leave no registers for that)
    shape.tile_rows = max_tokens * group <= 16 || cache.dim > 128 ? 16 : 32;
    // every row with tokens has one tile that it does not fill
    const uint64_t busy = rows.rows < tokens ? rows.rows : tokens;
    shape.most_tiles = static_cast<uint32_t>(tokens * group / shape.tile_rows + busy);
    // about three workgroups of a unit for each of the compute units
    shape.target = static_cast<uint32_t>(amd::ceil_div(3ull * handle->cu_count, cache.kv_heads));
    if ((static_cast<uint64_t>(shape.target) + shape.most_tiles) * cache.kv_heads > amd::max_grid_1d(256)) {
        return STATUS_BAD_TENSOR_SHAPE;
    }
    // Only tiles of several units use the workspace: of those, a tile of k keys is cut at every c of them where the
    // sum of all k is at most target * c, so they are at most 2 target units (ceil(x) <= 2 x from 1 on).
    const uint64_t units = 2ull * shape.target * cache.kv_heads;
    const uint64_t bytes = units * shape.tile_rows * (padded(cache.dim) + 2) * sizeof(float);
    auto *desc = new (std::nothrow) PagedAttentionAmdDescriptor{
        DevAmdGpu, handle->device_id, amd::same_dt(q->dt, BF16), cache, rows, static_cast<uint32_t>(tokens), static_cast<uint32_t>(group),
        static_cast<uint32_t>(max_tokens), q->strides[0], q->strides[1], out->strides[0], out->strides[1], scale, shape,
        tokens == 0 || rows.rows == 0 ? 0 : bytes};
    if (desc == nullptr) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    *desc_ptr = desc;
    return STATUS_SUCCESS;
}

infiniopStatus_t amdDestroyPagedAttentionDescriptor(PagedAttentionAmdDescriptor_t desc) {
    delete desc;
    return STATUS_SUCCESS;
}

// Create-time validation for PagedAttention on the amd-gpu device, and how its work is cut up.
#include "paged_attention_amd.h"
#include <cmath>
#include <new>

namespace {

// Sequences of up to this many query rows go to the kernel for decoding, in tiles of 32 that each read the keys (us, 64/8 heads x 128,
// there and with the kernel for prompts: 64 rows of 32 x 8192 keys 195 and 246, of 8 x 800 22.6 and 29.7; 96 rows of 32 x 8192 280 and 251).
constexpr uint32_t kFewRows = 64;

// Only tiles of several units use the workspace, and whatever offsets and lengths hold, of one head they are at most
//   * those of tiles of k steps that are cut at every c of them, where the sum of all k is at most (most_units - most_tiles) * c:
//     twice that many (ceil(x) <= 2 x from 1 on);
//   * for every tile that the rows can have, the units that a row as long as the table is cut into.
uint32_t slots_of(const PagedAttentionShape &s, const amd::PagedRows &rows, uint64_t page, uint64_t most_rows) {
    const uint64_t by_work = 2ull * (s.most_units - s.most_tiles);
    const uint64_t steps = amd::ceil_div(rows.cols * page, 32), units = amd::ceil_div(steps, s.least_steps);
    if (s.most_tiles == 0 || units < 2) return 0;
    const uint64_t tiles = rows.rows * amd::ceil_div(most_rows < s.most ? most_rows : s.most, s.tile_rows);
    return static_cast<uint32_t>(tiles >= by_work || tiles * units >= by_work ? by_work : tiles * units);
}
uint64_t workspace_of(const PagedAttentionShape &s, const amd::PagedCache &c) {
    return static_cast<uint64_t>(s.slots) * c.kv_heads * s.tile_rows * (paged_dim(c.dim) + 2) * sizeof(float);
}

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

    // a sequence with tokens has at most one tile that it does not fill
    const uint64_t busy = rows.rows < tokens ? rows.rows : tokens, query_rows = tokens * group, most_rows = max_tokens * group;
    const uint64_t cus = static_cast<uint64_t>(handle->cu_count);
    PagedAttentionShape few{}, many{};
    // two sets of 16 rows share what they read; heads wider than 128 leave no registers for that.  (us with tiles of 32 and of 16 rows,
    // 64/8 heads x 128, 32 rows of 8192 keys: 4 new tokens 123 and 172, 8 193 and 285; a call with a chunk of a prompt gives its single
    // tokens half-empty tiles: 8 beside a chunk of 500, 40/8 x 80, 253 and 246, 99 beside one of 600, 64/8 x 128, 285 and 272)
    few.tile_rows = most_rows <= 16 || cache.dim > 128 ? 16 : 32;
    few.least = 1;
    few.most = kFewRows;
    // (one sequence that may have many query rows goes to the kernel for prompts whatever it has: one launch less)
    few.most_tiles = busy == 1 && most_rows > kFewRows ? 0 : static_cast<uint32_t>(query_rows / few.tile_rows + busy);
    // as many units as the GPU holds, twice that where rows of unequal length meet (us, bf16, 64/8 heads x 128: 48 rows of
    // 100 to 131072 tokens 389 and 353, 32 of 8192 95 and 96; one of 131072 53 and 56); of 256 columns it holds one workgroup
    // a compute unit (32 rows of 100 to 32768 tokens 176 with twice the compute units, 182 with four times; of 8192 190 and 211)
    few.target = static_cast<uint32_t>(amd::ceil_div((rows.rows == 1 || paged_dim(cache.dim) == 256 ? 2 : 4) * cus, cache.kv_heads));
    few.most_units = few.target + few.most_tiles;
    many.tile_rows = 32 * paged_tile_waves(paged_dim(cache.dim));
    many.least = busy == 1 ? 1 : kFewRows + 1;
    many.most = UINT32_MAX;
    many.most_tiles = most_rows <= kFewRows ? 0 : static_cast<uint32_t>(query_rows / many.tile_rows + busy);
    many.target = static_cast<uint32_t>(amd::ceil_div(cus, cache.kv_heads));// one workgroup fills a compute unit
    many.at_once = rows.rows == 1 ? 0 : static_cast<uint32_t>(cus);
    many.most_units = (rows.rows == 1 ? 1 : 3) * many.target + many.most_tiles;// (one row is cut evenly)
    // (one sequence's units begin together, and a step for each wavefront is soonest done: 300 to 4000 keys, 32/8 heads x 128,
    // 11.2 to 12.8 us with 4, 13.1 to 14.2 with 8; where other rows' units wait, 8 of 2000 keys 20.0 with 4, 16.1 with 8)
    few.least_steps = rows.rows == 1 ? 4 : 8;
    few.whole_steps = 1;
    many.least_steps = 16;
    many.whole_steps = 2;// a tile of keys
    few.slots = slots_of(few, rows, cache.page, most_rows);
    many.slots = slots_of(many, rows, cache.page, most_rows);
    for (const PagedAttentionShape &s : {few, many}) {
        if (static_cast<uint64_t>(s.most_units) * cache.kv_heads > amd::max_grid_1d(512)) return STATUS_BAD_TENSOR_SHAPE;
    }
    const uint64_t for_few = workspace_of(few, cache), for_many = workspace_of(many, cache), most = for_few > for_many ? for_few : for_many;
    const uint64_t bytes = most > 16 ? most : 16;// (16: a call without a workspace is refused whether it needs one or not)
    auto *desc = new (std::nothrow) PagedAttentionAmdDescriptor{
        DevAmdGpu, handle->device_id, amd::same_dt(q->dt, BF16), cache, rows, static_cast<uint32_t>(tokens), static_cast<uint32_t>(group),
        static_cast<uint32_t>(max_tokens), q->strides[0], q->strides[1], out->strides[0], out->strides[1], scale, few, many,
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

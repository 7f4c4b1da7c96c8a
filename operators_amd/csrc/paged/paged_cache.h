// What the operators of the paged cache check alike at creation, and the image
// of a cache that their kernels get.  Host side; no HIP call.
#ifndef INFINIOP_AMD_PAGED_CACHE_H
#define INFINIOP_AMD_PAGED_CACHE_H

#include "../devices/amd/amd_handle.h"
#include "../devices/amd/common_amd.h"
#include "infiniop_paged.h"

namespace amd {

// Strides in elements: bytes for the codes, floats for the scales.
struct PagedStrides {
    int64_t page;    // codes, page to page
    uint32_t head;   // codes, head to head (a page spans less than 2^31)
    uint32_t token;  // codes, token to token
    int64_t s_page;  // scales, page to page
    int64_t s_head;  // scales, head to head
};

struct PagedCache {
    bool fp8;// F8E4M3, else I8
    uint32_t pages, kv_heads, page, dim, block;
    PagedStrides k, v;
};

// A stride's sign and size are free where its dimension has one entry.
inline infiniopStatus_t paged_strides(infiniopTensorDescriptor_t codes, infiniopTensorDescriptor_t scales, PagedStrides *out) {
    const uint64_t heads = codes->shape[1], page = codes->shape[2], dim = codes->shape[3], blocks = scales->shape[2];
    const int64_t sp = codes->strides[0], sh = heads > 1 ? codes->strides[1] : 0, st = codes->strides[2];
    if (codes->strides[3] != 1 || st < static_cast<int64_t>(dim) || st % 16 != 0 || sh < 0 || sh % 16 != 0) return STATUS_BAD_TENSOR_STRIDES;
    if (heads > 1 && sh < static_cast<int64_t>(dim)) return STATUS_BAD_TENSOR_STRIDES;
    if (codes->shape[0] > 1 && (sp < static_cast<int64_t>(dim) || sp % 16 != 0)) return STATUS_BAD_TENSOR_STRIDES;
    // 32-bit places within a page
    if (st >= (1ll << 31) || sh >= (1ll << 31)) return STATUS_BAD_TENSOR_STRIDES;
    const uint64_t span = (heads - 1) * static_cast<uint64_t>(sh) + (page - 1) * static_cast<uint64_t>(st) + dim;
    if (span >= (1ull << 31)) return STATUS_BAD_TENSOR_STRIDES;
    if (blocks > 1 && scales->strides[2] != 1) return STATUS_BAD_TENSOR_STRIDES;
    if ((heads > 1 && scales->strides[1] < 1) || (codes->shape[0] > 1 && scales->strides[0] < 1)) return STATUS_BAD_TENSOR_STRIDES;
    *out = PagedStrides{codes->shape[0] > 1 ? sp : 0, static_cast<uint32_t>(sh), static_cast<uint32_t>(st), codes->shape[0] > 1 ? scales->strides[0] : 0,
                        heads > 1 ? scales->strides[1] : 0};
    return STATUS_SUCCESS;
}

inline infiniopStatus_t paged_cache(infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache, infiniopTensorDescriptor_t k_scale,
                                    infiniopTensorDescriptor_t v_scale, PagedCache *out) {
    if (k_cache->ndim != 4 || v_cache->ndim != 4 || k_scale->ndim != 3 || v_scale->ndim != 3) return STATUS_BAD_TENSOR_SHAPE;
    const bool fp8 = same_dt(k_cache->dt, F8E4M3);
    if ((!fp8 && !same_dt(k_cache->dt, I8)) || !same_dt(v_cache->dt, k_cache->dt)) return STATUS_BAD_TENSOR_DTYPE;
    if (!same_dt(k_scale->dt, F32) || !same_dt(v_scale->dt, F32)) return STATUS_BAD_TENSOR_DTYPE;
    const uint64_t pages = k_cache->shape[0], heads = k_cache->shape[1], page = k_cache->shape[2], dim = k_cache->shape[3], blocks = k_scale->shape[2];
    for (int i = 0; i < 4; ++i) {
        if (v_cache->shape[i] != k_cache->shape[i]) return STATUS_BAD_TENSOR_SHAPE;
    }
    for (infiniopTensorDescriptor_t s : {k_scale, v_scale}) {
        if (s->shape[0] != pages || s->shape[1] != heads || s->shape[2] != blocks) return STATUS_BAD_TENSOR_SHAPE;
    }
    if (pages == 0 || pages >= (1ull << 31) || heads == 0 || heads >= (1ull << 16)) return STATUS_BAD_TENSOR_SHAPE;
    if (dim == 0 || dim % 16 != 0 || dim > 256) return STATUS_BAD_TENSOR_SHAPE;
    if (page == 0 || page % 16 != 0 || page >= (1ull << 20) || blocks == 0 || page % blocks != 0 || page / blocks % 16 != 0) return STATUS_BAD_TENSOR_SHAPE;
    if (heads * page * dim >= (1ull << 28)) return STATUS_BAD_TENSOR_SHAPE;
    *out = PagedCache{fp8, static_cast<uint32_t>(pages), static_cast<uint32_t>(heads), static_cast<uint32_t>(page), static_cast<uint32_t>(dim),
                      static_cast<uint32_t>(page / blocks), {}, {}};
    const infiniopStatus_t st = paged_strides(k_cache, k_scale, &out->k);
    return st != STATUS_SUCCESS ? st : paged_strides(v_cache, v_scale, &out->v);
}

// The rows of a batch: how many, how wide the table, and its row stride.
struct PagedRows {
    uint32_t rows, cols;
    int64_t stride;
};

inline infiniopStatus_t paged_table(infiniopTensorDescriptor_t table, uint64_t page, PagedRows *out) {
    if (table->ndim != 2) return STATUS_BAD_TENSOR_SHAPE;
    if (!same_dt(table->dt, I32)) return STATUS_BAD_TENSOR_DTYPE;
    const uint64_t rows = table->shape[0], cols = table->shape[1];
    // positions and table places below 2^31
    if (rows >= (1ull << 24) || cols == 0 || cols >= (1ull << 31) || cols * page >= (1ull << 31)) return STATUS_BAD_TENSOR_SHAPE;
    if (cols > 1 && table->strides[1] != 1) return STATUS_BAD_TENSOR_STRIDES;
    if (rows > 1 && table->strides[0] < static_cast<int64_t>(cols)) return STATUS_BAD_TENSOR_STRIDES;
    *out = PagedRows{static_cast<uint32_t>(rows), static_cast<uint32_t>(cols), rows > 1 ? table->strides[0] : static_cast<int64_t>(cols)};
    return STATUS_SUCCESS;
}

// A dense vector of n whole numbers.
inline infiniopStatus_t paged_vector(infiniopTensorDescriptor_t t, uint64_t n) {
    if (t->ndim != 1 || t->shape[0] != n) return STATUS_BAD_TENSOR_SHAPE;
    if (!same_dt(t->dt, I32)) return STATUS_BAD_TENSOR_DTYPE;
    return n > 1 && t->strides[0] != 1 ? STATUS_BAD_TENSOR_STRIDES : STATUS_SUCCESS;
}

// A dense list of pairs of whole numbers.
inline infiniopStatus_t paged_pairs(infiniopTensorDescriptor_t t) {
    if (t->ndim != 2 || t->shape[1] != 2 || t->shape[0] >= (1ull << 31)) return STATUS_BAD_TENSOR_SHAPE;
    if (!same_dt(t->dt, I32)) return STATUS_BAD_TENSOR_DTYPE;
    return t->strides[1] != 1 || (t->shape[0] > 1 && t->strides[0] != 2) ? STATUS_BAD_TENSOR_STRIDES : STATUS_SUCCESS;
}

// [tokens, heads, dim] (a launch spans less than 2^32 work-items) of 16-bit floating point with a unit innermost stride.
inline infiniopStatus_t paged_tokens(infiniopTensorDescriptor_t t) {
    if (t->ndim != 3) return STATUS_BAD_TENSOR_SHAPE;
    if (!same_dt(t->dt, F16) && !same_dt(t->dt, BF16)) return STATUS_BAD_TENSOR_DTYPE;
    if (t->shape[0] >= (1ull << 24) || t->shape[1] == 0 || t->shape[1] >= (1ull << 16)) return STATUS_BAD_TENSOR_SHAPE;
    return t->shape[2] > 1 && t->strides[2] != 1 ? STATUS_BAD_TENSOR_STRIDES : STATUS_SUCCESS;
}

}// namespace amd

#endif

// amd-gpu back end of PagedAttention.
#ifndef INFINIOP_AMD_PAGED_ATTENTION_H
#define INFINIOP_AMD_PAGED_ATTENTION_H

#include "../../paged_cache.h"

// The width that the kernels hold a head in.  192 for those that whole lanes of 12 columns make up.
constexpr uint32_t paged_dim(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 && dim % 48 == 0 ? 192 : 256; }
// Wavefronts of 32 query rows each that a workgroup of the kernel for prompts has.
constexpr int paged_tile_waves(int padded) { return padded <= 128 ? 8 : 4; }

// Steps of a unit that has at least `wanted`, at least `least`, in multiples of `whole` (a power of two).  No row has more than
// 2^26 (places below 2^31), so that 2^30 cut nothing; more wanted ones would not fit the whole number.
constexpr uint32_t paged_unit_steps(float wanted, uint32_t least, uint32_t whole) {
    const uint32_t steps = wanted < 0x1p30f ? static_cast<uint32_t>(wanted) + 1 : 1u << 30;
    return ((steps < least ? least : steps) + whole - 1) & ~(whole - 1);
}

// The work and the units of many rows, added up so that no sum wraps around whatever offsets and lengths hold.  A row's tiles are
// below 2^24 and its steps at most 2^26; of rows whose offsets name the same tokens there may be 2^24.
struct PagedSum {
    // Work of a workgroup's lane, at most 2^54 (of 2^9 lanes 2^63): units of that much divided among up to 2^10 are longer than any row.
    static constexpr uint64_t work(uint64_t sum, uint64_t tiles, uint64_t steps) {
        return sum + tiles * steps < (1ull << 54) ? sum + tiles * steps : 1ull << 54;
    }
    // Units in the low 48 bits, slots of the workspace (fewer than 2^16: slots_of in paged_attention_amd.cc) above.
    static constexpr uint64_t both(uint64_t units, uint64_t slots) { return units | slots << 48; }
    static constexpr uint64_t units(uint64_t sum) { return sum & ((1ull << 48) - 1); }
    static constexpr uint32_t slots(uint64_t sum) { return static_cast<uint32_t>(sum >> 48); }
};

// How a call's work is cut up.  A tile is up to `tile_rows` query rows (token by
// head of one K/V head's group) of one sequence; a unit is a tile over a range of
// keys, and what one workgroup computes.  `target` units of a K/V head or up to three
// times as many are aimed at; a tile is split over several where that gives fewer.  Sequences with
// at least `least` and at most `most` query rows are taken, the others left to the
// other kernel.
struct PagedAttentionShape {
    uint32_t tile_rows;
    uint32_t most_tiles;// of one K/V head, whatever the offsets; 0: the kernel is not needed
    uint32_t target, most_units;// most_units: of a head, whatever the lengths
    uint32_t at_once;// workgroups that the GPU holds, if units are made to fit that; 0 if not
    uint32_t least, most;
    uint32_t least_steps, whole_steps;// of a unit: at least, and what their number is a multiple of
    uint32_t slots;// of one K/V head: room in the workspace for the units of tiles that are cut
};

struct PagedAttentionAmdDescriptor {
    Device device;
    int device_id;
    bool bf16;// q and out, else F16
    amd::PagedCache cache;
    amd::PagedRows rows;
    uint32_t tokens, group, max_tokens;
    int64_t q_token, q_head, out_token, out_head;// elements
    float scale;
    PagedAttentionShape few, many;// query rows: decoding, prompts
    uint64_t workspace;
};
typedef PagedAttentionAmdDescriptor *PagedAttentionAmdDescriptor_t;

infiniopStatus_t amdCreatePagedAttentionDescriptor(AmdHandle_t handle, PagedAttentionAmdDescriptor_t *desc_ptr, infiniopTensorDescriptor_t out,
                                                   infiniopTensorDescriptor_t q, infiniopTensorDescriptor_t k_cache, infiniopTensorDescriptor_t v_cache,
                                                   infiniopTensorDescriptor_t k_scale, infiniopTensorDescriptor_t v_scale,
                                                   infiniopTensorDescriptor_t table, infiniopTensorDescriptor_t offsets,
                                                   infiniopTensorDescriptor_t lengths, uint64_t max_tokens, float scale);
infiniopStatus_t amdPagedAttention(PagedAttentionAmdDescriptor_t desc, void *workspace, uint64_t workspace_size, void *out, void const *q,
                                   void const *k_cache, void const *v_cache, void const *k_scale, void const *v_scale, void const *table,
                                   void const *offsets, void const *lengths, void *stream);
infiniopStatus_t amdDestroyPagedAttentionDescriptor(PagedAttentionAmdDescriptor_t desc);

#endif

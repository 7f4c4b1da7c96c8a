// Device side of page_table.h.  Include from .hip files only.
#ifndef INFINIOP_AMD_PAGE_TABLE_KERNEL_H
#define INFINIOP_AMD_PAGE_TABLE_KERNEL_H

#include "page_table.h"
#include "paged_kernel.h"

namespace amd {

// The workgroups of a launch, and which of them this is.
struct Crew {
    uint32_t index, count;
};

// The bits of `test(page)` for all pages of the crew's chunks, and how many are set in each chunk.
template<int WAVES, typename F>
__device__ __forceinline__ void mark_pages(Crew crew, uint32_t pages, uint64_t *words, uint32_t *counts, uint32_t *slots, F test) {
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t chunks = (pages + kChunkPages - 1) / kChunkPages;
    for (uint32_t c = crew.index; c < chunks; c += crew.count) {
        uint32_t set = 0;
        for (uint32_t w = wave; w < kChunkWords; w += WAVES) {
            const uint32_t p = c * kChunkPages + w * 64 + lane;
            const uint64_t bits = __builtin_amdgcn_ballot_w64(p < pages && test(p));
            if (lane == 0) words[c * kChunkWords + w] = bits;
            set += static_cast<uint32_t>(__builtin_popcountll(bits));
        }
        if (lane == 0) slots[wave] = set;
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t all = 0;
            for (int i = 0; i < WAVES; ++i) all += slots[i];
            counts[c] = all;
        }
        __syncthreads();
    }
}

}// namespace amd

#endif

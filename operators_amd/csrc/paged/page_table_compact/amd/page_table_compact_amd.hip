// gfx950 PageTableCompact: the i-th used page at or above `used` takes the i-th
// free page below it, so that pages 0 .. used-1 are the used ones:
//     rank(p) = used pages below p
//     p used, p >= used:  i = rank(p) - rank(used)        p free, p < used:  i = p - rank(p)
// Three phases: (1) used pages marked and counted by chunk, (2) ranks, the pairs,
// (3) table and counts.  Latency bound, a launch for each phase.
#include "../../page_table_kernel.h"
#include "page_table_compact_amd.h"

namespace {

using namespace amd;

constexpr int kTableWaves = 4;

struct CompactArgs {
    const int *table, *lengths, *refcount;
    int *new_table, *new_refcount, *pairs, *result;
    int64_t stride, new_stride;
    uint32_t rows, cols, pages, page, room;// room: pairs that there is space for
    FastDiv by_page;
    // workspace
    uint64_t *words;
    uint32_t *counts, *ranks;// used pages by chunk, and before each word
};

// used pages, and those among the pages below that number; to every lane
template<int WAVES>
__device__ __forceinline__ void totals(const CompactArgs &a, uint64_t *slots, uint32_t *used, uint32_t *below) {
    const uint32_t chunks = (a.pages + kChunkPages - 1) / kChunkPages;
    uint32_t unused, before;
    count_before<WAVES>(a.counts, 0, chunks, slots, &unused, used);
    count_before<WAVES>(a.counts, *used / kChunkPages, chunks, slots, &before, &unused);
    *below = *used == a.pages ? a.pages : before + bits_below(a.words, *used);
}

template<int WAVES>
__device__ void pair_up(const CompactArgs &a, Crew crew, uint64_t *slots) {
    const uint32_t lanes = WAVES * kWave, chunks = (a.pages + kChunkPages - 1) / kChunkPages;
    uint32_t used, below, unused;
    totals<WAVES>(a, slots, &used, &below);
    const uint32_t moved = used - below;
    for (uint32_t c = crew.index; c < chunks; c += crew.count) {
        uint32_t base;
        count_before<WAVES>(a.counts, c, chunks, slots, &base, &unused);
        for (uint32_t i = threadIdx.x; i < kChunkPages; i += lanes) {
            const uint32_t p = c * kChunkPages + i;
            if (p >= a.pages) continue;
            const uint32_t rank = base + bits_below(a.words, p);
            const bool is_used = ((a.words[p / 64] >> (p & 63)) & 1) != 0;
            if ((p & 63) == 0) a.ranks[p / 64] = rank;
            if (is_used && p >= used) a.pairs[2 * static_cast<uint64_t>(rank - below)] = static_cast<int>(p);
            if (!is_used && p < used) a.pairs[2 * static_cast<uint64_t>(p - rank) + 1] = static_cast<int>(p);
        }
    }
    for (uint64_t i = moved + static_cast<uint64_t>(crew.index) * lanes + threadIdx.x; i < a.room; i += static_cast<uint64_t>(crew.count) * lanes) {
        a.pairs[2 * i] = -1;
        a.pairs[2 * i + 1] = -1;
    }
    if (crew.index == 0 && threadIdx.x == 0) {
        a.result[0] = static_cast<int>(used);
        a.result[1] = static_cast<int>(moved);
    }
}

template<int WAVES>
__device__ void renumber(const CompactArgs &a, Crew crew) {
    const uint32_t lanes = WAVES * kWave;
    const uint32_t used = static_cast<uint32_t>(a.result[0]), moved = static_cast<uint32_t>(a.result[1]), below = used - moved;
    for (uint32_t r = crew.index; r < a.rows; r += crew.count) {
        const int length = a.lengths[r];
        const uint32_t tokens = length < 0 ? 0 : static_cast<uint32_t>(length) > a.cols * a.page ? a.cols * a.page : static_cast<uint32_t>(length);
        const uint32_t has = fast_quotient(tokens + a.page - 1, a.by_page), upto = a.new_table != a.table ? a.cols : has;
        for (uint32_t c = threadIdx.x; c < upto; c += lanes) {
            int e = a.table[r * a.stride + c];
            const uint32_t p = static_cast<uint32_t>(e);
            if (c < has && p < a.pages && p >= used) {
                const uint64_t word = a.words[p / 64];
                if (((word >> (p & 63)) & 1) != 0) {
                    const uint32_t rank = a.ranks[p / 64] + static_cast<uint32_t>(__builtin_popcountll(word & ((1ull << (p & 63)) - 1)));
                    e = a.pairs[2 * static_cast<uint64_t>(rank - below) + 1];
                }
            }
            a.new_table[r * a.new_stride + c] = e;
        }
    }
    const uint64_t first = static_cast<uint64_t>(crew.index) * lanes + threadIdx.x, step = static_cast<uint64_t>(crew.count) * lanes;
    // one lane for the two counts of a pair; those of other pages, where they go elsewhere
    for (uint64_t i = first; i < moved; i += step) {
        const int from = a.pairs[2 * i], to = a.pairs[2 * i + 1], n = a.refcount[from];
        a.new_refcount[from] = 0;
        a.new_refcount[to] = n;
    }
    if (a.new_refcount != a.refcount) {
        for (uint64_t p = first; p < a.pages; p += step) {
            const bool is_used = ((a.words[p / 64] >> (p & 63)) & 1) != 0;
            if (is_used == (p < used)) a.new_refcount[p] = is_used ? a.refcount[p] : 0;
        }
    }
}

__global__ __launch_bounds__(kTableWaves *kWave) void page_table_used(CompactArgs a) {
    __shared__ uint32_t slots[kTableWaves];
    mark_pages<kTableWaves>(Crew{blockIdx.x, gridDim.x}, a.pages, a.words, a.counts, slots, [&](uint32_t p) { return a.refcount[p] > 0; });
}
__global__ __launch_bounds__(kTableWaves *kWave) void page_table_pairs(CompactArgs a) {
    __shared__ uint64_t slots[kTableWaves];
    pair_up<kTableWaves>(a, Crew{blockIdx.x, gridDim.x}, slots);
}
__global__ __launch_bounds__(kTableWaves *kWave) void page_table_renumber(CompactArgs a) { renumber<kTableWaves>(a, Crew{blockIdx.x, gridDim.x}); }
}// namespace

infiniopStatus_t amdPageTableCompact(PageTableCompactAmdDescriptor_t desc, void *workspace, uint64_t workspace_size, void *new_table, void *new_refcount,
                                     void *pairs, void *result, void const *table, void const *lengths, void const *refcount, void *stream) {
    const PageTableCompactAmdDescriptor &d = *desc;
    const amd::TableSizes &z = d.sizes;
    if (workspace == nullptr || workspace_size < d.workspace) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    for (const void *p : {static_cast<const void *>(new_refcount), static_cast<const void *>(result), refcount}) {
        if (p == nullptr) return STATUS_BAD_PARAM;
    }
    if (z.old_rows.rows != 0 && (new_table == nullptr || table == nullptr || lengths == nullptr)) {
        return STATUS_BAD_PARAM;
    }
    if (d.pairs != 0 && pairs == nullptr) {
        return STATUS_BAD_PARAM;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 8 != 0 || (new_table == table && z.new_rows.stride != z.old_rows.stride)) {
        return STATUS_BAD_PARAM;
    }
    AMD_CHECK_HIP(hipSetDevice(d.device_id), STATUS_BAD_DEVICE);
    const uint64_t chunks = amd::chunks_of(z.pages), rows = z.old_rows.rows;
    auto *words = static_cast<uint64_t *>(workspace);
    auto *counts = reinterpret_cast<uint32_t *>(words + chunks * kChunkWords);
    const CompactArgs a{static_cast<const int *>(table), static_cast<const int *>(lengths), static_cast<const int *>(refcount),
                        static_cast<int *>(new_table), static_cast<int *>(new_refcount), static_cast<int *>(pairs), static_cast<int *>(result),
                        z.old_rows.stride, z.new_rows.stride, z.old_rows.rows, z.old_rows.cols, z.pages, z.page, d.pairs, amd::fast_div(z.page),
                        words, counts, counts + chunks};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned by_chunk = static_cast<unsigned>(chunks < 1024 ? chunks : 1024);
    const uint64_t rest = rows > by_chunk ? rows : by_chunk;
    page_table_used<<<by_chunk, kTableWaves * amd::kWave, 0, s>>>(a);
    page_table_pairs<<<by_chunk, kTableWaves * amd::kWave, 0, s>>>(a);
    page_table_renumber<<<static_cast<unsigned>(rest < 1024 ? rest : 1024), kTableWaves * amd::kWave, 0, s>>>(a);
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

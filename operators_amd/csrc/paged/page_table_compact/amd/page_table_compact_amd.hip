// gfx950 PageTableCompact: the i-th used page at or above `used` takes the i-th
// free page below it, so that pages 0 .. used-1 are the used ones:
//     rank(p) = used pages below p
//     p used, p >= used:  i = rank(p) - rank(used)        p free, p < used:  i = p - rank(p)
// Three phases: (1) used pages marked and counted by chunk, (2) ranks, the pairs,
// (3) table and counts.  Latency bound.  A launch for each phase, or, where one
// workgroup's LDS holds the pages, all in one (32 rows of 128, 4096 pages: 12.7 us in
// three launches, 6.7 in one).
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

template<int WAVES>
__device__ void pair_up(const CompactArgs &a, Crew crew, uint64_t *slots) {
    const uint32_t lanes = WAVES * kWave, chunks = (a.pages + kChunkPages - 1) / kChunkPages, lane = threadIdx.x & (kWave - 1);
    uint64_t words = lane < kChunkWords ? a.words[crew.index * kChunkWords + lane] : 0;
    // used pages in all and of the chunks before this workgroup's first, then of those before page `used`
    uint64_t count = 0, all;
    for (uint32_t c = threadIdx.x; c < chunks; c += lanes) {
        const uint64_t n = a.counts[c];
        count += n << 32 | (c < crew.index ? n : 0);
    }
    block_scan64<WAVES>(count, slots, &all);
    const uint32_t used = static_cast<uint32_t>(all >> 32), last = used / kChunkPages;
    uint32_t base = static_cast<uint32_t>(all);
    count = 0;
    for (uint32_t c = threadIdx.x; c < last; c += lanes) count += a.counts[c];
    uint64_t word = 0;// of the chunk that page `used` is in
    if (last < chunks && threadIdx.x < kChunkWords) word = a.words[last * kChunkWords + threadIdx.x];
    const uint32_t in_chunk = used % kChunkPages, whole = threadIdx.x * 64;
    count += static_cast<uint64_t>(__builtin_popcountll(whole + 64 <= in_chunk ? word : whole < in_chunk ? word & ((1ull << (in_chunk - whole)) - 1) : 0));
    block_scan64<WAVES>(count, slots, &all);
    const uint32_t below = static_cast<uint32_t>(all), moved = used - below;
    for (uint32_t c = crew.index; c < chunks;) {
        const uint32_t bits = static_cast<uint32_t>(__builtin_popcountll(words)), upto = wave_scan(bits);
        for (uint32_t w = threadIdx.x / kWave; w < kChunkWords; w += WAVES) {
            const uint64_t its = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(words), w)) |
                                 static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(words >> 32), w))) << 32;
            const uint32_t p = c * kChunkPages + w * 64 + lane;
            const uint32_t first = base + static_cast<uint32_t>(__builtin_amdgcn_readlane(upto - bits, w));
            const uint32_t rank = first + static_cast<uint32_t>(__builtin_popcountll(its & ((1ull << lane) - 1)));
            const bool is_used = ((its >> lane) & 1) != 0;
            if (p >= a.pages) continue;
            if (lane == 0) a.ranks[p / 64] = first;
            if (is_used && p >= used) a.pairs[2 * static_cast<uint64_t>(rank - below)] = static_cast<int>(p);
            if (!is_used && p < used) a.pairs[2 * static_cast<uint64_t>(p - rank) + 1] = static_cast<int>(p);
        }
        // (more chunks than workgroups: pools of over a million pages)
        const uint32_t next = c + crew.count;
        if (next < chunks) {
            for (uint32_t x = c; x < next; ++x) base += a.counts[x];
            words = lane < kChunkWords ? a.words[next * kChunkWords + lane] : 0;
        }
        c = next;
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
// All three phases in one workgroup of 1024 lanes, EACH pages a lane; where the pages go lies in LDS.
constexpr uint32_t kSmallLanes = 1024, kSmallEach = 8;
constexpr uint32_t kSmallEntries = kSmallLanes * kSmallEach, kSmallPages = kSmallLanes * kSmallEach;

template<uint32_t EACH>
__global__ __launch_bounds__(kSmallLanes) void page_table_compact_small(CompactArgs a, FastDiv by_cols) {
    constexpr int WAVES = kSmallLanes / kWave;
    __shared__ int goes[kSmallLanes * EACH];                 // where page p goes
    __shared__ int below_free[kSmallLanes * EACH / 2];       // the i-th free page below, at most half of all
    __shared__ uint64_t slots[WAVES];
    const uint32_t tid = threadIdx.x;
    // a lane's pages are neighbours, for their order
    int refs[EACH];
    uint64_t mine = 0, all;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t p = tid * EACH + i;
        refs[i] = p < a.pages ? a.refcount[p] : 0;
        mine += refs[i] > 0 ? 1 : 0;
    }
    const uint32_t first = static_cast<uint32_t>(block_scan64<WAVES>(mine, slots, &all)), used = static_cast<uint32_t>(all);
    uint64_t lower = 0, below_all;// used pages below page `used`
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) lower += refs[i] > 0 && tid * EACH + i < used ? 1 : 0;
    block_scan64<WAVES>(lower, slots, &below_all);
    const uint32_t below = static_cast<uint32_t>(below_all), moved = used - below;
    uint32_t rank = first;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t p = tid * EACH + i;
        if (refs[i] > 0) ++rank;
        else if (p < used) below_free[p - rank] = static_cast<int>(p);
    }
    __syncthreads();
    rank = first;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t p = tid * EACH + i;
        const bool is_used = refs[i] > 0;
        int to = static_cast<int>(p);
        if (is_used && p >= used) {
            to = below_free[rank - below];
            a.pairs[2 * (rank - below)] = static_cast<int>(p);
            a.pairs[2 * (rank - below) + 1] = to;
        }
        rank += is_used ? 1 : 0;
        goes[p] = to;
        // (a page that is used is written to by its own lane alone, a free one by the lane of the page that goes there)
        if (p < a.pages) {
            if (is_used) a.new_refcount[to] = refs[i];
            if (p >= used) a.new_refcount[p] = 0;
        }
    }
    for (uint32_t i = moved + tid; i < a.room; i += kSmallLanes) {
        a.pairs[2 * static_cast<uint64_t>(i)] = -1;
        a.pairs[2 * static_cast<uint64_t>(i) + 1] = -1;
    }
    if (tid == 0) {
        a.result[0] = static_cast<int>(used);
        a.result[1] = static_cast<int>(moved);
    }
    __syncthreads();
    for (uint32_t e = tid; e < a.rows * a.cols; e += kSmallLanes) {
        const uint32_t r = fast_quotient(e, by_cols), c = e - r * a.cols;
        const int length = a.lengths[r];
        const uint32_t tokens = length < 0 ? 0 : static_cast<uint32_t>(length) > a.cols * a.page ? a.cols * a.page : static_cast<uint32_t>(length);
        const bool held = c < fast_quotient(tokens + a.page - 1, a.by_page);
        const int p = a.table[r * a.stride + c];
        if (held || a.new_table != a.table) a.new_table[r * a.new_stride + c] = held && static_cast<uint32_t>(p) < a.pages ? goes[p] : p;
    }
}

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
    const uint64_t entries = rows * z.old_rows.cols;
    if (entries <= kSmallEntries && z.pages <= kSmallPages) {
        const amd::FastDiv by_cols = amd::fast_div(z.old_rows.cols);
        if (z.pages <= 4 * kSmallLanes) page_table_compact_small<4><<<1, kSmallLanes, 0, s>>>(a, by_cols);
        else page_table_compact_small<kSmallEach><<<1, kSmallLanes, 0, s>>>(a, by_cols);
    } else {
        const unsigned by_chunk = static_cast<unsigned>(chunks < 1024 ? chunks : 1024);
        const uint64_t rest = rows > by_chunk ? rows : by_chunk;
        page_table_used<<<by_chunk, kTableWaves * amd::kWave, 0, s>>>(a);
        page_table_pairs<<<by_chunk, kTableWaves * amd::kWave, 0, s>>>(a);
        page_table_renumber<<<static_cast<unsigned>(rest < 1024 ? rest : 1024), kTableWaves * amd::kWave, 0, s>>>(a);
    }
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

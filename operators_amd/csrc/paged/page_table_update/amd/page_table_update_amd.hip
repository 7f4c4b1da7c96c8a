// gfx950 PageTableUpdate: which row holds which pages after a step.
//     rows:    row r := row source[r]; refcount[p] += rows that got p - rows that gave it up
//     growth:  need[r] = pages(length + grow) - pages(length) + (1 if the last page is shared and grows)
//     fresh:   the k-th free page goes to the row whose need covers k in the running sum
// Four phases: (1) the rows that change are laid aside, (2) counts, (3) free pages marked
// and counted, needs worked out, rows written, (4) fresh pages handed out.  (3) and (4)
// need all of the one before, (2) of (1) the copy of the counts, where they go
// elsewhere, and of the rows its own.  Whole numbers throughout, added by
// atomics whose order does not matter.  Latency bound.  A launch for each phase, or, where
// the table fits the registers and the counts the LDS of one workgroup, all of them in
// one launch with three waits for memory (64 rows of 64, 4096 pages: 15.3 us in four
// launches, 8.6 in one).
#include "../../page_table_kernel.h"
#include "page_table_update_amd.h"

namespace {

using namespace amd;

constexpr int kTableWaves = 4;
// a row's growth: its pages (below 2^31; only pages of several tokens are copied, and then it is below 2^30), and whether
// the first of them takes the place of the last page
constexpr uint32_t kCopies = 1u << 31, kTooWide = ~0u;

struct UpdateArgs {
    const int *table, *lengths, *refcount, *source, *grow;
    int *new_table, *new_lengths, *new_refcount, *pairs, *result;
    int64_t stride, new_stride;
    uint32_t rows, cols, pages, page;
    FastDiv by_page;
    // workspace
    uint64_t *words;
    uint32_t *counts, *before, *need;// free pages by chunk; lengths before growth; growth
    int *aside;                      // [rows, cols]
};

__device__ __forceinline__ uint32_t in_range(const UpdateArgs &a, int length) {
    const uint32_t room = a.cols * a.page;// < 2^31
    return length < 0 ? 0 : static_cast<uint32_t>(length) > room ? room : static_cast<uint32_t>(length);
}
__device__ __forceinline__ uint32_t pages_of(const UpdateArgs &a, uint32_t tokens) { return fast_quotient(tokens + a.page - 1, a.by_page); }
__device__ __forceinline__ bool changes(const UpdateArgs &a, uint32_t r) { return a.source[r] != static_cast<int>(r); }

// (1) rows that change, laid aside; lengths before growth; the counts, where they go elsewhere
template<int WAVES>
__device__ void lay_aside(const UpdateArgs &a, Crew crew) {
    const uint32_t lanes = WAVES * kWave;
    for (uint32_t r = crew.index; r < a.rows; r += crew.count) {
        const uint32_t s = static_cast<uint32_t>(a.source[r]);
        const uint32_t length = s < a.rows ? in_range(a, a.lengths[s]) : 0, n = pages_of(a, length);
        if (threadIdx.x == 0) a.before[r] = length;
        if (s == r) continue;
        for (uint32_t c = threadIdx.x; c < a.cols; c += lanes) a.aside[static_cast<uint64_t>(r) * a.cols + c] = c < n ? a.table[s * a.stride + c] : -1;
    }
    if (a.new_refcount != a.refcount) {
        for (uint64_t p = static_cast<uint64_t>(crew.index) * lanes + threadIdx.x; p < a.pages; p += static_cast<uint64_t>(crew.count) * lanes)
            a.new_refcount[p] = a.refcount[p];
    }
}

// (2) what rows got, and what they gave up
template<int WAVES>
__device__ void count_rows(const UpdateArgs &a, Crew crew) {
    const uint32_t lanes = WAVES * kWave;
    for (uint32_t r = crew.index; r < a.rows; r += crew.count) {
        if (!changes(a, r)) continue;
        const uint32_t had = pages_of(a, in_range(a, a.lengths[r])), has = pages_of(a, a.before[r]);
        for (uint32_t c = threadIdx.x; c < had; c += lanes) {
            const uint32_t p = static_cast<uint32_t>(a.table[r * a.stride + c]);
            if (p < a.pages) atomicAdd(a.new_refcount + p, -1);
        }
        for (uint32_t c = threadIdx.x; c < has; c += lanes) {
            const uint32_t p = static_cast<uint32_t>(a.aside[static_cast<uint64_t>(r) * a.cols + c]);
            if (p < a.pages) atomicAdd(a.new_refcount + p, 1);
        }
    }
}

// (3) free pages, needs, rows without their growth
template<int WAVES>
__device__ void work_out(const UpdateArgs &a, Crew crew, uint32_t *slots) {
    const uint32_t lanes = WAVES * kWave;
    mark_pages<WAVES>(crew, a.pages, a.words, a.counts, slots, [&](uint32_t p) { return a.new_refcount[p] == 0; });
    for (uint32_t r = crew.index; r < a.rows; r += crew.count) {
        const bool changed = changes(a, r);
        const int *row = changed ? a.aside + static_cast<uint64_t>(r) * a.cols : a.table + r * a.stride;
        if (threadIdx.x == 0) {
            const uint32_t length = a.before[r], has = pages_of(a, length);
            const uint32_t by = a.grow[r] > 0 ? static_cast<uint32_t>(a.grow[r]) : 0;
            uint32_t need = kTooWide;
            if (by <= a.cols * a.page - length) {
                need = pages_of(a, length + by) - has;
                if (by != 0 && has * a.page != length) {
                    const uint32_t last = static_cast<uint32_t>(row[has - 1]);
                    if (last < a.pages && a.new_refcount[last] > 1) need = (need + 1) | kCopies;
                }
            }
            a.need[r] = need;
            a.pairs[2 * r] = -1;
            a.pairs[2 * r + 1] = -1;
        }
        if (changed || a.new_table != a.table) {
            for (uint32_t c = threadIdx.x; c < a.cols; c += lanes) a.new_table[r * a.new_stride + c] = row[c];
        }
    }
}

// (4) fresh pages to the rows that grow.  ends: LDS, for each row the sum of the needs up to it and its own.
// Everything that does not depend on something else is asked for at the start, and one scan adds up all of it.
template<int WAVES>
__device__ void hand_out(const UpdateArgs &a, Crew crew, uint32_t *ends, uint64_t *slots) {
    const uint32_t lanes = WAVES * kWave, chunks = (a.pages + kChunkPages - 1) / kChunkPages, lane = threadIdx.x & (kWave - 1);
    const uint32_t run = (a.rows + lanes - 1) / lanes, r0 = threadIdx.x * run;
    // a chunk's words, one for each of 16 lanes of every wavefront
    uint64_t words = lane < kChunkWords ? a.words[crew.index * kChunkWords + lane] : 0;
    // free pages of the chunks before the first of this workgroup, and of all
    uint64_t free = 0;
    for (uint32_t c = threadIdx.x; c < chunks; c += lanes) {
        const uint64_t n = a.counts[c];
        free += n << 32 | (c < crew.index ? n : 0);
    }
    // low half: pages, high half: rows too wide
    uint64_t mine = 0;
    for (uint32_t r = r0; r < r0 + run && r < a.rows; ++r) {
        const uint32_t n = a.need[r];
        mine += n == kTooWide ? 1ull << 40 : n & ~kCopies;
    }
    uint64_t total, all;
    uint64_t at = block_scan64<WAVES>(mine, slots, &total);
    block_scan64<WAVES>(free, slots, &all);
    for (uint32_t r = r0; r < r0 + run && r < a.rows; ++r) {
        const uint32_t n = a.need[r];
        at += n == kTooWide ? 0 : n & ~kCopies;
        ends[r] = static_cast<uint32_t>(at);// (sums beyond 2^32 do not fit into the pages, and nothing is handed out)
    }
    const uint64_t wanted = total & ((1ull << 40) - 1), all_free = all >> 32;
    const uint32_t wide = static_cast<uint32_t>(total >> 40);
    const bool fits = wide == 0 && wanted <= all_free;
    for (uint32_t r = crew.index * lanes + threadIdx.x; r < a.rows; r += crew.count * lanes) {
        a.new_lengths[r] = static_cast<int>(a.before[r] + (fits && a.grow[r] > 0 ? a.grow[r] : 0));
    }
    if (crew.index == 0 && threadIdx.x == 0) {
        const uint64_t lacks = wanted > all_free ? wanted - all_free : 0;
        a.result[0] = lacks > 0x7FFFFFFF ? 0x7FFFFFFF : static_cast<int>(lacks);
        a.result[1] = static_cast<int>(wide);
    }
    __syncthreads();
    if (!fits) return;// (uniform over the workgroup)
    uint32_t base = static_cast<uint32_t>(all);
    for (uint32_t c = crew.index; c < chunks && base < wanted;) {
        // the free pages before each word of the chunk, and in all of it
        const uint32_t bits = static_cast<uint32_t>(__builtin_popcountll(words)), upto = wave_scan(bits);
        for (uint32_t w = threadIdx.x / kWave; w < kChunkWords; w += WAVES) {
            const uint64_t word = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(words), w)) |
                                  static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(words >> 32), w))) << 32;
            const uint32_t p = c * kChunkPages + w * 64 + lane;
            const uint32_t k = base + static_cast<uint32_t>(__builtin_amdgcn_readlane(upto - bits, w)) + static_cast<uint32_t>(__builtin_popcountll(word & ((1ull << lane) - 1)));
            if (((word >> lane) & 1) == 0 || k >= wanted) continue;
            uint32_t lo = 0, hi = a.rows - 1;// the first row whose needs end beyond k
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (ends[mid] > k) hi = mid;
                else lo = mid + 1;
            }
            const uint32_t need = a.need[lo], nth = k - (ends[lo] - (need & ~kCopies)), has = pages_of(a, a.before[lo]);
            int *row = a.new_table + lo * a.new_stride;
            a.new_refcount[p] = 1;
            if ((need & kCopies) != 0 && nth == 0) {
                const int last = row[has - 1];
                a.pairs[2 * lo] = last;
                a.pairs[2 * lo + 1] = static_cast<int>(p);
                row[has - 1] = static_cast<int>(p);
                atomicAdd(a.new_refcount + last, -1);
            } else {
                row[has + nth - ((need & kCopies) != 0 ? 1 : 0)] = static_cast<int>(p);
            }
        }
        // (more chunks than workgroups: pools of over a million pages)
        const uint32_t next = c + crew.count;
        if (next < chunks) {
            for (uint32_t x = c; x < next; ++x) base += a.counts[x];
            words = lane < kChunkWords ? a.words[next * kChunkWords + lane] : 0;
        }
        c = next;
    }
}

__global__ __launch_bounds__(kTableWaves *kWave) void page_table_rows(UpdateArgs a) { lay_aside<kTableWaves>(a, Crew{blockIdx.x, gridDim.x}); }
__global__ __launch_bounds__(kTableWaves *kWave) void page_table_count(UpdateArgs a) { count_rows<kTableWaves>(a, Crew{blockIdx.x, gridDim.x}); }
__global__ __launch_bounds__(kTableWaves *kWave) void page_table_needs(UpdateArgs a) {
    __shared__ uint32_t slots[kTableWaves];
    work_out<kTableWaves>(a, Crew{blockIdx.x, gridDim.x}, slots);
}
__global__ __launch_bounds__(kTableWaves *kWave) void page_table_fresh(UpdateArgs a) {
    __shared__ uint32_t ends[kMostTableRows];
    __shared__ uint64_t slots[kTableWaves];
    hand_out<kTableWaves>(a, Crew{blockIdx.x, gridDim.x}, ends, slots);
}
// All four phases in one workgroup of 1024 lanes: the table's entries in registers, 8 a lane at most, the counts in LDS.
constexpr uint32_t kSmallLanes = 1024, kSmallEach = 8;
constexpr uint32_t kSmallEntries = kSmallLanes * kSmallEach, kSmallPages = kSmallLanes * kSmallEach, kSmallRows = kSmallLanes;

template<uint32_t EACH>// entries and pages of a lane
__global__ __launch_bounds__(kSmallLanes) void page_table_update_small(UpdateArgs a, FastDiv by_cols) {
    constexpr int WAVES = kSmallLanes / kWave;
    __shared__ int refs[kSmallLanes * EACH];
    __shared__ int source[kSmallRows], last[kSmallRows], grow[kSmallRows];
    __shared__ uint32_t had[kSmallRows], before[kSmallRows], need[kSmallRows], ends[kSmallRows];// pages, tokens, growth
    __shared__ uint64_t slots[WAVES];
    const uint32_t tid = threadIdx.x;
    if (tid < a.rows) {
        const uint32_t s = static_cast<uint32_t>(a.source[tid]);
        source[tid] = static_cast<int>(s);
        grow[tid] = a.grow[tid];
        had[tid] = pages_of(a, in_range(a, a.lengths[tid]));
        before[tid] = s < a.rows ? in_range(a, a.lengths[s]) : 0;
        last[tid] = -1;
    }
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t p = tid + i * kSmallLanes;
        refs[p] = p < a.pages ? a.refcount[p] : 1;
    }
    __syncthreads();
    int entry[EACH];
    const auto in_row = [&](uint32_t i, uint32_t *r, uint32_t *c) {
        const uint32_t e = tid + i * kSmallLanes;
        *r = fast_quotient(e, by_cols);
        *c = e - *r * a.cols;
        return e < a.rows * a.cols;
    };
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        uint32_t r, c;
        entry[i] = -1;
        if (!in_row(i, &r, &c)) continue;
        const uint32_t s = static_cast<uint32_t>(source[r]), has = pages_of(a, before[r]);
        const int own = a.table[r * a.stride + c];
        entry[i] = s == r ? own : c < has ? a.table[s * a.stride + c] : -1;
        if (s != r) {
            if (c < had[r] && static_cast<uint32_t>(own) < a.pages) atomicAdd(refs + own, -1);
            if (static_cast<uint32_t>(entry[i]) < a.pages) atomicAdd(refs + entry[i], 1);
        }
        if (c + 1 == has) last[r] = entry[i];
    }
    __syncthreads();
    uint64_t wanted = 0, total;// low half: pages, high half: rows too wide
    if (tid < a.rows) {
        const uint32_t length = before[tid], has = pages_of(a, length), by = grow[tid] > 0 ? static_cast<uint32_t>(grow[tid]) : 0;
        uint32_t n = kTooWide;
        if (by <= a.cols * a.page - length) {
            n = pages_of(a, length + by) - has;
            const uint32_t p = static_cast<uint32_t>(last[tid]);
            if (by != 0 && has * a.page != length && p < a.pages && refs[p] > 1) n = (n + 1) | kCopies;
        }
        need[tid] = n;
        wanted = n == kTooWide ? 1ull << 32 : n & ~kCopies;
        a.pairs[2 * tid] = -1;
        a.pairs[2 * tid + 1] = -1;
    }
    const uint64_t end = block_scan64<WAVES>(wanted, slots, &total) + wanted;// (fewer than 2^25 pages are wanted by rows that are not too wide)
    if (tid < a.rows) ends[tid] = static_cast<uint32_t>(end);
    // a lane's pages are neighbours, for the order in which they are handed out
    uint64_t mine = 0, all_free;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t p = tid * EACH + i;
        mine += p < a.pages && refs[p] == 0 ? 1 : 0;
    }
    uint32_t k = static_cast<uint32_t>(block_scan64<WAVES>(mine, slots, &all_free));
    const uint32_t all = static_cast<uint32_t>(total), wide = static_cast<uint32_t>(total >> 32);
    const bool fits = wide == 0 && all <= all_free;
    uint32_t is_free = 0;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t p = tid * EACH + i;
        is_free |= p < a.pages && refs[p] == 0 ? 1u << i : 0;
    }
    if (tid < a.rows) a.new_lengths[tid] = static_cast<int>(before[tid] + (fits && grow[tid] > 0 ? grow[tid] : 0));
    if (tid == 0) {
        a.result[0] = all > all_free ? static_cast<int>(all - all_free) : 0;
        a.result[1] = static_cast<int>(wide);
    }
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        uint32_t r, c;
        if (in_row(i, &r, &c) && (source[r] != static_cast<int>(r) || a.new_table != a.table)) a.new_table[r * a.new_stride + c] = entry[i];
    }
    __syncthreads();// refs read, the table written
    if (fits) {
#pragma unroll 1
        for (; is_free != 0 && k < all; is_free &= is_free - 1, ++k) {
            const uint32_t p = tid * EACH + static_cast<uint32_t>(__builtin_ctz(is_free));
            uint32_t lo = 0, hi = a.rows - 1;// the first row whose needs end beyond k
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (ends[mid] > k) hi = mid;
                else lo = mid + 1;
            }
            const uint32_t n = need[lo], nth = k - (ends[lo] - (n & ~kCopies)), has = pages_of(a, before[lo]);
            int *row = a.new_table + lo * a.new_stride;
            refs[p] = 1;
            if ((n & kCopies) != 0 && nth == 0) {
                a.pairs[2 * lo] = last[lo];
                a.pairs[2 * lo + 1] = static_cast<int>(p);
                row[has - 1] = static_cast<int>(p);
                atomicAdd(refs + last[lo], -1);
            } else {
                row[has + nth - ((n & kCopies) != 0 ? 1 : 0)] = static_cast<int>(p);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t p = tid + i * kSmallLanes;
        if (p < a.pages) a.new_refcount[p] = refs[p];
    }
}

}// namespace

infiniopStatus_t amdPageTableUpdate(PageTableUpdateAmdDescriptor_t desc, void *workspace, uint64_t workspace_size, void *new_table, void *new_lengths,
                                    void *new_refcount, void *pairs, void *result, void const *table, void const *lengths, void const *refcount,
                                    void const *source, void const *grow, void *stream) {
    const PageTableUpdateAmdDescriptor &d = *desc;
    const amd::TableSizes &z = d.sizes;
    if (workspace == nullptr || workspace_size < d.workspace) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    for (const void *p : {static_cast<const void *>(new_refcount), static_cast<const void *>(result), refcount}) {
        if (p == nullptr) return STATUS_BAD_PARAM;
    }
    // (no rows: the counts and the result are written all the same)
    for (const void *p : {static_cast<const void *>(new_table), static_cast<const void *>(new_lengths), static_cast<const void *>(pairs), table, lengths,
                          source, grow}) {
        if (p == nullptr && z.old_rows.rows != 0) return STATUS_BAD_PARAM;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 8 != 0 || (new_table == table && z.new_rows.stride != z.old_rows.stride)) {
        return STATUS_BAD_PARAM;
    }
    AMD_CHECK_HIP(hipSetDevice(d.device_id), STATUS_BAD_DEVICE);
    const uint64_t chunks = amd::chunks_of(z.pages), rows = z.old_rows.rows;
    auto *words = static_cast<uint64_t *>(workspace);
    auto *counts = reinterpret_cast<uint32_t *>(words + chunks * kChunkWords);
    const UpdateArgs a{static_cast<const int *>(table), static_cast<const int *>(lengths), static_cast<const int *>(refcount),
                       static_cast<const int *>(source), static_cast<const int *>(grow), static_cast<int *>(new_table),
                       static_cast<int *>(new_lengths), static_cast<int *>(new_refcount), static_cast<int *>(pairs), static_cast<int *>(result),
                       z.old_rows.stride, z.new_rows.stride, z.old_rows.rows, z.old_rows.cols, z.pages, z.page, amd::fast_div(z.page),
                       words, counts, counts + chunks, counts + chunks + rows, reinterpret_cast<int *>(counts + chunks + 2 * rows)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint64_t entries = rows * z.old_rows.cols;
    if (rows <= kSmallRows && entries <= kSmallEntries && z.pages <= kSmallPages) {
        const amd::FastDiv by_cols = amd::fast_div(z.old_rows.cols);
        const uint64_t most = entries > z.pages ? entries : z.pages;
        if (most <= 4 * kSmallLanes) page_table_update_small<4><<<1, kSmallLanes, 0, s>>>(a, by_cols);
        else page_table_update_small<kSmallEach><<<1, kSmallLanes, 0, s>>>(a, by_cols);
    } else {
        const unsigned by_row = static_cast<unsigned>(rows == 0 ? 1 : rows < 1024 ? rows : 1024), by_chunk = static_cast<unsigned>(chunks < 1024 ? chunks : 1024);
        page_table_rows<<<by_row, kTableWaves * amd::kWave, 0, s>>>(a);
        page_table_count<<<by_row, kTableWaves * amd::kWave, 0, s>>>(a);
        page_table_needs<<<by_row > by_chunk ? by_row : by_chunk, kTableWaves * amd::kWave, 0, s>>>(a);
        page_table_fresh<<<by_chunk, kTableWaves * amd::kWave, 0, s>>>(a);
    }
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

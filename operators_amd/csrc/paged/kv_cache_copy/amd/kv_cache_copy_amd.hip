// gfx950 KVCacheCopy: whole pages from place to place, codes and scales of k and
// v in one launch.  Bound by HBM, one byte read for each written.
// A workgroup, one wavefront, takes 4 KiB of a page's k or v of every grid-th pair, and
// all parts of a page fall to one XCD (workgroups are dealt to the eight in turn), whose
// address translation then meets each page once.  2000 pairs of random pages of
// 64 + 64 KiB: 99 us (5.3 TB/s); without that 103, in parts of 16 KiB by 256 lanes 104;
// of neighbouring pages 85 (6.2 TB/s).
// A list may be long and nearly empty (a compaction's has room for half the pool), so
// the wavefront reads 64 of its pairs at once and then goes through those that name pages.
#include "../../paged_kernel.h"
#include "kv_cache_copy_amd.h"

namespace {

using namespace amd;

constexpr int kCopyLanes = 64, kCopyVecs = 4;// 16-byte vectors of a lane and part

struct CopyArgs {
    uint8_t *codes[2];
    float *scales[2];
    PagedStrides at[2];
    const int *pairs;
    uint32_t count, pages, heads, page, blocks;
    uint32_t vecs, parts;       // 16-byte vectors of a page's k or v, and parts of it
    uint32_t per_token;         // vectors of a token
    bool dense;                 // a page is one run of codes, in k and in v
    FastDiv by_token, by_page, by_blocks;
};

__global__ __launch_bounds__(kCopyLanes) void kv_cache_copy(CopyArgs a) {
    const uint32_t lane = threadIdx.x & (kWave - 1);
    // eight lines of pairs at a time: pair y % 8 to XCD y % 8
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, both = 2 * a.parts;
    const bool eight = blockIdx.y < (gridDim.y & ~7u);
    const uint32_t y = eight ? id / (8 * both) * 8 + id % 8 : blockIdx.y, x = eight ? id / 8 % both : blockIdx.x;
    const int kv = x >= a.parts ? 1 : 0;
    const uint32_t part = kv ? x - a.parts : x;
    const PagedStrides at = a.at[kv];
    // where each of the lane's vectors lies in a page
    uint64_t place[kCopyVecs];
    bool mine[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i) {
        const uint32_t e = (part * kCopyVecs + i) * kCopyLanes + threadIdx.x;
        mine[i] = e < a.vecs;
        if (a.dense) {
            place[i] = static_cast<uint64_t>(e) * 16;
        } else {
            const uint32_t line = fast_quotient(e, a.by_token), head = fast_quotient(line, a.by_page);
            place[i] = static_cast<uint64_t>(head) * at.head + static_cast<uint64_t>(line - head * a.page) * at.token + (e - line * a.per_token) * 16u;
        }
    }
    for (uint64_t base = y; base < a.count; base += static_cast<uint64_t>(gridDim.y) * kWave) {
        const uint64_t p = base + static_cast<uint64_t>(lane) * gridDim.y;
        int from = -1, to = -1;
        if (p < a.count) {
            from = a.pairs[2 * p];
            to = a.pairs[2 * p + 1];
        }
        uint64_t todo = __builtin_amdgcn_ballot_w64(static_cast<uint32_t>(from) < a.pages && static_cast<uint32_t>(to) < a.pages);
        while (todo != 0) {
            const int l = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int64_t src = __builtin_amdgcn_readlane(from, l), dst = __builtin_amdgcn_readlane(to, l);
            const uint8_t *s = a.codes[kv] + src * at.page;
            uint8_t *d = a.codes[kv] + dst * at.page;
            u32x4 w[kCopyVecs];
#pragma unroll
            for (int i = 0; i < kCopyVecs; ++i) {
                if (mine[i]) w[i] = ld16_stream(s + place[i]);
            }
#pragma unroll
            for (int i = 0; i < kCopyVecs; ++i) {
                if (mine[i]) st16_stream(d + place[i], w[i]);
            }
            if (part == 0) {
                for (uint32_t e = threadIdx.x; e < a.heads * a.blocks; e += kCopyLanes) {
                    const uint32_t head = fast_quotient(e, a.by_blocks);
                    const int64_t o = head * at.s_head + (e - head * a.blocks);
                    a.scales[kv][dst * at.s_page + o] = a.scales[kv][src * at.s_page + o];
                }
            }
        }
    }
}

}// namespace

infiniopStatus_t amdKVCacheCopy(KVCacheCopyAmdDescriptor_t desc, void *k_cache, void *v_cache, void *k_scale, void *v_scale, void const *pairs,
                                void *stream) {
    const KVCacheCopyAmdDescriptor &d = *desc;
    if (d.pairs == 0) {
        return STATUS_SUCCESS;
    }
    for (const void *p : {static_cast<const void *>(k_cache), static_cast<const void *>(v_cache), static_cast<const void *>(k_scale),
                          static_cast<const void *>(v_scale), pairs}) {
        if (p == nullptr) return STATUS_BAD_PARAM;
    }
    if (!amd::aligned16(k_cache) || !amd::aligned16(v_cache)) {
        return STATUS_BAD_PARAM;
    }
    AMD_CHECK_HIP(hipSetDevice(d.device_id), STATUS_BAD_DEVICE);
    const amd::PagedCache &c = d.cache;
    const uint32_t vecs = static_cast<uint32_t>(static_cast<uint64_t>(c.kv_heads) * c.page * c.dim / 16);// a page spans less than 2^31
    const auto run = [&](const amd::PagedStrides &s) { return s.token == c.dim && (c.kv_heads == 1 || s.head == c.page * c.dim); };
    const uint32_t parts = static_cast<uint32_t>(amd::ceil_div(vecs, kCopyLanes * kCopyVecs));
    const CopyArgs a{{static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache)},
                     {static_cast<float *>(k_scale), static_cast<float *>(v_scale)},
                     {c.k, c.v},
                     static_cast<const int *>(pairs),
                     d.pairs,
                     c.pages,
                     c.kv_heads,
                     c.page,
                     c.page / c.block,
                     vecs,
                     parts,
                     c.dim / 16,
                     run(c.k) && run(c.v),
                     amd::fast_div(c.dim / 16),
                     amd::fast_div(c.page),
                     amd::fast_div(c.page / c.block)};
    const uint64_t wide = amd::ceil_div(65536, 2 * parts);// about 65 536 wavefronts, 256 for each compute unit, however long the list
    kv_cache_copy<<<dim3(2 * parts, static_cast<unsigned>(d.pairs < wide ? d.pairs : wide)), kCopyLanes, 0, static_cast<hipStream_t>(stream)>>>(a);
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

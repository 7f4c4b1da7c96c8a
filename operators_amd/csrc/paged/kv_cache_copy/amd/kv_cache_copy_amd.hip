// gfx950 KVCacheCopy: whole pages from place to place, codes and scales of k and
// v in one launch.  Bound by HBM, one byte read for each written.
// Workgroup (x, y) takes part y of the pairs x, x + grid, ...: a part is 16 KiB
// of a page's k or v.  A list may be long and nearly empty (a compaction's has
// room for half the pool), so a wavefront reads 64 of its pairs at once and then
// goes through those that name pages.
#include "../../paged_kernel.h"
#include "kv_cache_copy_amd.h"

namespace {

using namespace amd;

constexpr int kCopyLanes = 256, kCopyVecs = 4;// 16-byte vectors of a lane and part

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
    const int kv = blockIdx.y >= a.parts ? 1 : 0;
    const uint32_t part = kv ? blockIdx.y - a.parts : blockIdx.y;
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
    for (uint64_t base = blockIdx.x; base < a.count; base += static_cast<uint64_t>(gridDim.x) * kWave) {
        const uint64_t p = base + static_cast<uint64_t>(lane) * gridDim.x;
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
    const uint64_t wide = amd::ceil_div(16384, 2 * parts);// about 16 384 workgroups, 64 for each compute unit, however long the list
    kv_cache_copy<<<dim3(static_cast<unsigned>(d.pairs < wide ? d.pairs : wide), 2 * parts), kCopyLanes, 0, static_cast<hipStream_t>(stream)>>>(a);
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

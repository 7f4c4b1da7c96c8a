// Which unit of a call's work a workgroup computes.  The lengths are known on the
// GPU only, so every workgroup works it out for itself: the work of all rows is
// added up, keys per unit follow from it, and the unit's place among those of all
// rows gives the row.  One scan over the rows, a few hundred nanoseconds.
// Include from .hip files only.
#ifndef INFINIOP_AMD_PAGED_ATTENTION_UNITS_H
#define INFINIOP_AMD_PAGED_ATTENTION_UNITS_H

#include "../../paged_kernel.h"
#include "paged_attention_amd.h"

namespace amd {

constexpr uint32_t kStepKeys = 32;// keys that a wavefront takes at a time

struct AttentionArgs {
    RaggedRows rows;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    PagedStrides k_at, v_at;
    const uint16_t *q;
    uint16_t *out;
    int64_t q_token, q_head, out_token, out_head;
    uint32_t pages, kv_heads, dim, group, max_tokens, tile_rows;
    FastDiv by_group, by_block, by_tile;
    float scale;// of the scores, times log2(e)
    float units_each;// 1 / target
    uint32_t least_steps;// of a unit, and what their number is a multiple of
    uint32_t whole_steps;
    uint32_t least_rows, most_rows;// of a sequence that this kernel takes
    bool bf16;
    float *part_out, *part_stat;// [slot, kv head][tile row][padded dim], and [..][2]
};

struct Unit {
    uint32_t row, tile, chunk, chunks;// which tile of the row, which of its units
    uint32_t first, count, length;    // the row's tokens (RowSpan)
    uint32_t steps;                   // of a unit
    uint32_t slot;                    // where the tile's units begin in the workspace
};

struct RowWork {
    uint32_t tiles, steps;
};
__device__ __forceinline__ RowWork row_work(const AttentionArgs &a, const RowSpan &s) {
    const uint32_t tokens = s.count < a.max_tokens ? s.count : a.max_tokens;
    const uint32_t rows = tokens * a.group;
    if (rows < a.least_rows || rows > a.most_rows) return RowWork{0, 0};
    return RowWork{fast_quotient(rows + a.tile_rows - 1, a.by_tile), (s.length + kStepKeys - 1) / kStepKeys};
}

// Unit number `index` of all (SPLIT: tile number `index` of those that have several units); false if there are fewer.
template<int WAVES, bool SPLIT>
__device__ bool find_unit(const AttentionArgs &a, uint32_t index, uint64_t *slots, Unit *shared, Unit *out) {
    const uint32_t lanes = WAVES * kWave, run = (a.rows.rows + lanes - 1) / lanes, r0 = threadIdx.x * run;
    const uint32_t r1 = r0 + run < a.rows.rows ? r0 + run : a.rows.rows;
    uint64_t work = 0, total;
    for (uint32_t r = r0; r < r1; ++r) {
        const RowWork w = row_work(a, row_span(a.rows, r));
        work += static_cast<uint64_t>(w.tiles) * w.steps;
    }
    block_scan64<WAVES>(work, slots, &total);
    // at least total / target, with room for the rounding of the product
    uint32_t steps = static_cast<uint32_t>(static_cast<float>(total) * a.units_each * 1.000001f) + 1;
    steps = steps < a.least_steps ? a.least_steps : steps > 0x40000000u ? 0x40000000u : steps;
    steps = (steps + a.whole_steps - 1) & ~(a.whole_steps - 1);
    const auto chunks_of = [&](const RowWork &w) { return w.steps > steps ? (w.steps + steps - 1) / steps : 1u; };
    // low half: units (SPLIT: tiles of several), high half: slots of the workspace
    uint64_t mine = 0, all;
    for (uint32_t r = r0; r < r1; ++r) {
        const RowWork w = row_work(a, row_span(a.rows, r));
        const uint32_t c = chunks_of(w);
        const uint64_t units = static_cast<uint64_t>(w.tiles) * c;
        mine += (SPLIT ? (c > 1 ? w.tiles : 0) : units) | (c > 1 ? units << 32 : 0);
    }
    uint64_t before = block_scan64<WAVES>(mine, slots, &all);
    if (index >= static_cast<uint32_t>(all)) return false;
    if (index >= static_cast<uint32_t>(before) && index < static_cast<uint32_t>(before + mine)) {
        for (uint32_t r = r0; r < r1; ++r) {
            const RowSpan s = row_span(a.rows, r);
            const RowWork w = row_work(a, s);
            const uint32_t c = chunks_of(w);
            const uint64_t units = static_cast<uint64_t>(w.tiles) * c;
            const uint64_t n = (SPLIT ? (c > 1 ? w.tiles : 0) : units) | (c > 1 ? units << 32 : 0);
            if (index < static_cast<uint32_t>(before + n)) {
                const uint32_t i = index - static_cast<uint32_t>(before);
                // a prompt's last tiles see the most keys and begin first
                const uint32_t nth = SPLIT ? i : i / c;
                *shared = Unit{r, w.tiles - 1 - nth, SPLIT ? 0 : i - nth * c, c, s.first, s.count, s.length, steps,
                               static_cast<uint32_t>(before >> 32) + nth * c};
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    const auto same = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); };
    *out = Unit{same(shared->row), same(shared->tile), same(shared->chunk), same(shared->chunks), same(shared->first),
                same(shared->count), same(shared->length), same(shared->steps), same(shared->slot)};
    return true;
}

// 16-bit results, to nearest even
__device__ __forceinline__ uint32_t narrow2_rne(bool bf16, float a, float b) {
    if (bf16) return BF16Rne::narrow2_fast(a, b);
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

}// namespace amd

// paged_attention_tiles.hip: many query rows
void amdLaunchPagedAttentionTiles(const amd::AttentionArgs &a, bool fp8, unsigned units, hipStream_t s);

#endif

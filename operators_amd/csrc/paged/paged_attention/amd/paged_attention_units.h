// Which unit of a call's work a workgroup computes.  The lengths are known on the
// GPU only, so every workgroup works it out for itself: the work of all rows is
// added up, keys per unit follow from it, and the unit's place among those of all
// rows gives the row.  One scan over the rows, within a wavefront for up to 64.
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
    float units_each, rounds_each;// 1 / target; kv heads / workgroups at work at once, or 0
    uint32_t least_steps;// of a unit, and what their number is a multiple of
    uint32_t whole_steps;
    uint32_t least_rows, most_rows;// of a sequence that this kernel takes
    bool bf16;
    float *part_out, *part_stat;// [slot, kv head][tile row][padded dim]: a unit's own result, and [..][2]: m and l, its weight
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

// How many units a row's tiles are cut into where a unit has up to `steps`, and how many steps the longest then has.
__device__ __forceinline__ uint32_t unit_chunks(const RowWork &w, uint32_t steps) { return w.steps > steps ? (w.steps + steps - 1) / steps : 1u; }

__device__ __forceinline__ uint32_t unit_longest(const AttentionArgs &a, const RowWork &w, uint32_t chunks) {
    return ((w.steps + chunks - 1) / chunks + a.whole_steps - 1) & ~(a.whole_steps - 1);
}
// All rows' units, and the longest's steps.
struct UnitSum {
    float units, longest;
};

// Steps of a unit, from the work of all rows.  Cut into `target` parts, rows of unequal length leave odd ends.  Where
// many more workgroups wait than run (a.rounds_each is 0) these even out.  Otherwise the GPU takes the units in rounds,
// and of 2/3 to 3 times target parts those are taken whose rounds are the shortest together (a unit's
// beginning and end are worth 4 steps; 2505 query rows beside 8 of single ones: 3 units a tile in one round 243 us, 5 in two 275).
// sum(steps): of all rows.
template<typename F>
__device__ __forceinline__ uint32_t unit_steps(const AttentionArgs &a, float total, F sum) {
    const auto cut = [&](float by) {
        // at least total / target, with room for the roundings on the way
        return paged_unit_steps(total * a.units_each * by * 1.00001f, a.least_steps, a.whole_steps);
    };
    if (a.rounds_each == 0.0f) return cut(1.0f);
    float least = __builtin_inff();
    uint32_t best = 0, last = 0;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const uint32_t steps = cut(i == 0 ? 1.5f : i == 1 ? 1.25f : i == 2 ? 1.0f : i == 3 ? 2.0f / 3 : i == 4 ? 0.5f : 1.0f / 3);
        if (steps == last) break;// (the least there may be)
        last = steps;
        const UnitSum all = sum(steps);
        const float time = ceilf(all.units * a.rounds_each) * (all.longest + 4.0f);
        if (time < least) {
            least = time;
            best = steps;
        }
    }
    return best;
}

// Unit `i` of the row (JOIN: tile `i`), whose tiles' units begin at slot `slot`.
template<bool JOIN>
__device__ __forceinline__ Unit unit_of(const AttentionArgs &a, uint32_t r, const RowSpan &s, const RowWork &w, uint32_t chunks, uint32_t i, uint32_t slot) {
    const uint32_t nth = JOIN ? i : i / chunks;
    // a prompt's last tiles see the most keys and begin first
    return Unit{r, w.tiles - 1 - nth, JOIN ? 0 : i - nth * chunks, chunks, s.first, s.count, s.length,
                unit_longest(a, w, chunks), slot + nth * chunks};
}

// Unit number `index` of all (JOIN: tile number `index` of those that have several units); false if there are fewer.
template<int WAVES, bool JOIN>
__device__ __forceinline__ bool find_unit(const AttentionArgs &a, uint32_t index, uint64_t *slots, Unit *shared, Unit *out) {
    const auto same = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); };
    const uint32_t tid = threadIdx.x;
    if (a.rows.rows <= kWave) {// a row for each lane: every wavefront finds it for itself, without a barrier
        const uint32_t lane = tid & (kWave - 1);
        RowSpan s{0, 0, 0};
        if (lane < a.rows.rows) s = row_span(a.rows, lane);
        const RowWork w = row_work(a, s);
        const uint32_t steps = unit_steps(a, wave_sum(static_cast<float>(w.tiles) * static_cast<float>(w.steps)),
                                          [&](uint32_t n) {
                                              const uint32_t chunks = unit_chunks(w, n);
                                              return UnitSum{wave_sum(static_cast<float>(w.tiles * chunks)),
                                                             wave_max(w.tiles == 0 ? 0.0f : static_cast<float>(unit_longest(a, w, chunks)))};
                                          });
        const uint32_t chunks = unit_chunks(w, steps), units = w.tiles * chunks, mine = JOIN ? (chunks > 1 ? w.tiles : 0) : units;
        const uint32_t end = wave_scan(mine), in_slots = chunks > 1 ? units : 0, slot = wave_scan(in_slots) - in_slots;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(index < end && index >= end - mine);
        if (hit == 0) return false;
        const int l = __builtin_ctzll(hit);
        const auto at = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l)); };
        const RowSpan span{at(s.first), at(s.count), at(s.length)};
        const RowWork work{at(w.tiles), at(w.steps)};
        *out = unit_of<JOIN>(a, l, span, work, at(chunks), index - at(end - mine), at(slot));
        return true;
    }
    const uint32_t lanes = WAVES * kWave, run = (a.rows.rows + lanes - 1) / lanes, r0 = tid * run;
    const uint32_t r1 = r0 + run < a.rows.rows ? r0 + run : a.rows.rows;
    uint64_t work = 0, total;
    for (uint32_t r = r0; r < r1; ++r) {
        const RowWork w = row_work(a, row_span(a.rows, r));
        work = PagedSum::work(work, w.tiles, w.steps);
    }
    block_scan64<WAVES>(work, slots, &total);
    const uint32_t steps = unit_steps(a, static_cast<float>(total), [&](uint32_t n) {
        uint64_t units = 0, sum;
        float longest = 0.0f;
        for (uint32_t r = r0; r < r1; ++r) {
            const RowWork w = row_work(a, row_span(a.rows, r));
            const uint32_t chunks = unit_chunks(w, n);
            units += static_cast<uint64_t>(w.tiles) * chunks;
            if (w.tiles != 0) longest = fmaxf(longest, static_cast<float>(unit_longest(a, w, chunks)));
        }
        block_scan64<WAVES>(units, slots, &sum);
        return UnitSum{static_cast<float>(sum), block_max<WAVES>(longest, slots)};
    });
    // units (JOIN: tiles of several), and slots of the workspace
    const auto counts = [&](const RowWork &w, uint32_t chunks) {
        const uint64_t units = static_cast<uint64_t>(w.tiles) * chunks;
        return PagedSum::both(JOIN ? (chunks > 1 ? w.tiles : 0) : units, chunks > 1 ? units : 0);
    };
    uint64_t mine = 0, all;
    for (uint32_t r = r0; r < r1; ++r) {
        const RowWork w = row_work(a, row_span(a.rows, r));
        mine += counts(w, unit_chunks(w, steps));
    }
    uint64_t before = block_scan64<WAVES>(mine, slots, &all);
    if (index >= PagedSum::units(all)) return false;
    if (index >= PagedSum::units(before) && index < PagedSum::units(before + mine)) {
        for (uint32_t r = r0; r < r1; ++r) {
            const RowSpan s = row_span(a.rows, r);
            const RowWork w = row_work(a, s);
            const uint32_t chunks = unit_chunks(w, steps);
            const uint64_t n = counts(w, chunks);
            if (index < PagedSum::units(before + n)) {
                *shared = unit_of<JOIN>(a, r, s, w, chunks, index - static_cast<uint32_t>(PagedSum::units(before)), PagedSum::slots(before));
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    *out = Unit{same(shared->row), same(shared->tile), same(shared->chunk), same(shared->chunks), same(shared->first),
                same(shared->count), same(shared->length), same(shared->steps), same(shared->slot)};
    return true;
}

// log2, of subnormal numbers too, which the instruction by itself takes as 0; minus infinity of 0.
__device__ __forceinline__ float log2_of(float v) {
    return __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(v)) + static_cast<float>(__builtin_amdgcn_frexp_expf(v));
}
// A unit's weight beside others': l relative to 2^m, several of them together.
struct Weight {
    float m, l;
    __device__ __forceinline__ void add(float m2, float l2) {
        const float next = fmaxf(m, m2);
        l = l * __builtin_amdgcn_exp2f(m - next) + l2 * __builtin_amdgcn_exp2f(m2 - next);
        m = next;
    }
    __device__ __forceinline__ float inverse() const { return l > 0.0f ? 1.0f / l : 0.0f; }// 0 where nothing was seen
};
// What O is multiplied by, 2^exponent / l, as one factor or, where that may be out of range (V scales reach from 2^-149 to
// 2^127), as two.
struct WayBack {
    float first, second;
    bool two;// the same for the whole wavefront
    __device__ __forceinline__ WayBack(float l, float exponent) {
        two = __builtin_amdgcn_ballot_w64(fabsf(exponent) > 60.0f || l > 0x1p50f) != 0;
        second = two ? __builtin_amdgcn_exp2f(0.5f * exponent) : 1.0f;
        first = Weight{0.0f, l}.inverse() * (two ? second : __builtin_amdgcn_exp2f(exponent));
    }
};

// 16-bit results, to nearest even
__device__ __forceinline__ uint32_t narrow2_rne(bool bf16, float a, float b) {
    if (bf16) return BF16Rne::narrow2_fast(a, b);
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

}// namespace amd

// paged_attention_tiles.hip: many query rows.  `units` workgroups, and for what joins them the most tiles that are cut.
void amdLaunchPagedAttentionTiles(const amd::AttentionArgs &a, bool fp8, unsigned units, unsigned cut_tiles, hipStream_t s);

#endif

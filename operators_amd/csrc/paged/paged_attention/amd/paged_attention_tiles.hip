// gfx950 PagedAttention for many query rows: prompts and chunks of them.
//     S = K q^T,  P = exp2(scale S - m),  O = V^T P^T      transposed as in paged_attention_rows.hip
// A workgroup takes 256 query rows of one K/V head (tokens by heads of its group), a
// wavefront 32 of them, and all walk the keys together, 64 at a time (heads wider than
// 128: 128 rows, for one wavefront's registers are two's, and 32 keys).  A tile's codes
// are turned into fp16 once for all wavefronts on their way into LDS, keys by columns
// for K, columns by keys for V, so that either product reads its operand as 16-byte
// vectors; rows are 16 bytes longer than a power of two, which spreads eight
// neighbouring lanes over all banks.  Two tiles lie in LDS: while one is computed with,
// the next is written and the one behind it is on its way from memory.
// v_mfma_f32_32x32x16 leaves a lane 16 of the 32 keys of one query, and V's keys lie in
// the order in which those make up the second product's operand, so P is not exchanged.
// The V scale of a block, r times the largest so far, is added to the exponent, and taken out
// of its sum again, which saves a product for each score:
//     P = exp2(score + log2 r - m),  l = sum(P / r),  out = V^T P (largest V scale) / l
// m is the running maximum of score + log2 r less 10, each query row's own, so that what fp16
// holds of P depends only on what the row sees and gives weight to.  "The largest" is of the keys that
// some of the wavefront's 32 rows see; it keeps l in range, and a scale below 2^-80 of it counts as that.
// Two wavefronts share a SIMD and are a phase apart: one at its products, the other at
// its exponentials and the next tile's codes (when that took 330 us in the example
// below: 353 without, 390 with wavefronts of the same phase on a SIMD).
// 64 heads on 8 of 128 columns, a prompt of 4096 tokens: 291-318 us (from GPU to GPU), 0.9
// PFLOP/s; a library product of large fp16 matrices reaches 1.34.  Of that time (at 2.0 GHz)
// the matrix units are at work 40 %, the vector units 57 % (7 slots for each score, 4 of
// them the exponential), LDS 30 %.  Where the whole took 310 us, it took 231 without the products
// and 300 without the tiles' way from memory into LDS: bound by how far a SIMD does products and
// vector instructions of two wavefronts at once, and by the barrier after each phase.  Heads of
// 256 columns, 32 on 8, 2048 tokens: 169 us, 0.41 PFLOP/s; one wavefront a SIMD does its
// products and its exponentials one after the other.
#include "paged_attention_units.h"

namespace {

using namespace amd;

constexpr float kLift = 10.0f, kSlack = 4.0f, kNone = -1.0e30f;// as in paged_attention_rows.hip
constexpr float kLeastRatio = -80.0f;// log2 of a V scale to the largest: l stays below 2^(14 + 80 + 31)
constexpr float kZeroScale = -1000.0f;// log2 of a V scale of 0, and of one that nobody sees

__device__ __forceinline__ float pair_max(float v) {
    return across32(v, [](float a, float b) { return fmaxf(a, b); });
}

// What a wavefront's 32 query rows are: rows of the tile from `row0` on, tokens and heads of q and out.
struct TileRows {
    uint32_t row0, count, first, head;// count: how many there are of the 32
};

// 32 rows of q or out between memory, 16 bytes a lane and whole rows by neighbouring lanes, and LDS, a row every RP bytes.
template<int DP>
constexpr int kRowPitch = DP * 2 + 16;

template<int DP, int LANES = kWave, typename F>
__device__ __forceinline__ void each_piece(const AttentionArgs &a, const TileRows &t, uint32_t lane, int64_t token_step, int64_t head_step, F f) {
    constexpr int PIECES = DP / 8;
#pragma unroll
    for (int j = 0; j < (32 * PIECES + LANES - 1) / LANES; ++j) {
        const uint32_t index = lane + j * LANES, row = index / PIECES, piece = index % PIECES;
        const uint32_t r = t.row0 + row, token = fast_quotient(r, a.by_group);
        f(j, row < t.count && piece * 8 < a.dim, row * kRowPitch<DP> + piece * 16,
          static_cast<int64_t>(t.first + token) * token_step + static_cast<int64_t>(t.head * a.group + (r - token * a.group)) * head_step + piece * 8);
    }
}

// O times `by` into LDS, four of a lane's accumulators of each tile.  o[t][i] of lane (n, h) is column TD m' + t of
// row n, m' = 8 (i / 4) + 4 h + i % 4.
template<int DP, typename F>
__device__ __forceinline__ void put_four(const AttentionArgs &a, uint32_t n32, uint32_t h, uint8_t *scratch, uint32_t i4, F o_by) {
    constexpr int TD = DP / 32;
#pragma unroll
    for (int c = 0; c < 4 * TD; c += 2) {// columns side by side
        *reinterpret_cast<uint32_t *>(scratch + n32 * kRowPitch<DP> + ((8 * i4 + 4 * h) * TD + c) * 2) =
            narrow2_rne(a.bf16, o_by(c % TD, c / TD), o_by((c + 1) % TD, (c + 1) / TD));
    }
}
// Those rows to out.
template<int DP, int LANES = kWave>
__device__ __forceinline__ void put_rows(const AttentionArgs &a, const TileRows &rows, uint32_t lane, const uint8_t *scratch) {
    each_piece<DP, LANES>(a, rows, lane, a.out_token, a.out_head, [&](int, bool there, uint32_t in_lds, int64_t at) {
        if (there) st16_any(a.out + at, *reinterpret_cast<const u32x4 *>(scratch + in_lds));
    });
}

template<bool FP8, int DP>
__global__ __launch_bounds__(paged_tile_waves(DP) *kWave) void paged_attention_tiles(AttentionArgs a) {
    constexpr int kWaves = paged_tile_waves(DP), kLanes = kWaves * kWave;
    constexpr int BK = DP <= 128 ? 64 : 32;        // keys of a tile
    constexpr int KS = DP / 16, NC = DP / 16;      // steps of the first product; 16-byte pieces of a key
    constexpr int TD = DP / 32, NB = BK / 32, NG = BK / 16;
    constexpr int KP = DP * 2 + 16, VP = BK * 2 + 16;// bytes of a row in LDS
    constexpr int NT = DP == 96 ? 8 : NC;          // as many lanes as have a key's pieces (of 96 columns some are idle: 6 would make a wavefront's keys lie in two pages)
    constexpr int K_TASKS = BK * NT, V_TASKS = BK / 4 * (NT * 4);
    static_assert(K_TASKS == V_TASKS, "as many pieces of K as of V");
    constexpr int PER = (K_TASKS + kLanes - 1) / kLanes;// of a lane
    constexpr int TILES = 2 * (BK * KP + DP * VP), ROWS = kWaves * 32 * kRowPitch<DP>;
    __shared__ __attribute__((aligned(16))) uint8_t lds[TILES > ROWS ? TILES : ROWS];// two tiles; before and after, the query rows
    __shared__ uint64_t slots[kWaves];
    __shared__ Unit shared_unit;
    Unit u;
    const uint32_t head = blockIdx.x % a.kv_heads;
    if (!find_unit<kWaves, false>(a, blockIdx.x / a.kv_heads, slots, &shared_unit, &u)) return;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid / kWave)));
    const uint32_t n32 = lane & 31u, h = lane >> 5;
    const uint32_t tokens = u.count < a.max_tokens ? u.count : a.max_tokens;
    const uint32_t row0 = u.tile * a.tile_rows, rows = tokens * a.group;
    const int seen = static_cast<int>(u.length) - static_cast<int>(u.count);
    const auto sees = [&](uint32_t token) { return static_cast<uint32_t>(seen + static_cast<int>(token) < 0 ? 0 : seen + static_cast<int>(token) + 1); };
    const uint32_t row_end = row0 + a.tile_rows < rows ? row0 + a.tile_rows : rows;
    // this wavefront's rows, and what its first and its last see
    const uint32_t mine0 = row0 + wave * 32, mine1 = mine0 + 32 < row_end ? mine0 + 32 : row_end;
    const bool any = mine0 < row_end;
    const TileRows my_rows{mine0, any ? mine1 - mine0 : 0, u.first, head};
    const uint32_t all_see = any ? sees(fast_quotient(mine0, a.by_group)) : 0, some_see = any ? sees(fast_quotient(mine1 - 1, a.by_group)) : 0;
    const uint32_t tile_sees = sees(fast_quotient(row_end - 1, a.by_group));
    const uint32_t limit = mine0 + n32 < row_end ? sees(fast_quotient(mine0 + n32, a.by_group)) : 0;
    uint8_t *const scratch = lds + wave * 32 * kRowPitch<DP>;
    const auto k_lds = [&](uint32_t tile) { return lds + (tile & 1u) * (BK * KP); };
    const auto v_lds = [&](uint32_t tile) { return lds + 2 * BK * KP + (tile & 1u) * (DP * VP); };

    const uint32_t end = (tile_sees + kStepKeys - 1) / kStepKeys;
    const uint32_t s0 = u.chunk * u.steps, s1 = s0 + u.steps < end ? s0 + u.steps : end;
    const uint32_t first_key = s0 * kStepKeys, tiles = s1 > s0 ? (s1 - s0 + NB - 1) / NB : 0;
    const uint32_t my_tiles = some_see <= first_key ? 0 : (some_see - first_key + BK - 1) / BK < tiles ? (some_see - first_key + BK - 1) / BK : tiles;

    // a lane's pieces of a tile: 16 bytes of one key of K, 4 bytes of 4 keys of V
    const auto k_key = [&](int i) { return (tid + i * kLanes) / NT; };
    const auto k_piece = [&](int i) { return (tid + i * kLanes) % NT; };
    const auto v_keys = [&](int i) { return (tid + i * kLanes) / (NT * 4) * 4; };
    const auto v_col = [&](int i) { return (tid + i * kLanes) % (NT * 4) * 4; };
    const auto works = [&](int i) { return K_TASKS % kLanes == 0 || tid + i * kLanes < K_TASKS; };
    // (the 16 keys it is of: the same for the whole wavefront, for 16 keys are the pieces of whole wavefronts, or a
    // wavefront's pieces lie within 16 keys)
    const auto group_of = [](uint32_t key) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(key / 16))); };
    uint32_t k_off[PER], v_off[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        k_off[i] = (k_key(i) & 15u) * a.k_at.token + (k_piece(i) * 16 < a.dim ? k_piece(i) * 16 : 0);// (q is 0 behind dim)
        v_off[i] = (v_keys(i) & 15u) * a.v_at.token + (v_col(i) < a.dim ? v_col(i) : 0);             // (not stored behind dim)
    }
    const uint8_t *k_base = a.k + static_cast<uint64_t>(head) * a.k_at.head, *v_base = a.v + static_cast<uint64_t>(head) * a.v_at.head;
    const float *ks_base = a.k_scale + static_cast<int64_t>(head) * a.k_at.s_head, *vs_base = a.v_scale + static_cast<int64_t>(head) * a.v_at.s_head;
    const int *table = a.rows.table + u.row * a.rows.stride;

    // What tiles are loaded and computed with is read for 64 groups of 16 keys at once, one for each lane: the pages, ahead
    // for K and for V, and for the computation the scales.
    constexpr uint32_t kAhead = 64 / NG;// tiles of such a set
    // (worked out where it is needed, which is seldom: before the loop it would take registers that the loop needs)
    const auto seldom = [](uint32_t v) {
        asm volatile("" : "+v"(v));
        return v;
    };
    const auto page_of = [&](uint32_t tile, uint32_t upto) {// (upto: below it a key has to lie)
        const uint32_t key = first_key + tile * BK + seldom(lane) * 16;
        if (key >= upto) return -1;
        const int page = table[fast_quotient(key, a.rows.by_page)];
        return static_cast<uint32_t>(page) < a.pages ? page : -1;
    };
    const auto place_of = [&](uint32_t key) { return key - fast_quotient(key, a.rows.by_page) * a.rows.page; };
    const auto lane_of = [](float v, uint32_t l2) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l2)); };
    const auto lane_of64 = [](uint64_t v, uint32_t l2) {
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l2)) |
               static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), l2))) << 32;
    };
    // where a group's first key is; no page: page 0, for any place will do
    const auto bytes_of = [&](uint32_t tile, int page, const PagedStrides &at) {
        return static_cast<uint64_t>(static_cast<int64_t>(page < 0 ? 0 : page) * at.page) +
               static_cast<uint64_t>(place_of(first_key + tile * BK + seldom(lane) * 16)) * at.token;
    };
    uint64_t k_group, v_group, v_none, v_none_before;// v_none: a bit for each group without a page, of this set and the last
    {
        const int page = page_of(0, u.length);
        k_group = bytes_of(0, page, a.k_at);
        v_group = bytes_of(0, page, a.v_at);
        v_none = v_none_before = __builtin_amdgcn_ballot_w64(page < 0);
    }
    const auto k_set = [&](uint32_t tile) {
        if (tile % kAhead == 0) k_group = bytes_of(tile, page_of(tile, u.length), a.k_at);
    };
    const auto v_set = [&](uint32_t tile) {
        v_none_before = v_none;
        if (tile % kAhead == 0) {
            const int page = page_of(tile, u.length);
            v_group = bytes_of(tile, page, a.v_at);
            v_none = __builtin_amdgcn_ballot_w64(page < 0);
        }
    };
    u32x4 k_raw[PER];
    uint32_t v_raw[PER][4];
    const auto load_k = [&](uint32_t tile) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (!works(i)) continue;
            const uint8_t *p = k_base + lane_of64(k_group, tile % kAhead * NG + group_of(k_key(i)));
            asm("" : "+v"(k_off[i]));// (not added to k_base before the loop: a scalar base and a 32-bit offset make one instruction)
            k_raw[i] = ld16(p + k_off[i]);
        }
    };
    const auto load_v = [&](uint32_t tile) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (!works(i)) continue;
            const uint8_t *p = v_base + lane_of64(v_group, tile % kAhead * NG + group_of(v_keys(i)));
            asm("" : "+v"(v_off[i]));
#pragma unroll
            for (int j = 0; j < 4; ++j, p += a.v_at.token) v_raw[i][j] = *reinterpret_cast<const uint32_t *>(p + v_off[i]);
        }
    };
    const auto store_k = [&](uint32_t tile) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (!works(i)) continue;
            uint8_t *k = k_lds(tile) + k_key(i) * KP + k_piece(i) * 16;
            f16x8 half[2];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t c = prepare_codes<FP8>(k_raw[i][w]);
                const f16x2 x = pair_of<FP8, false>(c), y = pair_of<FP8, true>(c);
                f16x8 &to = half[w / 2];
                to[w % 2 * 4] = x.x;
                to[w % 2 * 4 + 1] = x.y;
                to[w % 2 * 4 + 2] = y.x;
                to[w % 2 * 4 + 3] = y.y;
            }
            if (NT != NC && k_piece(i) >= NC) continue;
            *reinterpret_cast<f16x8 *>(k) = half[0];
            *reinterpret_cast<f16x8 *>(k + NC * 16) = half[1];
        }
    };
    // 4 keys of column c of a lane's: 16 keys lie in order of the accumulator's halves, 0-3, 8-11, 4-7, 12-15, and
    // column d is row d / TD of the accumulator's tile d % TD
    const auto v_place = [&](uint32_t tile, uint32_t keys, uint32_t col, int c) {
        const uint32_t quad = keys / 4 & 3u, place = (keys & ~15u) + (quad & 1u) * 8 + (quad >> 1) * 4, d = col + c;
        return v_lds(tile) + (d % TD * 32 + d / TD) * VP + place * 2;
    };
    const auto store_v = [&](uint32_t tile) {// before the V of another tile is loaded
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (!works(i)) continue;
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = v_raw[i][j];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = prepare_codes<FP8>(x[j]);
            uint32_t pair[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                pair[j][0] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05010400u);
                pair[j][1] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07030602u);
            }
            if (NT != NC && v_col(i) >= DP) continue;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const auto two = [&](int j) { return __builtin_bit_cast(uint32_t, c % 2 ? pair_of<FP8, true>(pair[j][c / 2]) : pair_of<FP8, false>(pair[j][c / 2])); };
                *reinterpret_cast<u32x2 *>(v_place(tile, v_keys(i), v_col(i), c)) = u32x2{two(0), two(1)};
            }
        }
    };
    // What lies behind the row's end, or in no page, may be anything, and as e4m3 no number, which times 0 is not 0: a lane
    // puts zeros where it has just stored it.
    const auto clear_v = [&](uint32_t tile, uint64_t without) {
        if (!FP8) return;
        const uint32_t none = static_cast<uint32_t>(without >> (tile % kAhead * NG)) & ((1u << NG) - 1);
        if (none == 0 && first_key + tile * BK + BK <= u.length) return;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t keys = seldom(v_keys(i)), col = seldom(v_col(i));
            if (!works(i) || (NT != NC && col >= DP)) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if ((none >> group_of(v_keys(i)) & 1u) == 0 && first_key + tile * BK + keys + j < u.length) continue;
#pragma unroll
                for (int c = 0; c < 4; ++c) *reinterpret_cast<uint16_t *>(v_place(tile, keys, col, c) + j * 2) = 0;
            }
        }
    };
    load_k(0);
    load_v(0);

    // the query rows as the second operand: piece 2 s + h of K's order in LDS at step s
    f16x8 q[KS];
    float factor;
    {
        u32x4 w[KS];
        each_piece<DP>(a, my_rows, lane, a.q_token, a.q_head, [&](int j, bool there, uint32_t, int64_t at) {
            w[j] = u32x4{0, 0, 0, 0};
            if (there) w[j] = ld16_any(a.q + at);
        });
        each_piece<DP>(a, my_rows, lane, 0, 0, [&](int j, bool, uint32_t in_lds, int64_t) { *reinterpret_cast<u32x4 *>(scratch + in_lds) = w[j]; });
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint32_t piece = 2 * s + h, d8 = piece % NC * 2 + piece / NC;
            w[s] = *reinterpret_cast<const u32x4 *>(scratch + n32 * kRowPitch<DP> + d8 * 16);
            float x[8];
            if (a.bf16) widen8<BF16Rne>(w[s], x);
            else widen8<F16Ref>(w[s], x);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
        }
        top = pair_max(top);
        const int e = top > 0.0f ? static_cast<int>(__float_as_uint(top) >> 23) - 127 : 0;
        factor = ldexpf(fabsf(a.scale), e);// (its sign goes into q: the largest product is the largest score)
        const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float x[8];
            if (a.bf16) widen8<BF16Rne>(w[s], x);
            else widen8<F16Ref>(w[s], x);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[s][i] = static_cast<_Float16>(ldexpf(x[i] * sign, -e));
        }
    }
    f32x16 o[TD];
#pragma unroll
    for (int t = 0; t < TD; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    }
    // the running maximum less 10 of score + v_rel, which l is relative to, and log2 of the largest V scale so far, which O is too
    float m = kNone, l = 0.0f, v_top = kNone;
    float k_scale, v_rel, v_back;// of the lane's group: of V log2 relative to v_top, and the way back
    uint64_t no_page = 0;        // a bit for each group
    const auto scales = [&](uint32_t tile) {
        const int page = page_of(tile, some_see);// (what none of these rows sees counts as no page)
        float v_log = kZeroScale;
        k_scale = 0.0f;
        if (page >= 0) {
            const uint32_t block = fast_quotient(place_of(first_key + tile * BK + seldom(lane) * 16), a.by_block);
            k_scale = ks_base[page * a.k_at.s_page + block];
            v_log = fmaxf(log2_of(vs_base[page * a.v_at.s_page + block]), kZeroScale);
        }
        asm volatile("" : "+v"(k_scale));// (waited for here, not where this way and the one past it meet)
        no_page = __builtin_amdgcn_ballot_w64(page < 0);
        const float v_now = wave_max(v_log);
        if (v_now > v_top) {
            // all v_rel so far fall by `up`, and m with them, as far as l stays below 2^90; what O is beyond that goes into O
            const float up = v_now - v_top, down = fminf(up, fminf(120.0f, 90.0f - __builtin_amdgcn_logf(pair_max(l))));
            const float by = __builtin_amdgcn_exp2f(down - up);
            v_top = v_now;
            m -= down;
            l *= __builtin_amdgcn_exp2f(down);
#pragma unroll
            for (int t = 0; t < TD; ++t) o[t] *= by;
        }
        v_rel = fmaxf(v_log - v_top, kLeastRatio);
        v_back = __builtin_amdgcn_exp2f(-v_rel);
    };

    // The scores of a tile as the matrix units leave them, and what they are multiplied by.
    f32x16 s[NB];
    float f[NG], rel[NG], high = kNone;
    const auto products = [&](uint32_t tile) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < KS; ++e) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const f16x8 k = *reinterpret_cast<const f16x8 *>(k_lds(tile) + (b * 32 + n32) * KP + (2 * e + h) * 16);
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[e], s[b], 0, 0, 0);
            }
        }
    };
    // The largest score + v_rel, from the largest product of each group.
    const auto largest = [&](uint32_t tile) {
        const uint32_t at = tile % kAhead * NG;
        high = kNone;
#pragma unroll
        for (int g = 0; g < NG; ++g) rel[g] = lane_of(v_rel, at + g);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            // (above 0, so that what is not seen stays at minus infinity)
            f[g] = fmaxf(factor * lane_of(k_scale, at + g), 0x1p-126f);
            const f32x16 &x = s[g / 2];
            const int b = g % 2 * 8;
            const float top = fmaxf(fmaxf(fmaxf(fmaxf(x[b], x[b + 1]), x[b + 2]), fmaxf(fmaxf(x[b + 3], x[b + 4]), x[b + 5])), fmaxf(x[b + 6], x[b + 7]));
            high = fmaxf(high, __builtin_fmaf(top, f[g], rel[g]));
        }
    };
    // What a tile's scores need before their exponentials: the mask and the maximum.
    const auto ready = [&](uint32_t tile) {
        const uint32_t key0 = first_key + tile * BK;
        const uint32_t none = static_cast<uint32_t>(no_page >> (tile % kAhead * NG)) & ((1u << NG) - 1);
        if (none != 0 || key0 + BK > all_see) {
            const uint32_t mine = seldom(h * 4);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t key = key0 + b * 32 + 8 * (i / 4) + mine + i % 4;
                    const bool gone = key >= limit || (none >> (2 * b + i / 8) & 1u) != 0;
                    s[b][i] = gone ? -__builtin_inff() : s[b][i];
                }
            }
            largest(tile);
        }
        if (__builtin_amdgcn_ballot_w64(high > m + (kLift + kSlack)) != 0) {
            const float next = fmaxf(m, pair_max(high) - kLift), by = __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= by;
#pragma unroll
            for (int t = 0; t < TD; ++t) o[t] *= by;
        }
    };

    // Of eight wavefronts, two on each SIMD, the second four are a phase behind the first: while these use the matrix
    // units, those use the vector units for exponentials and for the codes on their way into LDS.  A barrier a phase.
    // What the first four write is needed in their next phase, what the others write in the phase after that.
    constexpr bool kTurns = kWaves == 8;
    const uint32_t lead = kTurns && wave < 4 ? 1 : 2;// K of tile + lead and V of the one before are written beside tile's exponentials
    if (tiles != 0) {
        scales(0);
        __syncthreads();// the query rows are read
        store_k(0);
        load_k(1);
        if (lead == 2) {
            store_v(0);
            clear_v(0, v_none);
            load_v(1);
            store_k(1);
            load_k(2);
        }
        __syncthreads();
        if (my_tiles != 0) {
            products(0);
            largest(0);
            ready(0);
        }
        __syncthreads();
        if (kTurns && wave >= 4) __syncthreads();
        for (uint32_t tile = 0; tile < tiles; ++tile) {
            k_set(tile + lead + 1);
            v_set(tile + lead);
            // (also behind the last tile, where nobody reads what is written, and of tiles that none of these rows sees: a
            // condition here would keep the rest from being mixed, and make the compiler wait for all loads where the ways meet)
            f16x8 p[NG];
            float sums = 0.0f;
            const uint32_t now = tile % kAhead * NG;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float less = rel[g] - m;
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g / 2][g % 2 * 8 + i], f[g], less));
                sums = __builtin_fmaf(((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7])), lane_of(v_back, now + g), sums);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const f16x2 w = __builtin_convertvector((f32x2{y[i], y[i + 1]}), f16x2);
                    p[g][i] = w.x;
                    p[g][i + 1] = w.y;
                }
            }
            store_k(tile + lead);
            store_v(tile + lead - 1);
            load_k(tile + lead + 1);
            load_v(tile + lead);
            l = tile < my_tiles ? l + sums : l;
            asm volatile("" : "+v"(l));// (not moved behind the barrier)
#pragma unroll
            for (int g = 0; g < NG; ++g) asm volatile("" : "+v"(p[g]));
            clear_v(tile + lead - 1, v_none_before);
            if (kTurns) __syncthreads();
            if (tile < my_tiles) {
                // the next tile's products (behind the last they are not used), and this one's sums
                if (kTurns) __builtin_amdgcn_s_setprio(1);
                products(tile + 1);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll
                    for (int t = 0; t < TD; ++t) {
                        const f16x8 x = *reinterpret_cast<const f16x8 *>(v_lds(tile) + (t * 32 + n32) * VP + g * 32 + h * 16);
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p[g], o[t], 0, 0, 0);
                    }
                }
                // eight operands are on their way from LDS while the matrix units are at work
                __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
                for (int i = 0; i < (KS * NB + NG * TD) - 8; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
                if (kTurns) __builtin_amdgcn_s_setprio(0);
                if ((tile + 1) % kAhead == 0) scales(tile + 1);
                largest(tile + 1);
                if (tile + 1 < my_tiles) ready(tile + 1);
            }
            __syncthreads();
        }
        if (kTurns && wave < 4) __syncthreads();
    }

    if (!any) return;
    l = across32(l, [](float x, float y) { return x + y; });
    const WayBack back(l, v_top);
#pragma unroll
    for (int t = 0; t < TD; ++t) o[t] *= back.first;
    if (back.two) {
#pragma unroll
        for (int t = 0; t < TD; ++t) o[t] *= back.second;
    }
    if (u.chunks > 1) {// as the lanes hold it, 16 bytes of each side by side
        const uint64_t at = (static_cast<uint64_t>(u.slot + u.chunk) * a.kv_heads + head) * kWaves + wave;
        if (h == 0) {
            a.part_stat[2 * (at * 32 + n32)] = m;
            a.part_stat[2 * (at * 32 + n32) + 1] = l;
        }
        float *p = a.part_out + at * (32 * DP) + lane * 4;
#pragma unroll
        for (int k = 0; k < 16 * TD; k += 4) {
            const auto of = [&](int j) { return o[(k + j) % TD][(k + j) / TD]; };
            *reinterpret_cast<f32x4 *>(p + k * kWave) = f32x4{of(0), of(1), of(2), of(3)};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i += 4) put_four<DP>(a, n32, h, scratch, i / 4, [&](int t, int j) { return o[t][i + j]; });
        put_rows<DP>(a, my_rows, lane, scratch);
    }
}

// The units of a tile together: 32 query rows a workgroup, in the lanes that held them, and a quarter of their sums a wavefront.
template<int DP>
__global__ __launch_bounds__(4 * kWave) void paged_attention_tiles_join(AttentionArgs a) {
    constexpr int TD = DP / 32;
    __shared__ __attribute__((aligned(16))) uint8_t scratch[32 * kRowPitch<DP>];
    __shared__ uint64_t slots[4];
    __shared__ Unit shared_unit;
    Unit u;
    const uint32_t waves = a.tile_rows / 32, part = blockIdx.x % waves, head = blockIdx.x / waves % a.kv_heads;
    if (!find_unit<4, true>(a, blockIdx.x / waves / a.kv_heads, slots, &shared_unit, &u)) return;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid / kWave)));
    const uint32_t n32 = lane & 31u;
    const uint32_t tokens = u.count < a.max_tokens ? u.count : a.max_tokens, rows = tokens * a.group, mine0 = u.tile * a.tile_rows + part * 32;
    if (mine0 >= rows) return;
    const auto at = [&](uint32_t c) { return (static_cast<uint64_t>(u.slot + c) * a.kv_heads + head) * waves + part; };
    const auto stat = [&](uint32_t c, int i) { return a.part_stat[2 * (at(c) * 32 + n32) + i]; };
    Weight all{kNone, 0.0f};
#pragma unroll 4
    for (uint32_t c = 0; c < u.chunks; ++c) all.add(stat(c, 0), stat(c, 1));
    const float each = all.inverse();
    f32x4 o[TD];
#pragma unroll
    for (int t = 0; t < TD; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t c = 0; c < u.chunks; ++c) {
        const float *p = a.part_out + at(c) * (32 * DP) + wave * (4 * TD * kWave) + lane * 4;
        const float by = stat(c, 1) * __builtin_amdgcn_exp2f(stat(c, 0) - all.m) * each;// its part of all weights
#pragma unroll
        for (int k = 0; k < TD; ++k) {
            const f32x4 x = ld16f(p + k * 4 * kWave);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[(k * 4 + j) % TD][(k * 4 + j) / TD] += x[j] * by;
        }
    }
    put_four<DP>(a, n32, lane >> 5, scratch, wave, [&](int t, int j) { return o[t][j]; });
    __syncthreads();
    put_rows<DP, 4 * kWave>(a, TileRows{mine0, rows - mine0 < 32 ? rows - mine0 : 32, u.first, head}, tid, scratch);
}

template<bool FP8, int DP>
void launch(const AttentionArgs &a, unsigned units, unsigned cut_tiles, hipStream_t s) {
    paged_attention_tiles<FP8, DP><<<units, paged_tile_waves(DP) * kWave, 0, s>>>(a);
    paged_attention_tiles_join<DP><<<cut_tiles * paged_tile_waves(DP), 4 * kWave, 0, s>>>(a);
}
template<bool FP8>
void launch(const AttentionArgs &a, unsigned units, unsigned cut_tiles, hipStream_t s) {
    // (96, which the kernel for decoding does not have, saves a quarter of 128's products)
    switch (a.dim > 64 && a.dim <= 96 ? 96 : paged_dim(a.dim)) {
        case 64: return launch<FP8, 64>(a, units, cut_tiles, s);
        case 96: return launch<FP8, 96>(a, units, cut_tiles, s);
        case 128: return launch<FP8, 128>(a, units, cut_tiles, s);
        case 192: return launch<FP8, 192>(a, units, cut_tiles, s);
        default: return launch<FP8, 256>(a, units, cut_tiles, s);
    }
}

}// namespace

void amdLaunchPagedAttentionTiles(const AttentionArgs &a, bool fp8, unsigned units, unsigned cut_tiles, hipStream_t s) {
    fp8 ? launch<true>(a, units, cut_tiles, s) : launch<false>(a, units, cut_tiles, s);
}

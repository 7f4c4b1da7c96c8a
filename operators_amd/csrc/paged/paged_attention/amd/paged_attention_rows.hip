// gfx950 PagedAttention for few query rows: decoding.
//     S = K q^T,  P = exp2(scale S - m),  O = V^T P^T      all transposed, keys down the accumulator's rows
// A wavefront takes 32 keys at a time, straight from the cache to registers, and up
// to 16 query rows (NT times) that share them.  Two v_mfma_f32_16x16x32 outputs hold
// 8 keys of one query in every lane, and those very 8 numbers, rounded to fp16, are
// that lane's share of the second product's operand: the matrix unit's k index is a
// label that both operands only have to agree on, so nothing of P is exchanged
// between lanes.  For V a lane holds the same 8 keys of dim / 16 neighbouring
// columns: byte permutations turn 8 keys x 4 columns round in registers.
// Codes are exact in fp16; q is multiplied by a power of two for each row that
// brings its largest element to [1, 2), so that it is off by at most 2^-25 of that
// element, whatever its type.  Scores, maxima, sums and O are fp32.
// The scale of a V block goes into P, whose running maximum is its own: with m_o of
// score + log2(V scale) and m of the scores,
//     P = exp2(score + log2(V scale) - m_o),  l = sum(exp2(score - m)),  out = V^T P 2^(m_o - m) / l
// so that what fp16 holds of P depends on nothing but what the query row sees and gives
// weight to, and neither O nor l on how large the values are.  P in fp16 costs each of
// these products at most 2^-11 of itself, as much as rounding `out` to fp16 does and an
// eighth of bf16.  It is lifted by 2^10, so that of one too small for that at most 2^-35 of
// the row's largest is lost, and the sum of very many small ones beside a large one is
// kept: m and m_o are the maxima less 10.
// The maxima are moved only when one is exceeded by 2^4 (P stays below 2^15), which
// leaves the usual step without an exchange between lanes.
// Bound by reading K and V once from HBM: 64 heads on 8 of 128 columns, 48 sequences of
// 100 to 131072 keys 347 us (5.5 TB/s; a large element-wise pass reaches 6.2), one of 131072
// 51 us (5.2), one of 1000 11 us, which is two launches and four waits for memory in turn.
#include "paged_attention_units.h"

namespace {

using namespace amd;

constexpr int kWaves = 4;
constexpr float kLift = 10.0f;   // log2 of P where it is the running maximum
constexpr float kSlack = 4.0f;   // log2 by which the running maximum may be exceeded
constexpr float kNone = -1.0e30f;// the maximum of no score
constexpr float kFar = 100.0f;   // log2 up to which P is exp2(score - m) times a power: what that loses below 2^-126 is nothing in fp16

// maximum and sum over the four lanes that hold one query row
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float quad_max(float v) { return across32(across16(v, larger), larger); }
__device__ __forceinline__ float quad_sum(float v) {
    const auto add = [](float a, float b) { return a + b; };
    return across32(across16(v, add), add);
}

// What a lane reads of 32 keys: of K, 16 bytes of each 64 columns of keys (lane % 16) of either half; of V,
// BYTES neighbouring columns of keys 4 (lane / 16) .. + 3 of either half.
template<int DP>
struct Tile {
    static constexpr int kChunks = DP / 64, kWords = DP / 64;
    u32x4 k[2][kChunks];
    uint32_t v[2][4][kWords];
};

template<int WORDS>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 1) {
        w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p));
    } else if constexpr (WORDS == 2) {
        const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p));
        w[0] = x.x;
        w[1] = x.y;
    } else if constexpr (WORDS == 3) {// at 4-byte boundaries
        typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
        typedef u32x3 __attribute__((aligned(4))) u32x3_any;
        const u32x3 x = __builtin_nontemporal_load(reinterpret_cast<const u32x3_any *>(p));
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
    } else {
        const u32x4 x = ld16_stream(p);
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
        w[3] = x.w;
    }
}

template<bool FP8, int DP, int NT>
__global__ __launch_bounds__(kWaves *kWave, DP > 192 ? 1 : DP > 128 ? 2 : (DP <= 64 ? 4 : 3) - (NT - 1)) void paged_attention_rows(AttentionArgs a) {
    constexpr int KS = DP / 32, CH = DP / 64, VB = DP / 16, WORDS = DP / 64;
    __shared__ uint64_t slots[kWaves];
    __shared__ Unit shared_unit;
    __shared__ float stat[3][kWaves][16 * NT];
    __shared__ f32x4 meet[2][NT * VB][kWave];
    Unit u;
    const uint32_t head = blockIdx.x % a.kv_heads;
    if (!find_unit<kWaves, false>(a, blockIdx.x / a.kv_heads, slots, &shared_unit, &u)) return;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid / kWave)));
    const uint32_t n16 = lane & 15u, g = lane >> 4;
    const uint32_t tokens = u.count < a.max_tokens ? u.count : a.max_tokens;
    const uint32_t row0 = u.tile * a.tile_rows, rows = tokens * a.group;
    // token i sees the places below seen + i + 1
    const int seen = static_cast<int>(u.length) - static_cast<int>(u.count);
    const auto sees = [&](uint32_t token) { return static_cast<uint32_t>(seen + static_cast<int>(token) < 0 ? 0 : seen + static_cast<int>(token) + 1); };
    const uint32_t row_end = row0 + a.tile_rows < rows ? row0 + a.tile_rows : rows;
    const uint32_t all_see = sees(fast_quotient(row0, a.by_group)), some_see = sees(fast_quotient(row_end - 1, a.by_group));

    // the lane's places within a page, relative to the half's first key
    uint32_t k_off[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) k_off[c] = n16 * a.k_at.token + (c * 64 + g * 16 < a.dim ? c * 64 + g * 16 : 0);// (q is 0 behind dim)
    const uint32_t v_off = g * 4 * a.v_at.token + (n16 * VB < a.dim ? n16 * VB : 0);                             // (not stored behind dim)
    const uint8_t *k_base = a.k + static_cast<uint64_t>(head) * a.k_at.head, *v_base = a.v + static_cast<uint64_t>(head) * a.v_at.head;
    const float *ks_base = a.k_scale + static_cast<int64_t>(head) * a.k_at.s_head, *vs_base = a.v_scale + static_cast<int64_t>(head) * a.v_at.s_head;
    const int *table = a.rows.table + u.row * a.rows.stride;

    const uint32_t end = (some_see + kStepKeys - 1) / kStepKeys;
    const uint32_t s0 = u.chunk * u.steps, s1 = s0 + u.steps < end ? s0 + u.steps : end;
    // steps s0 + wave, + 4, ...: page and scales of 32 of them are read at once, a half step by each lane;
    // the first of these are on their way while the queries are made ready
    int page = -1;
    float k_scale = 0.0f, v_log = 0.0f;
    const auto groups = [&](uint32_t base) {
        page = -1;
        k_scale = v_log = 0.0f;
        const uint32_t key = ((base + kWaves * (lane >> 1)) * 2 + (lane & 1)) * 16;
        if (key < u.length && base + kWaves * (lane >> 1) < s1) {
            const uint32_t col = fast_quotient(key, a.rows.by_page);
            page = table[col];
            if (static_cast<uint32_t>(page) < a.pages) {
                const uint32_t block = fast_quotient(key - col * a.rows.page, a.by_block);
                k_scale = ks_base[page * a.k_at.s_page + block];
                v_log = log2_of(vs_base[page * a.v_at.s_page + block]);
            } else {
                page = -1;
            }
        }
    };
    groups(s0 + wave);

    // the query rows, as the second operand of S: lane's row, 8 columns of each step of 32
    f16x8 q[NT][KS];
    float factor[NT];
    uint32_t limit[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t r = row0 + t * 16 + n16, token = fast_quotient(r, a.by_group);
        const bool mine = r < row_end;
        limit[t] = mine ? sees(token) : 0;
        float x[KS][8];
        float top = 0.0f;
        const uint16_t *p = a.q + static_cast<int64_t>(u.first + token) * a.q_token + static_cast<int64_t>(head * a.group + (r - token * a.group)) * a.q_head;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t d = c * 64 + g * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 w = {0, 0, 0, 0};
                if (mine && d < a.dim) w = ld16_any(p + d + h * 8);
                float y[8];
                if (a.bf16) widen8<BF16Rne>(w, y);
                else widen8<F16Ref>(w, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[2 * c + h][i] = y[i];
                    top = fmaxf(top, fabsf(y[i]));
                }
            }
        }
        top = quad_max(top);
        const int e = top > 0.0f ? static_cast<int>(__float_as_uint(top) >> 23) - 127 : 0;
        factor[t] = ldexpf(a.scale, e);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[t][s][i] = static_cast<_Float16>(ldexpf(x[s][i], -e));
        }
    }

    f32x4 o[NT][VB];
    float m[NT], l[NT], mo[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = mo[t] = kNone;
        l[t] = 0.0f;
#pragma unroll
        for (int j = 0; j < VB; ++j) o[t][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (uint32_t base = s0 + wave; base < s1; base += kWaves * 32) {
        if (base != s0 + wave) groups(base);
        const uint32_t count = (s1 - base + kWaves - 1) / kWaves < 32 ? (s1 - base + kWaves - 1) / kWaves : 32;
        // the next 32 keys' K is asked for before the scores of these are computed, their V after, in the place of this K
        const auto of_half = [&](uint32_t i, int h, uint32_t *at) {
            const uint32_t key = (base + kWaves * i) * kStepKeys + h * 16;
            *at = key - fast_quotient(key, a.rows.by_page) * a.rows.page;
            const int pg = __builtin_amdgcn_readlane(page, 2 * i + h);
            return static_cast<int64_t>(pg < 0 ? 0 : pg);// (no page: any place will do, the keys are masked)
        };
        const auto load_k = [&](uint32_t i, Tile<DP> &t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t at;
                const int64_t pg = of_half(i, h, &at);
                const uint8_t *p = k_base + pg * a.k_at.page + static_cast<uint64_t>(at) * a.k_at.token;
#pragma unroll
                for (int c = 0; c < CH; ++c) t.k[h][c] = ld16_stream(p + k_off[c]);
            }
        };
        const auto load_v = [&](uint32_t i, Tile<DP> &t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t at;
                const int64_t pg = of_half(i, h, &at);
                const uint8_t *p = v_base + pg * a.v_at.page + static_cast<uint64_t>(at) * a.v_at.token;
#pragma unroll
                for (int j = 0; j < 4; ++j) load_words<WORDS>(p + static_cast<uint64_t>(j) * a.v_at.token + v_off, t.v[h][j]);
            }
        };
        const auto step = [&](uint32_t i, Tile<DP> &t, Tile<DP> &next) {
            const uint32_t key0 = (base + kWaves * i) * kStepKeys;
            const int pg0 = __builtin_amdgcn_readlane(page, 2 * i), pg1 = __builtin_amdgcn_readlane(page, 2 * i + 1);
            const float ks[2] = {__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, k_scale), 2 * i)),
                                 __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, k_scale), 2 * i + 1))};
            const float vl[2] = {__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v_log), 2 * i)),
                                 __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v_log), 2 * i + 1))};
            f32x4 s[NT][2];
#pragma unroll
            for (int t2 = 0; t2 < NT; ++t2) s[t2][0] = s[t2][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int e = 0; e < KS; ++e) {
                    const uint32_t w0 = prepare_codes<FP8>(t.k[h][e / 2][e % 2 * 2]), w1 = prepare_codes<FP8>(t.k[h][e / 2][e % 2 * 2 + 1]);
                    f16x8 x;
                    const f16x2 p0 = pair_of<FP8, false>(w0), p1 = pair_of<FP8, true>(w0), p2 = pair_of<FP8, false>(w1), p3 = pair_of<FP8, true>(w1);
                    x = f16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
#pragma unroll
                    for (int t2 = 0; t2 < NT; ++t2) s[t2][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[t2][e], s[t2][h], 0, 0, 0);
                }
            }
            if (i + 1 < count) load_v(i + 1, next);
            const bool masked = pg0 < 0 || pg1 < 0 || key0 + kStepKeys > all_see;
            if (masked) {// also V's codes behind the row's end, which may be anything
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (key0 + h * 16 + g * 4 + j >= u.length || (h == 0 ? pg0 : pg1) < 0) {
#pragma unroll
                            for (int w = 0; w < WORDS; ++w) t.v[h][j][w] = 0;
                        }
                    }
                }
            }
            f16x8 p[NT];
#pragma unroll
            for (int t2 = 0; t2 < NT; ++t2) {
                float x[8];
                const float f0 = factor[t2] * ks[0], f1 = factor[t2] * ks[1];
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2) {
                    x[i2] = s[t2][0][i2] * f0;
                    x[4 + i2] = s[t2][1][i2] * f1;
                }
                if (masked) {
#pragma unroll
                    for (int i2 = 0; i2 < 8; ++i2) {
                        const bool gone = key0 + (i2 / 4) * 16 + g * 4 + i2 % 4 >= limit[t2] || (i2 < 4 ? pg0 : pg1) < 0;
                        x[i2] = gone ? -__builtin_inff() : x[i2];
                    }
                }
                const float high0 = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), high1 = fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]));
                const float high = fmaxf(high0, high1), high_o = fmaxf(high0 + vl[0], high1 + vl[1]);
                if (__builtin_amdgcn_ballot_w64(high > m[t2] + (kLift + kSlack) || high_o > mo[t2] + (kLift + kSlack)) != 0) {
                    const float next = fmaxf(m[t2], quad_max(high) - kLift), next_o = fmaxf(mo[t2], quad_max(high_o) - kLift);
                    l[t2] *= __builtin_amdgcn_exp2f(m[t2] - next);
                    const float by = __builtin_amdgcn_exp2f(mo[t2] - next_o);
                    m[t2] = next;
                    mo[t2] = next_o;
#pragma unroll
                    for (int j = 0; j < VB; ++j) o[t2][j] *= by;
                }
                float sum = 0.0f;
                float y[8];
#pragma unroll
                for (int i2 = 0; i2 < 8; ++i2) {
                    y[i2] = __builtin_amdgcn_exp2f(x[i2] - m[t2]);
                    sum += y[i2];
                }
                l[t2] += sum;
                const float r0 = vl[0] + (m[t2] - mo[t2]), r1 = vl[1] + (m[t2] - mo[t2]);
                if (__builtin_amdgcn_ballot_w64(fmaxf(r0, r1) > kFar) != 0) {
#pragma unroll
                    for (int i2 = 0; i2 < 8; ++i2) y[i2] = __builtin_amdgcn_exp2f(x[i2] + (vl[i2 / 4] - mo[t2]));
                } else {
                    const float by[2] = {__builtin_amdgcn_exp2f(r0), __builtin_amdgcn_exp2f(r1)};
#pragma unroll
                    for (int i2 = 0; i2 < 8; ++i2) y[i2] *= by[i2 / 4];
                }
#pragma unroll
                for (int i2 = 0; i2 < 8; i2 += 2) {
                    const f16x2 w = __builtin_convertvector((f32x2{y[i2], y[i2 + 1]}), f16x2);
                    p[t2][i2] = w.x;
                    p[t2][i2 + 1] = w.y;
                }
            }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                uint32_t x[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[h][j] = prepare_codes<FP8>(t.v[h][j][w]);
                }
                // columns 0 and 1 (2 and 3) of keys 0, 1 and of keys 2, 3
                uint32_t pair[2][2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        pair[h][j][0] = __builtin_amdgcn_perm(x[h][2 * j + 1], x[h][2 * j], 0x05010400u);
                        pair[h][j][1] = __builtin_amdgcn_perm(x[h][2 * j + 1], x[h][2 * j], 0x07030602u);
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const auto two = [&](int h, int j) { return c % 2 ? pair_of<FP8, true>(pair[h][j][c / 2]) : pair_of<FP8, false>(pair[h][j][c / 2]); };
                    const f16x2 y0 = two(0, 0), y1 = two(0, 1), y2 = two(1, 0), y3 = two(1, 1);
                    const f16x8 y = {y0.x, y0.y, y1.x, y1.y, y2.x, y2.y, y3.x, y3.y};
#pragma unroll
                    for (int t2 = 0; t2 < NT; ++t2) o[t2][w * 4 + c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, p[t2], o[t2][w * 4 + c], 0, 0, 0);
                }
            }
        };
        Tile<DP> even, odd;
        load_k(0, even);
        load_v(0, even);
        for (uint32_t i = 0; i < count; i += 2) {
            if (i + 1 < count) load_k(i + 1, odd);
            step(i, even, odd);
            if (i + 1 < count) {
                if (i + 2 < count) load_k(i + 2, even);
                step(i + 1, odd, even);
            }
        }
    }

    // the four wavefronts' sums, to the first: maxima, then O by halves
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        l[t] = quad_sum(l[t]);
        if (g == 0) {
            stat[0][wave][t * 16 + n16] = m[t];
            stat[1][wave][t * 16 + n16] = l[t];
            stat[2][wave][t * 16 + n16] = mo[t];
        }
    }
    __syncthreads();
    float total[NT], high[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float high_o = kNone;
        high[t] = kNone;
        total[t] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            high[t] = fmaxf(high[t], stat[0][w][t * 16 + n16]);
            high_o = fmaxf(high_o, stat[2][w][t * 16 + n16]);
        }
#pragma unroll
        for (int w = 0; w < kWaves; ++w) total[t] += stat[1][w][t * 16 + n16] * __builtin_amdgcn_exp2f(stat[0][w][t * 16 + n16] - high[t]);
        const WayBack back(total[t], high_o - high[t]);
        const float by = back.first * __builtin_amdgcn_exp2f(mo[t] - high_o);
#pragma unroll
        for (int j = 0; j < VB; ++j) o[t][j] *= by;
        if (back.two) {
#pragma unroll
            for (int j = 0; j < VB; ++j) o[t][j] *= back.second;
        }
    }
    if (wave >= 2) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int j = 0; j < VB; ++j) meet[wave - 2][t * VB + j][lane] = o[t][j];
        }
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int j = 0; j < VB; ++j) o[t][j] += meet[wave][t * VB + j][lane];
        }
    }
    if (wave == 1) {// (its own half of the room: only it has read that)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int j = 0; j < VB; ++j) meet[1][t * VB + j][lane] = o[t][j];
        }
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < VB; ++j) o[t][j] += meet[1][t * VB + j][lane];
        const uint32_t r = row0 + t * 16 + n16;
        if (r >= row_end) continue;
        // o[t][j][i] is column (4 g + i) VB + j of the row
        if (u.chunks > 1) {
            const uint64_t at = (static_cast<uint64_t>(u.slot + u.chunk) * a.kv_heads + head) * a.tile_rows + t * 16 + n16;
            if (g == 0) {
                a.part_stat[2 * at] = high[t];
                a.part_stat[2 * at + 1] = total[t];
            }
            if (total[t] == 0.0f) continue;// not read
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < VB; j += 4) {
                    *reinterpret_cast<f32x4 *>(a.part_out + at * DP + (4 * g + i) * VB + j) = f32x4{o[t][j][i], o[t][j + 1][i], o[t][j + 2][i], o[t][j + 3][i]};
                }
            }
        } else {
            const uint32_t token = fast_quotient(r, a.by_group);
            uint16_t *p = a.out + static_cast<int64_t>(u.first + token) * a.out_token + static_cast<int64_t>(head * a.group + (r - token * a.group)) * a.out_head;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t d = (4 * g + i) * VB;
                if (d >= a.dim) continue;
#pragma unroll
                for (int j = 0; j < VB; j += 4) {
                    *reinterpret_cast<u32x2_any *>(p + d + j) = u32x2{narrow2_rne(a.bf16, o[t][j][i], o[t][j + 1][i]), narrow2_rne(a.bf16, o[t][j + 2][i], o[t][j + 3][i])};
                }
            }
        }
    }
}

// The units of a tile together: a wavefront takes one query row, or, where the tile has many units, the four of a
// workgroup a quarter of a row's each (one sequence of 131072 keys in 64 units: 10.0 against 5.4 us).
template<int DP>
__global__ __launch_bounds__(kWaves *kWave) void paged_attention_join(AttentionArgs a) {
    constexpr int PER = DP / 64;
    __shared__ uint64_t slots[kWaves];
    __shared__ Unit shared_unit;
    __shared__ float meet[kWaves][PER][kWave];
    Unit u;
    const uint32_t head = blockIdx.x % a.kv_heads;
    if (!find_unit<kWaves, true>(a, blockIdx.x / a.kv_heads, slots, &shared_unit, &u)) return;
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / kWave)));
    const uint32_t tokens = u.count < a.max_tokens ? u.count : a.max_tokens, row0 = u.tile * a.tile_rows, left = tokens * a.group - row0;
    const uint32_t rows = left < a.tile_rows ? left : a.tile_rows;
    const bool four = u.chunks > 8;// wavefronts to a row
    const uint32_t quarter = (u.chunks + kWaves - 1) / kWaves, c0 = four ? wave * quarter : 0, c1 = four && c0 + quarter < u.chunks ? c0 + quarter : u.chunks;
    const uint32_t first = four ? blockIdx.y : blockIdx.y * kWaves + wave, step = four ? gridDim.y : gridDim.y * kWaves;
    for (uint32_t in_tile = first; in_tile < rows; in_tile += step) {
        const auto at = [&](uint32_t c) { return (static_cast<uint64_t>(u.slot + c) * a.kv_heads + head) * a.tile_rows + in_tile; };
        // a lane's unit of those that the wavefront adds up, and the weight of all
        const auto unit_weight = [&](uint32_t c) { return c < c1 ? Weight{a.part_stat[2 * at(c)], a.part_stat[2 * at(c) + 1]} : Weight{kNone, 0.0f}; };
        Weight mine = unit_weight(c0 + lane), all{kNone, 0.0f};
        for (uint32_t c = lane; c < u.chunks; c += kWave) all.add(a.part_stat[2 * at(c)], a.part_stat[2 * at(c) + 1]);
        const float high = wave_max(all.m);
        all = Weight{high, wave_sum(all.l * __builtin_amdgcn_exp2f(all.m - high))};
        const float each = all.inverse();
        float o[PER] = {};
        for (uint32_t base = c0; base < c1; base += kWave) {
            if (base != c0) mine = unit_weight(base + lane);
            const float by = mine.l * __builtin_amdgcn_exp2f(mine.m - high) * each;// the part of all weights
            const uint32_t n = c1 - base < kWave ? c1 - base : kWave;
            // 16 loads under way at a time; a unit that saw nothing has written nothing, and what is read of it is not used
            for (uint32_t k0 = 0; k0 < n; k0 += 16) {
                float x[16][PER];
#pragma unroll
                for (uint32_t k = 0; k < 16; ++k) {
                    const float *p = a.part_out + at(base + (k0 + k < n ? k0 + k : n - 1)) * DP + lane * PER;
#pragma unroll
                    for (int i = 0; i < PER; ++i) x[k][i] = p[i];
                }
#pragma unroll
                for (uint32_t k = 0; k < 16; ++k) {
                    const float w = k0 + k < n ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, by), k0 + k)) : 0.0f;
#pragma unroll
                    for (int i = 0; i < PER; ++i) o[i] += w != 0.0f ? w * x[k][i] : 0.0f;
                }
            }
        }
        if (four) {
#pragma unroll
            for (int i = 0; i < PER; ++i) meet[wave][i][lane] = o[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) o[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
#pragma unroll
                for (int i = 0; i < PER; ++i) o[i] += meet[w][i][lane];
            }
            __syncthreads();
            if (wave != 0) continue;
        }
        const uint32_t r = row0 + in_tile, token = fast_quotient(r, a.by_group);
        uint16_t *p = a.out + static_cast<int64_t>(u.first + token) * a.out_token + static_cast<int64_t>(head * a.group + (r - token * a.group)) * a.out_head;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (lane * PER + i < a.dim) p[lane * PER + i] = static_cast<uint16_t>(narrow2_rne(a.bf16, o[i], 0.0f));
        }
    }
}

// The kernel for few query rows, the one for many, and after either what joins its units.
template<bool FP8, int DP>
void launch(const PagedAttentionAmdDescriptor &d, AttentionArgs a, hipStream_t s) {
    const auto shape = [&](const PagedAttentionShape &z) {
        a.tile_rows = z.tile_rows;
        a.by_tile = fast_div(z.tile_rows);
        a.units_each = 1.0f / static_cast<float>(z.target);
        a.rounds_each = z.at_once == 0 ? 0.0f : static_cast<float>(d.cache.kv_heads) / static_cast<float>(z.at_once);
        a.least_rows = z.least;
        a.most_rows = z.most;
        a.least_steps = z.least_steps;
        a.whole_steps = z.whole_steps;
        // the workspace: weights of all slots, then their results
        a.part_out = a.part_stat + 2ull * z.slots * d.cache.kv_heads * z.tile_rows;
        return z.most_units * d.cache.kv_heads;
    };
    // a tile of several units has two at least
    const auto cut_tiles = [&](const PagedAttentionShape &z) {
        const uint32_t cut = z.most_units - z.most_tiles;
        return (cut < z.most_tiles ? cut : z.most_tiles) * d.cache.kv_heads;
    };
    if (d.few.most_tiles != 0) {
        const unsigned units = shape(d.few);
        if constexpr (DP <= 128) {
            if (d.few.tile_rows == 16) paged_attention_rows<FP8, DP, 1><<<units, kWaves * kWave, 0, s>>>(a);
            else paged_attention_rows<FP8, DP, 2><<<units, kWaves * kWave, 0, s>>>(a);
        } else {
            paged_attention_rows<FP8, DP, 1><<<units, kWaves * kWave, 0, s>>>(a);
        }
        const uint32_t rows = d.max_tokens * d.group;
        paged_attention_join<DP><<<dim3(cut_tiles(d.few), rows < 8 ? rows : 8), kWaves * kWave, 0, s>>>(a);
    }
    if (d.many.most_tiles != 0) {
        const unsigned units = shape(d.many);
        amdLaunchPagedAttentionTiles(a, FP8, units, cut_tiles(d.many), s);
    }
}

template<bool FP8>
void launch(const PagedAttentionAmdDescriptor &d, const AttentionArgs &a, hipStream_t s) {
    switch (paged_dim(d.cache.dim)) {
        case 64: return launch<FP8, 64>(d, a, s);
        case 128: return launch<FP8, 128>(d, a, s);
        case 192: return launch<FP8, 192>(d, a, s);
        default: return launch<FP8, 256>(d, a, s);
    }
}

}// namespace

infiniopStatus_t amdPagedAttention(PagedAttentionAmdDescriptor_t desc, void *workspace, uint64_t workspace_size, void *out, void const *q,
                                   void const *k_cache, void const *v_cache, void const *k_scale, void const *v_scale, void const *table,
                                   void const *offsets, void const *lengths, void *stream) {
    const PagedAttentionAmdDescriptor &d = *desc;
    if (d.tokens == 0 || d.rows.rows == 0) {
        return STATUS_SUCCESS;
    }
    if (workspace == nullptr || workspace_size < d.workspace) {
        return STATUS_MEMORY_NOT_ALLOCATED;
    }
    for (const void *p : {static_cast<const void *>(out), q, k_cache, v_cache, k_scale, v_scale, table, offsets, lengths}) {
        if (p == nullptr) return STATUS_BAD_PARAM;
    }
    if (!amd::aligned16(k_cache) || !amd::aligned16(v_cache) || !amd::aligned16(workspace)) {
        return STATUS_BAD_PARAM;
    }
    AMD_CHECK_HIP(hipSetDevice(d.device_id), STATUS_BAD_DEVICE);
    AttentionArgs a{};
    a.rows = amd::RaggedRows{static_cast<const int *>(table), static_cast<const int *>(offsets), static_cast<const int *>(lengths), d.rows.stride,
                             d.rows.rows, d.rows.cols, d.tokens, d.cache.page, amd::fast_div(d.cache.page)};
    a.k = static_cast<const uint8_t *>(k_cache);
    a.v = static_cast<const uint8_t *>(v_cache);
    a.k_scale = static_cast<const float *>(k_scale);
    a.v_scale = static_cast<const float *>(v_scale);
    a.k_at = d.cache.k;
    a.v_at = d.cache.v;
    a.q = static_cast<const uint16_t *>(q);
    a.out = static_cast<uint16_t *>(out);
    a.q_token = d.q_token;
    a.q_head = d.q_head;
    a.out_token = d.out_token;
    a.out_head = d.out_head;
    a.pages = d.cache.pages;
    a.kv_heads = d.cache.kv_heads;
    a.dim = d.cache.dim;
    a.group = d.group;
    a.max_tokens = d.max_tokens;
    a.by_group = amd::fast_div(d.group);
    a.by_block = amd::fast_div(d.cache.block);
    a.scale = d.scale * 1.44269504088896340736f;
    a.bf16 = d.bf16;
    a.part_stat = static_cast<float *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    d.cache.fp8 ? launch<true>(d, a, s) : launch<false>(d, a, s);
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

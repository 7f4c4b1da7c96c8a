// gfx950 KVCacheAppend: new tokens of every row, rounded to 8 bits with a scale
// for each block of tokens and head,
//     scale = max(top / 127, old scale)   or   max(2^ceil(log2(top / 448)), old scale)
//     code  = round(x / scale)
// A wavefront takes one head's k or v of one block of one row (a unit), for a
// scale belongs to exactly one of them: no two wavefronts share a number, and the
// result does not depend on their order.  The power of two makes rescaling e4m3
// codes exact but for what sinks below its smallest normal number.
// Prompts: 2 bytes read, 1 written per value, 8500 tokens of 8 heads x 128 12.7 us, 4.1 TB/s
// where a large element-wise pass reaches 6.2: all workgroups are one round, begin by looking
// for their units, then load, then store, and nothing of one overlaps another.  A few
// tokens: the chain table -> codes (256 rows of one 5.7 us).
#include "../../paged_kernel.h"
#include "kv_cache_append_amd.h"

namespace {

using namespace amd;

constexpr int kAppendWaves = 4;
// 16 values a lane and turn; blocks of up to this many turns stay in registers between the search for the top and the rounding
constexpr int kAppendHeld = 8;

struct AppendArgs {
    RaggedRows rows;
    uint8_t *codes[2];
    float *scales[2];
    const uint16_t *in[2];
    PagedStrides at[2];
    int64_t in_token[2], in_head[2];
    uint32_t pages, heads, dim, block;
    FastDiv by_block, by_vecs;// tokens per block, 16-value vectors per token
    bool by_token;
};

// A row's tokens; of more new ones than it has tokens, the last.
__device__ __forceinline__ RowSpan stored(const AppendArgs &a, uint32_t r) {
    RowSpan s = row_span(a.rows, r);
    if (s.count > s.length) {
        s.first += s.count - s.length;
        s.count = s.length;
    }
    return s;
}
// Units of a row: the blocks that its new tokens touch.
__device__ __forceinline__ uint32_t append_units(const AppendArgs &a, const RowSpan &s) {
    if (s.count == 0) return 0;
    return fast_quotient(s.length - 1, a.by_block) - fast_quotient(s.length - s.count, a.by_block) + 1;
}

template<typename T>
constexpr unsigned short kInfinity = 0;
template<>
constexpr unsigned short kInfinity<F16Ref> = 0x7C00;
template<>
constexpr unsigned short kInfinity<BF16Rne> = 0x7F80;

template<typename T>
__device__ __forceinline__ void widen16(const u32x4 (&w)[2], float (&x)[16]) {
    float lo[8], hi[8];
    widen8<T>(w[0], lo);
    widen8<T>(w[1], hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = lo[i];
        x[i + 8] = hi[i];
    }
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Two magnitudes as 16-bit codes, which are in order of the magnitudes.
__device__ __forceinline__ u16x2 top_codes(const u32x4 (&w)[2], u16x2 top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i / 4][i % 4] & 0x7FFF7FFFu));
    return top;
}
// The same of what is finite.
template<typename T>
__device__ __forceinline__ u16x2 top_finite(const u32x4 (&w)[2], u16x2 top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const u16x2 m = __builtin_bit_cast(u16x2, w[i / 4][i % 4] & 0x7FFF7FFFu);
        top = __builtin_elementwise_max(top, u16x2{m.x < kInfinity<T> ? m.x : static_cast<unsigned short>(0), m.y < kInfinity<T> ? m.y : static_cast<unsigned short>(0)});
    }
    return top;
}

// 16 values times inv, to the nearest code.  ANY: also beyond the codes (to the ends) and NaN (to 0); else the products are
// within the codes, for the scale is at least the top's.
template<bool FP8, bool ANY>
__device__ __forceinline__ u32x4 codes_of(const float (&x)[16], float inv) {
    constexpr float most = FP8 ? 448.0f : 127.0f;
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            y[j] = x[4 * i + j] * inv;
            if constexpr (ANY) y[j] = y[j] == y[j] ? fminf(fmaxf(y[j], -most), most) : 0.0f;
        }
        if constexpr (FP8) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            out[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true));
        } else {
            // 1.5 x 2^23 more, and the sum's rounding has left the whole number in its low bits
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(y[j] + 12582912.0f);
            const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(w[3], w[2], 0x0C0C0400u);
            out[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
        }
    }
    return out;
}

template<bool FP8>
__device__ __forceinline__ void values_of(u32x4 w, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t p = prepare_codes<FP8>(w[i]);
        const f16x2 lo = pair_of<FP8, false>(p), hi = pair_of<FP8, true>(p);
        x[4 * i] = static_cast<float>(lo.x);
        x[4 * i + 1] = static_cast<float>(lo.y);
        x[4 * i + 2] = static_cast<float>(hi.x);
        x[4 * i + 3] = static_cast<float>(hi.y);
    }
}

template<bool FP8>
__device__ __forceinline__ float scale_of(float top) {
    if (top < 0x1p-96f) return 0.0f;
    if constexpr (FP8) {
        // 448 = 1.75 x 2^8: the exponent of top less 8, one more where its mantissa is beyond 1.75
        const uint32_t u = __float_as_uint(top);
        return __uint_as_float(((u >> 23) - 8u + ((u & 0x7FFFFFu) > 0x600000u ? 1u : 0u)) << 23);
    } else {
        return top / 127.0f;
    }
}

// The unit of workgroup `index`: a row's tokens, and the first place of the block.
struct AppendUnit {
    uint32_t row;
    RowSpan span;
    uint32_t from;
};

// Few tokens a row: unit `token` is the block that this token is the first new one of, if it is.  Every wavefront looks
// for the token's row by itself: at first in the row of the token's number, where plain decoding has it.
__device__ __forceinline__ bool unit_of_token(const AppendArgs &a, uint32_t token, AppendUnit *out) {
    const auto has = [&](const RowSpan &s) { return token >= s.first && token - s.first < s.count; };
    out->row = token < a.rows.rows ? token : a.rows.rows - 1;
    out->span = stored(a, out->row);
    if (!has(out->span)) {
        const uint32_t lane = threadIdx.x & (kWave - 1);
        const auto at = [](uint32_t v, int l) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l)); };
        uint64_t hit = 0;
        for (uint32_t r0 = 0; r0 < a.rows.rows && hit == 0; r0 += kWave) {
            const RowSpan s = r0 + lane < a.rows.rows ? stored(a, r0 + lane) : RowSpan{0, 0, 0};
            hit = __builtin_amdgcn_ballot_w64(has(s));
            if (hit != 0) {
                const int l = __builtin_ctzll(hit);
                out->row = r0 + l;
                out->span = RowSpan{at(s.first, l), at(s.count, l), at(s.length, l)};
            }
        }
        if (hit == 0) return false;
    }
    const uint32_t pos = out->span.length - out->span.count + (token - out->span.first);
    out->from = fast_quotient(pos, a.by_block) * a.block;
    return token == out->span.first || pos == out->from;
}

// Many: unit `index` of all rows' blocks in order.
__device__ __forceinline__ bool unit_of_all(const AppendArgs &a, uint32_t index, AppendUnit *out) {
    __shared__ uint64_t slots[kAppendWaves];
    __shared__ AppendUnit found;
    const uint32_t run = (a.rows.rows + kAppendWaves * kWave - 1) / (kAppendWaves * kWave), r0 = threadIdx.x * run;
    uint64_t mine = 0, total;
    for (uint32_t r = r0; r < r0 + run && r < a.rows.rows; ++r) mine += append_units(a, stored(a, r));
    uint64_t before = block_scan64<kAppendWaves>(mine, slots, &total);
    if (index >= total) return false;// the grid holds the most units that so many tokens can make
    if (index >= before && index < before + mine) {
        for (uint32_t r = r0;; ++r) {
            const RowSpan s = stored(a, r);
            const uint32_t n = append_units(a, s);
            if (index < before + n) {
                found = AppendUnit{r, s, (fast_quotient(s.length - s.count, a.by_block) + static_cast<uint32_t>(index - before)) * a.block};
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    const auto same = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); };
    *out = AppendUnit{same(found.row), RowSpan{same(found.span.first), same(found.span.count), same(found.span.length)}, same(found.from)};
    return true;
}

template<typename T, bool FP8, bool HELD>
__global__ __launch_bounds__(kAppendWaves *kWave) void kv_cache_append(AppendArgs a) {
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / kWave)));
    AppendUnit u;
    if (!(a.by_token ? unit_of_token(a, blockIdx.x, &u) : unit_of_all(a, blockIdx.x, &u))) return;
    const uint32_t task = blockIdx.y * kAppendWaves + wave;// k of all heads, then v of all heads
    if (task >= 2 * a.heads) return;// (no barrier below)
    const int kv = task >= a.heads ? 1 : 0;
    const uint32_t head = kv ? task - a.heads : task;
    const RowSpan s = u.span;
    const uint32_t begin = s.length - s.count, from = u.from;
    const uint32_t lo = begin > from ? begin - from : 0, hi = s.length - from < a.block ? s.length - from : a.block;
    const uint32_t col = fast_quotient(from, a.rows.by_page), in_page = from - col * a.rows.page;
    // the new values are asked for before the page is known
    const int64_t step = a.in_token[kv];
    const uint16_t *in = a.in[kv] + (static_cast<int64_t>(s.first) + (from + lo) - begin) * step + static_cast<int64_t>(head) * a.in_head[kv];
    const uint32_t per_token = a.dim / 16, vecs = (hi - lo) * per_token;
    u32x4 held[HELD ? kAppendHeld : 1][2];
    const auto load = [&](uint32_t e, u32x4(&w)[2]) {
        const uint32_t token = fast_quotient(e, a.by_vecs);
        const uint16_t *p = in + token * step + (e - token * per_token) * 16;
        w[0] = ld16_any(p);
        w[1] = ld16_any(p + 8);
    };
    if constexpr (HELD) {
#pragma unroll
        for (int i = 0; i < kAppendHeld; ++i) {
            held[i][0] = held[i][1] = u32x4{0, 0, 0, 0};
            if (lane + i * kWave < vecs) load(lane + i * kWave, held[i]);
        }
    }
    const uint32_t page = static_cast<uint32_t>(a.rows.table[u.row * a.rows.stride + col]);
    if (page >= a.pages) return;
    const PagedStrides at = a.at[kv];
    uint8_t *codes = a.codes[kv] + static_cast<int64_t>(page) * at.page + static_cast<uint64_t>(head) * at.head + static_cast<uint64_t>(in_page) * at.token;
    float *scale = a.scales[kv] + static_cast<int64_t>(page) * at.s_page + static_cast<int64_t>(head) * at.s_head + fast_quotient(in_page, a.by_block);
    const float old = lo != 0 ? *scale : 0.0f;

    // the largest magnitude; where an infinity or NaN is among them, once more without those
    u16x2 tops = {0, 0};
    const auto search = [&](auto of) {
        tops = u16x2{0, 0};
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < kAppendHeld; ++i) tops = of(held[i], tops);
        } else {
            for (uint32_t e = lane; e < vecs; e += kWave) {
                load(e, held[0]);
                tops = of(held[0], tops);
            }
        }
    };
    search([](const u32x4(&w)[2], u16x2 t) { return top_codes(w, t); });
    const bool any = __builtin_amdgcn_ballot_w64(tops.x >= kInfinity<T> || tops.y >= kInfinity<T>) != 0;
    if (any) search([](const u32x4(&w)[2], u16x2 t) { return top_finite<T>(w, t); });
    const float now = fmaxf(scale_of<FP8>(wave_max(fmaxf(T::one(tops.x), T::one(tops.y)))), old);
    const float inv = now > 0.0f ? 1.0f / now : 0.0f;
    if (lo != 0 && now > old) {// the older tokens, to the scale that grew
        const float ratio = old / now;
        for (uint32_t e = lane; e < lo * per_token; e += kWave) {
            const uint32_t token = fast_quotient(e, a.by_vecs);
            uint8_t *p = codes + static_cast<uint64_t>(token) * at.token + (e - token * per_token) * 16;
            float x[16];
            values_of<FP8>(ld16(p), x);
            *reinterpret_cast<u32x4 *>(p) = codes_of<FP8, true>(x, ratio);
        }
    }
    const auto store = [&](uint32_t e, const u32x4(&w)[2]) {
        const uint32_t token = fast_quotient(e, a.by_vecs);
        float x[16];
        widen16<T>(w, x);
        u32x4 c;
        // (a scale below 2^-96 is 0, or an older one that values which count as 0 may exceed, or whose inverse is infinite)
        if (any || now < 0x1p-96f) c = codes_of<FP8, true>(x, inv);
        else c = codes_of<FP8, false>(x, inv);
        *reinterpret_cast<u32x4 *>(codes + static_cast<uint64_t>(lo + token) * at.token + (e - token * per_token) * 16) = c;
    };
    if constexpr (HELD) {
#pragma unroll
        for (int i = 0; i < kAppendHeld; ++i) {
            if (lane + i * kWave < vecs) store(lane + i * kWave, held[i]);
        }
    } else {
        for (uint32_t e = lane; e < vecs; e += kWave) {
            load(e, held[0]);
            store(e, held[0]);
        }
    }
    if (lane == 0) *scale = now;
}

// Decoding: where tokens are not many more than rows, a workgroup for each token looks its row up, without the scan
// over all rows that gives the units of long prompts (256 rows of a token, 8 heads x 128: 8.3 us with the scan, 5.7
// without).  Beyond 1024 rows the look takes longer than the scan.
bool by_token(const KVCacheAppendAmdDescriptor &d) { return d.tokens <= 2ull * d.rows.rows && d.rows.rows <= 1024; }

template<typename T, bool FP8>
void launch(const KVCacheAppendAmdDescriptor &d, AppendArgs &a, hipStream_t stream) {
    // a unit has at least one token, and a row at most two more than its tokens fill
    const uint64_t busy = d.rows.rows < d.tokens ? d.rows.rows : d.tokens;
    const uint64_t most = d.tokens / d.cache.block + 2 * busy;
    a.by_token = by_token(d);
    const dim3 grid(static_cast<unsigned>(a.by_token || most > d.tokens ? d.tokens : most),
                    static_cast<unsigned>(ceil_div(2 * d.cache.kv_heads, kAppendWaves)));
    if (d.cache.block * d.cache.dim <= 16 * kWave * kAppendHeld) {
        kv_cache_append<T, FP8, true><<<grid, kAppendWaves * kWave, 0, stream>>>(a);
    } else {
        kv_cache_append<T, FP8, false><<<grid, kAppendWaves * kWave, 0, stream>>>(a);
    }
}

}// namespace

infiniopStatus_t amdKVCacheAppend(KVCacheAppendAmdDescriptor_t desc, void *k_cache, void *v_cache, void *k_scale, void *v_scale, void const *k,
                                  void const *v, void const *table, void const *offsets, void const *lengths, void *stream) {
    const KVCacheAppendAmdDescriptor &d = *desc;
    if (d.tokens == 0 || d.rows.rows == 0) {
        return STATUS_SUCCESS;
    }
    for (const void *p : {static_cast<const void *>(k_cache), static_cast<const void *>(v_cache), static_cast<const void *>(k_scale),
                          static_cast<const void *>(v_scale), k, v, table, offsets, lengths}) {
        if (p == nullptr) return STATUS_BAD_PARAM;
    }
    if (!amd::aligned16(k_cache) || !amd::aligned16(v_cache)) {
        return STATUS_BAD_PARAM;
    }
    AMD_CHECK_HIP(hipSetDevice(d.device_id), STATUS_BAD_DEVICE);
    AppendArgs a{
        {static_cast<const int *>(table), static_cast<const int *>(offsets), static_cast<const int *>(lengths), d.rows.stride, d.rows.rows, d.rows.cols,
         d.tokens, d.cache.page, amd::fast_div(d.cache.page)},
        {static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache)},
        {static_cast<float *>(k_scale), static_cast<float *>(v_scale)},
        {static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v)},
        {d.cache.k, d.cache.v},
        {d.k_token, d.v_token},
        {d.k_head, d.v_head},
        d.cache.pages,
        d.cache.kv_heads,
        d.cache.dim,
        d.cache.block,
        amd::fast_div(d.cache.block),
        amd::fast_div(d.cache.dim / 16),
        false};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (d.elem == amd::Elem::F16) {
        d.cache.fp8 ? launch<amd::F16Ref, true>(d, a, s) : launch<amd::F16Ref, false>(d, a, s);
    } else {
        d.cache.fp8 ? launch<amd::BF16Rne, true>(d, a, s) : launch<amd::BF16Rne, false>(d, a, s);
    }
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

// gfx950 KVCacheAppend: new tokens of every row, rounded to 8 bits with a scale
// for each block of tokens and head,
//     scale = max(top / 127, old scale)   or   max(2^ceil(log2(top / 448)), old scale)
//     code  = round(x / scale)
// A wavefront takes one head's k or v of one block of one row (a unit), for a
// scale belongs to exactly one of them: no two wavefronts share a number, and the
// result does not depend on their order.  The power of two makes rescaling e4m3
// codes exact but for what sinks below its smallest normal number.
// Bound by HBM for prompts (2 bytes read, 1 written per value), by the chain
// table -> codes for a few tokens.
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

// the largest finite magnitude
template<typename T>
__device__ __forceinline__ float top_of(const u32x4 (&w)[2], float top) {
    float x[16];
    widen16<T>(w, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float m = fabsf(x[i]);
        top = fmaxf(top, m < __builtin_inff() ? m : 0.0f);
    }
    return top;
}

// 16 values times inv, to the nearest code; NaN to 0, infinities to the ends
template<bool FP8>
__device__ __forceinline__ u32x4 codes_of(const float (&x)[16], float inv) {
    constexpr float most = FP8 ? 448.0f : 127.0f;
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v = x[4 * i + j] * inv;
            y[j] = v == v ? fminf(fmaxf(v, -most), most) : 0.0f;
        }
        if constexpr (FP8) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            out[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true));
        } else {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) w |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(y[j]))) & 0xFFu) << (8 * j);
            out[i] = w;
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

template<typename T, bool FP8, bool HELD>
__global__ __launch_bounds__(kAppendWaves *kWave) void kv_cache_append(AppendArgs a) {
    __shared__ uint64_t slots[kAppendWaves];
    __shared__ uint32_t found[2];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1);
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid / kWave)));
    // which row and block: the unit's place among those of all rows, each lane a run of neighbouring rows
    const uint32_t run = (a.rows.rows + kAppendWaves * kWave - 1) / (kAppendWaves * kWave), r0 = tid * run;
    uint64_t mine = 0, total;
    for (uint32_t r = r0; r < r0 + run && r < a.rows.rows; ++r) mine += append_units(a, stored(a, r));
    uint64_t before = block_scan64<kAppendWaves>(mine, slots, &total);
    const uint32_t unit = blockIdx.x;
    if (unit >= total) return;// the grid holds the most units that so many tokens can make
    if (unit >= before && unit < before + mine) {
        uint32_t r = r0;
        for (;; ++r) {
            const uint32_t n = append_units(a, stored(a, r));
            if (unit < before + n) break;
            before += n;
        }
        found[0] = r;
        found[1] = static_cast<uint32_t>(unit - before);
    }
    __syncthreads();
    const uint32_t row = __builtin_amdgcn_readfirstlane(found[0]);
    const uint32_t task = blockIdx.y * kAppendWaves + wave;// k of all heads, then v of all heads
    if (task >= 2 * a.heads) return;// (no barrier below)
    const int kv = task >= a.heads ? 1 : 0;
    const uint32_t head = kv ? task - a.heads : task;
    const RowSpan s = stored(a, row);
    const uint32_t begin = s.length - s.count;
    const uint32_t from = (fast_quotient(begin, a.by_block) + found[1]) * a.block;// the block's first place
    const uint32_t lo = begin > from ? begin - from : 0, hi = s.length - from < a.block ? s.length - from : a.block;
    const uint32_t col = fast_quotient(from, a.rows.by_page), in_page = from - col * a.rows.page;
    const uint32_t page = static_cast<uint32_t>(a.rows.table[row * a.rows.stride + col]);
    if (page >= a.pages) return;
    const PagedStrides at = a.at[kv];
    uint8_t *codes = a.codes[kv] + static_cast<int64_t>(page) * at.page + static_cast<uint64_t>(head) * at.head + static_cast<uint64_t>(in_page) * at.token;
    float *scale = a.scales[kv] + static_cast<int64_t>(page) * at.s_page + static_cast<int64_t>(head) * at.s_head + fast_quotient(in_page, a.by_block);
    const int64_t step = a.in_token[kv];
    const uint16_t *in = a.in[kv] + (static_cast<int64_t>(s.first) + (from + lo) - begin) * step + static_cast<int64_t>(head) * a.in_head[kv];
    const float old = lo != 0 ? *scale : 0.0f;
    const uint32_t per_token = a.dim / 16, vecs = (hi - lo) * per_token;

    u32x4 held[HELD ? kAppendHeld : 1][2];
    float top = 0.0f;
    const auto load = [&](uint32_t e, u32x4(&w)[2]) {
        const uint32_t token = fast_quotient(e, a.by_vecs);
        const uint16_t *p = in + token * step + (e - token * per_token) * 16;
        w[0] = ld16_any(p);
        w[1] = ld16_any(p + 8);
    };
    if constexpr (HELD) {
#pragma unroll
        for (int i = 0; i < kAppendHeld; ++i) {
            if (lane + i * kWave < vecs) load(lane + i * kWave, held[i]);
        }
#pragma unroll
        for (int i = 0; i < kAppendHeld; ++i) {
            if (lane + i * kWave < vecs) top = top_of<T>(held[i], top);
        }
    } else {
        for (uint32_t e = lane; e < vecs; e += kWave) {
            load(e, held[0]);
            top = top_of<T>(held[0], top);
        }
    }
    const float now = fmaxf(scale_of<FP8>(wave_max(top)), old);
    const float inv = now > 0.0f ? 1.0f / now : 0.0f;
    if (lo != 0 && now > old) {// the older tokens, to the scale that grew
        const float ratio = old / now;
        for (uint32_t e = lane; e < lo * per_token; e += kWave) {
            const uint32_t token = fast_quotient(e, a.by_vecs);
            uint8_t *p = codes + static_cast<uint64_t>(token) * at.token + (e - token * per_token) * 16;
            float x[16];
            values_of<FP8>(ld16(p), x);
            *reinterpret_cast<u32x4 *>(p) = codes_of<FP8>(x, ratio);
        }
    }
    const auto store = [&](uint32_t e, const u32x4(&w)[2]) {
        const uint32_t token = fast_quotient(e, a.by_vecs);
        float x[16];
        widen16<T>(w, x);
        *reinterpret_cast<u32x4 *>(codes + static_cast<uint64_t>(lo + token) * at.token + (e - token * per_token) * 16) = codes_of<FP8>(x, inv);
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

template<typename T, bool FP8>
void launch(const KVCacheAppendAmdDescriptor &d, const AppendArgs &a, hipStream_t stream) {
    // a unit has at least one token, and a row at most two more than its tokens fill
    const uint64_t busy = d.rows.rows < d.tokens ? d.rows.rows : d.tokens;
    const uint64_t most = d.tokens / d.cache.block + 2 * busy;
    const dim3 grid(static_cast<unsigned>(most < d.tokens ? most : d.tokens), static_cast<unsigned>(ceil_div(2 * d.cache.kv_heads, kAppendWaves)));
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
    const AppendArgs a{
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
        amd::fast_div(d.cache.dim / 16)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (d.elem == amd::Elem::F16) {
        d.cache.fp8 ? launch<amd::F16Ref, true>(d, a, s) : launch<amd::F16Ref, false>(d, a, s);
    } else {
        d.cache.fp8 ? launch<amd::BF16Rne, true>(d, a, s) : launch<amd::BF16Rne, false>(d, a, s);
    }
    AMD_CHECK_HIP(hipGetLastError(), STATUS_EXECUTION_FAILED);
    return STATUS_SUCCESS;
}

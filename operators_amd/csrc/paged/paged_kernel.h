// Device-side pieces that the kernels of the paged cache share: the rows of a
// ragged batch, whole-number sums and scans over a workgroup, and 8-bit codes as
// fp16 pairs.  Include from .hip files only.
#ifndef INFINIOP_AMD_PAGED_KERNEL_H
#define INFINIOP_AMD_PAGED_KERNEL_H

#include "../devices/amd/kernel_amd.h"
#include "paged_cache.h"

namespace amd {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 __attribute__((aligned(2))) u32x2_any;
typedef float f32x16 __attribute__((ext_vector_type(16)));

// ---- the rows of a batch ----------------------------------------------------
struct RaggedRows {
    const int *table;// [rows, cols]
    const int *offsets, *lengths;
    int64_t stride;// of the table
    uint32_t rows, cols, tokens, page;
    FastDiv by_page;
};

// Row r's new tokens [first, first + count) of the call and its length with
// them, brought into range whatever the arrays hold: tokens within the call's,
// a length within the table.
struct RowSpan {
    uint32_t first, count, length;
};
__device__ __forceinline__ RowSpan row_span(const RaggedRows &b, uint32_t r) {
    const int tokens = static_cast<int>(b.tokens), room = static_cast<int>(b.cols * b.page);// < 2^31
    const int from = b.offsets[r], to = b.offsets[r + 1], len = b.lengths[r];
    const int lo = from < 0 ? 0 : from > tokens ? tokens : from, hi = to < lo ? lo : to > tokens ? tokens : to;
    return RowSpan{static_cast<uint32_t>(lo), static_cast<uint32_t>(hi - lo), static_cast<uint32_t>(len < 0 ? 0 : len > room ? room : len)};
}

// ---- within a wavefront, without LDS --------------------------------------------
// Sum of this lane's value and all lower lanes'.
template<int CTRL, int ROWS>
__device__ __forceinline__ uint32_t from_lane(uint32_t v) {// 0 where there is none
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
template<int CTRL, int ROWS>
__device__ __forceinline__ uint64_t from_lane(uint64_t v) {
    return from_lane<CTRL, ROWS>(static_cast<uint32_t>(v)) | static_cast<uint64_t>(from_lane<CTRL, ROWS>(static_cast<uint32_t>(v >> 32))) << 32;
}
template<typename U>
__device__ __forceinline__ U wave_scan(U v) {
    v += from_lane<0x111, 0xF>(v);       // row_shr:1
    v += from_lane<0x112, 0xF>(v);       // row_shr:2
    v += from_lane<0x114, 0xF>(v);       // row_shr:4
    v += from_lane<0x118, 0xF>(v);       // row_shr:8
    v += from_lane<0x142, 0xA>(v);       // row_bcast:15 -> rows 1, 3
    return v + from_lane<0x143, 0xC>(v); // row_bcast:31 -> rows 2, 3
}
// Lanes 16 and 32 apart, by exchanging rows of 16 lanes between two copies.
template<typename F>
__device__ __forceinline__ float across16(float v, F both) {
    const auto two = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return both(__uint_as_float(two[0]), __uint_as_float(two[1]));
}
template<typename F>
__device__ __forceinline__ float across32(float v, F both) {
    const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return both(__uint_as_float(two[0]), __uint_as_float(two[1]));
}

// ---- whole-number sums over a workgroup of WAVES wavefronts --------------------
// slots: LDS, WAVES values; one use of it has to end with a barrier before the next begins.
// The sum of the lower lanes' values (exclusive), and of all in `total`.
template<int WAVES>
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t *slots, uint64_t *total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint64_t sum = wave_scan(v);
    if (lane == kWave - 1) slots[wave] = sum;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        if (i < wave) before += slots[i];
        all += slots[i];
    }
    __syncthreads();
    *total = all;
    return before + sum - v;
}

// The largest of all lanes' values, which are not below 0.
template<int WAVES>
__device__ __forceinline__ float block_max(float v, uint64_t *slots) {
    v = wave_max(v);
    if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = __float_as_uint(v);
    __syncthreads();
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) top = fmaxf(top, __uint_as_float(static_cast<uint32_t>(slots[i])));
    __syncthreads();
    return top;
}

// ---- codes as fp16 ------------------------------------------------------------
// Both types are exact in fp16: whole numbers up to 128, and e4m3.
// An int8 with its sign bit turned over, as the low byte of 0x64xx, is the fp16
// number 1024 + 128 + value; one packed subtraction leaves the value.
__device__ __forceinline__ f16x2 bias_off(uint32_t pair) {
    return __builtin_bit_cast(f16x2, pair) + f16x2{static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
}
// int8 codes come with their sign bits turned over (prepare_codes)
template<bool FP8>
__device__ __forceinline__ uint32_t prepare_codes(uint32_t w) {
    return FP8 ? w : w ^ 0x80808080u;
}
// bytes 2 * HI and 2 * HI + 1 of a word
template<bool FP8, bool HI>
__device__ __forceinline__ f16x2 pair_of(uint32_t w) {
    if constexpr (FP8) {
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI);
    } else {
        return bias_off(__builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u));
    }
}

}// namespace amd

#endif

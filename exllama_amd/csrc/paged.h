// Shared pieces of the paged 8-bit key / value cache (paged.hip: block tables, slot maps and the append; paged_attention.hip).
//
// A page holds `block` tokens of one kv head: keys [blocks, kv_heads, block, hd16], values [blocks, kv_heads, hd16, block], hd16 =
// head_dim rounded up to 16 (the pad holds zeros), codes in e4m3 or int8, one scale per (page, head): x = code * scale.  Values lie
// with their TOKENS next to each other: the second product of attention reads 16 keys of one column as one 16-byte load, the
// MFMA operand as it is, and the append pays the transposition once.  Scales are powers of two: dividing by one is exact, so a code is
// ONE rounding of the exact value, growing a page's scale only shifts exponents, and the conversion instructions apply the scale
// for free.
#pragma once
#include "common.h"


// The scale's exponents.  Lower end: one step of the codes at this scale is fp16's own quantum (2^-24); upper end: the largest code
// stays a finite fp16 (448 * 2^7 = 57344, 127 * 2^9 = 65024; larger inputs saturate there).
template <int CODE> struct PagedRange;
template <> struct PagedRange<EXL_PAGE_FP8>  { static constexpr int lo = -15, hi = 7, top_exp = 8, top_mant = 0x600000; static constexpr float top = 448.f; };
template <> struct PagedRange<EXL_PAGE_INT8> { static constexpr int lo = -24, hi = 9, top_exp = 6, top_mant = 0x7e0000; static constexpr float top = 127.f; };

#ifdef __HIPCC__
typedef f16x4 f16x4_a4 __attribute__((aligned(4)));       // head_dim % 8 != 0: rows of a head are only 4- or 8-byte aligned
typedef f16x8 f16x8_a8 __attribute__((aligned(8)));
typedef f16x4 f16x4_a2 __attribute__((aligned(2)));       // sin and cos may begin anywhere
typedef f16x8 f16x8_a2 __attribute__((aligned(2)));

__device__ __forceinline__ float paged_pow2(int e) { return __uint_as_float((uint32_t) (e + 127) << 23); }

// the exponent of a scale in memory, brought into the range (whatever the memory holds)
template <int CODE> __device__ __forceinline__ int paged_scale_exp(float s)
{
    const int e = (int) ((__float_as_uint(s) >> 23) & 255) - 127;
    return min(max(e, PagedRange<CODE>::lo), PagedRange<CODE>::hi);
}

// the least e with amax <= top * 2^e, in the range: top = 1.75 * 2^8 or 1.984375 * 2^6, so the mantissa decides exactly
template <int CODE> __device__ __forceinline__ int paged_exp_for(float amax)
{
    typedef PagedRange<CODE> R;
    const uint32_t u = __float_as_uint(amax);
    const int e = (int) (u >> 23) - 127 - R::top_exp + ((int) (u & 0x7fffff) > R::top_mant ? 1 : 0);
    return min(max(e, R::lo), R::hi);
}

// four codes of x * inv, inv = 1 / scale: one rounding to nearest even; NaN stays NaN (e4m3) or becomes 0 (int8).  |x| * inv <= top, unless
// SATURATE (one instruction or two for a number where every comparison counts: the clamp is for pages with numbers beyond the last scale's)
template <int CODE, bool SATURATE> __device__ __forceinline__ uint32_t paged_encode4(float a, float b, float c, float d, float inv)
{
    if (SATURATE) {
        const float t = PagedRange<CODE>::top / inv;
        auto clamp = [&](float y) { return y > t ? t : y < -t ? -t : y; };
        a = clamp(a); b = clamp(b); c = clamp(c); d = clamp(d);
    }
    if (CODE == EXL_PAGE_FP8) {
        const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
        return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true);
    }
    // 1.5 * 2^23 + y has the nearest whole number in its low byte (two's complement); a NaN of fp16 or fp32 arithmetic has zeros there
    const float base = 12582912.f;
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(fmaf(b, inv, base)), __float_as_uint(fmaf(a, inv, base)), 0x0c0c0400u);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(fmaf(d, inv, base)), __float_as_uint(fmaf(c, inv, base)), 0x04000c0cu);
    return ab | cd;
}

// the four numbers of a word of codes
template <int CODE> __device__ __forceinline__ void paged_decode4(uint32_t w, float (&x)[4])
{
    if (CODE == EXL_PAGE_FP8) {
        x[0] = __builtin_amdgcn_cvt_f32_fp8((int) w, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8((int) w, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8((int) w, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8((int) w, 3);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float) (int) (int8_t) (w >> (8 * i));
    }
}
#endif

int paged_check_block(const char* what, int block_size, int num_blocks);
int paged_check_head(const char* what, int code, int head_dim);

// What a paged cache of keys and values holds, and where: rows [pages][heads][page][head dim] of int8, e4m3 or 16-bit values,
// for the 8-bit kinds with one float a row [pages][heads][page].  Head-major pages: 32 rows of a head, what one step of the
// attention reads, are one contiguous piece.
#pragma once

#include "bsa_device.hpp"

namespace bsa {

enum CacheKind : int { CACHE_16 = 0, CACHE_INT8 = 1, CACHE_E4M3 = 2 };
__host__ __device__ constexpr int cache_value_bytes(int kind) { return kind == CACHE_16 ? 2 : 1; }

// row of (slot, head), in rows of head_dim values; slot = page * page size + place
__device__ __forceinline__ long long cache_row(long long slot, int head, int heads, int page_shift)
{
    const long long page = slot >> page_shift;
    return ((page * heads + head) << page_shift) + (slot & ((1ll << page_shift) - 1));
}

// four values to the nearest of the cache's type, ties to even; |y| is at most 127 or 448
template <int KIND>
__device__ __forceinline__ unsigned narrow_held(float y0, float y1, float y2, float y3)
{
    if (KIND == CACHE_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y2, y3, w, true);
    }
    // adding 1.5 * 2^23 rounds to a whole number, whose two's complement is in the low byte
    const float magic = 12582912.f;
    const unsigned a = __float_as_uint(y0 + magic), b = __float_as_uint(y1 + magic), c = __float_as_uint(y2 + magic),
                   d = __float_as_uint(y3 + magic);
    const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return lo | (hi << 16);
}

template <int KIND>
__device__ __forceinline__ void widen_held(unsigned w, float *y)
{
    if (KIND == CACHE_E4M3) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        y[0] = lo.x, y[1] = lo.y, y[2] = hi.x, y[3] = hi.y;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (float)((int)(w << (24 - 8 * j)) >> 24);
}

// 8 values as 16-bit ones, all of them exactly
template <bool BF, int KIND>
__device__ __forceinline__ h8 widen_held_16(unsigned lo, unsigned hi)
{
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const unsigned w[2] = {lo, hi};
    unsigned o[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (KIND == CACHE_E4M3) {                // the conversion's own scale is 1
            if (BF) {
                o[2 * j] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j], 1.f, false));
                o[2 * j + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j], 1.f, true));
            } else {
                o[2 * j] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[j], 1.f, false));
                o[2 * j + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[j], 1.f, true));
            }
        } else if (BF) {
            float y[4];
            widen_held<KIND>(w[j], y);
            o[2 * j] = __builtin_bit_cast(unsigned, b2{(__bf16)y[0], (__bf16)y[1]});
            o[2 * j + 1] = __builtin_bit_cast(unsigned, b2{(__bf16)y[2], (__bf16)y[3]});
        } else {                                 // x + 128 in the low bits of 1024, less 1152
            const unsigned u = w[j] ^ 0x80808080u;
            const h2 off = {(half_t)-1152.f, (half_t)-1152.f};
            o[2 * j] = __builtin_bit_cast(unsigned, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
            o[2 * j + 1] = __builtin_bit_cast(unsigned, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
        }
    }
    return __builtin_bit_cast(h8, make_uint4(o[0], o[1], o[2], o[3]));
}

}  // namespace bsa

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

}  // namespace bsa

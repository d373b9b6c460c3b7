// Rows of keys and values into a paged cache and back out of it, quantised on the way in: one scale per token and head,
//   s = max |x| / top,   y = x top / max |x| rounded to the nearest value of the cache's type (ties to even),   x' = y s
// with top = 127 (int8) or 448 (e4m3); a 16-bit cache holds the rows as they are.  A row of zeros has scale 0; one that holds an
// infinity or a NaN has scale NaN and zeros, so that it reads back as NaN.
//
// The quotient is the exact one wherever that decides the rounding: x top has at most 20 significant bits and the
// maximum 11, so it either is a tie exactly, and then an fp32 value, or is further than 2^-19 of itself from every tie.  A
// reciprocal within one unit and one correction by the remainder (exact in a fused multiply-add) give the first kind to the
// bit and the second within one unit: three operations a value instead of a division's ten.
//
// What bounds it: 16 bytes a lane in, 8 out, 3 operations and a conversion a value between them: memory.  A row is 8 or 16
// lanes, which share its maximum in 3 or 4 exchanges; key and value rows of a token and head go together.  65521 tokens of 8 heads at
// head dim 64, written as int8 and read back: 69 us, 5.7 TB/s, where a copy of 1 GiB reaches 5.2 (part of it is still in the last
// cache); 8191 tokens in and out as e4m3 21 us, 4.7 TB/s; 48 rows 3.3 us: a launch.
#include "bsa_device.hpp"
#include "bsa_internal.hpp"
#include "cache_values.hpp"
#include "../../include/bsa.h"

namespace bsa {

namespace {

// one piece: 8 values of a row of HD, HD / 8 lanes a row
template <int HD, bool BF, int KIND>
__device__ __forceinline__ void quantise_piece(uint4 raw, uint2 &held, float &scale)
{
    const h8 x = as_h8(raw);
    unsigned top = 0;                            // largest magnitude, as the bits of a 16-bit value: NaN is above infinity
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned lo = w[j] & 0x7FFFu, hi = (w[j] >> 16) & 0x7FFFu;
        top = max(top, max(lo, hi));
    }
#pragma unroll
    for (int d = 1; d < HD / 8; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
    constexpr unsigned INFINITE = BF ? 0x7F80u : 0x7C00u;
    const float amax = widen_16<BF>(__builtin_bit_cast(half_t, (unsigned short)top));
    if (top >= INFINITE) {
        held = make_uint2(0, 0);
        scale = __builtin_nanf("");
        return;
    }
    constexpr float TOP = KIND == CACHE_INT8 ? 127.f : 448.f;
    scale = amax / TOP;
    // bf16 reaches where x TOP overflows and where the reciprocal of a maximum does
    const float unit = amax >= 0x1p64f ? 0x1p-64f : amax < 0x1p-64f ? 0x1p64f : 1.f;
    const float b = amax == 0.f ? 1.f : amax * unit, inv = __builtin_amdgcn_rcpf(b);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float a = widen_16<BF>(x[j]) * unit * TOP, y0 = a * inv;
        y[j] = __builtin_fmaf(__builtin_fmaf(-y0, b, a), inv, y0);
    }
    held = make_uint2(narrow_held<KIND>(y[0], y[1], y[2], y[3]), narrow_held<KIND>(y[4], y[5], y[6], y[7]));
}

template <int HD, bool BF, int KIND>
__global__ __launch_bounds__(256) void cache_write_kernel(
    const half_t *__restrict__ k, const half_t *__restrict__ v, const int32_t *__restrict__ slots, unsigned char *__restrict__ keys,
    unsigned char *__restrict__ values, float *__restrict__ key_scales, float *__restrict__ value_scales, long long rows, int heads,
    long long places, int page_shift, long long k_token, long long k_head, long long v_token, long long v_head)
{
    constexpr int LANES = HD / 8, WIDTH = cache_value_bytes(KIND);
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int piece = (int)(threadIdx.x % LANES);
    if (row >= rows) return;                     // whole rows of lanes leave together
    const long long token = row / heads;
    const int head = (int)(row - token * heads);
    const long long slot = slots[token];
    if (slot < 0 || slot >= places) return;
    const uint4 kr = ldg16(k + token * k_token + head * k_head + 8 * piece), vr = ldg16(v + token * v_token + head * v_head + 8 * piece);
    const long long at = cache_row(slot, head, heads, page_shift);
    const long long byte = (at * HD + 8 * piece) * WIDTH;
    if (KIND == CACHE_16) {
        stg16(keys + byte, kr);
        stg16(values + byte, vr);
        return;
    }
    uint2 kh, vh;
    float ks, vs;
    quantise_piece<HD, BF, KIND>(kr, kh, ks);
    quantise_piece<HD, BF, KIND>(vr, vh, vs);
    *reinterpret_cast<uint2 *>(keys + byte) = kh;
    *reinterpret_cast<uint2 *>(values + byte) = vh;
    if (piece == 0) {
        key_scales[at] = ks;
        value_scales[at] = vs;
    }
}

// What is read back leaves without a place in the caches: it would drive out the rows that the next calls read (65521 tokens in and out
// 69 us of kernels, with ordinary stores 91; 8191 21.0 and 21.7).  Streaming the write's loads as well gives 76 and 19.9.
// TO: 0 fp32, 1 fp16, 2 bf16 (the numbers of the ABI); FROM_BF: what a 16-bit cache holds
template <int TO>
__device__ __forceinline__ void store_values(void *out, long long at, const float (&y)[8])
{
    if (TO == BSA_F32) {
        float *p = reinterpret_cast<float *>(out) + at;
        stg16_stream(p, __builtin_bit_cast(uint4, make_float4(y[0], y[1], y[2], y[3])));
        stg16_stream(p + 4, __builtin_bit_cast(uint4, make_float4(y[4], y[5], y[6], y[7])));
    } else {
        h8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = narrow_16<TO == BSA_BF16>(y[j]);
        stg16_stream(reinterpret_cast<half_t *>(out) + at, __builtin_bit_cast(uint4, o));
    }
}

template <int HD, int TO, bool FROM_BF, int KIND>
__global__ __launch_bounds__(256) void cache_read_kernel(
    const unsigned char *__restrict__ keys, const unsigned char *__restrict__ values, const float *__restrict__ key_scales,
    const float *__restrict__ value_scales, const int32_t *__restrict__ slots, void *__restrict__ k_out, void *__restrict__ v_out,
    long long rows, int heads, long long places, int page_shift)
{
    constexpr int LANES = HD / 8, WIDTH = cache_value_bytes(KIND);
    const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int piece = (int)(threadIdx.x % LANES);
    if (row >= rows) return;
    const long long token = row / heads;
    const int head = (int)(row - token * heads);
    const long long slot = slots[token];
    const bool there = slot >= 0 && slot < places;
    float ky[8], vy[8];
    if (there) {
        const long long at = cache_row(slot, head, heads, page_shift), byte = (at * HD + 8 * piece) * WIDTH;
        if (KIND == CACHE_16) {
            const h8 a = as_h8(ldg16(keys + byte)), b = as_h8(ldg16(values + byte));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ky[j] = widen_16<FROM_BF>(a[j]);
                vy[j] = widen_16<FROM_BF>(b[j]);
            }
        } else {
            const uint2 a = *reinterpret_cast<const uint2 *>(keys + byte), b = *reinterpret_cast<const uint2 *>(values + byte);
            const float ks = key_scales[at], vs = value_scales[at];
            widen_held<KIND>(a.x, ky), widen_held<KIND>(a.y, ky + 4);
            widen_held<KIND>(b.x, vy), widen_held<KIND>(b.y, vy + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ky[j] *= ks;
                vy[j] *= vs;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) ky[j] = vy[j] = 0.f;
    }
    store_values<TO>(k_out, row * HD + 8 * piece, ky);
    store_values<TO>(v_out, row * HD + 8 * piece, vy);
}

unsigned cache_grid(const CacheRowsArgs &p)
{
    return (unsigned)(((long long)p.tokens * p.heads * (p.head_dim / 8) + 255) / 256);
}

template <int HD, bool BF, int KIND>
hipError_t write_rows(const CacheRowsArgs &p, hipStream_t st)
{
    cache_write_kernel<HD, BF, KIND><<<cache_grid(p), 256, 0, st>>>(
        (const half_t *)p.k, (const half_t *)p.v, p.slots, (unsigned char *)p.keys, (unsigned char *)p.values, p.key_scales,
        p.value_scales, (long long)p.tokens * p.heads, p.heads, (long long)p.pages << p.page_shift, p.page_shift, p.k_token,
        p.k_head, p.v_token, p.v_head);
    return hipGetLastError();
}
template <int HD, bool BF>
hipError_t write_rows_of(const CacheRowsArgs &p, hipStream_t st)
{
    if (p.kind == CACHE_INT8) return write_rows<HD, BF, CACHE_INT8>(p, st);
    if (p.kind == CACHE_E4M3) return write_rows<HD, BF, CACHE_E4M3>(p, st);
    return write_rows<HD, BF, CACHE_16>(p, st);
}

template <int HD, int TO, bool FROM_BF, int KIND>
hipError_t read_rows(const CacheRowsArgs &p, hipStream_t st)
{
    cache_read_kernel<HD, TO, FROM_BF, KIND><<<cache_grid(p), 256, 0, st>>>(
        (const unsigned char *)p.keys, (const unsigned char *)p.values, p.key_scales, p.value_scales, p.slots, (void *)p.k,
        (void *)p.v, (long long)p.tokens * p.heads, p.heads, (long long)p.pages << p.page_shift, p.page_shift);
    return hipGetLastError();
}
template <int HD, int TO>
hipError_t read_rows_of(const CacheRowsArgs &p, hipStream_t st)
{
    if (p.kind == CACHE_INT8) return read_rows<HD, TO, false, CACHE_INT8>(p, st);
    if (p.kind == CACHE_E4M3) return read_rows<HD, TO, false, CACHE_E4M3>(p, st);
    return p.held_bf16 ? read_rows<HD, TO, true, CACHE_16>(p, st) : read_rows<HD, TO, false, CACHE_16>(p, st);
}

}  // namespace

hipError_t launch_cache_write(int dtype, const CacheRowsArgs &p, hipStream_t st)
{
    if (p.head_dim == 64) return dtype == BSA_BF16 ? write_rows_of<64, true>(p, st) : write_rows_of<64, false>(p, st);
    return dtype == BSA_BF16 ? write_rows_of<128, true>(p, st) : write_rows_of<128, false>(p, st);
}

hipError_t launch_cache_read(int dtype, const CacheRowsArgs &p, hipStream_t st)
{
    if (p.head_dim == 64)
        return dtype == BSA_F32 ? read_rows_of<64, BSA_F32>(p, st) : dtype == BSA_F16 ? read_rows_of<64, BSA_F16>(p, st)
                                                                                      : read_rows_of<64, BSA_BF16>(p, st);
    return dtype == BSA_F32 ? read_rows_of<128, BSA_F32>(p, st) : dtype == BSA_F16 ? read_rows_of<128, BSA_F16>(p, st)
                                                                                   : read_rows_of<128, BSA_BF16>(p, st);
}

}  // namespace bsa

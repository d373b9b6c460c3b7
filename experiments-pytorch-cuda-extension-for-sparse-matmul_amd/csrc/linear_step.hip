// One token of every sequence against its recurrent state, in place:  S <- l S + k v^T,  o = scale q S.
//
// What bounds it: the state, 4 D^2 bytes a sequence and key head, read and written once; 3 to 4 operations a value.  250 sequences, 16 key heads,
// head dim 128: 524 MB in 84 to 88 us, 6.0 TB/s; 3 sequences, 4 heads, head dim 64: 3.2 us.  A workgroup has COLUMNS
// columns of one state, 16 bytes a lane, every lane all its loads in flight at once; the query heads of a key head share the pass.
// Results of the rows that different lanes have add up in LDS.
#include "bsa_device.hpp"
#include "bsa_internal.hpp"
#include "../../include/bsa.h"

namespace bsa {

namespace {

constexpr int STEP_HEADS = 4;            // query heads of a pass over the registers

template <int HD, int COLUMNS, bool BF>
__global__ __launch_bounds__(256) void linear_step_kernel(LinearStepArgs p)
{
    constexpr int LANES = COLUMNS / 4, ROWS = 256 / LANES, PER = HD / ROWS;      // lanes of a row, rows side by side, rows of a lane
    __shared__ float part[STEP_HEADS][ROWS][COLUMNS + 4];
    const int b = (int)blockIdx.z, key_head = (int)blockIdx.y, col0 = (int)blockIdx.x * COLUMNS;
    const int c = (int)threadIdx.x % LANES, r0 = (int)threadIdx.x / LANES, group = p.heads / p.key_heads;
    const int slot = p.at[b];
    half_t *const out = (half_t *)p.out + ((size_t)b * p.heads + (size_t)key_head * group) * HD + col0;
    if (slot < 0 || slot >= p.slots) {
        for (int i = (int)threadIdx.x; i < group * LANES; i += 256)
            *reinterpret_cast<uint2 *>(out + (size_t)(i / LANES) * HD + 4 * (i % LANES)) = make_uint2(0, 0);
        return;
    }
    float *const state = p.states + ((size_t)slot * p.key_heads + key_head) * HD * HD + col0 + 4 * c;
    const half_t *k = (const half_t *)p.k + b * p.k_token + key_head * p.k_head, *v = (const half_t *)p.v + b * p.v_token + key_head * p.v_head + col0 + 4 * c;
    f4v s[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = *reinterpret_cast<const f4v *>(state + (size_t)(r0 + ROWS * j) * HD);
    const float decay = __builtin_amdgcn_exp2f(p.log_decay[key_head] * 1.4426950408889634f);
    const h4 raw = *reinterpret_cast<const h4 *>(v);
    f4v value;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const half_t one = raw[e];
        value[e] = widen_16<BF>(one);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const float key = widen_16<BF>(k[r0 + ROWS * j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = __builtin_fmaf(decay, s[j][e], key * value[e]);
        *reinterpret_cast<f4v *>(state + (size_t)(r0 + ROWS * j) * HD) = s[j];
    }
    for (int g0 = 0; g0 < group; g0 += STEP_HEADS) {
        const int heads = min(STEP_HEADS, group - g0);
        for (int g = 0; g < heads; ++g) {
            const half_t *q = (const half_t *)p.q + b * p.q_token + (key_head * group + g0 + g) * p.q_head;
            f4v sum = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const float query = widen_16<BF>(q[r0 + ROWS * j]);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(query, s[j][e], sum[e]);
            }
            *reinterpret_cast<f4v *>(&part[g][r0][4 * c]) = sum;
        }
        __syncthreads();
        for (int i = (int)threadIdx.x; i < heads * COLUMNS; i += 256) {
            const int g = i / COLUMNS, at = i % COLUMNS;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) sum += part[g][r][at];
            out[(size_t)(g0 + g) * HD + at] = narrow_16<BF>(p.scale * sum);
        }
        __syncthreads();
    }
}

template <int HD, bool BF>
hipError_t step(const LinearStepArgs &p, hipStream_t st)
{
    linear_step_kernel<HD, 64, BF><<<dim3(HD / 64, p.key_heads, p.batch), 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_linear_step(const LinearStepArgs &p, hipStream_t st)
{
    if (p.head_dim == 64) return p.bf16 ? step<64, true>(p, st) : step<64, false>(p, st);
    return p.bf16 ? step<128, true>(p, st) : step<128, false>(p, st);
}

}  // namespace bsa

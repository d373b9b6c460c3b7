// Linear attention with a decay for each key head over sequences packed along the tokens, and its gradients:
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   l = exp(log_decay), S_0 given or zero.
//
// Chunks of 32 tokens: with a, b, c for q, k, v and P_ts = scale l^(t-s) (a_t . b_s) for s <= t inside the chunk,
//   o_t = sum_s P_ts c_s + scale l^(t+1) a_t S,      S <- l^32 S + sum_s l^(31-s) b_s c_s^T.
// The gradients are the same sum over other operands and, for dk and dv, from the end of the sequence (R: what dk and dv take the place of S):
//   dq: a, b, c = dO, V, K (the state is S^T);   dv: K, Q, dO backwards;   dk: V, dO, Q backwards (R^T).
//
// A sequence is cut into segments of p.segment tokens.  One workgroup walks a segment of one head, its wave w has columns 32 w .. of c and of
// the state, which stays in fp32 accumulators from chunk to chunk.  Where a sequence has several segments, two launches in front make
// the state that each begins with: every segment's own sum, then the running sum over segments.  Chunks travel
// straight to LDS two steps ahead of their use, in a ring of three.
#include "attention_tiles.hpp"
#include "bsa_device.hpp"
#include "bsa_internal.hpp"
#include "packed_tiles.hpp"
#include "../../include/bsa.h"

namespace bsa {

namespace {

constexpr int LA_ROWS = 32;              // tokens of a chunk
constexpr int LA_STAGES = 3;

struct LinearOperand {
    const half_t *x;
    long long token, head;               // strides in values
};

// one of the sums above, over all heads of its result
struct LinearSum {
    LinearOperand a, b, c;
    half_t *out;                         // dense [T][heads][HD]
    const float *first;                  // [sequences][key heads][HD][HD]: state at the walk's beginning, or null
    float *last;                         // the same at its end, or null
    int heads, inner;                    // heads of the result; heads of b and c that each of them sums over
    bool transposed;                     // states are read as their transposes
    float a_mul, b_mul;                  // of a_t S, of what enters the state
};

struct LinearWalk {
    const float *log_decay;              // [key heads]
    const int32_t *offsets;              // [sequences + 1]
    float *states;                       // [boundaries][key heads][HD][HD]: between segments, or null where there is none
    int tokens, sequences, key_heads, group;
    int shift;                           // a segment has 1 << shift tokens
    int units, unit_sets, slots;         // of the launch: results' heads, as packed_grid takes them; slots of a head
    float scale;
};

struct LinearItem {
    int unit, slot, sequence, begin, n;  // n: of the sequence
    int segment, segments;
    bool there;
};

__device__ __forceinline__ int linear_offset(const LinearWalk &p, int b)
{
    const int x = p.offsets[b];
    return x < 0 ? 0 : x > p.tokens ? p.tokens : x;
}

// Slot floor(offset / segment) + b is the first of sequence b, ascending in b, and an empty sequence has one: 64 lanes search together.
__device__ __forceinline__ LinearItem linear_item(const LinearWalk &p, int block)
{
    LinearItem item{0, 0, 0, 0, 0, 0, 0, false};
    const int x = block & 7, t = block >> 3;
    const int share = 8 / p.unit_sets, in_set = p.units / p.unit_sets;
    item.unit = x / share * in_set + t % in_set;
    item.slot = t / in_set * share + x % share;
    if (item.slot >= p.slots) return item;
    const int l = lane_id();
    int first = 0, count = p.sequences;
    while (true) {
        const int stride = (count + 63) / 64, b = first + l * stride;
        const bool before = b < first + count && (linear_offset(p, b) >> p.shift) + b <= item.slot;
        const int seen = __popcll(__builtin_amdgcn_ballot_w64(before));
        const int skip = (seen > 0 ? seen - 1 : 0) * stride;
        first += skip;
        count = count - skip < stride ? count - skip : stride;
        if (stride == 1) break;
    }
    item.sequence = __builtin_amdgcn_readfirstlane(first);
    item.begin = __builtin_amdgcn_readfirstlane(linear_offset(p, item.sequence));
    const int end = __builtin_amdgcn_readfirstlane(linear_offset(p, item.sequence + 1));
    item.n = end > item.begin ? end - item.begin : 0;
    item.segment = item.slot - ((item.begin >> p.shift) + item.sequence);
    item.segments = item.n > 0 ? (item.n + (1 << p.shift) - 1) >> p.shift : 1;
    item.there = item.segment >= 0 && item.segment < item.segments;
    return item;
}

// Place of the state between segments j - 1 and j of a sequence, j >= 1.  A sequence's last boundary has floor((n - 1) / segment) =: j, and
// floor(begin / segment) + j <= floor((begin + n - 1) / segment), so that the next sequence's first lies behind it and all are below
// (tokens - 1) / segment.
__device__ __forceinline__ size_t linear_boundary(const LinearWalk &p, int begin, int j, int key_head)
{
    return (size_t)((begin >> p.shift) + j - 1) * p.key_heads + key_head;
}

// exp(log_decay e): decays of e tokens
__device__ __forceinline__ float linear_power(float log2_decay, int e) { return e == 0 ? 1.f : at_exp2(log2_decay * (float)e); }

__device__ __forceinline__ float wave_most(float x)
{
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) x = fmaxf(x, __int_as_float(__builtin_amdgcn_ds_bpermute((lane_id() ^ d) << 2, __float_as_int(x))));
    return x;
}
// 2^e that brings a finite x > 0 to 2^9 .. 2^10
__device__ __forceinline__ float lift_of(float most)
{
    const int e = 10 - __builtin_amdgcn_frexp_expf(most);
    return __builtin_ldexpf(1.f, e > 120 ? 120 : e < -120 ? -120 : e);
}

// Chunks of two or three operands on their way to LDS, fetched by all W waves
template <int HD, bool WITH_A>
struct LinearTiles {
    static constexpr int W = HD / 32, TILE = 64 * HD, OPERANDS = WITH_A ? 3 : 2, STAGE = OPERANDS * TILE;
    static constexpr int PER_OPERAND = HD / 16 / W, REQUESTS = OPERANDS * PER_OPERAND;
    unsigned lds;                        // of this wave's first request in stage 0
    int row, piece;
    const unsigned char *base[OPERANDS];
    unsigned stride[OPERANDS];           // bytes between tokens
    __device__ __forceinline__ LinearTiles(unsigned char *lds_raw)
    {
        const int w = wave_id(), l = lane_id(), part = w & 3;
        lds = __builtin_amdgcn_readfirstlane(lds_address(lds_raw)) + 1024 * part;
        row = 8 * part + (l >> 3);
        piece = 16 * panel_src_piece(l, part);
    }
    static constexpr size_t lds_bytes() { return (size_t)LA_STAGES * STAGE; }
    __device__ __forceinline__ void set(int o, const LinearOperand &x, long long first_token, int head)
    {
        base[o] = (const unsigned char *)(x.x + first_token * x.token + head * x.head);
        stride[o] = (unsigned)(2 * x.token);
    }
    // `valid` tokens from `token` on, those behind as the last
    __device__ __forceinline__ void request(int o, int token, int valid, int stage) const
    {
        const unsigned char *from = base[o] + (long long)token * stride[o];
        const unsigned to = lds + (unsigned)(stage * STAGE + o * TILE);
#pragma unroll
        for (int i = 0; i < PER_OPERAND; ++i) {
            // HD 128: four waves, a panel a request; HD 64: two waves, 16 rows a request
            const int r = W == 4 ? row : row + 16 * i, there = r < valid ? r : valid - 1;
            dma16(from + (W == 4 ? 128 * i : 0), (unsigned)there * stride[o] + piece, to + (W == 4 ? 4096 * i : 2048 * i));
        }
    }
};

// TERMS: how many 16-bit values stand for what enters the state (its operand of the product): see linear_terms
template <int HD, bool BF, int TERMS, bool BACKWARDS, bool RESULT>
__device__ __forceinline__ void linear_walk(const LinearWalk &p, const LinearSum &sum, const LinearItem &item, int head, unsigned char *lds_raw)
{
    using Tiles = LinearTiles<HD, RESULT>;
    constexpr int KS = HD / 16, DT = HD / 32, B = RESULT ? 1 : 0, C = B + 1;
    const int w = wave_id(), l = lane_id(), i = l & 31, h = l >> 5;
    const int key_head = sum.inner > 1 || sum.heads == p.key_heads ? head : head / p.group;
    const int b_head = sum.inner > 1 ? head * sum.inner : key_head;
    const float log2_decay = p.log_decay[key_head] * 1.4426950408889634f;

    // tokens of the segment, in chunks; step s is chunk s / inner (from the end: BACKWARDS) and head s % inner of b and c
    const int from = item.segment << p.shift, here = min(item.n - from, 1 << p.shift);
    const int chunks = (here + LA_ROWS - 1) / LA_ROWS, inner = sum.inner, steps = chunks * inner;
    const long long begin = (long long)item.begin + from;
    Tiles tiles(lds_raw);
    if (RESULT) tiles.set(0, sum.a, begin, head);
    tiles.set(B, sum.b, begin, b_head);
    tiles.set(C, sum.c, begin, b_head);
    int next = 0, next_inner = 0, next_stage = 0;          // the chunk requested next
    auto request = [&]() {
        const int at = LA_ROWS * (BACKWARDS ? chunks - 1 - next : next), valid = min(here - at, LA_ROWS);
#pragma unroll
        for (int o = 0; o < Tiles::OPERANDS; ++o) tiles.request(o, at, valid, next_stage);
        next_stage = next_stage == LA_STAGES - 1 ? 0 : next_stage + 1;
        if (++next_inner == inner) {
            next_inner = 0;
            ++next;
            tiles.base[B] -= 2 * (inner - 1) * sum.b.head, tiles.base[C] -= 2 * (inner - 1) * sum.c.head;
        } else {
            tiles.base[B] += 2 * sum.b.head, tiles.base[C] += 2 * sum.c.head;
        }
    };
    if (steps > 0) request();
    if (steps > 1) request();

    // LDS addresses inside stage 0: rows as operands, b's columns (all), c's columns (this wave's)
    unsigned row_at[4], b_at[2][2], c_at[2];
    {
        const unsigned base = __builtin_amdgcn_readfirstlane(lds_address(lds_raw));
        const unsigned r = (unsigned)get_panel_addr(l, 0);
#pragma unroll
        for (int s = 0; s < 4; ++s) row_at[s] = base + (r ^ (32u * s));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const unsigned bt = (unsigned)get_panel_tr_ordered_addr(PANEL_SWAPPED, l, half), ct = (unsigned)get_panel_tr_ordered_addr(PANEL_PERM16, l, half);
            b_at[0][half] = base + bt;
            b_at[1][half] = base + (bt ^ 64u);
            c_at[half] = base + (ct ^ (64u * (w & 1))) + 4096u * (w >> 1);
        }
    }
    typedef const h8 __attribute__((address_space(3))) *lds_h8;
    typedef tr4 __attribute__((address_space(3))) *lds_tr4;
    auto rows = [&](unsigned tile, int s) { return *(lds_h8)(uintptr_t)(row_at[s % 4] + (tile + 4096u * (s / 4))); };
    auto columns = [&](const unsigned (&at)[2], unsigned tile) {
        const tr4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4)(uintptr_t)(at[0] + tile));
        const tr4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4)(uintptr_t)(at[1] + tile));
        return __builtin_shufflevector(__builtin_bit_cast(h4, lo), __builtin_bit_cast(h4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
    };

    // the state: value v of state[t] is row 32 t + swapped16(r), column 32 w + perm16(i), r = 8 (v / 4) + 4 h + v % 4;
    // times s_mul, a power of two (fp16: operands are made of it)
    f16v state[DT];
    float s_mul = 1.f;
    bool zero = true;                    // nothing entered so far
    const int column = 32 * w + perm16(i);
    auto row_of = [&](int t, int v) { return 32 * t + (v & 3) + 4 * ((v >> 2) & 1) + 8 * h + 16 * (v >> 3); };
    auto state_most = [&]() {
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) most = fmaxf(most, __builtin_fabsf(state[t][v]));
        return most;
    };
    auto scale_state = [&](float by) {
#pragma unroll
        for (int t = 0; t < DT; ++t) state[t] *= by;
    };
    {
        const bool given = BACKWARDS ? item.segment == item.segments - 1 : item.segment == 0;
        const size_t square = (size_t)HD * HD;
        const float *src = !RESULT ? nullptr
                         : given ? (sum.first ? sum.first + ((size_t)item.sequence * p.key_heads + key_head) * square : nullptr)
                                 : p.states + linear_boundary(p, item.begin, BACKWARDS ? item.segment + 1 : item.segment, key_head) * square;
#pragma unroll
        for (int t = 0; t < DT; ++t) state[t] = f16v{0};
        if (src != nullptr) {
            zero = false;
            if (sum.transposed) {
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const f4v x = *reinterpret_cast<const f4v *>(src + (size_t)column * HD + row_of(t, 4 * u));
#pragma unroll
                        for (int j = 0; j < 4; ++j) state[t][4 * u + j] = x[j];
                    }
            } else {
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int v = 0; v < 16; ++v) state[t][v] = src[(size_t)row_of(t, v) * HD + column];
            }
            // arrived: the compiler would wait for them inside the loop, and with them for the chunks on their way
#pragma unroll
            for (int t = 0; t < DT; ++t) asm volatile("" : "+v"(state[t]));
            if (!BF) {
                const float most = wave_most(state_most());
                if (most > 0.f && most < __builtin_inff()) {
                    s_mul = lift_of(most);
                    scale_state(s_mul);
                }
            }
        }
    }

    // decays inside a chunk of `valid` tokens: of P (and its mask), of what enters the state, of the state's way to this lane's token and
    // to the chunk's other end
    float within[16], entering[16], since = 0.f, over = 1.f;
    int decays_of = 0;
    auto set_decays = [&](int valid) {
        decays_of = valid;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int r = 8 * (v >> 2) + 4 * h + (v & 3);
            if (RESULT) {
                const bool sees = BACKWARDS ? r >= i && r < valid : r <= i;
                within[v] = sees ? p.scale * linear_power(log2_decay, BACKWARDS ? r - i : i - r) : 0.f;
            }
            entering[v] = r < valid ? sum.b_mul * linear_power(log2_decay, BACKWARDS ? r + 1 : valid - 1 - r) : 0.f;
        }
        if (RESULT) since = BACKWARDS ? (i < valid ? sum.a_mul * linear_power(log2_decay, valid - 1 - i) : 0.f) : sum.a_mul * linear_power(log2_decay, i + 1);
        over = linear_power(log2_decay, valid);
    };

    // whether the walk's end state is wanted
    const bool ends = RESULT ? sum.last != nullptr && (BACKWARDS ? item.segment == 0 : item.segment == item.segments - 1) : true;

    h8 aop[KS];
    f16v oacc;
    uint4 result[2];
    int stored = 0;                      // tokens of `result` that are to be stored
    half_t *to = nullptr;
    const long long width = (long long)sum.heads * HD;
    half_t *const out = RESULT ? sum.out + begin * width + (long long)head * HD + 32 * w + 16 * h : nullptr;
    auto store = [&]() {
        if (i < stored) {
            stg16(to, result[0]);
            stg16(to + 8, result[1]);
        }
        stored = 0;
    };
    int chunk = BACKWARDS ? chunks - 1 : 0, g = 0, stage = 0;
    for (int step = 0; step < steps; ++step) {
        if (step + 1 < steps) tile_wait<Tiles::REQUESTS>();
        else tile_wait<0>();
        asm volatile("s_barrier" ::: "memory");
        if (RESULT) store();
        if (step + 2 < steps) request();
        const int at = LA_ROWS * chunk, valid = min(here - at, LA_ROWS);
        const unsigned tile = (unsigned)(stage * Tiles::STAGE);
        if (valid != decays_of) set_decays(valid);
        h8 cop[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) cop[s] = columns(c_at, tile + C * Tiles::TILE + 2048u * s);
        if (RESULT && g == 0) {
#pragma unroll
            for (int s = 0; s < KS; ++s) aop[s] = rows(tile, s);
            float up = since;
            if (!BF && !zero) {          // operands of fp16 from the state
                const float most = state_most();
                const bool large = most >= 0x1p15f && most < __builtin_inff();
                if (__builtin_amdgcn_ballot_w64(large) != 0ull || __builtin_amdgcn_ballot_w64(most >= 0.25f || most != most) == 0ull) {
                    const float all = wave_most(most < __builtin_inff() ? most : 0.f);
                    if (all > 0.f) {
                        const float by = lift_of(all), to_mul = fminf(fmaxf(s_mul * by, 0x1p-120f), 0x1p120f);
                        scale_state(to_mul / s_mul);
                        s_mul = to_mul;
                    }
                }
                up = since / s_mul;
            }
            oacc = f16v{0};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                h8 op;
#pragma unroll
                for (int j = 0; j < 8; ++j) op[j] = narrow_16<BF>(state[s / 2][8 * (s % 2) + j]);
                oacc = mfma_16<BF>(op, aop[s], oacc);
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) oacc[v] *= up;
        }
        if (RESULT) {
            f16v prob = {0};
#pragma unroll
            for (int s = 0; s < KS; ++s) prob = mfma_16<BF>(rows(tile + B * Tiles::TILE, s), aop[s], prob);
            float most = 0.f, down = 1.f;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                prob[v] = within[v] == 0.f ? 0.f : prob[v] * within[v];      // whatever a hidden one is
                if (!BF) most = fmaxf(most, __builtin_fabsf(prob[v]));
            }
            if (!BF) {
                most = fmaxf(most, at_lane_xor32(most));
                const float mul = most > 0.f && most < __builtin_inff() ? lift_of(most) : 1.f;
                down = 1.f / mul;
#pragma unroll
                for (int v = 0; v < 16; ++v) prob[v] *= mul;
            }
            h8 pop[2];
#pragma unroll
            for (int v = 0; v < 16; ++v) pop[v >> 3][v & 7] = narrow_16<BF>(prob[v]);
            f16v part = {0};
            float sure = 0.f;
#pragma unroll
            for (int s = 0; s < 2; ++s) part = mfma_16<BF>(cop[s], pop[s], part);
#pragma unroll
            for (int v = 0; v < 16; ++v) sure += __builtin_fabsf(part[v]);
            if (__builtin_amdgcn_ballot_w64(!(sure < __builtin_inff())) != 0ull) {
                // An infinity or a NaN in c: zero times it is NaN, also for tokens that do not see it.  Left out of the product, it
                // makes NaN of its column for those that do.
                h8 clean[1][2] = {{cop[0], cop[1]}};
                take_out_not_finite<BF>(clean);
                part = f16v{0};
#pragma unroll
                for (int s = 0; s < 2; ++s) part = mfma_16<BF>(clean[0][s], pop[s], part);
                const unsigned first = __builtin_amdgcn_readfirstlane(lds_address(lds_raw)) + tile + C * Tiles::TILE + 4096u * (w >> 1);
#pragma unroll 1
                for (int r = 0; r < valid; ++r) {
                    const bool sees = BACKWARDS ? r >= i : r <= i;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const h8 x = *(lds_h8)(uintptr_t)(first + 128u * r + 16u * (unsigned)((4 * (w & 1) + 2 * h + half) ^ panel_swizzle(r)));
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float value = widen_16<BF>(x[j]);
                            if (sees && !(__builtin_fabsf(value) < __builtin_inff())) part[8 * half + j] = __builtin_nanf("");
                        }
                    }
                }
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) oacc[v] = BF ? oacc[v] + part[v] : __builtin_fmaf(part[v], down, oacc[v]);
        }
        if (ends || step + inner - g < steps) {            // the state is needed once more
            if (g == 0 && !zero) scale_state(over);
            float x[2][8], most = 0.f;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const half_t one = cop[s][j];
                    x[s][j] = widen_16<BF>(one) * entering[8 * s + j];
                    if (!BF) most = fmaxf(most, __builtin_fabsf(x[s][j]));
                }
            if (!BF) {
                const bool fits = most * s_mul < 0x1p15f || !(most < __builtin_inff());
                if (zero || __builtin_amdgcn_ballot_w64(!fits) != 0ull) {
                    const float all = wave_most(most < __builtin_inff() ? most : 0.f);
                    if (all > 0.f) {
                        const float to_mul = lift_of(all);
                        if (!zero) scale_state(to_mul / s_mul);
                        s_mul = to_mul;
                    }
                }
            }
            zero = false;
            h8 cw[TERMS][2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float left = BF ? x[s][j] : x[s][j] * s_mul;
#pragma unroll
                    for (int e = 0; e < TERMS; ++e) {
                        cw[e][s][j] = narrow_16<BF>(left);
                        const half_t one = cw[e][s][j];
                        if (e + 1 < TERMS) left -= widen_16<BF>(one);
                    }
                }
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const h8 bop = columns(b_at[t % 2], tile + B * Tiles::TILE + 4096u * (t / 2) + 2048u * s);
#pragma unroll
                    for (int e = 0; e < TERMS; ++e) state[t] = mfma_16<BF>(bop, cw[e][s], state[t]);
                }
        }
        stage = stage == LA_STAGES - 1 ? 0 : stage + 1;
        if (++g == inner) {
            if (RESULT) {
                pack16<BF>(oacc, result[0], result[1]);
                to = out + (long long)(at + i) * width;
                stored = valid;
            }
            g = 0;
            chunk += BACKWARDS ? -1 : 1;
        }
    }
    if (RESULT) store();
    if (ends) {
        float *dst = RESULT ? sum.last + ((size_t)item.sequence * p.key_heads + key_head) * HD * HD
                            : p.states + linear_boundary(p, item.begin, BACKWARDS ? item.segment : item.segment + 1, key_head) * HD * HD;
        if (RESULT && !BACKWARDS && sum.heads != p.key_heads && head % p.group != 0) return;
        const float down = BF ? 1.f : 1.f / s_mul;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) dst[(size_t)row_of(t, v) * HD + column] = state[t][v] * down;
    }
}

__device__ __forceinline__ void linear_clear(const LinearWalk &p, int part, half_t *rows, long long width)
{
    const int head = linear_offset(p, 0), tail = linear_offset(p, p.sequences);
    const long long pieces = width / 8, before = head < tail ? head : tail;
    auto clear = [&](long long from, long long to) {
        for (long long i = from * pieces + (long long)part * blockDim.x + threadIdx.x; i < to * pieces; i += (long long)PACKED_CLEARING * blockDim.x)
            stg16(rows + 8 * i, make_uint4(0, 0, 0, 0));
    };
    clear(0, before);
    clear(tail, p.tokens);
}

template <int HD, bool BF, int TERMS>
__global__ __launch_bounds__(2 * HD, 2) void linear_forward_kernel(LinearWalk p, LinearSum sum)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    const int cells = packed_grid(p.units, p.unit_sets, p.slots);
    if ((int)blockIdx.x >= cells) return linear_clear(p, (int)blockIdx.x - cells, sum.out, (long long)sum.heads * HD);
    const LinearItem item = linear_item(p, (int)blockIdx.x);
    if (!item.there) return;
    linear_walk<HD, BF, TERMS, false, true>(p, sum, item, item.unit, lds_raw);
}

// the three gradients: units are the query heads (dq), then for each key head dv and dk
struct LinearGradients {
    LinearSum dq, dv, dk;
    const float *states;                 // those of the forward pass
};
template <int HD, bool BF, int TERMS>
__global__ __launch_bounds__(2 * HD, 2) void linear_backward_kernel(LinearWalk p, LinearGradients g)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    const int cells = packed_grid(p.units, p.unit_sets, p.slots);
    if ((int)blockIdx.x >= cells) {
        const int part = (int)blockIdx.x - cells;
        linear_clear(p, part, g.dq.out, (long long)g.dq.heads * HD);
        linear_clear(p, part, g.dv.out, (long long)g.dv.heads * HD);
        return linear_clear(p, part, g.dk.out, (long long)g.dk.heads * HD);
    }
    const LinearItem item = linear_item(p, (int)blockIdx.x);
    if (!item.there) return;
    if (item.unit < g.dq.heads) {
        p.states = const_cast<float *>(g.states);
        return linear_walk<HD, BF, 2, false, true>(p, g.dq, item, item.unit, lds_raw);
    }
    const int at = item.unit - g.dq.heads;
    const bool values = (at & 1) == 0;
    linear_walk<HD, BF, TERMS, true, true>(p, values ? g.dv : g.dk, item, at >> 1, lds_raw);
}

// every segment's own sum, of those that have a neighbour behind (BACKWARDS: in front)
template <int HD, bool BF, int TERMS, bool BACKWARDS>
__global__ __launch_bounds__(2 * HD, 2) void linear_segments_kernel(LinearWalk p, LinearSum sum)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    const LinearItem item = linear_item(p, (int)blockIdx.x);
    if (!item.there || (BACKWARDS ? item.segment == 0 : item.segment == item.segments - 1)) return;
    linear_walk<HD, BF, TERMS, BACKWARDS, false>(p, sum, item, item.unit, lds_raw);
}

// the running sum over the segments of a sequence, in place: what each segment begins with
template <bool BACKWARDS>
__global__ __launch_bounds__(256) void linear_running_kernel(LinearWalk p, const float *__restrict__ first, int square)
{
    const int b = (int)blockIdx.z, key_head = (int)blockIdx.y;
    const int begin = linear_offset(p, b), n = linear_offset(p, b + 1) - begin, segments = (n + (1 << p.shift) - 1) >> p.shift;
    if (n <= 0 || segments < 2) return;
    const float log2_decay = p.log_decay[key_head] * 1.4426950408889634f;
    const size_t at = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x), stride = (size_t)p.key_heads * square;
    float *sums = p.states + linear_boundary(p, begin, 1, key_head) * square + at;       // of boundary 1
    f4v run = {0, 0, 0, 0};
    if (first != nullptr) run = *reinterpret_cast<const f4v *>(first + ((size_t)b * p.key_heads + key_head) * square + at);
    const float whole = linear_power(log2_decay, 1 << p.shift), rest = linear_power(log2_decay, n - ((segments - 1) << p.shift));
    auto place = [&](int j) { return reinterpret_cast<f4v *>(sums + (size_t)(BACKWARDS ? segments - 2 - j : j) * stride); };
    f4v own = *place(0);
    for (int j = 0; j + 1 < segments; ++j) {
        const f4v after = *place(j + 2 < segments ? j + 1 : j);
        run = run * (BACKWARDS && j == 0 ? rest : whole) + own;
        *place(j) = run;
        own = after;
    }
}

LinearWalk walk_of(const LinearArgs &a)
{
    LinearWalk p;
    p.log_decay = a.log_decay, p.offsets = a.offsets;
    p.states = nullptr;
    p.tokens = a.tokens, p.sequences = a.sequences, p.key_heads = a.key_heads, p.group = a.heads / a.key_heads;
    p.shift = __builtin_ctz((unsigned)a.segment);
    p.slots = packed_slots(a.tokens, a.sequences, a.segment);
    p.units = p.unit_sets = 0;
    p.scale = a.scale;
    return p;
}
LinearOperand operand(const void *x, long long token, long long head) { return LinearOperand{(const half_t *)x, token, head}; }

template <class Kernel, class... Args>
hipError_t run_linear(Kernel kernel, LinearWalk p, int units, int clearing, int hd, size_t lds, hipStream_t st, const Args &...args)
{
    if (lds > 65536) {
        const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (err != hipSuccess) return err;
    }
    p.units = units;
    p.unit_sets = packed_head_sets(units);
    kernel<<<packed_grid(units, p.unit_sets, p.slots) + clearing, 2 * hd, lds, st>>>(p, args...);
    return hipGetLastError();
}

template <int HD, bool BF, int TERMS, bool BACKWARDS>
hipError_t segment_states(LinearWalk p, const LinearSum &sum, const float *first, hipStream_t st)
{
    const hipError_t err = run_linear(linear_segments_kernel<HD, BF, TERMS, BACKWARDS>, p, p.key_heads, 0, HD, LinearTiles<HD, false>::lds_bytes(), st, sum);
    if (err != hipSuccess) return err;
    linear_running_kernel<BACKWARDS><<<dim3(HD * HD / 1024, p.key_heads, p.sequences), 256, 0, st>>>(p, first, HD * HD);
    return hipGetLastError();
}

template <int HD, bool BF, int TERMS>
hipError_t forward(const LinearArgs &a, hipStream_t st)
{
    LinearWalk p = walk_of(a);
    p.states = a.states;
    LinearSum sum{operand(a.q, a.q_token, a.q_head), operand(a.k, a.k_token, a.k_head), operand(a.v, a.v_token, a.v_head), (half_t *)a.out,
                  a.first, a.last, a.heads, 1, false, a.scale, 1.f};
    if (a.tokens > a.segment) {
        LinearSum own = sum;
        own.heads = a.key_heads;
        const hipError_t err = segment_states<HD, BF, TERMS, false>(p, own, a.first, st);
        if (err != hipSuccess) return err;
    }
    return run_linear(linear_forward_kernel<HD, BF, TERMS>, p, a.heads, PACKED_CLEARING, HD, LinearTiles<HD, true>::lds_bytes(), st, sum);
}

template <int HD, bool BF, int TERMS>
hipError_t backward(const LinearArgs &a, hipStream_t st)
{
    LinearWalk p = walk_of(a);
    p.states = a.back_states;
    const int group = a.heads / a.key_heads;
    const LinearOperand q = operand(a.q, a.q_token, a.q_head), k = operand(a.k, a.k_token, a.k_head), v = operand(a.v, a.v_token, a.v_head),
                        g = operand(a.dout, a.g_token, a.g_head);
    LinearGradients grads{LinearSum{g, v, k, (half_t *)a.dq, a.first, nullptr, a.heads, 1, true, a.scale, 1.f},
                          LinearSum{k, q, g, (half_t *)a.dv, a.dlast, a.dfirst, a.key_heads, group, false, 1.f, a.scale},
                          LinearSum{v, g, q, (half_t *)a.dk, a.dlast, nullptr, a.key_heads, group, true, 1.f, a.scale}, a.states};
    if (a.tokens > a.segment) {
        const hipError_t err = segment_states<HD, BF, TERMS, true>(p, grads.dv, a.dlast, st);
        if (err != hipSuccess) return err;
    }
    return run_linear(linear_backward_kernel<HD, BF, TERMS>, p, a.heads + 2 * a.key_heads, PACKED_CLEARING, HD, LinearTiles<HD, true>::lds_bytes(), st,
                      grads);
}

}  // namespace

// What enters the state is a 16-bit value times a decay.  Two 16-bit parts of it carry 16 bits (bf16) or 22 (fp16): with one, results would be
// 1.7 times as far off as their own rounding leaves them, with two 1.4.  States that are results themselves (fp32) take three in bf16.
static int linear_terms(const LinearArgs &a, const void *states_out) { return a.bf16 && states_out != nullptr ? 3 : 2; }

bool linear_fits(const LinearArgs &a)
{
    const long long slots = (long long)a.tokens / a.segment + a.sequences + 7;
    return ((long long)(a.heads + 2 * a.key_heads) * slots + PACKED_CLEARING) * 2 * a.head_dim < (1ll << 32) && a.sequences <= 65535;
}
size_t linear_workspace_bytes(const LinearArgs &a)
{
    if (a.tokens <= a.segment) return 0;
    return sizeof(float) * (size_t)((a.tokens - 1) / a.segment) * a.key_heads * a.head_dim * a.head_dim;
}
int linear_segment(int tokens, int sequences, int heads, int head_dim)
{
    (void)sequences, (void)head_dim;
    int segment = 256;
    while (segment < 4096 && (long long)tokens * heads / segment > 1024) segment *= 2;
    return segment;
}

hipError_t launch_linear_forward(const LinearArgs &a, hipStream_t st)
{
    const bool three = linear_terms(a, a.last) == 3;
    if (a.head_dim == 64) return !a.bf16 ? forward<64, false, 2>(a, st) : three ? forward<64, true, 3>(a, st) : forward<64, true, 2>(a, st);
    return !a.bf16 ? forward<128, false, 2>(a, st) : three ? forward<128, true, 3>(a, st) : forward<128, true, 2>(a, st);
}
hipError_t launch_linear_backward(const LinearArgs &a, hipStream_t st)
{
    const bool three = linear_terms(a, a.dfirst) == 3;
    if (a.head_dim == 64) return !a.bf16 ? backward<64, false, 2>(a, st) : three ? backward<64, true, 3>(a, st) : backward<64, true, 2>(a, st);
    return !a.bf16 ? backward<128, false, 2>(a, st) : three ? backward<128, true, 3>(a, st) : backward<128, true, 2>(a, st);
}

}  // namespace bsa

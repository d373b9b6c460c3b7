// Linear attention with a decay for each key head over sequences packed along the tokens, and its gradients:
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   l = exp(log_decay), S_0 given or zero.
//
// Chunks of 32 tokens: with a, b, c for q, k, v and P_ts = scale l^(t-s) (a_t . b_s) for s <= t inside the chunk,
//   o_t = sum_s P_ts c_s + scale l^(t+1) a_t S,      S <- l^32 S + sum_s l^(31-s) b_s c_s^T.
// The gradients are the same sum over other operands and, for dk and dv, from the end of the sequence, R in the place of S:
//   dq: a, b, c = dO, V, K (the state is S^T);   dv: K, Q, dO backwards;   dk: V, dO, Q backwards (R^T).
//
// A sequence is cut into segments of p.segment tokens.  One workgroup walks a segment of one key head with all query heads that share it; its
// wave w has columns 32 w .. of c and of the state, which stays in fp32 accumulators from chunk to chunk.  dv and dk, which read the
// same four operands, share a workgroup.  Where a sequence has several segments, two launches in front make the state that each begins
// with: every segment's own sum, then the running sum over segments.  Chunks travel straight to LDS two steps ahead of their use, in
// a ring of three.
//
// What bounds it (times of launches, the least of 60 and their median):
//   results: memory.  65519 tokens, 8 heads over 4, head dim 128, bf16: 104 us (121) for 430 MB, operands, result and states, 4.1 TB/s (3.6); one
//   workgroup of the two on a compute unit gets what the other leaves and ends a fifth later.  24575 tokens, 16 heads, fp16: 98 us (101), 4.4 TB/s.
//   segments' sums: memory, 134 MB in 37 us (45), 3.6 TB/s (3.0), 201 MB in 46 (47); with dq 139 us (141) together; the running sum over them 11 to
//   13 us (12 to 15) for 62 MB.
//   dv and dk: the clocks of a step, 24575 tokens, 16 heads, head dim 128: 205 us (209) for 600 MB; of 6.7k clocks a step the vector pipe works 45 %
//   and the matrix pipe 27 %, two waves on each side of a barrier.  512 threads and 97 KB of LDS: one workgroup a compute unit.
//   short texts: what a segment costs before its first product (5 us: its place, the state, the first chunks' way through memory) and
//   1 us a chunk.  368 tokens, 12 heads, head dim 64: 13.6 us (15).
#include "attention_tiles.hpp"
#include "bsa_device.hpp"
#include "bsa_internal.hpp"
#include "packed_tiles.hpp"
#include "../../include/bsa.h"

namespace bsa {

namespace {

constexpr int LA_ROWS = 32;              // tokens of a chunk
constexpr int LA_STAGES = 3;
// Behind the stages, floats: decays of P by how many tokens lie between, in four copies a float apart, so that four neighbours begin at a
// multiple of 16 bytes; then those of what enters the state, by token.
constexpr int LA_BETWEEN = 72, LA_TABLE = 4 * (4 * LA_BETWEEN + LA_ROWS);

struct LinearOperand {
    const half_t *x;
    long long token, head;               // strides in values
};

// One of the sums above.  A key head has a_inner heads of a (and of the result), or c_inner heads of b and c, whose sums add up; one of the two
// is 1.
struct LinearSum {
    LinearOperand a, b, c;
    half_t *out;                         // dense [T][key heads * a_inner][HD]
    const float *first;                  // [sequences][key heads][HD][HD]: state at the walk's beginning, or null
    float *last;                         // the same at its end, or null
    int a_inner, c_inner;
    bool transposed;                     // states are read as their transposes
    float a_mul, b_mul;                  // of a_t S, of what enters the state
};

struct LinearWalk {
    const float *log_decay;              // [key heads]
    const int32_t *offsets;              // [sequences + 1]
    float *states;                       // [boundaries][key heads][HD][HD]: between segments, or null where there is none
    int tokens, sequences, key_heads;
    int segment;                         // tokens, a multiple of LA_ROWS
    int head_sets, slots;                // of the launch, as packed_grid takes them; slots of a key head
    float scale;
};

struct LinearItem {
    int head, sequence, begin, n;        // head: key head; n: of the sequence
    int segment, segments;
    bool there;
};

__device__ __forceinline__ int linear_offset(const LinearWalk &p, int b)
{
    const int x = p.offsets[b];
    return x < 0 ? 0 : x > p.tokens ? p.tokens : x;
}

// Slot floor(offset / segment) + b is the first of sequence b, ascending in b, and an empty sequence has one: 64 lanes search together,
// up to 64 sequences by one look at the offsets.
__device__ __forceinline__ LinearItem linear_item(const LinearWalk &p, int block)
{
    LinearItem item{0, 0, 0, 0, 0, 0, false};
    const int x = block & 7, t = block >> 3;
    const int share = 8 / p.head_sets, in_set = p.key_heads / p.head_sets;
    item.head = x / share * in_set + t % in_set;
    const int slot = t / in_set * share + x % share;
    if (slot >= p.slots) return item;
    const unsigned length = (unsigned)p.segment;
    const int l = lane_id();
    int first = 0, count = p.sequences, stride, lane, from, to;
    do {
        stride = (count + WAVE - 1) / WAVE;
        const int b = first + l * stride;
        const bool there = b < first + count;
        from = linear_offset(p, there ? b : p.sequences), to = linear_offset(p, there ? b + 1 : p.sequences);
        const int seen = __popcll(__builtin_amdgcn_ballot_w64(there && (int)((unsigned)from / length) + b <= slot));
        lane = seen > 0 ? seen - 1 : 0;
        first += lane * stride;
        count = count - lane * stride < stride ? count - lane * stride : stride;
    } while (stride > 1);
    item.sequence = __builtin_amdgcn_readfirstlane(first);
    item.begin = __builtin_amdgcn_readlane(from, lane);
    const int end = __builtin_amdgcn_readlane(to, lane);
    item.n = end > item.begin ? end - item.begin : 0;
    item.segment = slot - ((int)((unsigned)item.begin / length) + item.sequence);
    item.segments = item.n > 0 ? (int)(((unsigned)item.n + length - 1) / length) : 1;
    item.there = item.segment >= 0 && item.segment < item.segments;
    return item;
}

// Place of the state between segments j - 1 and j of a sequence, j >= 1.  A sequence's last boundary has j = floor((n - 1) / segment), and
// floor(begin / segment) + j <= floor((begin + n - 1) / segment), so that the next sequence's first lies behind it and all are below
// (tokens - 1) / segment.
__device__ __forceinline__ size_t linear_boundary(const LinearWalk &p, int begin, int j, int key_head)
{
    return ((size_t)((unsigned)begin / (unsigned)p.segment) + j - 1) * p.key_heads + key_head;
}

// Decay of e tokens of one stretch: a chunk and what was put off before it, or a segment.  The exponent, x, is made from e and is off by about
// 2^-23 of itself.  Stretches multiply, each factor rounded: over m of them with exponents x1 .. xm what is left of a state is off by
// (x1 + .. + xm + m) 2^-23 of itself; a chunk ends one stretch at the most, a segment another.  Decays below 2^-126 are nothing.
__device__ __forceinline__ float linear_log2(float log_decay) { return log_decay * 1.4426950408889634f; }
__device__ __forceinline__ float linear_power(float log2_decay, int e) { return e == 0 ? 1.f : at_exp2(log2_decay * (float)e); }

__device__ __forceinline__ float wave_most(float x)
{
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) x = fmaxf(x, __int_as_float(__builtin_amdgcn_ds_bpermute((lane_id() ^ d) << 2, __float_as_int(x))));
    return x;
}
// 2^e that brings a finite x > 0 to 2^(to - 1) .. 2^to
__device__ __forceinline__ float lift_of(float most, int to)
{
    const int e = to - __builtin_amdgcn_frexp_expf(most);
    return __builtin_ldexpf(1.f, e > 120 ? 120 : e < -120 ? -120 : e);
}
__device__ __forceinline__ float larger(float most, float x)      // of magnitudes, NaN left out; one instruction
{
    return __builtin_amdgcn_fmed3f(most, __builtin_fabsf(x), __builtin_inff());
}
__device__ __forceinline__ bool is_finite(float x) { return __builtin_fabsf(x) < __builtin_inff(); }

typedef __fp16 fp16x2 __attribute__((ext_vector_type(2)));          // as builtins take them
// x y of a 16-bit x: fp16 is widened by the product itself
template <bool BF>
__device__ __forceinline__ float times(half_t x, float y) { return BF ? widen_16<BF>(x) * y : __builtin_fmaf((float)x, y, 0.f); }
// Two values as sums of TERMS 16-bit ones.  All but the last are cut, not rounded, in fp16 (one instruction for two); what is left is exact.
template <bool BF, int TERMS>
__device__ __forceinline__ void in_parts(float x0, float x1, h2 (&parts)[TERMS])
{
#pragma unroll
    for (int e = 0; e < TERMS; ++e) {
        if (!BF && e + 1 < TERMS) parts[e] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x0, x1));
        else parts[e] = h2{narrow_16<BF>(x0), narrow_16<BF>(x1)};
        if (e + 1 < TERMS) {
            const half_t a = parts[e][0], b = parts[e][1];
            float minus = -1.f;          // not known to the compiler, which would widen and subtract and round: three instructions in the place of one
            if (!BF) asm("" : "+s"(minus));
            x0 = BF ? x0 - widen_16<BF>(a) : __builtin_fmaf((float)a, minus, x0);
            x1 = BF ? x1 - widen_16<BF>(b) : __builtin_fmaf((float)b, minus, x1);
        }
    }
}

// Chunks of OPERANDS operands on their way to LDS, fetched by all NW waves of a workgroup
template <int HD, int OPERANDS, int NW>
struct LinearTiles {
    static constexpr int TILE = 64 * HD, STAGE = OPERANDS * TILE, WAVES = NW;
    static constexpr int EACH = HD / 16 / NW, REQUESTS = OPERANDS * EACH;        // of a wave
    static_assert(NW == 2 || NW == 4 || NW == 8, "rows and panels below");
    unsigned lds;                        // of this wave's first request in stage 0
    int row, piece;
    const unsigned char *base[OPERANDS];
    unsigned stride[OPERANDS];           // bytes between tokens
    __device__ __forceinline__ LinearTiles(unsigned char *lds_raw)
    {
        const int w = wave_id(), l = lane_id(), part = w & 3;
        lds = __builtin_amdgcn_readfirstlane(lds_address(lds_raw)) + 1024 * part + (NW == 8 ? 4096 * (w >> 2) : 0);
        row = 8 * part + (l >> 3);
        piece = 16 * panel_src_piece(l, part) + (NW == 8 ? 128 * (w >> 2) : 0);
    }
    static constexpr size_t lds_bytes() { return (size_t)LA_STAGES * STAGE + LA_TABLE; }
    __device__ __forceinline__ void set(int o, const LinearOperand &x, long long first_token, int head)
    {
        base[o] = (const unsigned char *)(x.x + first_token * x.token + head * x.head);
        stride[o] = (unsigned)(2 * x.token);
    }
    // `valid` tokens from base on, those behind as the last
    __device__ __forceinline__ void request(int o, int valid, int stage) const
    {
        const unsigned to = lds + (unsigned)(stage * STAGE + o * TILE);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            // a request is 8 rows of a panel of 64 columns: two waves fetch rows 16 apart, four a panel each time, eight both panels at once
            const int r = NW == 2 ? row + 16 * i : row, there = r < valid ? r : valid - 1;
            dma16(base[o] + (NW == 4 ? 128 * i : 0), (unsigned)there * stride[o] + piece, to + (NW == 2 ? 2048 * i : 4096 * i));
        }
    }
};

// What the waves of a workgroup read of a chunk: where their operands lie among the tiles
struct LinearPlaces {
    int a, b, c;
};

// TERMS: how many 16-bit values stand for what enters the state (its operand of the product): see linear_terms.  A wave is wave w of
// HD / 32 that share `sum`; the chunk's tiles are fetched by all waves of the workgroup.
template <int HD, bool BF, int TERMS, bool BACKWARDS, bool RESULT, class Tiles>
__device__ __forceinline__ void linear_walk(const LinearWalk &p, const LinearSum &sum, const LinearItem &item, int w, Tiles &tiles,
                                            const LinearPlaces places, const long long (&inner_step)[Tiles::STAGE / Tiles::TILE], int inner,
                                            unsigned char *lds_raw)
{
    constexpr int KS = HD / 16, DT = HD / 32, OPERANDS = Tiles::STAGE / Tiles::TILE;
    // The state's decay is put off until it passes this power of two: operands are made of the state, fp16 has no room for more.  In bf16 the state
    // is held smaller by as much, so that putting off makes nothing larger than it is: it goes as far up as fp32 does, and what is lost at
    // the other end is 2^-129 of what the parts of bf16 carry (until 2^23, at 2^-111: 1 % faster, 65519 tokens, 4 key heads).
    constexpr float PUT_OFF = 5.f;
    constexpr float HELD = 0x1p-5f, FREED = 0x1p5f;
    // P as an operand is this much larger (fp16 has least below 1), and the result until it is rounded
    constexpr float P_LIFT = BF ? 1.f : 64.f;
    const int l = lane_id(), i = l & 31, h = l >> 5, key_head = item.head;
    const float log2_decay = linear_log2(p.log_decay[key_head]);

    // tokens of the segment, in chunks; step s is chunk s / inner (from the end: BACKWARDS) and head s % inner
    const int from = item.segment * p.segment, here = min(item.n - from, p.segment);
    const int chunks = (here + LA_ROWS - 1) / LA_ROWS, steps = chunks * inner;
    const long long begin = (long long)item.begin + from;
    int next = 0, next_inner = 0, next_stage = 0;          // the step requested next, whose chunk and heads tiles.base has
#pragma unroll
    for (int o = 0; o < OPERANDS; ++o)
        if (BACKWARDS && chunks > 1) tiles.base[o] += (long long)LA_ROWS * (chunks - 1) * tiles.stride[o];
    auto request = [&]() {
        const int valid = min(here - LA_ROWS * (BACKWARDS ? chunks - 1 - next : next), LA_ROWS);
#pragma unroll
        for (int o = 0; o < OPERANDS; ++o) tiles.request(o, valid, next_stage);
        next_stage = next_stage == LA_STAGES - 1 ? 0 : next_stage + 1;
        // steps are made anew: kept, they are more scalars than there is room for
        if (++next_inner == inner) {
            next_inner = 0, ++next;
            int back = inner - 1;
            asm("" : "+s"(back));
#pragma unroll
            for (int o = 0; o < OPERANDS; ++o) {
                const long long chunk_step = (long long)LA_ROWS * tiles.stride[o];
                tiles.base[o] += (BACKWARDS ? -chunk_step : chunk_step) - back * inner_step[o];
            }
        } else {
#pragma unroll
            for (int o = 0; o < OPERANDS; ++o) tiles.base[o] += inner_step[o];
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
    const unsigned a_tile = (unsigned)(places.a * Tiles::TILE), b_tile = (unsigned)(places.b * Tiles::TILE), c_tile = (unsigned)(places.c * Tiles::TILE);
    typedef const h8 __attribute__((address_space(3))) *lds_h8;
    typedef tr4 __attribute__((address_space(3))) *lds_tr4;
    auto rows = [&](unsigned tile, int s) { return *(lds_h8)(uintptr_t)(row_at[s % 4] + (tile + 4096u * (s / 4))); };
    auto columns = [&](const unsigned (&at)[2], unsigned tile) {
        const tr4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4)(uintptr_t)(at[0] + tile));
        const tr4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4)(uintptr_t)(at[1] + tile));
        return __builtin_shufflevector(__builtin_bit_cast(h4, lo), __builtin_bit_cast(h4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
    };

    // The state: value v of state[t] is row 32 t + swapped16(8 (v / 4) + 4 h + v % 4), column 32 w + perm16(i); times s_mul, a power
    // of two (bf16: HELD), over the decay of the last `age` tokens, which it has not got yet.
    f16v state[DT];
    float s_mul = BF && steps > 0 ? HELD : 1.f, o_mul = 1.f;      // o_mul: of its operands besides, where what enters is much larger than it is
    int age = 0;
    float owed = 1.f;                    // that decay
    bool shrunk = false, dwarfed = false;        // it has got some of it, or was made small for what entered: too small for fp16 operands?
    bool zero = true;                    // nothing entered so far, or (fp16) only zeros
    const int column = 32 * w + perm16(i);
    auto row_of = [&](int t, int v) { return 32 * t + swapped16(8 * (v >> 2) + (v & 3)) + 8 * h; };
    auto lane_most = [&]() {
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) most = larger(most, state[t][v]);
        return most;
    };
    auto state_most = [&]() {
        const float most = lane_most();
        return wave_most(is_finite(most) ? most : 0.f);
    };
    auto scale_state = [&](float by) {
#pragma unroll
        for (int t = 0; t < DT; ++t) state[t] *= by;
    };
    // `by` as far as s_mul may go, which is at `mul`: from where the largest state of fp32 fits fp16, to where what enters next has room in fp32
    // (2^16, 2^5 of decay, a scale of 2^16); s_mul o_mul to 2^120
    constexpr float MUL_LEAST = 0x1p-113f, MUL_MOST = 0x1p90f, MUL_LAST = 0x1p120f;
    auto reach = [&](float mul, float by, float most) {
        const float under = __builtin_amdgcn_rcpf(mul);
        return fminf(fmaxf(by, MUL_LEAST * under), most * under);
    };
    auto lift_state = [&](float most) {  // to a size that fp16 operands have room around; by how much
        const float by = most > 0.f ? reach(s_mul, lift_of(most, 8), MUL_MOST) : 1.f;
        scale_state(by);
        s_mul *= by;
        o_mul = 1.f;
        dwarfed = false;
        return by;
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
            if (BF) scale_state(s_mul);
            if (!BF && steps > 0) {      // an empty sequence's comes out as it went in
                zero = __builtin_amdgcn_ballot_w64(lane_most() > 0.f) == 0ull;
                lift_state(state_most());
            }
        }
    }

    // Decays inside a chunk of `valid` tokens, in LDS, where all waves read them: of P (zero where a token does not see the other), of
    // what enters the state.  In a register: of the state's way to this lane's token.
    float since = 0.f, p_mul = 1.f;      // p_mul: of P's operands (fp16), a power of two
    int decays_of = 0;
    float *const table = reinterpret_cast<float *>(lds_raw + LA_STAGES * Tiles::STAGE);
    auto sees = [&](int r, int valid) { return BACKWARDS ? r >= i && r < valid : r <= i; };
    auto set_decays = [&](int valid) {
        decays_of = valid;
        const int thread = (int)threadIdx.x;
        if (RESULT && thread < 2 * LA_ROWS) {
            // entry 32 + r - i: zero where token r is hidden from token i
            const int e = thread - LA_ROWS, gap = BACKWARDS ? e : -e;
            const float x = gap >= 0 ? P_LIFT * p.scale * linear_power(log2_decay, gap) : 0.f;
#pragma unroll
            for (int copy = 0; copy < 4; ++copy) table[LA_BETWEEN * copy + thread + copy] = x;
        }
        if (thread < LA_ROWS) table[4 * LA_BETWEEN + thread] = thread < valid ? sum.b_mul * linear_power(log2_decay, BACKWARDS ? thread + 1 : valid - 1 - thread) : 0.f;
        if (RESULT) since = BACKWARDS ? (i < valid ? sum.a_mul * linear_power(log2_decay, valid - 1 - i) : 0.f) : sum.a_mul * linear_power(log2_decay, i + 1);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    // of this lane: entries 32 + r - i for r = 4 h .. + 3 and on in steps of 8, from the copy that has them at a multiple of four floats
    const float *const between = table + LA_BETWEEN * (i & 3) + (LA_ROWS + 4 * h - i + (i & 3)), *const entering = table + 4 * LA_BETWEEN + 4 * h;

    // whether the walk's end state is wanted
    const bool ends = RESULT ? sum.last != nullptr && (BACKWARDS ? item.segment == 0 : item.segment == item.segments - 1) : true;

    f16v oacc;
    uint4 result[2];
    int stored = 0;                      // tokens of `result` that are to be stored
    half_t *to = nullptr;
    const long long width = (long long)p.key_heads * sum.a_inner * HD;
    half_t *const out = RESULT ? sum.out + begin * width + (long long)key_head * sum.a_inner * HD + 32 * w + 16 * h : nullptr;
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
        const int at = LA_ROWS * chunk, valid = min(here - at, LA_ROWS);
        const unsigned tile = (unsigned)(stage * Tiles::STAGE);
        if (valid != decays_of) set_decays(valid);
        if (BACKWARDS && RESULT && valid < LA_ROWS) {        // tokens behind the sequence see nothing
            for (int e = (int)threadIdx.x; e < (Tiles::STAGE / 4096) * (LA_ROWS - valid) * 8; e += WAVE * Tiles::WAVES) {
                const int in = e % ((LA_ROWS - valid) * 8), panel = e / ((LA_ROWS - valid) * 8);
                *reinterpret_cast<uint4 *>(lds_raw + tile + 4096 * panel + 128 * valid + 16 * in) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        const bool last_inner = g == inner - 1;
        const bool fresh = !BACKWARDS || g == 0;             // of a token and head: the state's part comes first
        // every head of b and c enters the state, heads of a share one; after the segment's last chunk it may not be needed
        const bool enters = (BACKWARDS || last_inner) && (ends || step + inner - g < steps);
        // Operands are read from LDS ahead of the work that hides them; the compiler left to itself waits for each.
        h8 a[KS], b[KS], cop[2], bop[4];
        f4v decays[4], enter[4];
        auto read_b_columns = [&](int t) {
#pragma unroll
            for (int s = 0; s < 4; ++s) bop[s] = columns(b_at[s / 2], tile + b_tile + 4096u * (t / 2) + 2048u * (s % 2));
        };
        auto read_rows_of = [&](int first) {
#pragma unroll
            for (int s = first; s < first + 4; ++s) {
                a[s] = rows(tile + a_tile, s);
                b[s] = rows(tile + b_tile, s);
            }
        };
        if (RESULT) read_rows_of(0);
#pragma unroll
        for (int s = 0; s < 2; ++s) cop[s] = columns(c_at, tile + c_tile + 2048u * s);
#pragma unroll
        for (int u = 0; u < 4; ++u) enter[u] = *reinterpret_cast<const f4v *>(entering + 8 * u);
        if (!RESULT) read_b_columns(0);
        issue_order();
        // P's products run while what enters the state is made
        f16v prob = {0};
        if (RESULT) {
#pragma unroll
            for (int s = 0; s < 4; ++s) prob = mfma_16<BF>(b[s], a[s], prob);
            if (KS > 4) read_rows_of(4);
#pragma unroll
            for (int u = 0; u < 4; ++u) decays[u] = *reinterpret_cast<const f4v *>(between + 8 * u);
            issue_order();
#pragma unroll
            for (int s = 4; s < KS; ++s) prob = mfma_16<BF>(b[s], a[s], prob);
        }
        // What enters the state: c with its decay, times s_mul over the decay that the state has not got.
        const int aged = zero ? 0 : BACKWARDS && g > 0 ? age : age + valid;
        const bool gets = !(__builtin_fabsf(log2_decay * (float)aged) <= PUT_OFF);           // the state gets its decay with this chunk
        const float with = gets || aged == 0 ? 1.f : at_exp2(-log2_decay * (float)aged);
        // by, more: of the state and s_mul once the state has been an operand; what enters is made for them.  Beside a state so large (2^-20: beyond
        // what fp16's own values add up to) what enters may be less than fp32's least, and the state about to decay to that, or to nothing.
        float by = 1.f, more = 1.f;
        if (!BF && enters && gets && s_mul < 0x1p-20f) {
            const float left = state_most() * linear_power(log2_decay, aged), most = __builtin_amdgcn_rcpf(s_mul);
            by = left > 0.f ? fminf(most, fmaxf(1.f, lift_of(left, 8))) : most;
        }
        float x[2][8], x_most = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const half_t one = cop[u >> 1][4 * (u & 1) + j];
                float &to_enter = x[u >> 1][4 * (u & 1) + j];
                to_enter = times<BF>(one, enter[u][j] * with * (BF ? HELD : s_mul * by));
                if (!BF) x_most = larger(x_most, to_enter);
            }
        bool some_enters = true, small = false;
        auto look_at_entering = [&](float most) {
            some_enters = __builtin_amdgcn_ballot_w64(most > 0.f) != 0ull;
            small = __builtin_amdgcn_ballot_w64(most >= 1.f) == 0ull;
        };
        auto entering_most = [&]() {
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) most = larger(most, x[s][j]);
            return most;
        };
        auto scale_entering = [&](float by) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[s][j] *= by;
            look_at_entering(entering_most());
        };
        if (!BF) look_at_entering(x_most);
        if (!BF) {                       // it has to fit, and the state with it
            if ((zero || __builtin_amdgcn_ballot_w64(x_most >= 0x1p15f) != 0ull) && enters) {
                const float all = wave_most(is_finite(x_most) ? x_most : 0.f);
                if (zero ? all > 0.f : all >= 0x1p15f) {     // infinities fit nowhere and ask for nothing
                    const float to_fit = reach(s_mul * by, lift_of(all, 10), MUL_MOST);
                    if (by != 1.f) {
                        by *= to_fit;
                    } else {
                        s_mul *= to_fit;
                        if (!zero) {
                            scale_state(to_fit);
                            dwarfed = true;
                        }
                    }
                    scale_entering(to_fit);
                }
            }
            if (RESULT && fresh && (shrunk || dwarfed)) {
                if (dwarfed) {           // operands of another size than the state, as long as it is so
                    const float left = state_most();
                    o_mul = left > 0.f && left < 16.f ? fminf(lift_of(left, 8), MUL_LAST * __builtin_amdgcn_rcpf(s_mul)) : 1.f;
                    dwarfed = o_mul != 1.f;
                } else {                 // by a part of it: what has entered since most often makes up for it
                    float some = 0.f;
#pragma unroll
                    for (int v = 0; v < 16; ++v) some = larger(some, state[0][v]);
                    if (__builtin_amdgcn_ballot_w64(some >= 16.f) == 0ull) {
                        const float left = state_most(), up = left > 0.f ? reach(s_mul * by, lift_of(left, 8), MUL_MOST) : 1.f;
                        if (__builtin_amdgcn_ballot_w64(x_most * up >= 0x1p15f) == 0ull) {
                            scale_state(up);
                            s_mul *= up;
                            scale_entering(up);
                        } else {
                            o_mul = up;
                            dwarfed = true;
                        }
                    }
                }
                shrunk = false;
            }
        }
        float up = 0.f;
        if (RESULT) {
            auto meet = [&](float by) {
                oacc = f16v{0};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    h8 op;
#pragma unroll
                    for (int j = 0; j < 8; ++j) op[j] = narrow_16<BF>(state[s / 2][8 * (s % 2) + j] * by);
                    oacc = mfma_16<BF>(op, a[s], oacc);
                }
            };
            if (fresh) {
                oacc = f16v{0};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    h8 op;
#pragma unroll
                    for (int j = 0; j < 8; ++j) op[j] = narrow_16<BF>(state[s / 2][8 * (s % 2) + j]);
                    oacc = mfma_16<BF>(op, a[s], oacc);
                }
                if (!BF) {               // a state that has outgrown fp16, or is too small for it
                    float sure = 0.f;
#pragma unroll
                    for (int v = 0; v < 16; ++v) sure += __builtin_fabsf(oacc[v]);
                    // No number: brought back, and what enters with it, only if the state has outgrown fp16.  Otherwise a token of a, or what the
                    // state got before, is no number, which says nothing about its size: what enters has been fitted to s_mul already.
                    const float most = __builtin_amdgcn_ballot_w64(!is_finite(sure)) != 0ull ? state_most() : 0.f;
                    const bool outgrown = most >= 0x1p15f;
                    if (outgrown) scale_entering(lift_state(most));
                    if (outgrown || o_mul != 1.f) meet(o_mul);
                }
                up = since * (owed * (BF ? FREED : P_LIFT * __builtin_amdgcn_rcpf(s_mul * o_mul)));      // of a power of two: exact
            }
            issue_order();
            read_b_columns(0);
            issue_order();
            store();
        }
        // while the products run: memory takes its time to accept the next chunk's requests
        if (step + 2 < steps) request();
        const bool closes = RESULT && ends && step + inner - g >= steps && g == (BACKWARDS ? 0 : inner - 1);
        if (!BF && enters && some_enters && (closes || (gets && small))) {
            // Small beside the state, but not beside what its decay leaves of it: in the backward direction it comes with that decay itself.  What
            // closes the walk is no operand any more, and may be as large as its own parts can: a state of few tokens has all its bits.
            // An infinity has its column to itself, and the others their bits: lanes that have one are left out.
            const float most = entering_most(), all = wave_most(is_finite(most) ? most : 0.f);
            if (all > 0.f) {
                more = reach(s_mul * by, lift_of(all, closes ? 14 : 10), closes ? MUL_LAST : MUL_MOST);
                // the state comes along: it stays an operand or, at the end, in fp32 (it is below 2^44)
                if (!closes || more > 0x1p60f) {
                    const float held = state_most() * ((gets ? linear_power(log2_decay, aged) : 1.f) * by);
                    more = fminf(more, fmaxf(1.f, (closes ? 0x1p100f : 0x1p14f) * __builtin_amdgcn_rcpf(held)));
                }
                scale_entering(more);
            }
        }
        h8 cw[TERMS][2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                h2 parts[TERMS];
                in_parts<BF, TERMS>(x[s][j], x[s][j + 1], parts);
#pragma unroll
                for (int e = 0; e < TERMS; ++e) cw[e][s][j] = parts[e][0], cw[e][s][j + 1] = parts[e][1];
            }
        h8 pop[2];
        f16v part = {0};
        float p_size = 0.f;
        if (RESULT) {
            if (!BF && p_mul != 1.f) {
#pragma unroll
                for (int u = 0; u < 4; ++u) decays[u] *= p_mul;
            }
#pragma unroll
            for (int v = 0; v < 16; ++v)
                pop[v >> 3][v & 7] = narrow_16<BF>(BF ? prob[v] * decays[v >> 2][v & 3] : __builtin_fmaf(prob[v], decays[v >> 2][v & 3], 0.f));
            if (!BF) {                   // the sum of their squares tells their size in half the instructions
#pragma unroll
                for (int v = 0; v < 16; v += 2) {
                    const fp16x2 two = __builtin_bit_cast(fp16x2, h2{pop[v >> 3][v & 7], pop[v >> 3][(v & 7) + 1]});
                    p_size = __builtin_amdgcn_fdot2(two, two, p_size, false);
                }
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) part = mfma_16<BF>(cop[s], pop[s], part);
        }
        if (enters) {
            if (!BF) s_mul = s_mul * by * more;
            if (gets || more != 1.f) scale_state((gets ? linear_power(log2_decay, aged) : 1.f) * by * more);      // by: of what the decay leaves
            if (!BF) shrunk = shrunk || gets;
            age = gets ? 0 : aged;
            owed = gets ? 1.f : linear_power(log2_decay, age);
            zero = !BF && zero && !some_enters;
#pragma unroll
            for (int t = 0; t < DT; t += 2) {
                const h8 now[4] = {bop[0], bop[1], bop[2], bop[3]};
                if (t + 2 < DT) read_b_columns(t + 2);
#pragma unroll
                for (int e = 0; e < TERMS; ++e)
#pragma unroll
                    for (int s = 0; s < 4; ++s) state[t + s / 2] = mfma_16<BF>(now[s], cw[e][s % 2], state[t + s / 2]);
            }
        }
        if (RESULT) {
            float sure = 0.f;
#pragma unroll
            for (int v = 0; v < 16; ++v) sure += __builtin_fabsf(part[v]);
            if (!BF) {                   // P too large for fp16, or all of it too small
                if (__builtin_amdgcn_ballot_w64(p_size >= 0x1p30f) != 0ull || __builtin_amdgcn_ballot_w64(p_size >= 0x1p8f) == 0ull) {
                    float p_most = 0.f;
#pragma unroll
                    for (int v = 0; v < 16; ++v) p_most = larger(p_most, prob[v] * between[8 * (v >> 2) + (v & 3)]);
                    const float all = wave_most(is_finite(p_most) ? p_most : 0.f);
                    if (all > 0.f) {
                        p_mul = fminf(fmaxf(lift_of(all, 8), 0x1p-60f), 0x1p60f);
#pragma unroll
                        for (int v = 0; v < 16; ++v) pop[v >> 3][v & 7] = narrow_16<BF>(prob[v] * between[8 * (v >> 2) + (v & 3)] * p_mul);
                        part = f16v{0};
#pragma unroll
                        for (int s = 0; s < 2; ++s) part = mfma_16<BF>(cop[s], pop[s], part);
                        sure = 0.f;
#pragma unroll
                        for (int v = 0; v < 16; ++v) sure += __builtin_fabsf(part[v]);
                    }
                }
            }
            if (__builtin_amdgcn_ballot_w64(!is_finite(sure)) != 0ull) {
                // An infinity or a NaN: zero times it is NaN, also for tokens that do not see it.  Weights of hidden ones are put to zero,
                // and left out of c it makes NaN of its column for those that see it.
                if (!BF) {               // beside a NaN the sum of squares is silent about weights too large for fp16
                    float p_most = 0.f;
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const float weight = prob[v] * between[8 * (v >> 2) + (v & 3)];
                        p_most = larger(p_most, is_finite(weight) ? weight : 0.f);
                    }
                    const float all = wave_most(p_most);
                    if (all * p_mul >= 0x1p15f) p_mul = fmaxf(lift_of(all, 8), 0x1p-60f);
                }
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const float weight = prob[v] * between[8 * (v >> 2) + (v & 3)] * (BF ? 1.f : p_mul);
                    pop[v >> 3][v & 7] = narrow_16<BF>(sees(8 * (v >> 2) + 4 * h + (v & 3), valid) ? weight : 0.f);
                }
                h8 clean[1][2] = {{cop[0], cop[1]}};
                take_out_not_finite<BF>(clean);
                part = f16v{0};
#pragma unroll
                for (int s = 0; s < 2; ++s) part = mfma_16<BF>(clean[0][s], pop[s], part);
                const unsigned first = __builtin_amdgcn_readfirstlane(lds_address(lds_raw)) + tile + c_tile + 4096u * (w >> 1);
#pragma unroll 1
                for (int r = 0; r < valid; ++r) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const h8 one_row = *(lds_h8)(uintptr_t)(first + 128u * r + 16u * (unsigned)((4 * (w & 1) + 2 * h + half) ^ panel_swizzle(r)));
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const half_t one = one_row[j];
                            if (sees(r, valid) && !is_finite(widen_16<BF>(one))) part[8 * half + j] = __builtin_nanf("");
                        }
                    }
                }
            }
            if (!BF && p_mul != 1.f) part *= __builtin_amdgcn_rcpf(p_mul);
            if (fresh) {
#pragma unroll
                for (int v = 0; v < 16; ++v) oacc[v] = __builtin_fmaf(oacc[v], up, part[v]);
            } else {
                oacc += part;
            }
        }
        stage = stage == LA_STAGES - 1 ? 0 : stage + 1;
        if (RESULT && (!BACKWARDS || last_inner)) {
            if (BF) {
                pack16<BF>(oacc, result[0], result[1]);
            } else {
                h8 half[2];
#pragma unroll
                for (int v = 0; v < 16; ++v) half[v >> 3][v & 7] = narrow_16<BF>(__builtin_fmaf(oacc[v], 1.f / P_LIFT, 0.f));
                result[0] = __builtin_bit_cast(uint4, half[0]), result[1] = __builtin_bit_cast(uint4, half[1]);
            }
            to = out + (long long)(at + i) * width + (BACKWARDS ? 0 : g * HD);
            stored = valid;
        }
        g = last_inner ? 0 : g + 1;
        if (last_inner) chunk += BACKWARDS ? -1 : 1;
    }
    if (RESULT) store();
    if (ends) {
        float *dst = RESULT ? sum.last + ((size_t)item.sequence * p.key_heads + key_head) * HD * HD
                            : p.states + linear_boundary(p, item.begin, BACKWARDS ? item.segment : item.segment + 1, key_head) * HD * HD;
        const float down = owed * __builtin_amdgcn_rcpf(s_mul);
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

template <int HD> using ResultTiles = LinearTiles<HD, 3, HD / 32>;
template <int HD> using StateTiles = LinearTiles<HD, 2, HD / 32>;
template <int HD> using PairSumTiles = LinearTiles<HD, 4, HD / 16>;

// the forward pass, or dq, by packed_grid workgroups and PACKED_CLEARING
template <int HD, bool BF, int TERMS>
__device__ __forceinline__ void linear_result(const LinearWalk &p, const LinearSum &sum, int block, unsigned char *lds_raw)
{
    const int cells = packed_grid(p.key_heads, p.head_sets, p.slots);
    if (block >= cells) return linear_clear(p, block - cells, sum.out, (long long)p.key_heads * sum.a_inner * HD);
    const LinearItem item = linear_item(p, block);
    if (!item.there) return;
    const long long begin = (long long)item.begin + item.segment * p.segment;
    ResultTiles<HD> tiles(lds_raw);
    tiles.set(0, sum.a, begin, item.head * sum.a_inner);
    tiles.set(1, sum.b, begin, item.head);
    tiles.set(2, sum.c, begin, item.head);
    const long long inner_step[3] = {2 * sum.a.head, 0, 0};
    linear_walk<HD, BF, TERMS, false, true>(p, sum, item, wave_id(), tiles, LinearPlaces{0, 1, 2}, inner_step, sum.a_inner, lds_raw);
}
template <int HD, bool BF, int TERMS>
__global__ __launch_bounds__(2 * HD, 2) void linear_result_kernel(LinearWalk p, LinearSum sum)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    linear_result<HD, BF, TERMS>(p, sum, (int)blockIdx.x, lds_raw);
}

// dv by the first half of the waves, dk by the others: a, b, c of dv are K, Q, dO, of dk V, dO, Q
template <int HD, bool BF, int TERMS>
__global__ __launch_bounds__(4 * HD, 2) void linear_keys_kernel(LinearWalk p, LinearSum dv, LinearSum dk)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    const int cells = packed_grid(p.key_heads, p.head_sets, p.slots);
    if ((int)blockIdx.x >= cells) {
        linear_clear(p, (int)blockIdx.x - cells, dv.out, (long long)p.key_heads * HD);
        return linear_clear(p, (int)blockIdx.x - cells, dk.out, (long long)p.key_heads * HD);
    }
    const LinearItem item = linear_item(p, (int)blockIdx.x);
    if (!item.there) return;
    const long long begin = (long long)item.begin + item.segment * p.segment;
    PairSumTiles<HD> tiles(lds_raw);
    tiles.set(0, dv.a, begin, item.head);
    tiles.set(1, dk.a, begin, item.head);
    tiles.set(2, dv.b, begin, item.head * dv.c_inner);
    tiles.set(3, dv.c, begin, item.head * dv.c_inner);
    const long long inner_step[4] = {0, 0, 2 * dv.b.head, 2 * dv.c.head};
    const int w = wave_id(), half = w / (HD / 32);
    const LinearPlaces places = half == 0 ? LinearPlaces{0, 2, 3} : LinearPlaces{1, 3, 2};
    LinearSum sum = dv;
    if (half != 0) sum = dk;
    linear_walk<HD, BF, TERMS, true, true>(p, sum, item, w % (HD / 32), tiles, places, inner_step, dv.c_inner, lds_raw);
}

// every segment's own sum, of those that have a neighbour behind (BACKWARDS: in front): b and c are read once more than the results need them,
// which costs less than a chain over the segments would
template <int HD, bool BF, int TERMS, bool BACKWARDS>
__device__ __forceinline__ void linear_segment_sum(const LinearWalk &p, const LinearSum &sum, int block, unsigned char *lds_raw)
{
    const LinearItem item = linear_item(p, block);
    if (!item.there || (BACKWARDS ? item.segment == 0 : item.segment == item.segments - 1)) return;
    const long long begin = (long long)item.begin + item.segment * p.segment;
    StateTiles<HD> tiles(lds_raw);
    tiles.set(0, sum.b, begin, item.head * sum.c_inner);
    tiles.set(1, sum.c, begin, item.head * sum.c_inner);
    const long long inner_step[2] = {2 * sum.b.head, 2 * sum.c.head};
    linear_walk<HD, BF, TERMS, BACKWARDS, false>(p, sum, item, wave_id(), tiles, LinearPlaces{0, 0, 1}, inner_step, sum.c_inner, lds_raw);
}
template <int HD, bool BF, int TERMS>
__global__ __launch_bounds__(2 * HD, 2) void linear_segments_kernel(LinearWalk p, LinearSum sum)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    linear_segment_sum<HD, BF, TERMS, false>(p, sum, (int)blockIdx.x, lds_raw);
}
// the backward pass begins with two things that do not need one another: dq, and the sums from the end; walks differ in `states` alone
template <int HD, bool BF, int TERMS>
__global__ __launch_bounds__(2 * HD, 2) void linear_queries_kernel(LinearWalk p, LinearSum dq, LinearSum dv, float *back_states)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    const int results = packed_grid(p.key_heads, p.head_sets, p.slots) + PACKED_CLEARING;
    if ((int)blockIdx.x < results) return linear_result<HD, BF, 2>(p, dq, (int)blockIdx.x, lds_raw);
    p.states = back_states;
    linear_segment_sum<HD, BF, TERMS, true>(p, dv, (int)blockIdx.x - results, lds_raw);
}

// The running sum over the segments of a sequence, in place: what each segment begins with.  A lane has four values of a state; the
// segments' sums are requested RUN_AHEAD at a time: 30 states of each of 32 heads, 64 KB a state, 11.4 us (15.6 with one value a lane).
constexpr int RUN_AHEAD = 16;
template <bool BACKWARDS>
__global__ __launch_bounds__(256) void linear_running_kernel(LinearWalk p, const float *__restrict__ first, int square)
{
    const int b = (int)blockIdx.z, key_head = (int)blockIdx.y;
    const int begin = linear_offset(p, b), n = linear_offset(p, b + 1) - begin;
    if (n <= p.segment) return;
    const int bounds = (n - 1) / p.segment;
    const float log2_decay = linear_log2(p.log_decay[key_head]);
    const size_t at = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x), stride = (size_t)p.key_heads * square;
    float *sums = p.states + linear_boundary(p, begin, 1, key_head) * square + at;
    f4v run = {0, 0, 0, 0};
    if (first != nullptr) run = *reinterpret_cast<const f4v *>(first + ((size_t)b * p.key_heads + key_head) * square + at);
    const float whole = linear_power(log2_decay, p.segment), rest = linear_power(log2_decay, n - bounds * p.segment);
    auto place = [&](int j) { return reinterpret_cast<f4v *>(sums + (size_t)(BACKWARDS ? bounds - 1 - j : j) * stride); };
    for (int j0 = 0; j0 < bounds; j0 += RUN_AHEAD) {
        f4v own[RUN_AHEAD];
#pragma unroll
        for (int e = 0; e < RUN_AHEAD; ++e) own[e] = *place(j0 + e < bounds ? j0 + e : bounds - 1);
#pragma unroll
        for (int e = 0; e < RUN_AHEAD; ++e) {
            if (j0 + e >= bounds) break;
            run = run * (BACKWARDS && j0 + e == 0 ? rest : whole) + own[e];
            *place(j0 + e) = run;
        }
    }
}

LinearWalk walk_of(const LinearArgs &a, float *states)
{
    LinearWalk p;
    p.log_decay = a.log_decay, p.offsets = a.offsets, p.states = states;
    p.tokens = a.tokens, p.sequences = a.sequences, p.key_heads = a.key_heads;
    p.segment = a.segment;
    p.slots = packed_slots(a.tokens, a.sequences, a.segment);
    p.head_sets = packed_head_sets(a.key_heads);
    p.scale = a.scale;
    return p;
}
LinearOperand operand(const void *x, long long token, long long head) { return LinearOperand{(const half_t *)x, token, head}; }

template <class Kernel, class... Sums>
hipError_t run_linear(Kernel kernel, const LinearWalk &p, int clearing, int threads, size_t lds, hipStream_t st, const Sums &...sums)
{
    if (lds > 65536) {
        const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (err != hipSuccess) return err;
    }
    kernel<<<packed_grid(p.key_heads, p.head_sets, p.slots) + clearing, threads, lds, st>>>(p, sums...);
    return hipGetLastError();
}

template <bool BACKWARDS>
hipError_t running_sums(const LinearWalk &p, const float *first, int head_dim, hipStream_t st)
{
    linear_running_kernel<BACKWARDS><<<dim3(head_dim * head_dim / 1024, p.key_heads, p.sequences), 256, 0, st>>>(p, first, head_dim * head_dim);
    return hipGetLastError();
}

template <int HD, bool BF, int TERMS>
hipError_t forward(const LinearArgs &a, hipStream_t st)
{
    const LinearWalk p = walk_of(a, a.states);
    const LinearSum sum{operand(a.q, a.q_token, a.q_head), operand(a.k, a.k_token, a.k_head), operand(a.v, a.v_token, a.v_head), (half_t *)a.out,
                        a.first, a.last, a.heads / a.key_heads, 1, false, a.scale, 1.f};
    if (a.tokens > a.segment) {
        hipError_t err = run_linear(linear_segments_kernel<HD, BF, TERMS>, p, 0, 2 * HD, StateTiles<HD>::lds_bytes(), st, sum);
        if (err == hipSuccess) err = running_sums<false>(p, a.first, HD, st);
        if (err != hipSuccess) return err;
    }
    return run_linear(linear_result_kernel<HD, BF, TERMS>, p, PACKED_CLEARING, 2 * HD, ResultTiles<HD>::lds_bytes(), st, sum);
}

template <int HD, bool BF, int TERMS>
hipError_t backward(const LinearArgs &a, hipStream_t st)
{
    const int group = a.heads / a.key_heads;
    const LinearOperand q = operand(a.q, a.q_token, a.q_head), k = operand(a.k, a.k_token, a.k_head), v = operand(a.v, a.v_token, a.v_head),
                        g = operand(a.dout, a.g_token, a.g_head);
    const LinearSum dq{g, v, k, (half_t *)a.dq, a.first, nullptr, group, 1, true, a.scale, 1.f},
        dv{k, q, g, (half_t *)a.dv, a.dlast, a.dfirst, 1, group, false, 1.f, a.scale}, dk{v, g, q, (half_t *)a.dk, a.dlast, nullptr, 1, group, true, 1.f, a.scale};
    const LinearWalk towards = walk_of(a, a.states), p = walk_of(a, a.back_states);
    hipError_t err;
    if (a.tokens > a.segment) {
        const int sums = packed_grid(p.key_heads, p.head_sets, p.slots);
        err = run_linear(linear_queries_kernel<HD, BF, TERMS>, towards, PACKED_CLEARING + sums, 2 * HD, ResultTiles<HD>::lds_bytes(), st, dq, dv, a.back_states);
        if (err == hipSuccess) err = running_sums<true>(p, a.dlast, HD, st);
    } else {
        err = run_linear(linear_result_kernel<HD, BF, 2>, towards, PACKED_CLEARING, 2 * HD, ResultTiles<HD>::lds_bytes(), st, dq);
    }
    if (err != hipSuccess) return err;
    return run_linear(linear_keys_kernel<HD, BF, TERMS>, p, PACKED_CLEARING, 4 * HD, PairSumTiles<HD>::lds_bytes(), st, dv, dk);
}

}  // namespace

// What enters the state is a 16-bit value times a decay.  Two 16-bit parts of it carry 16 bits (bf16) or 22 (fp16): with one, results would be
// 1.7 times as far off as their own rounding leaves them, with two 1.4.  States that are results themselves (fp32) take three in bf16.
static int linear_terms(const LinearArgs &a, const void *states_out) { return a.bf16 && states_out != nullptr ? 3 : 2; }

bool linear_fits(const LinearArgs &a)
{
    const long long slots = (long long)a.tokens / a.segment + a.sequences + 7;
    return (2 * (long long)a.key_heads * slots + PACKED_CLEARING) * 4 * a.head_dim < (1ll << 32) && a.sequences <= 65535;
}
size_t linear_workspace_bytes(const LinearArgs &a)
{
    if (a.tokens <= a.segment) return 0;
    return sizeof(float) * (size_t)((a.tokens - 1) / a.segment) * a.key_heads * a.head_dim * a.head_dim;
}
// Large batches: segments of which every compute unit has its workgroups at once (two at head dim 128, four at 64) and no more: a second
// generation would leave most of the machine idle at its end, and every boundary is a state to write and read.  65519 tokens, 4 key
// heads, head dim 128: 168 us with the 500 workgroups of segments of 544 tokens, 200 with 512 tokens, 195 with 800.
// Others: two walks a segment long (0.06 us a token together) and the running sum over the boundaries (0.1 us each) are shortest
// together at sqrt(1.5 length).  One sequence of 65536, a head, head dim 64: 50 us with 320 or 384 tokens, 70 with 128, 77 with 1024; six texts of 1 to
// 1500, 12 heads: 31 us with 96, 30 with 128, 41 with 32, 38 with 384.  The lengths are on the device, so this goes by their mean; up to 192 the two
// launches in front of the walk take longer than they save.
int linear_segment(int tokens, int sequences, int key_heads, int head_dim)
{
    const int room = 512 * (head_dim == 64 ? 2 : 1) / key_heads;
    const int parts = room - (sequences < room / 2 ? sequences : room / 2);
    const long long fill = ((long long)tokens + (parts > 0 ? parts : 1) - 1) / (parts > 0 ? parts : 1);
    const int mean = tokens / sequences;
    int least = 512;
    if (mean > 192) {
        least = 96;
        while (least < 512 && (long long)least * least * 2 < 3ll * mean) least += LA_ROWS;
    }
    const long long segment = (fill + LA_ROWS - 1) / LA_ROWS * LA_ROWS;
    return segment < least ? least : segment > 8192 ? 8192 : (int)segment;
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

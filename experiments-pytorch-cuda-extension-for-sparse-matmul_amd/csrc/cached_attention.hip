// Attention of N new tokens a sequence over what a paged cache holds of it and over themselves: q [B, N, Hq, D], new k and v
// [B, N, Hk, D], cache positions 0 .. lengths[b] - 1 through pages[b], the new tokens under a mask tree[b][i][j] (a chain when
// there is none).  One new token a sequence is a decode step, a tree of drafted ones the check of a draft.
//
//   S_ij = scale (q_i . y_j) s_j     y: the 8-bit values as 16-bit ones (exact), s: the scale of the token's row
//   O_i  = sum_j softmax(S)_ij t_j z_j      the scales of the values ride on the probabilities; what is rounded is
//                                           exp2(S - m) t, m from the largest exp2(S) t that the row has met
//
// The query rows of a key head (N times the heads that share it) are the columns of 32 x 32 x 16 products; a tile is 32 tokens,
// which lie in one page.  A workgroup has four waves: RG groups of 32 rows times 4 / RG groups of tiles.  RG = 1: every wave walks
// tiles of its own through registers and its own LDS, with no barrier before the end.  RG = 4: 128 rows, whose waves share the
// tile, double buffered.
// What bounds it: with few rows the cache's bytes and the way of a chunk's first ones through page table, memory and LDS (one sequence of
// 131071 int8 tokens, 2 key heads: 23 us, 3.0 TB/s; 16 of 0 to 8192 e4m3 tokens, 4 key heads: 12); with many the widening of a tile, its exponentials and the
// barrier of a step (244 rows a sequence over 48 long ones: 235 us with the join, 281 TFLOP/s; the vector pipe is busy in 35 % of
// the clocks, the matrix pipe in 11 %, and waves wait in 46 %).  At head dim 128 RG = 1 needs 5 or 6 registers more than there
// are: they are spilled.
// The work is cut where it lies: a unit is a chunk of the tiles of one sequence and key head, the chunk chosen on the device
// from the lengths so that the units fill the machine, long sequences in many, short ones in one.  A sequence in several units
// leaves (max, sum, O) of each in a workspace, which a second launch joins in the order of the chunks.
#include "attention_tiles.hpp"
#include "bsa_device.hpp"
#include "bsa_internal.hpp"
#include "cache_values.hpp"
#include "packed_tiles.hpp"
#include "../../include/bsa.h"

namespace bsa {

namespace {

constexpr int CACHED_WAVES = 4;
// Rows are taken by 32 as long as a cached tile is then widened at most twice.  Measured (us, RG = 1 against 4): 64 rows of 64
// sequences of 2000 tokens 36 / 68, of one of 8000 15 / 20; 112 rows of 64 sequences 78 / 69, at head dim 128 144 / 93; 108
// rows of 4 sequences 40 / 34, 244 rows of 48 long ones 335 / 258.  (RG = 2 lost to RG = 1 up to 64 rows, 48 us for those 36.)
constexpr int cached_row_groups(int rows) { return rows <= 64 ? 1 : 4; }
// Tiles of 32 tokens that the waves of a tile group take at a time: two where registers allow (244 rows, head dim 64: 258 us, one
// 298), one at head dim 128 (the same time, where two spilled 25 registers).
constexpr int cached_subtiles(int hd, int rg) { return rg == 1 || hd == 128 ? 1 : 2; }
// K, V and the scales of them
constexpr int cached_set_bytes(int hd, int rg) { return cached_subtiles(hd, rg) * (128 * hd + 256) + 256; }
// The reference point of a row moves once a step's exponentials sum up to more.  Over an 8-bit cache a weight is at most 2^15 then, and
// the largest was 2^lift when the point was set: fp16 keeps all bits of those down to 2^-18 of it.  48 trees over int8 caches, fp16:
// lift 6 248 us, 4 234, 0 226; lift 6 and a point that moves once the sum passes 256: 305.
constexpr float CACHED_LAZY_SUM = 256.f, CACHED_LAZY_WEIGHTS = 32768.f;
constexpr float cached_lift(bool bf) { return bf ? 0.f : 4.f; }
// Scales count in the reference point from 2^-32 on, so that exponentials without them, whose sum the row is divided by, stay
// within fp32, and up to 2^64 in bf16, so that those of other tokens do; what fp16 rows over larger ones give is infinite.
constexpr float CACHED_LEAST_SCALE = -32.f;
constexpr float cached_most_scale(bool bf) { return bf ? 64.f : 124.f; }

struct CachedOperands {
    const half_t *q, *k, *v;
    half_t *out;
    const unsigned char *keys, *values;
    const float *key_scales, *value_scales;
    const int32_t *table, *lengths;
    const unsigned char *tree;                   // [B or 1][N][N], may be null
    float *parts;                                // [units][key heads][row blocks][rows of a block][HD], then (max, sum)
    float2 *stats;
    int batch, drafts, heads, key_heads, group;
    int pages, page_shift, width;                // width: of the page table
    int rows, row_blocks, least, together, target;   // rows: drafts * group; a chunk has `least` tiles or more, a
                                                 // multiple of `together`; target: units wanted
    int step_shift;                              // log2 of the tiles of a step: a sequence's cached ones are counted up to a multiple
    int tree_batch;                              // values between the masks of two sequences, 0: one mask for all
    float scale2;
    long long q_batch, q_token, q_head, k_batch, k_token, k_head, v_batch, v_token, v_head;
};

__device__ __forceinline__ int cached_length(const CachedOperands &p, int b)
{
    const int n = p.lengths[b];
    const long long room = (long long)p.width << p.page_shift;
    return n < 0 ? 0 : n > room ? (int)room : n;
}
// inclusive sums over the lanes of a wave, by additions across lanes without LDS (they stand in front of everything else)
__device__ __forceinline__ int wave_sums(int x)
{
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);              // from 1, 2, 4 and 8 lanes below in a row of 16,
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);              // from the last lane of the row below to rows 1 and 3,
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);              // from the last lane of the lower half to the upper
    return x;
}

// the largest of lanes 32 .. 63, in lane 63
__device__ __forceinline__ float upper_half_most(float x)
{
    auto with = [&](int y) { x = fmaxf(x, __int_as_float(y)); };
    with(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x111, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x112, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x114, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x118, 0xF, 0xF, false));
    with(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x142, 0xA, 0xF, false));
    return x;
}

// How the lengths cut the work: the tiles of a chunk, as many units as wanted and none shorter than `least` tiles, and the
// sequence of a unit, or, with `unit` < 0, the units of sequence `of`.  Up to 64 sequences the lengths are loaded once.
struct CachedUnit {
    int b, len, part, parts, first, chunk;       // first: unit of part 0; chunk: its tiles; b < 0: nothing to do
};
__device__ __forceinline__ CachedUnit cached_unit(const CachedOperands &p, int unit, int of)
{
    const int l = lane_id(), drafted = (p.drafts + 31) / 32, shift = p.step_shift;
    auto held = [&](int len) { return (len + (32 << shift) - 1) >> (5 + shift) << shift; };
    auto length = [&](int b0) { return b0 + l < p.batch ? cached_length(p, b0 + l) : 0; };
    auto tiles = [&](int b0, int len) { return b0 + l < p.batch ? held(len) + drafted : 0; };
    int len = length(0);
    long long total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += WAVE)
        total += __builtin_amdgcn_readlane(wave_sums(tiles(b0, b0 == 0 ? len : length(b0))), WAVE - 1);
    const long long wanted = (total * p.key_heads * p.row_blocks + p.target - 1) / p.target;
    const int chunk = ((int)(wanted < p.least ? p.least : wanted) + p.together - 1) / p.together * p.together;
    int before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += WAVE) {
        if (b0 > 0) len = length(b0);
        const int mine = (tiles(b0, len) + chunk - 1) / chunk, upto = before + wave_sums(mine);
        const unsigned long long found = __builtin_amdgcn_ballot_w64(unit >= 0 ? upto - mine <= unit && unit < upto : b0 + l == of);
        if (found != 0ull) {
            const int at = __builtin_ctzll(found);
            const int parts = __builtin_amdgcn_readlane(mine, at), first = __builtin_amdgcn_readlane(upto, at) - parts;
            // as many units as such chunks make, but of even lengths: 48 trees over uneven sequences 239 us, 260 with a short last one
            const int length = __builtin_amdgcn_readlane(len, at), even = (held(length) + drafted + parts - 1) / parts;
            return CachedUnit{b0 + at, length, unit - first, parts, first, (even + p.together - 1) / p.together * p.together};
        }
        before = __builtin_amdgcn_readlane(upto, WAVE - 1);
    }
    return CachedUnit{-1, 0, 0, 0, 0, 0};
}

template <int HD, bool BF, int KIND, int RG>
__global__ __launch_bounds__(64 * CACHED_WAVES, 2) void cached_attention_kernel(CachedOperands p)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    constexpr int KS = HD / 16, KG = CACHED_WAVES / RG, BUFFERS = RG > 1 ? 2 : 1, THREADS = 64 * RG, SUBT = cached_subtiles(HD, RG);
    constexpr int WIDTH = cache_value_bytes(KIND), PIECES = 32 * HD * WIDTH / 16, EACH = SUBT * PIECES / THREADS;
    constexpr int TILE = 64 * HD, SET = cached_set_bytes(HD, RG), SCALES = 2 * SUBT * TILE;
    constexpr bool SCALED = KIND != CACHE_16;
    static_assert(EACH * THREADS == SUBT * PIECES && PIECES % 64 == 0, "a wave's pieces lie in one subtile");
    const float NEG_INF = -__builtin_inff();

    const int xcd = (int)(blockIdx.x & 7u), turn = (int)(blockIdx.x >> 3);
    const int rb = turn % p.row_blocks, pair = turn / p.row_blocks * 8 + xcd;    // row blocks of a chunk share an L2
    const int key_head = pair % p.key_heads, unit = pair / p.key_heads;
    const CachedUnit u = cached_unit(p, unit, 0);
    if (u.b < 0) return;
    const int b = u.b, len = u.len, chunk = u.chunk;
    // tiles of the cache; the new tokens' begin a step of their own: their values come as they are, with scale 1, and beside weights of
    // that size those of a cached tile with small values would lose bits
    const int cached = (len + 31) / 32, held = (cached + SUBT - 1) / SUBT * SUBT, tiles = held + (p.drafts + 31) / 32;
    const int begin = u.part * chunk, end = min(tiles, begin + chunk);

    const int w = wave_id(), l = lane_id(), qq = l & 31, h = l >> 5, rg = w % RG, kg = w / RG;
    const int thread = l + 64 * rg;              // among those that share a tile
    unsigned char *set0 = lds_raw + kg * BUFFERS * SET;
    const TileReader rd(set0);

    // Where the tiles of a step lie: rows of the cache, and how many of their tokens are there (0: drafts, behind the end, or on a page
    // that the cache does not have).
    struct Step {
        int t0;
        long long first[SUBT];
        int there[SUBT];
    };
    int window = -1, page_of_lane = -1;          // page numbers of 64 pages from `window` on, one a lane
    auto locate = [&](int t0) {
        Step step;
        step.t0 = t0;
#pragma unroll
        for (int s = 0; s < SUBT; ++s) {
            const int t = t0 + s;
            step.there[s] = 0;
            step.first[s] = 0;
            if (t >= cached || t >= end) continue;
            const int page_index = t >> (p.page_shift - 5);
            if (window < 0 || page_index - window >= WAVE) {
                window = page_index;
                page_of_lane = window + l < p.width ? p.table[(long long)b * p.width + window + l] : -1;
            }
            const int page = __builtin_amdgcn_readlane(page_of_lane, page_index - window);
            if (page < 0 || page >= p.pages) continue;
            step.there[s] = min(32, len - 32 * t);
            step.first[s] = (((long long)page * p.key_heads + key_head) << p.page_shift) + ((32 * t) & ((1 << p.page_shift) - 1));
        }
        return step;
    };
    auto tokens_of = [&](const Step &step, int s) {
        const int t = step.t0 + s;
        return t >= end ? 0 : t < held ? step.there[s] : min(32, p.drafts - 32 * (t - held));
    };
    auto subtile_of = [&](int i) { return SUBT == 1 ? 0 : (THREADS * i + 64 * rg) / PIECES; };
    auto load = [&](const Step &step, const unsigned char *rows, uint4 (&raw)[EACH]) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int s = subtile_of(i), piece = thread + THREADS * i - PIECES * s;
            const bool low = SUBT == 1 || s == 0;
            if ((low ? step.there[0] : step.there[SUBT - 1]) > 0)
                raw[i] = ldg16_stream(rows + (low ? step.first[0] : step.first[SUBT - 1]) * HD * WIDTH + 16 * piece);
        }
    };
    auto load_scales = [&](const Step &step, float (&raw)[SUBT]) {
        if (SCALED && rg == 0)
#pragma unroll
            for (int s = 0; s < SUBT; ++s)
                if (step.there[s] > 0) raw[s] = (l < 32 ? p.key_scales : p.value_scales)[step.first[s] + (l & 31)];
    };
    // 8 values of token r of a tile into the panels that TileReader reads
    auto put = [&](unsigned char *tile, int r, int piece, uint4 x) {
        *reinterpret_cast<uint4 *>(tile + 4096 * (piece >> 3) + 128 * r + 16 * ((piece & 7) ^ panel_swizzle(r))) = x;
    };
    // the tiles of a step in LDS, as 16-bit values; tokens that the sequence does not have are zeros, whatever the page holds
    auto stage = [&](const Step &step, const uint4 (&raw)[EACH], unsigned char *tiles_lds) {
        const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int s = subtile_of(i), piece = thread + THREADS * i - PIECES * s;
            const int has = SUBT == 1 || s == 0 ? step.there[0] : step.there[SUBT - 1];
            unsigned char *tile = tiles_lds + s * TILE;
            if (step.t0 + s >= held) continue;
            if (SCALED) {
                const int r = piece / (HD / 16), c = 2 * (piece % (HD / 16)), swap = (c >> 3) & 1;       // the panels' halves in turn: banks
                const uint4 x = r < has ? raw[i] : none;
                const h8 lo = widen_held_16<BF, KIND>(x.x, x.y), hi = widen_held_16<BF, KIND>(x.z, x.w);
                put(tile, r, c + swap, __builtin_bit_cast(uint4, swap ? hi : lo));
                put(tile, r, c + 1 - swap, __builtin_bit_cast(uint4, swap ? lo : hi));
            } else {
                const int r = piece / (HD / 8), c = piece % (HD / 8);
                put(tile, r, c, r < has ? raw[i] : none);
            }
        }
    };
    auto stage_new = [&](const Step &step, bool values, unsigned char *tiles_lds) {
#pragma unroll
        for (int s = 0; s < SUBT; ++s) {
            const int t = step.t0 + s, j0 = 32 * (t - held);
            if (t < held) continue;              // behind the last new token: zeros
            const half_t *rows = values ? p.v + b * p.v_batch + key_head * p.v_head : p.k + b * p.k_batch + key_head * p.k_head;
            const long long stride = values ? p.v_token : p.k_token;
#pragma unroll 1
            for (int piece = thread; piece < 32 * HD / 8; piece += THREADS) {
                const int r = piece / (HD / 8), c = piece % (HD / 8), j = j0 + r;
                put(tiles_lds + s * TILE, r, c, j < p.drafts ? ldg16(rows + j * stride + 8 * c) : make_uint4(0, 0, 0, 0));
            }
        }
    };
    // scales of the keys, times the call's, of the values, and behind them the largest of the values'; those of what is hidden are
    // the call's, which is not zero
    auto stage_scales = [&](const Step &step, const float (&raw)[SUBT], float *scales) {
        if (!SCALED || rg != 0) return;
#pragma unroll
        for (int s = 0; s < SUBT; ++s) {
            const bool fresh = step.t0 + s >= held, is = (l & 31) < step.there[s];
            const float x = fresh ? (l < 32 ? p.scale2 : 1.f) : is ? (l < 32 ? raw[s] * p.scale2 : raw[s]) : l < 32 ? p.scale2 : 0.f;
            scales[64 * s + l] = x;
            const float most = upper_half_most(__builtin_fabsf(x));
            if (l == 63) scales[64 * SUBT + s] = most;
        }
    };

    uint4 kraw[EACH], vraw[EACH];
    float sraw[SUBT];
    Step step = locate(begin + kg * SUBT);
    load(step, p.keys, kraw);
    load(step, p.values, vraw);
    load_scales(step, sraw);

    // query rows: row = draft * group + head of the group; those behind the last repeat it and are not stored
    const int row = 32 * (rb * RG + rg) + qq, mine = min(row, p.rows - 1), draft = mine / p.group, sub = mine - draft * p.group;
    h8 qop[KS];
    const half_t *q_row = p.q + b * p.q_batch + draft * p.q_token + (long long)(key_head * p.group + sub) * p.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) qop[s] = as_h8(ldg16(q_row + 16 * s + 8 * h));

    // Reference point of the row's exponentials, which its sum and results are relative to: the largest score, over an 8-bit cache the
    // largest score + log2(scale of the value row).  A large value row of no weight is then no measure for the others: 4096 fp16
    // tokens, one 1e4 times as large and of weight 1e-8, were off by 2.4e-3 when the largest scale was it, by 3.4e-4 as
    // without that row with this.
    float m = NEG_INF, lsum = 0.f, minus_ref = 0.f;
    float most_sum = CACHED_LAZY_SUM;            // of a step's exponentials; declared in the step it costs 30 registers more
    constexpr float LEAST_SCALE = CACHED_LEAST_SCALE, MOST_SCALE = cached_most_scale(BF);
    RowTile<HD> oacc;
    clear<HD>(oacc);
    auto scores = [&](unsigned k_tiles, f16v (&sacc)[SUBT]) {
#pragma unroll
        for (int s = 0; s < SUBT; ++s) {
            sacc[s] = f16v{0};
#pragma unroll
            for (int k = 0; k < KS; ++k) sacc[s] = mfma_16<BF>(rd.rows(k_tiles + s * TILE, k), qop[k], sacc[s]);
        }
    };
    // a step from its scores on
    auto weigh_values = [&](const Step &step, f16v (&sacc)[SUBT], unsigned set) {
        const float *scales = reinterpret_cast<const float *>(set0 + set + SCALES);
        bool partial = false;
#pragma unroll
        for (int s = 0; s < SUBT; ++s) partial = partial || step.t0 + s >= held || step.there[s] < 32;
        if (SCALED) {
            float most = scales[64 * SUBT];      // the largest value scale of the step
            if (SUBT > 1) most = fmaxf(most, scales[64 * SUBT + 1]);
            most_sum = CACHED_LAZY_WEIGHTS * __builtin_amdgcn_rcpf(__builtin_amdgcn_fmed3f(most, at_exp2(LEAST_SCALE), at_exp2(MOST_SCALE)));
        }
        unsigned sees[SUBT];                     // bit v: the key of accumulator value v is seen
        if (partial) {
            const float hidden = p.scale2 < 0.f ? __builtin_inff() : NEG_INF;    // -inf once scaled
#pragma unroll
            for (int s = 0; s < SUBT; ++s) {
                sees[s] = 0;
                const bool drafted = step.t0 + s >= held;
                const int j0 = 32 * (step.t0 + s - held), have = tokens_of(step, s);
                const unsigned char *mask = p.tree + (long long)b * p.tree_batch + (long long)draft * p.drafts + j0;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int r = 8 * (v >> 2) + 4 * h + (v & 3);
                    bool seen = r < have;
                    if (drafted && seen) seen = p.tree != nullptr ? mask[r] != 0 : j0 + r <= draft;
                    sees[s] |= seen ? 1u << v : 0u;
                }
                asm volatile("" : "+v"(sees[s]));        // as bits of one register: the compiler would keep 16 masks
#pragma unroll
                for (int v = 0; v < 16; ++v) sacc[s][v] = (sees[s] >> v) & 1u ? sacc[s][v] : hidden;
            }
        }
        auto scale_of = [&](int s, int g) {
            if (SCALED) return *reinterpret_cast<const f4v *>(scales + 64 * s + 8 * g + 4 * h);
            return f4v{p.scale2, p.scale2, p.scale2, p.scale2};
        };
        float psum;
        h8 pop[SUBT][2];
        auto exponentials = [&]() {
            psum = 0.f;
#pragma unroll
            for (int s = 0; s < SUBT; ++s)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    __builtin_amdgcn_sched_barrier(0xF);         // products may pass, reads from LDS not: 64 scales would wait in registers
                    const f4v ks = scale_of(s, g);
                    f4v vs = {1.f, 1.f, 1.f, 1.f};
                    if (SCALED) vs = *reinterpret_cast<const f4v *>(scales + 64 * s + 32 + 8 * g + 4 * h);
                    half_t pair[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float pv = at_exp2(__builtin_fmaf(sacc[s][4 * g + j], ks[j], minus_ref));
                        if (SCALED) psum += pv;
                        pair[j] = narrow_16<BF>(SCALED ? pv * vs[j] : pv);
                        pop[s][g >> 1][4 * (g & 1) + j] = pair[j];
                    }
                    if (!SCALED) psum = add_pair<BF>(pair[2], pair[3], add_pair<BF>(pair[0], pair[1], psum));
                }
        };
        exponentials();
        // A row moves its reference point by itself, so that its bits are its own: a row beside it, of NaN say, changes nothing.
        bool move = m == NEG_INF || psum > most_sum;
        if (__builtin_amdgcn_ballot_w64(move) != 0ull) {
            const int other_moves = __builtin_amdgcn_ds_bpermute((l ^ 32) << 2, (int)move);
            move = move || other_moves != 0;
            float bm = NEG_INF;
#pragma unroll
            for (int s = 0; s < SUBT; ++s)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f4v ks = scale_of(s, g);
                    f4v vs = {1.f, 1.f, 1.f, 1.f};
                    if (SCALED) vs = *reinterpret_cast<const f4v *>(scales + 64 * s + 32 + 8 * g + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float point = sacc[s][4 * g + j] * ks[j];
                        if (SCALED) point += __builtin_amdgcn_fmed3f(__builtin_amdgcn_logf(__builtin_fabsf(vs[j])), LEAST_SCALE, MOST_SCALE);
                        bm = fmaxf(bm, point);
                    }
                }
            if (SCALED) bm -= cached_lift(BF);
            bm = fmaxf(bm, at_lane_xor32(bm));
            const float m_new = move ? fmaxf(m, bm) : m;
            const float keep = m == NEG_INF ? 0.f : at_exp2(m - at_finite_or_zero(m_new));       // nothing accumulated so far: 0
            m = m_new;
            minus_ref = -at_finite_or_zero(m_new);
            lsum *= keep;
            each<HD>(oacc, [&](float x, int) { return x * keep; });
            exponentials();
        }
        lsum += psum;
#pragma unroll
        for (int s = 0; s < SUBT; ++s) {
            const unsigned v_tile = set + (SUBT + s) * TILE;
            if (weigh_tile<HD, BF>(rd, v_tile, pop[s], oacc, step.t0 + s >= held)) {
                const unsigned other = (unsigned)__builtin_amdgcn_ds_bpermute((l ^ 32) << 2, (int)sees[s]);
                const unsigned lower = h == 0 ? sees[s] : other, upper = h == 0 ? other : sees[s];
                add_not_finite<HD, BF>(rd, v_tile, oacc, [&](int r) {
                    return (((r & 4 ? upper : lower) >> (4 * (r >> 3) + (r & 3))) & 1u) != 0u;
                });
            }
        }
    };

    constexpr int ALL = KG * SUBT;
    const int rounds = (end - begin + ALL - 1) / ALL;
    for (int round = 0; round < rounds; ++round) {
        // One tile group alone needs one buffer; the next step is on its way while this one is worked on.  Making the scores of the next
        // step beside the exponentials, as the packed walk does, took 430 us where this takes 260 (48 trees of 61 drafts): with
        // the rows on their way and their scales there are too few registers.
        const unsigned set = (RG > 1 ? round & 1 : 0) * SET;
        const Step now = step;
        bool any = false;
        if (now.t0 < end) {
#pragma unroll
            for (int s = 0; s < SUBT; ++s) any = any || tokens_of(now, s) > 0;
            stage(now, kraw, set0 + set);
            stage(now, vraw, set0 + set + SUBT * TILE);
            stage_scales(now, sraw, reinterpret_cast<float *>(set0 + set + SCALES));
            stage_new(now, false, set0 + set);
            stage_new(now, true, set0 + set + SUBT * TILE);
            step = locate(now.t0 + ALL);
            load(step, p.keys, kraw);
            load(step, p.values, vraw);
            load_scales(step, sraw);
        }
        if (RG > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else wave_lds_fence();
        if (!any) continue;
        f16v sacc[SUBT];
        scores(set, sacc);
        weigh_values(now, sacc, set);
        if (RG == 1) wave_lds_fence();
    }
    lsum += at_lane_xor32(lsum);

    // join the tile groups of the workgroup: all but the first park (max, sum) and O^T in LDS
    __syncthreads();
    if constexpr (KG > 1) {
        constexpr int PARK = 2 * TILE + 256;     // O^T of a wave: 32 HD floats, and (max, sum) of 32 rows
        static_assert(CACHED_WAVES * PARK <= KG * BUFFERS * SET, "the parked results take the tiles' place");
        unsigned char *park = lds_raw + w * PARK;
        if (kg > 0) {
            each<HD>(oacc, [&](float x, int at) { return reinterpret_cast<float *>(park)[at] = x; });
            if (h == 0) reinterpret_cast<float2 *>(park + 2 * TILE)[qq] = make_float2(m, lsum);
        }
        __syncthreads();
        if (kg > 0) return;
        float most = m;
#pragma unroll
        for (int o = 1; o < KG; ++o) most = fmaxf(most, reinterpret_cast<const float2 *>(park + o * RG * PARK + 2 * TILE)[qq].x);
        const float to = at_finite_or_zero(most), own = at_exp2(m - to);
        lsum *= own;
        each<HD>(oacc, [&](float x, int) { return x * own; });
#pragma unroll
        for (int o = 1; o < KG; ++o) {
            const unsigned char *from = park + o * RG * PARK;
            const float2 st = reinterpret_cast<const float2 *>(from + 2 * TILE)[qq];
            const float f = at_exp2(st.x - to);
            lsum += st.y * f;
            each<HD>(oacc, [&](float x, int at) { return x + reinterpret_cast<const float *>(from)[at] * f; });
        }
        m = most;
    }
    if (u.parts > 1) {
        const long long block = ((long long)unit * p.key_heads + key_head) * p.row_blocks + rb;
        const long long at = block * (32 * RG) + 32 * rg + qq;
        if (row < p.rows) {
            float *part = p.parts + at * HD;
#pragma unroll
            for (int t = 0; t < HD / 32; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f4v *>(part + 32 * t + 8 * g + 4 * h) =
                        f4v{oacc[t][4 * g], oacc[t][4 * g + 1], oacc[t][4 * g + 2], oacc[t][4 * g + 3]};
            if (h == 0) p.stats[at] = make_float2(m, lsum);
        }
        return;
    }
    if (row < p.rows) {
        const float inv = lsum > 0.f || lsum != lsum ? 1.f / lsum : 0.f;
        half_t *dst = p.out + (((long long)b * p.drafts + draft) * p.heads + key_head * p.group + sub) * HD;
#pragma unroll
        for (int t = 0; t < HD / 32; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                h4 o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = narrow_16<BF>(oacc[t][4 * g + j] * inv);
                *reinterpret_cast<h4 *>(dst + 32 * t + 8 * g + 4 * h) = o;
            }
    }
}

// Joins the chunks of the rows of a sequence and key head: HD / 4 lanes a row and list, the chunks of a row dealt to `lists` lists,
// which are then joined pair by pair.  JOIN_BATCH chunks are loaded at a time: with one at a time each waited for the one before (384
// chunks: 9.8 us).  The order of the sums is given by the number of chunks and of lists.  Bound by latency: lengths, chunks, LDS.
// 256 threads a workgroup: 108 rows of 4 sequences, walk and join 28.7 us, with 512 threads 32.8, with 1024 34.3.
constexpr int JOIN_BATCH = 8, JOIN_THREADS = 256;
struct JoinPart {
    float m, sum;
    f4v acc;
    __device__ __forceinline__ void add(float om, float osum, f4v oacc)
    {
        const float top = fmaxf(m, om), to = at_finite_or_zero(top), keep = at_exp2(m - to), f = at_exp2(om - to);
        m = top;
        sum = sum * keep + osum * f;
        acc = acc * keep + oacc * f;
    }
};
template <int HD, bool BF>
__global__ __launch_bounds__(JOIN_THREADS) void cached_join_kernel(CachedOperands p, int block_rows, int lists)
{
    constexpr int LANES = HD / 4, GROUPS = JOIN_THREADS / LANES;
    __shared__ f4v sums[GROUPS][LANES];
    __shared__ float2 stats[GROUPS];
    const int rows = GROUPS / lists;                    // rows of this workgroup
    const int per = (p.rows + rows - 1) / rows, group = (int)blockIdx.x;
    const int key_head = group / per % p.key_heads, b = group / per / p.key_heads;
    const int place = (int)threadIdx.x / LANES, lane = (int)threadIdx.x % LANES, list = place % lists;
    const int row = group % per * rows + place / lists;
    const CachedUnit u = cached_unit(p, -1, b);
    if (u.parts <= 1) return;                    // the walk has stored the rows
    JoinPart mine = {-__builtin_inff(), 0.f, {0.f, 0.f, 0.f, 0.f}};
    if (row < p.rows) {
        const long long stride = (long long)p.key_heads * p.row_blocks * block_rows;
        const long long first = (((long long)u.first * p.key_heads + key_head) * p.row_blocks + row / block_rows) * block_rows + row % block_rows;
        for (int part0 = list; part0 < u.parts; part0 += JOIN_BATCH * lists) {
            float2 st[JOIN_BATCH];
            f4v x[JOIN_BATCH];
#pragma unroll
            for (int i = 0; i < JOIN_BATCH; ++i) {
                const int part = part0 + i * lists;
                const long long at = first + stride * (part < u.parts ? part : part0);
                st[i] = p.stats[at];
                x[i] = *reinterpret_cast<const f4v *>(p.parts + at * HD + 4 * lane);
            }
#pragma unroll
            for (int i = 0; i < JOIN_BATCH; ++i)
                if (part0 + i * lists < u.parts) mine.add(st[i].x, st[i].y, x[i]);
        }
    }
    for (int apart = 1; apart < lists; apart *= 2) {
        if (list % (2 * apart) == apart) {
            sums[place][lane] = mine.acc;
            if (lane == 0) stats[place] = make_float2(mine.m, mine.sum);
        }
        __syncthreads();
        if (list % (2 * apart) == 0) mine.add(stats[place + apart].x, stats[place + apart].y, sums[place + apart][lane]);
    }
    if (list != 0 || row >= p.rows) return;
    const float inv = mine.sum > 0.f || mine.sum != mine.sum ? 1.f / mine.sum : 0.f;
    const int draft = row / p.group, sub = row - draft * p.group;
    h4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = narrow_16<BF>(mine.acc[j] * inv);
    *reinterpret_cast<h4 *>(p.out + (((long long)b * p.drafts + draft) * p.heads + key_head * p.group + sub) * HD + 4 * lane) = o;
}

// ---- launchers ----------------------------------------------------------------------------------------
// Units wanted in a launch.  RG = 1: the 512 workgroups that the machine holds at once (1024: 36 us where 512 take 30, one long
// sequence a key head).  RG = 4 is better balanced with more (48 uneven sequences: 512 292 us, 768 258, 1536 250), but
// 1536 took 171 us where 768 take 157 (64 sequences of 500 to 4000 tokens, 120 rows).
constexpr int cached_units(int rg) { return rg == 1 ? 512 : 768; }
// Tiles of a chunk, 4 / 8 / 16 (us a pass).  RG = 1, two of 8 for each wave: 16 sequences of 0 to 8192 tokens, one row a head,
// 15.1 / 15.4 / 19.2, one of 131071 30.7 in each.  RG = 4, 8 steps or 4 of two: 108 rows of 4 sequences 32.1 / 28.5 / 36.3, 244 rows of 48
// long ones 235 in each.
constexpr int CACHED_LEAST = 8;

CachedOperands operands(const CachedArgs &a)
{
    CachedOperands p;
    p.q = (const half_t *)a.q, p.k = (const half_t *)a.k, p.v = (const half_t *)a.v, p.out = (half_t *)a.out;
    p.keys = (const unsigned char *)a.keys, p.values = (const unsigned char *)a.values;
    p.key_scales = a.key_scales, p.value_scales = a.value_scales;
    p.table = a.table, p.lengths = a.lengths, p.tree = a.tree;
    p.batch = a.batch, p.drafts = a.drafts, p.heads = a.heads, p.key_heads = a.key_heads, p.group = a.heads / a.key_heads;
    p.pages = a.pages, p.page_shift = a.page_shift, p.width = a.width;
    p.tree_batch = a.tree_shared ? 0 : a.drafts * a.drafts;
    // a hidden score is an infinity whose product with this is -inf: never zero (1e-30 leaves every exponent of a zero scale at 0)
    p.scale2 = a.scale == 0.f ? 1e-30f : a.scale * 1.4426950408889634f;
    p.q_batch = a.q_batch, p.q_token = a.q_token, p.q_head = a.q_head;
    p.k_batch = a.k_batch, p.k_token = a.k_token, p.k_head = a.k_head;
    p.v_batch = a.v_batch, p.v_token = a.v_token, p.v_head = a.v_head;
    p.rows = a.drafts * p.group;
    const int rg = cached_row_groups(p.rows);
    p.row_blocks = (p.rows + 32 * rg - 1) / (32 * rg);
    p.least = CACHED_LEAST;
    p.together = CACHED_WAVES / rg * cached_subtiles(a.head_dim, rg);
    p.step_shift = cached_subtiles(a.head_dim, rg) - 1;
    static_assert(cached_subtiles(64, 4) <= 2, "the logarithm above");
    p.target = cached_units(rg);
    // A sequence may have one unit more than its share of the wanted ones.  With few of them the wanted ones make room, so that all
    // run at once: 33 sequences of 300 to 16000 tokens 64 us, without 78; 64 sequences 51 and 50.
    if (rg == 1 && 2ll * a.batch * a.key_heads * p.row_blocks <= p.target) p.target -= a.batch * a.key_heads * p.row_blocks;
    p.parts = (float *)a.workspace;
    p.stats = (float2 *)(p.parts + cached_attention_parts(a) * a.head_dim);
    return p;
}

template <int HD, bool BF, int KIND, int RG>
hipError_t walk(const CachedArgs &a, hipStream_t st)
{
    const CachedOperands p = operands(a);
    constexpr size_t lds = (CACHED_WAVES / RG) * (RG > 1 ? 2 : 1) * cached_set_bytes(HD, RG);
    auto kernel = cached_attention_kernel<HD, BF, KIND, RG>;
    if (lds > 65536) {
        const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (err != hipSuccess) return err;
    }
    const long long pairs = (cached_attention_units(a) * a.key_heads + 7) / 8 * 8;
    kernel<<<(unsigned)(pairs * p.row_blocks), 64 * CACHED_WAVES, lds, st>>>(p);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess || !cached_attention_splits(a)) return err;
    // as many lists as give the machine a workgroup a compute unit
    constexpr int GROUPS = JOIN_THREADS / (HD / 4);
    int lists = 1;
    auto workgroups = [&]() { return (long long)a.batch * a.key_heads * ((p.rows + GROUPS / lists - 1) / (GROUPS / lists)); };
    while (lists < GROUPS && workgroups() < 256) lists *= 2;
    cached_join_kernel<HD, BF><<<(unsigned)workgroups(), JOIN_THREADS, 0, st>>>(p, 32 * RG, lists);
    return hipGetLastError();
}
template <int HD, bool BF, int KIND>
hipError_t walk_rows(const CachedArgs &a, hipStream_t st)
{
    const int rg = cached_row_groups(a.drafts * (a.heads / a.key_heads));
    return rg == 1 ? walk<HD, BF, KIND, 1>(a, st) : walk<HD, BF, KIND, 4>(a, st);
}
template <int HD, bool BF>
hipError_t walk_kind(const CachedArgs &a, hipStream_t st)
{
    if (a.kind == CACHE_INT8) return walk_rows<HD, BF, CACHE_INT8>(a, st);
    if (a.kind == CACHE_E4M3) return walk_rows<HD, BF, CACHE_E4M3>(a, st);
    return walk_rows<HD, BF, CACHE_16>(a, st);
}

}  // namespace

// most tiles a sequence can have
static long long most_tiles(const CachedArgs &a)
{
    const long long step = 32 * cached_subtiles(a.head_dim, cached_row_groups(a.drafts * (a.heads / a.key_heads)));
    return (((long long)a.width << a.page_shift) + step - 1) / step * (step / 32) + (a.drafts + 31) / 32;
}
bool cached_attention_splits(const CachedArgs &a) { return most_tiles(a) > CACHED_LEAST; }
// Most units (of all sequences) a launch can have: the chunk is at least total key_heads row_blocks / target, so that the whole
// chunks are at most target / (key_heads row_blocks), and every sequence has one that is not.
long long cached_attention_units(const CachedArgs &a)
{
    const int rows = a.drafts * (a.heads / a.key_heads), rg = cached_row_groups(rows), blocks = (rows + 32 * rg - 1) / (32 * rg);
    return a.batch + (cached_attention_splits(a) ? cached_units(rg) / (a.key_heads * blocks) : 0);
}
long long cached_attention_parts(const CachedArgs &a)
{
    if (!cached_attention_splits(a)) return 0;
    const int rows = a.drafts * (a.heads / a.key_heads), rg = cached_row_groups(rows), blocks = (rows + 32 * rg - 1) / (32 * rg);
    return cached_attention_units(a) * a.key_heads * blocks * 32 * rg;
}
size_t cached_attention_workspace_bytes(const CachedArgs &a)
{
    return (size_t)cached_attention_parts(a) * (a.head_dim + 2) * sizeof(float);
}

hipError_t launch_cached_attention(const CachedArgs &a, hipStream_t st)
{
    if (a.head_dim == 64) return a.bf16 ? walk_kind<64, true>(a, st) : walk_kind<64, false>(a, st);
    return a.bf16 ? walk_kind<128, true>(a, st) : walk_kind<128, false>(a, st);
}

}  // namespace bsa

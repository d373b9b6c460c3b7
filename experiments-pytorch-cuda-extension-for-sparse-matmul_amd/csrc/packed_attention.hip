// Causal (or full) attention over sequences of different lengths packed along the tokens, with grouped heads, and its gradients:
// q [T, Hq, D], k and v [T, Hk, D], sequence b = rows offsets[b] .. offsets[b + 1] - 1, query head h over key head h / (Hq / Hk).
//
// One workgroup holds 32 W query rows of one head; its W waves share tiles of 64 keys and values in LDS (double buffered, loaded
// straight to LDS, one barrier a tile), and each wave has 32 of the rows:
//   S^T = K Q^T             a lane holds ONE query column and 32 of the 64 keys (the others sit in lane ^ 32)
//   online softmax          per-lane reference point and sum; the point moves only when a tile's sum of exponentials passes 256
//   O^T += V^T P^T          the probabilities go from accumulators to operands without leaving the registers
// What bounds it: a tile has 32 exponentials a lane (8 clocks each, as much again for scaling, rounding and sums) beside 16 products of 32
// clocks at head dim 64 and 32 at 128, so the scores of the next tile are made beside the exponentials of this one, and two waves a
// SIMD fill what is left.  Causal, 16384 tokens, 16 heads at head dim 64: 611 to 632 us, 870 to 900 TFLOP/s; sequences of 4096 to 97 tokens at head
// dim 128: 108 to 112 us, 860 to 890 TFLOP/s (a library product of 8192^3 1217 on the same card).  W = 4: eight waves, which read K and V
// half as often, took 124 us for those 112 and 660 for 620: twice as many waves wait at a barrier, and half as many workgroups share
// the uneven rows.
//
// The lengths stay on the device: a launch has slots for the most tiles that T tokens in B sequences can make, and every workgroup
// finds its sequence by a search over the offsets.  Slots that no sequence uses end at once.  Offsets are clamped to [0, T]
// before anything is addressed with them.
#include "attention_tiles.hpp"
#include "bsa_device.hpp"
#include "bsa_internal.hpp"
#include "packed_tiles.hpp"
#include "../../include/bsa.h"

namespace bsa {

namespace {

constexpr float PACKED_LAZY_SUM = 256.f;         // fp16 holds what stays below it

// TRAIN: the row statistics and the result's rest are wanted.  The result is normalised by the sum of the rounded probabilities, so that
// their common error cancels; the statistics are of the exponentials before that, which is what the backward walks make again.
template <int HD, bool BF, int W, bool TRAIN>
__global__ __launch_bounds__(64 * W, 2) void packed_forward_kernel(PackedOperands p)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    constexpr int KS = HD / 16, ROWS = 32 * W;
    const int cells = packed_grid(p.heads, p.head_sets, p.slots);
    if ((int)blockIdx.x >= cells) return packed_clear(p, (int)blockIdx.x - cells, p.out, (long long)p.heads * HD);
    const PackedItem item = packed_item<ROWS>(p, p.heads, false);
    if (item.n == 0) return;
    const int w = wave_id(), l = lane_id(), qq = l & 31, h = l >> 5, n = item.n, key_head = item.head / p.group;
    const int row0 = item.tile * ROWS + 32 * w, row = row0 + qq;                 // rows and keys count from the sequence's start
    const long long begin = item.begin;
    const float NEG_INF = -__builtin_inff();

    PairTiles<HD, W, 2> tiles(p.k + begin * p.k_token + key_head * p.k_head, p.k_token,
                           p.v + begin * p.v_token + key_head * p.v_head, p.v_token, lds_raw);
    const int last_row = min(n, item.tile * ROWS + ROWS) - 1;
    const int steps = p.causal ? last_row / 64 + 1 : (n + 63) / 64;
    tiles.request(0, 0, n, 0);

    h8 qop[KS];
    const half_t *q_row = p.q + (begin + min(row, n - 1)) * p.q_token + item.head * p.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) qop[s] = as_h8(ldg16(q_row + 16 * s + 8 * h));
    loaded(qop);

    // reference point of the query (both lane halves agree), minus it (0 while nothing was seen), this half's sum
    float m = NEG_INF, minus_m = 0.f, lsum = 0.f, exact_sum = 0.f;
    RowTile<HD> oacc;
    clear<HD>(oacc);

    auto scores = [&](int buffer, f16v (&sacc)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            h8 kop[KS];
            read_rows<HD>(tiles.rd, tiles.at(buffer, 0, u), kop);
            sacc[u] = f16v{0};
            product<BF>(kop, qop, sacc[u]);
        }
    };
    float psum, pexact;
    h8 pop[2][2];
    auto exponentials = [&](const f16v (&sacc)[2], float mul) {
        psum = 0.f, pexact = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int v = 0; v < 16; v += 2) {
                const float p0 = at_exp2(__builtin_fmaf(sacc[u][v], mul, minus_m)), p1 = at_exp2(__builtin_fmaf(sacc[u][v + 1], mul, minus_m));
                pop[u][v >> 3][v & 7] = narrow_16<BF>(p0);
                pop[u][v >> 3][(v & 7) + 1] = narrow_16<BF>(p1);
                psum = add_pair<BF>(pop[u][v >> 3][v & 7], pop[u][v >> 3][(v & 7) + 1], psum);
                if (TRAIN) pexact += p0 + p1;
            }
    };
    // A row moves its reference point by itself, so that its bits are its own: a row beside it, of NaN say, changes nothing.
    auto settle = [&](const f16v (&sacc)[2], float mul) {
        bool move = m == NEG_INF || psum > PACKED_LAZY_SUM;
        if (__builtin_amdgcn_ballot_w64(move) != 0ull) {
            const int other_moves = __builtin_amdgcn_ds_bpermute((l ^ 32) << 2, (int)move);
            move = move || other_moves != 0;
            float bm = sacc[0][0] * mul;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int v = 0; v < 16; ++v) bm = fmaxf(bm, sacc[u][v] * mul);
            bm = fmaxf(bm, at_lane_xor32(bm));
            const float m_new = move ? fmaxf(m, bm) : m;
            const float keep = m == NEG_INF ? 0.f : at_exp2(m - at_finite_or_zero(m_new));       // nothing accumulated so far: 0
            m = m_new;
            minus_m = -at_finite_or_zero(m_new);
            lsum *= keep, exact_sum *= keep;
            each<HD>(oacc, [&](float x, int) { return x * keep; });
            exponentials(sacc, mul);
        }
        lsum += psum, exact_sum += pexact;
    };
    // Round r has the keys of tile r and the values of tile r - 1, in buffer r % 2.
    auto enter = [&](int r) {
        tiles.arrived();
        if (r >= steps) return;
        if (r + 1 < steps) tiles.request(0, r + 1, n, (r & 1) ^ 1);
        tiles.request(1, r, n, (r & 1) ^ 1);
    };
    // a tile that all queries of the wave see whole; the scores of the next one are made beside its exponentials
    auto whole_tile = [&](int r, int buffer, const f16v (&sacc)[2], f16v (&next)[2]) {
        enter(r);
        scores(buffer, next);
        exponentials(sacc, p.scale2);
        settle(sacc, p.scale2);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            h8 vop[HD / 32][2];
            read_columns<HD>(tiles.rd, tiles.at(buffer, 1, u), vop);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < HD / 32; ++t) oacc[t] = mfma_16<BF>(vop[t][s], pop[u][s], oacc[t]);
        }
    };
    const int mine = row0 >= n ? 0 : p.causal ? min(steps, (row0 + 31) / 64 + 1) : steps;        // tiles that this wave needs
    const int whole = row0 >= n ? 0 : p.causal ? (row0 + 1) / 64 : n / 64;                       // that are whole to it
    f16v sacc[2], next[2];
    enter(0);
    if (mine > 0) scores(0, sacc);
    int r = 1;
    for (; r + 1 <= whole; r += 2) {
        whole_tile(r, 1, sacc, next);
        whole_tile(r + 1, 0, next, sacc);
    }
    if (r <= whole) {
        whole_tile(r, 1, sacc, next);
        sacc[0] = next[0], sacc[1] = next[1];
        ++r;
    }
    for (; r <= mine; ++r) {                     // the last ones, with places that are hidden
        enter(r);
        const int seen = (p.causal ? min(row, n - 1) : n - 1) - 64 * (r - 1);    // last key of the tile that the query sees
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int v = 0; v < 16; ++v)         // -inf only once scaled, whatever the scale's sign
                sacc[u][v] = 32 * u + 8 * (v >> 2) + (v & 3) > seen - 4 * h ? NEG_INF : sacc[u][v] * p.scale2;
        exponentials(sacc, 1.f);
        settle(sacc, 1.f);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (weigh_tile<HD, BF>(tiles.rd, tiles.at(r & 1, 1, u), pop[u], oacc, true))
                add_not_finite<HD, BF>(tiles.rd, tiles.at(r & 1, 1, u), oacc, [&](int at) { return 32 * u + at <= seen; });
        if (r < mine) scores(r & 1, sacc);
    }
    for (; r <= steps; ++r) enter(r);            // of the rows below
    lsum += at_lane_xor32(lsum);                 // both halves used the same reference point
    const bool any = lsum > 0.f || lsum != lsum;
    if (TRAIN) exact_sum += at_lane_xor32(exact_sum);
    if (TRAIN && h == 0 && row < n)              // log2 of the row's sum, +inf for a row that sees nothing
        p.lse[(size_t)item.head * p.tokens + begin + row] =
            any ? at_finite_or_zero(m) + __builtin_amdgcn_logf(exact_sum) : __builtin_inff();
    __syncthreads();                             // all are done with the tiles, whose place the results take
    store_token_rows<HD, BF>(oacc, any ? 1.f / lsum : 0.f, lds_raw + 64 * HD * w,
                             p.out + ((begin + row0) * p.heads + item.head) * HD, (long long)p.heads * HD, n - row0);
    if (TRAIN)
        store_token_rows<HD, BF, true>(oacc, any ? 1.f / lsum : 0.f, lds_raw + 64 * HD * w,
                                       p.rest + ((begin + row0) * p.heads + item.head) * HD, (long long)p.heads * HD, n - row0);
}

// ---------------------------------------------------------------------------
// Gradients, as two walks that each rebuild the probabilities from the row statistics and write every result once (no atomics:
// the same bits every time):
//   rows      as the forward walk:  P = exp2(scale2 S - lse),  dS = P (dO V^T - delta),  dq^T += K^T dS^T;
//             delta = rowsum(dO O) is made here, O with what its rounding took, and left for the other walk.  From the rounded O
//             alone its error moves a whole row of dS the same way: dq and dk were 1.6 times as far from float64 as their own
//             rounding leaves them, with it 1.46, at no time that could be measured, and 1.44 with the statistics of the exponentials
//             before they are rounded (1 % of a training step).  dS itself in 16 bits gives 1.42 of that; its low parts as a
//             second operand would leave 1.05 but take 8 % (bf16, head dim 64)
//   columns   a workgroup holds 64 keys of one key head and walks the queries of all heads that share it:
//             dv^T += dO^T P,  dk^T += Q^T dS
// Sequences of 4096, 2976 and 1119 tokens, 16 heads over 4, head dim 128 (55 GFLOP a product): forward 135 to 140 us, rows 197 to 205, columns 311
// to 319 (800, 820 and 700 TFLOP/s); 12 heads at head dim 64, six sequences of 1 to 1500 tokens 27, 39 and 36 us, one
// generation of workgroups, as long as the 24 steps of the longest sequence.  Rows have the forward walk's bounds with three products to the exponentials' one.
// ---------------------------------------------------------------------------
// fp16 holds dS only times a power of two: with gradients of 1e-3 and 4096 keys dS is 3e-6, a few steps of fp16's smallest, and
// dq was 5.1 times as far off as its own rounding leaves it, now 1.2; above 65504 it was infinite where dq is not.  A row takes the
// power from the largest dS of the first keys it sees, so that that is below 2^4, and a smaller one once one would pass
// 2^15.  The walk over the keys does the same for dk, where the error was 47 times that of dk's own rounding,
// now 1.3.  A training step of the first case above 648 us, without both 638.
constexpr float DS_MOST = 0x1p15f, DS_LAZY_SQUARES = DS_MOST * DS_MOST;
__device__ __forceinline__ float ds_lift(float most)              // where all are hidden or zero: the largest, there is room downwards only
{
    return most == 0.f ? 40.f : fminf(4.f - (float)__builtin_amdgcn_frexp_expf(most), 40.f);
}

template <int HD, bool BF, int W>
__global__ __launch_bounds__(64 * W, 2) void packed_rows_kernel(PackedOperands p)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    constexpr int KS = HD / 16, ROWS = 32 * W;
    const int cells = packed_grid(p.heads, p.head_sets, p.slots);
    if ((int)blockIdx.x >= cells) return packed_clear(p, (int)blockIdx.x - cells, p.out, (long long)p.heads * HD);
    const PackedItem item = packed_item<ROWS>(p, p.heads, false);
    if (item.n == 0) return;
    const int w = wave_id(), l = lane_id(), qq = l & 31, h = l >> 5, n = item.n, key_head = item.head / p.group;
    const int row0 = item.tile * ROWS + 32 * w, row = row0 + qq;
    const long long begin = item.begin;

    PairTiles<HD, W, 2> tiles(p.k + begin * p.k_token + key_head * p.k_head, p.k_token,
                           p.v + begin * p.v_token + key_head * p.v_head, p.v_token, lds_raw);
    const int last_row = min(n, item.tile * ROWS + ROWS) - 1;
    const int steps = p.causal ? last_row / 64 + 1 : (n + 63) / 64;
    tiles.request(0, n, 0);

    h8 qop[KS], dop[KS];
    float delta = 0.f;
    const long long token = begin + min(row, n - 1);
    const half_t *q_row = p.q + token * p.q_token + item.head * p.q_head, *g_row = p.dout + token * p.g_token + item.head * p.g_head,
                 *o_row = p.o + (token * p.heads + item.head) * HD, *rest_row = p.o_rest + (token * p.heads + item.head) * HD;
    const float minus_lse = -p.lse[(size_t)item.head * p.tokens + token];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        qop[s] = as_h8(ldg16(q_row + 16 * s + 8 * h));
        dop[s] = as_h8(ldg16(g_row + 16 * s + 8 * h));
        const h8 o = as_h8(ldg16(o_row + 16 * s + 8 * h)), rest = as_h8(ldg16(rest_row + 16 * s + 8 * h));
#pragma unroll
        for (int j = 0; j < 8; ++j) delta += widen_16<BF>(dop[s][j]) * (widen_16<BF>(o[j]) + widen_16<BF>(rest[j]));
    }
    delta += at_lane_xor32(delta);               // the other half of the head dim sits in lane ^ 32
    // Rows whose keys all lie in the first tile make their delta again as sum P dP, of their own probabilities: with few keys the
    // rounding of the forward pass's probabilities, which O has, weighs most (a bf16 batch of short sequences: dq and dk 1.65 times as far
    // off as their own rounding, so 1.35; 37 tokens 1.48 and 1.446, which is dS's to three digits).  One more look at one tile, by the
    // waves that have the fewest: 1 % of a training step.
    const bool few = (p.causal ? min(row0 + 32, n) : n) <= 64;
    if (!few && h == 0 && row < n) p.delta[(size_t)item.head * p.tokens + token] = delta;
    loaded(qop);
    loaded(dop);

    RowTile<HD> dq;
    clear<HD>(dq);
    float lift = BF ? 0.f : __builtin_inff();    // dS of the row and dq are times 2^lift; not chosen yet
    for (int step = 0; step < steps; ++step) {
        const int k0 = 64 * step;
        const int buffer = step & 1;
        tiles.arrived();
        if (step + 1 < steps) tiles.request(step + 1, n, buffer ^ 1);
        if (row0 >= n || (p.causal && k0 > row0 + 31)) continue;
        const bool masked = k0 + 64 > n || (p.causal && k0 + 63 > row0);
        const int seen = (p.causal ? min(row, n - 1) : n - 1) - k0;
        if (few) {
            delta = 0.f;
#pragma unroll 1
            for (int u = 0; u < 2; ++u) {
                f16v sacc = {0}, dpacc = {0};
                h8 op[KS];
                read_rows<HD>(tiles.rd, tiles.at(buffer, 0, u), op);
                product<BF>(op, qop, sacc);
                read_rows<HD>(tiles.rd, tiles.at(buffer, 1, u), op);
                product<BF>(op, dop, dpacc);
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const float part = at_exp2(__builtin_fmaf(sacc[v], p.scale2, minus_lse)) * dpacc[v];
                    delta += 32 * u + 8 * (v >> 2) + (v & 3) > seen - 4 * h ? 0.f : part;
                }
            }
            delta += at_lane_xor32(delta);
            if (h == 0 && row < n) p.delta[(size_t)item.head * p.tokens + token] = delta;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f16v sacc = {0}, dpacc = {0};
            h8 ktr[HD / 32][2], ds[2];
            {
                h8 kop[KS], vop[KS];
                read_rows<HD>(tiles.rd, tiles.at(buffer, 0, u), kop);
                read_rows<HD>(tiles.rd, tiles.at(buffer, 1, u), vop);
                issue_order();
                product<BF>(kop, qop, sacc);
                product<BF>(vop, dop, dpacc);
            }
            read_columns<HD>(tiles.rd, tiles.at(buffer, 0, u), ktr);
            issue_order();
            const float up = BF ? minus_lse : minus_lse + lift;
            float squares = 0.f;
            auto gradient = [&](int v, float minus, bool some_hidden) {  // a hidden score has no probability and no gradient, whatever it is
                const float grad = at_exp2(__builtin_fmaf(sacc[v], p.scale2, minus)) * (dpacc[v] - delta);
                return some_hidden && 32 * u + 8 * (v >> 2) + (v & 3) > seen - 4 * h ? 0.f : grad;
            };
            auto gradients = [&](float minus, bool some_hidden) {
#pragma unroll
                for (int v = 0; v < 16; v += 2) {
                    const half_t a = narrow_16<BF>(gradient(v, minus, some_hidden)), b = narrow_16<BF>(gradient(v + 1, minus, some_hidden));
                    ds[v >> 3][v & 7] = a;
                    ds[v >> 3][(v & 7) + 1] = b;
                    if (!BF) squares = __builtin_amdgcn_fdot2(h2{a, b}, h2{a, b}, squares, false);
                }
            };
            if (masked) gradients(up, true);
            else gradients(up, false);
            bool move = !BF && !(squares <= DS_LAZY_SQUARES);
            if (__builtin_amdgcn_ballot_w64(move) != 0ull) {
                const int other_moves = __builtin_amdgcn_ds_bpermute((l ^ 32) << 2, (int)move);
                move = move || other_moves != 0;
                float most = 0.f;
#pragma unroll
                for (int v = 0; v < 16; ++v) most = fmaxf(most, __builtin_fabsf(gradient(v, minus_lse, masked)));
                most = fmaxf(most, at_lane_xor32(most));
                const float to = move ? fminf(lift, ds_lift(most)) : lift, keep = move ? at_exp2(to - lift) : 1.f;
                lift = to;
                each<HD>(dq, [&](float x, int) { return x * keep; });
                // those of rows that stay are kept: made again, with another choice of fused instructions, they may differ by a bit
                const h8 kept[2] = {ds[0], ds[1]};
                gradients(minus_lse + lift, masked);
#pragma unroll
                for (int s = 0; s < 2; ++s) ds[s] = move ? ds[s] : kept[s];
            }
            if (weigh<HD, BF>(ktr, ds, dq, masked))
                add_not_finite<HD, BF>(tiles.rd, tiles.at(buffer, 0, u), dq, [&](int at) { return 32 * u + at <= seen; });
            issue_order();
        }
    }
    __syncthreads();
    store_token_rows<HD, BF>(dq, BF ? p.scale : p.scale * at_exp2(-lift), lds_raw + 64 * HD * w, p.out + ((begin + row0) * p.heads + item.head) * HD,
                             (long long)p.heads * HD, n - row0);
}

// A workgroup has two tiles of 32 keys, each wave one of them for one of the SUB subtiles of 32 queries of a tile; the subtiles'
// parts add up in LDS at the end.  128 queries a tile at head dim 128, 64 at 64.  K stays in registers, V in LDS: with the
// accumulators they would leave too few for two waves a SIMD at head dim 128 (256 registers each, none spilled: what is spilled
// is waited for behind the tiles on their way).  One wave a SIMD with 512 registers and both key tiles, which reads Q and dO half
// as often, took 430 us where this took 338, now 311 to 319 (sequences of 4096, 2976 and 1119 tokens, 16 heads over 4, 700 TFLOP/s of the four
// products): nothing runs beside what a wave waits for.  What bounds it: a step of the workgroup takes 6.3k clocks, of which the
// products fill 2.0k, LDS 2.6k (Q and dO are read both ways) and the exponentials 1.0k, and the two waves of a SIMD, which the barrier
// keeps in step, overlap little of it; and the first keys of the longest sequence have 128 steps where a compute unit has 106 on
// average.  A static priority for one of the two waves changed nothing (622 us a training step for 619).
// Behind the tiles of PairTiles: lse and delta of a tile's queries, per buffer, and the workgroup's V.
template <int HD, bool BF, int SUB>
__global__ __launch_bounds__(128 * SUB, 2) void packed_columns_kernel(PackedOperands p)
{
    extern __shared__ __align__(16) unsigned char lds_raw[];
    constexpr int KS = HD / 16, ROWS = 64, TOKENS = 32 * SUB, W = 2 * SUB;
    using Tiles = PairTiles<HD, W, SUB>;
    const int key_heads = p.heads / p.group;
    const int cells = packed_grid(key_heads, p.head_sets, p.slots);
    if ((int)blockIdx.x >= cells) {
        packed_clear(p, (int)blockIdx.x - cells, p.dk, (long long)key_heads * HD);
        return packed_clear(p, (int)blockIdx.x - cells, p.dv, (long long)key_heads * HD);
    }
    const PackedItem item = packed_item<ROWS>(p, key_heads, p.causal);
    if (item.n == 0) return;
    const int w = wave_id(), sub = w % SUB, l = lane_id(), kk = l & 31, h = l >> 5, n = item.n, tile0 = item.tile * ROWS;
    const int key0 = tile0 + 32 * (w / SUB), key = key0 + kk;                     // of this wave, of this lane
    const long long begin = item.begin;

    constexpr unsigned V_TILES = (unsigned)Tiles::lds_bytes() + 16 * TOKENS;
    const unsigned v_tile = V_TILES + w / SUB * Tiles::TILE;
    const int there = min(key0, n - 1);
    if (sub == 0)
        request_rows<HD>(p.v + (begin + there) * p.v_token + item.head * p.v_head, p.v_token, n - there,
                         __builtin_amdgcn_readfirstlane(lds_address(lds_raw)) + v_tile);
    h8 kop[KS];
    const half_t *k_row = p.k + (begin + min(key, n - 1)) * p.k_token + item.head * p.k_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) kop[s] = as_h8(ldg16(k_row + 16 * s + 8 * h));
    loaded(kop);
    RowTile<HD> dk, dv;
    clear<HD>(dk);
    clear<HD>(dv);

    const int first = p.causal ? tile0 / TOKENS : 0, last = (n + TOKENS - 1) / TOKENS, steps = (last - first) * p.group;
    float *stats = reinterpret_cast<float *>(lds_raw + Tiles::lds_bytes());      // [2][lse, delta][TOKENS]
    const unsigned stats_lds = __builtin_amdgcn_readfirstlane(lds_address(stats));
    const int head0 = item.head * p.group;
    Tiles tiles(p.q + begin * p.q_token + head0 * p.q_head, p.q_token, p.dout + begin * p.g_token + head0 * p.g_head, p.g_token, lds_raw);
    constexpr int STAT_WAVES = TOKENS / WAVE;    // waves that fetch lse and delta of 64 queries each
    const float *lse = p.lse + (size_t)head0 * p.tokens + begin, *delta = p.delta + (size_t)head0 * p.tokens + begin;
    int next = first;                            // of the step requested next, whose head is in the pointers
    auto request = [&](int buffer) {
        tiles.request(next, n, buffer);
        if (w < STAT_WAVES) {
            const int query = min(TOKENS * next + WAVE * w + l, n - 1);
            dma4_gather(lse + query, stats_lds + 8 * TOKENS * buffer + 256 * w);
            dma4_gather(delta + query, stats_lds + 8 * TOKENS * buffer + 4 * TOKENS + 256 * w);
        }
        if (++next == last) {
            next = first;
            tiles.base[0] += 2 * p.q_head, tiles.base[1] += 2 * p.g_head, lse += p.tokens, delta += p.tokens;
        }
    };
    // fp16 probabilities of long sequences would be subnormal: they travel times 256
    constexpr float UP = BF ? 1.f : 256.f, DOWN = 1.f / UP, LOG_UP = BF ? 0.f : 8.f;
    // dS and dk of the key: times this, a power of two as in the row walk; not chosen yet
    float ds_mul = BF ? 1.f : __builtin_inff();

    request(0);
    int q_tile = first;
    for (int step = 0; step < steps; ++step) {
        const int buffer = step & 1, at = TOKENS * q_tile + 32 * sub;            // first query of this wave
        // Some wave has hidden places in this tile: see the products with such places in packed_tiles.hpp.  A dO that is no number is
        // cleaned out of the tile, and its delta, which is none either, moves into the lse.
        const bool masked = TOKENS * q_tile + TOKENS > n || (p.causal && TOKENS * q_tile < tile0 + ROWS);
        if (masked) {
            tiles.template clean<BF>(buffer);
            if (w < STAT_WAVES) {
                float *mine = stats + 2 * TOKENS * buffer + WAVE * w + l;
                const float d = mine[TOKENS];
                if (!(__builtin_fabsf(d) < __builtin_inff())) {
                    mine[0] = __builtin_nanf("");
                    mine[TOKENS] = 0.f;
                }
            }
        }
        tiles.arrived();
        if (step + 1 < steps) request(buffer ^ 1);
        q_tile = q_tile + 1 < last ? q_tile + 1 : first;

        const float *stat_lds = stats + 2 * TOKENS * buffer + 32 * sub;
        const unsigned q_at = tiles.at(buffer, 0, sub), do_at = tiles.at(buffer, 1, sub);
        f16v prob = {0}, dpacc = {0};
        {
            h8 op[KS];
            read_rows<HD>(tiles.rd, q_at, op);
            product<BF>(op, kop, prob);
        }
        {
            h8 op[KS];
            read_rows<HD>(tiles.rd, do_at, op);
#pragma unroll
            for (int s = 0; s < KS; ++s) dpacc = mfma_16<BF>(op[s], tiles.rd.rows(v_tile, s), dpacc);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f4v ls = *reinterpret_cast<const f4v *>(stat_lds + 8 * g + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) prob[4 * g + j] = at_exp2(__builtin_fmaf(prob[4 * g + j], p.scale2, LOG_UP - ls[j]));
        }
        if (masked) {
            int low = (p.causal ? key : 0) - at - 4 * h, high = n - at - 4 * h;  // queries of the subtile that see the key
            asm volatile("" : "+v"(low));        // the comparisons stay here: the compiler would keep 16 masks through the walk
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int r = 8 * (v >> 2) + (v & 3);
                prob[v] = ((r < low) | (r >= high)) ? 0.f : prob[v];
            }
        }
        h8 pop[2], ds[2];
        float most = 0.f;                        // largest dS of the lane
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f4v dl = *reinterpret_cast<const f4v *>(stat_lds + TOKENS + 8 * g + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int v = 4 * g + j;
                pop[v >> 3][v & 7] = narrow_16<BF>(prob[v]);
                dpacc[v] = prob[v] * (dpacc[v] - dl[j]);
                if (!BF) most = fmaxf(most, __builtin_fabsf(dpacc[v]));
            }
        }
        bool move = !BF && !(most * ds_mul <= DS_MOST);
        if (__builtin_amdgcn_ballot_w64(move) != 0ull) {
            const int other_moves = __builtin_amdgcn_ds_bpermute((l ^ 32) << 2, (int)move);
            move = move || other_moves != 0;
            most = fmaxf(most, at_lane_xor32(most));
            const float to = move ? fminf(ds_mul, at_exp2(ds_lift(most))) : ds_mul, keep = move ? to * __builtin_amdgcn_rcpf(ds_mul) : 1.f;
            ds_mul = to;
            issue_order();                       // one accumulator after the other: all at once spill 14 registers, 12 of them K's
#pragma unroll
            for (int t = 0; t < HD / 32; ++t) {
                dk[t] *= keep;
                issue_order();
            }
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) ds[v >> 3][v & 7] = narrow_16<BF>(BF ? dpacc[v] : dpacc[v] * ds_mul);
#pragma unroll
        for (int t = 0; t < HD / 32; ++t) {
            h8 qc[2], dc[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                qc[s] = tiles.rd.columns(q_at, t, s);
                dc[s] = tiles.rd.columns(do_at, t, s);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                dk[t] = mfma_16<BF>(qc[s], ds[s], dk[t]);
                dv[t] = mfma_16<BF>(dc[s], pop[s], dv[t]);
            }
        }
    }
    // the parts of a key tile add up in order of the subtiles, one accumulator set at a time in the tiles' place
    const long long width = (long long)key_heads * HD, out = (begin + key0) * width + (long long)item.head * HD;
    static_assert((size_t)W * 2 * Tiles::TILE <= Tiles::lds_bytes(), "the parked parts take the tiles' place");
    float *park = reinterpret_cast<float *>(lds_raw + (size_t)w * 2 * Tiles::TILE);
    const float *parts = reinterpret_cast<const float *>(lds_raw + (size_t)(w - sub) * 2 * Tiles::TILE);
#pragma unroll
    for (int set = 0; set < 2; ++set) {          // subtile `set` of each key tile sums and stores it
        RowTile<HD> &acc = set == 0 ? dv : dk;
        const float out_scale = set == 0 ? DOWN : BF ? p.scale : p.scale * DOWN * __builtin_amdgcn_rcpf(ds_mul);     // of each wave's own key
        __syncthreads();                         // all are done with the tiles, or with the set before
        each<HD>(acc, [&](float x, int i) { return park[i] = x * out_scale; });
        __syncthreads();
        if (sub != set) continue;
        clear<HD>(acc);
#pragma unroll 1
        for (int o = 0; o < SUB; ++o) each<HD>(acc, [&](float x, int i) { return x + parts[o * 32 * HD + i]; });
        store_token_rows<HD, BF>(acc, 1.f, reinterpret_cast<unsigned char *>(park), (set == 0 ? p.dv : p.dk) + out, width,
                                 n - key0);
    }
}

// ---- launchers ----------------------------------------------------------------------------------------
constexpr int PACKED_WAVES = 4;
constexpr int packed_subtiles(int hd) { return hd == 64 ? 2 : 4; }       // of queries in the walk over the keys

PackedOperands operands(const PackedArgs &a)
{
    PackedOperands p;
    p.q = (const half_t *)a.q, p.k = (const half_t *)a.k, p.v = (const half_t *)a.v;
    p.dout = (const half_t *)a.dout, p.o = (const half_t *)a.o, p.o_rest = (const half_t *)a.o_rest;
    p.out = (half_t *)a.out, p.rest = (half_t *)a.rest, p.dk = (half_t *)a.dk, p.dv = (half_t *)a.dv;
    p.lse = a.lse, p.delta = a.delta;
    p.offsets = a.offsets;
    p.tokens = a.tokens, p.sequences = a.sequences, p.heads = a.heads, p.group = a.heads / a.key_heads;
    p.causal = a.causal;
    p.scale = a.scale, p.scale2 = a.scale * 1.4426950408889634f;
    p.q_token = a.q_token, p.q_head = a.q_head, p.k_token = a.k_token, p.k_head = a.k_head;
    p.v_token = a.v_token, p.v_head = a.v_head, p.g_token = a.g_token, p.g_head = a.g_head;
    return p;
}

// a launch gets 64 KB of LDS without asking
template <class Kernel>
hipError_t run_walk(Kernel kernel, PackedOperands p, int heads, int rows, int waves, size_t lds, hipStream_t st)
{
    if (lds > 65536) {
        const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (err != hipSuccess) return err;
    }
    p.head_sets = packed_head_sets(heads);
    p.slots = packed_slots(p.tokens, p.sequences, rows);
    kernel<<<packed_grid(heads, p.head_sets, p.slots) + PACKED_CLEARING, 64 * waves, lds, st>>>(p);
    return hipGetLastError();
}

template <int HD, bool BF>
hipError_t forward(const PackedArgs &a, hipStream_t st)
{
    constexpr int W = PACKED_WAVES;
    return run_walk(a.lse != nullptr ? packed_forward_kernel<HD, BF, W, true> : packed_forward_kernel<HD, BF, W, false>, operands(a), a.heads,
                    32 * W, W, PairTiles<HD, W, 2>::lds_bytes(), st);
}
template <int HD, bool BF>
hipError_t backward(const PackedArgs &a, hipStream_t st)
{
    constexpr int W = PACKED_WAVES;
    const PackedOperands p = operands(a);
    const hipError_t err = run_walk(packed_rows_kernel<HD, BF, W>, p, a.heads, 32 * W, W, PairTiles<HD, W, 2>::lds_bytes(), st);
    if (err != hipSuccess || a.dk == nullptr) return err;
    constexpr int SUB = packed_subtiles(HD);
    return run_walk(packed_columns_kernel<HD, BF, SUB>, p, a.key_heads, 64, 2 * SUB,
                    PairTiles<HD, 2 * SUB, SUB>::lds_bytes() + 16 * 32 * SUB + 2 * 64 * HD, st);
}

}  // namespace

bool packed_fits(const PackedArgs &a, bool key_gradients)
{
    // packed_grid rounds the slots of a head up to at most 7 more; in 64 bits
    auto fits = [&](int heads, int rows, int threads) {
        return ((long long)heads * ((long long)a.tokens / rows + a.sequences + 7) + PACKED_CLEARING) * threads < (1ll << 32);
    };
    return fits(a.heads, 32 * PACKED_WAVES, 64 * PACKED_WAVES) && (!key_gradients || fits(a.key_heads, 64, 128 * packed_subtiles(a.head_dim)));
}

hipError_t launch_packed_forward(const PackedArgs &a, hipStream_t st)
{
    if (a.head_dim == 64) return a.bf16 ? forward<64, true>(a, st) : forward<64, false>(a, st);
    return a.bf16 ? forward<128, true>(a, st) : forward<128, false>(a, st);
}

hipError_t launch_packed_backward(const PackedArgs &a, hipStream_t st)
{
    if (a.head_dim == 64) return a.bf16 ? backward<64, true>(a, st) : backward<64, false>(a, st);
    return a.bf16 ? backward<128, true>(a, st) : backward<128, false>(a, st);
}

}  // namespace bsa

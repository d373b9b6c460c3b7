// What the walks over packed sequences share: finding the sequence of a workgroup, pairs of operand tiles of 64 tokens that all
// waves of a workgroup read, products with hidden places, results of 32 tokens on their way out.
#pragma once

#include "attention_tiles.hpp"
#include "bsa_device.hpp"

namespace bsa {

struct PackedOperands {
    const half_t *q, *k, *v, *dout, *o, *o_rest; // o: the forward result, [T][heads][HD], for the backward walks
    half_t *out, *rest, *dk, *dv;                // out: the result, or dq; rest, o_rest: what its rounding took; all dense
    float *lse, *delta;                          // [heads][T]
    const int32_t *offsets;                      // [sequences + 1]
    int tokens, sequences, heads, group;         // heads: query heads, group: of them to a key head
    int head_sets, slots;                        // of a launch: sets of heads that XCDs share, workgroup slots of a head
    int causal;
    float scale, scale2;                         // scale2 = scale log2(e)
    long long q_token, q_head, k_token, k_head, v_token, v_head, g_token, g_head;    // strides in values; g: dout
};

// Slots of a head: the most workgroups of `rows` tokens that `tokens` in `sequences` can need.
__host__ __device__ __forceinline__ int packed_slots(int tokens, int sequences, int rows) { return tokens / rows + sequences; }
// Workgroups that clear the results of tokens outside every sequence, behind those of the slots.
constexpr int PACKED_CLEARING = 32;
// Workgroup ids go round the 8 XCDs.  With `sets` = gcd(8, heads) the heads are cut into that many sets of neighbours, each set on
// 8 / sets XCDs of its own, which take its slots in turn: a key head is read into as few L2s as the balance allows.
__host__ __forceinline__ int packed_head_sets(int heads) { return heads % 8 == 0 ? 8 : heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1; }
__host__ __device__ __forceinline__ int packed_grid(int heads, int sets, int slots)
{
    const int share = 8 / sets;
    return 8 * (heads / sets) * ((slots + share - 1) / share);
}

struct PackedItem {
    int head, tile;              // tile: of the sequence, in workgroups' rows
    int begin, n;                // first token, tokens; n == 0: nothing to do
};

__device__ __forceinline__ int packed_offset(const PackedOperands &p, int b)
{
    const int x = p.offsets[b];
    return x < 0 ? 0 : x > p.tokens ? p.tokens : x;
}

// The workgroup's head and tile.  The hardware starts workgroups in order, so the long ones come first: up to 64 sequences the
// tiles of all of them are dealt by their index in the sequence, the highest first (from_end: the distance to the sequence's
// end), each lane of a wave holding one sequence.  With more, slot floor(offset / ROWS) + b is the first of sequence b, strictly
// ascending in b, so 64 lanes search together, and a sequence's own tiles come longest first.  `heads`: of the launch.
template <int ROWS>
__device__ __forceinline__ PackedItem packed_item(const PackedOperands &p, int heads, bool from_end)
{
    PackedItem item{0, 0, 0, 0};
    const int x = (int)(blockIdx.x & 7u), t = (int)(blockIdx.x >> 3);
    const int share = 8 / p.head_sets, in_set = heads / p.head_sets;
    item.head = x / share * in_set + t % in_set;
    const int slot = t / in_set * share + x % share;
    if (slot >= p.slots) return item;
    const int l = lane_id();
    if (p.sequences <= WAVE) {
        const int from = packed_offset(p, l < p.sequences ? l : p.sequences), to = packed_offset(p, l < p.sequences ? l + 1 : p.sequences);
        const int tiles = to > from ? (to - from + ROWS - 1) / ROWS : 0;
        // tiles with an index of at least `index`
        auto beyond = [&](int index) {
            int sum = 0;
            for (int b = 0; b < p.sequences; ++b) {
                const int more = __builtin_amdgcn_readlane(tiles, b) - index;
                sum += more > 0 ? more : 0;
            }
            return sum;
        };
        // the highest index with more than `slot` tiles from it on, 64 candidates at a time, the first of which always has them
        int index = 0, stride = p.slots, behind = 0;
        do {
            stride = (stride + WAVE - 1) / WAVE;
            const int left = beyond(index + stride * l);
            const int with = __popcll(__builtin_amdgcn_ballot_w64(left > slot));
            if (with == 0) return item;          // the first time: there are fewer tiles
            behind = with < WAVE ? __builtin_amdgcn_readlane(left, with) : beyond(index + stride * WAVE);
            index += stride * (with - 1);
        } while (stride > 1);
        index = __builtin_amdgcn_readfirstlane(index);
        const int place = slot - __builtin_amdgcn_readfirstlane(behind);         // among the sequences with such a tile
        const unsigned long long with = __builtin_amdgcn_ballot_w64(tiles > index);
        const int mine = __builtin_amdgcn_mbcnt_hi((unsigned)(with >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)with, 0u));
        const int b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(tiles > index && mine == place));
        item.begin = __builtin_amdgcn_readlane(from, b);
        item.n = __builtin_amdgcn_readlane(to, b) - item.begin;
        item.tile = from_end ? __builtin_amdgcn_readlane(tiles, b) - 1 - index : index;
        return item;
    }
    int first = 0, count = p.sequences;
    while (true) {
        const int stride = (count + 63) / 64, b = first + l * stride;
        const bool before = b < first + count && packed_offset(p, b) / ROWS + b <= slot;
        const int seen = __popcll(__builtin_amdgcn_ballot_w64(before));
        const int skip = (seen > 0 ? seen - 1 : 0) * stride;
        first += skip;
        count = count - skip < stride ? count - skip : stride;
        if (stride == 1) break;
    }
    first = __builtin_amdgcn_readfirstlane(first);
    const int begin = __builtin_amdgcn_readfirstlane(packed_offset(p, first));
    const int end = __builtin_amdgcn_readfirstlane(packed_offset(p, first + 1));
    const int tile = slot - (begin / ROWS + first), tiles = (end - begin + ROWS - 1) / ROWS;
    if (end <= begin || tile < 0 || tile >= tiles) return item;
    item.begin = begin;
    item.n = end - begin;
    item.tile = from_end ? tile : tiles - 1 - tile;
    return item;
}

// the tokens before the first and behind the last sequence
__device__ __forceinline__ void packed_clear(const PackedOperands &p, int part, half_t *rows, long long width)
{
    const int head = packed_offset(p, 0), tail = packed_offset(p, p.sequences);
    const long long pieces = width / 8, before = head < tail ? head : tail;
    auto clear = [&](long long from, long long to) {
        for (long long i = from * pieces + (long long)part * blockDim.x + threadIdx.x; i < to * pieces;
             i += (long long)PACKED_CLEARING * blockDim.x)
            stg16(rows + 8 * i, make_uint4(0, 0, 0, 0));
    };
    clear(0, before);
    clear(tail, p.tokens);
}

// sum + a + b of two 16-bit values in one instruction (subnormal ones count).  Rows are normalised by the sum of the probabilities
// as the products take them, so their rounding cancels where all of them share it.
template <bool BF>
__device__ __forceinline__ float add_pair(half_t a, half_t b, float sum)
{
    if (BF) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        const b2 x = {__builtin_bit_cast(__bf16, a), __builtin_bit_cast(__bf16, b)}, ones = {(__bf16)1.f, (__bf16)1.f};
        return __builtin_amdgcn_fdot2_f32_bf16(x, ones, sum, false);
    }
    const h2 x = {a, b}, ones = {(half_t)1.f, (half_t)1.f};
    return __builtin_amdgcn_fdot2(x, ones, sum, false);
}

// Keeps what is above in front of what is below: operands are requested from LDS before the work that hides their latency.
__device__ __forceinline__ void issue_order() { __builtin_amdgcn_sched_barrier(0); }
// Values loaded in front of a loop have arrived: otherwise the compiler waits for them inside it, and with them for the loads to
// LDS that it does not know of.
template <int N>
__device__ __forceinline__ void loaded(h8 (&op)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(op[i]));
}

template <int HD>
__device__ __forceinline__ void read_rows(const TileReader &rd, unsigned tile, h8 (&op)[HD / 16])
{
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) op[s] = rd.rows(tile, s);
}
template <int HD>
__device__ __forceinline__ void read_columns(const TileReader &rd, unsigned tile, h8 (&op)[HD / 32][2])
{
#pragma unroll
    for (int t = 0; t < HD / 32; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s) op[t][s] = rd.columns(tile, t, s);
}
template <bool BF, int N>
__device__ __forceinline__ void product(const h8 (&a)[N], const h8 (&b)[N], f16v &acc)
{
#pragma unroll
    for (int s = 0; s < N; ++s) acc = mfma_16<BF>(a[s], b[s], acc);
}
// Products with some weights zero because their place is hidden: an infinity or a NaN in a token must not reach the results of
// those that do not see it, and zero times it would be NaN.  Where anything is hidden the operands are looked at and such values left
// out of the products.  add_not_finite then adds them to the results of the lanes for which sees(row of the tile) holds.  In the walk over
// the keys nothing has to be added: such a query's statistics are no numbers either, and with them the weights of all that it sees.
template <bool BF, int T>
__device__ __forceinline__ bool take_out_not_finite(h8 (&columns)[T][2])
{
    typedef unsigned short us8 __attribute__((ext_vector_type(8)));
    constexpr unsigned short INFINITE = BF ? 0x7F80 : 0x7C00;
    us8 top = 0;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s)
            top = __builtin_elementwise_max(top, (us8)(__builtin_bit_cast(us8, columns[t][s]) & (unsigned short)0x7FFF));
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) finite = finite && top[j] < INFINITE;
    if (__builtin_amdgcn_ballot_w64(!finite) == 0ull) return false;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            us8 x = __builtin_bit_cast(us8, columns[t][s]);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (x[j] & 0x7FFF) < INFINITE ? x[j] : (unsigned short)0;
            columns[t][s] = __builtin_bit_cast(h8, x);
        }
    return true;
}
template <int HD, bool BF, class Sees>
__device__ __forceinline__ void add_not_finite(const TileReader &rd, unsigned tile, RowTile<HD> &acc, Sees sees)
{
    constexpr unsigned short INFINITE = BF ? 0x7F80 : 0x7C00;
    const int h = lane_id() >> 5;
    typedef const h4 __attribute__((address_space(3))) *lds_h4;
    const unsigned first = (unsigned)__builtin_amdgcn_readfirstlane((int)(rd.row[0] - (unsigned)get_panel_addr(lane_id(), 0))) + tile;
#pragma unroll 1
    for (int r = 0; r < 32; ++r) {
        const bool seen = sees(r);
#pragma unroll
        for (int t = 0; t < HD / 32; ++t) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int piece = 4 * (t & 1) + g;
                const h4 raw = *(lds_h4)(uintptr_t)(first + 4096 * (t / 2) + 128 * r + 16 * (piece ^ panel_swizzle(r)) + 8 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const half_t one = raw[j];   // a bit cast of a vector's element itself takes the first one
                    const float value = widen_16<BF>(one);
                    if (seen && (__builtin_bit_cast(unsigned short, one) & 0x7FFF) >= INFINITE)
                        acc[t][4 * g + j] += value;
                }
            }
            issue_order();
        }
    }
}

// acc[t] += columns 32 t .. of a 32-row tile, its rows weighted by op; the columns have been read; whether values were left out
template <int HD, bool BF>
__device__ __forceinline__ bool weigh(h8 (&columns)[HD / 32][2], const h8 (&op)[2], RowTile<HD> &acc, bool hidden)
{
    const bool out = hidden && take_out_not_finite<BF>(columns);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int t = 0; t < HD / 32; ++t) acc[t] = mfma_16<BF>(columns[t][s], op[s], acc[t]);
    return out;
}
// the same, 64 columns read at a time
template <int HD, bool BF>
__device__ __forceinline__ bool weigh_tile(const TileReader &rd, unsigned tile, const h8 (&op)[2], RowTile<HD> &acc, bool hidden = false)
{
    bool out = false;
#pragma unroll
    for (int t0 = 0; t0 < HD / 32; t0 += 2) {
        h8 tr[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < 2; ++s) tr[t][s] = rd.columns(tile, t0 + t, s);
        if (hidden && take_out_not_finite<BF>(tr)) out = true;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) acc[t0 + t] = mfma_16<BF>(tr[t][s], op[s], acc[t0 + t]);
        if (HD > 64) issue_order();
    }
    return out;
}

// 32 rows `stride` values apart, of which `valid` are there (those behind as the last), to a tile at LDS address `to`, by one wave
template <int HD>
__device__ __forceinline__ void request_rows(const half_t *rows, long long stride, int valid, unsigned to)
{
    const int l = lane_id();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int r = 8 * c + (l >> 3), there = r < valid ? r : valid - 1;
        const unsigned off = (unsigned)(there > 0 ? there : 0) * (unsigned)(2 * stride) + 16 * panel_src_piece(l, c);
#pragma unroll
        for (int u = 0; u < HD / 64; ++u) dma16((const unsigned char *)rows + 128 * u, off, to + 4096 * u + 1024 * c);
    }
}

// Two operands (K and V, or Q and dO) in tiles of 32 SUB tokens, double buffered, read by all W waves.  LDS of a buffer: the first
// operand's 32-row tiles (TileRequests' panels), then the second's.  A wave fetches SUB HD / 16 / W kilobytes of each.
template <int HD, int W, int SUB>
struct PairTiles {
    static constexpr int TOKENS = 32 * SUB, TILE = 64 * HD, BUFFER = 2 * SUB * TILE, REQUESTS = SUB * HD / 16 / W;
    const TileReader rd;         // of buffer 0
    const unsigned char *base[2];
    long long stride[2];         // bytes between tokens
    unsigned lds, row, piece;    // row: of this lane inside a 32-row tile
    unsigned whole[2];           // what a lane fetches, from the first of its rows and pieces on
    int wave;
    __device__ __forceinline__ PairTiles(const half_t *a, long long a_token, const half_t *b, long long b_token, unsigned char *lds_raw)
        : rd(lds_raw)
    {
        wave = wave_id();
        const int l = lane_id(), chunk = wave & 3;
        base[0] = (const unsigned char *)a, base[1] = (const unsigned char *)b;
        stride[0] = 2 * a_token, stride[1] = 2 * b_token;
        lds = __builtin_amdgcn_readfirstlane(lds_address(lds_raw));
        row = 8 * chunk + (l >> 3);
        piece = 16 * panel_src_piece(l, chunk);
#pragma unroll
        for (int o = 0; o < 2; ++o) whole[o] = row * (unsigned)stride[o] + piece;
    }
    static constexpr size_t lds_bytes() { return 2 * (size_t)BUFFER; }
    __device__ __forceinline__ int subtile(int i) const { return (i * W + wave) / (HD / 16); }
    __device__ __forceinline__ int panel(int i) const { return (i * W + wave) % (HD / 16) / 4; }
    // tokens TOKENS step .. of n of one operand, those from n on as token n - 1 (what they give is hidden)
    __device__ __forceinline__ void request(int o, int step, int n, int buffer) const
    {
        const unsigned char *from = base[o] + (long long)TOKENS * step * stride[o];
        const unsigned to = lds + (unsigned)(buffer * BUFFER + o * SUB * TILE + 1024 * (wave & 3));
        if (TOKENS * step + TOKENS <= n) {
#pragma unroll
            for (int i = 0; i < REQUESTS; ++i)
                dma16(from + 32 * subtile(i) * stride[o] + 128 * panel(i), whole[o], to + TILE * subtile(i) + 4096 * panel(i));
            return;
        }
        const unsigned last = (unsigned)(n - 1 - TOKENS * step);
#pragma unroll
        for (int i = 0; i < REQUESTS; ++i) {
            unsigned r = 32 * subtile(i) + row;
            r = r < last ? r : last;
            dma16(from + 128 * panel(i), r * (unsigned)stride[o] + piece, to + TILE * subtile(i) + 4096 * panel(i));
        }
    }
    __device__ __forceinline__ void request(int step, int n, int buffer) const
    {
        request(0, step, n, buffer);
        request(1, step, n, buffer);
    }
    // Zeros in the place of infinities and NaN in what this wave has fetched of a buffer, once it has arrived and before the others
    // read it.
    template <bool BF>
    __device__ __forceinline__ void clean(int buffer) const
    {
        typedef unsigned short us8 __attribute__((ext_vector_type(8)));
        typedef us8 __attribute__((address_space(3))) *lds_us8;
        constexpr unsigned short INFINITE = BF ? 0x7F80 : 0x7C00;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int i = 0; i < REQUESTS; ++i) {
                const unsigned to = lds + (unsigned)(buffer * BUFFER + o * SUB * TILE + 1024 * (wave & 3)) + TILE * subtile(i) + 4096 * panel(i);
                const lds_us8 at = (lds_us8)(uintptr_t)(to + 16u * (unsigned)lane_id());
                us8 x = *at;
                bool finite = true;
#pragma unroll
                for (int j = 0; j < 8; ++j) finite = finite && (x[j] & 0x7FFF) < INFINITE;
                if (!finite) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = (x[j] & 0x7FFF) < INFINITE ? x[j] : (unsigned short)0;
                    *at = x;
                }
            }
    }
    // this wave's part of what was requested has arrived, and everyone's; all waves are done with the buffer before
    __device__ __forceinline__ void arrived() const { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
    // subtile u of an operand in a buffer, as TileReader's tile
    static __device__ __forceinline__ constexpr unsigned at(int buffer, int operand, int u)
    {
        return (unsigned)(buffer * BUFFER + (SUB * operand + u) * TILE);
    }
};

// 32 result rows `stride` values apart, of which the first `valid` are stored; through 64 HD bytes of LDS, so that they leave
// as whole lines.  REST: what the rounding takes from them instead.
template <int HD, bool BF, bool REST = false>
__device__ __forceinline__ void store_token_rows(const RowTile<HD> &acc, float mul, unsigned char *scratch, half_t *dst,
                                                 long long stride, int valid)
{
    const int l = lane_id(), row = l & 31, h = l >> 5;
    wave_lds_fence();
#pragma unroll
    for (int t = 0; t < HD / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            h4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = acc[t][4 * g + j] * mul;
                o[j] = narrow_16<BF>(REST ? x - widen_16<BF>(narrow_16<BF>(x)) : x);
            }
            *reinterpret_cast<h4 *>(scratch + out_row_addr(HD, row, 4 * t + g, h)) = o;
        }
    wave_lds_fence();
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
        const int slot = l + 64 * j, r = slot / (HD / 8), p = slot % (HD / 8);
        if (r < valid) stg16(dst + r * stride + 8 * p, *reinterpret_cast<const uint4 *>(scratch + out_row_addr(HD, r, p, 0)));
    }
}

}  // namespace bsa

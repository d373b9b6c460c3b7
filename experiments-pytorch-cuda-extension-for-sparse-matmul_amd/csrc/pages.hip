// Which pages of a cache each sequence has, kept on the device, and copies of pages.
//
//   table [sequences][width]   page numbers, -1 behind the last;  lengths [sequences]: tokens;  uses [pages]: sequences that have a page
//
// Whole pages may belong to several sequences, the last page of one that is not full belongs to it alone: a fork shares the whole pages
// and copies that one.  New pages are the lowest free ones, in the order of the call's sequences, so that equal tables and equal
// calls give equal tables.  Counting is by integer atomics, whose order changes nothing.
//
// What bounds it: latency.  Ranks of free pages are found by one workgroup that reads `uses` 16 bytes a lane and sums up in LDS, as far as it
// has to; rows of the table are read and written by a workgroup each.  Least of 60 launches and their median: a step of 64
// sequences 4.5 us (4.7), 24 prompts of 64 to 4096 tokens 6.3 (6.6) and, their slots, 2.6 (3.8); a fork of 8 sequences to 504 children of up to 235
// pages 8.9 (11.4), 8.2 (8.4) and 4.2 (4.8), three launches; a compaction of 6650 pages 8.2 (8.4) and 2.8 (4.6).  The end
// of 8 sequences of 22 pages 3.0 us (3.9), of 504 of 235 pages 3.6 (4.3): a launch, each page's use an atomic.
// Copies of pages: memory, 5.7 TB/s (217 MB each way in 76 us, 78).
#include "bsa_device.hpp"
#include "bsa_internal.hpp"

namespace bsa {

namespace {

constexpr int PG_THREADS = 1024, PG_WAVES = PG_THREADS / WAVE;
constexpr int PG_MOST = PAGES_MOST_SEQUENCES, PG_PER = PG_MOST / PG_THREADS;

__device__ __forceinline__ int wave_prefix(int x)        // inclusive, over the wave
{
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) {
        const int below = __builtin_amdgcn_ds_bpermute((lane_id() - d) << 2, x);
        x += lane_id() >= d ? below : 0;
    }
    return x;
}
// exclusive prefix over the PG_THREADS threads of a workgroup, and the sum of all
__device__ __forceinline__ int block_prefix(int x, int *parts, int &all)
{
    const int inclusive = wave_prefix(x);
    __syncthreads();                                     // parts may still be read
    if (lane_id() == WAVE - 1) parts[wave_id()] = inclusive;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) {
        before += w < wave_id() ? parts[w] : 0;
        all += parts[w];
    }
    return before + inclusive - x;
}

// taken(rank, page) for the `wanted` lowest pages for which free(uses), by rank; how many there are, at most `wanted`
template <class Taken>
__device__ __forceinline__ int lowest_free(const int32_t *uses, int pages, int wanted, int *parts, Taken taken)
{
    int found = 0, next[4];
    auto fetch = [&](int at) {
        if (at + 4 <= pages) {
            const int4 x = *reinterpret_cast<const int4 *>(uses + at);
            next[0] = x.x, next[1] = x.y, next[2] = x.z, next[3] = x.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) next[j] = at + j < pages ? uses[at + j] : 1;
        }
    };
    if (wanted > 0) fetch(4 * (int)threadIdx.x);
    for (int first = 0; first < pages && found < wanted; first += 4 * PG_THREADS) {
        const int at = first + 4 * (int)threadIdx.x;
        int use[4], mine = 0, all;
#pragma unroll
        for (int j = 0; j < 4; ++j) use[j] = next[j];
        fetch(at + 4 * PG_THREADS);                      // on their way while these are counted
#pragma unroll
        for (int j = 0; j < 4; ++j) mine += use[j] == 0 ? 1 : 0;
        int rank = found + block_prefix(mine, parts, all);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (use[j] == 0) {
                if (rank < wanted) taken(rank, at + j);
                ++rank;
            }
        found += all;
    }
    return found < wanted ? found : wanted;
}

__device__ __forceinline__ int pages_of(long long tokens, int page_shift) { return (int)((tokens + (1 << page_shift) - 1) >> page_shift); }
__device__ __forceinline__ int length_of(const PagesArgs &p, int b)
{
    const long long n = p.lengths[b], most = (long long)p.width << p.page_shift;
    return (int)(n < 0 ? 0 : n > most ? most : n);
}
__device__ __forceinline__ bool is_page(const PagesArgs &p, int x) { return x >= 0 && x < p.pages; }

// ---- new tokens ---------------------------------------------------------------------------------------
__device__ __forceinline__ int new_offset(const PagesArgs &p, int b)
{
    const int x = p.offsets[b];
    return x < 0 ? 0 : x > p.tokens ? p.tokens : x;
}
// started[b]: the length before, -1 for a sequence whose tokens have no place
__device__ __forceinline__ void write_slots(const PagesArgs &p, int first, int stride, const int32_t *started)
{
    for (int t = first; t < p.tokens; t += stride) {
        int low = 0, count = p.sequences;                // the last sequence that begins at t or before
        while (count > 1) {
            const int half = count / 2;
            if (new_offset(p, low + half) <= t) {
                low += half;
                count -= half;
            } else {
                count = half;
            }
        }
        int slot = -1;
        const int from = new_offset(p, low);
        if (from <= t && t < new_offset(p, low + 1) && started[low] >= 0) {
            const int place = started[low] + (t - from), at = place >> p.page_shift;
            const int page = at < p.width ? p.table[(size_t)low * p.width + at] : -1;
            if (is_page(p, page)) slot = (page << p.page_shift) + (place & ((1 << p.page_shift) - 1));
        }
        p.slots[t] = slot;
    }
}

__global__ __launch_bounds__(PG_THREADS) void pages_append_kernel(PagesArgs p, bool with_slots)
{
    __shared__ int parts[PG_WAVES], ends[PG_MOST], had[PG_MOST];
    int need[PG_PER], sum = 0, all;
    bool wide[PG_PER];
    // sequences PG_PER x thread .. of this thread; ends: pages that the sequences up to and with one need
#pragma unroll
    for (int j = 0; j < PG_PER; ++j) {
        const int b = PG_PER * (int)threadIdx.x + j;
        need[j] = 0, wide[j] = false;
        if (b < p.sequences) {
            const int from = new_offset(p, b), to = new_offset(p, b + 1), held = length_of(p, b);
            const long long length = (long long)held + (to > from ? to - from : 0);
            had[b] = pages_of(held, p.page_shift);
            wide[j] = pages_of(length, p.page_shift) > p.width;
            need[j] = wide[j] ? 0 : pages_of(length, p.page_shift) - had[b];
        }
        sum += need[j];
    }
    int end = block_prefix(sum, parts, all);
#pragma unroll
    for (int j = 0; j < PG_PER; ++j) {
        end += need[j];
        ends[PG_PER * threadIdx.x + j] = end;
    }
    __syncthreads();
    // the sequence that the page of this rank goes to: the first whose end lies behind it
    auto owner = [&](int rank) {
        int low = 0, count = p.sequences;
        while (count > 0) {
            const int half = count / 2;
            if (ends[low + half] <= rank) {
                low += half + 1;
                count -= half + 1;
            } else {
                count = half;
            }
        }
        return low;
    };
    const int found = lowest_free(p.uses, p.pages, all, parts, [&](int rank, int page) {
        const int b = owner(rank), begin = b > 0 ? ends[b - 1] : 0;
        p.table[(size_t)b * p.width + had[b] + (rank - begin)] = page;
        p.uses[page] = 1;
    });
    __syncthreads();
    if (found < all) {                                   // the sequence that got a part of its pages only gives them back
        const int b = owner(found), begin = b > 0 ? ends[b - 1] : 0;
        for (int r = begin + (int)threadIdx.x; r < found; r += PG_THREADS) {
            int32_t *at = p.table + (size_t)b * p.width + had[b] + (r - begin);
            p.uses[*at] = 0;
            *at = -1;
        }
    }
    int refused = 0;
#pragma unroll
    for (int j = 0; j < PG_PER; ++j) {
        const int b = PG_PER * (int)threadIdx.x + j;
        if (b >= p.sequences) continue;
        const int from = new_offset(p, b), to = new_offset(p, b + 1), held = length_of(p, b);
        const bool fits = !wide[j] && (need[j] == 0 || ends[b] <= found);
        p.scratch[b] = fits ? held : -1;
        p.lengths[b] = held + (fits && to > from ? to - from : 0);
        refused += fits ? 0 : 1;
    }
    if (refused > 0) atomicAdd(p.missing, refused);
    __syncthreads();
    if (with_slots) write_slots(p, (int)threadIdx.x, PG_THREADS, p.scratch);
}
__global__ __launch_bounds__(256) void pages_slots_kernel(PagesArgs p)
{
    write_slots(p, (int)(blockIdx.x * 256 + threadIdx.x), (int)(gridDim.x * 256), p.scratch);
}

// ---- sequences that end -------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void pages_free_kernel(PagesArgs p)
{
    __shared__ int length;
    const int b = p.children[blockIdx.x];
    if (b < 0 || b >= p.sequences) return;
    if (threadIdx.x == 0) length = atomicExch(p.lengths + b, 0);         // of several entries for a sequence one finds it
    __syncthreads();
    const long long most = (long long)p.width << p.page_shift;
    const int count = pages_of(length < 0 ? 0 : length > most ? most : length, p.page_shift);
    for (int j = (int)threadIdx.x; j < count; j += 256) {
        int32_t *at = p.table + (size_t)b * p.width + j;
        if (is_page(p, *at)) atomicAdd(p.uses + *at, -1);
        *at = -1;
    }
}

// ---- sequences that others continue -------------------------------------------------------------------
// Scratch of an entry: its parent's row, then these
struct ForkEntry {
    int32_t tokens;                      // of the parent; -1: an entry that is left out
    int32_t old_pages;                   // that the child had
    int32_t copies;                      // the parent's last page is copied
    int32_t unused;
};
__device__ __forceinline__ int32_t *fork_row(const PagesArgs &p, int i) { return p.scratch + (size_t)i * (p.width + 4); }
__device__ __forceinline__ ForkEntry &fork_entry(const PagesArgs &p, int i) { return *reinterpret_cast<ForkEntry *>(fork_row(p, i) + p.width); }

// Of the entries for a child the first counts; of the entries that continue a parent which is itself replaced, the first keeps its last
// page.  by_child, by_parent: their places among the entries, or none; heirs: how many entries continue a sequence.
struct ForkClaims {
    int by_child[PG_MOST], by_parent[PG_MOST], heirs[PG_MOST];
};
constexpr int PG_NONE = 0x7FFFFFFF;
__device__ __forceinline__ void fork_claims(const PagesArgs &p, ForkClaims &claims)
{
    for (int b = (int)threadIdx.x; b < p.sequences; b += (int)blockDim.x) {
        claims.by_child[b] = claims.by_parent[b] = PG_NONE;
        claims.heirs[b] = 0;
    }
    __syncthreads();
    auto inside = [&](int x) { return x >= 0 && x < p.sequences; };
    for (int i = (int)threadIdx.x; i < p.entries; i += (int)blockDim.x)
        if (inside(p.parents[i]) && inside(p.children[i])) atomicMin(claims.by_child + p.children[i], i);
    __syncthreads();
    for (int i = (int)threadIdx.x; i < p.entries; i += (int)blockDim.x)
        if (inside(p.parents[i]) && inside(p.children[i]) && claims.by_child[p.children[i]] == i) {
            atomicMin(claims.by_parent + p.parents[i], i);
            atomicAdd(claims.heirs + p.parents[i], 1);
        }
    __syncthreads();
}

// One entry, by the threads `thread` of `threads`: its parent's row into scratch, uses of what the child had and, by a parent's first heir
// for all of them, of what they share.  The parent's last page, where it is not full, is the first heir's if the parent itself is
// replaced, and nobody's share.
__device__ __forceinline__ void fork_share(const PagesArgs &p, int i, const ForkClaims &claims, int thread, int threads)
{
    const int parent = p.parents[i], child = p.children[i];
    const bool there = parent >= 0 && parent < p.sequences && child >= 0 && child < p.sequences && claims.by_child[child] == i;
    ForkEntry entry{-1, 0, 0, 0};
    if (there) {
        entry.tokens = length_of(p, parent);
        entry.old_pages = pages_of(length_of(p, child), p.page_shift);
        const bool first = claims.by_parent[parent] == i;
        const int whole = entry.tokens >> p.page_shift, count = pages_of(entry.tokens, p.page_shift);
        entry.copies = count > whole && (claims.by_child[parent] == PG_NONE || !first);
        int32_t *row = fork_row(p, i);
        for (int j = thread; j < count; j += threads) {
            const int page = p.table[(size_t)parent * p.width + j];
            row[j] = page;
            if (first && is_page(p, page) && (j < whole || entry.copies == 0)) atomicAdd(p.uses + page, j < whole ? claims.heirs[parent] : 1);
        }
        for (int j = thread; j < entry.old_pages; j += threads) {
            const int page = p.table[(size_t)child * p.width + j];
            if (is_page(p, page)) atomicAdd(p.uses + page, -1);
        }
    }
    if (thread == 0) fork_entry(p, i) = entry;
}

// pages for the copies, by one workgroup; an entry that gets none leaves its child empty
__device__ __forceinline__ void fork_allocate(const PagesArgs &p, int *parts)
{
    int wanted = 0;
    const int rounds = (p.entries + PG_THREADS - 1) / PG_THREADS;
    // ranks: the copying entries in their order; p.targets holds the rank's entry until its page is known
    for (int r = 0; r < rounds; ++r) {
        const int i = r * PG_THREADS + (int)threadIdx.x;
        const bool copies = i < p.entries && fork_entry(p, i).copies != 0;
        int all;
        const int rank = wanted + block_prefix(copies ? 1 : 0, parts, all);
        if (copies) fork_entry(p, rank).unused = i;
        wanted += all;
        if (i < p.entries) p.sources[i] = p.targets[i] = -1;
    }
    __syncthreads();
    const int found = lowest_free(p.uses, p.pages, wanted, parts, [&](int rank, int page) {
        const int i = fork_entry(p, rank).unused, last = fork_entry(p, i).tokens >> p.page_shift;
        p.sources[i] = fork_row(p, i)[last];
        p.targets[i] = page;
        fork_row(p, i)[last] = page;
        p.uses[page] = 1;
    });
    __syncthreads();
    for (int rank = found; rank < wanted; ++rank) {
        const int i = fork_entry(p, rank).unused, shared = fork_entry(p, i).tokens >> p.page_shift;
        for (int j = (int)threadIdx.x; j < shared; j += PG_THREADS)
            if (is_page(p, fork_row(p, i)[j])) atomicAdd(p.uses + fork_row(p, i)[j], -1);
        __syncthreads();
        if (threadIdx.x == 0) {
            fork_entry(p, i).tokens = 0;
            atomicAdd(p.missing, 1);
        }
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < p.entries; i += PG_THREADS)
        if (fork_entry(p, i).tokens >= 0) p.lengths[p.children[i]] = fork_entry(p, i).tokens;
}

__device__ __forceinline__ void fork_place(const PagesArgs &p, int i, int thread, int threads)
{
    const ForkEntry entry = fork_entry(p, i);
    if (entry.tokens < 0) return;
    const int count = pages_of(entry.tokens, p.page_shift), old = entry.old_pages;
    int32_t *to = p.table + (size_t)p.children[i] * p.width;
    for (int j = thread; j < (count > old ? count : old); j += threads) to[j] = j < count ? fork_row(p, i)[j] : -1;
}

// an entry a workgroup, or, where there are more of them, a wave
template <class Work>
__device__ __forceinline__ void each_entry(const PagesArgs &p, Work work)
{
    if ((int)gridDim.x == p.entries) return work((int)blockIdx.x, (int)threadIdx.x, 256);
    for (int i = 4 * (int)blockIdx.x + wave_id(); i < p.entries; i += 4 * (int)gridDim.x) work(i, lane_id(), WAVE);
}
__global__ __launch_bounds__(256) void pages_share_kernel(PagesArgs p)
{
    __shared__ ForkClaims claims;
    fork_claims(p, claims);
    each_entry(p, [&](int i, int thread, int threads) { fork_share(p, i, claims, thread, threads); });
}
__global__ __launch_bounds__(PG_THREADS) void pages_allocate_kernel(PagesArgs p)
{
    __shared__ int parts[PG_WAVES];
    fork_allocate(p, parts);
}
__global__ __launch_bounds__(256) void pages_place_kernel(PagesArgs p)
{
    each_entry(p, [&](int i, int thread, int threads) { fork_place(p, i, thread, threads); });
}
// the three in one, a wave an entry
__global__ __launch_bounds__(PG_THREADS) void pages_fork_kernel(PagesArgs p)
{
    __shared__ ForkClaims claims;
    __shared__ int parts[PG_WAVES];
    fork_claims(p, claims);
    for (int i = wave_id(); i < p.entries; i += PG_WAVES) fork_share(p, i, claims, lane_id(), WAVE);
    __threadfence();                                     // counts of uses are made in memory, by atomics
    __syncthreads();
    fork_allocate(p, parts);
    __syncthreads();
    for (int i = wave_id(); i < p.entries; i += PG_WAVES) fork_place(p, i, lane_id(), WAVE);
}

// ---- what is left moves together ----------------------------------------------------------------------
// The used pages number `used` and up move, in their order, into the free ones below.  scratch: [0] used, then the new number of every page.
__global__ __launch_bounds__(PG_THREADS) void pages_moves_kernel(PagesArgs p)
{
    __shared__ int parts[PG_WAVES];
    int mine = 0, used;
#pragma unroll 8
    for (int i = (int)threadIdx.x; i < p.pages; i += PG_THREADS) mine += p.uses[i] > 0 ? 1 : 0;
    block_prefix(mine, parts, used);
    if (threadIdx.x == 0) p.scratch[0] = used;
    const int holes = lowest_free(p.uses, used, used, parts, [&](int rank, int page) { p.targets[rank] = page; });
    __syncthreads();
    int moved = 0;
    for (int first = used; first < p.pages && moved < holes; first += 4 * PG_THREADS) {
        const int at = first + 4 * (int)threadIdx.x;
        int use[4], some = 0, all;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            use[j] = at + j < p.pages ? p.uses[at + j] : 0;
            some += use[j] > 0 ? 1 : 0;
        }
        int rank = moved + block_prefix(some, parts, all);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (use[j] > 0 && rank < holes) {
                const int to = p.targets[rank];
                p.sources[rank] = at + j;
                p.scratch[1 + at + j] = to;
                p.uses[to] = use[j];
                p.uses[at + j] = 0;
                ++rank;
            }
        moved += all;
    }
    for (int i = holes + (int)threadIdx.x; i < p.entries; i += PG_THREADS) p.sources[i] = p.targets[i] = -1;
}
__global__ __launch_bounds__(256) void pages_renumber_kernel(PagesArgs p)
{
    const int b = (int)blockIdx.x, used = p.scratch[0], count = pages_of(length_of(p, b), p.page_shift);
    for (int j = (int)threadIdx.x; j < count; j += 256) {
        int32_t *at = p.table + (size_t)b * p.width + j;
        const int page = *at;
        if (page >= used && page < p.pages) *at = p.scratch[1 + page];
    }
}

// ---- copies of pages ----------------------------------------------------------------------------------
// Pieces of 16 KB of a page's keys or values, dealt to the workgroups in order; the scales go with the first of each.
constexpr int COPY_PIECE = 16384;
__device__ __forceinline__ void copy_bytes(const unsigned char *from, unsigned char *to, int bytes)
{
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = 16 * (256 * j + (int)threadIdx.x);
        if (at < bytes) x[j] = ldg16_stream(from + at);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = 16 * (256 * j + (int)threadIdx.x);
        if (at < bytes) stg16_stream(to + at, x[j]);
    }
}
__global__ __launch_bounds__(256) void pages_copy_kernel(PageCopyArgs p)
{
    const int per = (int)((p.page_bytes + COPY_PIECE - 1) / COPY_PIECE), whole = 2 * per;
    const long long pieces = (long long)p.count * whole;
    for (long long piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
        const int pair = (int)(piece / whole), part = (int)(piece - (long long)pair * whole), at = part % per;
        const int from = p.sources[pair], to = p.targets[pair];
        if (from < 0 || from >= p.from_pages || to < 0 || to >= p.pages) continue;
        const bool values = part >= per;
        const size_t first = (size_t)at * COPY_PIECE;
        const int bytes = (int)(p.page_bytes - (long long)first < COPY_PIECE ? p.page_bytes - (long long)first : COPY_PIECE);
        copy_bytes((const unsigned char *)(values ? p.from_values : p.from_keys) + (size_t)from * p.page_bytes + first,
                   (unsigned char *)(values ? p.values : p.keys) + (size_t)to * p.page_bytes + first, bytes);
        if (at == 0)
            for (long long s = 0; s < p.scale_bytes; s += COPY_PIECE)
                copy_bytes((const unsigned char *)(values ? p.from_value_scales : p.from_key_scales) + (size_t)from * p.scale_bytes + s,
                           (unsigned char *)(values ? p.value_scales : p.key_scales) + (size_t)to * p.scale_bytes + s,
                           (int)(p.scale_bytes - s < COPY_PIECE ? p.scale_bytes - s : COPY_PIECE));
    }
}

}  // namespace

constexpr int FORK_GROUPS = 512;

size_t pages_fork_scratch(int entries, int width) { return (size_t)entries * (width + 4) * sizeof(int32_t); }

hipError_t launch_pages_append(const PagesArgs &p, hipStream_t st)
{
    constexpr int ALONE = 4096;                          // tokens whose slots the one workgroup writes itself
    pages_append_kernel<<<1, PG_THREADS, 0, st>>>(p, p.tokens <= ALONE);
    if (p.tokens > ALONE) {
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
        pages_slots_kernel<<<(p.tokens + 255) / 256 < 2048 ? (p.tokens + 255) / 256 : 2048, 256, 0, st>>>(p);
    }
    return hipGetLastError();
}
hipError_t launch_pages_free(const PagesArgs &p, hipStream_t st)
{
    pages_free_kernel<<<p.entries, 256, 0, st>>>(p);
    return hipGetLastError();
}
hipError_t launch_pages_fork(const PagesArgs &p, hipStream_t st)
{
    // An entry a wave and a row one load: 11 us in one launch, 10.5 in three, which take the host 4 us longer.  16 entries of 256 pages: 14.3
    // and 11.1 us, 64 of 32: 17.2 and 11.1.
    if (p.entries <= PG_WAVES && p.width <= WAVE) {
        pages_fork_kernel<<<1, PG_THREADS, 0, st>>>(p);
        return hipGetLastError();
    }
    // every workgroup goes through all entries for the claims: 4000 entries 99 us with a workgroup each, 55 with 512 of them
    const int groups = p.entries < FORK_GROUPS ? p.entries : FORK_GROUPS;
    pages_share_kernel<<<groups, 256, 0, st>>>(p);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    pages_allocate_kernel<<<1, PG_THREADS, 0, st>>>(p);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
    pages_place_kernel<<<groups, 256, 0, st>>>(p);
    return hipGetLastError();
}
hipError_t launch_pages_compact(const PagesArgs &p, hipStream_t st)
{
    pages_moves_kernel<<<1, PG_THREADS, 0, st>>>(p);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    pages_renumber_kernel<<<p.sequences, 256, 0, st>>>(p);
    return hipGetLastError();
}
hipError_t launch_pages_copy(const PageCopyArgs &p, hipStream_t st)
{
    const long long pieces = (long long)p.count * 2 * ((p.page_bytes + COPY_PIECE - 1) / COPY_PIECE);
    pages_copy_kernel<<<(unsigned)(pieces < 4096 ? pieces : 4096), 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace bsa

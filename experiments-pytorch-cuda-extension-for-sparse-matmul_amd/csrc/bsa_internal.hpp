// Host-side launchers behind the C ABI (one per kernel family).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bsa {

hipError_t launch_layout_build(const uint8_t *mask, int R, int C, int32_t *row_blocks,
                               int32_t *row_off, int32_t *col_blocks, int32_t *col_off,
                               int32_t *nnz_out, void *workspace, hipStream_t stream);

hipError_t launch_layout_finish(const int32_t *row_in, const int32_t *col_in, int nnz, int C, int32_t *row_blocks,
                                int32_t *col_blocks, int64_t *positions, int64_t *cells, hipStream_t stream);

hipError_t launch_schedule_build(const int32_t *offsets, int groups, int cap, int waves,
                                 int flags, int slice_max, int slices, int32_t *sched, int64_t capacity,
                                 int32_t *counts_out, hipStream_t stream);

hipError_t launch_to_sparse(int elem_size, const void *dense, void *sparse, const int32_t *row_blocks,
                            int nnz, int batches, int R, int C, hipStream_t stream);
hipError_t launch_to_dense(int elem_size, const void *sparse, void *dense, const uint8_t *mask,
                           const int32_t *ordinal_of, int nnz, int batches, int R, int C, hipStream_t stream);

struct MatmulArgs {
    const void *a, *b;
    void *c;
    const int32_t *blocks;
    const int32_t *sched;      // group records, then wavefront slots
    int groups;
    int sched_wgs, sched_waves;
    int tile_slots, split_groups;   // partial tiles / counters one (batch, strip) needs
    void *workspace;
    int nnz, batches;
    int M, N, K;
    bool tr_a, tr_b;
    bool sparse_shared;   // DSD / DDS: the sparse operand has no batch dimension
    bool row_table = false;   // DSD / DDS: `blocks` is the row-major table, whose pair p names block p
};

hipError_t launch_sdd(int dtype, const MatmulArgs &p, hipStream_t stream);
size_t gw_counter_bytes(int split_groups, int batches, int free_dim);
size_t gw_workspace_bytes(int tile_slots, int split_groups, int batches, int free_dim);
// group walk shared by DSD (dsd = true) and DDS
hipError_t launch_group_walk(int dtype, bool dsd, const MatmulArgs &p, hipStream_t stream);
// the same walk with the split-group workspace in the library's static device buffer (p.workspace is ignored)
hipError_t launch_group_walk_static_scratch(int dtype, bool dsd, const MatmulArgs &p, hipStream_t stream);

// DSD on a mask of 64 x 64 blocks (coarse tables: one pair per block)
struct Block64Args {
    const void *a, *b;
    void *c;
    const int32_t *blocks, *offsets;   // row table of the coarse mask
    const int32_t *sched;              // schedule of that table, built without splitting
    int coarse_rows, coarse_cols, coarse_nnz;
    int sched_wgs, sched_waves;
    int batches, N;
    bool sparse_shared;
};
hipError_t launch_dsd_block64(int dtype, const Block64Args &p, hipStream_t stream);

// DSD over runs of block rows with the dense strips of a run resident in LDS (dsd_runs.hip)
constexpr int RUN_RECORD_BYTES = 160;      // one record per run; the schedule is [records x mask rows][one byte per pair]
constexpr int RUN_MAX_STRIPS = 39;         // 4 KB each, next to the per-wave flags, in the 160 KB of a compute unit
constexpr int RUN_MAX_WAVES = 12;
hipError_t launch_run_schedule_build(const int32_t *row_blocks, const int32_t *row_offsets, int rows, int nnz,
                                     int target_pairs, int max_strips, void *sched, int32_t *counts_out,
                                     hipStream_t stream);
struct RunsArgs {
    const void *a, *b;
    void *c;
    const int32_t *blocks, *offsets;   // row table
    const void *sched;                 // run schedule of that table
    int n_runs, waves, strips;         // strips: the widest run's (counts_out[1] of the build)
    int mask_rows, mask_cols, nnz;
    int batches, N;
    bool sparse_shared;
};
hipError_t launch_dsd_runs(int dtype, const RunsArgs &p, hipStream_t stream);

// products of a block-sparse weight with many dense rows, and the weight's gradient (weight_panels.hip)
// Dense rows of a workgroup: 64 to 160, chosen by the launch; 96 is what callers that weigh this walk against bsa_matmul's
// reckon with (their line was measured with it).
constexpr int PANEL_ROWS = 96;
constexpr int PANEL_MAX_KBLOCKS = 1024;            // the lists of eight groups: 32 KB of LDS
constexpr int PANEL_MAX_NNZ = (1 << 20) - 1;       // 2 KB blocks within a 31-bit buffer range
struct WeightPanelArgs {
    const void *dense, *sparse;
    void *out;
    const int32_t *blocks, *offsets;
    int groups, nnz, rows, KT, batches;            // rows: dense rows of one launch entry
    bool row_groups, sparse_shared;
};
hipError_t launch_weight_panels(int dtype, const WeightPanelArgs &p, hipStream_t stream);
struct WeightGradArgs {
    const void *a, *b;
    void *out;
    float *parts;                                  // [shares][nnz][1024]
    const int32_t *blocks, *offsets;               // row table
    int mask_rows, mask_cols, nnz;
    int tokens, shares;
};
int weight_grad_shares(int mask_rows, int mask_cols, int tokens);
hipError_t launch_weight_grad(int dtype, const WeightGradArgs &p, hipStream_t stream);

struct SoftmaxArgs {
    const void *x;    // forward: scores; backward: y
    const void *dy;   // backward only
    void *out;
    const int32_t *blocks;
    const int32_t *sched;
    int groups;
    int sched_wgs, sched_waves;
    int nnz, batches;
    float scale;
    bool causal;
};

hipError_t launch_softmax_forward(int dtype, const SoftmaxArgs &p, hipStream_t stream);
hipError_t launch_softmax_backward(int dtype, const SoftmaxArgs &p, hipStream_t stream);

struct AttentionArgs {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void *out = nullptr;            // forward: result; backward: the forward result (read)
    void *lse = nullptr;            // forward: optional output; backward: input
    const void *dout = nullptr;     // backward only
    void *p_out = nullptr, *ds_out = nullptr;   // row walk of the backward pass, both or neither: [batches, nnz, 32, 32]
    void *dq_out = nullptr;         // row walk, may be null: [batches, 32 mask_rows, head_dim]
    void *delta = nullptr;          // float [batches, 32 mask_rows], rowsum(dout o out): written by the row walk (may be
                                    // null there), read by the column walk
    void *dk_out = nullptr, *dv_out = nullptr;  // column walk: [batches, 32 mask_cols, head_dim]
    int nnz = 0;
    const int32_t *blocks = nullptr;
    const int32_t *sched = nullptr;
    int groups = 0;                 // block rows (block columns for the column walk)
    int sched_wgs = 0, sched_waves = 0;
    int tile_slots = 0, split_groups = 0;   // parked tiles / counters one batch entry needs for the split groups of this walk
    void *workspace = nullptr;
    int mask_rows = 0, mask_cols = 0, batches = 0;
    float scale = 1.f;
    bool causal = false;
    bool bf16 = false;      // operands are bfloat16, not fp16
    int head_dim = 64;      // 64 or 128
};

size_t attention_workspace_bytes(int tile_slots, int split_groups, int batches, int head_dim);
// row walk region first, then the column walk's; either may be empty
size_t attention_backward_workspace_bytes(int row_tile_slots, int row_split_groups, int col_tile_slots,
                                          int col_split_groups, int batches, int head_dim);
hipError_t launch_attention_forward(const AttentionArgs &p, hipStream_t stream);
hipError_t launch_attention_backward_scores(const AttentionArgs &p, hipStream_t stream);
constexpr int AT_COLUMN_WAVES_128 = 4;    // waves per workgroup the column walk takes at head dim 128
hipError_t launch_attention_backward_dkdv(const AttentionArgs &p, hipStream_t stream);   // groups = block columns

// attention over packed sequences (packed_attention.hip); strides in values
struct PackedArgs {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    const void *dout = nullptr, *o = nullptr, *o_rest = nullptr;     // backward only; o: the forward result, o_rest: its rest; dense
    void *out = nullptr;                         // forward: the result; backward: dq
    void *rest = nullptr;                        // forward: what the result's rounding took; null with lse
    void *dk = nullptr, *dv = nullptr;           // both or neither
    float *lse = nullptr;                        // [heads][tokens]; forward: written, may be null; backward: read
    float *delta = nullptr;                      // backward: scratch of the same size
    const int32_t *offsets = nullptr;
    int tokens = 0, sequences = 0, heads = 0, key_heads = 0, head_dim = 64;
    long long q_token = 0, q_head = 0, k_token = 0, k_head = 0, v_token = 0, v_head = 0, g_token = 0, g_head = 0;
    float scale = 1.f;
    bool causal = true, bf16 = false;
};
// whether every launch has fewer than 2^32 threads; key_gradients: those of the backward call's walk over the keys too (a forward call whose
// statistics are wanted asks for them, so that a training step is refused before it has begun)
bool packed_fits(const PackedArgs &p, bool key_gradients);
hipError_t launch_packed_forward(const PackedArgs &p, hipStream_t stream);
hipError_t launch_packed_backward(const PackedArgs &p, hipStream_t stream);

// linear attention over packed sequences (linear_attention.hip); strides in values
struct LinearArgs {
    const void *q = nullptr, *k = nullptr, *v = nullptr, *dout = nullptr;
    void *out = nullptr, *dq = nullptr, *dk = nullptr, *dv = nullptr;
    const float *log_decay = nullptr;            // [key_heads]
    const int32_t *offsets = nullptr;
    const float *first = nullptr;                // [sequences][key_heads][head_dim][head_dim], may be null; the same for the next three
    float *last = nullptr;                       // forward
    const float *dlast = nullptr;                // backward: gradients of the last states
    float *dfirst = nullptr;                     // backward: of the first
    float *states = nullptr, *back_states = nullptr;     // between segments: written by the forward pass; scratch of the backward pass
    int tokens = 0, sequences = 0, heads = 0, key_heads = 0, head_dim = 64, segment = 0;     // segment: tokens, a multiple of 32
    long long q_token = 0, q_head = 0, k_token = 0, k_head = 0, v_token = 0, v_head = 0, g_token = 0, g_head = 0;
    float scale = 1.f;
    bool bf16 = false;
};
int linear_segment(int tokens, int sequences, int key_heads, int head_dim);
size_t linear_workspace_bytes(const LinearArgs &p);
bool linear_fits(const LinearArgs &p);
hipError_t launch_linear_forward(const LinearArgs &p, hipStream_t stream);
hipError_t launch_linear_backward(const LinearArgs &p, hipStream_t stream);

// one token of every sequence against states in slots (linear_step.hip)
struct LinearStepArgs {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void *out = nullptr;
    const float *log_decay = nullptr;
    float *states = nullptr;                     // [slots][key_heads][head_dim][head_dim]
    const int32_t *at = nullptr;                 // [batch]
    int batch = 0, slots = 0, heads = 0, key_heads = 0, head_dim = 64;
    long long q_token = 0, q_head = 0, k_token = 0, k_head = 0, v_token = 0, v_head = 0;
    float scale = 1.f;
    bool bf16 = false;
};
hipError_t launch_linear_step(const LinearStepArgs &p, hipStream_t stream);

// rows into and out of a paged cache (cache_rows.hip); strides in values
struct CacheRowsArgs {
    const void *k = nullptr, *v = nullptr;       // write: read; read: the results
    void *keys = nullptr, *values = nullptr;
    float *key_scales = nullptr, *value_scales = nullptr;
    const int32_t *slots = nullptr;
    int tokens = 0, heads = 0, head_dim = 0, pages = 0, page_shift = 0, kind = 0;
    bool held_bf16 = false;                      // what a 16-bit cache holds
    long long k_token = 0, k_head = 0, v_token = 0, v_head = 0;
};
hipError_t launch_cache_write(int dtype, const CacheRowsArgs &p, hipStream_t stream);
hipError_t launch_cache_read(int dtype, const CacheRowsArgs &p, hipStream_t stream);

// new tokens over a paged cache and themselves (cached_attention.hip); strides in values
struct CachedArgs {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void *out = nullptr;                         // dense [batch][drafts][heads][head_dim]
    const void *keys = nullptr, *values = nullptr;
    const float *key_scales = nullptr, *value_scales = nullptr;
    const int32_t *table = nullptr, *lengths = nullptr;
    const unsigned char *tree = nullptr;
    void *workspace = nullptr;
    int batch = 0, drafts = 0, heads = 0, key_heads = 0, head_dim = 0, kind = 0, pages = 0, page_shift = 0, width = 0;
    bool bf16 = false, tree_shared = false;
    float scale = 1.f;
    long long q_batch = 0, q_token = 0, q_head = 0, k_batch = 0, k_token = 0, k_head = 0, v_batch = 0, v_token = 0, v_head = 0;
};
bool cached_attention_splits(const CachedArgs &p);       // a sequence may have several chunks
long long cached_attention_units(const CachedArgs &p);
long long cached_attention_parts(const CachedArgs &p);   // rows that chunks can leave in the workspace
size_t cached_attention_workspace_bytes(const CachedArgs &p);
hipError_t launch_cached_attention(const CachedArgs &p, hipStream_t stream);

// which pages each sequence has (pages.hip)
constexpr int PAGES_MOST_SEQUENCES = 4096;       // and entries of a call: the workgroup that deals pages has them in LDS
struct PagesArgs {
    int32_t *table = nullptr, *lengths = nullptr, *uses = nullptr, *missing = nullptr;
    const int32_t *offsets = nullptr;            // append: of the new tokens, [sequences + 1]
    int32_t *slots = nullptr;                    // append: [tokens]
    const int32_t *parents = nullptr, *children = nullptr;       // fork; free: children
    int32_t *sources = nullptr, *targets = nullptr;              // [entries]
    int32_t *scratch = nullptr;
    int tokens = 0, entries = 0, sequences = 0, width = 0, pages = 0, page_shift = 0;
};
size_t pages_fork_scratch(int entries, int width);
hipError_t launch_pages_append(const PagesArgs &p, hipStream_t stream);
hipError_t launch_pages_free(const PagesArgs &p, hipStream_t stream);
hipError_t launch_pages_fork(const PagesArgs &p, hipStream_t stream);
hipError_t launch_pages_compact(const PagesArgs &p, hipStream_t stream);
struct PageCopyArgs {
    const void *from_keys = nullptr, *from_values = nullptr, *from_key_scales = nullptr, *from_value_scales = nullptr;
    void *keys = nullptr, *values = nullptr, *key_scales = nullptr, *value_scales = nullptr;
    const int32_t *sources = nullptr, *targets = nullptr;
    int count = 0, pages = 0, from_pages = 0;
    long long page_bytes = 0, scale_bytes = 0;
};
hipError_t launch_pages_copy(const PageCopyArgs &p, hipStream_t stream);

}  // namespace bsa

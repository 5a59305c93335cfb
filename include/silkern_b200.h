/*
 * silkern_b200 -- C ABI of the B200 (sm_100a) sparse-index localization converter.
 *
 * The converter turns one selection batch of global logical token positions
 * (batch, width) int32 into the rank-local physical KV slots that one decode
 * context-parallel (DCP) rank owns, compacted to the front of each row in the
 * selector's order, plus an exact valid count per row.
 *
 * Per element t of row r (request q = req_ids[r], table row = block_table[q]):
 *   owner = (t / interleave) % dcp_size                       (t >= 0 only)
 *   local = (t / (dcp_size * interleave)) * interleave + t % interleave
 *   lb, off = local / block_size, local % block_size
 *   valid  = t >= 0 && owner == dcp_rank && lb < table_width
 *   phys   = block_table[q][lb] * block_size + off            (int32 wrap)
 * With compaction (compact_valid_to_front && dcp_size > 1) the valid values
 * fill out[r][0:count] in input order and the rest of the row is -1; without
 * it every column keeps its own value (phys, or -1 when invalid).
 *
 * Conventions shared by every entry point:
 *   - every buffer is caller-owned int32 device memory, contiguous, on the
 *     device that is current on the calling thread; nothing is allocated and
 *     nothing is synchronised, so calls may be captured in a CUDA graph;
 *   - `stream` is a cudaStream_t (NULL = legacy default stream);
 *   - launches use programmatic dependent launch: each kernel waits on the
 *     previous grid in the stream before it reads any input;
 *   - `status` may be NULL; otherwise a row whose request id is outside
 *     [0, table_rows) is emitted as all -1 with count 0 and the kernel stores
 *     SILKERN_STATUS_BAD_REQUEST into *status, and a cluster whose count
 *     exchange ran out of its wait bound ORs in SILKERN_STATUS_EXCHANGE_TIMEOUT
 *     (the kernel never clears *status);
 *   - return value: 0 on success, a positive SILKERN_E* code when an argument
 *     is rejected before launch (nothing is enqueued), or -(cudaError_t) when
 *     the launch itself fails.
 */
#ifndef SILKERN_B200_H_
#define SILKERN_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SILKERN_ABI_VERSION 1

#define SILKERN_OK 0
#define SILKERN_E_NULL 1         /* a required pointer is NULL */
#define SILKERN_E_SHAPE 2        /* batch/width/table dimensions out of range */
#define SILKERN_E_DCP 3          /* invalid dcp_size / dcp_rank / interleave */
#define SILKERN_E_BLOCK_SIZE 4   /* block_size < 1 or not divisible by interleave */
#define SILKERN_E_TILE 5         /* unsupported tile_size */
#define SILKERN_E_ALIAS 6        /* an output overlaps an input, another output or itself */
#define SILKERN_E_GEOMETRY 7     /* explicit launch geometry rejected */
#define SILKERN_E_SCRATCH 8      /* batch x tiles exceeds SILKERN_NOALLOC_MAX_TILES */
#define SILKERN_E_CACHE 9        /* unsupported cache geometry, stride or alignment */
#define SILKERN_E_HEADS 10       /* heads not a positive multiple of the cache's heads */
#define SILKERN_E_TYPE 11        /* element type is neither SILKERN_BF16 nor SILKERN_F16 */
#define SILKERN_E_ATTEND 12      /* window, sinks or softmax scale out of range */

#define SILKERN_STATUS_BAD_REQUEST 1
/* Status bit of the converter entry points (OR-ed into *status): a row split
 * over a thread-block cluster whose CTAs did not complete their count
 * exchange within the kernel's wait bound. The CTAs that gave up store
 * nothing for that row (out, counts and tiles keep their previous contents).
 * It does not occur in a working cluster launch. */
#define SILKERN_STATUS_EXCHANGE_TIMEOUT 4
/* Status bit of the fused top-k entry point (OR-ed into *status). */
#define SILKERN_STATUS_BAD_LENGTH 2 /* a seq_len outside [0, logits_width]; clamped */

/* Widest selection row either entry point accepts. */
#define SILKERN_MAX_ROW_WIDTH 16384
/* Hierarchical tile sizes accepted by the workspace geometry. */
#define SILKERN_MIN_TILE_SIZE 64
#define SILKERN_MAX_TILE_SIZE 1024

/*
 * Row-wise stable localization: one launch; each row is scanned by one CTA
 * or by a group of threads inside one (or, for long rows with few requests,
 * by a thread-block cluster that exchanges per-CTA counts through distributed
 * shared memory).
 * Replaces silkern/kernels.py:318-434 (localize_rowwise and _rowwise_kernel,
 * kernels.py:51-125). block_table is (table_rows, table_width); tokens and
 * out are (batch, width); req_ids and counts are (batch,).
 */
int silkern_localize_rowwise_v1(const int32_t* req_ids, const int32_t* block_table,
                                int64_t table_rows, int64_t table_width,
                                const int32_t* tokens, int32_t* out, int32_t* counts,
                                int64_t batch, int64_t width, int32_t block_size,
                                int32_t dcp_size, int32_t dcp_rank, int32_t dcp_interleave,
                                int32_t compact_valid_to_front, int32_t* status,
                                void* stream);

/*
 * Hierarchical stable localization for wide rows: each row is split into
 * tiles of tile_size columns; the CTAs of one row form a thread-block cluster,
 * compose their tile-prefix offsets deterministically (no atomics) and
 * publish them into the caller-owned workspace: tile_counts[r][k] is the
 * number of valid elements in tile k and tile_offsets[r][k] the exclusive
 * prefix of those counts, both (batch, ceil(width / tile_size)).
 * mapped_ws and local_positions_ws, (batch, width), are accepted for
 * interface compatibility and are neither read nor written (may be NULL).
 * Replaces silkern/kernels.py:436-633 (localize_hierarchical and the
 * _map_tiles / _tile_prefix / _fill_output / _scatter_tiles kernels,
 * kernels.py:127-315).
 */
int silkern_localize_hierarchical_v1(const int32_t* req_ids, const int32_t* block_table,
                                     int64_t table_rows, int64_t table_width,
                                     const int32_t* tokens, int32_t* out, int32_t* counts,
                                     int32_t* mapped_ws, int32_t* local_positions_ws,
                                     int32_t* tile_counts_ws, int32_t* tile_offsets_ws,
                                     int64_t batch, int64_t width, int32_t block_size,
                                     int32_t dcp_size, int32_t dcp_rank, int32_t dcp_interleave,
                                     int32_t compact_valid_to_front, int32_t tile_size,
                                     int32_t* status, void* stream);

/*
 * Exact caller-owned workspace shapes for the hierarchical entry point, as
 * four (rows, cols) pairs in the order mapped, local_positions, tile_counts,
 * tile_offsets. Host only; touches no device. Replaces
 * silkern/workspace.py:22-53 (workspace_shapes).
 */
int silkern_workspace_shapes_v1(int64_t batch, int64_t width, int32_t tile_size,
                                int64_t out_shapes[8]);

/*
 * Row-wise or hierarchical localization with an explicit launch geometry, for
 * conformance sweeps and tuning: cluster_size CTAs per row (1, 2, 4 or 8),
 * stage_table = 1 stages the request's block-table row in shared memory
 * (table_width <= 4096), 0 gathers it from global memory, -1 lets the
 * library decide; prefetch_table likewise for the L2 bulk prefetch of the
 * whole table; chunks_per_thread (1, 2, 4 or 8; 0 = library choice) makes
 * each thread map a run of 4 x chunks_per_thread consecutive columns.
 * tile_size = 0 selects row-wise semantics (no workspace).
 * Same semantics and outputs as the entry points above. No counterpart in the
 * reference (its launch geometry is fixed inside each launcher).
 */
int silkern_localize_explicit_v1(const int32_t* req_ids, const int32_t* block_table,
                                 int64_t table_rows, int64_t table_width,
                                 const int32_t* tokens, int32_t* out, int32_t* counts,
                                 int32_t* tile_counts_ws, int32_t* tile_offsets_ws,
                                 int64_t batch, int64_t width, int32_t block_size,
                                 int32_t dcp_size, int32_t dcp_rank, int32_t dcp_interleave,
                                 int32_t compact_valid_to_front, int32_t tile_size,
                                 int32_t cluster_size, int32_t stage_table,
                                 int32_t prefetch_table, int32_t chunks_per_thread,
                                 int32_t* status, void* stream);

/*
 * Hierarchical localization for callers that cannot allocate device memory:
 * the same computation and outputs (out, counts) as
 * silkern_localize_hierarchical_v1, but without workspace arguments. Its
 * tile workspace (tile counts and tile offsets) lives in a fixed array inside
 * this library, SILKERN_NOALLOC_MAX_TILES entries for each, 256 KiB in total,
 * which every GPU that loads the library holds until the process exits.
 * Callers whose memory is planned outside their control use it: plugin hosts
 * and serving runtimes whose enqueue path forbids cudaMalloc, or code run
 * while another framework records a CUDA graph, where a new allocation would
 * break the recording or stall it.
 *   - batch * ceil(width / tile_size) above SILKERN_NOALLOC_MAX_TILES is
 *     rejected with SILKERN_E_SCRATCH before anything is launched;
 *   - the first call on a device looks up the array's device address with
 *     that device current, so make that first call before any stream capture;
 *   - every call shares the one array and leaves its tile decomposition there
 *     (nothing in it has to start at zero: each call writes every entry it
 *     uses before reading any), so calls that overlap on the GPU, from two
 *     streams or two threads, race on it and must be serialised.
 * Nothing is allocated or freed. No counterpart in the reference (its
 * hierarchical launcher always takes caller-owned workspace).
 */
#define SILKERN_NOALLOC_MAX_TILES 32768
int silkern_localize_hierarchical_noalloc_v1(const int32_t* req_ids, const int32_t* block_table,
                                             int64_t table_rows, int64_t table_width,
                                             const int32_t* tokens, int32_t* out,
                                             int32_t* counts, int64_t batch, int64_t width,
                                             int32_t block_size, int32_t dcp_size,
                                             int32_t dcp_rank, int32_t dcp_interleave,
                                             int32_t compact_valid_to_front, int32_t tile_size,
                                             int32_t* status, void* stream);

/*
 * Device-side equality check used by the CUDA-graph replay gate: adds the
 * number of positions i < n with a[i] != b[i] to *mismatches (one atomic add
 * per CTA). No counterpart in the reference (its replay check copies to the
 * host, silkern/verify.py:362-372).
 */
int silkern_count_mismatches_v1(const int32_t* a, const int32_t* b, int64_t n,
                                int32_t* mismatches, void* stream);

/*
 * silkern_count_mismatches_v1 per segment, for the decode-step replay gate:
 * a and b hold `segments` consecutive segments of segment_elems int32 each
 * (one per layer of a step), and counters[s] (int32, segments entries) is
 * increased by the number of positions of segment s where a and b differ.
 * One launch; segments <= 65535. No counterpart in the reference.
 */
int silkern_count_segment_mismatches_v1(const int32_t* a, const int32_t* b, int64_t segments,
                                        int64_t segment_elems, int32_t* counters, void* stream);

/*
 * Measurement reference, not the product: dst[0..n) = src[0..n) (int32) with
 * the converter's data movement and launch mode and none of its work. CTAs of
 * `threads` threads (a multiple of 32, at most 1024) each copy a contiguous
 * chunk of threads * run elements, each thread a run of `run` (8 or 16)
 * elements with 256-bit accesses where aligned; programmatic dependent launch,
 * with a bulk L2 prefetch of the chunk issued before the wait on the previous
 * grid. ctas_per_sm in 1..8 reserves shared memory so that at most that many
 * of these CTAs share an SM (the converter's residency control); 0 reserves
 * none. The time of back-to-back calls over the converter's tokens and output
 * is the floor a converter call of the same size runs against. src and dst
 * must not overlap (SILKERN_E_ALIAS). No counterpart in the reference.
 */
int silkern_copy_floor_v1(const int32_t* src, int32_t* dst, int64_t n, int32_t run, int32_t threads,
                          int32_t ctas_per_sm, void* stream);

/*
 * Comparison baseline, not the product: the atomic-reservation converter of
 * the reference's bench/atomic_baseline.py:40-111 and :313-385 (itself a
 * restatement of the upstream vLLM converter). Same set and counts as the
 * entry points above, but each 128-column tile reserves its output segment
 * with an atomicAdd on scratch[row] (int32, (batch,)), so the order of the
 * segments varies from run to run. Three stream operations: reset, reserve
 * and scatter, counts <- scratch.
 */
int silkern_atomic_baseline_v1(const int32_t* req_ids, const int32_t* block_table,
                               int64_t table_rows, int64_t table_width, const int32_t* tokens,
                               int32_t* out, int32_t* counts, int32_t* scratch, int64_t batch,
                               int64_t width, int32_t block_size, int32_t dcp_size,
                               int32_t dcp_rank, int32_t dcp_interleave, void* stream);

/*
 * Fused indexer top-k + localization: selection and conversion in one launch,
 * without the (batch, top_k) selection round trip through HBM. This is the
 * "fuse the converter into the indexer's top-k epilogue" step beyond the
 * reference's converter boundary; its localization half is the contract above
 * (silkern/contract.py:67-158), applied to the selected positions.
 *
 * logits is float32 (batch, logits_width) with row stride logits_stride
 * (elements, >= logits_width); row r scores the positions [0, L) with
 * L = seq_lens[r] (values outside [0, logits_width] are clamped and flagged
 * with SILKERN_STATUS_BAD_LENGTH); columns at and beyond L are never read.
 * Selection: every position when L <= top_k; otherwise the top_k positions
 * with the largest keys, where key(x) orders the float bit patterns totally
 * (-NaN < -inf < ... < -0 < +0 < ... < +inf < +NaN), ties going to the lower
 * position. The selected positions, in ascending order and padded with -1 to
 * top_k, form the selection row that is localized into out (batch, top_k)
 * and counts (batch,), exactly as silkern_localize_rowwise_v1 would localize
 * it. positions (batch, top_k) may be NULL; otherwise it receives that
 * selection row. 1 <= top_k <= SILKERN_MAX_ROW_WIDTH; logits_width <=
 * SILKERN_TOPK_MAX_WIDTH. One CTA per row: a sampled estimate of the
 * threshold, one streaming pass over the row that keeps candidate bit masks,
 * an exact radix select over the candidates in shared memory (or over the
 * whole row when the estimate misses), and the converter's compaction.
 */
#define SILKERN_TOPK_MAX_WIDTH 262144
int silkern_topk_localize_v1(const float* logits, int64_t logits_stride, int64_t logits_width,
                             const int32_t* seq_lens, const int32_t* req_ids,
                             const int32_t* block_table, int64_t table_rows, int64_t table_width,
                             int32_t* positions, int32_t* out, int32_t* counts, int64_t batch,
                             int32_t top_k, int32_t block_size, int32_t dcp_size, int32_t dcp_rank,
                             int32_t dcp_interleave, int32_t compact_valid_to_front,
                             int32_t* status, void* stream);

/*
 * silkern_topk_localize_v1 with explicit internals (tuning and test hook):
 * candidate_capacity entries in the shared-memory candidate list (0 =
 * automatic; top_k .. the shared-memory budget; a capacity of top_k sends
 * almost every row down the whole-row path) and stage_table (-1 automatic,
 * 0 gather the block table from global memory, 1 stage the request's row in
 * shared memory, which needs table_width <= 4096). SILKERN_E_GEOMETRY when
 * either is out of range.
 */
int silkern_topk_localize_explicit_v1(const float* logits, int64_t logits_stride,
                                      int64_t logits_width, const int32_t* seq_lens,
                                      const int32_t* req_ids, const int32_t* block_table,
                                      int64_t table_rows, int64_t table_width, int32_t* positions,
                                      int32_t* out, int32_t* counts, int64_t batch, int32_t top_k,
                                      int32_t block_size, int32_t dcp_size, int32_t dcp_rank,
                                      int32_t dcp_interleave, int32_t compact_valid_to_front,
                                      int32_t candidate_capacity, int32_t stage_table,
                                      int32_t* status, void* stream);

/*
 * silkern_topk_localize_explicit_v1 with the CTA shape pinned as well:
 * cta_threads 0 (automatic: 1024 threads, one CTA per SM, when batch is at
 * most the device's SM count, else 512 threads, two per SM), 512 or 1024.
 * SILKERN_E_GEOMETRY for any other value.
 */
int silkern_topk_localize_explicit_v2(const float* logits, int64_t logits_stride,
                                      int64_t logits_width, const int32_t* seq_lens,
                                      const int32_t* req_ids, const int32_t* block_table,
                                      int64_t table_rows, int64_t table_width, int32_t* positions,
                                      int32_t* out, int32_t* counts, int64_t batch, int32_t top_k,
                                      int32_t block_size, int32_t dcp_size, int32_t dcp_rank,
                                      int32_t dcp_interleave, int32_t compact_valid_to_front,
                                      int32_t candidate_capacity, int32_t stage_table,
                                      int32_t cta_threads, int32_t* status, void* stream);

/*
 * The 8-bit paged cache. A page (block) holds block_size consecutive
 * rank-local tokens; slot = block * block_size + offset is what the converter
 * emits. Keys and values are e4m3 codes, and every (block, head) pair has one
 * float32 scale for its keys and one for its values: the stored value is
 * scale * code. k is (num_blocks, block_size, kv_heads, key_dim) with strides
 * in bytes, multiples of 16, for the first three dimensions and 1 for the
 * last; v likewise with value_dim; k_scale and v_scale are contiguous
 * (num_blocks, kv_heads). A latent cache has one head, key_dim 576, v and
 * v_scale NULL and value_dim 512: the first 512 columns of a key are its
 * value, and k_scale is the scale of both. Scales lie in [2^-100, 2^100], or
 * are 0 (every value of the pair is 0) or NaN (every use gives NaN); codes of
 * visible tokens are finite (neither 0x7f nor 0xff). num_blocks * block_size
 * is below 2^31 and block_size at most 65536. Addresses of k and v are multiples
 * of 16.
 *
 * SILKERN_E_ALIAS: what a call writes shares memory with what it reads, or two
 * of its own elements do (a stride below what the smaller ones span). Buffers
 * with equal largest strides may lie between one another's rows; others are
 * compared as whole ranges of memory.
 */
typedef struct silkern_cache_v1 {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t num_blocks;
  int32_t block_size;
  int32_t kv_heads;
  int32_t key_dim;
  int32_t value_dim;
  int64_t k_block, k_token, k_head;
  int64_t v_block, v_token, v_head;
} silkern_cache_v1;

/* Element types of queries, new tokens and outputs. */
#define SILKERN_BF16 0
#define SILKERN_F16 1

/* Status bits of the cache entry points (OR-ed into *status, with
 * SILKERN_STATUS_BAD_REQUEST and SILKERN_STATUS_BAD_LENGTH): a slot past the
 * cache, or a token whose page is outside its table row or the cache. Such a
 * token is left out. */
#define SILKERN_STATUS_BAD_SLOT 8
/* Status bit of the attention entry points: a wait inside the kernel ran out
 * of its bound, and the pipeline of warps concerned gave up. The results of all
 * of its work items, and those of an item that it shared with others, are NaN.
 * It does not occur in a working launch. */
#define SILKERN_STATUS_WAIT_TIMEOUT 16

/*
 * Append tokens to the 8-bit cache. Sequence b (of `sequences`) has the new
 * tokens [cu_tokens[b], cu_tokens[b + 1]) of keys (tokens, kv_heads, key_dim)
 * and values (tokens, kv_heads, value_dim; NULL for a latent cache), at the
 * positions starts[b], starts[b] + 1, ... of the request req_ids[b]; the
 * positions that this rank owns are stored through block_table, the others
 * are skipped. keys and values have unit column stride and strides in
 * elements for tokens and heads.
 *
 * Scales are powers of two. With m the largest magnitude among the call's
 * tokens in one (page, head), the scale becomes max(old, w), w the smallest
 * power of two with 448 w >= m (within [2^-100, 2^100]; 0 where m is 0). A
 * page whose first token is among the call's is new: old counts as 0.
 * Otherwise, where the scale grows, the codes that the page holds are
 * rescaled (exact for a power of two, but for codes that become subnormal).
 * An infinity or NaN among a page's new values makes that scale NaN until the
 * page is new again. A page takes tokens from one sequence of the call at
 * most (a page shared by several requests is copied before one of them
 * appends to it). Nothing else is written.
 */
int silkern_append_quantized_v1(const silkern_cache_v1* cache, const void* keys, int64_t key_token,
                                int64_t key_head, const void* values, int64_t value_token,
                                int64_t value_head, int32_t type, int64_t tokens,
                                const int32_t* cu_tokens, const int32_t* starts,
                                const int32_t* req_ids, int64_t sequences,
                                const int32_t* block_table, int64_t table_rows,
                                int64_t table_width, int32_t dcp_size, int32_t dcp_rank,
                                int32_t dcp_interleave, int32_t* status, void* stream);

/*
 * Attention of each query row over its selected slots:
 *   out[r][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(softmax_scale * q[r][h] . k_j)
 *   lse[r][h] = log(sum_j p_j)
 * over j in [0, counts[r]) (counts may be NULL: the whole width) with
 * slots[r][j] >= 0; a row without such a j gets out 0 and lse -inf. q is
 * (rows, heads, key_dim) and out (rows, heads, value_dim), both of `type`,
 * with unit column stride, strides in elements for rows and heads (q's are
 * multiples of 8 and its address of 16); lse is float32 (rows, heads),
 * contiguous; slots has row stride slots_row. Query head h reads cache head
 * h / (heads / kv_heads). key_dim is 64 or 128 with value_dim the same, or
 * the cache is latent. A count outside [0, width] is clamped and flagged with
 * SILKERN_STATUS_BAD_LENGTH.
 */
int silkern_attend_selected_v1(const silkern_cache_v1* cache, const void* q, int64_t q_row,
                               int64_t q_head, int32_t type, int64_t rows, int32_t heads,
                               const int32_t* slots, int64_t slots_row, int64_t width,
                               const int32_t* counts, void* out, int64_t out_row, int64_t out_head,
                               float* lse, float softmax_scale, int32_t* status, void* stream);

/*
 * Attention through the block table. Sequence b has the queries
 * [cu_tokens[b], cu_tokens[b + 1]) of q, the last tokens of the request
 * req_ids[b], whose length is lengths[b] with them; the query at position t
 * sees the positions [max(0, t + 1 - window), t] and the first `sinks`
 * positions up to t (window 0: every position up to t), as far as this rank
 * owns them. Rows of q at and past cu_tokens[sequences] are not touched in
 * out and lse. Outputs, types and layouts as for silkern_attend_selected_v1.
 * A length below the number of queries is flagged with
 * SILKERN_STATUS_BAD_LENGTH; queries at negative positions see nothing.
 */
int silkern_attend_window_v1(const silkern_cache_v1* cache, const void* q, int64_t q_row,
                             int64_t q_head, int32_t type, int64_t rows, int32_t heads,
                             const int32_t* cu_tokens, const int32_t* lengths,
                             const int32_t* req_ids, int64_t sequences,
                             const int32_t* block_table, int64_t table_rows, int64_t table_width,
                             int64_t window, int64_t sinks, int32_t dcp_size, int32_t dcp_rank,
                             int32_t dcp_interleave, void* out, int64_t out_row, int64_t out_head,
                             float* lse, float softmax_scale, int32_t* status, void* stream);

/*
 * Join the partial results of `ranks` context-parallel ranks:
 *   lse[r][h] = log(sum_i exp(lses[i][r][h]))
 *   out[r][h] = sum_i exp(lses[i][r][h] - lse[r][h]) outs[i][r][h]
 * outs is (ranks, rows, heads, dim) with unit column stride and strides in
 * elements, lses float32 (ranks, rows, heads) contiguous, out (rows, heads,
 * dim) of the same type with strides, lse float32 (rows, heads) contiguous or
 * NULL. A partial result whose lse is -inf is not read; where all are, out
 * is 0 and lse -inf. The ranks are added in order.
 */
int silkern_merge_partials_v1(const void* outs, int64_t outs_rank, int64_t outs_row,
                              int64_t outs_head, const float* lses, int32_t type, int64_t ranks,
                              int64_t rows, int64_t heads, int64_t dim, void* out, int64_t out_row,
                              int64_t out_head, float* lse, void* stream);

/*
 * Bound, in cycles of an SM's clock, on each wait of the attention kernels for
 * another warp's part of one tile of 128 keys (waits over several tiles have as
 * many times the bound). 0 to 2^32; 4e9, about two seconds, to begin with. Holds
 * for launches, and captures into graphs, from then on in the whole process.
 * Returns the bound before; with a value out of range, changes nothing. For
 * debuggers and other slow surroundings, and for tests: with 0 a kernel gives up
 * at once, and says so as SILKERN_STATUS_WAIT_TIMEOUT does.
 */
int64_t silkern_attend_wait_bound_v1(int64_t cycles);

/* Static text for a return code (positive SILKERN_E*, 0, or -cudaError_t). */
const char* silkern_status_string_v1(int code);

/* SILKERN_ABI_VERSION of the loaded library. */
int silkern_abi_version_v1(void);

/*
 * Host check of the invariant-divisor division the kernels use: returns the
 * number of n in [n_begin, n_begin + n_count) (all < 2^31) for which the fast
 * quotient differs from n / divisor. Test hook; touches no device.
 */
int64_t silkern_fastdiv_selftest_v1(uint32_t divisor, uint32_t n_begin, uint32_t n_count);

#ifdef __cplusplus
}
#endif

#endif /* SILKERN_B200_H_ */

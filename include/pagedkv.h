/*
 * pagedkv.h — C ABI of the MI355X (gfx950) paged-KV library.
 *
 * Plain pointers, sizes and a HIP stream handle (hipStream_t passed as void*;
 * NULL means the null stream). Every device pointer is an ordinary device
 * allocation (or pinned host memory where stated). No torch types cross this
 * boundary. Every call is asynchronous on `stream` unless stated otherwise;
 * the kernels never read or write out of bounds: an out-of-range page id or
 * slot is skipped and reported through `status_word` (a device int32 whose
 * bits are OR-ed in; see PKV_STATUS_*), which the caller reads at a declared
 * check point.
 *
 * Return value: PKV_OK, or an error code with a message in pkv_last_error()
 * (thread-local, valid until the next call on the same thread).
 *
 * Pool layout (the reference's, serving/backends/paged_torch.py:127-137):
 * one allocation of `n_layers * 2` planes, plane (layer, kv) at
 * base + (layer * 2 + kv) * plane_bytes, each plane a contiguous
 * [num_blocks, page_size, n_kv_heads, head_dim] array. A per-layer K (or V)
 * pool is exactly one plane, so a caller that only has per-layer tensors
 * passes that plane's address to the per-layer entry points.
 */
#ifndef PAGEDKV_H
#define PAGEDKV_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types of the pool, q, k, v and out */
#define PKV_DTYPE_F16 0
#define PKV_DTYPE_BF16 1
#define PKV_DTYPE_F32 2

/* return codes */
#define PKV_OK 0
#define PKV_ERR_INVALID 1     /* argument or metadata error (Python: ValueError) */
#define PKV_ERR_RANGE 2       /* block id out of range (Python: IndexError) */
#define PKV_ERR_HIP 3         /* HIP runtime error */
#define PKV_ERR_CAPACITY 4    /* caller-provided buffer too small */

/* bits OR-ed into *status_word by the kernels */
#define PKV_STATUS_BAD_SLOT 1   /* slot_mapping entry outside [0, num_slots) */
#define PKV_STATUS_BAD_PAGE 2   /* kv_indices entry outside [0, num_blocks) */
#define PKV_STATUS_BAD_BLOCK 4  /* copy/gather/scatter id outside [0, num_blocks) */
#define PKV_STATUS_BAD_POSITION 8  /* position without a row of the rotation table */

/* Version of this ABI; bumped on any signature change. */
int pkv_abi_version(void);

/* Message for the last non-zero return on this thread ("" if none). */
const char* pkv_last_error(void);

/*
 * KV append — replaces PagedTorchBackend.append_kv
 * (serving/backends/paged_torch.py:209-276) and FlashInfer's
 * append_paged_kv_cache call (serving/backends/flashinfer_backend.py:502-512):
 * for t < n_tokens, row slot_mapping[t] of the flat [num_slots, n_kv_heads,
 * head_dim] view of k_pool / v_pool receives row t of k / v. k and v are
 * contiguous [n_tokens, n_kv_heads, head_dim] in the pool dtype.
 * Idempotent. Slots outside [0, num_slots) are skipped and flagged.
 */
int pkv_append_kv(void* k_pool, void* v_pool, int64_t num_slots,
                  const void* k, const void* v, const int32_t* slot_mapping,
                  int64_t n_tokens, int32_t n_kv_heads, int32_t head_dim,
                  int32_t dtype, int32_t* status_word, void* stream);

/*
 * KV append with the position rotation on the way — no counterpart in the
 * reference, whose models rotate q and k before append_kv. Row t of q is
 * rotated into row t of q_out, row t of k is rotated into row slot_mapping[t]
 * of the K pool, row t of v copied into that row of the V pool. q, k and v
 * have heads of head_dim consecutive elements, one head after another, and
 * rows q_stride / k_stride / v_stride elements apart (slices of one
 * projection's output); q_out is contiguous. Of each head the first rotary_dim
 * elements (even, at most head_dim) form pairs, (i, i + rotary_dim / 2) or,
 * with interleaved != 0, (2 i, 2 i + 1); pair i of a token at position p =
 * positions[t] becomes (a c - b s, b c + a s) with c = table[p][0][i], s =
 * table[p][1][i] of the float [max_positions][2][rotary_dim / 2] table, in 32
 * bits with one rounding to the pool dtype. Slots outside [0, num_slots) are
 * skipped and flagged; positions outside [0, max_positions) are flagged, write
 * no row and get a zero row of q_out. No two tokens may share a slot, and
 * q_out may not overlap the inputs.
 */
int pkv_append_rotated(void* k_pool, void* v_pool, int64_t num_slots, const void* q,
                       int64_t q_stride, void* q_out, const void* k, int64_t k_stride,
                       const void* v, int64_t v_stride, const int32_t* slot_mapping,
                       const int64_t* positions, int64_t n_tokens, const float* table,
                       int64_t max_positions, int32_t rotary_dim, int32_t interleaved,
                       int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                       int32_t* status_word, void* stream);

/*
 * pkv_append_rotated with the arguments that do not change from layer to layer
 * set once, and, where n_complete is not 0, pkv_page_bounds of the pages
 * `complete` that these rows complete, in the layer whose bounds lo and hi are.
 */
typedef struct pkv_rotated {
  int64_t num_blocks, n_tokens, max_positions, n_complete;
  const int32_t* slot_mapping;
  const int64_t* positions;
  const float* table;
  const int32_t* complete;
  int32_t* status_word;
  int32_t n_heads, n_kv_heads, head_dim, page_size, dtype, rotary_dim, interleaved, reserved;
} pkv_rotated;

int pkv_append_rotated_batch(const void* batch, void* k_pool, void* v_pool, const void* q,
                             int64_t q_stride, void* q_out, const void* k, int64_t k_stride,
                             const void* v, int64_t v_stride, void* lo, void* hi, void* stream);

/*
 * Decode plan (host function, synchronous, no device access) — the
 * counterpart of the reference fast path's plan step
 * (serving/backends/flashinfer_backend.py:566-676), computed once per batch
 * and reused by every layer. Checks that every sequence has
 * ceil(kv_len / page_size) pages and that kv_last_page_len agrees
 * (PKV_ERR_INVALID, message naming kv_last_page_len, as
 * serving/backends/paged_torch.py:379-392 does).
 *
 * Each sequence of np pages is cut into pieces of part_pages pages, the
 * remainder last, a remainder shorter than both 4 pages and half a piece
 * joining the piece before it (a function of its own length only: at most
 * ceil(np / part_pages) pieces of at most part_pages + 3 pages); the pieces
 * are
 * dealt longest first to the least-loaded of at most
 * max_workgroups / (n_kv_heads / heads-per-workgroup) bins. The plan is
 * bins blocks of *plan_stride_out ints: {n_items, n_pages, 0, 0}, n_pages
 * page words (kv_indices entries, with the page's live row count - 1 in bits
 * 27..30 and an out-of-range flag in bit 31), and n_items items {seq,
 * n_pages, first token, kv_len, partial slot (-1: a whole sequence), pieces
 * of the sequence, its first slot, flags (bit 0: the piece holds the
 * sequence's last page; from bit 1: the sequence's row of q, out, k_new, v_new
 * and slot_mapping, its index as planned -- a caller whose batch is part of
 * a larger one may set it to a row of the larger one's arrays)} at the end of
 * the block, item i at 8 (i + 1) ints before the next block -- pieces of cut sequences before their last, whole
 * sequences, then the last pieces; then 64 zero ints. *plan_stride_out is at
 * least 68, and a multiple of 8 if every bin holds one item, 4 more than one
 * otherwise: by it (and the sizes) a launch picks the kernel for few pieces or
 * the one that streams bins. Either serves any plan, with the same bits.
 * *plan_needed (if not NULL) receives the ints required; a plan larger than
 * plan_capacity returns PKV_ERR_CAPACITY and writes nothing else.
 * *n_work_out is the grid size (workgroups), *n_slots_out the partial slots
 * (workspace size). num_blocks must not exceed 2^27.
 */
int pkv_plan_decode(const int32_t* kv_indptr, const int32_t* kv_indices,
                    const int32_t* kv_lens, const int32_t* kv_last_page_len,
                    int32_t n_seqs, int32_t page_size, int64_t num_blocks,
                    int32_t n_kv_heads, int32_t part_pages, int32_t max_workgroups,
                    int32_t* plan, int64_t plan_capacity, int64_t* plan_needed,
                    int32_t* n_work_out, int32_t* n_slots_out, int32_t* plan_stride_out);

/*
 * Workgroups a decode plan should be dealt into on the current device: the
 * device's compute units times the fast decode kernel's resident workgroups
 * per compute unit for this geometry, capped at per_cu. 0 if the geometry has
 * no fast kernel (or no device is current). No reference counterpart: it is
 * the grid-size half of the plan step FlashInfer's plan performs internally
 * (serving/backends/flashinfer_backend.py:658-670).
 */
int pkv_decode_workgroups(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                          int32_t dtype, int32_t per_cu);

/*
 * Bytes of workspace pkv_attend_decode needs: arrival counters for
 * n_seqs * n_kv_heads (zero before the first launch that uses the workspace;
 * every launch leaves them zero) then n_slots partial results. 0 when
 * n_slots is 0 (no sequence is cut; no workspace is read).
 */
int64_t pkv_decode_workspace_bytes(int32_t n_seqs, int32_t n_slots, int32_t n_heads,
                                   int32_t n_kv_heads, int32_t head_dim);

/*
 * 1 if pkv_attend_decode runs its fast kernel for this geometry (and so
 * accepts a fused append), 0 if it falls back to the generic kernel.
 */
int pkv_decode_fast_path(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                         int32_t page_size, int32_t dtype, int32_t part_pages);

/*
 * Paged decode attention — replaces PagedTorchBackend.attend
 * (serving/backends/paged_torch.py:280-485) and FlashInfer's decode wrapper
 * run (serving/backends/flashinfer_backend.py:556-562, planned at :658-670)
 * for batches where every sequence contributes exactly one query token
 * (token i belongs to sequence i). q, out: [n_seqs, n_heads, head_dim];
 * query head h reads KV head h / (n_heads / n_kv_heads); no mask (the
 * single query is the last position). `plan` is the device copy of
 * pkv_plan_decode's output, with its n_work, n_slots and plan_stride. Cut
 * sequences merge inside the launch through `workspace` (256-byte aligned,
 * pkv_decode_workspace_bytes long); launches that share a workspace must not
 * overlap in time (same stream is fine).
 *
 * Fused append: if k_new / v_new ([n_seqs, n_kv_heads, head_dim]) and
 * slot_mapping ([n_seqs]) are given, the launch also performs pkv_append_kv
 * of those rows, with the same result as the two calls in sequence (fast
 * path only). Pass NULL for all three otherwise.
 *
 * Geometries outside the fast kernel (head_dim not 64/128, more than 16
 * query heads per KV head, page_size != 16, fp32) read kv_indptr /
 * kv_indices / kv_lens instead of the plan: fp32 at head_dim 64/128 and
 * page_size 16 on its own matrix-core kernel, the rest on the generic one.
 */
int pkv_attend_decode(const void* q, void* out,
                      void* k_pool, void* v_pool, int64_t num_blocks,
                      const int32_t* kv_indptr, const int32_t* kv_indices,
                      const int32_t* kv_lens, int32_t n_seqs,
                      int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                      int32_t page_size, float scale, int32_t dtype,
                      const int32_t* plan, int32_t n_work, int32_t n_slots,
                      int32_t plan_stride,
                      const void* k_new, const void* v_new, const int32_t* slot_mapping,
                      void* workspace, int64_t workspace_bytes,
                      int32_t* status_word, void* stream);

/*
 * No-allocation decode — no counterpart in the reference. For callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc): the same launch as
 * pkv_attend_decode, same arguments without the workspace. The split-K
 * workspace is a file-scope device array of PKV_DECODE_SCRATCH_BYTES on each
 * GPU the library runs on (held until the process ends); a plan whose
 * pkv_decode_workspace_bytes exceeds it is rejected with PKV_ERR_CAPACITY.
 * Allocates nothing: no hipMalloc, hipFree or allocating library call. The
 * arrival counters are cleared by a fill kernel on `stream` before each launch.
 * Every call on one GPU shares that GPU's array, so calls that overlap in
 * time on one GPU (different streams, or threads) race; calls in order on one
 * stream do not.
 */
#define PKV_DECODE_SCRATCH_BYTES (64LL * 1024 * 1024)

int pkv_attend_decode_noalloc(const void* q, void* out,
                              void* k_pool, void* v_pool, int64_t num_blocks,
                              const int32_t* kv_indptr, const int32_t* kv_indices,
                              const int32_t* kv_lens, int32_t n_seqs,
                              int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                              int32_t page_size, float scale, int32_t dtype,
                              const int32_t* plan, int32_t n_work, int32_t n_slots,
                              int32_t plan_stride,
                              const void* k_new, const void* v_new, const int32_t* slot_mapping,
                              int32_t* status_word, void* stream);

/*
 * Prefill plan (host function) — tiles each sequence's query rows for
 * pkv_attend_prefill. Output `plan` = n_tiles items {seq, q_start, q_len,
 * 0}, ordered by descending work.
 */
int pkv_plan_prefill(const int32_t* cu_query_lens, const int32_t* kv_indptr,
                     const int32_t* kv_lens, const int32_t* kv_last_page_len,
                     int32_t n_seqs, int32_t page_size, int32_t q_tile,
                     int32_t* plan, int64_t plan_capacity, int32_t* n_tiles_out);

/*
 * Query tile (tokens per plan tile) for which pkv_attend_prefill runs its
 * matrix-core kernel on this geometry: 128 / (n_heads / n_kv_heads), so a
 * tile is 128 query rows of one KV head; for fp32, 32 / (n_heads /
 * n_kv_heads), at least 1 (its kernel takes any q_tile, this one without
 * idle workgroups). 0 if the geometry has no such kernel (any q_tile then
 * runs the generic kernel). Counterpart of the
 * tile choice inside FlashInfer's prefill plan
 * (serving/backends/flashinfer_backend.py:635-649).
 */
int pkv_prefill_q_tile(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                       int32_t page_size, int32_t dtype);

/*
 * Paged attention for arbitrary per-sequence query lengths (chunked prefill,
 * mixed prefill+decode) — replaces PagedTorchBackend.attend
 * (serving/backends/paged_torch.py:280-485) and FlashInfer's prefill wrapper
 * run (serving/backends/flashinfer_backend.py:556-562, planned with
 * causal=True at :635-649). Query j of sequence i (q_len_i queries,
 * kv_len_i keys) attends keys [0, kv_len_i - q_len_i + j] (bottom-right
 * causal). q, out: [n_tokens, n_heads, head_dim]. `batch_indices` maps each
 * token to its sequence. `plan` is the device copy of pkv_plan_prefill's
 * output (q_tile must match the one given to the plan). The matrix-core
 * kernel runs when q_tile == pkv_prefill_q_tile(...) != 0 (fp32: any q_tile,
 * with 16-byte aligned q, out and pools); otherwise the generic kernel runs
 * (it reads cu_query_lens / batch_indices, not the plan; fp32 without a plan
 * too).
 */
int pkv_attend_prefill(const void* q, void* out,
                       const void* k_pool, const void* v_pool, int64_t num_blocks,
                       const int32_t* cu_query_lens, const int32_t* kv_indptr,
                       const int32_t* kv_indices, const int32_t* kv_lens,
                       const int32_t* batch_indices,
                       int32_t n_seqs, int32_t n_tokens,
                       int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                       int32_t page_size, float scale, int32_t dtype,
                       const int32_t* plan, int32_t n_tiles, int32_t q_tile,
                       int32_t* status_word, void* stream);

/*
 * pkv_attend_prefill over the chunks of a mixed batch and pkv_attend_decode
 * over its one-token sequences, with the same result as the two calls: one
 * launch where neither fills the chip. prefill_plan covers the multi-token
 * sequences only; decode_plan is pkv_plan_decode's output over the n_decodes
 * one-token sequences, its items' rows set to their token rows of q and out.
 * With n_decodes > 0 the geometry must have the fast decode path
 * (pkv_decode_fast_path; else PKV_ERR_INVALID, nothing launched: run such a
 * batch whole through pkv_attend_prefill) and q be 16-byte aligned.
 * No reference counterpart: the reference attends a mixed batch sequence by
 * sequence (serving/backends/paged_torch.py:280-485).
 */
int pkv_attend_mixed(const void* q, void* out, void* k_pool, void* v_pool, int64_t num_blocks,
                     const int32_t* cu_query_lens, const int32_t* kv_indptr,
                     const int32_t* kv_indices, const int32_t* kv_lens,
                     const int32_t* batch_indices, int32_t n_seqs, int32_t n_tokens,
                     int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t page_size,
                     float scale, int32_t dtype, const int32_t* prefill_plan, int32_t n_tiles,
                     int32_t q_tile, const int32_t* decode_plan, int32_t n_decodes,
                     int32_t n_work, int32_t n_slots, int32_t plan_stride, void* workspace,
                     int64_t workspace_bytes, int32_t* status_word, void* stream);

/*
 * A batch's arguments that do not change from layer to layer, set once per
 * step, and the two calls of a layer that read them: the same work as
 * pkv_append_kv of the batch's n_tokens rows, and as pkv_attend_decode
 * (is_prefill 0; k_new and v_new may be NULL), pkv_attend_prefill (n_decodes 0)
 * or pkv_attend_mixed, at a third of the arguments a launch. The struct is
 * read on the host before the call returns. No reference counterpart.
 */
typedef struct pkv_batch {
  int64_t num_blocks;
  const int32_t* cu_query_lens;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_lens;
  const int32_t* batch_indices;
  const int32_t* slot_mapping;
  const int32_t* prefill_plan;
  const int32_t* decode_plan;
  void* workspace;
  int64_t workspace_bytes;
  int32_t* status_word;
  int32_t n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, page_size, dtype, is_prefill;
  int32_t n_tiles, q_tile, n_decodes, n_work, n_slots, plan_stride;
} pkv_batch;

int pkv_append_batch(const void* batch, void* k_pool, void* v_pool, const void* k,
                     const void* v, void* stream);
int pkv_attend_batch(const void* batch, const void* q, void* out, void* k_pool, void* v_pool,
                     float scale, const void* k_new, const void* v_new, void* stream);

/*
 * Shared-prefix plan (host function) — no counterpart in the reference, whose
 * radix cache shares pages but whose attention reads them once a sequence.
 * Page lists that begin with the same ids form a tree; each of its runs of at
 * least min_pages pages with n >= 2 sequences below it that saves more bytes a
 * KV head ((n - 1) * pages * page_bytes, page_bytes a page's of a KV head) than
 * it costs (n * part_bytes, a part more for each sequence) becomes tiles of
 * pkv_attend_shared, 128 / (n_heads / n_kv_heads) sequences and a split of the
 * run each, splits sized for about tile_target workgroups. A sequence's last
 * page is never shared. `plan` is pkv_plan_decode's over the remaining pages
 * (arguments and outputs as there), with each sequence's shared parts counted
 * among its pieces and given its first partial slots. `tiles` receives
 * *n_tiles_out items {index of the first page in kv_indices, pages, first
 * member, members, split, 0, 0, 0}, *n_merges_out merges {sequence, parts,
 * first partial slot, 0} of the sequences with shared parts, then the members
 * {row of q, partial slot of split 0}; *tiles_needed ints in all. A buffer too small
 * gives PKV_ERR_CAPACITY with the needed sizes set (tiles_needed once plan
 * suffices). Where all runs together save less than least_bytes over the KV
 * heads nothing is shared: *n_tiles_out is 0 and no plan is written.
 */
int pkv_plan_shared(const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_lens,
                    const int32_t* kv_last_page_len, int32_t n_seqs, int32_t page_size,
                    int64_t num_blocks, int32_t n_heads, int32_t n_kv_heads, int32_t part_pages,
                    int32_t max_workgroups, int32_t min_pages, int64_t page_bytes,
                    int64_t part_bytes, int64_t least_bytes, int32_t tile_target, int32_t* plan,
                    int64_t plan_capacity, int64_t* plan_needed, int32_t* n_work_out,
                    int32_t* n_slots_out, int32_t* plan_stride_out, int32_t* tiles,
                    int64_t tiles_capacity, int64_t* tiles_needed, int32_t* n_tiles_out,
                    int32_t* n_merges_out);

/*
 * pkv_attend_decode with pkv_plan_shared's tiles and plan (device copies): the
 * same result up to rounding, with each shared run of pages read once per tile
 * of sequences. kv_indices is the device copy of the planned one; workspace
 * and fused append as for pkv_attend_decode (no shared page may be a slot's of
 * slot_mapping). Needs at least one tile, the fast decode path and a positive
 * scale (PKV_ERR_INVALID otherwise, nothing launched).
 */
int pkv_attend_shared(const void* q, void* out, void* k_pool, void* v_pool, int64_t num_blocks,
                      const int32_t* kv_indices, int32_t n_seqs, int32_t n_heads,
                      int32_t n_kv_heads, int32_t head_dim, int32_t page_size, float scale,
                      int32_t dtype, const int32_t* tiles, int32_t n_tiles, int32_t n_merges,
                      const int32_t* plan, int32_t n_work, int32_t n_slots, int32_t plan_stride,
                      const void* k_new, const void* v_new, const int32_t* slot_mapping,
                      void* workspace, int64_t workspace_bytes, int32_t* status_word,
                      void* stream);

/*
 * pkv_attend_shared with the arguments that do not change from layer to layer
 * set once.
 */
typedef struct pkv_shared {
  int64_t num_blocks, workspace_bytes;
  const int32_t* kv_indices;
  const int32_t* tiles;
  const int32_t* plan;
  const int32_t* slot_mapping;
  void* workspace;
  int32_t* status_word;
  int32_t n_seqs, n_heads, n_kv_heads, head_dim, page_size, dtype;
  int32_t n_tiles, n_merges, n_work, n_slots, plan_stride, reserved;
} pkv_shared;

int pkv_attend_shared_batch(const void* batch, const void* q, void* out, void* k_pool,
                            void* v_pool, float scale, const void* k_new, const void* v_new,
                            void* stream);

/*
 * Key bounds of pages — no counterpart in the reference. For each of the
 * n_ids pages of ids (NULL: pages 0 .. n_ids - 1) and each of n_layers layers,
 * row id of lo and hi ([num_blocks, n_kv_heads, head_dim], the pool dtype)
 * receives the elementwise minimum and maximum of the page's page_size key
 * rows; a NaN among them gives NaN. Layer l's K plane, lo and hi start
 * l * pool_step and l * bounds_step bytes from the given ones. Ids outside
 * [0, num_blocks) are skipped and flagged; equal ids are harmless.
 */
int pkv_page_bounds(const void* k_pool, int64_t pool_step, void* lo, void* hi,
                    int64_t bounds_step, int32_t n_layers, int64_t num_blocks,
                    const int32_t* ids, int64_t n_ids, int32_t n_kv_heads, int32_t head_dim,
                    int32_t page_size, int32_t dtype, int32_t* status_word, void* stream);

/*
 * Choice of pages for a batch of one-token sequences — no counterpart in the
 * reference. A sequence of np pages gets, per KV head, all of them if np <=
 * pages; else its last page and the pages - 1 of the others with the largest
 * score, the largest over the KV head's query heads of sum_d q_d * (q_d < 0 ?
 * lo_d : hi_d) in 64 bits (equal scores: the lower index; a NaN beats every
 * number). lo and hi are one layer's bounds (pkv_page_bounds). ids and
 * ordinals, int32 [n_seqs, n_kv_heads, min(pages, max_pages)], receive the
 * chosen pages' kv_indices entries and indices in the sequence's page list, in
 * ascending order, -1 behind shorter lists. max_pages is at least every
 * sequence's page count; scores holds n_seqs * n_kv_heads * max_pages doubles
 * (NULL if max_pages <= pages). Out-of-range page ids are scored by page 0's
 * bounds and flagged. With `words` the chosen pages go there instead of ids, as
 * page words of pkv_plan_selected's plan (its places, part_pages, and head_words
 * its size), KV head h's at words + h * head_words.
 */
int pkv_select_pages(const void* q, const void* lo, const void* hi, int64_t num_blocks,
                     const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_lens,
                     int32_t n_seqs, int32_t max_pages, int32_t pages, int32_t n_heads,
                     int32_t n_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype,
                     double* scores, int32_t* ids, int32_t* ordinals, int32_t* words,
                     const int32_t* places, int64_t head_words, int32_t part_pages,
                     int32_t* status_word, void* stream);

/*
 * Plan over chosen pages (host function), for batches whose pieces fill the
 * device: pkv_plan_decode's over lists of min(pages, pages of the sequence)
 * pages, whose page words pkv_select_pages fills in on the device, and
 * `places`, where each list's words go: {first piece, pieces} a sequence, then
 * the position of each piece's first word. Needs the fast decode path.
 */
int pkv_plan_selected(const int32_t* kv_lens, int32_t n_seqs, int32_t pages, int32_t n_heads,
                      int32_t n_kv_heads, int32_t head_dim, int32_t dtype, int32_t part_pages,
                      int32_t max_workgroups, int32_t* plan, int64_t plan_capacity,
                      int64_t* plan_needed, int32_t* n_work_out, int32_t* n_slots_out,
                      int32_t* plan_stride_out, int32_t* places, int64_t places_capacity,
                      int64_t* places_needed);

/*
 * Decode attention over the pages pkv_select_pages chose (its ids, n_seqs,
 * max_pages and pages): sequence i's single query attends the rows of its
 * chosen pages, of the last one those below kv_lens[i]. Lists are cut into
 * pieces of part_pages pages (8 is what the kernel stages at a time), the
 * remainder last, and cut ones merge through `workspace` (256-byte aligned, pkv_selected_workspace_bytes
 * long; zero before the first launch that uses it, and left with zero
 * counters by each; launches that share it must not overlap in time).
 * Geometries without the fast decode path run a generic kernel, with no
 * workspace. With a plan (pkv_plan_selected's, its words filled by
 * pkv_select_pages) the streaming decode kernel runs it, with the workspace of
 * pkv_decode_workspace_bytes for its n_slots; ids and part_pages are not read.
 */
int64_t pkv_selected_workspace_bytes(int32_t n_seqs, int32_t max_pages, int32_t pages,
                                     int32_t part_pages, int32_t n_heads, int32_t n_kv_heads,
                                     int32_t head_dim, int32_t page_size, int64_t num_blocks,
                                     int32_t dtype);
int pkv_attend_selected(const void* q, void* out, void* k_pool, void* v_pool, int64_t num_blocks,
                        const int32_t* ids, const int32_t* kv_lens, int32_t n_seqs,
                        int32_t max_pages, int32_t pages, int32_t part_pages, int32_t n_heads,
                        int32_t n_kv_heads, int32_t head_dim, int32_t page_size, float scale,
                        int32_t dtype, const int32_t* plan, int32_t n_work, int32_t n_slots,
                        int32_t plan_stride, const int32_t* words, int64_t head_words,
                        void* workspace, int64_t workspace_bytes, int32_t* status_word,
                        void* stream);

/*
 * pkv_select_pages and pkv_attend_selected of one layer, with the arguments
 * that do not change from layer to layer set once. lo and hi are the layer's
 * bounds.
 */
typedef struct pkv_selected {
  int64_t num_blocks, workspace_bytes, head_words;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_lens;
  double* scores;
  int32_t* ids;
  int32_t* words;
  const int32_t* places;
  const int32_t* plan;
  void* workspace;
  int32_t* status_word;
  int32_t n_seqs, max_pages, pages, part_pages;
  int32_t n_heads, n_kv_heads, head_dim, page_size, dtype;
  int32_t n_work, n_slots, plan_stride;
} pkv_selected;

int pkv_attend_selected_batch(const void* batch, const void* q, void* out, void* k_pool,
                              void* v_pool, const void* lo, const void* hi, int32_t* ordinals,
                              float scale, void* stream);

/*
 * The 4-bit cache — no counterpart in the reference. A block's K (or V) is
 * pkv_block_bytes_4bit bytes (0 for a geometry that has none: odd head_dim or
 * above 256), laid out as csrc/fourbit.h says; a pool is a contiguous array of
 * num_blocks of them, which pkv_copy_blocks, pkv_gather_blocks and
 * pkv_scatter_blocks move like any other. A row of a KV head is cut into groups
 * of 64 elements (one group where head_dim is no multiple of 64); a group keeps
 * a float16 zero, a float16 step and 4-bit codes, and reads as zero + step c.
 *
 * pkv_append_4bit: for t < n_tokens, row t of k / v (heads one after another,
 * rows k_stride / v_stride elements apart, f16, bf16 or f32) goes to slot
 * slot_mapping[t]. Slots outside the pool are skipped and flagged. No two tokens
 * may share a slot.
 *
 * pkv_read_4bit: row i of k / v (contiguous [n_rows, n_kv_heads, head_dim])
 * receives what slot slots[i] holds, rounded to dtype once; zeros (and the flag)
 * for slots outside the pool.
 */
int64_t pkv_block_bytes_4bit(int32_t n_kv_heads, int32_t head_dim, int32_t page_size);
int pkv_append_4bit(void* k_pool, void* v_pool, int64_t num_blocks, const void* k,
                    int64_t k_stride, const void* v, int64_t v_stride,
                    const int32_t* slot_mapping, int64_t n_tokens, int32_t n_kv_heads,
                    int32_t head_dim, int32_t page_size, int32_t dtype, int32_t* status_word,
                    void* stream);
int pkv_read_4bit(const void* k_pool, const void* v_pool, int64_t num_blocks,
                  const int32_t* slots, int64_t n_rows, void* k, void* v, int32_t n_kv_heads,
                  int32_t head_dim, int32_t page_size, int32_t dtype, int32_t* status_word,
                  void* stream);

/*
 * Causal attention over the 4-bit cache, any query lengths: sequence i's query
 * tokens are the last of its kv_lens[i] tokens. q and out are contiguous
 * [n_tokens, n_heads, head_dim] in dtype; a batch's arguments are set once and
 * serve every layer.
 *
 * pkv_plan_4bit (host, synchronous) checks the metadata as pkv_plan_decode does (a
 * kv_len is at most 2^31 - 129)
 * and fills items (capacity ints; *needed of them, PKV_ERR_CAPACITY if there are
 * fewer) with pieces of 28 ints {first token's row in q, tokens, its position,
 * kv_len, first page in kv_indices, pages, first tile of 64 keys, tiles, partial
 * slot or -1, the first piece's slot, pieces, arrival counter, the pages of the
 * first 256 keys' 16 units}, n_few those of sequences with
 * at most 16 query rows (tokens x query heads a KV head), n_wide of 32 rows, n_tall
 * of 128, and the plan
 * fields of *plan; long rows are cut to fill compute_units compute units. Geometries without a matrix-core kernel (head_dim
 * other than 64 and 128, f32, pages that are no power of two times 16, more than
 * 32 query heads a KV head, 256 KV heads) need no items.
 *
 * `workspace` (256-byte aligned, workspace_bytes long): arrival counters, zero
 * before the first launch and left so by each (pkv_counter_bytes_4bit from the
 * front), then the partial results; launches that share it must not overlap in time. Page ids
 * outside [0, num_blocks) read as zeros and are flagged.
 */
typedef struct pkv_4bit {
  int64_t num_blocks, workspace_bytes;
  const int32_t* cu_query_lens;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_lens;
  const int32_t* batch_indices;
  const int32_t* items;
  void* workspace;
  int32_t* status_word;
  int32_t n_seqs, n_tokens, n_heads, n_kv_heads, head_dim, page_size, dtype;
  int32_t n_few, n_wide, n_tall, few_rows, few_waves, part_rows, n_slots, n_cuts;   /* the plan's */
} pkv_4bit;

int pkv_plan_4bit(const int32_t* cu_query_lens, const int32_t* kv_indptr,
                  const int32_t* kv_indices, const int32_t* kv_lens,
                  const int32_t* kv_last_page_len, int32_t n_seqs, int32_t n_heads,
                  int32_t n_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype,
                  int32_t compute_units, int32_t* items, int64_t capacity, int64_t* needed,
                  pkv_4bit* plan);
int64_t pkv_counter_bytes_4bit(int32_t n_cuts, int32_t n_kv_heads);
int pkv_attend_4bit(const void* batch, const void* q, void* out, const void* k_pool,
                    const void* v_pool, float scale, void* stream);

/*
 * Batched block copy over every layer, K and V — replaces
 * PagedTorchBackend.copy_block (serving/backends/paged_torch.py:181-207),
 * called once per pair by RadixCache.ensure_writable
 * (serving/cache/radix.py:672-674). For each pair p, block dst[p] of every
 * plane becomes a copy of block src[p]. All sources are read before any
 * destination is written only if no dst appears among the srcs; the caller
 * guarantees that (and that dsts are distinct). Ids outside
 * [0, num_blocks) are skipped and flagged.
 */
int pkv_copy_blocks(void* pool_base, int32_t n_layers, int64_t plane_bytes,
                    int64_t block_bytes, int64_t num_blocks,
                    const int32_t* src, const int32_t* dst, int32_t n_pairs,
                    int32_t* status_word, void* stream);

/*
 * Metadata upload — replaces the host-to-device tensor builds of
 * build_batch_meta (serving/engine_iface/batch.py:246-318; one pinned buffer
 * per step here): `bytes` bytes of the pinned host buffer `host` (allocated
 * pinned, hence mapped for the device) are copied to device memory `dst` by
 * a kernel on `stream` that reads the buffer through its device mapping, so
 * the copy is ordered on the launch stream like the kernels that read it,
 * with no copy-engine hand-off. `host` must stay unchanged until the copy
 * has run (the caller records an event after it). PKV_ERR_INVALID if `host`
 * is not pinned memory mapped for the device.
 */
int pkv_upload_pinned(void* dst, const void* host, int64_t bytes, void* stream);

/*
 * Swap-out gather — the device half of KVSwapSpace._to_host
 * (serving/scheduler/preemption.py:490-509): staging[kv][layer][i] = block
 * ids[i] of plane (layer, kv), i.e. staging is [2][n_layers][n_ids][block]
 * (K half first), the reference's SwapHandle.k / .v layout
 * (serving/scheduler/preemption.py:303-332). `staging` may be device memory
 * or pinned host memory mapped for the device.
 */
int pkv_gather_blocks(const void* pool_base, int32_t n_layers, int64_t plane_bytes,
                      int64_t block_bytes, int64_t num_blocks,
                      const int32_t* ids, int32_t n_ids, void* staging,
                      int32_t* status_word, void* stream);

/*
 * Swap-in scatter — the device half of KVSwapSpace._from_host
 * (serving/scheduler/preemption.py:511-523): the inverse of
 * pkv_gather_blocks; block ids[i] of plane (layer, kv) receives
 * staging[kv][layer][i]. ids must be distinct.
 */
int pkv_scatter_blocks(void* pool_base, int32_t n_layers, int64_t plane_bytes,
                       int64_t block_bytes, int64_t num_blocks,
                       const int32_t* ids, int32_t n_ids, const void* staging,
                       int32_t* status_word, void* stream);

/*
 * Greedy sampling — the scheduler's torch.argmax(logits, dim=-1)
 * (serving/scheduler/scheduler.py:752-757) on the device: out_ids[r] = the
 * index of the largest of the `vocab` logits of row r (row r starts at
 * element r * row_stride), with torch's order: a NaN beats every number
 * and between equal values the smaller index wins. logits are f16, bf16 or
 * f32 (dtype); out_ids is a device int64 array of n_rows entries. n_rows = 0
 * does nothing.
 */
int pkv_argmax_rows(const void* logits, int64_t n_rows, int64_t vocab, int64_t row_stride,
                    int32_t dtype, int64_t* out_ids, void* stream);

/*
 * Verification of drafted tokens — no counterpart in the reference, which
 * decodes greedily. Rows of logits (row r at element r * row_stride) belong to
 * n_seqs sequences, rows cu_query_lens[i] .. cu_query_lens[i + 1] to sequence i
 * (batch_indices[r]: row r's sequence); tokens[r] is the token that row r
 * follows, so those behind a sequence's first are its drafts. Draft j, x =
 * tokens[r + 1] at its row r = cu_query_lens[i] + j, stands if numbers[r] *
 * q(x) < p(x): p the softmax of row r's logits / temperature, q row r - i of
 * draft_probs ([n_rows - n_seqs, vocab], row stride probs_stride; NULL: 1 at x).
 * accepted[i] is how many stand before the first that does not; ids[i] (width
 * entries, at least a sequence's rows) holds them, one more token, and -1. The
 * one more is drawn from max(p - q, 0) at the first row whose draft falls (p
 * without x where draft_probs is NULL; p itself where nothing is left), or from
 * the last row's p: the first token whose running sum of weights exceeds the
 * last row's number times their sum. All of it as in 64 bits; weights below
 * 2^-1000 of a row's largest count as 0. At temperatures of 0 or below a draft
 * stands if it is the row's pkv_argmax_rows id, which is the token otherwise. In
 * a row without a distribution (a NaN, +inf, or nothing but -inf) no draft
 * stands, and that id is taken; a draft outside [0, vocab) does not stand.
 * temperatures: one a sequence, or NULL: `temperature` for all; one above the
 * largest finite float (and +inf) counts as that. `workspace`:
 * pkv_verify_workspace_bytes, aligned to 16, in any state; calls that overlap in
 * time need one each.
 */
int64_t pkv_verify_workspace_bytes(int64_t n_rows, int64_t n_seqs, int64_t vocab, int32_t dtype);
int pkv_verify_drafts(const void* logits, int64_t n_rows, int64_t vocab, int64_t row_stride,
                      int32_t dtype, const int64_t* tokens, const int32_t* cu_query_lens,
                      const int32_t* batch_indices, int64_t n_seqs, const float* numbers,
                      const void* draft_probs, int64_t probs_stride, int32_t probs_dtype,
                      const float* temperatures, float temperature, int64_t* ids, int64_t width,
                      int64_t* accepted, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PAGEDKV_H */

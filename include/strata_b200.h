/*
 * strata_b200.h — what libstrata_b200.so adds on top of strata_plugin.h.
 *
 * 1. A vendor extension on the plugin's extension chain
 *    (StrataPluginV1::extension_start, raw.rs:51-85).  The reference's ABI 0.1
 *    allocates a buffer per value per run and copies host bytes in and out
 *    (crates/ferrite-strata-plugin-api/src/host/plugin.rs:382-534); that path
 *    is kept unchanged.  The extension lets a host keep buffers resident on
 *    the device across runs (weights, KV caches), wrap device memory it
 *    already owns, enqueue a run without blocking, and join a tensor-parallel
 *    group.  A host that does not know the extension type skips it
 *    (loader.rs:279-316), so ABI 0.1 hosts are unaffected.
 *
 * 2. Kernel-level entry points with plain device pointers, used by the
 *    plugin's own executor and callable directly (for example from ctypes)
 *    to check one kernel in isolation.  Pointers are device pointers; `stream`
 *    is a cudaStream_t passed as void* (null = the legacy default stream).
 *    Every entry point returns 0 on success and a negative STRATA_* status on
 *    a rejected argument or a launch failure; kernels are asynchronous.
 *
 * bf16 tensors are passed as uint16_t bit patterns.
 */
#ifndef STRATA_B200_H
#define STRATA_B200_H

#include "strata_plugin.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------ */
/* Extension on the plugin's chain                                          */
/* ------------------------------------------------------------------------ */

/* Vendor-chosen tag ("B2DV"), outside the ABI's own 0..2 range. */
#define STRATA_B200_EXT_DEVICE 0x56443242u
#define STRATA_B200_EXT_DEVICE_VERSION 1u

typedef struct StrataB200DeviceExt {
  StrataExtBase base; /* ty == STRATA_B200_EXT_DEVICE */
  uint32_t version;   /* STRATA_B200_EXT_DEVICE_VERSION */
  uint32_t reserved;

  /* Wrap `bytes` of device memory the caller owns as a buffer.  The plugin
   * never frees it; buffer_release only drops the handle. */
  int32_t (*buffer_wrap)(void *ctx, void *device_ptr, uint64_t bytes,
                         StrataBuffer **out_buffer);
  /* The device address and byte size behind a buffer. */
  int32_t (*buffer_device_ptr)(void *ctx, const StrataBuffer *buffer,
                               void **out_ptr, uint64_t *out_bytes);
  /* Enqueue a run on the plugin's stream and return without waiting.
   * Device-side failures surface at the next synchronize or buffer_read. */
  int32_t (*run_async)(void *ctx, const StrataRunArgs *args,
                       StrataError **out_error);
  /* Wait for everything enqueued, then report any device-side failure. */
  int32_t (*synchronize)(void *ctx, StrataError **out_error);
  /* The cudaStream_t the plugin launches on. */
  void *(*stream)(void *ctx);
  /* Number of kernel launches the plugin has enqueued since load (CUDA-graph
   * replays count every kernel inside the graph). */
  uint64_t (*launch_count)(void *ctx);
  /* Tensor parallelism: rank 0 creates an id (128 bytes), every rank passes
   * it to tp_init with its own rank.  Collective; call before compile. */
  int32_t (*tp_unique_id)(void *ctx, uint8_t out_id[128]);
  int32_t (*tp_init)(void *ctx, int32_t rank, int32_t world_size,
                     const uint8_t id[128], StrataError **out_error);
  /* Select the CUDA device for this context (before any other call). */
  int32_t (*set_device)(void *ctx, int32_t device);
} StrataB200DeviceExt;

/* ------------------------------------------------------------------------ */
/* Step profile                                                             */
/* ------------------------------------------------------------------------ */

/* With STRATA_B200_STEP_TIMES=1 in the environment when the library loads,
 * every run is eager (no CUDA graph) and each of its steps is bracketed by
 * CUDA events on the plugin's stream; the device time accumulates per step
 * class ("gemv:swiglu", "attention", "all_reduce_add_norm", ...).  This
 * writes {"class": [steps, milliseconds], ...} into buf (NUL-terminated when
 * it fits), clears the totals when reset is non-zero, and returns the bytes
 * the JSON needs.  No counterpart in the reference. */
uint64_t strata_b200_step_times(char *buf, uint64_t cap, int32_t reset);

/* ------------------------------------------------------------------------ */
/* Kernel-level entry points                                                */
/* ------------------------------------------------------------------------ */

/* Quantisation, bit-exact with the CPU oracle.  w is f32 [n, k]. */
int32_t strata_b200_quant_w4g32(const float *w, int64_t n, int64_t k,
                                uint8_t *packed, uint16_t *scale_bf16,
                                void *stream);
int32_t strata_b200_quant_w8pc(const float *w, int64_t n, int64_t k,
                               int8_t *q, float *scale, void *stream);
int32_t strata_b200_dequant_w4g32(const uint8_t *packed,
                                  const uint16_t *scale_bf16, int64_t n,
                                  int64_t k, float *w, void *stream);
int32_t strata_b200_dequant_w8pc(const int8_t *q, const float *scale,
                                 int64_t n, int64_t k, float *w, void *stream);

/* y[m, n] = sum_k x[m, k] * deq(W)[n, k]  (+ residual[m, n] when non-null);
 * bf16 in and out, f32 accumulation.  k must be a multiple of 32 (w4g32) or
 * 16 (w8pc). */
int32_t strata_b200_linear_w4g32(const uint16_t *x, int64_t m, int64_t k,
                                 const uint8_t *packed,
                                 const uint16_t *scale_bf16, int64_t n,
                                 const uint16_t *residual, uint16_t *y,
                                 void *stream);
int32_t strata_b200_linear_w8pc(const uint16_t *x, int64_t m, int64_t k,
                                const int8_t *q, const float *scale,
                                int64_t n, const uint16_t *residual,
                                uint16_t *y, void *stream);

/* The same with MX weights (OCP Microscaling; the element types of
 * crates/ferrite-strata/src/dtype.rs:41-85, DType::microscaled): codes E4M3
 * [n, k] one byte each (mxfp8) or E2M1 [n, k] packed two per byte, even k in
 * the low nibble (mxfp4); scales E8M0 [n, k/32], one byte each.  Weights are
 * dequantised exactly (code * 2^(e - 127)).  k % 128 == 0 and n % 16 == 0 for
 * m <= 64 (the tensor-core GEMV). */
int32_t strata_b200_linear_mxfp8(const uint16_t *x, int64_t m, int64_t k,
                                 const uint8_t *codes,
                                 const uint8_t *scale_e8m0, int64_t n,
                                 const uint16_t *residual, uint16_t *y,
                                 void *stream);
int32_t strata_b200_linear_mxfp4(const uint16_t *x, int64_t m, int64_t k,
                                 const uint8_t *codes,
                                 const uint8_t *scale_e8m0, int64_t n,
                                 const uint16_t *residual, uint16_t *y,
                                 void *stream);

/* y[m, n] = sum_k x[m, k] * w[n, k]  (+ residual[m, n] when non-null) with
 * bf16 weights [n, k]: the reference's f32 `linear` (crates/ferrite-strata-cpu/
 * src/backend.rs:607-637) in bf16 storage with f32 accumulation.  k must be a
 * multiple of 8.  Batches of more than 64 rows run on the tcgen05 tensor cores
 * (so do the int4, int8 and MX entry points, after expanding the weights into
 * a bf16 scratch buffer the library keeps per device and stream; a call that
 * needs a larger one than it has allocates it with cudaMalloc, also while the
 * stream is being captured, and the smaller one stays allocated for graphs
 * that name it). */
int32_t strata_b200_linear_bf16(const uint16_t *x, int64_t m, int64_t k,
                                const uint16_t *w, int64_t n,
                                const uint16_t *residual, uint16_t *y,
                                void *stream);

int32_t strata_b200_rms_norm_bf16(const uint16_t *x, const uint16_t *gamma,
                                  int64_t rows, int64_t cols, float eps,
                                  uint16_t *y, void *stream);
int32_t strata_b200_rope_bf16(const uint16_t *x, const int32_t *pos,
                              int64_t rows, int64_t heads, int64_t head_dim,
                              float theta, uint16_t *y, void *stream);
int32_t strata_b200_swiglu_bf16(const uint16_t *gate, const uint16_t *up,
                                int64_t n, uint16_t *y, void *stream);

/* Decode attention.  q [batch, heads*head_dim]; k_new/v_new
 * [batch, kv_heads*head_dim] are written into the caches
 * [batch, kv_heads, max_len, head_dim] at position pos[b], then row b attends
 * to positions 0..pos[b].  `scratch` must hold
 * strata_b200_attention_decode_scratch_bytes(...) bytes. */
uint64_t strata_b200_attention_decode_scratch_bytes(int64_t batch,
                                                    int64_t heads,
                                                    int64_t head_dim,
                                                    int64_t max_len);
int32_t strata_b200_attention_decode_bf16(
    const uint16_t *q, const uint16_t *k_new, const uint16_t *v_new,
    uint16_t *k_cache, uint16_t *v_cache, const int32_t *pos, int64_t batch,
    int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_len,
    void *scratch, uint16_t *out, void *stream);

/* Decode attention that allocates nothing.  No counterpart in the reference:
 * it exists for callers that cannot call cudaMalloc -- for example code running
 * while a stream is captured in a mode that refuses allocation, or a runtime
 * whose device memory is all owned by its own pool.  The split-KV partials go
 * to a scratch area inside the library (a __device__ array of
 * strata_b200_noalloc_scratch_capacity() bytes, 32 MiB, reserved on every GPU
 * that loads the library until the process exits) instead of a caller buffer.
 * Same arguments and results as strata_b200_attention_decode_bf16 otherwise.
 * Returns STRATA_RESOURCE_EXHAUSTED if the shape needs more scratch than the
 * capacity.  The first call on a device looks up the scratch address there;
 * make that first call before any stream capture.  Calls that overlap on the
 * GPU share the scratch and race: serialise them (one stream, or events). */
uint64_t strata_b200_noalloc_scratch_capacity(void);
int32_t strata_b200_attention_decode_bf16_noalloc(
    const uint16_t *q, const uint16_t *k_new, const uint16_t *v_new,
    uint16_t *k_cache, uint16_t *v_cache, const int32_t *pos, int64_t batch,
    int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_len,
    uint16_t *out, void *stream);

int32_t strata_b200_embed_bf16(const int32_t *ids, int64_t rows,
                               const uint16_t *table, int64_t vocab,
                               int64_t dim, uint16_t *out, void *stream);
int32_t strata_b200_argmax_bf16(const uint16_t *x, int64_t rows, int64_t cols,
                                int32_t *out, void *stream);

/* ------------------------------------------------------------------------ */
/* Several continuations of a sequence: drafted trees and beams             */
/* ------------------------------------------------------------------------ */
/* No counterpart in the reference.  Shared conventions:
 *  - Caches are contiguous [batch, kv_heads, max_len, head_dim] when
 *    block_table is null, else page pools [num_pages, kv_heads, page_size,
 *    head_dim] with a block table I32 [batch, max_len / page_size] (page_size a
 *    power of two from 16 to 4096); batch (or pool) * kv_heads * positions is
 *    below 2^31.  No two caches, pools or outputs of a call overlap.
 *  - A workspace is device memory of at least the bytes its *_workspace_bytes
 *    function gives (0 for a shape the entry point refuses), 16-byte aligned,
 *    whose contents do not matter before or after a call.  Two calls that may
 *    overlap on the GPU need two workspaces; so do two CUDA graphs that may be
 *    replayed at once.
 *  - `status` (null, or one I32 on the device) is set when a device-side
 *    input is wrong, and left alone otherwise: 2 a length, position or index
 *    out of range, 6 a block-table entry that names no page of the pool; 4 is a
 *    fault of the library's own (a wait inside a kernel ran out; outputs are then
 *    incomplete).
 *  - Calls allocate nothing and may be captured into a CUDA graph.  Launches
 *    go to the current device, which must be the stream's.  What a call writes
 *    is there for every later call on its stream, without a wait between. */

/* Attention of a tree of drafted tokens over the cached prompt.  q
 * [batch * tokens, heads * head_dim]; k_new, v_new [batch * tokens,
 * kv_heads * head_dim].  Sequence b has base[b] cached positions and count[b]
 * live nodes (null: `tokens` for all).  Node i's k and v are written at position
 * base + i, and node t attends to the positions below base and to the live
 * nodes j whose bit j % 32 of word j / 32 is set in mask [batch, tokens,
 * ceil(tokens / 32)] row t (set a node's own bit to let it see itself).  out
 * [batch * tokens, heads * head_dim]; a node that sees nothing, and rows at or
 * past count, are zeros.  Scores, softmax sums and accumulators are f32; each
 * probability is rounded to bf16 (by at most 2^-8 of it) for its product with v,
 * as in the library's other attention, so an output is within
 * 2^-8 sum_p(w_p |v_p|) + 2^-8 |o| and 32-bit rounding.  A sequence with
 * base < 0, count outside 0..tokens or base + count > max_len gets status 2:
 * zeros, and nothing is appended.  Positions on missing pages get status 6 and
 * read as zero rows.  tokens <= 1024, head_dim 64 or 128, at most 128 query
 * heads per kv head, pointers 16-byte aligned; a call whose 128-position tiles
 * over all sequences and kv heads could pass 2^31 is refused.  Two sequences
 * must not append to the same page. */
uint64_t strata_b200_tree_attention_workspace_bytes(int64_t tokens,
                                                    int64_t heads,
                                                    int64_t kv_heads,
                                                    int64_t head_dim);
int32_t strata_b200_tree_attention_bf16(
    const uint16_t *q, const uint16_t *k_new, const uint16_t *v_new,
    uint16_t *k_cache, uint16_t *v_cache, const int32_t *block_table,
    const int32_t *base, const int32_t *count, const uint32_t *mask,
    int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
    int64_t head_dim, int64_t max_len, int64_t page_size, int64_t num_pages,
    void *workspace, uint16_t *out, int32_t *status, void *stream);

/* A beam step's selection.  logits [batch * beams, vocab]; scores
 * [batch * beams], the beams' accumulated log probabilities (-inf or NaN: an
 * empty beam, which offers nothing); done [batch * beams] (may be null),
 * non-zero for a beam that has ended.  A live beam w offers score + log_softmax(logits)[v] for every v (a NaN
 * logit counts as -inf; +inf logits share their row's probability equally and
 * the others get none); an ended one offers its unchanged score with token
 * eos.  Writes the `keep` best of every batch entry, best first, ties to the
 * lowest w * vocab + v: out_scores, out_parent (the row b * beams + w),
 * out_token and out_done (the parent had ended, or the token is eos), each
 * [batch, keep].  Where no candidate above -inf is left: -inf, -1, -1, 0.
 * eos -1: no token ends a beam (an ended beam's token is then -1).  keep <=
 * 64, beams <= 1024, batch * beams <= 65535, vocab <= 2^30.  Scores are added
 * and compared in f64 and rounded once; the softmax's terms are f32, and the
 * logarithm of their sum is within 2^-20.  Each beam enters with its `keep`
 * largest logits (the lowest ids on ties): where two different logits of a beam
 * are so close beside its score that f64 gives both the same score, the larger
 * logit may be kept and not the lower id. */
uint64_t strata_b200_beam_select_workspace_bytes(int64_t batch, int64_t beams,
                                                 int64_t vocab, int64_t keep);
int32_t strata_b200_beam_select_bf16(
    const uint16_t *logits, const float *scores, const int32_t *done,
    int64_t batch, int64_t beams, int64_t vocab, int64_t keep, int64_t eos,
    float *out_scores, int32_t *out_parent, int32_t *out_token,
    int32_t *out_done, void *workspace, void *stream);
int32_t strata_b200_beam_select_f32(
    const float *logits, const float *scores, const int32_t *done,
    int64_t batch, int64_t beams, int64_t vocab, int64_t keep, int64_t eos,
    float *out_scores, int32_t *out_parent, int32_t *out_token,
    int32_t *out_done, void *workspace, void *stream);

/* Keeps the accepted branch of a drafted tree: in each of n_caches caches or
 * pools (a host array of device pointers, at most 256, 16-byte aligned; rows
 * of row_bytes bytes, a multiple of 16), row base[b] + path[b, i] moves to
 * base[b] + i for i < n_path[b].  path [batch, max_path] is strictly increasing
 * from 0 or more; a sequence whose path is not, or leaves max_len, is left
 * alone (status 2; 6 for a missing page).  max_path <= 1024.  The rows from
 * base on must belong to the sequence alone. */
int32_t strata_b200_kv_accept(
    void *const *caches, int64_t n_caches, int64_t row_bytes,
    const int32_t *block_table, const int32_t *base, const int32_t *path,
    const int32_t *n_path, int64_t batch, int64_t kv_heads, int64_t max_len,
    int64_t max_path, int64_t page_size, int64_t num_pages, int32_t *status,
    void *stream);

/* Gives every row of a block table a new parent: row r continues old row
 * parents[r] (-1: becomes empty) with its length.  Pools are page pools as
 * above with rows of row_bytes bytes, at most 256; refs [num_pages] counts who
 * holds a page (every table entry >= 0 is one reference; more may be held
 * elsewhere).  Full pages are shared.  A partly filled last page stays with
 * the lowest row that takes it when nobody else holds it; every other row gets
 * a copy of its filled rows in a free page, in every pool.  Then each
 * non-empty row gets free pages until len + reserve positions fit; entries
 * past those are -1 (pages an old row held beyond its length are let go).
 * Pages no entry names any more and nobody else holds become free (refs 0);
 * free pages are dealt out lowest id first, to rows in ascending order.
 * Outputs: table_out [rows, pages_per_seq], lens_out, refs_out (none may be its
 * input) and report I32 [4]: error, pages copied, pages newly reserved, pages
 * left free.  Errors: 2 a parent or length out of range (or len + reserve past
 * the row), 3 refs below the table's references, 5 too few free pages (report
 * [3] is how many more are needed), 6 a needed entry that names no page; where
 * several hold, 6 goes before 3 before 2 before 5.  The outputs are then copies
 * of the inputs and the pools are not touched.
 * rows <= 65536, rows * pages_per_seq < 2^31 - 8192; a call with no rows writes
 * nothing. */
uint64_t strata_b200_kv_fork_workspace_bytes(int64_t rows,
                                             int64_t pages_per_seq,
                                             int64_t num_pages);
int32_t strata_b200_kv_fork(
    void *const *pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads,
    int64_t page_size, int64_t num_pages, const int32_t *table_in,
    const int32_t *lens_in, const int32_t *refs_in, const int32_t *parents,
    int64_t rows, int64_t pages_per_seq, int64_t reserve, int32_t *table_out,
    int32_t *lens_out, int32_t *refs_out, int32_t *report, void *workspace,
    void *stream);

/* Moves the used pages (refs > 0) of the pools together: of n used pages, the
 * i-th with an id of n or more moves to the i-th free id below n.  Outputs:
 * table_out, refs_out (neither may be its input), remap [num_pages] (a page's
 * new id, -1 for a free page; for other holders of page ids) and report I32
 * [4]: error, used pages, pages moved, free pages.  Errors: 3 a negative count
 * or a table entry on a page without references, 6 an entry past the pool;
 * the outputs are then copies of the inputs (remap the identity) and the pools
 * are not touched.  The same pool arguments as kv_fork. */
uint64_t strata_b200_kv_compact_workspace_bytes(int64_t num_pages);
int32_t strata_b200_kv_compact(
    void *const *pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads,
    int64_t page_size, int64_t num_pages, const int32_t *table_in,
    const int32_t *refs_in, int64_t rows, int64_t pages_per_seq,
    int32_t *table_out, int32_t *refs_out, int32_t *remap, int32_t *report,
    void *workspace, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* STRATA_B200_H */

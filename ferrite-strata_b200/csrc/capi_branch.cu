// Kernel-level C entry points for several continuations of a sequence
// (include/strata_b200.h): argument checks, then the launchers of
// k_branch.cuh.
#include "../../include/strata_b200.h"
#include "k_branch.cuh"

using namespace sb;

namespace {

cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }

bool aligned(const void* p, uintptr_t n) { return p && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool fits(int64_t v, int64_t lo, int64_t hi = INT32_MAX) { return v >= lo && v <= hi; }

// The paged-cache arguments every entry point shares: no table means
// contiguous caches (page_size is then not looked at).
bool make_pages(const int32_t* table, int64_t max_len, int64_t kv_heads, int64_t page_size, int64_t num_pages,
                KvPages* kp) {
  *kp = KvPages{};
  if (!table) return true;
  if (!aligned(table, 4) || !kv_page_size_ok(page_size) || max_len % page_size || !fits(num_pages, 1)) return false;
  // rows of the pool, as the kernels number them
  if (num_pages > INT32_MAX / kv_heads / page_size) return false;
  kp->table = table;
  kp->page_size = int(page_size);
  kp->pages_per_seq = int(max_len / page_size);
  kp->num_pages = int(num_pages);
  return true;
}

bool make_pools(void* const* pools, int64_t n, int64_t row_bytes, KvPools* out) {
  if (!fits(n, 0, kMaxPools) || (n && !pools) || row_bytes < 16 || row_bytes % 16 || row_bytes > (1 << 20)) return false;
  *out = KvPools{};
  for (int64_t i = 0; i < n; ++i) {
    if (!aligned(pools[i], 16)) return false;
    out->p[i] = pools[i];
  }
  return true;
}

}  // namespace

extern "C" {

uint64_t strata_b200_tree_attention_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads,
                                                    int64_t head_dim) {
  return tree_attention_supported(tokens, heads, kv_heads, head_dim)
             ? tree_attention_workspace_bytes(tokens, heads, kv_heads, head_dim)
             : 0;
}

int32_t strata_b200_tree_attention_bf16(const uint16_t* q, const uint16_t* k_new, const uint16_t* v_new,
                                        uint16_t* k_cache, uint16_t* v_cache, const int32_t* block_table,
                                        const int32_t* base, const int32_t* count, const uint32_t* mask,
                                        int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                        int64_t head_dim, int64_t max_len, int64_t page_size, int64_t num_pages,
                                        void* workspace, uint16_t* out, int32_t* status, void* stream) {
  if (!fits(batch, 0, 65535) || !tree_attention_supported(tokens, heads, kv_heads, head_dim) || !fits(max_len, 1))
    return SB_INVALID_ARGUMENT;
  if (batch == 0) return SB_OK;
  TreeArgs a{q, k_new, v_new, k_cache, v_cache, base, count, mask, batch, tokens, heads, kv_heads, head_dim, max_len,
             KvPages{}, workspace, out, status};
  if (!make_pages(block_table, max_len, kv_heads, page_size, num_pages, &a.kp)) return SB_INVALID_ARGUMENT;
  if (!block_table && max_len > INT32_MAX / kv_heads / batch) return SB_INVALID_ARGUMENT;
  if (!aligned(base, 4) || !aligned(mask, 4) || (count && !aligned(count, 4)) || (status && !aligned(status, 4)))
    return SB_INVALID_ARGUMENT;
  return launch_tree_attention(a, S(stream));
}

uint64_t strata_b200_beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
  return beam_select_workspace_bytes(batch, beams, vocab, keep);
}

}  // extern "C"

template <typename T>
static int32_t beam_common(const T* logits, const float* scores, const int32_t* done, int64_t batch, int64_t beams,
                           int64_t vocab, int64_t keep, int64_t eos, float* out_scores, int32_t* out_parent,
                           int32_t* out_token, int32_t* out_done, void* workspace, void* stream) {
  if (!beam_select_supported(batch, beams, vocab, keep) || eos < -1 || eos >= vocab) return SB_INVALID_ARGUMENT;
  if (batch == 0) return SB_OK;
  if (!aligned(logits, sizeof(T)) || !aligned(scores, 4) || (done && !aligned(done, 4)) || !aligned(out_scores, 4) ||
      !aligned(out_parent, 4) || !aligned(out_token, 4) || !aligned(out_done, 4) || !aligned(workspace, 16))
    return SB_INVALID_ARGUMENT;
  return launch_beam_select<T>(logits, scores, done, batch, beams, vocab, keep, eos, out_scores, out_parent,
                               out_token, out_done, workspace, S(stream));
}

extern "C" {

int32_t strata_b200_beam_select_bf16(const uint16_t* logits, const float* scores, const int32_t* done, int64_t batch,
                                     int64_t beams, int64_t vocab, int64_t keep, int64_t eos, float* out_scores,
                                     int32_t* out_parent, int32_t* out_token, int32_t* out_done, void* workspace,
                                     void* stream) {
  return beam_common(logits, scores, done, batch, beams, vocab, keep, eos, out_scores, out_parent, out_token,
                     out_done, workspace, stream);
}

int32_t strata_b200_beam_select_f32(const float* logits, const float* scores, const int32_t* done, int64_t batch,
                                    int64_t beams, int64_t vocab, int64_t keep, int64_t eos, float* out_scores,
                                    int32_t* out_parent, int32_t* out_token, int32_t* out_done, void* workspace,
                                    void* stream) {
  return beam_common(logits, scores, done, batch, beams, vocab, keep, eos, out_scores, out_parent, out_token,
                     out_done, workspace, stream);
}

int32_t strata_b200_kv_accept(void* const* caches, int64_t n_caches, int64_t row_bytes, const int32_t* block_table,
                              const int32_t* base, const int32_t* path, const int32_t* n_path, int64_t batch,
                              int64_t kv_heads, int64_t max_len, int64_t max_path, int64_t page_size,
                              int64_t num_pages, int32_t* status, void* stream) {
  KvPools p;
  KvPages kp;
  if (!make_pools(caches, n_caches, row_bytes, &p) || !fits(batch, 0, 65535) || !fits(kv_heads, 1, 65535) ||
      !fits(max_len, 1) || !fits(max_path, 0, kTreeMaxTokens) ||
      !make_pages(block_table, max_len, kv_heads, page_size, num_pages, &kp))
    return SB_INVALID_ARGUMENT;
  if (batch == 0 || n_caches == 0 || max_path == 0) return SB_OK;
  if (!aligned(base, 4) || !aligned(path, 4) || !aligned(n_path, 4) || (status && !aligned(status, 4)))
    return SB_INVALID_ARGUMENT;
  return launch_kv_accept(p, n_caches, row_bytes, base, path, n_path, batch, kv_heads, max_len, max_path, kp, status,
                          S(stream));
}

// The arguments kv_fork and kv_compact share.
static bool pool_args(void* const* pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads, int64_t page_size,
                      int64_t num_pages, int64_t rows, int64_t pages_per_seq, KvPools* p) {
  return make_pools(pools, n_pools, row_bytes, p) && fits(kv_heads, 1, 65535) && kv_page_size_ok(page_size) &&
         fits(num_pages, 1, INT32_MAX / 2) && num_pages <= INT32_MAX / kv_heads / page_size && fits(rows, 0, 65536) &&
         fits(pages_per_seq, 1) && pages_per_seq <= INT32_MAX / page_size &&
         rows * pages_per_seq <= INT32_MAX - kPlanStep;
}

uint64_t strata_b200_kv_fork_workspace_bytes(int64_t rows, int64_t pages_per_seq, int64_t num_pages) {
  return fits(rows, 0, 65536) && fits(pages_per_seq, 1) && fits(num_pages, 1, INT32_MAX / 2)
             ? kv_fork_workspace_bytes(rows, pages_per_seq, num_pages)
             : 0;
}

int32_t strata_b200_kv_fork(void* const* pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads,
                            int64_t page_size, int64_t num_pages, const int32_t* table_in, const int32_t* lens_in,
                            const int32_t* refs_in, const int32_t* parents, int64_t rows, int64_t pages_per_seq,
                            int64_t reserve, int32_t* table_out, int32_t* lens_out, int32_t* refs_out,
                            int32_t* report, void* workspace, void* stream) {
  KvPools p;
  if (!pool_args(pools, n_pools, row_bytes, kv_heads, page_size, num_pages, rows, pages_per_seq, &p) ||
      !fits(reserve, 0))
    return SB_INVALID_ARGUMENT;
  if (rows == 0) return SB_OK;
  if (!aligned(table_in, 4) || !aligned(lens_in, 4) || !aligned(refs_in, 4) || !aligned(parents, 4) ||
      !aligned(table_out, 4) || !aligned(lens_out, 4) || !aligned(refs_out, 4) || !aligned(report, 4) ||
      !aligned(workspace, 16) || table_in == table_out || lens_in == lens_out || refs_in == refs_out)
    return SB_INVALID_ARGUMENT;
  return launch_kv_fork(p, n_pools, row_bytes, kv_heads, page_size, num_pages, table_in, lens_in, refs_in, parents,
                        rows, pages_per_seq, reserve, table_out, lens_out, refs_out, report, workspace, S(stream));
}

uint64_t strata_b200_kv_compact_workspace_bytes(int64_t num_pages) {
  return fits(num_pages, 1, INT32_MAX / 2) ? kv_compact_workspace_bytes(num_pages) : 0;
}

int32_t strata_b200_kv_compact(void* const* pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads,
                               int64_t page_size, int64_t num_pages, const int32_t* table_in, const int32_t* refs_in,
                               int64_t rows, int64_t pages_per_seq, int32_t* table_out, int32_t* refs_out,
                               int32_t* remap, int32_t* report, void* workspace, void* stream) {
  KvPools p;
  if (!pool_args(pools, n_pools, row_bytes, kv_heads, page_size, num_pages, rows, pages_per_seq, &p))
    return SB_INVALID_ARGUMENT;
  if (!aligned(refs_in, 4) || !aligned(refs_out, 4) || !aligned(remap, 4) || !aligned(report, 4) ||
      (rows && (!aligned(table_in, 4) || !aligned(table_out, 4) || table_in == table_out)) ||
      !aligned(workspace, 16) || refs_in == refs_out)
    return SB_INVALID_ARGUMENT;
  return launch_kv_compact(p, n_pools, row_bytes, kv_heads, page_size, num_pages, table_in, refs_in, rows,
                           pages_per_seq, table_out, refs_out, remap, report, workspace, S(stream));
}

}  // extern "C"

// Launcher declarations of the kernels for several continuations of a
// sequence: drafted trees and beams over KV caches.
#pragma once

#include "common.cuh"

namespace sb {

// Error codes the kernels leave in a caller's status word (the executor's
// error word uses the same numbers).
constexpr int kBadPosition = 2;  // a length, position, index or parent outside its range
constexpr int kBadRefs = 3;      // a page's reference count is below the table's own references
constexpr int kNoPages = 5;      // the pool has too few free pages
constexpr int kBadPage = 6;      // a block-table entry that is needed names no page of the pool

// Attention of a tree of drafted tokens over the cached prompt (k_tree.cu).
constexpr int kTreeMaxTokens = 1024;
struct TreeArgs {
  const uint16_t *q, *k_new, *v_new;  // [batch * tokens, heads * d], [batch * tokens, kv_heads * d]
  uint16_t *k_cache, *v_cache;
  const int32_t* base;    // [batch]: positions cached before the tree
  const int32_t* count;   // [batch]: live nodes, null for `tokens` everywhere
  const uint32_t* mask;   // [batch, tokens, ceil(tokens / 32)]
  int64_t batch, tokens, heads, kv_heads, head_dim, max_len;
  KvPages kp;
  void* workspace;
  uint16_t* out;
  int* err;
};
uint64_t tree_attention_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim);
bool tree_attention_supported(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim);
int launch_tree_attention(const TreeArgs& a, cudaStream_t st);

// Beam selection (k_beam.cu).
constexpr int kBeamMaxKeep = 64;
constexpr int kBeamMaxBeams = 1024;
uint64_t beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep);
bool beam_select_supported(int64_t batch, int64_t beams, int64_t vocab, int64_t keep);
template <typename T>
int launch_beam_select(const T* logits, const float* scores, const int32_t* done, int64_t batch, int64_t beams,
                       int64_t vocab, int64_t keep, int64_t eos, float* out_scores, int32_t* out_parent,
                       int32_t* out_token, int32_t* out_done, void* workspace, cudaStream_t st);

// Cache upkeep (k_kvpages.cu).  The caches or pools of every layer, passed to
// a kernel by value.
constexpr int kMaxPools = 256;
struct KvPools {
  void* p[kMaxPools];
};
int launch_kv_accept(const KvPools& caches, int64_t n_caches, int64_t row_bytes, const int32_t* base,
                     const int32_t* path, const int32_t* n_path, int64_t batch, int64_t kv_heads, int64_t max_len,
                     int64_t max_path, const KvPages& kp, int* err, cudaStream_t st);
// Table entries that a planning kernel steps over at once; a table ends that far below 2^31.
constexpr int kPlanStep = 8192;
uint64_t kv_fork_workspace_bytes(int64_t rows, int64_t pages_per_seq, int64_t num_pages);
int launch_kv_fork(const KvPools& pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads, int64_t page_size,
                   int64_t num_pages, const int32_t* table_in, const int32_t* lens_in, const int32_t* refs_in,
                   const int32_t* parents, int64_t rows, int64_t pages_per_seq, int64_t reserve, int32_t* table_out,
                   int32_t* lens_out, int32_t* refs_out, int32_t* report, void* workspace, cudaStream_t st);
uint64_t kv_compact_workspace_bytes(int64_t num_pages);
int launch_kv_compact(const KvPools& pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads, int64_t page_size,
                      int64_t num_pages, const int32_t* table_in, const int32_t* refs_in, int64_t rows,
                      int64_t pages_per_seq, int32_t* table_out, int32_t* refs_out, int32_t* remap, int32_t* report,
                      void* workspace, cudaStream_t st);

}  // namespace sb

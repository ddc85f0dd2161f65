// Attention of a tree of drafted tokens over a cached prompt.
//
// Sequence b has base[b] cached positions and count[b] live nodes.  Node i's k
// and v rows are appended at position base + i, and node t attends to every
// position below base and to the nodes whose bit is set in its mask row.  A
// node at or past count, and one that sees nothing, gives zeros.
#include "common.cuh"
#include "k_branch.cuh"

namespace sb {

namespace {

struct TreeSeq {
  int base, count;  // count 0 where the sequence is unusable
  bool bad;
};

__device__ __forceinline__ TreeSeq tree_seq(const int32_t* base, const int32_t* count, int tokens, int max_len, int b) {
  TreeSeq s{base[b], count ? count[b] : tokens, false};
  if (s.count < 0 || s.count > tokens || s.base < 0 || s.base > max_len - s.count) {
    s.count = 0;
    s.bad = true;
  }
  return s;
}

__global__ void tree_append_kernel(const TreeArgs a) {
  const int b = int(blockIdx.y), t = int(blockIdx.x);
  const TreeSeq s = tree_seq(a.base, a.count, int(a.tokens), int(a.max_len), b);
  if (s.bad && threadIdx.x == 0 && a.err) atomicExch(a.err, kBadPosition);
  const int d = int(a.head_dim), w = int(a.kv_heads) * d;
  const int64_t r = int64_t(b) * a.tokens + t;
  if (t >= s.count) {
    for (int i = threadIdx.x; i < int(a.heads) * d; i += blockDim.x) a.out[r * a.heads * d + i] = 0;
    return;
  }
  for (int i = threadIdx.x; i < w; i += blockDim.x) {
    const int64_t row = kv_row(a.kp, b, i / d, int(a.kv_heads), int(a.max_len), s.base + t);
    if (row < 0) {
      if (a.err) atomicExch(a.err, kBadPage);
      continue;
    }
    a.k_cache[row * d + i % d] = a.k_new[r * w + i];
    a.v_cache[row * d + i % d] = a.v_new[r * w + i];
  }
}

// One warp per (node, head): each position's product is summed over the lanes,
// with a running maximum and sum.
__global__ void tree_warp_kernel(const TreeArgs a) {
  const int b = int(blockIdx.z), h = int(blockIdx.y) * int(blockDim.y) + int(threadIdx.y), t = int(blockIdx.x);
  const int lane = threadIdx.x, d = int(a.head_dim), per = d / 32;
  const TreeSeq s = tree_seq(a.base, a.count, int(a.tokens), int(a.max_len), b);
  if (h >= a.heads || t >= s.count) return;
  const int kvh = h / int(a.heads / a.kv_heads);
  const int64_t r = int64_t(b) * a.tokens + t;
  const uint32_t* mask = a.mask + r * ((a.tokens + 31) / 32);
  float q[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
  for (int e = 0; e < per; ++e) q[e] = bf2f(a.q[(r * a.heads + h) * d + lane * per + e]) * rsqrtf(float(d));
  for (int p = 0; p < s.base + s.count; ++p) {
    const int j = p - s.base;
    if (j >= 0 && !(mask[j / 32] >> (j % 32) & 1)) continue;
    const int64_t row = kv_row(a.kp, b, kvh, int(a.kv_heads), int(a.max_len), p);
    if (row < 0) {
      if (a.err) atomicExch(a.err, kBadPage);
      continue;
    }
    float x = 0.0f;
    for (int e = 0; e < per; ++e) x += q[e] * bf2f(a.k_cache[row * d + lane * per + e]);
    x = warp_sum(x);
    const float mn = fmaxf(m, x), c = m == -INFINITY ? 0.0f : expf(m - mn), w = expf(x - mn);
    l = l * c + w;
    for (int e = 0; e < per; ++e) o[e] = o[e] * c + w * bf2f(a.v_cache[row * d + lane * per + e]);
    m = mn;
  }
  for (int e = 0; e < per; ++e)
    a.out[(r * a.heads + h) * d + lane * per + e] = f2bf(l > 0.0f || l != l ? o[e] / l : 0.0f);
}

}  // namespace

uint64_t tree_attention_workspace_bytes(int64_t, int64_t, int64_t, int64_t) { return 256; }

bool tree_attention_supported(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  return tokens >= 1 && tokens <= kTreeMaxTokens && kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0 &&
         heads / kv_heads <= 128 && heads <= 65535 && (head_dim == 64 || head_dim == 128);
}

int launch_tree_attention(const TreeArgs& a, cudaStream_t st) {
  if (!tree_attention_supported(a.tokens, a.heads, a.kv_heads, a.head_dim)) return SB_INVALID_ARGUMENT;
  if (a.batch == 0) return SB_OK;
  tree_append_kernel<<<dim3(unsigned(a.tokens), unsigned(a.batch)), 128, 0, st>>>(a);
  SB_LAUNCH_CHECK();
  tree_warp_kernel<<<dim3(unsigned(a.tokens), unsigned((a.heads + 3) / 4), unsigned(a.batch)), dim3(32, 4), 0, st>>>(a);
  SB_LAUNCH_CHECK();
  return SB_OK;
}

}  // namespace sb

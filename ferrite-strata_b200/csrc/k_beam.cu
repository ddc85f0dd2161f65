// Beam selection: the `keep` best continuations of every batch entry over its
// beams and the vocabulary.
//
//   logp[w, v] = l[w, v] - lse_w,  lse_w = m_w + log(sum_v exp(l[w, v] - m_w))
//   candidates (score[w] + logp[w, v], parent w, token v), best first, the
//   lowest w * V + v on ties
//
// Within a beam the order of the candidates is the order of its logits, so
// one pass over the logits is enough: the first kernel reads a run of one
// row's logits, keeps its maximum, the sum of exponentials against it and the
// run's `keep` largest logits; the second joins the runs of a row, turns what
// is left into scores and selects over the beams.  The read of the logits
// bounds it (HBM) for large calls, latency for small ones.
//
// Scores are compared in 64 bits: two beams' candidates can lie closer than
// 32 bits resolve at a score of some tens.  A sum of exponentials is kept in
// 32 bits over the 32 logits a thread holds and in 64 from there on.
#include <algorithm>

#include "common.cuh"
#include "k_branch.cuh"

namespace sb {

namespace {

constexpr int kBmThreads = 256;
constexpr int kBmPer = 32;                        // logits a thread holds
constexpr int kBmTile = kBmThreads * kBmPer;      // logits per block step
constexpr int kBmCap = 1024;                      // candidates taken directly against the running threshold
constexpr int kBmList = kBeamMaxKeep + (kBeamMaxKeep - 1) * kBmPer + 1;  // the most candidates at once
static_assert(kBmCap + kBeamMaxKeep <= kBmList, "candidate list");
constexpr int kMgThreads = 1024;
constexpr int kMgMost = 65536;  // candidates the joining block takes: beams * runs * keep

// Order-preserving map of a float's bits to unsigned.
__device__ __forceinline__ uint32_t ord32(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unord32(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// A candidate of one row: larger key = larger logit, then lower id.  -inf
// (and NaN, read as -inf) is never a candidate; key 0 stands for none.
__device__ __forceinline__ uint64_t cand_key(float x, uint32_t id) {
  return (uint64_t(ord32(x)) << 32) | uint32_t(~id);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2eF = 1.4426950408889634f;

struct RunStat {
  double sum;
  float max;
  int pad;
};

// 16 bytes of logits from byte address `p`, which need not be aligned: the one
// or two aligned 16-byte blocks that hold them, shifted together.  A block is
// read only if it holds a byte below `end`.
__device__ __forceinline__ uint4 load16(const uint8_t* p, const uint8_t* end) {
  const uint32_t mis = uint32_t(reinterpret_cast<uintptr_t>(p)) & 15;
  const uint4* a = reinterpret_cast<const uint4*>(p - mis);
  const uint4 lo = __ldg(a);
  if (mis == 0) return lo;
  uint4 hi = make_uint4(0, 0, 0, 0);
  if (reinterpret_cast<const uint8_t*>(a + 1) < end) hi = __ldg(a + 1);
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (mis & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (mis & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const uint32_t sh = (mis & 2) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh), __funnelshift_r(w[2], w[3], sh),
                    __funnelshift_r(w[3], w[4], sh));
}

template <typename T>
struct BeamArgs {
  const T* logits;
  const float* scores;
  const int32_t* done;
  int beams, keep, runs;  // runs: blocks per row
  int vocab, span;        // span: logits per block, a multiple of kBmTile
  int eos;
  float* out_scores;
  int32_t *out_parent, *out_token, *out_done;
  RunStat* stats;   // [rows][runs]
  uint64_t* cands;  // [rows][runs][keep], best first, 0 past the last
};

// The rank of every key among n distinct ones, best first; the first `keep` go
// to out in order.  All threads.
__device__ __forceinline__ void select_sorted(const uint64_t* in, int n, int keep, uint64_t* out) {
  for (int i = threadIdx.x; i < n; i += kBmThreads) {
    const uint64_t k = in[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += in[j] > k;
    if (rank < keep) out[rank] = k;
  }
}

template <typename T>
__global__ void __launch_bounds__(kBmThreads) beam_run_kernel(const BeamArgs<T> a) {
  constexpr int kVec = 16 / int(sizeof(T));
  __shared__ uint64_t s_list[kBmList];
  __shared__ uint64_t s_best[kBeamMaxKeep];
  __shared__ uint64_t s_tkey[kBmThreads], s_cut;
  __shared__ double s_red[kBmThreads / 32];
  __shared__ float s_max[kBmThreads / 32];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = blockIdx.x, row = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  const float score = a.scores[row];
  if (!(score > -INFINITY) || (a.done && a.done[row])) return;  // no candidate of this row is looked at
  const int v0 = run * a.span, v1 = min(a.vocab, v0 + a.span);
  const uint8_t* base = reinterpret_cast<const uint8_t*>(a.logits + int64_t(row) * a.vocab);
  const uint8_t* end = base + int64_t(a.vocab) * int(sizeof(T));
  float m_run = -INFINITY;
  double sum = 0.0;   // thread's share, against m_run
  int have = 0;       // candidates in s_best
  float tau = -INFINITY;  // the keep-th best so far (have == keep)
  for (int t0 = v0; t0 < v1; t0 += kBmTile) {
    float x[kBmPer];
#pragma unroll
    for (int v = 0; v < kBmPer / kVec; ++v) {
      const int e = t0 + (v * kBmThreads + tid) * kVec;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (e < v1) u = load16(base + int64_t(e) * int(sizeof(T)), end);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        float f;
        if constexpr (sizeof(T) == 2) f = (j & 1) ? bf_hi(w[j / 2]) : bf_lo(w[j / 2]);
        else f = __uint_as_float(w[j]);
        x[v * kVec + j] = e + j < v1 ? fmaxf(f, -INFINITY) : -INFINITY;  // NaN -> -inf
      }
    }
    float tm = -INFINITY;
#pragma unroll
    for (int i = 0; i < kBmPer; ++i) tm = fmaxf(tm, x[i]);
    const float wm = warp_max(tm);
    if (lane == 0) s_max[warp] = wm;
    if (tid == 0) s_n = 0;
    __syncthreads();
    float bm = s_max[0];
#pragma unroll
    for (int w = 1; w < kBmThreads / 32; ++w) bm = fmaxf(bm, s_max[w]);
    // ---- sum of exponentials against the running maximum -----------------------
    const float m_new = fmaxf(m_run, bm);
    if (m_new == -INFINITY) {  // nothing but -inf so far
      __syncthreads();
      continue;
    }
    // In pairs, so that many small terms beside a large one are not each
    // rounded against it (32 in a row were off by 28 halves of its last bit).
    float part = 0.0f, quad[kBmPer / 8];
    if (m_new == INFINITY) {  // only the infinite logits share the probability
#pragma unroll
      for (int i = 0; i < kBmPer; ++i) part += x[i] == INFINITY ? 1.0f : 0.0f;
      sum = m_run == INFINITY ? sum : 0.0;
    } else {
#pragma unroll
      for (int i = 0; i < kBmPer; i += 8) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = ex2((x[i + j] - m_new) * kLog2eF);
        quad[i / 8] = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
      }
      part = (quad[0] + quad[1]) + (quad[2] + quad[3]);
      if (m_new != m_run) sum = m_run == -INFINITY ? 0.0 : sum * exp(double(m_run) - double(m_new));
    }
    sum += double(part);
    m_run = m_new;
    // ---- candidates ------------------------------------------------------------
    // With a full list only logits above its last one count (an equal one has
    // a higher id).  Without, or when too many are above, the keep-th best of
    // the threads' best ones is a bound that at least `keep` logits reach; a
    // thread can hold several logits past it only if its best one is past it,
    // so at most (keep - 1) * 32 + 1 do.
    bool direct = have == a.keep;
    if (direct) {
      int above = 0;
#pragma unroll
      for (int i = 0; i < kBmPer; ++i) above += x[i] > tau;
      if (above) atomicAdd(&s_n, above);
      __syncthreads();
      const int n = s_n;
      if (n == 0) {
        __syncthreads();
        continue;
      }
      direct = n <= kBmCap;
    }
    auto id_of = [&](int i) { return uint32_t(t0 + ((i / kVec) * kBmThreads + tid) * kVec + i % kVec); };
    uint64_t cut = 0;
    if (!direct) {
      int first = 0;
#pragma unroll
      for (int i = kBmPer - 1; i >= 0; --i)
        if (x[i] == tm) first = i;
      const uint64_t key = tm > -INFINITY ? cand_key(tm, id_of(first)) : 0;
      s_tkey[tid] = key;
      if (tid == 0) s_cut = 0;
      __syncthreads();
      int rank = 0;
      for (int j = 0; j < kBmThreads; ++j) rank += s_tkey[j] > key;
      if (key && rank == a.keep - 1) s_cut = key;
      __syncthreads();
      cut = s_cut;
    }
    for (int i = tid; i < have; i += kBmThreads) s_list[i] = s_best[i];
    __syncthreads();
    if (tid == 0) s_n = have;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBmPer; ++i) {
      const float f = x[i];
      if (f > (have == a.keep ? tau : -INFINITY)) {
        const uint64_t k = cand_key(f, id_of(i));
        if (k >= cut) s_list[atomicAdd(&s_n, 1)] = k;
      }
    }
    __syncthreads();
    const int n = s_n;
    select_sorted(s_list, n, a.keep, s_best);
    have = min(n, a.keep);
    __syncthreads();
    if (have == a.keep) tau = unord32(uint32_t(s_best[a.keep - 1] >> 32));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_red[warp] = sum;
  __syncthreads();
  const int64_t slot = int64_t(row) * a.runs + run;
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < kBmThreads / 32; ++w) t += s_red[w];
    a.stats[slot] = RunStat{t, m_run, 0};
  }
  for (int i = tid; i < a.keep; i += kBmThreads) a.cands[slot * a.keep + i] = i < have ? s_best[i] : 0;
}

// A candidate of a batch entry: better = higher score, then lower `flat`
// (beam << 32 | token).
struct Scored {
  double score;
  uint64_t flat;
};
__device__ __forceinline__ bool better(const Scored& a, const Scored& b) {
  return a.score > b.score || (a.score == b.score && a.flat < b.flat);
}
constexpr uint64_t kNoFlat = ~uint64_t(0);

template <typename T>
__global__ void __launch_bounds__(kMgThreads) beam_join_kernel(const BeamArgs<T> a) {
  extern __shared__ __align__(16) uint8_t smem[];
  double* s_log = reinterpret_cast<double*>(smem);             // [beams] log of the row's sum
  float* s_m = reinterpret_cast<float*>(s_log + a.beams);      // [beams] the row's maximum
  Scored* s_top = reinterpret_cast<Scored*>(smem + ((size_t(a.beams) * 12 + 15) & ~size_t(15)));  // [threads] best of each
  Scored* s_list = s_top + kMgThreads;                         // survivors
  __shared__ int s_n;
  __shared__ Scored s_cut;
  const int tid = threadIdx.x, b = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  if (tid == 0) {
    s_n = 0;
    s_cut = Scored{-INFINITY, kNoFlat};
  }
  for (int w = tid; w < a.beams; w += kMgThreads) {
    const int64_t row = int64_t(b) * a.beams + w;
    const bool dead = !(a.scores[row] > -INFINITY), done = a.done && a.done[row];
    float m = -INFINITY;
    double sum = 0.0;
    if (!dead && !done) {
      for (int r = 0; r < a.runs; ++r) m = fmaxf(m, a.stats[row * a.runs + r].max);
      for (int r = 0; r < a.runs; ++r) {
        const RunStat s = a.stats[row * a.runs + r];
        if (s.max > -INFINITY) sum += s.max == m ? s.sum : m == INFINITY ? 0.0 : s.sum * exp(double(s.max) - double(m));
      }
    }
    s_m[w] = m;
    s_log[w] = log(sum);
  }
  __syncthreads();
  // Candidate i of the entry: (beam, run, place) with the place fastest.  A
  // thread takes i = tid, tid + 1024, ...
  const int per_beam = a.runs * a.keep, total = a.beams * per_beam;
  auto get = [&](int i) {
    const int w = i / per_beam, j = i % per_beam;
    const int64_t row = int64_t(b) * a.beams + w;
    Scored c{-INFINITY, kNoFlat};
    const float s = a.scores[row];
    if (!(s > -INFINITY)) return c;
    if (a.done && a.done[row]) {
      if (j == 0) c = Scored{double(s), uint64_t(w) << 32 | uint32_t(max(a.eos, 0))};
      return c;
    }
    const uint64_t k = a.cands[row * per_beam + j];
    if (k == 0) return c;
    const float x = unord32(uint32_t(k >> 32)), m = s_m[w];
    c.score = double(s) + ((x == m ? 0.0 : double(x) - double(m)) - s_log[w]);
    c.flat = uint64_t(w) << 32 | uint32_t(~uint32_t(k));
    if (!(c.score > -INFINITY)) c = Scored{-INFINITY, kNoFlat};
    return c;
  };
  Scored best{-INFINITY, kNoFlat};
  for (int i = tid; i < total; i += kMgThreads) {
    const Scored c = get(i);
    if (better(c, best)) best = c;
  }
  s_top[tid] = best;
  __syncthreads();
  // The keep-th best of the threads' best ones bounds the answer from below.
  const int live = min(total, kMgThreads);
  if (tid < live && best.flat != kNoFlat) {
    int rank = 0;
    for (int j = 0; j < live; ++j) rank += better(s_top[j], best);
    if (rank == a.keep - 1) s_cut = best;
  }
  __syncthreads();
  const Scored cut = s_cut;
  if (best.flat != kNoFlat && !better(cut, best)) {
    for (int i = tid; i < total; i += kMgThreads) {
      const Scored c = get(i);
      if (c.flat != kNoFlat && !better(cut, c)) s_list[atomicAdd(&s_n, 1)] = c;
    }
  }
  __syncthreads();
  const int n = s_n;
  const int64_t o0 = int64_t(b) * a.keep;
  for (int i = tid; i < n; i += kMgThreads) {
    const Scored c = s_list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += better(s_list[j], c);
    if (rank < a.keep) {
      const int w = int(c.flat >> 32), token = int(uint32_t(c.flat));
      const int64_t row = int64_t(b) * a.beams + w;
      const bool done = a.done && a.done[row];
      a.out_scores[o0 + rank] = float(c.score);
      a.out_parent[o0 + rank] = int(row);
      a.out_token[o0 + rank] = done && a.eos < 0 ? -1 : token;
      a.out_done[o0 + rank] = done || (a.eos >= 0 && token == a.eos) ? 1 : 0;
    }
  }
  for (int i = n + tid; i < a.keep; i += kMgThreads) {
    a.out_scores[o0 + i] = -INFINITY;
    a.out_parent[o0 + i] = -1;
    a.out_token[o0 + i] = -1;
    a.out_done[o0 + i] = 0;
  }
}

// Blocks per row: enough for four blocks on every SM, each with at least one
// tile, at most what the joining block takes.
int beam_runs(int64_t rows, int64_t beams, int64_t vocab, int64_t keep) {
  const int64_t tiles = (vocab + kBmTile - 1) / kBmTile;
  int64_t runs = (4 * kNumSMs + rows - 1) / rows;
  runs = std::min(runs, tiles);
  runs = std::min(runs, kMgMost / (beams * keep));
  runs = std::max<int64_t>(runs, 1);
  const int64_t per = (tiles + runs - 1) / runs;
  return int((tiles + per - 1) / per);
}

constexpr uint64_t up256(uint64_t x) { return (x + 255) & ~uint64_t(255); }

}  // namespace

bool beam_select_supported(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
  return batch >= 0 && beams >= 1 && beams <= kBeamMaxBeams && vocab >= 1 && vocab <= (int64_t(1) << 30) &&
         keep >= 1 && keep <= kBeamMaxKeep && batch * beams <= 65535;
}

uint64_t beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
  if (!beam_select_supported(batch, beams, vocab, keep) || batch == 0) return 0;
  const uint64_t slots = uint64_t(batch * beams) * uint64_t(beam_runs(batch * beams, beams, vocab, keep));
  return up256(slots * sizeof(RunStat)) + up256(slots * uint64_t(keep) * sizeof(uint64_t));
}

template <typename T>
int launch_beam_select(const T* logits, const float* scores, const int32_t* done, int64_t batch, int64_t beams,
                       int64_t vocab, int64_t keep, int64_t eos, float* out_scores, int32_t* out_parent,
                       int32_t* out_token, int32_t* out_done, void* workspace, cudaStream_t st) {
  if (!beam_select_supported(batch, beams, vocab, keep)) return SB_INVALID_ARGUMENT;
  if (batch == 0) return SB_OK;
  const int64_t rows = batch * beams;
  const int runs = beam_runs(rows, beams, vocab, keep);
  const int64_t tiles = (vocab + kBmTile - 1) / kBmTile;
  BeamArgs<T> a{logits, scores, done, int(beams), int(keep), runs, int(vocab),
                int((tiles + runs - 1) / runs * kBmTile), int(eos), out_scores, out_parent, out_token, out_done,
                nullptr, nullptr};
  a.stats = static_cast<RunStat*>(workspace);
  a.cands = reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(workspace) +
                                        up256(uint64_t(rows) * uint64_t(runs) * sizeof(RunStat)));
  if (launch_pdl(beam_run_kernel<T>, dim3(unsigned(runs), unsigned(rows)), dim3(kBmThreads), 0, st, a) != cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  // Survivors of the joining block: fewer than keep threads hold more than one.
  const int64_t each = (beams * runs * keep + kMgThreads - 1) / kMgThreads;
  const size_t smem = ((size_t(beams) * 12 + 15) & ~size_t(15)) +
                      sizeof(Scored) * size_t(kMgThreads + keep * each);
  static PerDeviceOnce configured;
  if (!configured.run([] {
        return cudaFuncSetAttribute(beam_join_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024) ==
               cudaSuccess;
      }))
    return SB_INTERNAL;
  if (launch_pdl(beam_join_kernel<T>, dim3(unsigned(batch)), dim3(kMgThreads), smem, st, a) != cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  return SB_OK;
}

template int launch_beam_select<uint16_t>(const uint16_t*, const float*, const int32_t*, int64_t, int64_t, int64_t,
                                          int64_t, int64_t, float*, int32_t*, int32_t*, int32_t*, void*,
                                          cudaStream_t);
template int launch_beam_select<float>(const float*, const float*, const int32_t*, int64_t, int64_t, int64_t, int64_t,
                                       int64_t, float*, int32_t*, int32_t*, int32_t*, void*, cudaStream_t);

}  // namespace sb

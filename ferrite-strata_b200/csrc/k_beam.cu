// Beam selection: the `keep` best continuations of every batch entry over its
// beams and the vocabulary.
//
//   logp[w, v] = l[w, v] - lse_w,  lse_w = m_w + log(sum_v exp(l[w, v] - m_w))
//   candidates (score[w] + logp[w, v], parent w, token v), best first, the
//   lowest w * V + v on ties
//
// Within a beam the order of the candidates is the order of its logits, so
// one pass over the logits is enough: the first kernel reads a run of one
// row's logits, sums exponentials and keeps the run's `keep` largest logits; the
// second joins the runs of a row, turns what is left into scores and selects
// over the beams.  Large calls are bound by issuing the sums' instructions (with the
// logits read at 4.7 of 6.6 TB/s) and by the blocks' ends, small ones by latency.
//
// The first kernel works a warp at a time, 1024 logits a step, with no barrier
// until the run's end.  A lane sums exponentials against a reference of its own
// that moves only when a logit exceeds it by 4 (so the sums are seldom
// rescaled), and notes the maximum of its 32 logits of each step.
// At the end the keep-th largest of the 256 lanes' maxima bounds the answer from
// below, and in random logits little more than `keep` reach it: only the noted
// groups of 32 whose maximum does are read again, and what reaches the bound is
// placed by counting.  Checking every step against a running bound instead took
// about as many instructions as the sums (56 us, and 105 with each warp going by
// a list of its own, against 37, for 512 rows of 128001 bf16, keep 32); a ring of
// asynchronous copies to shared memory cost more in resident blocks than it hid
// (54 us).  Without the last part the pass takes 28 us, 4.7 TB/s.  With the joining
// kernel, about 7 us, the call takes 46 us; 4 rows of 32000 f32 take 11 us, which is
// the latency of two kernels.
//
// Scores are compared in 64 bits: two beams' candidates can lie closer than
// 32 bits resolve at a score of some tens.  A sum of exponentials is kept in
// 32 bits over the 32 logits a lane holds (in pairs, so that many small terms
// beside a large one are not each rounded against it) and in 64 from there on.
#include <algorithm>

#include "common.cuh"
#include "k_branch.cuh"

namespace sb {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kPer = 32;           // logits a lane holds
constexpr int kStep = 32 * kPer;   // logits a warp takes at once
constexpr int kTile = kWarps * kStep;
// How far a logit may exceed a lane's reference.  A term's exponent (x - ref) log2(e) is formed
// in f32: up to 4 above, x - ref and the product are off by 2^-23 and 2^-22 and the constant adds
// 2^-23.6, so the term by 1.5 x 2^-22 relative and ex2's 2^-22; with five additions of 2^-24 the
// sum, and the logarithm, is within 2^-20.  At 16 a term alone was off by 1.4 x 2^-20; 4 costs
// 0.2 to 0.8 us of 45 (512 rows of 128001 bf16), 2 costs 2.6.
constexpr float kLag = 4.0f;
constexpr int kMaxSteps = 24;      // of a run: one noted maximum per lane and step
constexpr uint32_t kAll = 0xffffffffu;

// Order-preserving map of a float's bits to unsigned; -0 counts as 0.
__device__ __forceinline__ uint32_t ord32(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unord32(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// A candidate of one row: larger key = larger logit, then lower id.  Key 0
// stands for none.
__device__ __forceinline__ uint64_t cand_key(float x, uint32_t id) {
  return (uint64_t(ord32(x)) << 32) | uint32_t(~id);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
constexpr float kLog2eF = 1.4426950408889634f;

struct RunStat {
  double sum;  // of exp(l - ref)
  float ref;
  int pad;
};

// ---------------------------------------------------------------------------
// Lists sorted across a warp: entry j * 32 + lane, best first
// ---------------------------------------------------------------------------
struct Key {
  uint64_t k;
  __device__ static Key none() { return Key{0}; }
  __device__ bool better(const Key& o) const { return k > o.k; }
  __device__ Key shfl(int lane) const { return Key{__shfl_sync(kAll, k, lane)}; }
  __device__ Key shfl_xor(int m) const { return Key{__shfl_xor_sync(kAll, k, m)}; }
};

// A candidate of a batch entry: the score's order-preserving bits, then the
// lower `flat` (beam << 32 | token).  Score 0 stands for none.
struct Scored {
  uint64_t score;
  uint64_t flat;
  __device__ static Scored none() { return Scored{0, ~uint64_t(0)}; }
  __device__ bool better(const Scored& o) const { return score > o.score || (score == o.score && flat < o.flat); }
  __device__ Scored shfl(int lane) const { return Scored{__shfl_sync(kAll, score, lane), __shfl_sync(kAll, flat, lane)}; }
  __device__ Scored shfl_xor(int m) const {
    return Scored{__shfl_xor_sync(kAll, score, m), __shfl_xor_sync(kAll, flat, m)};
  }
};
__device__ __forceinline__ uint64_t ord64(double x) {
  const uint64_t b = uint64_t(__double_as_longlong(x + 0.0));
  return b >> 63 ? ~b : b | uint64_t(1) << 63;
}
__device__ __forceinline__ double unord64(uint64_t u) {
  return __longlong_as_double(int64_t(u >> 63 ? u & ~(uint64_t(1) << 63) : ~u));
}

// Compare-exchange of all entries with those `stride` further on: the better
// one goes to the lower place where `up` is set, to the higher one otherwise.
template <typename E, int N>
__device__ __forceinline__ void exchange(E (&v)[N], int stride, int block) {
  const int lane = threadIdx.x & 31;
  if (stride >= 32) {
    const int d = stride / 32;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j & d) continue;
      const bool up = ((j * 32 + lane) & block) == 0;
      if (v[j + d].better(v[j]) == up) {
        const E t = v[j];
        v[j] = v[j + d];
        v[j + d] = t;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const E o = v[j].shfl_xor(stride);
      const bool up = ((j * 32 + lane) & block) == 0;
      const bool low = (lane & stride) == 0;
      if (o.better(v[j]) == (low == up)) v[j] = o;
    }
  }
}

// Sorts N * 32 entries, best first.
template <typename E, int N>
__device__ __forceinline__ void sort_list(E (&v)[N]) {
#pragma unroll
  for (int block = 2; block <= N * 32; block *= 2)
#pragma unroll
    for (int stride = block / 2; stride > 0; stride /= 2) exchange(v, stride, block == N * 32 ? 0 : block);
}

// v becomes the best N * 32 of two sorted lists, sorted: the better of v[i]
// and o[last - i] is a bitonic sequence of exactly those.
template <typename E, int N>
__device__ __forceinline__ void merge_list(E (&v)[N], const E (&o)[N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const E x = o[N - 1 - j].shfl(31 - lane);
    if (x.better(v[j])) v[j] = x;
  }
#pragma unroll
  for (int stride = N * 16; stride > 0; stride /= 2) exchange(v, stride, 0);
}

// Entry i of a list, to every lane.
template <typename E, int N>
__device__ __forceinline__ E entry(const E (&v)[N], int i) {
  if (N > 1 && i >= 32) return v[N - 1].shfl(i & 31);
  return v[0].shfl(i & 31);
}

template <typename T>
struct BeamArgs {
  const T* logits;
  const float* scores;
  const int32_t* done;
  int beams, keep, runs;  // runs: blocks per row
  int vocab, span;        // span: logits per block, a multiple of kTile
  int eos;
  float* out_scores;
  int32_t *out_parent, *out_token, *out_done;
  RunStat* stats;   // [rows][runs]
  uint64_t* cands;  // [rows][runs][keep], best first, 0 past the last
};

template <typename T>
__device__ __forceinline__ float logit_at(const uint8_t* row, int i) {
  if constexpr (sizeof(T) == 2) return bf2f(reinterpret_cast<const uint16_t*>(row)[i]);
  else return reinterpret_cast<const float*>(row)[i];
}

// 16 bytes at a byte offset `Words` * 4 + (sh ? 2 : 0) into two aligned blocks.
template <int Words>
__device__ __forceinline__ uint4 shift16(const uint4& lo, const uint4& hi, uint32_t sh) {
  const uint32_t w[9] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w, 0};
  return make_uint4(__funnelshift_r(w[Words], w[Words + 1], sh), __funnelshift_r(w[Words + 1], w[Words + 2], sh),
                    __funnelshift_r(w[Words + 2], w[Words + 3], sh), __funnelshift_r(w[Words + 3], w[Words + 4], sh));
}

// Asks for n 16-byte blocks from p on to be brought into L2.
__device__ __forceinline__ void prefetch_l2(const uint4* p, int n) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(n * 16) : "memory");
}

// Logits come from the kernel ahead, which may run when this one starts: their
// loads keep their place behind the wait, which __ldg does not promise.
__device__ __forceinline__ uint4 ld_logits(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// N is 1 for lists of 32 (keep <= 32), 2 for lists of 64.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) beam_run_kernel(const BeamArgs<T> a) {
  constexpr int kVec = 16 / int(sizeof(T)), kLoads = kPer / kVec;
  constexpr int kCollect = kWarps * N * 32;
  __shared__ Key s_all[kCollect];  // logits that reach the bound
  constexpr int kHot = 256;
  __shared__ int s_hot[kHot];  // groups of 32 logits with one that reaches the bound
  __shared__ int s_count, s_hots;
  __shared__ double s_sum[kWarps];
  __shared__ float s_ref[kWarps];
  __shared__ float s_note[kMaxSteps][kThreads];  // the maximum of each lane's logits of each step
  __shared__ float s_max[kWarps][N * 32];
  __shared__ float s_bound;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int run = blockIdx.x, row = blockIdx.y;
  const int v0 = run * a.span, v1 = min(a.vocab, v0 + a.span);
  if (threadIdx.x == 0) s_count = s_hots = 0;
  pdl_trigger();
  pdl_wait();
  const float score = a.scores[row];
  if (!(score > -INFINITY) || (a.done && a.done[row])) return;  // no candidate of this row is looked at
  const uint8_t* base = reinterpret_cast<const uint8_t*>(a.logits + int64_t(row) * a.vocab);
  // A row may start anywhere.  16 logits' bytes come from the one or two aligned
  // blocks that hold them, so that lane and place of a logit depend on its id
  // alone and equal rows give equal sums.
  const uint32_t mis = uint32_t(reinterpret_cast<uintptr_t>(base)) & 15;
  const uint4* blocks = reinterpret_cast<const uint4*>(base - mis);
  const int last_block = int((mis + int64_t(a.vocab) * int(sizeof(T)) - 1) / 16);

  float ref = -INFINITY;
  double sum = 0.0;
  float most = -INFINITY;
  int step = 0;
  for (int t0 = v0 + warp * kStep; t0 < v1; t0 += kTile) {
    uint4 u[kLoads];
    const int blk = t0 / kVec + lane;
    // The step after next, on its way to L2.
    const int ahead = (t0 + 2 * kTile) / kVec;
    if (lane == 0 && t0 + 2 * kTile < v1) prefetch_l2(blocks + ahead, min(kStep / kVec, last_block + 1 - ahead));
    if (mis == 0) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) u[i] = ld_logits(blocks + min(blk + i * 32, last_block));
    } else {
      uint4 hi[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        u[i] = ld_logits(blocks + min(blk + i * 32, last_block));
        hi[i] = ld_logits(blocks + min(blk + i * 32 + 1, last_block));
      }
      const uint32_t sh = (mis & 2) * 8;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        switch (mis >> 2) {
          case 0: u[i] = shift16<0>(u[i], hi[i], sh); break;
          case 1: u[i] = shift16<1>(u[i], hi[i], sh); break;
          case 2: u[i] = shift16<2>(u[i], hi[i], sh); break;
          default: u[i] = shift16<3>(u[i], hi[i], sh); break;
        }
      }
    }
    auto id_of = [&](int i, int j) { return t0 + (i * 32 + lane) * kVec + j; };  // logit j of load i
    auto get = [&](int i, int j) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
      if constexpr (sizeof(T) == 2) return (j & 1) ? bf_hi(w[j / 2]) : bf_lo(w[j / 2]);
      else return __uint_as_float(w[j]);
    };
    if (t0 + kStep > v1) {  // the row's or run's end: -inf past it
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (id_of(i, j) >= v1) {
            if constexpr (sizeof(T) == 2) w[j / 2] = (j & 1) ? (w[j / 2] & 0xffffu) | 0xff800000u
                                                             : (w[j / 2] & 0xffff0000u) | 0xff80u;
            else w[j] = 0xff800000u;
          }
        u[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    float tm = -INFINITY;  // NaN is passed over
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int j = 0; j < kVec; j += 2) tm = fmax3(tm, get(i, j), get(i, j + 1));
    if (tm > ref + kLag || ref == -INFINITY) {
      if (ref != -INFINITY) sum = tm == INFINITY ? 0.0 : sum * exp(double(ref) - double(tm));
      ref = tm;
    }
    // ---- sum of exponentials ---------------------------------------------------
    {
      const uint64_t neg = pack_f2(-ref, -ref), scale = pack_f2(kLog2eF, kLog2eF);
      uint64_t quad[kPer / 8];
#pragma unroll
      for (int g = 0; g < kPer / 8; ++g) {
        uint64_t e[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int k = g * 8 + p * 2;
          float x0, x1;
          unpack_f2(mul_f2(add_f2(pack_f2(get(k / kVec, k % kVec), get(k / kVec, k % kVec + 1)), neg), scale), x0, x1);
          e[p] = pack_f2(ex2(x0), ex2(x1));
        }
        quad[g] = add_f2(add_f2(e[0], e[1]), add_f2(e[2], e[3]));
      }
      float p0, p1;
      unpack_f2(add_f2(add_f2(quad[0], quad[1]), add_f2(quad[2], quad[3])), p0, p1);
      float part = p0 + p1;
      if (part != part) {  // NaN logits, infinite ones, or nothing but -inf so far
        part = 0.0f;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const float x = get(i, j);
            if (x == ref && ref != -INFINITY) part += 1.0f;
            else if (x > -INFINITY && x < ref) part += ref == INFINITY ? 0.0f : ex2((x - ref) * kLog2eF);
            else if (x > ref && ref != -INFINITY) part += ex2((x - ref) * kLog2eF);
          }
      }
      sum += double(part);
    }
    s_note[step++][threadIdx.x] = tm;
    most = fmaxf(most, tm);
  }
  // ---- the bound: the keep-th largest of the lanes' maxima -----------------------
  float tops[N];
  tops[0] = most;
  if (N > 1) tops[N - 1] = -INFINITY;
#pragma unroll
  for (int block = 2; block <= 32; block *= 2)
#pragma unroll
    for (int stride = block / 2; stride > 0; stride /= 2) {
      const float o = __shfl_xor_sync(kAll, tops[0], stride);
      tops[0] = ((lane & stride) == 0) == ((lane & (block & 31)) == 0) ? fmaxf(tops[0], o) : fminf(tops[0], o);
    }
#pragma unroll
  for (int half = kWarps / 2; half > 0; half /= 2) {
    if (warp >= half && warp < 2 * half) {
#pragma unroll
      for (int j = 0; j < N; ++j) s_max[warp][j * 32 + lane] = tops[j];
    }
    __syncthreads();
    if (warp < half) {
#pragma unroll
      for (int j = 0; j < N; ++j) tops[j] = fmaxf(tops[j], s_max[warp + half][N * 32 - 1 - j * 32 - lane]);
      if (N > 1) {
        const float x = tops[0], y = tops[N - 1];
        tops[0] = fmaxf(x, y);
        tops[N - 1] = fminf(x, y);
      }
#pragma unroll
      for (int stride = 16; stride > 0; stride /= 2)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float o = __shfl_xor_sync(kAll, tops[j], stride);
          tops[j] = (lane & stride) == 0 ? fmaxf(tops[j], o) : fminf(tops[j], o);
        }
    }
  }
  if (warp == 0 && lane == (a.keep - 1) % 32) s_bound = tops[N > 1 && a.keep > 32 ? N - 1 : 0];
  __syncthreads();
  const float bound = s_bound;
  // ---- the logits that reach it ---------------------------------------------------
  // The hot groups of all warps, up to kHot; then a warp takes every 8th of
  // them, four at a time, and the block collects up to kCollect logits.
  auto group_id = [&](int g) {  // this lane's logit of group g = step * kThreads + thread
    const int s = g / kThreads, t = g % kThreads;
    return v0 + (s * kWarps + t / 32) * kStep + ((lane / kVec) * 32 + t % 32) * kVec + lane % kVec;
  };
  for (int s = 0; s < step; ++s) {
    const float note = s_note[s][threadIdx.x];
    if (note >= bound && note > -INFINITY) {
      const int at = atomicAdd(&s_hots, 1);
      if (at < kHot) s_hot[at] = s * kThreads + int(threadIdx.x);
    }
  }
  __syncthreads();
  const int hots = s_hots;
  if (hots <= kHot) {
    for (int g0 = warp; g0 < hots; g0 += 4 * kWarps) {
      float x[4];
      int id[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int g = g0 + q * kWarps;
        id[q] = g < hots ? group_id(s_hot[g]) : v1;
        x[q] = id[q] < v1 ? logit_at<T>(base, id[q]) : -INFINITY;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (x[q] >= bound && x[q] > -INFINITY) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kCollect) s_all[at] = Key{cand_key(x[q], uint32_t(id[q]))};
        }
    }
  }
  // ---- the block's sum and list ------------------------------------------------
  const float top = warp_max(ref);
  double part = ref == top || sum == 0.0 ? sum : top == INFINITY ? 0.0 : sum * exp(double(ref) - double(top));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(kAll, part, o);
  if (lane == 0) {
    s_sum[warp] = part;
    s_ref[warp] = top;
  }
  __syncthreads();
  const int count = hots <= kHot ? s_count : kCollect + 1;
  const int64_t place = int64_t(row) * a.runs + run;
  uint64_t* out = a.cands + place * a.keep;
  if (warp == 0) {
    const float own = s_ref[lane % kWarps], r = warp_max(own);
    double t = lane < kWarps ? s_sum[lane] : 0.0;
    if (own != r && t != 0.0) t = r == INFINITY ? 0.0 : t * exp(double(own) - double(r));
#pragma unroll
    for (int o = kWarps / 2; o > 0; o /= 2) t += __shfl_xor_sync(kAll, t, o);
    if (lane == 0) a.stats[place] = RunStat{t, r, 0};
  }
  if (count <= kCollect) {
    // A logit's place is the number of better ones.
    for (int i = int(threadIdx.x); i < max(count, a.keep); i += kThreads) {
      if (i < count) {
        const Key k = s_all[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += s_all[j].better(k);
        if (rank < a.keep) out[rank] = k.k;
      } else {
        out[i] = 0;
      }
    }
  } else {
    // Very many equal logits, or a bound far too low: each warp keeps a sorted
    // list of its own, and the lists are joined in pairs.
    Key list[N];
#pragma unroll
    for (int j = 0; j < N; ++j) list[j] = Key::none();
    Key worst = Key::none();  // list entry keep - 1
    int pending = 0;          // collected logits
    Key* mine = s_all + warp * N * 32;
    auto flush = [&]() {
      __syncwarp();
      Key fresh[N];
#pragma unroll
      for (int j = 0; j < N; ++j) fresh[j] = j * 32 + lane < pending ? mine[j * 32 + lane] : Key::none();
      sort_list(fresh);
      merge_list(list, fresh);
      worst = entry(list, a.keep - 1);
      pending = 0;
      __syncwarp();
    };
    for (int s = 0; s < step; ++s) {
      const float note = s_note[s][threadIdx.x];
      uint32_t hot = __ballot_sync(kAll, note >= bound && note > -INFINITY);
      while (hot) {
        const int h = __ffs(hot) - 1;
        hot &= hot - 1;
        const int id = group_id(s * kThreads + warp * 32 + h);
        const float x = id < v1 ? logit_at<T>(base, id) : -INFINITY;
        const Key k{cand_key(x, uint32_t(id))};
        const uint32_t takes = __ballot_sync(kAll, x >= bound && x > -INFINITY && k.better(worst));
        if (pending + __popc(takes) > N * 32) flush();
        if (takes >> lane & 1) mine[pending + __popc(takes & ((1u << lane) - 1))] = k;
        pending += __popc(takes);
      }
    }
    if (pending) flush();
#pragma unroll
    for (int half = kWarps / 2; half > 0; half /= 2) {
      __syncthreads();
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int j = 0; j < N; ++j) mine[j * 32 + lane] = list[j];
      }
      __syncthreads();
      if (warp < half) {
        Key other[N];
#pragma unroll
        for (int j = 0; j < N; ++j) other[j] = s_all[(warp + half) * N * 32 + j * 32 + lane];
        merge_list(list, other);
      }
    }
    if (warp != 0) return;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j * 32 + lane < a.keep) out[j * 32 + lane] = list[j].k;
  }
}

// One block per batch entry; a warp takes every 16th list (a run of a beam) and
// merges it, as scores, into a list of its own; the warps' lists are joined in
// pairs.
constexpr int kJoinWarps = 16;
template <typename T, int N>
__global__ void __launch_bounds__(kJoinWarps * 32) beam_join_kernel(const BeamArgs<T> a) {
  extern __shared__ __align__(16) uint8_t smem[];
  double* s_log = reinterpret_cast<double*>(smem);           // [beams] log of the row's sum
  float* s_ref = reinterpret_cast<float*>(s_log + a.beams);  // [beams]
  int* s_done = reinterpret_cast<int*>(s_ref + a.beams);     // [beams]
  __shared__ Scored s_list[kJoinWarps][N * 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const int lists = a.beams * a.runs;
  // The keys of list i, if it is one of a live beam.
  uint64_t keys[N];
  float score = -INFINITY;
  bool ended = false;
  auto fetch = [&](int i) {
    const int w = i / a.runs;
    const int64_t row = int64_t(b) * a.beams + w;
    score = a.scores[row];
    ended = a.done && a.done[row];
    const uint64_t* p = a.cands + (row * a.runs + i % a.runs) * a.keep;
#pragma unroll
    for (int j = 0; j < N; ++j) keys[j] = j * 32 + lane < a.keep ? p[j * 32 + lane] : 0;
  };
  if (warp < lists) fetch(warp);
  for (int w = threadIdx.x; w < a.beams; w += kJoinWarps * 32) {
    const int64_t row = int64_t(b) * a.beams + w;
    // All loads at once; a row that is not looked at leaves its statistics unwritten.
    const float sc = a.scores[row];
    const int dn = a.done ? a.done[row] : 0;
    const RunStat* st = a.stats + row * a.runs;
    RunStat s0 = st[0];
    float r = s0.ref;
    for (int k = 1; k < a.runs; ++k) r = fmaxf(r, st[k].ref);
    double sum = 0.0;
    if (sc > -INFINITY && !dn) {
      for (int k = 0; k < a.runs; ++k) {
        const RunStat s = k ? st[k] : s0;
        if (s.sum != 0.0) sum += s.ref == r ? s.sum : r == INFINITY ? 0.0 : s.sum * exp(double(s.ref) - double(r));
      }
    }
    s_ref[w] = r;
    s_log[w] = log(sum);
    s_done[w] = dn != 0;
  }
  __syncthreads();
  Scored list[N];
#pragma unroll
  for (int j = 0; j < N; ++j) list[j] = Scored::none();
  Scored worst = Scored::none();
  for (int i = warp; i < lists; i += kJoinWarps) {
    if (i != warp) fetch(i);
    const int w = i / a.runs;
    Scored fresh[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = j * 32 + lane;
      double v = -INFINITY;
      uint32_t token = ~uint32_t(keys[j]);
      if (ended) {
        if (e == 0 && i % a.runs == 0) v = double(score);  // an ended beam's one candidate
        token = uint32_t(max(a.eos, 0));
      } else if (score > -INFINITY && keys[j]) {
        const float x = unord32(uint32_t(keys[j] >> 32)), r = s_ref[w];
        v = double(score) + ((x == r ? 0.0 : double(x) - double(r)) - s_log[w]);
      }
      fresh[j] = v > -INFINITY ? Scored{ord64(v), uint64_t(w) << 32 | token} : Scored::none();
    }
    // In the order of its logits, so of its scores, unless scores that differ by
    // less than f64 resolves have become equal.
    bool off = false;
    Scored last = Scored::none();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Scored left = fresh[j].shfl((lane + 31) & 31);
      if (j > 0 && lane == 0) left = last;
      last = fresh[j].shfl(31);
      off |= (lane || j) && fresh[j].better(left);
    }
    if (__any_sync(kAll, off)) sort_list(fresh);
    if (!__any_sync(kAll, fresh[0].better(worst))) continue;  // its first entries are its best
    merge_list(list, fresh);
    worst = entry(list, a.keep - 1);
  }
#pragma unroll
  for (int half = kJoinWarps / 2; half > 0; half /= 2) {
    if (half >= lists) continue;
    if (warp >= half && warp < 2 * half) {
#pragma unroll
      for (int j = 0; j < N; ++j) s_list[warp][j * 32 + lane] = list[j];
    }
    __syncthreads();
    if (warp < half && warp + half < lists) {
      Scored other[N];
#pragma unroll
      for (int j = 0; j < N; ++j) other[j] = s_list[warp + half][j * 32 + lane];
      merge_list(list, other);
    }
  }
  if (warp != 0) return;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int e = j * 32 + lane;
    if (e >= a.keep) continue;
    const int64_t o = int64_t(b) * a.keep + e;
    const Scored c = list[j];
    if (c.score == 0) {
      a.out_scores[o] = -INFINITY;
      a.out_parent[o] = a.out_token[o] = -1;
      a.out_done[o] = 0;
      continue;
    }
    const int w = int(c.flat >> 32);
    const bool done = s_done[w];
    const int token = done ? a.eos : int(uint32_t(c.flat));
    a.out_scores[o] = float(unord64(c.score));
    a.out_parent[o] = b * a.beams + w;
    a.out_token[o] = token;
    a.out_done[o] = done || token == a.eos ? 1 : 0;
  }
}

// Blocks per row: enough for kRunsPerSm blocks on every SM, each with at least
// one tile and at most kMaxSteps.  3 against 2, 4 and 6: 128 rows of 128256 bf16 18.0 us
// (20.8, 18.0, 22.2), 512 rows of 128001 f32 52.9 (52.9, 58.8, 58.6), 300 rows of 50257 f32
// 25.1 (21.8, 25.1, 28.6), 512 rows of 128001 bf16 44.6 (44.7, 44.1, 43.8).
constexpr int kRunsPerSm = 3;
int beam_runs(int64_t rows, int64_t vocab) {
  const int64_t tiles = (vocab + kTile - 1) / kTile;
  int64_t runs = std::min((kRunsPerSm * kNumSMs + rows - 1) / rows, tiles);
  runs = std::max(runs, (tiles + kMaxSteps - 1) / kMaxSteps);
  const int64_t per = (tiles + runs - 1) / runs;
  return int((tiles + per - 1) / per);
}

constexpr uint64_t up256(uint64_t x) { return (x + 255) & ~uint64_t(255); }

template <typename T, int N>
int launch_beam(const BeamArgs<T>& a, int64_t batch, cudaStream_t st) {
  if (launch_pdl(beam_run_kernel<T, N>, dim3(unsigned(a.runs), unsigned(batch * a.beams)), dim3(kThreads), 0, st, a) !=
      cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  if (launch_pdl(beam_join_kernel<T, N>, dim3(unsigned(batch)), dim3(kJoinWarps * 32), size_t(a.beams) * 16, st, a) !=
      cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  return SB_OK;
}

}  // namespace

bool beam_select_supported(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
  return batch >= 0 && beams >= 1 && beams <= kBeamMaxBeams && vocab >= 1 && vocab <= (int64_t(1) << 30) &&
         keep >= 1 && keep <= kBeamMaxKeep && batch * beams <= 65535;
}

uint64_t beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
  if (!beam_select_supported(batch, beams, vocab, keep) || batch == 0) return 0;
  const uint64_t slots = uint64_t(batch * beams) * uint64_t(beam_runs(batch * beams, vocab));
  return up256(slots * sizeof(RunStat)) + up256(slots * uint64_t(keep) * sizeof(uint64_t));
}

template <typename T>
int launch_beam_select(const T* logits, const float* scores, const int32_t* done, int64_t batch, int64_t beams,
                       int64_t vocab, int64_t keep, int64_t eos, float* out_scores, int32_t* out_parent,
                       int32_t* out_token, int32_t* out_done, void* workspace, cudaStream_t st) {
  if (!beam_select_supported(batch, beams, vocab, keep)) return SB_INVALID_ARGUMENT;
  if (batch == 0) return SB_OK;
  const int64_t rows = batch * beams;
  const int runs = beam_runs(rows, vocab);
  const int64_t tiles = (vocab + kTile - 1) / kTile;
  BeamArgs<T> a{logits, scores, done, int(beams), int(keep), runs, int(vocab),
                int((tiles + runs - 1) / runs * kTile), int(eos), out_scores, out_parent, out_token, out_done,
                nullptr, nullptr};
  a.stats = static_cast<RunStat*>(workspace);
  a.cands = reinterpret_cast<uint64_t*>(static_cast<uint8_t*>(workspace) +
                                        up256(uint64_t(rows) * uint64_t(runs) * sizeof(RunStat)));
  return keep <= 32 ? launch_beam<T, 1>(a, batch, st) : launch_beam<T, 2>(a, batch, st);
}

template int launch_beam_select<uint16_t>(const uint16_t*, const float*, const int32_t*, int64_t, int64_t, int64_t,
                                          int64_t, int64_t, float*, int32_t*, int32_t*, int32_t*, void*,
                                          cudaStream_t);
template int launch_beam_select<float>(const float*, const float*, const int32_t*, int64_t, int64_t, int64_t, int64_t,
                                       int64_t, float*, int32_t*, int32_t*, int32_t*, void*, cudaStream_t);

}  // namespace sb

// Upkeep of KV caches when a sequence has several continuations: keeping the
// rows of an accepted branch (kv_accept), giving every row of a block table a
// new parent (kv_fork: shares full pages, copies partly filled ones, frees
// what is no longer named) and moving the used pages of a pool together
// (kv_compact).
//
// All three move whole 16-byte pieces and compute nothing on them, so they
// are exact in any element type; what bounds them is HBM (every moved byte is
// read once and written once) or, for a few rows, latency.  Measured, device time
// back to back in a graph: accepting one sequence's path in 64 caches 2.8 us (the
// host's launch takes 9), 32 paths of up to 33 nodes in 160 pools 17.5 us; forking 4
// rows of 64 pools 11.5 us, most of it the plan's chain of dependent reads; 128 rows of
// 32 pools 47 us, the copies alone (220 MB) 41 us with nothing cached, 5.4 TB/s;
// compacting 3000 pages of 32 pools 241 us, the copies 238 us, 6.0 TB/s.
//
// What these kernels write, the decode attention may read before its wait (rows
// below a position, the block table, positions).  So no later kernel may start
// before it is written: the last kernel of each operator does not trigger its
// dependents, which then start when it has ended, and its writes are fenced, since the
// end of a kernel is not yet the end of its writes for one that starts early.  And nothing that a kernel ahead
// may write is read through const __restrict__ or __ldg here: either says that the
// data stays as it is while the kernel runs, so the compiler may move such a load
// above the wait.  (Block tables are: only the planning kernels write them.)
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "k_branch.cuh"

namespace sb {

namespace {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------
// kv_accept
// ---------------------------------------------------------------------------
constexpr int kAcThreads = 256;
constexpr int kAcBatch = 8;  // rows in flight per thread

// Row base + path[i] -> row base + i of every cache, i < n.  A block works for
// one sequence; a thread owns one 16-byte column of one (cache, kv head) and
// takes the path's rows in order, eight at a time: path is strictly
// increasing, so path[i] >= i and the rows written by earlier groups lie
// below every row a later group reads.  The moves with path[i] == i are a
// prefix of the path and are skipped.
__global__ void __launch_bounds__(kAcThreads)
    kv_accept_kernel(const __grid_constant__ KvPools pools, int n_caches, int chunks, const int32_t* base,
                     const int32_t* path, const int32_t* n_path, int kv_heads, int max_len, int max_path, KvPages kp,
                     int* err) {
  __shared__ int64_t s_src[kTreeMaxTokens], s_dst[kTreeMaxTokens];
  __shared__ int s_first;
  pdl_wait();  // no trigger: later kernels may read the rows before their own wait
  const int b = blockIdx.y;
  const int p0 = base[b], n = n_path[b];
  if (threadIdx.x == 0) s_first = n;
  __syncthreads();
  int bad = n < 0 || n > max_path || p0 < 0 || p0 > max_len ? kBadPosition : 0;
  if (!bad) {
    for (int i = threadIdx.x; i < n; i += kAcThreads) {
      const int x = path[int64_t(b) * max_path + i];
      const int prev = i ? path[int64_t(b) * max_path + i - 1] : -1;
      if (x <= prev || x < 0 || x >= max_len - p0) {
        bad = kBadPosition;
        continue;
      }
      const int64_t src = kv_row(kp, b, 0, kv_heads, max_len, p0 + x), dst = kv_row(kp, b, 0, kv_heads, max_len, p0 + i);
      if (src < 0 || dst < 0) bad = max(bad, kBadPage);
      s_src[i] = src;
      s_dst[i] = dst;
      if (x != i) atomicMin(&s_first, i);
    }
  }
  if (__syncthreads_or(bad)) {  // nothing of this sequence moves
    if (bad && err && blockIdx.x == 0) atomicExch(err, bad);
    return;
  }
  const int first = s_first;
  const int64_t u = int64_t(blockIdx.x) * kAcThreads + threadIdx.x;
  const int c = int(u % chunks);
  const int64_t ch = u / chunks;
  const int h = int(ch % kv_heads);
  const int64_t cache = ch / kv_heads;
  const bool on = cache < n_caches;  // the last block may reach past the last cache
  const int64_t head_rows = int64_t(h) * (kp.paged() ? kp.page_size : max_len);
  uint4* at = static_cast<uint4*>(pools.p[on ? cache : 0]) + head_rows * chunks + c;
  for (int i0 = on ? first : n; i0 < n; i0 += kAcBatch) {
    uint4 v[kAcBatch];
#pragma unroll
    for (int j = 0; j < kAcBatch; ++j)
      if (i0 + j < n) v[j] = at[s_src[i0 + j] * chunks];
#pragma unroll
    for (int j = 0; j < kAcBatch; ++j)
      if (i0 + j < n) at[s_dst[i0 + j] * chunks] = v[j];
  }
  // One fence for the block's rows; by each thread it cost another 1.1 us of 17.6 (32 paths, 160 pools).
  __syncthreads();
  if (threadIdx.x == 0) __threadfence();
}

// ---------------------------------------------------------------------------
// Page copies
// ---------------------------------------------------------------------------
constexpr int kCpThreads = 256;
constexpr int kPiece = 256;  // 16-byte pieces a warp moves at once (4 KB): eight loads in flight per lane

struct PageCopy {
  int src, dst, rows, pad;
};

// Copies the first `rows` rows of every kv head of page src to page dst, in
// every pool, for the n copies a planning kernel listed.  A page is
// [kv_heads, page_size, row]; a warp moves up to 4 KB of one head's rows.
__global__ void __launch_bounds__(kCpThreads)
    page_copy_kernel(const __grid_constant__ KvPools pools, int n_pools, int kv_heads, int page_size, int chunks,
                     const PageCopy* list, const int* n_list) {
  pdl_wait();  // no trigger: later kernels may read the pages, and what the plan wrote, before their own wait
  const int lane = threadIdx.x & 31;
  const uint32_t pieces = uint32_t(page_size * chunks + kPiece - 1) / kPiece;
  const uint32_t per = uint32_t(n_pools) * uint32_t(kv_heads) * pieces;  // below 2^31 (launcher)
  const uint32_t warps = gridDim.x * (kCpThreads / 32), first = blockIdx.x * (kCpThreads / 32) + (threadIdx.x >> 5);
  // (copy, unit within it), carried along instead of divided out: with all copies
  // together a unit's number may pass 32 bits.
  uint32_t copy = first / per, in = first - copy * per;
  const uint32_t step_copy = warps / per, step_in = warps - step_copy * per;
  uint32_t copies;  // by a load that keeps its place behind the wait: the entries below it are then written, too
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(copies) : "l"(n_list) : "memory");
  for (; copy < copies; copy += step_copy, in += step_in, copy += in >= per, in -= in >= per ? per : 0) {
    const PageCopy cp = list[copy];
    const uint32_t hp = in / pieces;
    const int piece = int(in - hp * pieces), pool = int(hp / uint32_t(kv_heads)), h = int(hp) - pool * kv_heads;
    const int end = cp.rows * chunks, c0 = piece * kPiece;
    if (c0 >= end) continue;
    uint4* p = static_cast<uint4*>(pools.p[pool]);
    const int64_t head = int64_t(page_size) * chunks;
    const uint4* src = p + (int64_t(cp.src) * kv_heads + h) * head + c0 + lane;
    uint4* dst = p + (int64_t(cp.dst) * kv_heads + h) * head + c0 + lane;
    uint4 v[kPiece / 32];
#pragma unroll
    for (int j = 0; j < kPiece / 32; ++j)
      if (c0 + j * 32 + lane < end) v[j] = src[j * 32];
#pragma unroll
    for (int j = 0; j < kPiece / 32; ++j)
      if (c0 + j * 32 + lane < end) dst[j * 32] = v[j];
  }
  __threadfence();
}

// ---------------------------------------------------------------------------
// Planning, by one thread-block cluster
// ---------------------------------------------------------------------------
constexpr int kPlThreads = 1024;
constexpr int kPlMaxCluster = 8;
static_assert(kPlThreads * kPlMaxCluster <= kPlanStep, "indexes of table entries stay below 2^31");
constexpr int kPlItems = 4 * kPlThreads;  // table entries and pages that one block plans alone

// Division of numbers below 2^31 by a fixed positive one: floor(n m / 2^(31 + s))
// with m = ceil(2^(31 + s) / d) and 2^s >= d (Granlund and Montgomery 1994).
struct FastDiv {
  uint32_t m = 0;
  int s = 0, d = 1;
  FastDiv() = default;
  explicit FastDiv(int div) : d(div) {
    while ((int64_t(1) << s) < div) ++s;
    m = uint32_t(((uint64_t(1) << (31 + s)) + unsigned(div) - 1) / unsigned(div));
  }
  __device__ __forceinline__ int div(int n) const { return int(uint64_t(uint32_t(n)) * m >> (31 + s)); }
};

// Exclusive prefix sum over the block's threads; *total gets the sum.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* warp_sums, T* total) {
  static_assert(kPlThreads == 1024, "one warp adds up the warps' sums");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = v;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    T s = warp_sums[lane];
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  *total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

struct ForkArgs {
  const int32_t *table_in, *lens_in, *refs_in, *parents;
  int32_t *table_out, *lens_out, *refs_out, *report;
  int rows, per, page_shift, num_pages, reserve;
  bool copies_follow;  // the copying kernel is launched behind the plan
  FastDiv by_per;
  // workspace; the first four in shared memory where one block plans
  int *left, *cand, *free_list, *row_off;
  PageCopy* copies;
  int* n_copies;
};

constexpr int kNobody = 0x7fffffff;

// What row r becomes: its new length, full pages, pages it needs and its
// parent's row of the old table.
struct ForkRow {
  int parent, len, full, part, need;
  bool bad;
};

__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int r) {
  ForkRow f{a.parents[r], 0, 0, 0, 0, false};
  if (f.parent < -1 || f.parent >= a.rows) {
    f.bad = true;
    f.parent = -1;
  }
  if (f.parent < 0) return f;
  f.len = a.lens_in[f.parent];
  const int most = a.per << a.page_shift;  // below 2^31
  if (f.len < 0 || f.len > most || a.reserve > most - f.len) {
    f.bad = true;
    f.len = 0;
    f.parent = -1;
    return f;
  }
  f.full = f.len >> a.page_shift;
  f.part = f.len - (f.full << a.page_shift);
  f.need = int((uint32_t(f.len + a.reserve) + (1u << a.page_shift) - 1) >> a.page_shift);
  return f;
}

// One cluster plans the whole call.  left[g] counts the references to page g
// that remain when the old table lets go and every row has taken its parent's
// full pages, first the one and then the other; integer atomics, so the order of
// the threads does not matter.
// A partly filled page with left[g] == 0 stays with the lowest row that wants
// it (cand[g]), everyone else gets a copy.  A page is free when nobody holds
// or wants it; the free pages are dealt out in ascending order to the rows in
// ascending order.  When something is wrong or the pool is short, the outputs
// are the inputs and nothing is copied.
__global__ void __launch_bounds__(kPlThreads) kv_fork_plan_kernel(const __grid_constant__ ForkArgs args) {
  extern __shared__ int s_plan[];
  cg::cluster_group cluster = cg::this_cluster();
  const int nranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = rank * kPlThreads + threadIdx.x, nthreads = nranks * kPlThreads;
  __shared__ long long s_warp[32];
  __shared__ int s_err, s_low, s_free;
  ForkArgs a = args;
  if (nranks == 1) {
    a.left = s_plan;
    a.cand = a.left + a.num_pages;
    a.free_list = a.cand + a.num_pages;
    a.row_off = a.free_list + a.num_pages;
  }
  if (threadIdx.x == 0) {
    s_err = 0;
    s_low = 0;
  }
  if (a.copies_follow) pdl_trigger();
  pdl_wait();
#pragma unroll 1
  for (int g = tid; g < a.num_pages; g += nthreads) {
    a.left[g] = a.refs_in[g];
    a.cand[g] = kNobody;
  }
  cluster.sync();
  int err = 0;
  const int entries = a.rows * a.per;
  // The old table lets go of everything before the new one takes anything: a count
  // below the old references would not show among the new ones.
#pragma unroll 1
  for (int e = tid; e < entries; e += nthreads) {
    const int old = a.table_in[e];
    if (old >= a.num_pages) err = max(err, kBadPage);
    else if (old >= 0 && atomicSub(&a.left[old], 1) <= 0) err = max(err, kBadRefs);
  }
  cluster.sync();
#pragma unroll 1
  for (int e = tid; e < entries; e += nthreads) {
    const int r = a.by_per.div(e), i = e - r * a.per;
    const ForkRow f = fork_row(a, r);
    if (f.bad) err = max(err, kBadPosition);
    if (f.parent < 0 || i > f.full || (i == f.full && !f.part)) continue;
    const int mine = a.table_in[f.parent * a.per + i];
    if (mine < 0 || mine >= a.num_pages) err = max(err, kBadPage);
    else if (i < f.full) atomicAdd(&a.left[mine], 1);
    else atomicMin(&a.cand[mine], r);
  }
  if (err) atomicMax(&s_err, err);
  cluster.sync();
  err = 0;
#pragma unroll 1
  for (int k = 0; k < nranks; ++k) err = max(err, *cluster.map_shared_rank(&s_err, k));
  // Pages each row takes from the free list, and which rows copy: every block
  // scans all rows for itself, block 0 writes the offsets down.
  int total = 0, copies = 0;
#pragma unroll 1
  for (int r0 = 0; r0 < a.rows; r0 += kPlThreads) {
    const int r = r0 + threadIdx.x;
    int take = 0, copy = 0, tail = -1;
    ForkRow f{-1, 0, 0, 0, 0, false};
    if (!err && r < a.rows) {
      f = fork_row(a, r);
      if (f.parent >= 0) {
        bool keep = false;
        if (f.part) {
          tail = a.table_in[f.parent * a.per + f.full];
          keep = a.left[tail] == 0 && a.cand[tail] == r;
          copy = !keep;
        }
        take = f.need - f.full - (keep ? 1 : 0);
      }
    }
    // Both sums in one scan: a block's rows copy at most 1024 pages.
    long long sum;
    const long long both = block_scan(static_cast<long long>(take) << 16 | copy, s_warp, &sum);
    const int off = total + int(both >> 16), at = copies + int(both & 0xffff);
    total += int(sum >> 16);
    copies += int(sum & 0xffff);
    if (rank == 0 && r < a.rows) {
      a.row_off[r] = off;
      if (copy) a.copies[at] = PageCopy{tail, -1, f.part, r};
    }
  }
  // Free pages: every block counts its run of pages, then numbers them.
  const int slice = (a.num_pages + nranks - 1) / nranks;
  const int run = (slice + kPlThreads - 1) / kPlThreads;
  const int g0 = min(rank * slice + int(threadIdx.x) * run, min(a.num_pages, (rank + 1) * slice));
  const int g1 = min(g0 + run, min(a.num_pages, (rank + 1) * slice));
  int mine = 0;
  bool low = false;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    const int l = a.left[g];
    mine += l == 0 && a.cand[g] == kNobody;
    low |= l < 0;
  }
  long long sum;
  const int before = int(block_scan(static_cast<long long>(mine), s_warp, &sum));
  if (threadIdx.x == 0) s_free = int(sum);
  if (low) s_low = kBadRefs;
  cluster.sync();
  int free_pages = 0, ahead = 0;
#pragma unroll 1
  for (int k = 0; k < nranks; ++k) {
    err = max(err, *cluster.map_shared_rank(&s_low, k));
    const int f = *cluster.map_shared_rank(&s_free, k);
    free_pages += f;
    if (k < rank) ahead += f;
  }
  if (!err && total > free_pages) err = kNoPages;
  int nth = ahead + before;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    int refs = a.refs_in[g];
    if (!err) {
      refs = a.left[g];
      if (refs == 0) {
        if (a.cand[g] != kNobody) {
          refs = 1;  // the lowest row keeps it
        } else if (nth < total) {
          a.free_list[nth] = g;
          refs = 1;
          ++nth;
        } else {
          ++nth;
        }
      }
    }
    a.refs_out[g] = refs;
  }
  cluster.sync();
#pragma unroll 1
  for (int e = tid; e < entries; e += nthreads) {
    const int r = a.by_per.div(e), i = e - r * a.per;
    int v = a.table_in[e];
    if (!err) {
      const ForkRow f = fork_row(a, r);
      const int got = f.parent >= 0 ? a.table_in[f.parent * a.per + i] : -1;
      v = -1;
      if (f.parent >= 0 && i < f.need) {
        bool keep = false;
        if (f.part) {
          const int tail = i == f.full ? got : a.table_in[f.parent * a.per + f.full];
          keep = a.left[tail] == 0 && a.cand[tail] == r;
        }
        if (i < f.full || (keep && i == f.full)) v = got;
        else v = a.free_list[a.row_off[r] + i - f.full - (keep ? 1 : 0)];
      }
    }
    a.table_out[e] = v;
  }
#pragma unroll 1
  for (int r = tid; r < a.rows; r += nthreads) a.lens_out[r] = err ? a.lens_in[r] : fork_row(a, r).len;
  if (!err)
#pragma unroll 1
    for (int k = tid; k < copies; k += nthreads) a.copies[k].dst = a.free_list[a.row_off[a.copies[k].pad]];
  if (tid == 0) {
    *a.n_copies = err ? 0 : copies;
    a.report[0] = err;
    a.report[1] = err ? 0 : copies;
    a.report[2] = err ? 0 : total - copies;
    a.report[3] = err == kNoPages ? total - free_pages : err ? 0 : free_pages - total;
  }
  __threadfence();
  cluster.sync();  // no block leaves while another may still read its shared memory
}

struct CompactArgs {
  const int32_t *table_in, *refs_in;
  int32_t *table_out, *refs_out, *remap, *report;
  int rows, per, page_size, num_pages;
  bool copies_follow;  // as in ForkArgs
  int* holes;
  PageCopy* copies;
  int* n_copies;
};

// n pages are used; the i-th used page with an id of n or more moves into the
// i-th free page below n.  Both numberings come from one prefix sum over
// "used": free pages before g are g - used(before g), and used pages from n on
// are used(before g) - used(before n).
__global__ void __launch_bounds__(kPlThreads) kv_compact_plan_kernel(const CompactArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int nranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = rank * kPlThreads + threadIdx.x, nthreads = nranks * kPlThreads;
  __shared__ int s_warp[32], s_used, s_low, s_err;
  if (threadIdx.x == 0) {
    s_low = 0;
    s_err = 0;
  }
  if (a.copies_follow) pdl_trigger();
  pdl_wait();
  const int slice = (a.num_pages + nranks - 1) / nranks;
  const int run = (slice + kPlThreads - 1) / kPlThreads;
  const int g0 = min(rank * slice + int(threadIdx.x) * run, min(a.num_pages, (rank + 1) * slice));
  const int g1 = min(g0 + run, min(a.num_pages, (rank + 1) * slice));
  int mine = 0;
  bool bad = false;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    const int c = a.refs_in[g];
    mine += c > 0;
    bad |= c < 0;
  }
  int sum;
  int before = block_scan(mine, s_warp, &sum);
  if (threadIdx.x == 0) s_used = sum;
  if (bad) atomicMax(&s_err, kBadRefs);
  const int entries = a.rows * a.per;
#pragma unroll 1
  for (int e = tid; e < entries; e += nthreads) {
    const int g = a.table_in[e];
    if (g >= a.num_pages) atomicMax(&s_err, kBadPage);
    else if (g >= 0 && a.refs_in[g] <= 0) atomicMax(&s_err, kBadRefs);
  }
  cluster.sync();
  int n = 0, err = 0;
#pragma unroll 1
  for (int k = 0; k < nranks; ++k) {
    const int u = *cluster.map_shared_rank(&s_used, k);
    n += u;
    if (k < rank) before += u;
    err = max(err, *cluster.map_shared_rank(&s_err, k));
  }
  // used(before n), found by the thread whose run holds page n (none does
  // when every page is used: then nothing moves).
  int used = before;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    const bool u = a.refs_in[g] > 0;
    if (g == n) s_low = used;
    if (!err && !u && g < n) a.holes[g - used] = g;
    used += u;
  }
  cluster.sync();
  int low = 0;
#pragma unroll 1
  for (int k = 0; k < nranks; ++k) low += *cluster.map_shared_rank(&s_low, k);
  if (n == a.num_pages) low = n;
  const int moves = err ? 0 : n - low;
  used = before;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    const int c = a.refs_in[g];
    const bool u = c > 0;
    int to = u ? g : -1;
    if (err) {
      a.refs_out[g] = c;
      to = g;
    } else if (g < n) {
      if (u) a.refs_out[g] = c;
    } else {
      a.refs_out[g] = 0;
      if (u) {
        to = a.holes[used - low];
        a.refs_out[to] = c;
        a.copies[used - low] = PageCopy{g, to, a.page_size, 0};
      }
    }
    a.remap[g] = to;
    used += u;
  }
  cluster.sync();
#pragma unroll 1
  for (int e = tid; e < entries; e += nthreads) {
    const int g = a.table_in[e];
    a.table_out[e] = err ? g : g < 0 ? -1 : a.remap[g];
  }
  if (tid == 0) {
    *a.n_copies = moves;
    a.report[0] = err;
    a.report[1] = err ? 0 : n;
    a.report[2] = moves;
    a.report[3] = err ? 0 : a.num_pages - n;
  }
  __threadfence();
  cluster.sync();
}

template <typename Args>
int launch_plan(void (*kern)(Args), const Args& a, int64_t items, size_t shared, cudaStream_t st) {
  // One block up to kPlItems: its barriers cost a tenth of a cluster's, and what it
  // notes per page lies in shared memory.  Then as many blocks as give each that many.
  int blocks = 1;
  while (blocks < kPlMaxCluster && int64_t(blocks) * kPlItems < items) blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(kPlThreads);
  cfg.dynamicSmemBytes = blocks == 1 ? shared : 0;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = unsigned(blocks);
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) return SB_INTERNAL;
  count_launch();
  return SB_OK;
}

// What warps share out of one copied page; the copying kernel counts it in 31 bits.
int64_t units_per_copy(int64_t n_pools, int64_t row_bytes, int64_t kv_heads, int64_t page_size) {
  return n_pools * kv_heads * ((page_size * (row_bytes / 16) + kPiece - 1) / kPiece);
}

int launch_copies(const KvPools& pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads, int64_t page_size,
                  int64_t most, const PageCopy* list, const int* n_list, cudaStream_t st) {
  const int chunks = int(row_bytes / 16);
  const int64_t units = most * units_per_copy(n_pools, row_bytes, kv_heads, page_size);
  const int64_t blocks = std::min<int64_t>((units + kCpThreads / 32 - 1) / (kCpThreads / 32), int64_t(kNumSMs) * 8);
  if (launch_pdl(page_copy_kernel, dim3(unsigned(std::max<int64_t>(blocks, 1))), dim3(kCpThreads), 0, st, pools,
                 int(n_pools), int(kv_heads), int(page_size), chunks, list, n_list) != cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  return SB_OK;
}

constexpr uint64_t up256(uint64_t x) { return (x + 255) & ~uint64_t(255); }

// Carves typed pieces out of a workspace, 256-byte aligned.
struct Carve {
  uint8_t* p;
  template <typename T>
  T* take(uint64_t n) {
    T* r = reinterpret_cast<T*>(p);
    p += up256(n * sizeof(T));
    return r;
  }
};

}  // namespace

int launch_kv_accept(const KvPools& caches, int64_t n_caches, int64_t row_bytes, const int32_t* base,
                     const int32_t* path, const int32_t* n_path, int64_t batch, int64_t kv_heads, int64_t max_len,
                     int64_t max_path, const KvPages& kp, int* err, cudaStream_t st) {
  if (batch == 0 || n_caches == 0) return SB_OK;
  const int chunks = int(row_bytes / 16);
  const int64_t units = n_caches * kv_heads * chunks;
  const int64_t blocks = (units + kAcThreads - 1) / kAcThreads;
  if (blocks > INT32_MAX || batch > 65535) return SB_INVALID_ARGUMENT;
  if (launch_pdl(kv_accept_kernel, dim3(unsigned(blocks), unsigned(batch)), dim3(kAcThreads), 0, st, caches,
                 int(n_caches), chunks, base, path, n_path, int(kv_heads), int(max_len), int(max_path), kp,
                 err) != cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  return SB_OK;
}

uint64_t kv_fork_workspace_bytes(int64_t rows, int64_t pages_per_seq, int64_t num_pages) {
  (void)pages_per_seq;
  return 3 * up256(uint64_t(num_pages) * 4) + up256(uint64_t(rows) * 4) + up256(uint64_t(rows) * sizeof(PageCopy)) +
         256;
}

int launch_kv_fork(const KvPools& pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads, int64_t page_size,
                   int64_t num_pages, const int32_t* table_in, const int32_t* lens_in, const int32_t* refs_in,
                   const int32_t* parents, int64_t rows, int64_t pages_per_seq, int64_t reserve, int32_t* table_out,
                   int32_t* lens_out, int32_t* refs_out, int32_t* report, void* workspace, cudaStream_t st) {
  if (units_per_copy(n_pools, row_bytes, kv_heads, page_size) > INT32_MAX) return SB_INVALID_ARGUMENT;
  ForkArgs a{table_in, lens_in, refs_in, parents, table_out, lens_out, refs_out, report, int(rows),
             int(pages_per_seq), __builtin_ctz(unsigned(page_size)), int(num_pages), int(reserve),
             n_pools > 0, FastDiv(int(pages_per_seq)), nullptr, nullptr, nullptr, nullptr,
             nullptr, nullptr};
  Carve w{static_cast<uint8_t*>(workspace)};
  a.left = w.take<int>(uint64_t(num_pages));
  a.cand = w.take<int>(uint64_t(num_pages));
  a.free_list = w.take<int>(uint64_t(num_pages));
  a.row_off = w.take<int>(uint64_t(rows));
  a.copies = w.take<PageCopy>(uint64_t(rows));
  a.n_copies = w.take<int>(1);
  // The pages and rows of a call that one block plans are at most kPlItems together.
  static PerDeviceOnce configured;
  if (!configured.run([] {
        return cudaFuncSetAttribute(kv_fork_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    3 * kPlItems * 4) == cudaSuccess;
      }))
    return SB_INTERNAL;
  const int rc = launch_plan(kv_fork_plan_kernel, a, rows * pages_per_seq + num_pages,
                             size_t(3 * num_pages + rows) * 4, st);
  if (rc || n_pools == 0) return rc;
  return launch_copies(pools, n_pools, row_bytes, kv_heads, page_size, rows, a.copies, a.n_copies, st);
}

uint64_t kv_compact_workspace_bytes(int64_t num_pages) {
  return up256(uint64_t(num_pages) * 4) + up256(uint64_t(num_pages) * sizeof(PageCopy)) + 256;
}

int launch_kv_compact(const KvPools& pools, int64_t n_pools, int64_t row_bytes, int64_t kv_heads, int64_t page_size,
                      int64_t num_pages, const int32_t* table_in, const int32_t* refs_in, int64_t rows,
                      int64_t pages_per_seq, int32_t* table_out, int32_t* refs_out, int32_t* remap, int32_t* report,
                      void* workspace, cudaStream_t st) {
  if (units_per_copy(n_pools, row_bytes, kv_heads, page_size) > INT32_MAX) return SB_INVALID_ARGUMENT;
  CompactArgs a{table_in, refs_in, table_out, refs_out, remap, report, int(rows), int(pages_per_seq),
                int(page_size), int(num_pages), n_pools > 0, nullptr, nullptr, nullptr};
  Carve w{static_cast<uint8_t*>(workspace)};
  a.holes = w.take<int>(uint64_t(num_pages));
  a.copies = w.take<PageCopy>(uint64_t(num_pages));
  a.n_copies = w.take<int>(1);
  const int rc = launch_plan(kv_compact_plan_kernel, a, rows * pages_per_seq + num_pages, 0, st);
  if (rc || n_pools == 0) return rc;
  return launch_copies(pools, n_pools, row_bytes, kv_heads, page_size, num_pages / 2 + 1, a.copies, a.n_copies, st);
}

}  // namespace sb

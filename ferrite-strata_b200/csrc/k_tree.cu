// Attention of a tree of drafted tokens over a cached prompt, on the
// 5th-generation tensor cores (tcgen05, TMEM, TMA): bf16, head_dim 64 or 128.
//
// Sequence b has base[b] cached positions and count[b] live nodes.  Node i's k
// and v rows are appended at position base + i, and node t attends to every
// position below base and to the nodes whose bit is set in its mask row:
//   o[t, h] = sum_p softmax_p(q[t, h] . k[p] / sqrt d) v[p]
// A node at or past count, and one that sees nothing, gives zeros.
//
// Work.  The query rows of one (sequence, kv head) are its nodes times the
// group's heads (row = node * G + head), so a kv head's cache is read once for
// all of them.  An item is 128 such rows (up to 256 when there are more than
// 128), and its KV is a list of 128-position tiles: the cached positions, read
// from the cache or its pages, then the nodes, read from k_new and v_new
// directly (so nothing waits for the append, which a warp of its own does while
// the first tiles are on their way).  All items are numbered in one line and each
// block takes an equal run of it, whatever the sequences' lengths; an item cut by
// a block's end leaves (max, sum, O) of each part in the workspace and a second
// kernel joins the parts in order, so results do not depend on timing.
//
// What bounds it (heads of 128 on 8 kv heads, 4096 positions, 32 sequences; 148
// blocks).  Up to 128 rows a kv head, reading the cache: a tile of K and V takes
// 1.45 us a block, 6.6 TB/s, the rate of a plain stream of the same copies; 128 rows,
// contiguous, 108 us, 5.1 TB/s over the call: 4 us to the first products, 5 us for each
// further item, 4 us for the last output and 4 us for the join stand beside it.
// 16-row pages, eight boxes a tile, 116 us.  With 256 rows, the chain S, softmax,
// P V of each group: 2.7 us a tile, 880 TFLOP/s (158 us); the two products alone
// would take 1.1 us and the exponentials as long, and neither is the limit.
//
// Block.  Warp 0 walks the block's run and loads by TMA through one ring of
// 128-row tiles in the order they are used (K0, K1, V0, K2, V1, ...); a thread of
// warp 1 issues the products
//   S = Q K^T    (A, B in shared memory; 128 x 128 f32 in TMEM)
//   O += P V     (A = P in TMEM, written over S; B = the V tile as loaded)
// warp 2 appends the new rows, warp 3 cleans V tiles (below), and warps 4-11 and
// 12-19 are two softmax groups: two threads per query row, 64 positions each (the
// step from one thread and 128 positions, with the walk and the append moved to warps
// of their own, took 32 x 32 nodes from 218 to 171 us).  With more than 128 rows
// the two groups take a query tile each and share every KV tile; with up to 128
// rows both work for the same query tile, one on the even and one on the odd KV
// tiles (each with a maximum, sum and O of its own, joined at the end), so that
// one group's softmax runs during the other's products.
//
// Softmax in base 2: a row's reference moves, and O is rescaled in TMEM, only
// when a score exceeds the reference by more than 8, so probabilities stay
// below 2^8.  The two threads of a row agree by one barrier vote per tile that
// nothing moves; only when something does they exchange their maxima.  P is
// rounded to bf16 for the second product, whose operands have to be of V's type
// (f32 terms would take a second product for what the rounding leaves); each
// probability is then off by at most 2^-8, which for values without a common sign
// adds as much error as rounding the output does.  Reference, sum and O are f32.
//
// Masked places.  A masked score becomes -inf whatever it was.  0 * NaN must
// not reach O either: V rows at or past a tile's end are zeroed in shared
// memory, and so are non-finite values of a node's v; the rows that do see
// such a node get its non-finite values added to their output.  Warp 3 does this
// as soon as such a tile has arrived.
//
// Every wait is bounded; one that runs out sets error word 4 and the block
// winds down (loads land, products finish, TMEM is freed).
#include <algorithm>

#include "common.cuh"
#include "k_branch.cuh"
#include "k_tc.cuh"

namespace sb {

namespace {

using namespace tc;

constexpr int kTile = 128;   // query rows per tile, positions per KV tile
constexpr int kHalf = 64;    // positions per softmax thread
constexpr int kThreads = 640;
constexpr int kStart = 2;    // what starting an item costs, in tiles (see the walk)
constexpr int kSegs = 4;     // segments the walking warp is ahead at most, rounded up
constexpr uint32_t kTmemCols = 512;  // S_0, S_1 (128 columns each), O_0, O_1 (head_dim each)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.0f;  // log2 of the largest P before O is rescaled

struct Seq {
  int base, count;  // count 0 where the sequence is unusable or has no nodes
  int prefix;       // tiles of cached positions
  int nt;           // all tiles
  int pairs;        // items per kv head
};

// A block's stretch of one item: tiles [j0, j1) of nt.
struct Seg {
  Seq s;
  int b, kvh, pair, j0, j1;
  int last;  // the block's last one
};

// Shared memory: the item's query tile (two when wide), the ring, the softmax
// threads' statistics, the next segments, the barriers.
template <int D, bool Wide>
struct Lay {
  static constexpr int kKB = D / 64;              // 64-wide blocks of head_dim
  static constexpr int kBytesTile = 128 * D * 2;  // a query tile: kKB blocks of [128 rows][128 bytes]
  static constexpr int kGroup = kKB * 1024;       // a K or V tile: 16 groups of kKB blocks of [8 rows][128 bytes]
  static constexpr int kSlots = D == 128 ? (Wide ? 5 : 6) : (Wide ? 11 : 12);
  static constexpr int kQ = 0;
  static constexpr int kRing = (Wide ? 2 : 1) * kBytesTile;
  static constexpr int kStat = kRing + kSlots * kBytesTile;  // [2 groups][128]: sum and reference, or each half's sum (wide)
  static constexpr int kSeg = kStat + 4 * 128 * 4;
  static constexpr int kBar = kSeg + kSegs * int(sizeof(Seg));
  static constexpr int kBars = 3 * kSlots + 12 + kSegs;
  static constexpr int kUse = kBar + kBars * 8 + 8 + 20;  // and the TMEM address, the failure word, four notes
  static constexpr int kBytes = kUse + 1024 < 232448 ? kUse + 1024 : 232448;
  static constexpr uint32_t kOCol = 256;
  static_assert(kUse <= 232448 && kBar % 8 == 0, "shared memory");
  // One part of a cut item and query tile: O as [D / 4][128 rows] float4, then (reference, sum) [128 rows].
  static constexpr size_t kPart = size_t(D / 4) * 128 * 16 + 128 * 8;
};

// What the joining kernel needs to know of the item a block's run starts in.
struct Meta {
  int b, kvh, pair, count;
  int j0;  // the item's tile the run starts at (0: the run starts with the item)
  int nt;  // tiles of the item
  int share, extra;  // blocks below `extra` have share + 1 units, the others share
};

struct Args {
  const int32_t *base, *count;
  const uint32_t* mask;
  const uint16_t *k_new, *v_new;
  uint16_t *k_cache, *v_cache, *out;
  int batch, tokens, heads, kv_heads, max_len;
  int group, tpt;  // query heads per kv head; nodes per query tile (tpt * group <= 128)
  int per_item;    // nodes per item
  uint32_t item_mul;  // ceil(2^20 / per_item)
  int words;       // mask words per node
  KvPages kp;
  int pool_rows;
  int page_shift;  // log2 of the page size
  int box_rows;  // rows of a K or V box: 8, or a multiple of 8 that a map of whole groups gives
  Meta* meta;
  uint8_t* parts;
  int* err;
};

// Whether the call can serve the sequence; one that it cannot has nothing.
__device__ __forceinline__ bool usable(const Args& a, int base, int count) {
  return count >= 0 && count <= a.tokens && base >= 0 && base <= a.max_len - count;
}

template <bool Wide>
__device__ __forceinline__ Seq seq_of(const Args& a, int b) {
  Seq s{a.base[b], a.count ? a.count[b] : a.tokens, 0, 0, 0};
  if (!usable(a, s.base, s.count)) s.base = s.count = 0;
  s.prefix = (s.base + kTile - 1) / kTile;
  s.nt = s.count ? s.prefix + (s.count + kTile - 1) / kTile : 0;
  // By multiplication: exact for what a tree can have (kTreeMaxTokens is below 2^11).
  s.pairs = Wide ? int(uint32_t(s.count + a.per_item - 1) * a.item_mul >> 20) : s.count > 0;
  return s;
}

// The line that blocks share out is counted in units: an item is kStart units
// that stand for starting it and then its tiles, one unit each.
struct Walk {
  Seq s;  // of sequence b
  int b, left;   // units left of the block's run
  uint32_t off;  // within sequence b's units
};

// Units of a sequence.  The host bounds those of a call below 2^31.
__device__ __forceinline__ uint32_t units_of(const Args& a, const Seq& s) {
  return s.nt ? uint32_t(s.nt + kStart) * uint32_t(a.kv_heads) * uint32_t(s.pairs) : 0;
}

// The next segment; false at the run's end.  A run holds a tile whenever `left`
// is not 0: what remains of it is dropped when only start units do.
template <bool Wide>
__device__ __forceinline__ bool next_seg(const Args& a, Walk& w, Seg& g) {
  if (w.left <= 0) return false;
  for (;;) {
    if (w.off < units_of(a, w.s)) break;
    w.off = 0;  // runs end where sequences do
    if (++w.b >= a.batch) return false;
    w.s = seq_of<Wide>(a, w.b);
  }
  g.s = w.s;
  g.b = w.b;
  const uint32_t per = uint32_t(w.s.nt + kStart), item = w.off / per;
  const int at = int(w.off - item * per), units = min(int(per) - at, w.left);
  g.j0 = max(0, at - kStart);
  g.kvh = int(Wide ? item / uint32_t(w.s.pairs) : item);
  g.pair = int(item - uint32_t(g.kvh) * uint32_t(w.s.pairs));
  g.j1 = at + units - kStart;
  w.off += uint32_t(units);
  w.left -= units;
  if (w.left <= kStart) w.left = 0;
  g.last = w.left == 0;
  return true;
}

// Bounded wait for the phase with parity `parity` (mbar_wait, kept small: it
// stands at two dozen places).
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity) {
  const uint32_t at = su32(bar);
#pragma unroll 1
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(at), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
// The same by a converged warp, whose lanes stay together.
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t parity) {
  const uint32_t at = su32(bar);
#pragma unroll 1
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(at), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done)) return true;
  }
  return false;
}

// An arrival by the lanes with `on`, without a branch: a warp that splits at
// every arrival loses more than the arrival costs.
__device__ __forceinline__ void arrive_if(bool on, uint64_t* bar) {
  asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %1, 0;\n @p mbarrier.arrive.shared::cta.b64 _, [%0];\n}" ::"r"(su32(bar)),
               "r"(uint32_t(on))
               : "memory");
}
__device__ __forceinline__ void expect_if(bool on, uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n @p mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(
          su32(bar)),
      "r"(bytes), "r"(uint32_t(on))
      : "memory");
}

// Tile j of a segment: valid positions, and for a tile of nodes the first node (-1 for cached positions).
__device__ __forceinline__ int tile_valid(const Seq& s, int j, int& node0) {
  if (j < s.prefix) {
    node0 = -1;
    return min(kTile, s.base - j * kTile);
  }
  node0 = (j - s.prefix) * kTile;
  return min(kTile, s.count - node0);
}

// The n lowest bits (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// 2^x by the hardware approximation (relative error about 2^-22).
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
// Packed pairs of f32.
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Both halves of a bf16 pair: the non-finite ones set to zero (keep = false) or all others (keep = true).
__device__ __forceinline__ uint32_t split_finite(uint32_t v, bool keep) {
  const bool lo = (v & 0x7F80u) == 0x7F80u, hi = (v & 0x7F800000u) == 0x7F800000u;
  return (lo == keep ? v & 0xFFFFu : 0u) | (hi == keep ? v & 0xFFFF0000u : 0u);
}

__device__ __forceinline__ bool all_finite(uint32_t v) {
  return (v & 0x7F80u) != 0x7F80u && (v & 0x7F800000u) != 0x7F800000u;
}

// Whether a V tile has rows past its end or nodes' rows.
__device__ __forceinline__ bool needs_cleaning(int nv, int node0) { return nv < kTile || node0 >= 0; }

// Appends the block's share of the new rows, and zeroes the output rows of
// dead nodes.  One warp.
template <int D>
__device__ void append_rows(const Args& a, int tid) {
  constexpr int kT = 32, kU = 4;  // threads; pieces in flight of each
  constexpr int kPer = D / 8;  // 16-byte pieces per head
  const int rows = a.batch * a.tokens, pieces = a.kv_heads * kPer;
#pragma unroll 1
  for (int r = int(blockIdx.x); r < rows; r += int(gridDim.x)) {
    const int b = r / a.tokens, t = r % a.tokens;
    const int base = a.base[b], count = a.count ? a.count[b] : a.tokens;
    const bool good = usable(a, base, count);
    if (!good && t == 0 && tid == 0 && a.err) atomicExch(a.err, kBadPosition);
    if (!good || t >= count) {
      uint4* o = reinterpret_cast<uint4*>(a.out) + int64_t(r) * a.heads * kPer;
#pragma unroll 1
      for (int i = tid; i < a.heads * kPer; i += kT) o[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const uint4* kn = reinterpret_cast<const uint4*>(a.k_new) + int64_t(r) * pieces;
    const uint4* vn = reinterpret_cast<const uint4*>(a.v_new) + int64_t(r) * pieces;
    const int64_t row0 = kv_row(a.kp, b, 0, a.kv_heads, a.max_len, base + t);
    if (row0 < 0) {
      if (tid == 0 && a.err) atomicExch(a.err, kBadPage);
      continue;
    }
    const int64_t step = a.kp.paged() ? a.kp.page_size : a.max_len;  // rows between kv heads
#pragma unroll 1
    for (int i0 = tid; i0 < pieces; i0 += kT * kU) {
      uint4 k[kU], v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (i0 + u * kT < pieces) {
          k[u] = kn[i0 + u * kT];
          v[u] = vn[i0 + u * kT];
        }
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (i0 + u * kT < pieces) {
          const int i = i0 + u * kT;
          const int64_t at = (row0 + i / kPer * step) * kPer + i % kPer;
          reinterpret_cast<uint4*>(a.k_cache)[at] = k[u];
          reinterpret_cast<uint4*>(a.v_cache)[at] = v[u];
        }
    }
  }
}

// Whether `p` holds in any thread of the two warps that share barrier `id`.
__device__ __forceinline__ bool pair_any(int id, bool p) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 64, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(uint32_t(p)), "r"(id)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ void pair_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory");
}

template <int D, bool Wide>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap knmap,
                          const __grid_constant__ CUtensorMap vnmap, const Args a) {
  using L = Lay<D, Wide>;
  constexpr int kNS = L::kSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u);
  if (smem - smem_raw + L::kUse > L::kBytes) {  // the 128-byte swizzle needs the tiles on 1024 bytes
    if (threadIdx.x == 0 && a.err) atomicExch(a.err, 4);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* full = bars;              // [kNS] ring slot loaded (and clean)
  uint64_t* empty = bars + kNS;       // [kNS] ring slot read by its products
  uint64_t* raw = bars + 2 * kNS;     // [kNS] a V tile that warp 3 cleans first is loaded
  uint64_t* seg_full = bars + 3 * kNS;  // [kSegs] segment written
  uint64_t* q_full = seg_full + kSegs;  // the segment's query tiles are loaded
  uint64_t* q_empty = q_full + 1;     // its S products are complete
  uint64_t* s_full = q_full + 2;      // [2] per group: S is in TMEM
  uint64_t* p_full = q_full + 4;      // [2] per group: P is in TMEM (8 warps arrive)
  uint64_t* o_done = q_full + 6;      // [2] per group: the segment's last P V is complete
  uint64_t* st_full = q_full + 8;     // [2] per group: its statistics are written (8 warps)
  uint64_t* o_free = q_full + 10;     // O and the statistics have been read (16 warps)
  uint64_t* mma_done = q_full + 11;   // every product of the block is complete
  int* words = reinterpret_cast<int*>(bars + L::kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(words);
  int* s_fail = words + 1;
  int* s_odd = words + 2;  // [4]: s_odd[i % 4] == i + 1: segment i holds non-finite node values
  float* s_stat = reinterpret_cast<float*>(smem + L::kStat);  // [group][2][row]
  Seg* s_seg = reinterpret_cast<Seg*>(smem + L::kSeg);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_item = a.per_item;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kNS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&raw[s], 1);
    }
    for (int s = 0; s < kSegs; ++s) mbar_init(&seg_full[s], 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 8);
      mbar_init(&o_done[s], 1);
      mbar_init(&st_full[s], 8);
    }
    mbar_init(o_free, 16);
    mbar_init(mma_done, 1);
    *s_fail = 0;
    s_odd[0] = s_odd[1] = s_odd[2] = s_odd[3] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&qmap);
    prefetch_map(&kmap);
    prefetch_map(&vmap);
    prefetch_map(&knmap);
    prefetch_map(&vnmap);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();  // every operand may come from the kernels before
  auto fail = [&]() { atomicExch(s_fail, 1); };
  auto failed = [&]() { return *reinterpret_cast<volatile int*>(s_fail) != 0; };

  static_assert(kNS > 2, "a step of two loads passes the ring's end at most once");
  struct Place {  // of a ring load
    uint32_t slot, parity;
    __device__ void step(uint32_t by) {
      slot += by;
      if (slot >= uint32_t(kNS)) {
        slot -= kNS;
        parity ^= 1;
      }
    }
  };
  // Every role takes the same segments from warp 0 and counts ring loads, S
  // tiles and segments for itself, so each barrier's phase is known without
  // any block-wide synchronisation.  Ring loads of a segment of n tiles that
  // starts at load c0:  K_0: c0;  K_j: c0 + 2j - 1;  V_j: c0 + 2j + 2, the last
  // one c0 + 2n - 1.  A segment's slot is written again four segments later:
  // then warp 0 has waited for the S products of two segments later, before
  // which warp 1 has waited for every softmax warp to be done with this one.
  auto wait_seg = [&](int si) { return wait_bar(&seg_full[si % kSegs], (si / kSegs) & 1); };
  if (warp == 0) {
    // ---- the walk and the loads --------------------------------------------------
    // All items in one line, an equal run of it per block.  A block that goes on to
    // another item drains its products, writes O and fills up again meanwhile: blocks
    // with three segments finished 4 to 8 us behind those with two.  So a start counts
    // as kStart tiles: 16 nodes over 500 positions, 32 heads, 14.5 -> 12.4 us (3: 12.6,
    // 5: 13.8); 8 x 25 nodes over 1100 to 2048, 55.9 -> 53.7 us.
    uint32_t sum = 0, share = 0, extra = 0, w0 = 0, len = 0;
    Walk w{Seq{}, a.batch, 0, 0};
    const int sets = (a.batch + 31) / 32;
    Seq s{};
#pragma unroll 1
    for (int r = 0; r < 2 * sets; ++r) {  // the sum of all tiles; then where this block's run starts
      const int b0 = (r < sets ? r : r - sets) * 32;
      if (r != 1 || sets > 1) {  // a single set of sequences is read once
        s = Seq{};
        if (b0 + lane < a.batch) s = seq_of<Wide>(a, b0 + lane);
      }
      const uint32_t u = units_of(a, s);
      if (r < sets) {
        sum += u;
        if (r < sets - 1) continue;
        const uint32_t total = __reduce_add_sync(0xffffffffu, sum);
        // A part costs about as much as a tile, so runs have two units at least
        // (16 nodes over 500 positions, 32 heads: 15.6 -> 14.9 us).
        const uint32_t blocks = min(gridDim.x, (total + 1) / 2);
        share = blocks ? total / blocks : 0;
        extra = total - share * blocks;
        w0 = share * blockIdx.x + min(blockIdx.x, extra);
        len = blockIdx.x < blocks ? share + (blockIdx.x < extra) : 0;
        sum = 0;  // now of the sequences before
        if (len == 0) break;
        continue;
      }
      uint32_t end = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += y;
      }
      end += sum;
      const uint32_t hit = __ballot_sync(0xffffffffu, w0 < end);
      if (hit) {
        const int l = __ffs(hit) - 1;
        w.b = b0 + l;
        w.off = w0 - __shfl_sync(0xffffffffu, end - u, l);
        w.s = Seq{__shfl_sync(0xffffffffu, s.base, l), __shfl_sync(0xffffffffu, s.count, l),
                  __shfl_sync(0xffffffffu, s.prefix, l), __shfl_sync(0xffffffffu, s.nt, l),
                  __shfl_sync(0xffffffffu, s.pairs, l)};
        w.left = int(len);
        const uint32_t at = w.off % uint32_t(w.s.nt + kStart);
        if (at + len <= kStart) w.left = 0;  // the next block has the item's first tile
        break;
      }
      sum = __shfl_sync(0xffffffffu, end, 31);
    }
    int nl = 0, si = 0;
    bool ok = true;
    Place next_load{0, 0};
    const int br = a.box_rows, nbox = kTile / br;
    Seg g;
    Meta m{0, 0, 0, 0, 0, 0, int(share), int(extra)};
    if (w.left == 0 && lane == 0) {  // nothing to do: an empty segment ends every role
      s_seg[0] = Seg{Seq{}, 0, 0, 0, 0, 0, 1};
      mbar_arrive(&seg_full[0]);
    }
    while (ok && next_seg<Wide>(a, w, g)) {
      if (__any_sync(0xffffffffu, failed())) break;
      if (!(ok = si == 0 || wait_bar_warp(q_empty, (si - 1) & 1))) break;
      if (lane == 0) {
        s_seg[si % kSegs] = g;
        mbar_arrive(&seg_full[si % kSegs]);
      }
      const int t0 = g.pair * per_item;
      const int qtiles = Wide && t0 + a.tpt < g.s.count ? 2 : 1;
      if (lane == 0) mbar_expect_tx(q_full, uint32_t(qtiles * L::kKB * a.tpt * a.group * 128));
      __syncwarp();
      if (lane < qtiles * L::kKB) {
        const int t = lane / L::kKB, kb = lane % L::kKB;
        tma_load_3d(smem + L::kQ + t * L::kBytesTile + kb * 16384, &qmap, q_full, kb * 64, g.kvh * a.group,
                    g.b * a.tokens + t0 + t * a.tpt);
      }
      // This lane's box of tile j: the map row of its first position.  A page
      // that is missing is read past the map's end, which gives zeros.
      auto box_row = [&](int j) {
        if (j >= g.s.prefix || lane >= nbox) return 0;
        const int p = j * kTile + lane * br;
        if (!a.kp.paged()) return (g.b * a.kv_heads + g.kvh) * a.max_len + p;
        const int lp = p >> a.page_shift;
        const int pg = lp < a.kp.pages_per_seq ? __ldg(a.kp.table + int64_t(g.b) * a.kp.pages_per_seq + lp) : -1;
        if (uint32_t(pg) < uint32_t(a.kp.num_pages))
          return ((pg * a.kv_heads + g.kvh) << a.page_shift) + (p & (a.kp.page_size - 1));
        if (p < g.s.base && a.err) atomicExch(a.err, kBadPage);
        return a.pool_rows;
      };
      auto load = [&](int tile, int map_row, bool is_v) {
        uint64_t* bar = &full[next_load.slot];
        uint8_t* dst = smem + L::kRing + next_load.slot * L::kBytesTile;
        if (nl >= kNS && !wait_bar_warp(&empty[next_load.slot], next_load.parity ^ 1)) ok = false;
        int node0;
        const int nv = tile_valid(g.s, tile, node0);
        if (is_v && needs_cleaning(nv, node0)) bar = &raw[next_load.slot];
        if (!ok) return;
        if (node0 < 0) {
          expect_if(lane == 0, bar, L::kBytesTile);
          if (lane < nbox) {
            if (br > 8) tma_load_4d(dst + lane * (br / 8) * L::kGroup, is_v ? &vmap : &kmap, bar, 0, 0, 0, map_row / 8);
            else tma_load_3d(dst + lane * L::kGroup, is_v ? &vmap : &kmap, bar, 0, map_row, 0);
          }
        } else {  // the 8-row groups that hold nodes
          expect_if(lane == 0, bar, (nv + 7) / 8 * L::kGroup);
          if (lane < (nv + 7) / 8)
            tma_load_4d(dst + lane * L::kGroup, is_v ? &vnmap : &knmap, bar, 0, g.b * a.tokens + node0 + lane * 8, 0,
                        g.kvh);
        }
        next_load.step(1);
        ++nl;
      };
      // K_0, then K_1, V_0, K_2, V_1, ..., and the last V.  A tile's map rows are
      // found two tiles before its K is loaded, so that the block table's latency is hidden.
      int row = 0, next = 0, later = 0;  // of tiles j, j + 1, j + 2
#pragma unroll 1
      for (int j = g.j0 - 2; j < g.j1; ++j) {
        row = next;
        next = later;
        if (j + 2 < g.j1) later = box_row(j + 2);
        if (j >= g.j0 - 1 && j + 1 < g.j1) load(j + 1, next, false);
        if (j >= g.j0) load(j, row, true);
      }
      if (si == 0) {
        m.b = g.b;
        m.kvh = g.kvh;
        m.pair = g.pair;
        m.count = g.s.count;
        m.j0 = g.j0;
        m.nt = g.s.nt;
      }
      ++si;
    }
    if (!ok) fail();
    if (lane == 0) {
      a.meta[blockIdx.x] = m;
      // Let the loads in flight land before the block can end.
#pragma unroll 1
      for (int c = max(0, nl - kNS); c < nl; ++c) wait_bar(&full[c % kNS], (c / kNS) & 1);
      if (si > 0) wait_bar(q_full, (si - 1) & 1);
    }
  } else if (warp == 1) {
    // ---- products: one thread --------------------------------------------------------
    // It shares its scheduler with the softmax, so what it does per product is
    // kept short: no votes, descriptors differ by an addition, ring places by a step.
    if (elect_one()) {
      constexpr uint32_t kIdS = idesc_bf16(kTile, kTile), kIdO = idesc_bf16(kTile, D, true);
      constexpr uint32_t kSlotStep = L::kBytesTile >> 4;  // in descriptor units
      const uint64_t q_desc = sw128_desc(smem + L::kQ), k_desc = sw128_desc(smem + L::kRing, L::kGroup),
                     v_desc = sw128_desc_mn(smem + L::kRing, 1024, L::kGroup);
      Place first{0, 0};  // the segment's first load
      int si = 0;
      uint32_t np = 0;  // parity of each group's next P tile
      bool ok = true;
      auto wait_load = [&](const Place& c) { return wait_bar(&full[c.slot], c.parity); };
      auto wait_p = [&](int t) {
        const bool r = wait_bar(&p_full[t], np >> t & 1);
        np ^= 1u << t;
        return r;
      };
      auto issue_s = [&](int t, uint32_t tile, const Place& k) {
        const uint64_t da = q_desc + uint64_t(tile * kSlotStep), db = k_desc + uint64_t(k.slot * kSlotStep);
#pragma unroll
        for (int kb = 0; kb < L::kKB; ++kb)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_bf16(tmem + uint32_t(t * 128), da + uint64_t(kb * (16384 >> 4) + 2 * kk),
                      db + uint64_t(kb * (1024 >> 4) + 2 * kk), kIdS, (kb | kk) != 0);
        umma_commit(&s_full[t]);
      };
      for (;;) {
        if (!(ok = wait_seg(si))) break;
        const Seg g = s_seg[si % kSegs];
        const int n = g.j1 - g.j0;
        if (n == 0) break;
        const bool second = Wide ? g.pair * per_item + a.tpt < g.s.count : n > 1;  // the second group has work
        Place k = first, v = first;  // of the next K tile and the next V tile
        v.step(n > 1 ? 2 : 1);
        if (!(ok = wait_bar(q_full, si & 1) && wait_load(k))) break;
        tc_fence_after();
        issue_s(0, 0, k);
        if (Wide && second) issue_s(1, 1, k);
        umma_commit(&empty[k.slot]);
        k.step(1);
        if constexpr (!Wide) {
          if (second) {
            if (!(ok = wait_load(k))) break;
            issue_s(1, 0, k);
            umma_commit(&empty[k.slot]);
            k.step(2);
          }
        }
        if (n == 1 || (!Wide && n == 2)) umma_commit(q_empty);
        // O of the segment before must have been read before this one's first P V.
        if (si >= 1 && !(ok = wait_bar(o_free, (si - 1) & 1))) break;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
          int node0;
          const int steps = (tile_valid(g.s, g.j0 + i, node0) + 15) / 16;
          const uint64_t dv = v_desc + uint64_t(v.slot * kSlotStep);
          auto issue_o = [&](int t, bool first_pv, bool last_pv) {
            const uint32_t tP = tmem + uint32_t(t * 128), tO = tmem + L::kOCol + uint32_t(t * D);
            tc_fence_after();
            umma_bf16_ts(tO, tP, dv, kIdO, !first_pv);
#pragma unroll
            for (int kk = 1; kk < kTile / 16; ++kk)
              if (kk < steps) umma_bf16_ts(tO, tP + uint32_t(kk * 8), dv + uint64_t(kk * (2 * L::kGroup >> 4)), kIdO, 1);
            if (last_pv) umma_commit(&o_done[t]);
          };
          const int ahead = Wide ? i + 1 : i + 2;  // the tile whose S follows this one's P V
          if (!(ok = wait_load(v) && (ahead >= n || wait_load(k)))) break;
          if constexpr (Wide) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (t == 1 && !second) break;
              if (!(ok = wait_p(t))) break;
              issue_o(t, i == 0, i == n - 1);
              if (ahead < n) issue_s(t, t, k);
            }
            if (!ok) break;
            umma_commit(&empty[v.slot]);
          } else {
            const int t = i & 1;
            if (!(ok = wait_p(t))) break;
            issue_o(t, i < 2, ahead >= n);
            umma_commit(&empty[v.slot]);
            if (ahead < n) issue_s(t, 0, k);
          }
          if (ahead < n) {
            umma_commit(&empty[k.slot]);
            k.step(2);
            if (ahead == n - 1) umma_commit(q_empty);
          }
          v.step(i + 2 >= n ? 1 : 2);  // the last V follows its K; past it the next segment starts
        }
        if (!ok) break;
        first = v;
        ++si;
        if (g.last) break;
      }
      if (!ok) fail();
      umma_commit(mma_done);
      wait_bar(mma_done, 0);
    }
    __syncwarp();
  } else if (warp == 2) {
    append_rows<D>(a, lane);
  } else if (warp == 3) {
    // ---- cleaning of V tiles ------------------------------------------------------------
    // Such a tile's load signals raw[slot], and this warp signals full[slot].
    int c0 = 0;
    uint32_t parity = 0;  // of each slot's next such tile
    bool ok = true;
    for (int si = 0;; ++si) {
      if (!(ok = __all_sync(0xffffffffu, wait_seg(si)))) break;
      const Seg g = s_seg[si % kSegs];
      const int n = g.j1 - g.j0;
      for (int i = 0; i < n; ++i) {
        int node0;
        const int nv = tile_valid(g.s, g.j0 + i, node0), nv16 = (nv + 15) & ~15;
        if (!needs_cleaning(nv, node0)) continue;
        const int c = i == n - 1 ? c0 + 2 * n - 1 : c0 + 2 * i + 2, slot = c % kNS;
        if (!(ok = wait_bar_warp(&raw[slot], parity >> slot & 1))) break;
        parity ^= 1u << slot;
        uint8_t* v = smem + L::kRing + slot * L::kBytesTile;
        // Rows past the tile's end, up to the last 16-row step of the product.
#pragma unroll 1
        for (int e = lane; e < (nv16 - nv) * L::kKB * 8; e += 32) {
          const int piece = e & 7, kb = (e >> 3) % L::kKB, r = nv + (e >> 3) / L::kKB;
          *reinterpret_cast<uint4*>(v + (r / 8) * L::kGroup + kb * 1024 + (r % 8) * 128 + piece * 16) =
              make_uint4(0, 0, 0, 0);
        }
        if (node0 >= 0) {
          bool odd = false;
#pragma unroll 2
          for (int e = lane; e < nv * L::kKB * 8; e += 32) {  // the swizzle only permutes a row's pieces
            const int piece = e & 7, kb = (e >> 3) % L::kKB, r = (e >> 3) / L::kKB;
            uint4* p = reinterpret_cast<uint4*>(v + (r / 8) * L::kGroup + kb * 1024 + (r % 8) * 128 + piece * 16);
            const uint4 x = *p;
            if (!(all_finite(x.x) && all_finite(x.y) && all_finite(x.z) && all_finite(x.w))) {
              *p = make_uint4(split_finite(x.x, false), split_finite(x.y, false), split_finite(x.z, false),
                              split_finite(x.w, false));
              odd = true;
            }
          }
          if (__any_sync(0xffffffffu, odd) && lane == 0) *reinterpret_cast<volatile int*>(&s_odd[si & 3]) = si + 1;
        }
        __threadfence_block();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[slot]);
      }
      if (!ok || n == 0 || g.last) break;
      c0 += 2 * n;
    }
    if (!ok) fail();
  } else {
    // ---- softmax and output: two threads per query row --------------------------------
    const int t = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1;
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const int pair_bar = 1 + t * 4 + quarter;  // shared with the warp of the other half
    const uint32_t lane_addr = uint32_t(quarter * 32) << 16;
    const uint32_t tS = tmem + lane_addr + uint32_t(t * 128);
    const uint32_t tO = tmem + lane_addr + L::kOCol;
    const float sl = kLog2e / sqrtf(float(D));
    const int node = row / a.group, head = row % a.group;
    int ns = 0, no[2] = {0, 0};  // S tiles and finished O's so far
    // After a wait that ran out nothing waits any more and nothing is written,
    // but every step is still taken, so that the pairs' barriers stay complete.
    bool ok = true;
    for (int si = 0;; ++si) {
      if (failed()) ok = false;
      if (ok && !wait_bar_warp(&seg_full[si % kSegs], (si / kSegs) & 1)) ok = false;
      ok = !pair_any(pair_bar, !ok);
      if (!ok) {  // the segments may not be there: all softmax warps leave here
        fail();
        break;
      }
      const Seg g = s_seg[si % kSegs];
      const int n = g.j1 - g.j0;
      if (n == 0) break;
      const int tok = g.pair * per_item + (Wide ? t * a.tpt : 0) + node;  // this row's node
      const bool live = node < a.tpt && tok < g.s.count;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const bool mine = !Wide || t == 0 || g.pair * per_item + a.tpt < g.s.count;
      const int64_t qrow = int64_t(g.b) * a.tokens + tok;
      float m_ref = -INFINITY, l = 0.0f;
      if (mine) {
        for (int i = Wide ? 0 : t; i < n; i += Wide ? 1 : 2) {
          int node0;
          const int nv = tile_valid(g.s, g.j0 + i, node0) - half * kHalf;  // of this thread's positions
          // The positions this row sees, of this thread's 64.
          uint32_t seen[2] = {low_bits(nv), low_bits(nv - 32)};
          if (node0 >= 0) {
            const int w = node0 / 32 + half * 2;
            seen[0] &= live && w < a.words ? a.mask[qrow * a.words + w] : 0u;
            seen[1] &= live && w + 1 < a.words ? a.mask[qrow * a.words + w + 1] : 0u;
          }
          if (ok && !wait_bar_warp(&s_full[t], ns & 1)) ok = false;
          ++ns;
          tc_fence_after();
          if (warp_live) {
            uint32_t r[kHalf];
            tmem_ld64(tS + uint32_t(half * kHalf), r);
            if (node0 >= 0 || nv < kHalf) {
#pragma unroll
              for (int e = 0; e < kHalf; ++e)
                if (!(seen[e / 32] >> (e % 32) & 1)) r[e] = 0xFF800000u;
            }
            // Maximum of the raw scores, four independent chains; the scale is
            // positive, so it is applied once to the maximum (base 2).
            float mc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < kHalf; e += 8)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                mc[c] = fmax3(mc[c], __uint_as_float(r[e + 2 * c]), __uint_as_float(r[e + 2 * c + 1]));
            float mt = fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])) * sl;
            // The vote also stands between this thread's read of S and the other's P in its columns.
            tc_fence_before();
            const bool moves = pair_any(pair_bar, mt > m_ref + kRescale);
            tc_fence_after();
            if (moves) {  // also the first tile with anything to see
              // Both threads of a row take the larger maximum: exchanged in two
              // columns of S, which both have read.
              tmem_st1(tS + uint32_t(kHalf + half), __float_as_uint(mt));
              tc_fence_before();
              pair_sync(pair_bar);
              tc_fence_after();
              mt = fmaxf(mt, __uint_as_float(tmem_ld1(tS + uint32_t(kHalf + 1 - half))));
              bool rescale = false;
              float corr = 1.0f;
              if (mt > m_ref + kRescale) {
                if (m_ref != -INFINITY) {
                  corr = ex2(m_ref - mt);
                  rescale = true;
                }
                l *= corr;
                m_ref = mt;
              }
              // O is settled: its last P V completed before this S was published.
              if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 16) {
                  uint32_t o16[16];
                  const uint32_t at = tO + uint32_t(t * D + half * (D / 2) + c);
                  tmem_ld16(at, o16);
#pragma unroll
                  for (int e = 0; e < 16; ++e) o16[e] = __float_as_uint(__uint_as_float(o16[e]) * corr);
                  tmem_st16(at, o16);
                }
              }
            }
            // P = 2^(s sl - m_ref) as bf16 pairs, packed in place; -inf gives 0 (a row
            // that sees nothing yet uses 0 for the reference: no inf - inf).  All
            // exponentials on the special-function unit: a quarter of them as cubic
            // polynomials on the others took as long, half of them 6 % longer.
            const float mneg = m_ref == -INFINITY ? 0.0f : -m_ref;
            const uint64_t sl2 = pack_f2(sl, sl), mneg2 = pack_f2(mneg, mneg);
            uint64_t acc[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < kHalf; e += 2) {
              float x0, x1;
              unpack_f2(fma_f2(pack_f2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), sl2, mneg2), x0, x1);
              x0 = ex2(x0);
              x1 = ex2(x1);
              acc[(e >> 1) & 1] = add_f2(acc[(e >> 1) & 1], pack_f2(x0, x1));
              asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r[e / 2]) : "f"(x1), "f"(x0));
            }
            float a0, a1;
            unpack_f2(add_f2(acc[0], acc[1]), a0, a1);
            l += a0 + a1;
            tmem_st32p(tS + uint32_t(half * 32), r);
          }
          tc_fence_before();
          __syncwarp();
          arrive_if(lane == 0, &p_full[t]);
        }
      }
      // ---- output ----------------------------------------------------------------------
      // The statistics of the segment before have been read by everyone.
      if (si >= 1 && ok && !wait_bar_warp(o_free, (si - 1) & 1)) ok = false;
      s_stat[(t * 2 + half) * 128 + row] = l;
      if (!Wide) {  // the other group wants the row's sum and its reference
        pair_sync(pair_bar);
        if (half == 0) s_stat[t * 256 + row] = l + s_stat[t * 256 + 128 + row];
        pair_sync(pair_bar);
        if (half == 1) s_stat[t * 256 + 128 + row] = m_ref;
      }
      __syncwarp();
      arrive_if(lane == 0, &st_full[t]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (Wide && x != t) continue;
        if (ok && !wait_bar_warp(&st_full[x], si & 1)) ok = false;
        if (Wide ? mine : x < n) {
          if (ok && !wait_bar_warp(&o_done[x], no[x] & 1)) ok = false;
          ++no[x];
        }
      }
      __syncwarp();
      tc_fence_after();
      if (mine && warp_live && __all_sync(0xffffffffu, ok)) {
        float w0 = 1.0f, w1 = 0.0f;  // weights of O_0 and O_1 (not wide: both belong to the row)
        if (Wide) {
          l = s_stat[t * 256 + row] + s_stat[t * 256 + 128 + row];
        } else {
          const float m0 = s_stat[128 + row], m1 = n > 1 ? s_stat[384 + row] : -INFINITY;
          const float l0 = s_stat[row], l1 = s_stat[256 + row];
          m_ref = fmaxf(m0, m1);
          w1 = n > 1 ? 1.0f : 0.0f;
          if (m_ref != -INFINITY) {
            w0 = ex2(m0 - m_ref);
            w1 = ex2(m1 - m_ref);
          }
          l = l0 * w0 + l1 * w1;
        }
        const bool whole = g.j0 == 0 && g.j1 == g.s.nt;
        const bool odd = *reinterpret_cast<volatile int*>(&s_odd[si & 3]) == si + 1;
        const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);  // a row that sees nothing: O is 0
        // A cut item: this part's place (0: the block's run starts in it).
        const uint32_t slot = (blockIdx.x * 2 + (si == 0 ? 0 : 1)) * (Wide ? 2 : 1) + (Wide ? t : 0);
        float4* po = reinterpret_cast<float4*>(a.parts + slot * uint32_t(L::kPart));
        float2* pm = reinterpret_cast<float2*>(po + (D / 4) * 128);
        uint16_t* orow = a.out + (qrow * a.heads + g.kvh * a.group + head) * D;
        constexpr int kCols = Wide ? D / 2 : D / 4;  // this thread's columns
        const int col0 = (Wide ? half : t * 2 + half) * kCols;
#pragma unroll 1
        for (int c = col0; c < col0 + kCols; c += 16) {
          float o[16];
          {
            uint32_t r[16];
            tmem_ld16(tO + uint32_t((Wide ? t * D : 0) + c), r);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __uint_as_float(r[e]);
          }
          if (!Wide && n > 1) {
            uint32_t r[16];
            tmem_ld16(tO + uint32_t(D + c), r);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = o[e] * w0 + __uint_as_float(r[e]) * w1;
          }
          if (odd && live) {
#pragma unroll 1
            for (int j = max(0, (g.j0 - g.s.prefix) * kTile); j < min(g.s.count, (g.j1 - g.s.prefix) * kTile); ++j) {
              if (!(a.mask[qrow * a.words + j / 32] >> (j % 32) & 1)) continue;
              const uint32_t* v = reinterpret_cast<const uint32_t*>(
                  a.v_new + ((int64_t(g.b) * a.tokens + j) * a.kv_heads + g.kvh) * D + c);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t x = split_finite(v[e], true);
                o[2 * e] += bf_lo(x);
                o[2 * e + 1] += bf_hi(x);
              }
            }
          }
          if (live && whole) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              uint32_t w4[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w4[e] = pack_bf2(o[8 * v + 2 * e] * inv, o[8 * v + 2 * e + 1] * inv);
              *reinterpret_cast<uint4*>(orow + c + 8 * v) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
            }
          } else if (live) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              po[(c / 4 + v) * 128 + row] = make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
          }
        }
        if (live && !whole && half == 0 && (Wide || t == 0)) pm[row] = make_float2(m_ref, l);
      }
      // O and the statistics have been read.
      tc_fence_before();
      __syncwarp();
      arrive_if(lane == 0, o_free);
      if (g.last) break;
    }
    if (!ok) fail();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
  if (threadIdx.x == 0 && *s_fail && a.err) atomicExch(a.err, 4);
}

// Joins the parts of the item that block c's run starts in the middle of, when
// c is the first block whose run does.  Thread = query row, blockIdx.y = 8
// columns of one query tile; parts are taken four at a time, all their loads in
// flight together.
constexpr int kJoinParts = 4;
template <int D, bool Wide>
__global__ void __launch_bounds__(128) tree_join_kernel(const Args a) {
  using L = Lay<D, Wide>;
  // Wait, then trigger: a kernel behind this one may read the cache before its own
  // wait (the decode attention does), and the appended rows have to be there by then.
  pdl_wait();
  pdl_trigger();
  const int c = int(blockIdx.x), row = int(threadIdx.x);
  const int t = Wide ? int(blockIdx.y) / (D / 8) : 0, col = int(blockIdx.y) % (D / 8);
  const Meta m = a.meta[c];
  const int before = m.share + (c - 1 < m.extra);  // units of block c - 1
  if (m.j0 == 0 || m.j0 > before) return;
  const int tok = m.pair * a.tpt * (Wide ? 2 : 1) + t * a.tpt + row / a.group;
  if (row / a.group >= a.tpt || tok >= m.count) return;
  // Block c - 1's part, then those of c, c + 1, ...: first the longer blocks, then the others.
  const int rest = m.nt - m.j0, longer = max(0, m.extra - c), in_longer = longer * (m.share + 1);
  const int parts = 1 + (rest <= in_longer ? (rest + m.share) / (m.share + 1)
                                           : longer + (rest - in_longer + m.share - 1) / m.share);
  float best = -INFINITY, l = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int k0 = 0; k0 < parts; k0 += kJoinParts) {
    float2 ml[kJoinParts];
    float4 x[kJoinParts][2];
#pragma unroll
    for (int q = 0; q < kJoinParts; ++q) {
      const int k = k0 + q;
      ml[q] = make_float2(-INFINITY, 0.0f);
      x[q][0] = x[q][1] = make_float4(0, 0, 0, 0);
      if (k < parts) {
        const int64_t slot = (int64_t(c - 1 + k) * 2 + (k == 0 && m.j0 + kStart < before ? 1 : 0)) * (Wide ? 2 : 1) + t;
        const uint8_t* p = a.parts + slot * L::kPart;
        ml[q] = reinterpret_cast<const float2*>(p + size_t(D / 4) * 128 * 16)[row];
        x[q][0] = reinterpret_cast<const float4*>(p)[(col * 2) * 128 + row];
        x[q][1] = reinterpret_cast<const float4*>(p)[(col * 2 + 1) * 128 + row];
      }
    }
    float top = best;
#pragma unroll
    for (int q = 0; q < kJoinParts; ++q) top = fmaxf(top, ml[q].x);
    // Nothing seen so far: every O is 0, or a non-finite node's value.
    const float w0 = best == top ? 1.0f : ex2(best - top);
    l *= w0;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= w0;
#pragma unroll
    for (int q = 0; q < kJoinParts; ++q) {
      const float w = ml[q].x == top ? 1.0f : ex2(ml[q].x - top);
      l += w * ml[q].y;
      o[0] += w * x[q][0].x;
      o[1] += w * x[q][0].y;
      o[2] += w * x[q][0].z;
      o[3] += w * x[q][0].w;
      o[4] += w * x[q][1].x;
      o[5] += w * x[q][1].y;
      o[6] += w * x[q][1].z;
      o[7] += w * x[q][1].w;
    }
    best = top;
  }
  const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
  uint16_t* orow = a.out + ((int64_t(m.b) * a.tokens + tok) * a.heads + m.kvh * a.group + row % a.group) * D + col * 8;
  *reinterpret_cast<uint4*>(orow) = make_uint4(pack_bf2(o[0] * inv, o[1] * inv), pack_bf2(o[2] * inv, o[3] * inv),
                                               pack_bf2(o[4] * inv, o[5] * inv), pack_bf2(o[6] * inv, o[7] * inv));
}

constexpr size_t kMetaBytes = size_t(kNumSMs) * sizeof(Meta);

template <int D, bool Wide>
int launch(const TreeArgs& t, cudaStream_t st) {
  using L = Lay<D, Wide>;
  static PerDeviceOnce configured;
  if (!configured.run([] {
        return cudaFuncSetAttribute(tree_attention_kernel<D, Wide>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    L::kBytes) == cudaSuccess;
      }))
    return SB_INTERNAL;
  const int group = int(t.heads / t.kv_heads), tpt = kTile / group, per_item = tpt * (Wide ? 2 : 1);
  const bool paged = t.kp.paged();
  const uint64_t rows = uint64_t(t.batch) * uint64_t(t.tokens);
  const uint64_t kv_rows = paged ? uint64_t(t.kp.num_pages) * uint64_t(t.kv_heads) * uint64_t(t.kp.page_size)
                                 : uint64_t(t.batch) * uint64_t(t.kv_heads) * uint64_t(t.max_len);
  // K and V tiles lie in shared memory as groups of 8 rows, a group's 64-wide
  // blocks side by side, so that one box brings whole groups: a page, or a tile
  // of a contiguous cache whose sequences start on 8 rows.  One box of 128 rows
  // instead of two of 64 columns, and 8 instead of 16 for 16-row pages: 32 x 16
  // nodes over 4096 positions in 16-row pages 149 -> 131 us.  Rows that start
  // anywhere (the nodes' own, and other contiguous caches) come 8 at a time.
  constexpr uint64_t kKB = D / 64;
  const bool grouped = paged || t.max_len % 8 == 0;
  const uint32_t box = !grouped ? 8u : paged ? uint32_t(std::min(t.kp.page_size, kTile)) : uint32_t(kTile);
  auto cache_map = [&](CUtensorMap* m, const void* p) {
    if (grouped) {
      const uint64_t dims[4] = {64, 8, kKB, kv_rows / 8}, strides[3] = {D, 64, 8 * D};
      const uint32_t bx[4] = {64, 8, uint32_t(kKB), box / 8};
      return make_map_bf16(m, p, 4, dims, strides, bx);
    }
    const uint64_t dims[3] = {64, kv_rows, kKB}, strides[2] = {D, 64};
    const uint32_t bx[3] = {64, 8, uint32_t(kKB)};
    return make_map_bf16(m, p, 3, dims, strides, bx);
  };
  auto node_map = [&](CUtensorMap* m, const void* p) {
    const uint64_t dims[4] = {64, rows, kKB, uint64_t(t.kv_heads)}, strides[3] = {uint64_t(t.kv_heads) * D, 64, D};
    const uint32_t bx[4] = {64, 8, uint32_t(kKB), 1};
    return make_map_bf16(m, p, 4, dims, strides, bx);
  };
  const uint64_t qdims[3] = {D, uint64_t(t.heads), rows}, qstrides[2] = {D, uint64_t(t.heads) * D};
  const uint32_t qbox[3] = {64, uint32_t(group), uint32_t(tpt)};
  CUtensorMap qm, km, vm, knm, vnm;
  if (!make_map_bf16(&qm, t.q, 3, qdims, qstrides, qbox) || !cache_map(&km, t.k_cache) || !cache_map(&vm, t.v_cache) ||
      !node_map(&knm, t.k_new) || !node_map(&vnm, t.v_new))
    return SB_INTERNAL;
  Args a{t.base, t.count, t.mask, t.k_new, t.v_new, t.k_cache, t.v_cache, t.out, int(t.batch), int(t.tokens),
         int(t.heads), int(t.kv_heads), int(t.max_len), group, tpt, per_item, ((1u << 20) + unsigned(per_item) - 1) / unsigned(per_item), int((t.tokens + 31) / 32), t.kp, int(kv_rows), paged ? __builtin_ctz(unsigned(t.kp.page_size)) : 0, int(box),
         static_cast<Meta*>(t.workspace), static_cast<uint8_t*>(t.workspace) + kMetaBytes, t.err};
  // A block per SM, fewer when there are not that many tiles even at full lengths.
  const int64_t tiles = (t.max_len + kTile - 1) / kTile + (t.tokens + kTile - 1) / kTile + kStart;  // and start units
  const int64_t items = t.batch * t.kv_heads * ((t.tokens + per_item - 1) / per_item);
  if (items > INT32_MAX / tiles) return SB_INVALID_ARGUMENT;
  const int64_t most = items * tiles;
  const unsigned grid = unsigned(std::min<int64_t>(most, kNumSMs));
  if (launch_pdl(tree_attention_kernel<D, Wide>, dim3(grid), dim3(kThreads), size_t(L::kBytes), st, qm, km, vm, knm,
                 vnm, a) != cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  // Also where nothing is cut: it holds later kernels back until the rows are appended.
  if (launch_pdl(tree_join_kernel<D, Wide>, dim3(grid, unsigned(D / 8 * (Wide ? 2 : 1))), dim3(128), 0, st, a) !=
      cudaSuccess)
    return SB_INTERNAL;
  count_launch();
  return SB_OK;
}

bool wide(int64_t tokens, int64_t heads, int64_t kv_heads) {
  const int64_t group = heads / kv_heads;
  return tokens > kTile / group;
}

}  // namespace

uint64_t tree_attention_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  const uint64_t part = head_dim == 128 ? Lay<128, false>::kPart : Lay<64, false>::kPart;
  return kMetaBytes + uint64_t(kNumSMs) * 2 * part * (wide(tokens, heads, kv_heads) ? 2 : 1);
}

bool tree_attention_supported(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  return tokens >= 1 && tokens <= kTreeMaxTokens && kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0 &&
         heads / kv_heads <= kTile && heads <= 65535 && (head_dim == 64 || head_dim == 128);
}

int launch_tree_attention(const TreeArgs& a, cudaStream_t st) {
  if (!tree_attention_supported(a.tokens, a.heads, a.kv_heads, a.head_dim)) return SB_INVALID_ARGUMENT;
  if (a.batch == 0) return SB_OK;
  for (const void* p : {static_cast<const void*>(a.q), static_cast<const void*>(a.k_new),
                        static_cast<const void*>(a.v_new), static_cast<const void*>(a.k_cache),
                        static_cast<const void*>(a.v_cache), static_cast<const void*>(a.out),
                        static_cast<const void*>(a.workspace)})
    if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return SB_INVALID_ARGUMENT;  // TMA and 16-byte accesses
  if (wide(a.tokens, a.heads, a.kv_heads))
    return a.head_dim == 128 ? launch<128, true>(a, st) : launch<64, true>(a, st);
  return a.head_dim == 128 ? launch<128, false>(a, st) : launch<64, false>(a, st);
}

}  // namespace sb

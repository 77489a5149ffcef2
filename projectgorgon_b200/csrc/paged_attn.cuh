// Attention over a paged cache: the launch description, the visibility rule,
// and the schedule that the tensor-core kernels share.
//
// A unit of work is M packed query rows of one (sequence, kv head): packed row
// r is (new row r / group, query head r % group of the kv head's group), so a
// unit's rows are close in position and share a causal frontier.  A unit's
// keys are tiles of `bn` positions: the tiles that hold its sink rows, then
// those from its window's first position to its last visible one.
//
// The tiles of all units, in the order (sequence, kv head, row block), form one
// list that the grid's CTAs share out in equal contiguous ranges, so ragged
// batches, long single sequences and windows balance by themselves, without
// the host knowing any length.  A unit also costs its start and end (loading
// Q, joining warps, writing rows), which counts as `unit_cost` empty places
// before its tiles: a batch of short sequences would otherwise load some CTAs
// with many units.  A unit inside one CTA's range is finished there; one cut between CTAs leaves unnormalised fp32 rows with their running
// max and sum in the workspace (slot 0: the piece that a CTA starts with, slot
// 1: the one that it ends with), and paged_merge_kernel joins them in the
// order of the CTAs, so results do not depend on timing.
#pragma once

#include <type_traits>

#include "paged.cuh"

namespace gorgon {

constexpr int kPagedMaxNodes = 1024;  // tree rows per sequence

struct PagedAttn {
  PagedPool pool;
  NewRows nr;
  const char* q;
  int64_t q_sb, q_sh, q_sn;  // bytes
  char* out;
  int64_t o_sb, o_sh, o_sn;  // elements (dtype of the pool)
  float* lse;
  int64_t l_sb, l_sh, l_sn;
  const int32_t* parents;
  int64_t par_sb;
  int max_depth;
  int window, sinks;  // window 0: none
  int hq, group, n;   // n: largest count of new rows
  int rows;           // packed rows of q and out (with nr.cu)
  float scale_log2;   // softmax scale * log2(e)
  // tensor-core schedule
  int m, bn_shift;    // packed rows per unit, log2 of the positions per tile
  uint32_t group_m;   // with group_s: division by `group` (group_div)
  int group_s;
  int qblocks;        // units per (sequence, kv head) at most
  int unit_cost;      // places in the list that a unit's start and end take
  int grid;
  float* part_o;      // [grid * 2][m][d]
  float2* part_ml;    // [grid * 2][m]  running max (log2 units) and sum
  struct CutUnit* cut;  // [grid]
  uint64_t wait_ns;
  int tma;            // (tcgen05) pages come by TMA
};

// n / group for 0 <= n < 2^31, by a multiplication (m = floor(2^32 (2^s - group)
// / group) + 1, s = ceil(log2 group)).
__device__ __forceinline__ int group_div(const PagedAttn& a, int n) {
  return static_cast<int>((__umulhi(static_cast<uint32_t>(n), a.group_m) + static_cast<uint32_t>(n)) >> a.group_s);
}
inline void set_group_div(PagedAttn* a) {
  int s = 0;
  while ((1 << s) < a->group) ++s;
  a->group_s = s;
  a->group_m = static_cast<uint32_t>((((uint64_t(1) << s) - a->group) << 32) / a->group + 1);
}

// What CTA c leaves for the merge: the unit that its range starts inside of.
// pieces == 0: none, or an earlier CTA's entry names the unit.
struct CutUnit {
  int b, kvh, qb;
  int pieces;      // CTAs c - 1, c, ..., c - 2 + pieces
  int first_slot;  // slot of CTA c - 1's piece (the others are in slot 0)
};

// A sequence's state: P cached rows before its c new ones.
struct Seq {
  int L, c, P;
  bool ok;  // has rows to compute
};

// The sequence's rows lie inside q and out.
__device__ __forceinline__ bool rows_inside(const PagedAttn& a, int b, int c) {
  return !a.nr.cu || (a.nr.cu[b] >= 0 && c >= 0 && a.nr.cu[b] <= a.rows - c);
}

__device__ __forceinline__ Seq sequence(const PagedAttn& a, int b, bool report) {
  Seq s;
  s.L = a.pool.lens[b];
  s.c = a.nr.count(b);
  s.P = s.L - s.c;
  const bool bad_len = s.L != 0 && (s.c > s.L || s.c > a.n || s.c < 0 || !rows_inside(a, b, s.c));
  const bool bad_table = static_cast<int64_t>(s.L) > static_cast<int64_t>(a.pool.table_cols) * a.pool.page_size;
  if (report && bad_len) raise_device_error(a.pool.err, kErrBadSeqlen);
  if (report && bad_table) raise_device_error(a.pool.err, kErrBadPage);
  s.ok = s.L > 0 && s.c > 0 && !bad_len && !bad_table;
  return s;
}

// Keys of a unit of rows [t0, t1): its union is [0, s_end) and [lo, hi).
struct UnitKeys {
  int s_end, lo, hi;
  int s_tiles, lo_tile, tiles;
  __device__ __forceinline__ int tile(int i) const { return i < s_tiles ? i : lo_tile + (i - s_tiles); }
  __device__ __forceinline__ bool wanted(int j) const { return j < hi && (j >= lo || j < s_end); }
};

__device__ __forceinline__ UnitKeys unit_keys(const PagedAttn& a, const Seq& s, int t0, int t1) {
  UnitKeys u;
  u.hi = a.parents ? s.L : s.P + t1;
  const int first = s.P + (a.parents ? 0 : t0);  // the smallest position of the unit's rows, at least
  u.lo = a.window ? max(0, first - a.window + 1) : 0;
  u.s_end = min(a.sinks, u.lo);
  const int up = (1 << a.bn_shift) - 1;
  u.lo_tile = u.lo >> a.bn_shift;
  u.s_tiles = min((u.s_end + up) >> a.bn_shift, u.lo_tile);
  u.tiles = u.s_tiles + ((u.hi + up) >> a.bn_shift) - u.lo_tile;
  return u;
}

// Rows [t0, t1) of row block qb; false when the block is past the sequence's rows.
__device__ __forceinline__ bool block_rows(const PagedAttn& a, const Seq& s, int qb, int& t0, int& t1) {
  const int r0 = qb * a.m, R = s.c * a.group;
  if (r0 >= R) return false;
  t0 = qb == 0 ? 0 : group_div(a, r0);
  t1 = r0 + a.m >= R ? s.c : group_div(a, r0 + a.m - 1) + 1;
  return true;
}

// Places of every row block of one (sequence, kv head).
__device__ __forceinline__ int head_places(const PagedAttn& a, const Seq& s) {
  int n = 0;
  int t0, t1;
  if (!s.ok) return 0;
  for (int qb = 0; block_rows(a, s, qb, t0, t1); ++qb) n += unit_keys(a, s, t0, t1).tiles + a.unit_cost;
  return n;
}

// A tile in the list.
struct TileCursor {
  int b, kvh, qb;
  int i;        // tile within the unit
  int t0, t1;   // the unit's new rows
  int at;       // the tile's place, counted from the CTA's first place
  Seq s;
  UnitKeys u;
  __device__ __forceinline__ int tile() const { return u.tile(i); }
  // To the unit after this one; false when there is none.
  __device__ __forceinline__ bool next_unit(const PagedAttn& a) {
    at += u.tiles - i + a.unit_cost;
    i = 0;
    ++qb;
    if (!block_rows(a, s, qb, t0, t1)) {
      qb = 0;
      if (++kvh == a.pool.hkv) {
        kvh = 0;
        do {
          if (++b >= a.pool.batch) return false;
          s = sequence(a, b, false);
        } while (!s.ok);
      }
      block_rows(a, s, qb, t0, t1);
    }
    u = unit_keys(a, s, t0, t1);
    return true;
  }
  // Whether the CTA, whose share ends at place `end`, has a tile after this unit.
  __device__ __forceinline__ bool more(const PagedAttn& a, int end) const { return at + u.tiles - i + a.unit_cost < end; }
  // To the next tile before place `end`; false when there is none.
  __device__ __forceinline__ bool next(const PagedAttn& a, int end) {
    if (i + 1 < u.tiles) {
      ++i;
      ++at;
      return at < end;
    }
    return more(a, end) && next_unit(a) && at < end;
  }
};

// The CTA's share of the list's T places, [g0, g1) (G CTAs have one), and its
// first tile (called by all THREADS threads of the CTA; `sh` is shared
// scratch); false when it has no tile.  Thread t counts the places of sequences
// [t * per, (t + 1) * per), a block scan places them, and the thread that
// owns g0 names its sequence.
struct ShareScratch {
  int warp_sum[32];
  int rem, b;
  Seq s;
};
struct Share {
  int g0, g1, T, G;  // (the planner keeps T below 2^31)
  // The first place of CTA c: c T / G, in 32 bits.
  __device__ __forceinline__ int start(int c) const {
    const uint32_t q = static_cast<uint32_t>(T) / static_cast<uint32_t>(G), r = static_cast<uint32_t>(T) - q * G;
    return static_cast<int>(c * q + c * r / static_cast<uint32_t>(G));  // (c r < G^2)
  }
};
template <int THREADS>
__device__ __forceinline__ bool cta_share(const PagedAttn& a, ShareScratch* sh, Share& r, TileCursor& cur) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.pool.batch + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, a.pool.batch), b1 = min(b0 + per, a.pool.batch);
  int mine = 0;
  Seq last{};
  for (int b = b0; b < b1; ++b) {
    last = sequence(a, b, blockIdx.x == 0);
    mine += head_places(a, last) * a.pool.hkv;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sh->warp_sum[warp] = incl;
  __syncthreads();
  int before = 0, T = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int x = sh->warp_sum[w];
    if (w < warp) before += x;
    T += x;
  }
  r.T = T;
  r.G = min(a.grid, T);
  const bool work = static_cast<int>(blockIdx.x) < r.G;
  r.g0 = work ? r.start(blockIdx.x) : T;
  r.g1 = work ? r.start(blockIdx.x + 1) : T;
  const int g0 = r.g0;
  const int start = before + incl - mine;
  if (work && g0 >= start && g0 < start + mine) {
    int rem = g0 - start;
    int b = b1 - 1;
    if (per > 1) {
      for (b = b0; b < b1 - 1; ++b) {
        const int n = head_places(a, sequence(a, b, false)) * a.pool.hkv;
        if (rem < n) break;
        rem -= n;
      }
      last = sequence(a, b, false);
    }
    sh->b = b;
    sh->rem = rem;
    sh->s = last;
  }
  __syncthreads();
  if (!work) return false;
  cur.b = sh->b;
  cur.s = sh->s;
  const uint32_t per_head = head_places(a, cur.s);
  cur.kvh = static_cast<int>(static_cast<uint32_t>(sh->rem) / per_head);
  int rem = sh->rem - cur.kvh * per_head;
  for (cur.qb = 0;; ++cur.qb) {
    block_rows(a, cur.s, cur.qb, cur.t0, cur.t1);
    cur.u = unit_keys(a, cur.s, cur.t0, cur.t1);
    if (rem < cur.u.tiles + a.unit_cost) break;
    rem -= cur.u.tiles + a.unit_cost;
  }
  cur.i = max(0, rem - a.unit_cost);
  cur.at = cur.i + a.unit_cost - rem;
  return cur.at < r.g1 - r.g0;
}

// CTA c's note for the merge; `cur` is at the CTA's first tile.  When the CTA
// starts inside a unit's tiles, the tile before is CTA c - 1's; the unit's
// first tile is too unless an earlier CTA names it.  CTA c - 1 began with this
// unit if its range starts in it (the place before a unit is a tile).
__device__ __forceinline__ void note_cut(const PagedAttn& a, bool work, const TileCursor& cur, const Share& r) {
  CutUnit n{};
  if (work && cur.i > 0) {
    const int c = blockIdx.x;
    const int first = r.g0 - cur.i, end = first + cur.u.tiles;  // places of the unit's tiles
    const int prev = r.start(c - 1);
    if (first >= prev) {
      int last = c;  // the CTA of place end - 1
      if (r.g1 < end) last = static_cast<int>((static_cast<int64_t>(end) * r.G - 1) / r.T);
      n = CutUnit{cur.b, cur.kvh, cur.qb, last - c + 2, prev >= first - a.unit_cost ? 0 : 1};
    }
  }
  a.cut[blockIdx.x] = n;
}

// Rows of sequences that have nothing to compute: zeros, log-sum-exp -inf.
template <typename T, int THREADS>
__device__ __forceinline__ void clear_unused(const PagedAttn& a) {
  for (int b = blockIdx.x; b < a.pool.batch; b += gridDim.x) {
    if (sequence(a, b, false).ok) continue;
    const int c = a.nr.count(b);
    if (c <= 0 || !rows_inside(a, b, c)) continue;
    const int64_t first = a.nr.cu ? a.nr.cu[b] : 0;
    T* out = reinterpret_cast<T*>(a.out) + (a.nr.cu ? 0 : b * a.o_sb);
    const int64_t values = static_cast<int64_t>(c) * a.hq * a.pool.d;
    for (int64_t e = threadIdx.x; e < values; e += THREADS) {
      const int d = static_cast<int>(e % a.pool.d);
      const int64_t rh = e / a.pool.d;
      const int64_t r = first + rh / a.hq, h = rh % a.hq;
      out[r * a.o_sn + h * a.o_sh + d] = Cvt<T>::from_f(0.f);
      if (a.lse && d == 0) a.lse[(a.nr.cu ? 0 : b * a.l_sb) + r * a.l_sn + h * a.l_sh] = -INFINITY;
    }
  }
}

// Ancestor bits of tree row i (bit j: new row j is visible to it) and its
// depth.  `bits` has (c + 31) / 32 words, zeroed.
__device__ __forceinline__ int tree_bits(const PagedAttn& a, const Seq& s, int b, int i, uint32_t* bits) {
  const int32_t* par = a.parents + static_cast<int64_t>(b) * a.par_sb;
  int cur = i, hop = 0;
  for (; hop <= s.c; ++hop) {
    const bool near = hop <= a.max_depth;
    const bool in = !a.window || hop < a.window || s.P + cur < a.sinks;
    if (near && in) bits[cur >> 5] |= 1u << (cur & 31);
    const int up = par[cur];
    if (up < -1 || up >= s.c) raise_device_error(a.pool.err, kErrBadParent);
    if (up < 0 || up >= s.c) break;
    cur = up;
  }
  return hop;
}

// f16 weights over 16-bit pages are taken against the running max less 7 (log2
// units): at most 2^15, as far up in f16 as they go, so that weights keep their bits
// down to 2^-21 of the largest and count down to 2^-32.  (A first key may take
// nearly all weight and hold next to nothing.)  bf16 has the range.
template <typename X, bool kWide>
__host__ __device__ constexpr float headroom() { return kWide && std::is_same_v<X, __half> ? 7.f : 0.f; }

// The unit of 8-bit rows' weights.  A weight (at most 2^8) times its V scale
// enters the products as f16, in units of 2^(e - kUnit), where its scale lies in
// [2^(e - 1 - kSpan), 2^e): it stays below 2^15, and what f16 takes off a weight
// is at most half a step of 2^-10 of it, or 2^-27 (half of f16's smallest step,
// at the smallest scale; a row's largest weight is 1 or more).  Rows outside that
// span are not taken by the products: they are added in fp32, so that a large
// row, seen or hidden, takes nothing from the small ones.  e follows the tiles up
// and down, but stays within kRise of the smallest scale met: above, what f16
// takes off a large row of little weight would count beside small rows of much.
// The output row follows e by exact powers of two in fp32, which holds it while e
// is within kReach of the largest scale met; scales that spread by more than both
// allow leave every row to fp32 (only terms below 2^-130 of the largest leave its
// range).  Scales below 2^-106, those of rows below 2^-100, do not count as
// small: rows of zeros have them.
// (Weights held below 2^4 and kUnit 11 would take 2^-31 off at most: 64-node trees
// over 16 x 8192 e4m3 rows took 22 us more, for the output row's corrections.)
constexpr int kUnit = 7, kSpan = 5, kRise = 10, kReach = 64;
constexpr int kNoExp = -116;  // nothing met yet
constexpr uint32_t kFloorBits = 21u << 23;  // 2^-106

__device__ __forceinline__ float pow2(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }
// The scale's bits above the floor's, for a minimum; wraps to the top below it.
__device__ __forceinline__ uint32_t above_floor(float scale) { return (__float_as_uint(scale) & 0x7fffffffu) - kFloorBits; }

struct VUnit {
  int e = kNoExp;                   // the unit's exponent
  int top = kNoExp, low = 1 << 20;  // the largest and smallest met (scale < 2^)
  bool closed = false;              // every row is outside
  // The tile's scales, largest `hi` (bits of a float) and smallest `lo`
  // (above_floor), lie within the unit's span.
  __device__ __forceinline__ bool fits(int hi, uint32_t lo) const {
    return !closed && hi < (e + 127) << 23 && lo >= static_cast<uint32_t>(max(e - kSpan + 126 - 21, 0)) << 23;
  }
  // A scale in units of 2^(e - kUnit) is outside the span (a NaN is not).
  static __device__ __forceinline__ bool outside(float f) {
    return fabsf(f) >= static_cast<float>(1 << kUnit) || fabsf(f) < static_cast<float>(1 << kUnit) / (2 << kSpan);
  }
  // Follows a tile; true when rows outside the span remain.
  __device__ __forceinline__ bool follow(int hi, uint32_t lo) {
    if (fits(hi, lo)) return false;
    const int e_hi = min((hi >> 23) - 126, 128);
    const int e_lo = lo >> 31 ? e_hi : static_cast<int>((lo + kFloorBits) >> 23) - 126;
    top = max(top, e_hi);
    if (!(lo >> 31)) low = min(low, e_lo);
    const int most = low + kRise;
    // a tile that spreads keeps the unit; the first one takes its large rows, unless they are too large
    const int want = e_hi - e_lo <= kSpan ? e_hi : e != kNoExp ? e : e_hi <= most ? e_hi : e_lo + kSpan;
    e = max(min(want, most), max(top - kReach, kNoExp));
    closed = e > most;
    return !fits(hi, lo);
  }
};

// Launches a kernel so that it may start while the one before it in the stream
// ends (it waits for that itself, by griddepcontrol.wait).
template <typename K, typename... More>
int launch_early(K kern, const PagedAttn& a, int threads, int smem, cudaStream_t st, int grid_y = 1, const More&... more) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.grid), static_cast<unsigned>(grid_y));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, more...), "gorgon_paged_attn launch");
}

int launch_paged_simt(const PagedAttn& a, cudaStream_t st);
int launch_paged_merge(const PagedAttn& a, cudaStream_t st);
// Tensor-core kernel for few packed rows per (sequence, kv head).
bool paged_mma_supported(const PagedAttn& a);
void paged_mma_plan(PagedAttn* a);
int launch_paged_mma(const PagedAttn& a, cudaStream_t st);
// tcgen05 kernel for many.
bool paged_tc_supported(const PagedAttn& a);
void paged_tc_plan(PagedAttn* a);
int launch_paged_tc(const PagedAttn& a, cudaStream_t st);

}  // namespace gorgon

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
// the host knowing any length.  A unit inside one CTA's range is finished
// there; one cut between CTAs leaves unnormalised fp32 rows with their running
// max and sum in the workspace, and paged_merge_kernel joins them in a fixed
// order, so results do not depend on timing.
#pragma once

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
  float scale_log2;   // softmax scale * log2(e)
  // tensor-core schedule
  int m, bn;          // packed rows per unit, positions per tile
  int qblocks;        // units per (sequence, kv head) at most
  int grid;
  float* part_o;      // [grid * 2][m][d]
  float2* part_ml;    // [grid * 2][m]  running max (log2 units) and sum
  int* tile_start;    // [batch + 1]
  uint64_t wait_ns;
};

// A sequence's state: P cached rows before its c new ones.
struct Seq {
  int L, c, P;
  bool ok;  // has rows to compute
};

__device__ __forceinline__ Seq sequence(const PagedAttn& a, int b, bool report) {
  Seq s;
  s.L = a.pool.lens[b];
  s.c = a.nr.count(b);
  s.P = s.L - s.c;
  const bool bad_len = s.L != 0 && (s.c > s.L || s.c > a.n || s.c < 0);
  const bool bad_table = static_cast<int64_t>(s.L) > static_cast<int64_t>(a.pool.table_cols) * a.pool.page_size;
  if (report && bad_len) raise_device_error(a.pool.err, kErrBadSeqlen);
  if (report && bad_table) raise_device_error(a.pool.err, kErrBadPage);
  s.ok = s.L > 0 && s.c > 0 && !bad_len && !bad_table;
  return s;
}

// What a row sees: position j <= hi, and (window) j >= lo or j < sinks; a tree
// row's hi is P - 1, and its own tree's rows go by its ancestor bits.
struct RowView {
  int hi, lo;
};

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
  u.lo_tile = u.lo / a.bn;
  u.s_tiles = min((u.s_end + a.bn - 1) / a.bn, u.lo_tile);
  u.tiles = u.s_tiles + (u.hi + a.bn - 1) / a.bn - u.lo_tile;
  return u;
}

// Rows [t0, t1) of row block qb; false when the block is past the sequence's rows.
__device__ __forceinline__ bool block_rows(const PagedAttn& a, const Seq& s, int qb, int& t0, int& t1) {
  const int r0 = qb * a.m, R = s.c * a.group;
  if (r0 >= R) return false;
  t0 = r0 / a.group;
  t1 = min(s.c, (min(r0 + a.m, R) - 1) / a.group + 1);
  return true;
}

// Tiles of every row block of one (sequence, kv head).
__device__ __forceinline__ int head_tiles(const PagedAttn& a, const Seq& s) {
  int n = 0, t0, t1;
  if (!s.ok) return 0;
  for (int qb = 0; block_rows(a, s, qb, t0, t1); ++qb) n += unit_keys(a, s, t0, t1).tiles;
  return n;
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
    if (up < 0) break;
    if (up >= s.c) {
      raise_device_error(a.pool.err, kErrBadParent);
      break;
    }
    cur = up;
  }
  return hop;
}

int launch_paged_simt(const PagedAttn& a, cudaStream_t st);

}  // namespace gorgon

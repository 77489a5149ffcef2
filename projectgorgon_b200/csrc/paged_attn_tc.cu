// Paged attention for many packed rows per (sequence, kv head): prompt chunks,
// draft trees.  tcgen05 products with TMEM accumulators.
//
// A unit is MT x 128 packed rows of one (sequence, kv head), row t * group + g;
// a tile is 64 positions of its cache.  One CTA per SM walks its share of the
// tile list (paged_attn.cuh).  Warp roles:
//   warp 0        Q K^T issuer (one thread)
//   warp 1        P V issuer (one thread); the warp allocates TMEM
//   warps 2, 3    TMA loads of K and V tiles (one thread each)
//   warps 4, 5    K, 32 rows of every tile each
//   warps 6, 7    V
//   warps 8 - 11  softmax and epilogue of M-tile 0, a thread per row
//   warps 12 - 15 (MT = 2) of M-tile 1
// Pages of 8, 16, 32 rows or a multiple of 64 come by TMA, a box per page (or
// per 64 rows of one) and 128-byte column block.  16-bit rows land in the SW128
// tiles that the products read.  8-bit rows land in a ring of raw bytes, and
// warps 4 to 7 widen their 32 rows from there to f16, exactly (paged_widen.cuh),
// so that the products see the stored numbers and the scales are applied in
// fp32: K's to the scores, V's to the weights (see VUnit; rows outside its span
// are added before the tile's product, add_far).  Pages of other sizes are
// gathered row by row by warps 4 to 7 with 16-byte cp.async copies (which took
// 1700 cycles a tile, most of them waiting for issue slots, so TMA is used where
// it can be).  V rows that no row of the unit sees are made zeros.
//
// Softmax per row is owned by one thread (TMEM lane = row): no shuffles.  The
// running max moves only when a tile's max exceeds it by more than 8 (log2
// units), which bounds weights by 2^8 and makes corrections of O rare.  Tiles
// that every row of the unit sees whole run a loop without masks.  In the
// others a 64-bit word per row says which columns it sees, and their V rows
// are searched for infinities and NaN (0 times those would reach every row):
// the search replaces them by zeros, and the epilogue adds them to the rows
// that do see them.
//
// Measured: 2048 new tokens over 32768 bf16 rows (32 heads on 8, 128 wide) 930 to
// 1026 us by the card's power, 1.04 to 1.14 PFLOP/s, the tensor pipe busy 75 % and
// the exponentials' 61 % of the time; 64-node trees of 16 sequences over 8192 e4m3
// rows 280 us with nothing saturated (shared memory 67 %, issue slots 42 %, tensor
// pipe 33 %): the producers' chain of wait, widening and hand-over; bf16 pages of 16
// rows cost 5 % over pages of 64.

// Every mbarrier wait is bounded; a wait that runs out raises kErrTimeout, and
// the CTA drains its copies and products, frees TMEM and returns.
#include <algorithm>
#include <type_traits>

#include <cuda.h>

#include <mutex>

#include "attn_tc_common.cuh"
#include "paged_attn.cuh"
#include "paged_widen.cuh"

namespace gorgon {
namespace {
using namespace sm100;

constexpr int kTile = 64;  // positions per tile
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0;    // + (buf * MT + mt) * kTile
constexpr uint32_t kColO = 256;  // + mt * D
constexpr int kMaxTree = 256;    // tree rows (8 words of ancestor bits)

template <typename T, int ST, int D_, int MT_>
struct TcCfg {
  static constexpr int D = D_, MT = MT_;
  static constexpr bool kWide = ST == GORGON_KV_NATIVE;
  using X = std::conditional_t<kWide, T, __half>;
  static constexpr int kHalves = D / 64;                 // 128-byte column blocks of a row
  static constexpr int M = MT * 128;
  static constexpr int kThreads = 256 + MT * 128;
  static constexpr uint32_t kQTile = kHalves * kQHalf;   // one M-tile of Q
  static constexpr uint32_t kBlock = kTile * 128;        // 64 rows of one column block
  static constexpr uint32_t kTileBytes = kHalves * kBlock;
  static constexpr int kStages = kWide ? (MT == 2 ? 4 : 5) : 3;
  static constexpr int kRawStages = kWide ? 0 : (MT == 2 ? 3 : 5);
  static constexpr uint32_t kRawRows = 32 * D;           // bytes of a producer's 32 rows
  static constexpr uint32_t kRawBytes = 2 * kRawRows + 768;  // a tile of K or V, and (cp.async) its scales, for each half
  static constexpr int kInfo = 8;                        // (more than the tiles a producer has in flight)
  static constexpr int kLag = kWide ? kStages - 2 : 0;   // tiles in flight behind the newest
  // With two M-tiles each softmax warpgroup frees a K stage once it has seen its
  // scores, which takes a commit off the Q K^T issuer, the busiest thread.
  static constexpr bool kSoftmaxFreesK = MT == 2;
  static constexpr uint32_t kOffK = MT * kQTile;
  static constexpr uint32_t kOffV = kOffK + kStages * kTileBytes;
  static constexpr uint32_t kOffRaw = kOffV + kStages * kTileBytes;         // [K, V][stages]
  static constexpr uint32_t kOffMeta = kOffRaw + 2 * kRawStages * kRawBytes;  // [stages] Meta
  static constexpr uint32_t kMetaBytes = kWide ? 16 : 16 + 8 * kTile;       // 2 words of valid keys, E, partly hidden; K and V factors
  static constexpr uint32_t kOffBits = kOffMeta + kStages * kMetaBytes;     // [M][8] ancestor words
  static constexpr uint32_t kOffQs = kOffBits + M * (kMaxTree / 32) * 4;    // [M] undoes Q's power of two
  static constexpr uint32_t kOffInfo = kOffQs + M * 4;                      // [4 producers][kInfo] valid keys, plain
  static constexpr uint32_t kOffCur = kOffInfo + 4 * kInfo * 8;             // [softmax warps] TileCursor
  static constexpr uint32_t kOffBar = (kOffCur + 4 * MT * static_cast<uint32_t>(sizeof(TileCursor)) + 15) / 16 * 16;
  static constexpr uint32_t kSmem = kOffBar + 512 + 1024;                   // + alignment slack
  static_assert(kSmem <= 232448, "shared memory per block");
};

template <typename C>
struct TcBars {
  uint64_t k_full[C::kStages], k_empty[C::kStages], v_full[C::kStages], v_empty[C::kStages];
  // TMA: 16-bit V tiles land, 8-bit K and V tiles land, and their raw bytes are done with
  uint64_t land[2][C::kWide ? C::kStages : C::kRawStages], raw_empty[2][C::kWide ? 1 : C::kRawStages];
  uint64_t q_full;
  uint64_t s_full[2 * C::MT], p_full[2 * C::MT];  // buf * MT + mt
  uint64_t p_free[2];            // every M-tile's P V of the buffer has completed
  int bad;   // a wanted page is out of the pool: tiles are checked for it
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort;
  int odd;  // bit 0: infinities or NaN were taken out of partly hidden V rows, bit 1: of a tile with a bad page
  ShareScratch sh;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
  const int n = take ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool take) {
  const int n = take ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// True on one lane of a converged warp, in a form that the compiler knows to be
// one: a TMA copy behind it is issued in a few cycles, behind `lane == 0` it took
// about 250 (2048 new tokens over 16384 rows in pages of 16: 574 -> 472 us).
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(yes));
  return yes != 0;
}

template <int N>
struct Slot {  // ring position
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

// The unit's positions that every row sees: [all_lo, all_hi], and the sinks.
struct Common {
  int all_hi, all_lo;
  __device__ __forceinline__ Common(const PagedAttn& a, const TileCursor& c) {
    all_hi = a.parents ? c.s.P - 1 : c.s.P + c.t0;
    const int last = c.s.P + (a.parents ? c.s.c : c.t1) - 1;
    all_lo = a.window ? max(0, last - a.window + 1) : 0;
  }
  __device__ __forceinline__ bool plain(const PagedAttn& a, int j0) const {
    return j0 + kTile - 1 <= all_hi && (j0 >= all_lo || j0 + kTile <= a.sinks);
  }
};

// Bits [lo, hi) of a 64-bit word, clipped to it.
__device__ __forceinline__ uint64_t bit_range(int lo, int hi) {
  lo = max(0, min(64, lo));
  hi = max(0, min(64, hi));
  if (lo >= hi) return 0;
  const uint64_t up = hi == 64 ? ~0ull : (1ull << hi) - 1;
  return up & ~((1ull << lo) - 1);
}

// ------------------------------------------------------------ tiles
// A producer's 32 rows of raw bytes (row-major at src) to the f16 tile at st;
// rows without their bit in `keep` become zeros.
template <int ST, typename C>
__device__ __forceinline__ void widen_rows(const uint8_t* src, uint8_t* st, int half, uint32_t keep) {
  constexpr int kRow = C::D, kCpr = kRow / 16, kRpi = 32 / kCpr;
  const int lane = threadIdx.x & 31, piece = lane % kCpr, rsub = lane / kCpr;
  uint8_t* blk = st + (piece >> 2) * C::kBlock;
#pragma unroll 4
  for (int it = 0; it < 32 / kRpi; ++it) {
    const int r = it * kRpi + rsub;
    uint4 w = *reinterpret_cast<const uint4*>(src + r * kRow + piece * 16);
    if (!((keep >> r) & 1u)) w = make_uint4(0, 0, 0, 0);
    uint32_t x[8];
    widen_word<ST>(w.x, x[0], x[1]);
    widen_word<ST>(w.y, x[2], x[3]);
    widen_word<ST>(w.z, x[4], x[5]);
    widen_word<ST>(w.w, x[6], x[7]);
    *reinterpret_cast<uint4*>(blk + sw128(half * 32 + r, (2 * piece) & 7)) = make_uint4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<uint4*>(blk + sw128(half * 32 + r, (2 * piece + 1) & 7)) = make_uint4(x[4], x[5], x[6], x[7]);
  }
}

// Takes infinities and NaN out of 32 rows of a 16-bit V tile (rows without their
// bit in `keep` become zeros); true on lanes that found some in kept rows.
template <typename T, typename C>
__device__ __forceinline__ bool strip_rows(uint8_t* st, int half, uint32_t keep) {
  constexpr int kCpr = C::D / 8, kRpi = 32 / kCpr;
  const int lane = threadIdx.x & 31, piece = lane % kCpr, rsub = lane / kCpr;
  bool odd = false;
#pragma unroll 4
  for (int it = 0; it < 32 / kRpi; ++it) {
    const int r = it * kRpi + rsub;
    uint4* w = reinterpret_cast<uint4*>(st + (piece >> 3) * C::kBlock + sw128(half * 32 + r, piece & 7));
    uint32_t x[4] = {w->x, w->y, w->z, w->w};
    constexpr uint32_t top = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
    const bool kept = (keep >> r) & 1u;
    bool here = !kept;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!kept) x[e] = 0;
      if ((x[e] & top) == top) {
        x[e] &= 0xffff0000u;
        odd = here = true;
      }
      if (((x[e] >> 16) & top) == top) {
        x[e] &= 0xffffu;
        odd = here = true;
      }
    }
    if (here) *w = make_uint4(x[0], x[1], x[2], x[3]);
  }
  return odd;
}

// What the softmax needs of a tile: the half's valid word, and (8-bit) K's scales
// times the softmax scale and V's scales in the unit of the tile (VUnit).  Both
// halves know all 64 V scales (`vs` its own, `vo` the other half's), and so the
// same unit.  Rows outside its span keep their factor; the softmax knows them by it.
constexpr uint32_t kFar = 2, kAllFar = 4;  // in the tile's word: it has such rows, all are
template <typename C>
__device__ __forceinline__ void write_meta(const PagedAttn& a, uint8_t* smem, uint32_t stage, int half, uint32_t valid, float ks, float vs,
                                           float vo, bool first, VUnit& unit, bool plain) {
  const int lane = threadIdx.x & 31;
  uint8_t* meta = smem + C::kOffMeta + stage * C::kMetaBytes;
  if (lane == 0) reinterpret_cast<uint32_t*>(meta)[half] = valid;
  if constexpr (!C::kWide) {
    if (first) unit = VUnit{};
    const float big = fmaxf(fmaxf(0.f, fabsf(vs)), fabsf(vo));  // (NaN never wins)
    const bool far = unit.follow(__reduce_max_sync(0xffffffffu, __float_as_int(big)),
                                 __reduce_min_sync(0xffffffffu, min(above_floor(vs), above_floor(vo))));
    // (each half says whether its rows are whole and seen by all, in its half of the word)
    if (lane == 0) reinterpret_cast<uint16_t*>(meta + 12)[half] = (plain && valid == 0xffffffffu ? 0 : 1) | (far ? kFar : 0) | (unit.closed ? kAllFar : 0);
    if (lane == 0 && half == 0) reinterpret_cast<int*>(meta)[2] = unit.e;
    reinterpret_cast<float*>(meta + 16)[half * 32 + lane] = ks * a.scale_log2;
    reinterpret_cast<float*>(meta + 16)[kTile + half * 32 + lane] = vs * pow2(kUnit - unit.e);
  }
}

// Rows of a page that one TMA box covers, 0 when pages of this size go row by row.
__host__ __device__ __forceinline__ int box_rows(int page_size) {
  return page_size % kTile == 0 ? kTile : page_size >= 8 && kTile % page_size == 0 ? page_size : 0;
}

// ------------------------------------------------------------ TMA loads
template <typename C>
__device__ void load_tiles(const PagedAttn& a, const CUtensorMap* map, TileCursor f, int end, uint8_t* smem, TcBars<C>* bars, int is_v) {
  constexpr int kSlots = C::kWide ? C::kStages : C::kRawStages;
  const int lane = threadIdx.x & 31;
  volatile int* abort = &bars->abort;
  uint64_t* full = C::kWide && !is_v ? bars->k_full : bars->land[is_v];
  uint64_t* empty = C::kWide ? (is_v ? bars->v_empty : bars->k_empty) : bars->raw_empty[is_v];
  uint8_t* ring = smem + (C::kWide ? (is_v ? C::kOffV : C::kOffK) : C::kOffRaw + is_v * C::kRawStages * C::kRawBytes);
  constexpr uint32_t kSlotBytes = C::kWide ? C::kTileBytes : C::kRawBytes;
  const int R = box_rows(a.pool.page_size), boxes = kTile / R;
  const uint32_t box_bytes = static_cast<uint32_t>(R) * (C::kWide ? C::D * 2 : C::D);
  // Page of box `lane` of a tile (-2: not wanted, -1: bad), and the tile's row in it
  // (a page smaller than a tile begins with its box).
  auto look_up = [&](int& row) {
    int page = -2;
    const int p = f.tile() * kTile + lane * R;
    if (lane < boxes && p < f.u.hi && (p + R > f.u.lo || p < f.u.s_end)) {
      int col;
      a.pool.split(p, col, row);
      page = max(-1, __ldg(a.pool.table + static_cast<int64_t>(f.b) * a.pool.table_sb + col));
    }
    return page;
  };
  int next_row = 0, next_page = look_up(next_row);
  Slot<kSlots> s;
  int64_t issued = 0;
  bool more = true;
  while (more) {
    const int page = next_page, row = __shfl_sync(0xffffffffu, next_row, 0), kvh = f.kvh;
    more = f.next(a, end);
    if (more) next_page = look_up(next_row);  // (in flight while this tile's boxes are sent)
    if (!warp_wait(&empty[s.stage], s.phase ^ 1u, abort, a.wait_ns)) break;
    const uint32_t go = __ballot_sync(0xffffffffu, page >= 0 && page < a.pool.num_pages);
    if (page != -2 && !((go >> lane) & 1u)) {
      raise_device_error(a.pool.err, kErrBadPage);
      *reinterpret_cast<volatile int*>(&bars->bad) = 1;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive_expect_tx(&full[s.stage], __popc(go) * box_bytes);
    __syncwarp();
    uint8_t* dst = ring + s.stage * kSlotBytes;
#pragma unroll 1
    for (int x = 0; x < boxes; ++x, dst += R * (C::kWide ? 128 : C::D)) {
      const int pg = __shfl_sync(0xffffffffu, page, x);
      if (((go >> x) & 1u) && elect_one()) {
        if constexpr (C::kWide) {
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h) tma_load_4d(dst + h * C::kBlock, map, &full[s.stage], h * 64, row, kvh, pg);
        } else {
          tma_load_4d(dst, map, &full[s.stage], 0, row, kvh, pg);
        }
      }
      __syncwarp();
    }
    __syncwarp();
    ++issued;
    s.next();
  }
  // Every issued load must land before the CTA leaves.
  if (lane == 0)
    for (int64_t k = issued > kSlots ? issued - kSlots : 0; k < issued; ++k)
      drain_wait(&full[k % kSlots], static_cast<uint32_t>(k / kSlots) & 1u);
}

// What is left to do for 32 rows of every tile that lands by TMA: their valid
// word and scales, hidden rows of 16-bit V, widening of 8-bit rows.
template <typename T, int ST, typename C>
__device__ void finish_tiles(const PagedAttn& a, TileCursor f, int end, uint8_t* smem, TcBars<C>* bars, int is_v, int half) {
  const int lane = threadIdx.x & 31;
  volatile int* abort = &bars->abort;
  uint64_t* full = is_v ? bars->v_full : bars->k_full;
  uint64_t* empty = is_v ? bars->v_empty : bars->k_empty;
  uint8_t* ring = smem + (is_v ? C::kOffV : C::kOffK);
  // This lane's row (and, for V's scales, the same row of the other half): its page
  // two tiles ahead, its scales one tile ahead, so that nothing waits for them.
  int page[2] = {-2, -2}, row[2] = {}, kvh = 0;
  bool next_first = true;
  auto look_up = [&]() {
    kvh = f.kvh;
#pragma unroll
    for (int k = 0; k < (C::kWide ? 1 : 2); ++k) {
      page[k] = -2;
      const int j = f.tile() * kTile + (k ? 1 - half : half) * 32 + lane;
      if (f.u.wanted(j)) {
        int col;
        a.pool.split(j, col, row[k]);
        page[k] = __ldg(a.pool.table + static_cast<int64_t>(f.b) * a.pool.table_sb + col);
      }
    }
  };
  bool held = false;
  float ks = 0.f, vs = 0.f, vo = 0.f;
  auto take = [&]() {  // the looked-up pages' validity and scales
    held = page[0] >= 0 && page[0] < a.pool.num_pages;
    if constexpr (!C::kWide) {
      ks = vs = vo = 0.f;
      if (is_v && held) {
        ks = __ldg(a.pool.ks + page[0] * a.pool.ks_sp + kvh * a.pool.ks_sh + row[0] * a.pool.ks_ss);
        vs = __ldg(a.pool.vs + page[0] * a.pool.vs_sp + kvh * a.pool.vs_sh + row[0] * a.pool.vs_ss);
      }
      if (is_v && page[1] >= 0 && page[1] < a.pool.num_pages)
        vo = __ldg(a.pool.vs + page[1] * a.pool.vs_sp + kvh * a.pool.vs_sh + row[1] * a.pool.vs_ss);
    }
  };
  VUnit unit;
  bool first = true;  // the tile is the unit's first here
  bool plain = Common(a, f).plain(a, f.tile() * kTile), next_plain = false;
  look_up();
  take();
  bool more = f.next(a, end);
  if (more) {
    next_plain = Common(a, f).plain(a, f.tile() * kTile);
    next_first = f.i == 0;
    look_up();
  }
  constexpr int kSlots = C::kWide ? C::kStages : C::kRawStages;
  Slot<kSlots> ls;
  Slot<C::kStages> hs;
  while (true) {
    const uint32_t valid = __ballot_sync(0xffffffffu, held);
    const float k1 = ks, v1 = vs, o1 = vo;
    const bool p1 = plain, f1 = first, again = more;
    if (more) {  // the next tile's scales, and the page of the one after
      take();
      plain = next_plain;
      first = next_first;
      more = f.next(a, end);
      if (more) {
        next_plain = Common(a, f).plain(a, f.tile() * kTile);
        next_first = f.i == 0;
        look_up();
      }
    }
    if (!warp_wait(&bars->land[is_v][ls.stage], ls.phase, abort, a.wait_ns)) return;
    uint8_t* st = ring + hs.stage * C::kTileBytes;
    if constexpr (C::kWide) {
      if (!(p1 && valid == 0xffffffffu)) {
        if (strip_rows<T, C>(st, half, valid)) atomicOr(&bars->odd, p1 ? 2 : 1);
        fence_proxy_async_smem();
      }
    } else {
      if (!warp_wait(&empty[hs.stage], hs.phase ^ 1u, abort, a.wait_ns)) return;
      const uint8_t* src = smem + C::kOffRaw + (is_v * C::kRawStages + ls.stage) * C::kRawBytes + half * C::kRawRows;
      widen_rows<ST, C>(src, st, half, is_v ? valid : 0xffffffffu);
      fence_proxy_async_smem();
    }
    if (is_v) write_meta<C>(a, smem, hs.stage, half, valid, k1, v1, o1, f1, unit, p1);
    __syncwarp();
    if (lane == 0) {
      if constexpr (!C::kWide) mbar_arrive(&bars->raw_empty[is_v][ls.stage]);
      mbar_arrive(&full[hs.stage]);
    }
    ls.next();
    hs.next();
    if (!again) return;
  }
}

// ------------------------------------------------------------ row by row
// One of the two warps that fetch K (is_v 0) or V rows; `half` picks its 32 of a tile's rows.
template <typename T, int ST, typename C>
__device__ void produce(const PagedAttn& a, TileCursor cur, int end, uint8_t* smem, TcBars<C>* bars, int is_v, int half) {
  const int lane = threadIdx.x & 31;
  volatile int* abort = &bars->abort;
  uint64_t* full = is_v ? bars->v_full : bars->k_full;
  uint64_t* empty = is_v ? bars->v_empty : bars->k_empty;
  uint8_t* ring = smem + (is_v ? C::kOffV : C::kOffK);
  uint8_t* raw = smem + C::kOffRaw + is_v * C::kRawStages * C::kRawBytes;
  const int64_t sp = is_v ? a.pool.v_sp : a.pool.k_sp, ss = is_v ? a.pool.v_ss : a.pool.k_ss, sh = is_v ? a.pool.v_sh : a.pool.k_sh;
  const char* pages = is_v ? a.pool.v : a.pool.k;
  constexpr int kRow = C::kWide ? C::D * 2 : C::D;       // bytes of a row
  constexpr int kCpr = kRow / 16, kRpi = 32 / kCpr;
  const int piece = lane % kCpr, rsub = lane / kCpr;

  // The fetch runs ahead of the hand-over by kLag tiles (16-bit) or by the raw ring (8-bit).
  constexpr int kAhead = C::kWide ? C::kLag : C::kRawStages - 1;
  // Of a fetched tile: which rows it has, and whether every row of the unit sees it whole.
  uint2* info = reinterpret_cast<uint2*>(smem + C::kOffInfo) + (is_v * 2 + half) * C::kInfo;
  static_assert(kAhead + 1 < C::kInfo, "info ring");
  TileCursor f = cur;
  bool more = true;
  int f_tile = 0;             // tiles fetched
  Slot<C::kStages> fs;        // (16-bit) the stage fetched into
  // The page of this lane's row of the next tile (-2: not wanted), looked up a tile ahead.
  int next_page = -2, next_row = 0, next_other = -2, next_other_row = 0;
  auto look_up = [&]() {
    auto one = [&](int j, int& pg, int& rw) {
      pg = -2;
      if (f.u.wanted(j)) {
        int col;
        a.pool.split(j, col, rw);
        pg = max(-1, __ldg(a.pool.table + static_cast<int64_t>(f.b) * a.pool.table_sb + col));
      }
    };
    one(f.tile() * kTile + half * 32 + lane, next_page, next_row);
    if (!C::kWide && is_v) one(f.tile() * kTile + (1 - half) * 32 + lane, next_other, next_other_row);
  };
  look_up();
  auto fetch = [&]() -> bool {
    if constexpr (C::kWide) {
      if (!warp_wait(&empty[fs.stage], fs.phase ^ 1u, abort, a.wait_ns)) return false;
    }
    int page = next_page;
    const int prow = next_row;
    [[maybe_unused]] const int other = next_other, other_row = next_other_row;
    if (page != -2 && (page < 0 || page >= a.pool.num_pages)) {
      raise_device_error(a.pool.err, kErrBadPage);
      *reinterpret_cast<volatile int*>(&bars->bad) = 1;  // before the tile is handed over
      page = -2;
    }
    const uint32_t valid = __ballot_sync(0xffffffffu, page >= 0);
    if (lane == 0)
      info[f_tile % C::kInfo] = make_uint2(valid, (Common(a, f).plain(a, f.tile() * kTile) ? 1u : 0u) | (f.i == 0 ? 2u : 0u));
    const int64_t off = page >= 0 ? page * sp + prow * ss : 0;
    const char* base = pages + f.kvh * sh + piece * 16;
#pragma unroll
    for (int it = 0; it < 32 / kRpi; ++it) {
      const int r = it * kRpi + rsub;
      const int64_t o = __shfl_sync(0xffffffffu, off, r);
      uint32_t at;
      if constexpr (C::kWide)
        at = smem_u32(ring + fs.stage * C::kTileBytes + (piece >> 3) * C::kBlock) + sw128(half * 32 + r, piece & 7);
      else
        at = smem_u32(raw + (f_tile % C::kRawStages) * C::kRawBytes) + half * C::kRawRows + r * kRow + piece * 16;
      cp16(at, base + o, (valid >> r) & 1u);
    }
    if constexpr (!C::kWide) {
      if (is_v) {  // its rows' K and V scales, and the other half's V scales
        const int64_t pg = page >= 0 ? page : 0, pr = page >= 0 ? prow : 0;
        const bool other_held = other >= 0 && other < a.pool.num_pages;
        const int64_t og = other_held ? other : 0, orow = other_held ? other_row : 0;
        const uint32_t at = smem_u32(raw + (f_tile % C::kRawStages) * C::kRawBytes) + 2 * C::kRawRows + half * 384 + lane * 4;
        cp4(at, a.pool.ks + pg * a.pool.ks_sp + f.kvh * a.pool.ks_sh + pr * a.pool.ks_ss, page >= 0);
        cp4(at + 128, a.pool.vs + pg * a.pool.vs_sp + f.kvh * a.pool.vs_sh + pr * a.pool.vs_ss, page >= 0);
        cp4(at + 256, a.pool.vs + og * a.pool.vs_sp + f.kvh * a.pool.vs_sh + orow * a.pool.vs_ss, other_held);
      }
    }
    cp_commit();
    if constexpr (C::kWide) fs.next();
    ++f_tile;
    more = f.next(a, end);
    if (more) look_up();
    return true;
  };
  Slot<C::kStages> hs;  // the stage handed over
  int done = 0;
  VUnit unit;
  // Hands tile `done` over: its copies have landed.
  auto hand_over = [&]() -> bool {
    const uint2 h = info[done % C::kInfo];
    uint8_t* st = ring + hs.stage * C::kTileBytes;
    __syncwarp();  // every lane's copies
    if constexpr (!C::kWide) {
      if (!warp_wait(&empty[hs.stage], hs.phase ^ 1u, abort, a.wait_ns)) return false;
      widen_rows<ST, C>(raw + (done % C::kRawStages) * C::kRawBytes + half * C::kRawRows, st, half, h.x);
    }
    if (is_v) {
      float ks = 0.f, vs = 0.f, vo = 0.f;
      if constexpr (!C::kWide) {
        const float* sc = reinterpret_cast<const float*>(raw + (done % C::kRawStages) * C::kRawBytes + 2 * C::kRawRows + half * 384);
        ks = sc[lane];
        vs = sc[32 + lane];
        vo = sc[64 + lane];
      } else if (!((h.y & 1u) && h.x == 0xffffffffu)) {
        if (strip_rows<T, C>(st, half, h.x)) atomicOr(&bars->odd, h.y & 1u ? 2 : 1);
      }
      write_meta<C>(a, smem, hs.stage, half, h.x, ks, vs, vo, done == 0 || (h.y & 2u), unit, h.y & 1u);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&full[hs.stage]);
    hs.next();
    ++done;
    return true;
  };
  bool ok = true;
  while (ok && more && f_tile < kAhead) ok = fetch();
  while (ok && more) {
    ok = fetch();
    if (!ok) break;
    cp_wait<kAhead>();
    ok = hand_over();
  }
  cp_wait<0>();
  while (ok && done < f_tile) ok = hand_over();
}

// ------------------------------------------------------------ issuers
// M-tiles of the cursor's unit that hold rows.
template <typename C>
__device__ __forceinline__ int live_tiles(const PagedAttn& a, const TileCursor& c) {
  return C::MT == 1 || c.s.c * a.group - c.qb * C::M <= 128 ? 1 : 2;
}

template <typename C>
__device__ void issue_scores(const PagedAttn& a, TileCursor cur, int end, uint8_t* smem, TcBars<C>* bars, uint32_t tmem, uint32_t fmt) {
  volatile int* abort = &bars->abort;
  const uint64_t q0 = umma_desc_sw128(smem_u32(smem), 16, 1024);
  const uint64_t k0 = umma_desc_sw128(smem_u32(smem + C::kOffK), 16, 1024);
  const uint32_t idesc = umma_idesc_f16(fmt, 128, kTile, 0, 0);
  Slot<C::kStages> kr;
  uint32_t i = 0, unit = 0;
  bool ok = true;
  while (ok) {
    if (!spin_wait(&bars->q_full, unit & 1u, abort, a.wait_ns)) break;
    ++unit;
    const int n = min(cur.u.tiles - cur.i, end - cur.at), live = live_tiles<C>(a, cur);
    for (int t = 0; t < n && ok; ++t, ++i) {
      // Both probes before either result is used: the round trips overlap when the
      // K tile and the S buffer (its weights of two tiles ago) are ready, as they usually are.
      const uint32_t pf = ((i - 2) >> 1) & 1u;
      const bool k_ready = mbar_test_wait(&bars->k_full[kr.stage], kr.phase);
      const bool p_ready = i < 2 || mbar_test_wait(&bars->p_free[i & 1u], pf);
      if (!(k_ready && p_ready) && (!spin_wait(&bars->k_full[kr.stage], kr.phase, abort, a.wait_ns) ||
                                    (i >= 2 && !spin_wait(&bars->p_free[i & 1u], pf, abort, a.wait_ns)))) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int mt = 0; mt < C::MT; ++mt) {
        if (mt < live)
#pragma unroll
        for (int ks = 0; ks < C::D / 16; ++ks)
          umma_f16_ss(tmem + kColS + ((i & 1u) * C::MT + mt) * kTile,
                      q0 + static_cast<uint64_t>((mt * C::kHalves + (ks >> 2)) * (kQHalf >> 4) + (ks & 3) * 2),
                      k0 + static_cast<uint64_t>(kr.stage * (C::kTileBytes >> 4) + (ks >> 2) * (C::kBlock >> 4) + (ks & 3) * 2), idesc,
                      ks > 0 ? 1u : 0u);
        umma_commit(&bars->s_full[(i & 1u) * C::MT + mt]);
        // The second M-tile's scores follow the first one's weights of the tile before, so
        // that the two warpgroups' exponentials and the P V products alternate.
        if (C::MT == 2 && mt == 0 && i > 0 && !spin_wait(&bars->p_full[((i - 1) & 1u) * C::MT], ((i - 1) >> 1) & 1u, abort, a.wait_ns)) {
          ok = false;
          break;
        }
      }
      if (!C::kSoftmaxFreesK) umma_commit(&bars->k_empty[kr.stage]);
      kr.next();
    }
    cur.at += n - 1;
    cur.i += n - 1;
    if (!ok || !cur.next(a, end)) break;
  }
  umma_commit(&bars->drain[0]);
  drain_wait(&bars->drain[0], 0);
}

template <typename C>
__device__ void issue_outputs(const PagedAttn& a, TileCursor cur, int end, uint8_t* smem, TcBars<C>* bars, uint32_t tmem, uint32_t fmt) {
  volatile int* abort = &bars->abort;
  const uint64_t v0 = umma_desc_sw128(smem_u32(smem + C::kOffV), C::kBlock, 1024);
  const uint32_t idesc = umma_idesc_f16(fmt, 128, C::D, 0, 1);
  Slot<C::kStages> vr;
  uint32_t i = 0;
  bool ok = true;
  while (ok) {
    const int n = min(cur.u.tiles - cur.i, end - cur.at), live = live_tiles<C>(a, cur);
    for (int t = 0; t < n && ok; ++t, ++i) {
      const uint32_t buf = i & 1u;
      if (!spin_wait(&bars->v_full[vr.stage], vr.phase, abort, a.wait_ns)) {
        ok = false;
        break;
      }
      for (int mt = 0; mt < C::MT; ++mt) {
        if (!spin_wait(&bars->p_full[buf * C::MT + mt], (i >> 1) & 1u, abort, a.wait_ns)) {
          ok = false;
          break;
        }
        if (mt >= live) continue;
        tc_fence_after();
        // A unit's output begins with its first product, or with what the softmax put there (add_far).
        const bool begun = t > 0 || (!C::kWide && (reinterpret_cast<const uint32_t*>(smem + C::kOffMeta + vr.stage * C::kMetaBytes)[3] & kFar));
#pragma unroll
        for (int ks = 0; ks < kTile / 16; ++ks)
          umma_f16_ts(tmem + kColO + mt * C::D, tmem + kColS + (buf * C::MT + mt) * kTile + ks * 8,
                      v0 + static_cast<uint64_t>(vr.stage * (C::kTileBytes >> 4) + ks * (2048 >> 4)), idesc, (ks > 0 || begun) ? 1u : 0u);
      }
      if (!ok) break;
      umma_commit(&bars->p_free[buf]);
      umma_commit(&bars->v_empty[vr.stage]);
      vr.next();
    }
    cur.at += n - 1;
    cur.i += n - 1;
    if (!ok || !cur.next(a, end)) break;
  }
  umma_commit(&bars->drain[1]);
  drain_wait(&bars->drain[1], 0);
}

// ------------------------------------------------------------ softmax
// Which columns of the tile at j0 the row sees.
__device__ __forceinline__ uint64_t row_word(const PagedAttn& a, const TileCursor& c, int pos, bool ok, const uint32_t* bits, int j0) {
  if (!ok) return 0;
  const int P = c.s.P;
  const int hi = a.parents ? P - 1 : pos;
  uint64_t w = bit_range(0, hi - j0 + 1);
  if (a.window) w &= bit_range(pos - a.window + 1 - j0, 64) | bit_range(0, a.sinks - j0);
  if (a.parents && j0 + 64 > P) {  // its own tree's columns by its ancestor bits
    const int o = j0 - P;          // the tile's first tree row (negative: the tree starts inside the tile)
    const int words = (c.s.c + 31) >> 5;
    auto word = [&](int k) -> uint64_t { return k >= 0 && k < words ? bits[k] : 0u; };
    const int k = o >> 5, sh = o & 31;  // floor
    uint64_t t = (word(k) | (word(k + 1) << 32)) >> sh;
    if (sh) t |= word(k + 2) << (64 - sh);
    w |= t;
  }
  return w;
}

// The rare correction of a warp's output rows before a tile's product: they are
// multiplied by alpha and regrade (or begin at 0, `fresh`), and the tile's columns
// whose rows lie outside the unit's span (`far`) are added, key by key from the V
// tile `v`.  x: a row's scores less its running max; `factor`: V's scales in the unit.
// Out of the loop's registers.
template <typename C>
__device__ __noinline__ void add_far(uint32_t o_addr, bool fresh, float alpha, float regrade, uint64_t far, const float* x,
                                     const uint8_t* v, const float* factor) {
#pragma unroll 1
  for (int c0 = 0; c0 < C::D; c0 += 32) {
    float o[32];
    if (fresh) {
#pragma unroll
      for (int k = 0; k < 32; ++k) o[k] = 0.f;
    } else {
      uint32_t ov[32];
      tmem_ld32(o_addr + c0, ov);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < 32; ++k) o[k] = __uint_as_float(ov[k]) * alpha * regrade;
    }
    const uint8_t* blk = v + (c0 >> 6) * C::kBlock;
#pragma unroll 1
    for (uint64_t rest = far; rest; rest &= rest - 1) {
      const int c = __ffsll(static_cast<long long>(rest)) - 1;
      const float p = ex2_approx(x[c]);
      if (!__any_sync(0xffffffffu, p != 0.f)) continue;  // (rows that were not fetched, too)
      const float w = p == 0.f ? 0.f : p * factor[c];    // (a hidden row's factor may be an infinity)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint4 b = *reinterpret_cast<const uint4*>(blk + sw128(static_cast<uint32_t>(c), static_cast<uint32_t>(((c0 & 63) >> 3) + q)));
        const uint32_t b4[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b4[e]));
          o[q * 8 + 2 * e] = fmaf(w, y.x, o[q * 8 + 2 * e]);
          o[q * 8 + 2 * e + 1] = fmaf(w, y.y, o[q * 8 + 2 * e + 1]);
        }
      }
    }
    uint32_t ov[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) ov[k] = __float_as_uint(o[k]);
    tmem_st32(o_addr + c0, ov);
  }
  tmem_wait_st();
}

template <typename T, int ST, typename C>
__device__ void softmax(const PagedAttn& a, const TileCursor& start, int end, uint8_t* smem, TcBars<C>* bars, uint32_t tmem) {
  using X = typename C::X;
  constexpr bool kScaleQ = !C::kWide && std::is_same_v<T, __nv_bfloat16>;
  constexpr float kHead = headroom<X, C::kWide>();
  constexpr int MT = C::MT, D = C::D;
  constexpr int kChunks = D / 8;          // 16-byte pieces of a 16-bit row
  constexpr int kRows = 32 / kChunks;     // rows that a warp instruction covers
  volatile int* abort = &bars->abort;
  const int wg = (threadIdx.x >> 7) - 2;  // M-tile
  const int wq = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int r = threadIdx.x & 127, qrow = wg * 128 + r;
  const uint32_t lane_base = tmem + (static_cast<uint32_t>(wq * 32) << 16);
  uint8_t* q_tile = smem + wg * C::kQTile;
  uint32_t* s_bits = reinterpret_cast<uint32_t*>(smem + C::kOffBits);
  float* s_qs = reinterpret_cast<float*>(smem + C::kOffQs);
  constexpr int kWords = kMaxTree / 32;
  const int chunk = lane % kChunks, rsub = lane / kChunks;
  // a row of the warp's 32: 16-byte pieces in the SW128 order of Q
  auto stage_row = [&](int rr, int j) -> uint8_t* {
    return q_tile + (j >> 3) * kQHalf + sw128(static_cast<uint32_t>(wq * 32 + rr), static_cast<uint32_t>(j & 7));
  };
  const bool vec_out = (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0 && ((a.o_sb | a.o_sh | a.o_sn) & 7) == 0;
  // The warp's cursor lives in shared memory: the loop over tiles needs little of it.
  TileCursor& cur = reinterpret_cast<TileCursor*>(smem + C::kOffCur)[(threadIdx.x >> 5) - 8];
  if (lane == 0) cur = start;
  __syncwarp();
  uint32_t i = 0;
  Slot<C::kStages> vr;
  bool first_unit = true;
  bool cut_start = cur.i > 0;
  while (true) {
    const int n = min(cur.u.tiles - cur.i, end - cur.at);
    const int R = cur.s.c * a.group;
    const int64_t first = a.nr.cu ? a.nr.cu[cur.b] : 0;
    const int pr = cur.qb * C::M + qrow;
    const bool row_ok = pr < R;
    const int t = row_ok ? group_div(a, pr) : cur.t0;
    const int h = cur.kvh * a.group + (row_ok ? pr - t * a.group : 0);
    // ---- Q rows -> shared memory; the previous unit's last product is complete
    {
      const char* qb = a.q + (a.nr.cu ? 0 : cur.b * a.q_sb) + first * a.q_sn + static_cast<int64_t>(cur.kvh) * a.group * a.q_sh;
      const int p0 = cur.qb * C::M + wg * 128 + wq * 32;
      if constexpr (!kScaleQ) {
#pragma unroll
        for (int k = 0; k < 32; k += kRows) {
          const int p = p0 + k + rsub;
          const int tt = group_div(a, p), gg = p - tt * a.group;
          cp16(smem_u32(stage_row(k + rsub, chunk)), p < R ? qb + tt * a.q_sn + gg * a.q_sh + chunk * 16 : qb, p < R);
        }
        cp_commit();
        cp_wait<0>();
      }
      constexpr int kBatch = 8;
#pragma unroll 1
      for (int k0 = kScaleQ ? 0 : 32; k0 < 32; k0 += kBatch * kRows) {
        uint4 qv[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int p = p0 + k0 + k * kRows + rsub;
          const int tt = group_div(a, p), gg = p - tt * a.group;
          qv[k] = p < R ? __ldg(reinterpret_cast<const uint4*>(qb + tt * a.q_sn + gg * a.q_sh) + chunk) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int rr = k0 + k * kRows + rsub;
          if constexpr (kScaleQ) {
            uint32_t x[4] = {qv[k].x, qv[k].y, qv[k].z, qv[k].w};
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max((x[e] << 16) & 0x7f800000u, x[e] & 0x7f800000u));
#pragma unroll
            for (int o = 1; o < kChunks; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e2 = max(static_cast<int>(top >> 23) - 127, -100);
            const float f = pow2(15 - e2);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[e] = pack16x2(__uint_as_float(x[e] << 16) * f, __uint_as_float(x[e] & 0xffff0000u) * f, false);
            qv[k] = make_uint4(x[0], x[1], x[2], x[3]);
            if (chunk == 0) s_qs[wg * 128 + wq * 32 + rr] = pow2(e2 - 15);
          }
          *reinterpret_cast<uint4*>(stage_row(rr, chunk)) = qv[k];
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full);
    }
    // ---- this row's ancestor bits.  The warp copies parents[] to its own rows' place
    // for the bits, every lane walks its row's chain there, and the bits go over it
    // (rows of one node repeat the walk, but no barrier stands between warps that
    // may give up a wait).
    int pos = cur.s.P + t;
    uint32_t* bits = s_bits + qrow * kWords;
    if (a.parents) {
      int32_t* par = reinterpret_cast<int32_t*>(s_bits + (wg * 128 + wq * 32) * kWords);
      const int32_t* src = a.parents + static_cast<int64_t>(cur.b) * a.par_sb;
      const int c = cur.s.c, P = cur.s.P;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        if (lane + 32 * k < c) par[lane + 32 * k] = __ldg(src + lane + 32 * k);
      __syncwarp();
      uint32_t word[kWords] = {};
      int at = row_ok ? t : -1, hop = 0;
      for (; at >= 0 && hop <= c; ++hop) {
        if (hop <= a.max_depth && (!a.window || hop < a.window || P + at < a.sinks)) {
#pragma unroll
          for (int k = 0; k < kWords; ++k)
            if ((at >> 5) == k) word[k] |= 1u << (at & 31);
        }
        const int up = par[at];
        if (up < -1 || up >= c) raise_device_error(a.pool.err, kErrBadParent);
        if (up < 0 || up >= c) break;
        at = up;
      }
      pos += hop - t;
      if (hop > c) pos = P + c;  // (a cycle: no position is its own)
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kWords; ++k) bits[k] = word[k];
      __syncwarp();
    }
    const Common common(a, cur);
    // (8-bit: K's factors hold the softmax scale)
    const float qs = C::kWide ? a.scale_log2 : kScaleQ ? s_qs[qrow] : 1.f;
    float m_used = -INFINITY, l = 0.f;
    int unit_exp = kNoExp;
    // One tile of this row: scores to weights against the lazy running max.
    auto tile = [&](auto mask_tag, auto far_tag, int j0, bool fresh) -> bool {
      constexpr bool kMask = decltype(mask_tag)::value, kHasFar = decltype(far_tag)::value;
      const uint32_t bi = (i & 1u) * MT + wg;
      [[maybe_unused]] const uint8_t* meta = smem + C::kOffMeta + vr.stage * C::kMetaBytes;
      if (kMask && C::kWide) {  // the tile's valid keys (8-bit: the caller waited for them and the scales)
        if (!warp_wait(&bars->v_full[vr.stage], vr.phase, abort, a.wait_ns)) return false;
      }
      uint64_t vw = ~0ull;
      if (kMask) vw = row_word(a, cur, pos, row_ok, bits, j0) & *reinterpret_cast<const uint64_t*>(meta);
      if (!warp_wait(&bars->s_full[bi], (i >> 1) & 1u, abort, a.wait_ns)) return false;
      if (!kMask && C::kWide && *reinterpret_cast<volatile int*>(&bars->bad)) return true;  // (the caller looks at it too)
      if (C::kSoftmaxFreesK && wq == 0 && lane == 0) mbar_arrive(&bars->k_empty[i % C::kStages]);
      tc_fence_after();
      const uint32_t s_addr = lane_base + kColS + bi * kTile;
      float x[kTile];
      {
        uint32_t rr[2][32];
        tmem_ld32(s_addr, rr[0]);
        tmem_ld32(s_addr + 32, rr[1]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < kTile; ++c) x[c] = __uint_as_float(rr[c >> 5][c & 31]);
      }
      // Wide: x stays the raw score.  8-bit: x becomes the score (in log2 units) less
      // the running max.
      [[maybe_unused]] const float base = C::kWide || m_used == -INFINITY ? 0.f : m_used;
      if constexpr (!C::kWide) {
        const float4* ks = reinterpret_cast<const float4*>(meta + 16);
        const uint64_t qb = f2_pack(qs, qs), nb = f2_pack(-base, -base);
#pragma unroll
        for (int c = 0; c < kTile; c += 4) {
          const float4 f = ks[c >> 2];
          uint64_t f0 = f2_pack(f.x, f.y), f1 = f2_pack(f.z, f.w);
          if (kScaleQ) {
            f0 = f2_mul(f0, qb);
            f1 = f2_mul(f1, qb);
          }
          f2_unpack(f2_fma(f2_pack(x[c], x[c + 1]), f0, nb), x[c], x[c + 1]);
          f2_unpack(f2_fma(f2_pack(x[c + 2], x[c + 3]), f1, nb), x[c + 2], x[c + 3]);
        }
      }
      if (kMask) {
        const uint32_t w[2] = {static_cast<uint32_t>(vw), static_cast<uint32_t>(vw >> 32)};
#pragma unroll
        for (int c = 0; c < kTile; ++c) x[c] = ((w[c >> 5] >> (c & 31)) & 1u) ? x[c] : -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < kTile; c += 2) mx[(c >> 1) & 3] = fmax3(mx[(c >> 1) & 3], x[c], x[c + 1]);
      const float top = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]);
      float alpha = 1.f;
      [[maybe_unused]] float regrade = 1.f;
      bool need = false;
      if constexpr (C::kWide) {
        const float tmax = top * qs - kHead;
        if (fresh) {
          m_used = tmax;
        } else if (tmax > m_used + 8.f) {
          alpha = ex2_approx(m_used - tmax);
          m_used = tmax;
          need = true;
        }
      } else {
        const bool move = fresh || m_used == -INFINITY ? top > -INFINITY : top > 8.f;
        if (__any_sync(0xffffffffu, move)) {
          const float d = move ? top : 0.f;
          if (move) {
            alpha = m_used == -INFINITY ? 0.f : ex2_approx(-d);
            m_used = base + d;
            need = !fresh;
          }
          const uint64_t d2 = f2_pack(-d, -d);
#pragma unroll
          for (int c = 0; c < kTile; c += 2) f2_unpack(f2_add(f2_pack(x[c], x[c + 1]), d2), x[c], x[c + 1]);
        }
      }
      l *= alpha;
      if constexpr (!C::kWide) {
        const int e = reinterpret_cast<const int*>(meta)[2];
        if (e != unit_exp) {
          const int half = (unit_exp - e) / 2;  // (the whole step may pass fp32's range)
          alpha *= pow2(half);
          regrade = pow2(unit_exp - e - half);
          unit_exp = e;
          need = !fresh;
        }
      }
      // Columns whose rows lie outside the unit's span: their scores are kept for add_far.
      [[maybe_unused]] uint64_t far = 0;
      [[maybe_unused]] float far_x[kHasFar ? kTile : 1];
      if constexpr (kHasFar) {
        const float* f = reinterpret_cast<const float*>(meta + 16) + kTile;
        const bool all = reinterpret_cast<const uint32_t*>(meta)[3] & kAllFar;
        far = __ballot_sync(0xffffffffu, all || VUnit::outside(f[lane])) |
              static_cast<uint64_t>(__ballot_sync(0xffffffffu, all || VUnit::outside(f[32 + lane]))) << 32;
#pragma unroll
        for (int c = 0; c < kTile; ++c) far_x[c] = x[c];
      }
      const float nmb = m_used == -INFINITY ? 0.f : -m_used;
      [[maybe_unused]] const uint64_t qs2 = f2_pack(qs, qs), nmb2 = f2_pack(nmb, nmb);
      uint64_t acc[4] = {0, 0, 0, 0};
      [[maybe_unused]] const float4* vs = reinterpret_cast<const float4*>(meta + 16 + 4 * kTile);
      // Weights go to TMEM 32 columns at a time (over this tile's scores, which are in
      // registers), so that few are held beside them.
#pragma unroll
      for (int c0 = 0; c0 < kTile; c0 += 32) {
      uint32_t packed[16];
#pragma unroll
      for (int c = c0; c < c0 + 32; c += 4) {
        float y[4] = {x[c], x[c + 1], x[c + 2], x[c + 3]};
        if constexpr (C::kWide) {
          f2_unpack(f2_fma(f2_pack(x[c], x[c + 1]), qs2, nmb2), y[0], y[1]);
          f2_unpack(f2_fma(f2_pack(x[c + 2], x[c + 3]), qs2, nmb2), y[2], y[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = ex2_approx(y[e]);
        uint64_t p0 = f2_pack(y[0], y[1]), p1 = f2_pack(y[2], y[3]);
        acc[(c >> 1) & 3] = f2_add(acc[(c >> 1) & 3], p0);
        acc[((c >> 1) + 1) & 3] = f2_add(acc[((c >> 1) + 1) & 3], p1);
        if constexpr (!C::kWide) {
          const float4 f = vs[c >> 2];
          p0 = f2_mul(p0, f2_pack(f.x, f.y));
          p1 = f2_mul(p1, f2_pack(f.z, f.w));
          float z[4];
          f2_unpack(p0, z[0], z[1]);
          f2_unpack(p1, z[2], z[3]);
          if (kMask) {  // a hidden key's weight is 0 whatever its scale
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = y[e] == 0.f || (kHasFar && ((far >> (c + e)) & 1u)) ? 0.f : z[e];
          }
          packed[(c - c0) >> 1] = pack16x2(z[0], z[1], false);
          packed[((c - c0) >> 1) + 1] = pack16x2(z[2], z[3], false);
        } else {
          packed[(c - c0) >> 1] = pack16x2(y[0], y[1], std::is_same_v<X, __nv_bfloat16>);
          packed[((c - c0) >> 1) + 1] = pack16x2(y[2], y[3], std::is_same_v<X, __nv_bfloat16>);
        }
      }
      tmem_st16(s_addr + (c0 >> 1), packed);
      }
      {
        float s0, s1;
        f2_unpack(f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3])), s0, s1);
        l += s0 + s1;
      }
      if (kHasFar || __any_sync(0xffffffffu, need)) {
        const uint32_t o_addr = lane_base + kColO + wg * D;
        if (!fresh) {  // (before a unit's first tile the epilogue has waited)
          const uint32_t pv = i - 1;
          if (!warp_wait(&bars->p_free[pv & 1u], (pv >> 1) & 1u, abort, a.wait_ns)) return false;
          tc_fence_after();
        }
        if constexpr (kHasFar) {
          add_far<C>(o_addr, fresh, alpha, regrade, far, far_x, smem + C::kOffV + vr.stage * C::kTileBytes,
                     reinterpret_cast<const float*>(meta + 16) + kTile);
        } else {
#pragma unroll
          for (int ch = 0; ch < D / 32; ++ch) {
            uint32_t ov[32];
            tmem_ld32(o_addr + ch * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(C::kWide ? __uint_as_float(ov[c]) * alpha : __uint_as_float(ov[c]) * alpha * regrade);
            tmem_st32(o_addr + ch * 32, ov);
          }
          tmem_wait_st();
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[bi]);
      vr.next();
      return true;
    };
    // Whether the warp has rows in this unit: its lanes of the products are not read otherwise.
    auto live = [&]() { return cur.qb * C::M + wg * 128 + wq * 32 < cur.s.c * a.group; };
    const uint32_t done = i + n;
    if (!live()) {
      for (; i < done; ++i) {
        const uint32_t bi = (i & 1u) * MT + wg;
        if (!warp_wait(&bars->s_full[bi], (i >> 1) & 1u, abort, a.wait_ns)) return;
        if (lane == 0) {
          if (C::kSoftmaxFreesK && wq == 0) mbar_arrive(&bars->k_empty[i % C::kStages]);
          mbar_arrive(&bars->p_full[bi]);
        }
        vr.next();
      }
    }
#pragma unroll 1
    for (int k = 0; i < done; ++k, ++i) {
      if constexpr (C::kWide) {
        // (a plain tile lacks keys only where a page is bad, which is known before its scores are)
        const uint32_t stage = vr.stage;
        const int j0 = cur.u.tile(cur.i + k) * kTile;
        if (common.plain(a, j0) && !tile(std::false_type(), std::false_type(), j0, k == 0)) return;
        if (vr.stage == stage && !tile(std::true_type(), std::false_type(), j0, k == 0)) return;
      } else {
        if (!warp_wait(&bars->v_full[vr.stage], vr.phase, abort, a.wait_ns)) return;
        const uint32_t word = reinterpret_cast<const uint32_t*>(smem + C::kOffMeta + vr.stage * C::kMetaBytes)[3];
        if (word == 0) {
          if (!tile(std::false_type(), std::false_type(), 0, k == 0)) return;
        } else if (!(word & kFar)) {
          if (!tile(std::true_type(), std::false_type(), cur.u.tile(cur.i + k) * kTile, k == 0)) return;
        } else {
          if (!tile(std::true_type(), std::true_type(), cur.u.tile(cur.i + k) * kTile, k == 0)) return;
        }
      }
    }
    // ---- epilogue
    const uint32_t lastv = i - 1;
    if (!warp_wait(&bars->p_free[lastv & 1u], (lastv >> 1) & 1u, abort, a.wait_ns)) return;
    tc_fence_after();
    const bool has_rows = live();
    const bool whole = cur.i + n == cur.u.tiles && !cut_start;
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (first_unit ? 0 : 1);
    const uint32_t o_addr = lane_base + kColO + wg * D;
    const float back = C::kWide ? 1.f : pow2(unit_exp - kUnit);
    const bool none = m_used == -INFINITY && !(whole && l != 0.f);  // nothing but hidden keys (l: NaN where a score was)
    const float f = whole ? back / l : back;
    const int odd = C::kWide ? *reinterpret_cast<volatile int*>(&bars->odd) : 0;
    // Adds what the producers took out of partly hidden V rows to a row that sees
    // it: columns [c0, c0 + 32), key by key from the pages.
    auto put_back = [&](int c0, float (&v)[32]) {
      for (int k = 0; k < n; ++k) {
        const int j0 = cur.u.tile(cur.i + k) * kTile;
        if (!(odd & 2) && common.plain(a, j0)) continue;
        const uint64_t see = row_word(a, cur, pos, row_ok, bits, j0);
        for (int j = j0; j < j0 + kTile; ++j) {
          if (!((see >> (j - j0)) & 1ull) || !cur.u.wanted(j)) continue;
          int col, prow;
          a.pool.split(j, col, prow);
          const int page = a.pool.page(cur.b, col);
          if (page < 0) continue;
          const T* src = reinterpret_cast<const T*>(a.pool.v + page * a.pool.v_sp + cur.kvh * a.pool.v_sh + prow * a.pool.v_ss) + c0;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float y = Cvt<T>::to_f(src[c]);
            if (!(fabsf(y) < INFINITY)) v[c] += y;
          }
        }
      }
    };
    T* out = reinterpret_cast<T*>(a.out) + (a.nr.cu ? 0 : cur.b * a.o_sb);
    // Rows go out through the warp's staging rows (its slice of the Q tile, free
    // now), so that a store instruction writes whole rows: 16-bit rows in one
    // pass, the fp32 rows of a piece in two.
    constexpr int kPass = kChunks * 4;  // fp32 columns that a staging row holds
    float* part = a.part_o + (slot * C::M + wg * 128 + wq * 32) * D;
#pragma unroll
    for (int ch = 0; ch < D / 32; ++ch) {
      if (!has_rows) break;
      uint32_t ov[32];
      tmem_ld32(o_addr + ch * 32, ov);
      tmem_wait_ld();
      float v[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = none ? 0.f : __uint_as_float(ov[c]) * f;
      if (odd) put_back(ch * 32, v);
      if (!whole) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          *reinterpret_cast<float4*>(stage_row(lane, (ch * 32 % kPass) / 4 + u)) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        if ((ch + 1) * 32 % kPass == 0) {
          __syncwarp();
#pragma unroll 4
          for (int k = 0; k < 32; k += kRows)
            *reinterpret_cast<float4*>(part + (k + rsub) * D + (ch * 32 / kPass) * kPass + chunk * 4) =
                *reinterpret_cast<const float4*>(stage_row(k + rsub, chunk));
          __syncwarp();
        }
      } else if (vec_out) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = pack16x2(v[8 * u + 2 * e], v[8 * u + 2 * e + 1], std::is_same_v<T, __nv_bfloat16>);
          *reinterpret_cast<uint4*>(stage_row(lane, ch * 4 + u)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else if (row_ok) {
#pragma unroll
        for (int c = 0; c < 32; ++c) out[h * a.o_sh + (first + t) * a.o_sn + ch * 32 + c] = Cvt<T>::from_f(v[c]);
      }
    }
    if (!has_rows) {
    } else if (whole) {
      if (vec_out) {
        __syncwarp();
        const int p0 = cur.qb * C::M + wg * 128 + wq * 32;
        T* ob = out + first * a.o_sn + static_cast<int64_t>(cur.kvh) * a.group * a.o_sh + chunk * 8;
#pragma unroll 4
        for (int k = 0; k < 32; k += kRows) {
          const int p = p0 + k + rsub;
          const int tt = group_div(a, p), gg = p - tt * a.group;
          const uint4 w = *reinterpret_cast<const uint4*>(stage_row(k + rsub, chunk));
          if (p < R) *reinterpret_cast<uint4*>(ob + tt * a.o_sn + gg * a.o_sh) = w;
        }
        __syncwarp();
      }
      if (row_ok && a.lse)
        a.lse[(a.nr.cu ? 0 : cur.b * a.l_sb) + h * a.l_sh + (first + t) * a.l_sn] = (m_used + log2f(l)) * 0.6931471805599453f;
    } else {
      a.part_ml[slot * C::M + qrow] = make_float2(m_used, l);
    }
    first_unit = cut_start = false;
    __syncwarp();
    int more = 0;
    if (lane == 0) {
      TileCursor c = cur;
      c.at += n - 1;
      c.i += n - 1;
      more = c.next(a, end);
      cur = c;
    }
    if (!__shfl_sync(0xffffffffu, more, 0)) return;
    __syncwarp();
  }
}

template <typename T, int ST, int D, int MT>
__global__ void __launch_bounds__(TcCfg<T, ST, D, MT>::kThreads, 1) paged_tc_kernel(const __grid_constant__ PagedAttn a,
                const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = TcCfg<T, ST, D, MT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcBars<C>* bars = reinterpret_cast<TcBars<C>*>(smem + C::kOffBar);
  static_assert(sizeof(TcBars<C>) <= 1024, "barrier block");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.tma && (warp == 2 || warp == 3) && lane == 0) prefetch_tensormap(warp == 3 ? &vmap : &kmap);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars->k_full[s], a.tma && C::kWide ? 1 : 2);  // the TMA thread, or the two warps of its rows
      mbar_init(&bars->k_empty[s], C::kSoftmaxFreesK ? MT : 1);
      mbar_init(&bars->v_full[s], 2);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int v = 0; v < 2; ++v)
      for (int s = 0; s < (C::kWide ? C::kStages : C::kRawStages); ++s) {
        mbar_init(&bars->land[v][s], 1);
        if (!C::kWide) mbar_init(&bars->raw_empty[v][s], 2);
      }
    mbar_init(&bars->q_full, 4 * MT);
    for (int b = 0; b < 2 * MT; ++b) {
      mbar_init(&bars->s_full[b], 1);
      mbar_init(&bars->p_full[b], 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->p_free[b], 1);
      mbar_init(&bars->drain[b], 1);
    }
    bars->bad = 0;
    bars->abort = 0;
    bars->odd = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  // Launched while the kernel before it ends; nothing is read before that has.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Share share;
  TileCursor cur;
  const bool work = cta_share<C::kThreads>(a, &bars->sh, share, cur);
  if (threadIdx.x == 0) note_cut(a, work, cur, share);
  clear_unused<T, C::kThreads>(a);
  const int end = static_cast<int>(share.g1 - share.g0);
  constexpr uint32_t fmt = std::is_same_v<typename C::X, __nv_bfloat16> ? 1u : 0u;
  if (warp < 8) {
    if (work) {
      if (warp == 0) {
        if (elect_one()) issue_scores<C>(a, cur, end, smem, bars, tmem, fmt);
      } else if (warp == 1) {
        // (elected, P V goes out too closely packed for the exponentials beside it: pages of 16 rows 469 -> 514 us)
        if (lane == 0) issue_outputs<C>(a, cur, end, smem, bars, tmem, fmt);
      } else if (warp < 4) {
        if (a.tma) load_tiles<C>(a, warp == 3 ? &vmap : &kmap, cur, end, smem, bars, warp - 2);
      } else if (a.tma) {
        if (!C::kWide || warp >= 6) finish_tiles<T, ST, C>(a, cur, end, smem, bars, (warp - 4) >> 1, warp & 1);
      } else {
        produce<T, ST, C>(a, cur, end, smem, bars, (warp - 4) >> 1, warp & 1);
      }
    }
  } else {
    if (work) softmax<T, ST, C>(a, cur, end, smem, bars, tmem);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (bars->abort && threadIdx.x == 0) raise_device_error(a.pool.err, kErrTimeout);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  });
  return fn;
}

// The pages of K or V as a 4-D tensor (column, row in the page, head, page);
// false where TMA does not take the layout, and rows are gathered instead.
bool page_map(const PagedAttn& a, bool v, CUtensorMap* map) {
  EncodeFn enc = encoder();
  if (!enc || a.pool.num_pages < 1) return false;
  const bool wide = a.pool.storage == GORGON_KV_NATIVE;
  const int64_t sp = v ? a.pool.v_sp : a.pool.k_sp, sh = v ? a.pool.v_sh : a.pool.k_sh, ss = v ? a.pool.v_ss : a.pool.k_ss;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.pool.d), static_cast<cuuint64_t>(a.pool.page_size),
                              static_cast<cuuint64_t>(a.pool.hkv), static_cast<cuuint64_t>(a.pool.num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(ss), static_cast<cuuint64_t>(sh), static_cast<cuuint64_t>(sp)};
  const cuuint32_t box[4] = {wide ? 64u : static_cast<cuuint32_t>(a.pool.d), static_cast<cuuint32_t>(box_rows(a.pool.page_size)), 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType dt = !wide ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : a.pool.dtype == GORGON_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, dt, 4, v ? a.pool.v : a.pool.k, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             wide ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename F>
int by_config(const PagedAttn& a, F&& f) {
  auto rows = [&](auto t, auto s, auto d) {
    return a.m == 128 ? f(t, s, d, std::integral_constant<int, 1>()) : f(t, s, d, std::integral_constant<int, 2>());
  };
  auto dims = [&](auto t, auto s) {
    return a.pool.d == 128 ? rows(t, s, std::integral_constant<int, 128>()) : rows(t, s, std::integral_constant<int, 64>());
  };
  auto store = [&](auto t) {
    switch (a.pool.storage) {
      case GORGON_KV_NATIVE: return dims(t, std::integral_constant<int, GORGON_KV_NATIVE>());
      case GORGON_KV_INT8: return dims(t, std::integral_constant<int, GORGON_KV_INT8>());
      default: return dims(t, std::integral_constant<int, GORGON_KV_E4M3>());
    }
  };
  return a.pool.dtype == GORGON_BF16 ? store(__nv_bfloat16{}) : store(__half{});
}

}  // namespace

bool paged_tc_supported(const PagedAttn& a) { return paged_mma_supported(a) && !(a.parents && a.n > kMaxTree); }

void paged_tc_plan(PagedAttn* a) {
  const int64_t rows = static_cast<int64_t>(a->n) * a->group;
  a->m = rows <= 128 ? 128 : 256;
  a->bn_shift = 6;
  a->qblocks = static_cast<int>(ceil_div(rows, a->m));
  a->unit_cost = 4;
  const int64_t keys = static_cast<int64_t>(a->pool.table_cols) * a->pool.page_size;
  const int64_t tiles = static_cast<int64_t>(a->pool.batch) * a->pool.hkv * a->qblocks * std::max<int64_t>(1, ceil_div(keys, kTile));
  a->grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count(), tiles)));
}

int launch_paged_tc(const PagedAttn& args, cudaStream_t st) {
  PagedAttn a = args;
  CUtensorMap kmap{}, vmap{};
  a.tma = box_rows(a.pool.page_size) > 0 && page_map(a, false, &kmap) && page_map(a, true, &vmap);
  return by_config(a, [&](auto t, auto s, auto d, auto mt) {
    using C = TcCfg<decltype(t), decltype(s)::value, decltype(d)::value, decltype(mt)::value>;
    auto kern = paged_tc_kernel<decltype(t), decltype(s)::value, decltype(d)::value, decltype(mt)::value>;
    constexpr int smem = C::kSmem + 512;
    static_assert(smem <= 232448, "shared memory per block");
    int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "gorgon_paged_attn smem attribute");
    if (rc) return rc;
    return launch_early(kern, a, C::kThreads, smem, st, 1, kmap, vmap);
  });
}

}  // namespace gorgon

// Paged attention for few packed rows per (sequence, kv head): single tokens of
// grouped heads, short drafts.  Bound by the bytes of the cache where it holds 16
// bits (16 x 8192 rows 98 us, 0.83 of measured HBM), by latency where it holds 8.
//
// Two CTAs per SM walk their shares of the tile list (paged_attn.cuh).  A tile is
// one group of 16 or 32 keys for each warp, and the warps work on their own:
// each streams its groups' K and V rows into its own ring of shared memory
// with 16-byte cp.async copies (three stages of 8 KB a warp, about 200 KB an SM
// in flight or in use, well above what covers the memory latency) and keeps
// its own running softmax, so there is no barrier in the loop.  Rows are
// gathered one by one, so pages may be of any size and stride; the table entry
// of a group is fetched one group ahead.  (Bulk copies of a row, which would
// need fewer instructions, are issued lane by lane: they took more.)
//
// Products run on mma.sync m16n8k16 with the keys as M: S^T = K Q^T and
// O^T = V^T P^T, so that a tile is 16 keys by 8 packed rows and a group of up to
// 8 query heads fills it (with the rows as M, half of every product and of the
// softmax was padding).  P^T's fragment is S^T's transposed, by movmatrix.
// 8-bit rows are widened in registers to f16, exactly, whatever the type of
// Q: f16 takes the fewest instructions per value.  The K scale is applied to
// the score and the V scale to the weight, in fp32 (see VUnit).  bf16 queries enter as f16
// times a power of two per row that puts the row's largest value at 2^15 or above, just
// inside f16: exact, but for values below 2^-32 of it.  So that a thread widens whole 16-byte pieces, the head
// dimension is taken in another order than the fragments': thread c of a quad
// holds values 16 (c + 4 i) + 4 s .. + 3 for K step (i, s), Q in the same
// order, and row r of output tile t is value D / 8 (r % 8) + 2 t + r / 8.
//
// At the end of a unit the warps' rows meet in shared memory.
//
// Measured (with the merge): 16 sequences of up to 8192 int8 rows, 32 heads on 8,
// 46 us, 2.9 TB/s with every byte read once; 24 of up to 16384 e4m3 rows in a
// window of 4096 52 us, 3.5 TB/s; one of 2048 bf16 rows 12 us, of which 3.5 are
// the merge's launch and most of the rest the schedule and the first loads.
#include <type_traits>

#include "paged_attn.cuh"
#include "paged_widen.cuh"

namespace gorgon {
namespace {

constexpr int kCtasPerSm = 2;
constexpr int kRedFloats = 2480;

template <typename T, int ST, int D_, int NT_>
struct Cfg {
  static constexpr int D = D_, NT = NT_;
  static constexpr bool kWide = ST == GORGON_KV_NATIVE;  // 16-bit pages
  using X = std::conditional_t<kWide, T, __half>;        // type of the products' operands
  static constexpr int kRowBytes = kWide ? D * 2 : D;
  static constexpr int KB = kRowBytes == 256 ? 1 : 2;    // blocks of 16 keys per group
  static constexpr int G = 16 * KB;                      // keys per warp and tile
  // A stage: K rows, V rows, the group's two words, then K and V scales.
  static constexpr int kHalf = G * kRowBytes;
  static constexpr int kOffWord = 2 * kHalf;
  static constexpr int kStage = kOffWord + (kWide ? 16 : 16 + 8 * G);
  // Two CTAs an SM, so that one's unit ends (barriers, the next unit's Q) pass
  // under the other's loads.
  static constexpr int kWarps = 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStages = kRowBytes == 64 ? 6 : 3;
  static constexpr int BN = G * kWarps;
  static constexpr int M = 8 * NT;
  // 16-byte pieces: kCpr to a row, kRpi rows to a copy instruction.  Piece p of
  // row r lies at p ^ (r % 8) (rows of 64 bytes: p ^ (r / 2 % 4)), so that a
  // fragment's reads meet no bank twice; a lane's pieces follow one of
  // kSwizzles patterns.
  static constexpr int kCpr = kRowBytes / 16, kRpi = 32 / kCpr, kSwizzles = kRpi >= 8 ? 1 : 8 / kRpi;
  static __device__ __forceinline__ uint32_t at(int row, int piece) {
    if constexpr (kCpr >= 8) return static_cast<uint32_t>(row * kCpr + (piece ^ (row & 7))) * 16u;
    return static_cast<uint32_t>(row * kCpr + (piece ^ ((row >> 1) & (kCpr - 1)))) * 16u;
  }
  static constexpr int kRing = kStages * kStage;
  // The block where the warps' rows meet; before that, the scratch of the
  // schedule, and while a unit runs, its tree's bits and depths and the warps'
  // maxima and sums.
  static constexpr int kOffRed = kWarps * kRing;
  static constexpr int kOffBits = kOffRed;                                  // [M][32] ancestor words
  static constexpr int kOffDepth = kOffBits + M * (kPagedMaxNodes / 32) * 4;
  static constexpr int kOffMl = kOffRed + 4096;                             // [warps][M] max, sum
  static_assert(kOffDepth + M * 4 <= kOffMl && kOffMl + kWarps * M * 8 <= kOffRed + kRedFloats * 4, "shared block");
  static constexpr int kOffRow = kOffRed + kRedFloats * 4;                  // [M] max, sum over the warps
  static constexpr int kOffCur = kOffRow + M * 8;                           // TileCursor of the unit worked on, and each warp's of the unit fetched
  static constexpr int kSmem = kOffCur + (kWarps + 1) * static_cast<int>(sizeof(TileCursor));
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
  const int n = take ? 16 : 0;  // 0: zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool take) {
  const int n = take ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// What the loop does rarely lives in calls, so that the loop itself stays short
// and in the instruction cache.

// Bit 4 nt + e: the thread's score (nt, e) is hidden.  `row` is the first of its
// packed rows, j[] its two keys' positions, held[] whether they were fetched.
__device__ __noinline__ uint32_t hidden_scores(const PagedAttn& a, const TileCursor* cur, const uint32_t* bits,
                                               const int* depth, int row, int tiles, int j0, int j1, bool held0, bool held1) {
  uint32_t out = 0;
  const int P = cur->s.P, R = cur->s.c * a.group;
  for (int k = 0; k < tiles * 4; ++k) {
    const int pr = row + (k >> 2) * 8 + (k & 1), j = k & 2 ? j1 : j0;
    bool see = (k & 2 ? held1 : held0) && pr < R;
    if (see) {
      const int t = group_div(a, pr);
      if (a.parents && j >= P) {
        see = j - P < cur->s.c && ((bits[(t - cur->t0) * (kPagedMaxNodes / 32) + ((j - P) >> 5)] >> ((j - P) & 31)) & 1u);
      } else {
        const int pos = P + (a.parents ? depth[t - cur->t0] : t);
        see = j <= pos && (!a.window || j > pos - a.window || j < a.sinks);
      }
    }
    out |= see ? 0u : 1u << k;
  }
  return out;
}

// A cursor in shared memory to the next unit (one lane); its `at` is `end` or
// more when the CTA has no tile there.
__device__ __noinline__ void step_unit(const PagedAttn& a, TileCursor* cur, int end) {
  TileCursor n = *cur;
  n.at += n.u.tiles - 1 - n.i;
  n.i = n.u.tiles - 1;
  if (!n.next(a, end)) n.at = end;
  *cur = n;
}

template <typename T, int ST, int D, int NT>
__global__ void __launch_bounds__(Cfg<T, ST, D, NT>::kThreads, kCtasPerSm) paged_mma_kernel(const __grid_constant__ PagedAttn a) {
  using C = Cfg<T, ST, D, NT>;
  using X = typename C::X;
  constexpr int KB = C::KB, G = C::G;
  constexpr uint32_t kAll = G == 32 ? 0xffffffffu : (1u << (G & 31)) - 1u;
  constexpr bool kScaleQ = !C::kWide && std::is_same_v<T, __nv_bfloat16>;
  constexpr float kHead = headroom<X, C::kWide>();
  extern __shared__ __align__(128) uint8_t smem[];
  static_assert(sizeof(ShareScratch) <= kRedFloats * 4, "scratch");
  ShareScratch* sh = reinterpret_cast<ShareScratch*>(smem + C::kOffRed);
  // Launched while the kernel before it ends; nothing is read before that has.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  Share share;
  TileCursor first_tile;
  const bool work = cta_share<C::kThreads>(a, sh, share, first_tile);
  if (threadIdx.x == 0) note_cut(a, work, first_tile, share);
  clear_unused<T, C::kThreads>(a);
  if (!work) return;

  uint8_t* ring = smem + warp * C::kRing;
  const uint32_t ring_s = smem_addr(ring);
  uint32_t* s_bits = reinterpret_cast<uint32_t*>(smem + C::kOffBits);
  int* s_depth = reinterpret_cast<int*>(smem + C::kOffDepth);
  float* s_red = reinterpret_cast<float*>(smem + C::kOffRed);
  float2* s_ml = reinterpret_cast<float2*>(smem + C::kOffMl);
  float2* s_row = reinterpret_cast<float2*>(smem + C::kOffRow);
  // The unit being worked on, and the unit whose tiles are being fetched.  They
  // live in shared memory: the loop needs little of them.
  TileCursor& cur = *reinterpret_cast<TileCursor*>(smem + C::kOffCur);
  TileCursor& ahead = reinterpret_cast<TileCursor*>(smem + C::kOffCur)[1 + warp];
  if (threadIdx.x == 0) cur = first_tile;
  if (lane == 0) ahead = first_tile;
  __syncthreads();

  // ---- loads: `page` is the page of key lane % G of the next tile to fetch
  // (-2: not wanted), fetched when the cursor got there.  A stage's words say
  // which keys it holds, and the first one's position with, in the top bit,
  // whether every row of the unit sees them all.
  constexpr uint32_t kPlain = 1u << 31;
  bool cut_start = first_tile.i > 0;  // the CTA's first unit began in another CTA
  const int end = static_cast<int>(share.g1 - share.g0);
  UnitKeys u;              // of `ahead`
  int tile = 0, left = 0;  // the tile to fetch, and how many of the unit's are left to fetch with it
  bool more = false;       // the CTA has tiles of a later unit
  int page = -2, prow = 0;
  const bool in_pages = a.pool.page_size % 16 == 0;  // 16 keys from a multiple of 16 on lie in one page
  const int piece = lane % C::kCpr, rsub = lane / C::kCpr;
  uint32_t swizzled[C::kSwizzles];
#pragma unroll
  for (int k = 0; k < C::kSwizzles; ++k) swizzled[k] = C::at(k * C::kRpi + rsub, piece) - k * C::kRpi * C::kRowBytes;
  const uint32_t k_sp = static_cast<uint32_t>(a.pool.k_sp), v_sp = static_cast<uint32_t>(a.pool.v_sp);
  const uint32_t k_ss = static_cast<uint32_t>(a.pool.k_ss), v_ss = static_cast<uint32_t>(a.pool.v_ss);
  // per unit: the head's rows, and the positions that every row of the unit sees, [all_lo, all_hi] and the sinks before
  // it (the rows' last position is at most last: a tree row's depth is below c)
  const char *kb = nullptr, *vb = nullptr;
  const float *ksb = nullptr, *vsb = nullptr;
  const int32_t* tb = nullptr;
  int all_hi = 0, all_lo = 0;
  auto enter = [&]() {
    u = ahead.u;
    tile = ahead.i;
    left = min(u.tiles - tile, end - ahead.at);
    more = ahead.more(a, end);
    kb = a.pool.k + ahead.kvh * a.pool.k_sh + piece * 16;
    vb = a.pool.v + ahead.kvh * a.pool.v_sh + piece * 16;
    if constexpr (!C::kWide) {
      ksb = a.pool.ks + ahead.kvh * a.pool.ks_sh;
      vsb = a.pool.vs + ahead.kvh * a.pool.vs_sh;
    }
    tb = a.pool.table + static_cast<int64_t>(ahead.b) * a.pool.table_sb;
    all_hi = a.parents ? ahead.s.P - 1 : ahead.s.P + ahead.t0;
    const int last = ahead.s.P + (a.parents ? ahead.s.c : ahead.t1) - 1;
    all_lo = a.window ? max(0, last - a.window + 1) : 0;
  };
  auto look_up = [&]() {
    page = -2;
    const int j = u.tile(tile) * C::BN + warp * G + (lane & (G - 1));
    if (u.wanted(j)) {
      int col;
      a.pool.split(j, col, prow);
      page = max(-1, __ldg(tb + col));  // col is inside: L fits the table
    }
  };
  auto issue = [&](int stage) {
    if (left > 0) {
      const bool held = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pool.num_pages);
      if (page != -2 && !held) raise_device_error(a.pool.err, kErrBadPage);
      const uint32_t valid = __ballot_sync(0xffffffffu, held) & kAll;
      const uint32_t dst = ring_s + stage * C::kStage;
      const int j0 = u.tile(tile) * C::BN + warp * G;
      const bool plain = valid == kAll && j0 + G - 1 <= all_hi && (j0 >= all_lo || j0 + G <= a.sinks);
      if (lane == 0)
        *reinterpret_cast<uint2*>(ring + stage * C::kStage + C::kOffWord) =
            make_uint2(valid, static_cast<uint32_t>(j0) | (plain ? kPlain : 0u));
      if (valid) {
        if (in_pages) {
#pragma unroll
          for (int kbk = 0; kbk < KB; ++kbk) {
            const uint32_t mine = (valid >> (16 * kbk)) & 0xffffu;
            const int src = __ffs(mine | 0x10000u) - 1;  // a wanted key of the block: its page is the block's
            const uint32_t pg = __shfl_sync(0xffffffffu, page, 16 * kbk + (src & 15));
            const uint32_t r0 = __shfl_sync(0xffffffffu, prow, 16 * kbk + (src & 15)) - (src & 15) + rsub;
            const char* kr = kb + static_cast<uint64_t>(pg) * k_sp + static_cast<uint64_t>(r0) * k_ss;
            const char* vr = vb + static_cast<uint64_t>(pg) * v_sp + static_cast<uint64_t>(r0) * v_ss;
            if (mine == 0xffffu) {
#pragma unroll
              for (int it = 0; it < 16 / C::kRpi; ++it) {
                const uint32_t at = dst + (kbk * 16 + it * C::kRpi) * C::kRowBytes + swizzled[it % C::kSwizzles];
                cp16(at, kr + it * C::kRpi * static_cast<uint64_t>(k_ss), true);
                cp16(at + C::kHalf, vr + it * C::kRpi * static_cast<uint64_t>(v_ss), true);
              }
            } else {
#pragma unroll 1
              for (int it = 0; it < 16 / C::kRpi; ++it) {
                const bool take = (mine >> (it * C::kRpi + rsub)) & 1u;
                const uint32_t at = dst + C::at(kbk * 16 + it * C::kRpi + rsub, piece);
                cp16(at, take ? kr + it * C::kRpi * static_cast<uint64_t>(k_ss) : kb, take);
                cp16(at + C::kHalf, take ? vr + it * C::kRpi * static_cast<uint64_t>(v_ss) : vb, take);
              }
            }
          }
        } else {
          const uint32_t pg = held ? page : 0, pr = held ? prow : 0;
          const uint64_t ko = static_cast<uint64_t>(pg) * k_sp + static_cast<uint64_t>(pr) * k_ss;
          const uint64_t vo = static_cast<uint64_t>(pg) * v_sp + static_cast<uint64_t>(pr) * v_ss;
#pragma unroll 1
          for (int it = 0; it < G / C::kRpi; ++it) {
            const int r = it * C::kRpi + rsub;
            const bool take = (valid >> r) & 1u;
            const uint32_t at = dst + C::at(r, piece);
            cp16(at, kb + __shfl_sync(0xffffffffu, ko, r), take);
            cp16(at + C::kHalf, vb + __shfl_sync(0xffffffffu, vo, r), take);
          }
        }
        if constexpr (!C::kWide) {
          static_assert(C::kWide || G == 32, "a lane for each key's scales");
          const uint32_t pg = held ? page : 0, pr = held ? prow : 0;
          const uint32_t at = dst + C::kOffWord + 16 + lane * 4;
          cp4(at, ksb + static_cast<uint64_t>(pg) * static_cast<uint32_t>(a.pool.ks_sp) + static_cast<uint64_t>(pr) * static_cast<uint32_t>(a.pool.ks_ss), held);
          cp4(at + 4 * G, vsb + static_cast<uint64_t>(pg) * static_cast<uint32_t>(a.pool.vs_sp) + static_cast<uint64_t>(pr) * static_cast<uint32_t>(a.pool.vs_ss), held);
        }
      }
      ++tile;
      if (--left == 0 && more) {
        if (lane == 0) step_unit(a, &ahead, end);
        __syncwarp();
        more = false;
        if (ahead.at < end) enter();
        __syncwarp();
      }
      if (left > 0) look_up();
    }
    cp_commit();
  };
  enter();
  look_up();
#pragma unroll 1
  for (int k = 0; k < C::kStages; ++k) issue(k);

  // ---- the unit's state.  A thread's rows are nt * 8 + 2 c + {0, 1} for scores
  // and output, nt * 8 + g for Q.
  uint32_t qf[NT][D / 16][2];
  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2], qscale[NT][2];
  VUnit vunit;  // of the warp's weights times V scales
  float unit_scale = 1.f;
  bool first_unit = true;
  int stage = 0;
  while (true) {
    const int in_unit = min(cur.u.tiles - cur.i, end - cur.at);  // of the unit, in this CTA
    if (a.parents) {
      for (int k = threadIdx.x; k < C::M * (kPagedMaxNodes / 32); k += C::kThreads) s_bits[k] = 0;
      __syncthreads();
      for (int t = cur.t0 + threadIdx.x; t < cur.t1; t += C::kThreads)
        s_depth[t - cur.t0] = tree_bits(a, cur.s, cur.b, t, s_bits + (t - cur.t0) * (kPagedMaxNodes / 32));
      __syncthreads();
    }
    {
      const int R = cur.s.c * a.group;
      const int64_t first = a.nr.cu ? a.nr.cu[cur.b] : 0;
      const char* qb = a.q + (a.nr.cu ? 0 : cur.b * a.q_sb);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int pr = cur.qb * C::M + nt * 8 + g;
        const bool ok = pr < R;
        const int t = ok ? group_div(a, pr) : 0;
        const int h = cur.kvh * a.group + (ok ? pr - t * a.group : 0);
        const char* row = qb + (first + t) * a.q_sn + static_cast<int64_t>(h) * a.q_sh;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          if constexpr (C::kWide) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(row + ks * 32) + c;
            qf[nt][ks][0] = ok ? __ldg(w) : 0u;
            qf[nt][ks][1] = ok ? __ldg(w + 4) : 0u;
          } else {
            const int d = (c + 4 * (ks >> 2)) * 16 + (ks & 3) * 4;
            const uint2 w = ok ? __ldg(reinterpret_cast<const uint2*>(row + d * 2)) : make_uint2(0u, 0u);
            qf[nt][ks][0] = w.x;
            qf[nt][ks][1] = w.y;
          }
        }
        float back = 1.f;  // undoes the power of two below, for row g
        if constexpr (kScaleQ) {
          uint32_t top = 0;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int k = 0; k < 2; ++k) top = max(top, max(qf[nt][ks][k] << 16 & 0x7f800000u, qf[nt][ks][k] & 0x7f800000u));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // (an infinity or a NaN stays one; a row below 2^-100 is small enough to enter as it is scaled for 2^-100)
          const int e = max(static_cast<int>(top >> 23) - 127, -100);
          const float f = pow2(15 - e);
          back = pow2(e - 15);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              qf[nt][ks][k] = pack2(__uint_as_float(qf[nt][ks][k] << 16) * f, __uint_as_float(qf[nt][ks][k] & 0xffff0000u) * f, __half{});
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[nt][e] = -INFINITY;
          l[nt][e] = 0.f;
          qscale[nt][e] = a.scale_log2 * (kScaleQ ? __shfl_sync(0xffffffffu, back, (2 * c + e) * 4) : 1.f);
        }
#pragma unroll
        for (int t2 = 0; t2 < D / 16; ++t2)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][t2][e] = 0.f;
      }
      vunit = VUnit{};
      unit_scale = pow2(kUnit - kNoExp);
    }

#pragma unroll 1
    for (int done = 0; done < in_unit; ++done) {
      uint8_t* st = ring + stage * C::kStage;
      const uint32_t st_s = ring_s + stage * C::kStage;
      cp_wait<C::kStages - 1>();
      __syncwarp();
      const uint2 word = *reinterpret_cast<const uint2*>(st + C::kOffWord);
      if (word.x) {
        const uint32_t valid = word.x;
        const int j0 = static_cast<int>(word.y & ~kPlain);
        const bool plain = word.y & kPlain;
        float x[KB][NT][4];  // S^T of a block: key g of row 2 c, of row 2 c + 1, key g + 8 of both
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[b][nt][e] = 0.f;
        // ---- scores
        if constexpr (C::kWide) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              uint32_t k[4];
              ldsm4(k, st_s + C::at(b * 16 + (lane & 15), ks * 2 + (lane >> 4)));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma(x[b][nt], k, qf[nt][ks][0], qf[nt][ks][1], X{});
            }
        } else {
#pragma unroll
          for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              const uint4 w0 = *reinterpret_cast<const uint4*>(st + C::at(b * 16 + g, c + 4 * i));
              const uint4 w1 = *reinterpret_cast<const uint4*>(st + C::at(b * 16 + g + 8, c + 4 * i));
              const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                uint32_t k[4];
                widen_word<ST>(u0[s], k[0], k[2]);
                widen_word<ST>(u1[s], k[1], k[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(x[b][nt], k, qf[nt][i * 4 + s][0], qf[nt][i * 4 + s][1], X{});
              }
            }
        }
        // ---- softmax
        const float* sc = reinterpret_cast<const float*>(st + C::kOffWord + 16);
        float vsc[KB][2];
        uint32_t slow = 0;  // keys whose rows are added one by one: those outside the unit's span, or (16-bit) all
        if constexpr (!C::kWide) {
          float top = 0.f;
          uint32_t low = 0xffffffffu;
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              vsc[b][hh] = sc[G + b * 16 + hh * 8 + g];  // (0 for keys that were not fetched)
              top = fmaxf(top, fabsf(vsc[b][hh]));        // (NaN never wins)
              low = min(low, above_floor(vsc[b][hh]));
            }
          if (__any_sync(0xffffffffu, !vunit.fits(__float_as_int(top), low))) {
            const int was = vunit.e;
            const bool far = vunit.follow(__reduce_max_sync(0xffffffffu, __float_as_int(top)), __reduce_min_sync(0xffffffffu, low));
            if (far) slow = __ballot_sync(0xffffffffu, vunit.closed || vunit.outside(sc[G + lane] * pow2(kUnit - vunit.e)));
            if (vunit.e != was) {
              unit_scale = pow2(kUnit - vunit.e);
              const int half = (was - vunit.e) / 2;  // (the whole step may pass fp32's range)
              const float r0 = pow2(half), r1 = pow2(was - vunit.e - half);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < D / 16; ++t)
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[nt][t][e] = o[nt][t][e] * r0 * r1;
            }
          }
        }
        bool move = false;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const float k0 = C::kWide ? 1.f : sc[b * 16 + g], k1 = C::kWide ? 1.f : sc[b * 16 + 8 + g];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[b][nt][e] *= C::kWide ? qscale[nt][e & 1] : qscale[nt][e & 1] * (e < 2 ? k0 : k1);
        }
        uint32_t hidden[KB] = {};
        if (!plain) {
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            const int k0 = b * 16 + g;
            hidden[b] = hidden_scores(a, &cur, s_bits, s_depth, cur.qb * C::M + 2 * c, NT, j0 + k0, j0 + k0 + 8, (valid >> k0) & 1u,
                                      (valid >> (k0 + 8)) & 1u);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((hidden[b] >> (4 * nt + e)) & 1u) x[b][nt][e] = -INFINITY;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(x[0][nt][e], x[0][nt][e + 2]);
            if constexpr (KB == 2) top = fmaxf(top, fmaxf(x[KB - 1][nt][e], x[KB - 1][nt][e + 2]));
            move |= top > m[nt][e] + (8.f + kHead);
          }
        // The running max moves only when a score exceeds it by 8 (log2 units), so
        // the usual group needs no shuffles and no rescaling.  (m is the max less kHead.)
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float alpha[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = -INFINITY;
#pragma unroll
              for (int b = 0; b < KB; ++b) top = fmaxf(top, fmaxf(x[b][nt][e], x[b][nt][e + 2]));
              top = fmaxf(top - kHead, m[nt][e]);
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
              alpha[e] = ex2(m[nt][e] - (top == -INFINITY ? 0.f : top));
              m[nt][e] = top;
              l[nt][e] *= alpha[e];
            }
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
              o[nt][t][0] *= alpha[0];
              o[nt][t][1] *= alpha[1];
              o[nt][t][2] *= alpha[0];
              o[nt][t][3] *= alpha[1];
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float base = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
              x[b][nt][e] = ex2(x[b][nt][e] - base);
              x[b][nt][e + 2] = ex2(x[b][nt][e + 2] - base);
              l[nt][e] += x[b][nt][e] + x[b][nt][e + 2];
            }
          }
        // ---- a partly hidden group of 16-bit rows: 0 * infinity must not reach a row that does not see it
        if constexpr (C::kWide) {
          if (!plain) {
            bool odd = false;
            for (int it = lane; it < G * C::kCpr; it += 32) {
              const uint4 w = *reinterpret_cast<const uint4*>(st + C::kHalf + it * 16);
              constexpr uint32_t top = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
              const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) odd |= (ww[e] & top) == top || ((ww[e] >> 16) & top) == top;
            }
            if (__any_sync(0xffffffffu, odd)) slow = kAll;
          }
        }
        // ---- output rows
        if (slow) {
          // Keys one at a time on the CUDA cores.  The weights go over the K rows, which are done with.
          float* w = reinterpret_cast<float*>(st);
          static_assert(C::M * G * 4 <= C::kHalf, "weights fit the K block");
          __syncwarp();
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[(nt * 8 + 2 * c + (e & 1)) * G + b * 16 + g + 8 * (e >> 1)] =
                    (hidden[b] >> (4 * nt + e)) & 1u ? -1.f : x[b][nt][e];
          __syncwarp();
#pragma unroll 1
          for (uint32_t rest = slow; rest; rest &= rest - 1) {
            const int k = __ffs(rest) - 1;
            const float f = C::kWide ? 1.f : sc[G + k] * unit_scale;
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                float v;
                if constexpr (C::kWide) {
                  v = Cvt<T>::to_f(*(reinterpret_cast<const T*>(st + C::kHalf + C::at(k, 2 * t + hh)) + g));
                } else {
                  const int d = g * (D / 8) + 2 * t + hh;
                  v = byte_value<ST>(st[C::kHalf + C::at(k, d >> 4) + (d & 15)]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float p = w[(nt * 8 + 2 * c + e) * G + k];
                    if (!(p < 0.f)) o[nt][t][2 * hh + e] = fmaf(C::kWide ? p : p * f, v, o[nt][t][2 * hh + e]);
                  }
              }
          }
        }
        if (!C::kWide || !slow) {
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                float p0 = x[b][nt][2 * hh], p1 = x[b][nt][2 * hh + 1];
                if constexpr (!C::kWide) {
                  const float f = vsc[b][hh] * unit_scale;
                  // (a hidden key's weight is 0 whatever its scale)
                  const bool done = slow && ((slow >> (b * 16 + hh * 8 + g)) & 1u);
                  p0 = done || (!plain && p0 == 0.f) ? 0.f : p0 * f;
                  p1 = done || (!plain && p1 == 0.f) ? 0.f : p1 * f;
                }
                pf[nt][hh] = transpose8(pack2(p0, p1, X{}));
              }
            if constexpr (C::kWide) {
#pragma unroll
              for (int t = 0; t < D / 16; ++t) {
                uint32_t v[4];
                ldsm4t(v, st_s + C::kHalf + C::at(b * 16 + (lane & 7) + ((lane >> 4) << 3), t * 2 + ((lane >> 3) & 1)));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(o[nt][t], v, pf[nt][0], pf[nt][1], X{});
              }
            } else {
              uint32_t w[4][D / 32];  // keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9: D / 8 values from g on
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int key = b * 16 + (k >> 1) * 8 + 2 * c + (k & 1);
                if constexpr (D == 128) {
                  const uint4 r = *reinterpret_cast<const uint4*>(st + C::kHalf + C::at(key, g));
                  w[k][0] = r.x;
                  w[k][1] = r.y;
                  w[k][2] = r.z;
                  w[k][3] = r.w;
                } else {
                  const uint2 r = *reinterpret_cast<const uint2*>(st + C::kHalf + C::at(key, g >> 1) + (g & 1) * 8);
                  w[k][0] = r.x;
                  w[k][1] = r.y;
                }
              }
#pragma unroll
              for (int q = 0; q < D / 32; ++q) {
                const uint32_t v0[4] = {widen<ST, 0, 4>(w[0][q], w[1][q]), widen<ST, 1, 5>(w[0][q], w[1][q]),
                                        widen<ST, 0, 4>(w[2][q], w[3][q]), widen<ST, 1, 5>(w[2][q], w[3][q])};
                const uint32_t v1[4] = {widen<ST, 2, 6>(w[0][q], w[1][q]), widen<ST, 3, 7>(w[0][q], w[1][q]),
                                        widen<ST, 2, 6>(w[2][q], w[3][q]), widen<ST, 3, 7>(w[2][q], w[3][q])};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma(o[nt][2 * q], v0, pf[nt][0], pf[nt][1], X{});
                  mma(o[nt][2 * q + 1], v1, pf[nt][0], pf[nt][1], X{});
                }
              }
            }
          }
        }
      }
      __syncwarp();  // every lane is done with the stage
      issue(stage);
      stage = stage + 1 == C::kStages ? 0 : stage + 1;
    }

    // ---- the end of the unit, or of the CTA's part of it
    const bool unit_done = cur.i + in_unit == cur.u.tiles;
    const bool whole = unit_done && !cut_start;
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (first_unit ? 0 : 1);
    const int R = cur.s.c * a.group;
    const int64_t first = a.nr.cu ? a.nr.cu[cur.b] : 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], w);
        if (g == 0) s_ml[warp * C::M + nt * 8 + 2 * c + e] = make_float2(m[nt][e], l[nt][e]);
      }
    __syncthreads();
    if (threadIdx.x < C::M) {
      float top = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) top = fmaxf(top, s_ml[w * C::M + threadIdx.x].x);
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) {
        const float2 y = s_ml[w * C::M + threadIdx.x];
        L += y.x == -INFINITY ? y.y : y.y * ex2(y.x - top);  // (a warp that met only NaN has its sum alone)
      }
      s_row[threadIdx.x] = make_float2(top, L);
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int rows = min(8, R - cur.qb * C::M - nt * 8);
      if (rows <= 0) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float f = ex2(m[nt][e] - s_row[nt * 8 + 2 * c + e].x);
        if constexpr (!C::kWide) f *= pow2(vunit.e - kUnit);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          o[nt][t][e] = m[nt][e] == -INFINITY ? 0.f : o[nt][t][e] * f;  // (nothing seen: weight 0)
          o[nt][t][e + 2] = m[nt][e] == -INFINITY ? 0.f : o[nt][t][e + 2] * f;
        }
      }
      // as many tiles of 16 columns per pass as fit the buffer for the rows in use
      const int rp = rows <= 4 ? 4 : 8;
      const int tiles = min(D / 16, (kRedFloats / (C::kWarps * rp) - 4) / 16);
      const int pitch = tiles * 16 + 4;
      for (int p0 = 0; p0 < D / 16; p0 += tiles) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          if (t < p0 || t >= p0 + tiles || 2 * c >= rp) continue;
          float* at = s_red + (warp * rp + 2 * c) * pitch + (t - p0) * 16 + g;
          at[0] = o[nt][t][0];
          at[pitch] = o[nt][t][1];
          at[8] = o[nt][t][2];
          at[pitch + 8] = o[nt][t][3];
        }
        __syncthreads();
        const int cols = min(tiles, D / 16 - p0) * 16;
        for (int e = threadIdx.x; e < rows * cols; e += C::kThreads) {
          const int r = e / cols, v = e - r * cols;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < C::kWarps; ++w) sum += s_red[(w * rp + r) * pitch + v];
          const int t = p0 + (v >> 4);
          const int d = C::kWide ? t * 16 + (v & 15) : (v & 7) * (D / 8) + 2 * t + ((v >> 3) & 1);
          const int row = nt * 8 + r;
          const float top = s_row[row].x, L = s_row[row].y;
          if (whole) {
            const int pr = cur.qb * C::M + row, tt = group_div(a, pr), h = cur.kvh * a.group + pr - tt * a.group;
            T* out = reinterpret_cast<T*>(a.out) + (a.nr.cu ? 0 : cur.b * a.o_sb) + h * a.o_sh + (first + tt) * a.o_sn;
            out[d] = Cvt<T>::from_f(L == 0.f ? 0.f : sum * (1.f / L));
            if (a.lse && d == 0)
              a.lse[(a.nr.cu ? 0 : cur.b * a.l_sb) + h * a.l_sh + (first + tt) * a.l_sn] = (top + log2f(L)) * 0.6931471805599453f;
          } else {
            a.part_o[(slot * C::M + row) * D + d] = sum;
            if (d == 0) a.part_ml[slot * C::M + row] = make_float2(top, L);
          }
        }
        __syncthreads();
      }
    }
    first_unit = cut_start = false;
    if (!cur.more(a, end)) break;
    __syncthreads();
    if (threadIdx.x == 0) step_unit(a, &cur, end);
    __syncthreads();  // (the rows' maxima and sums, too, are read before the next unit writes them)
    if (cur.at >= end) break;
  }
  cp_wait<0>();
}

template <typename T, int ST, int D, int NT>
int launch_t(const PagedAttn& a, cudaStream_t st) {
  using C = Cfg<T, ST, D, NT>;
  static_assert(C::kSmem <= 233472 / kCtasPerSm - 1024, "shared memory per block");
  auto kern = paged_mma_kernel<T, ST, D, NT>;
  int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem),
                      "gorgon_paged_attn smem attribute");
  if (rc) return rc;
  return launch_early(kern, a, C::kThreads, C::kSmem, st);
}

// Calls f with the configuration's constants as types.
template <typename F>
int by_config(const PagedAttn& a, F&& f) {
  auto rows = [&](auto t, auto s, auto d) {
    return a.m == 8 ? f(t, s, d, std::integral_constant<int, 1>()) : f(t, s, d, std::integral_constant<int, 2>());
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

bool paged_mma_supported(const PagedAttn& a) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  auto m16 = [](int64_t x, int64_t y, int64_t z) { return ((x | y | z) & 15) == 0; };
  auto small = [](int64_t x) { return x >= 0 && x <= UINT32_MAX; };  // strides that the kernels keep in 32 bits
  const bool strides = small(a.pool.k_sp) && small(a.pool.v_sp) && small(a.pool.k_ss) && small(a.pool.v_ss) &&
                       small(a.pool.ks_sp) && small(a.pool.vs_sp) && small(a.pool.ks_ss) && small(a.pool.vs_ss);
  return strides && a.pool.dtype != GORGON_F32 && (a.pool.d == 64 || a.pool.d == 128) && al(a.pool.k) && al(a.pool.v) && al(a.q) &&
         m16(a.pool.k_sp, a.pool.k_sh, a.pool.k_ss) && m16(a.pool.v_sp, a.pool.v_sh, a.pool.v_ss) &&
         m16(a.q_sb, a.q_sh, a.q_sn);
}

void paged_mma_plan(PagedAttn* a) {
  const int64_t rows = static_cast<int64_t>(a->n) * a->group;
  a->m = rows <= 8 ? 8 : 16;
  by_config(*a, [&](auto t, auto s, auto d, auto nt) {
    constexpr int bn = Cfg<decltype(t), decltype(s)::value, decltype(d)::value, decltype(nt)::value>::BN;
    static_assert((bn & (bn - 1)) == 0, "tiles of a power of two");
    for (a->bn_shift = 0; (1 << a->bn_shift) < bn; ++a->bn_shift) {
    }
    return 0;
  });
  a->qblocks = static_cast<int>(ceil_div(rows, a->m));
  a->unit_cost = 2;
  // no more CTAs than there can be tiles
  const int64_t keys = static_cast<int64_t>(a->pool.table_cols) * a->pool.page_size;
  const int64_t tiles = static_cast<int64_t>(a->pool.batch) * a->pool.hkv * a->qblocks * std::max<int64_t>(1, ceil_div(keys, int64_t(1) << a->bn_shift));
  a->grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(static_cast<int64_t>(kCtasPerSm) * sm_count(), tiles)));
}

int launch_paged_mma(const PagedAttn& a, cudaStream_t st) {
  return by_config(a, [&](auto t, auto s, auto d, auto nt) {
    return launch_t<decltype(t), decltype(s)::value, decltype(d)::value, decltype(nt)::value>(a, st);
  });
}

}  // namespace gorgon

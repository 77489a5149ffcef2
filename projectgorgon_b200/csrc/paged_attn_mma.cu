// Paged attention for few packed rows per (sequence, kv head): single tokens of
// grouped heads, short drafts.  Bound by the bytes of the cache.
//
// A CTA of 8 warps per SM walks its share of the tile list (paged_attn.cuh).  A
// tile is one group of G keys for each warp, and the warps work on their own:
// each streams its groups' K and V rows into its own ring of shared memory
// with 16-byte cp.async copies (8 KB a stage, 3 stages: about 190 KB an SM in
// flight or in use, well above what the memory latency takes to cover), and
// keeps its own running softmax, so there is no barrier in the loop.  Rows
// are gathered one by one, so pages may be of any size and stride; the table
// entry of a group is fetched one group ahead.
//
// Products run on mma.sync m16n8k16: M = 16 packed rows (few of them used when
// the group of query heads is small; the tensor pipe has the time: at 512
// bytes a key an SM's share of the memory bandwidth is one key in 22 cycles).
// 8-bit rows are widened in registers: the byte's exact value as bf16 or f16,
// with the K scale applied to the score and the V scale to the weight, both in
// fp32.  So that a thread widens whole 16-byte pieces, the head dimension is
// taken in another order than the fragment's: thread c of a quad holds values
// 16 (c + 4 i) + 4 s .. + 3 for K step (i, s) (Q is loaded in the same order),
// and column n of output tile t is value n * D / 8 + t.
//
// At the end of a unit the 8 warps' rows meet in shared memory.
#include <type_traits>

#include "paged_attn.cuh"

namespace gorgon {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kRedFloats = 5120;  // 8 warps x 4 rows x 136, 8 rows x 72 or 16 rows x 40 columns

template <typename T, int ST, int D_, int MT>
struct Cfg {
  static constexpr int D = D_;
  static constexpr bool kWide = ST == GORGON_KV_NATIVE;  // 16-bit pages
  static constexpr int kRowBytes = kWide ? D * 2 : D;
  static constexpr int G = kRowBytes == 256 ? 16 : 32;   // keys per warp and tile
  static constexpr int BN = G * kWarps;
  static constexpr int M = 16 * MT;
  static constexpr int kCpr = kRowBytes / 16;            // 16-byte pieces per row
  static constexpr int kRpi = 32 / kCpr;                 // rows per copy instruction
  static constexpr int kHalf = G * kRowBytes;            // K (or V) bytes of a stage
  static constexpr int kMeta = kWide ? 16 : 16 + 8 * G;  // valid-key word, then K and V scales
  static constexpr int kStage = 2 * kHalf + kMeta;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kOffRed = kWarps * kRing;
  static constexpr int kOffMl = kOffRed + kRedFloats * 4;            // [8][M] max, sum
  static constexpr int kOffBits = kOffMl + kWarps * M * 8;           // [M][32] ancestor words
  static constexpr int kOffDepth = kOffBits + M * (kPagedMaxNodes / 32) * 4;
  static constexpr int kSmem = kOffDepth + M * 4;
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
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

// Bytes E of words a and b (the same word twice: two neighbours) as a pair of
// 16-bit floats, exactly.
//   int8 to bf16: 2^7 + (low 7 bits) is the bf16 0x4300 | bits; less 2^7, or 2^8
//     (0x4380) when the sign bit is set.
//   int8 to f16: 2^10 + (byte + 128) is the f16 0x6400 | (byte ^ 0x80); less 1152.
//   e4m3: sign and the seven low bits moved to the wider type's fields; its
//     exponent bias is 7, so times 2^(127 - 7) (bf16) or 2^(15 - 7) (f16), which
//     also makes subnormals right.
template <int ST, uint32_t SEL_LO, uint32_t SEL_HI>
__device__ __forceinline__ uint32_t widen(uint32_t a, uint32_t b, __nv_bfloat16) {
  if constexpr (ST == GORGON_KV_INT8) {
    const uint32_t t = __byte_perm(a, b, SEL_LO);
    const uint32_t x = (t & 0x007f007fu) | 0x43004300u, y = (t & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t t = __byte_perm(a, b, SEL_HI);
    const uint32_t x = (t & 0x80008000u) | ((t >> 4) & 0x07f007f0u);
    const uint32_t f = 0x7b807b80u;  // 2^120
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <int ST, uint32_t SEL_LO, uint32_t SEL_HI>
__device__ __forceinline__ uint32_t widen(uint32_t a, uint32_t b, __half) {
  if constexpr (ST == GORGON_KV_INT8) {
    const uint32_t t = __byte_perm(a, b, SEL_LO);
    const uint32_t x = ((t & 0x00ff00ffu) ^ 0x00800080u) | 0x64006400u;
    const uint32_t f = 0x64806480u;  // 1152
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&f));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t t = __byte_perm(a, b, SEL_HI);
    const uint32_t x = (t & 0x80008000u) | ((t >> 1) & 0x3f803f80u);
    const uint32_t f = 0x5c005c00u;  // 2^8
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
// Byte e of a to the low byte (LO) or the high byte (HI) of the low half, byte
// f of b (numbered 4 .. 7 by __byte_perm) likewise of the high half; the other
// bytes are whatever is there, and masked off.
constexpr uint32_t sel_lo(int e, int f) { return static_cast<uint32_t>(e | (e << 4) | (f << 8) | (f << 12)); }

// f16 weights times V scales need f16's range: they are taken in units of
// 2^(E - 10), with 2^E above the largest V scale that the warp has met in the
// unit, so that they are below 2^10 and keep a row's full precision down to
// 2^-24 of the largest (E only grows; the output row follows it as it follows
// the running max).  bf16 has the range.
template <typename T, int ST>
constexpr bool kUnits = ST != GORGON_KV_NATIVE && std::is_same_v<T, __half>;
__device__ __forceinline__ float pow2(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }

template <int CPR>
__device__ __forceinline__ uint32_t piece_at(int row, int piece) {  // byte offset within a K or V block
  if constexpr (CPR >= 8) return static_cast<uint32_t>(row * CPR + (piece ^ (row & 7))) * 16u;
  return static_cast<uint32_t>(row * CPR + (piece ^ ((row >> 1) & (CPR - 1)))) * 16u;
}

template <typename T, int ST, int D, int MT>
__global__ void __launch_bounds__(kThreads, 1) paged_mma_kernel(const __grid_constant__ PagedAttn a) {
  using C = Cfg<T, ST, D, MT>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ ShareScratch sh;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  Share share;
  TileCursor cur;
  const bool work = cta_share<kThreads>(a, &sh, share, cur);
  if (threadIdx.x == 0) note_cut(a, work, cur, share);
  clear_unused<T, kThreads>(a);
  if (!work) return;

  uint8_t* ring = smem + warp * C::kRing;
  const uint32_t ring_s = smem_addr(ring);
  uint32_t* s_bits = reinterpret_cast<uint32_t*>(smem + C::kOffBits);
  int* s_depth = reinterpret_cast<int*>(smem + C::kOffDepth);
  float* s_red = reinterpret_cast<float*>(smem + C::kOffRed);
  float2* s_ml = reinterpret_cast<float2*>(smem + C::kOffMl);

  // ---- loads: `ahead` is the cursor of the next tile to fetch, `page` this
  // lane's page there (-2: not wanted), fetched when the cursor got there
  TileCursor ahead = cur;
  int64_t to_issue = share.g1 - share.g0;
  int page = -2, prow = 0;
  auto look_up = [&]() {
    page = -2;
    const int j = ahead.tile() * C::BN + warp * C::G + lane;
    if (lane < C::G && ahead.u.wanted(j)) {
      int col;
      a.pool.split(j, col, prow);
      page = __ldg(a.pool.table + static_cast<int64_t>(ahead.b) * a.pool.table_sb + col);  // col is inside: L fits the table
    }
  };
  auto issue = [&](int stage) {
    if (to_issue > 0) {
      --to_issue;
      if (page != -2 && (page < 0 || page >= a.pool.num_pages)) {
        raise_device_error(a.pool.err, kErrBadPage);
        page = -2;
      }
      const uint32_t valid = __ballot_sync(0xffffffffu, page != -2);
      const uint32_t dst = ring_s + stage * C::kStage;
      if (lane == 0) *reinterpret_cast<uint32_t*>(ring + stage * C::kStage + 2 * C::kHalf) = valid;
      if (valid) {
        const int64_t pg = page == -2 ? 0 : page, pr = page == -2 ? 0 : prow;
        const int64_t ko = pg * a.pool.k_sp + pr * a.pool.k_ss, vo = pg * a.pool.v_sp + pr * a.pool.v_ss;
        const char* kb = a.pool.k + ahead.kvh * a.pool.k_sh;
        const char* vb = a.pool.v + ahead.kvh * a.pool.v_sh;
        const int piece = lane % C::kCpr;
#pragma unroll
        for (int it = 0; it < C::G / C::kRpi; ++it) {
          const int r = it * C::kRpi + lane / C::kCpr;
          const bool take = (valid >> r) & 1u;
          const int64_t kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
          const uint32_t at = piece_at<C::kCpr>(r, piece);
          cp16(dst + at, kb + kr + piece * 16, take);
          cp16(dst + C::kHalf + at, vb + vr + piece * 16, take);
        }
        if constexpr (!C::kWide) {
          if (lane < C::G) {
            const uint32_t m = dst + 2 * C::kHalf + 16 + lane * 4;
            cp4(m, a.pool.ks + pg * a.pool.ks_sp + ahead.kvh * a.pool.ks_sh + pr * a.pool.ks_ss, page != -2);
            cp4(m + 4 * C::G, a.pool.vs + pg * a.pool.vs_sp + ahead.kvh * a.pool.vs_sh + pr * a.pool.vs_ss, page != -2);
          }
        }
      }
      if (to_issue > 0) {
        ahead.next(a);
        look_up();
      }
    }
    cp_commit();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < kStages; ++s) issue(s);

  // ---- this unit's state
  uint32_t qf[MT][D / 16][4];
  float o[MT][D / 8][4];
  float m[MT][2], l[MT][2];
  int unit_exp = -116;  // (kUnits) E; -116: nothing met yet
  int hi[MT][2], lo[MT][2];     // what each of the thread's rows sees (paged rows; a tree row's hi is P - 1)
  int all_hi = 0, all_lo = 0;   // positions that every row sees: [all_lo, all_hi]
  bool fresh = true;            // the unit's state is to be set up

  auto sees = [&](int mt, int hh, int j) -> bool {
    if (a.parents && j >= cur.s.P) {
      const int t = (cur.qb * C::M + mt * 16 + g + 8 * hh) / a.group - cur.t0;
      const int n = j - cur.s.P;
      return hi[mt][hh] >= -1 && n < cur.s.c && ((s_bits[t * (kPagedMaxNodes / 32) + (n >> 5)] >> (n & 31)) & 1u);
    }
    return j <= hi[mt][hh] && (j >= lo[mt][hh] || j < a.sinks);
  };

  int stage = 0;
  for (int64_t left = share.g1 - share.g0; left > 0; --left) {
    if (fresh) {
      fresh = false;
      if (a.parents) {
        __syncthreads();  // every warp is done with the last unit's bits
        for (int k = threadIdx.x; k < C::M * (kPagedMaxNodes / 32); k += kThreads) s_bits[k] = 0;
        __syncthreads();
        for (int t = cur.t0 + threadIdx.x; t < cur.t1; t += kThreads)
          s_depth[t - cur.t0] = tree_bits(a, cur.s, cur.b, t, s_bits + (t - cur.t0) * (kPagedMaxNodes / 32));
        __syncthreads();
      }
      const int R = cur.s.c * a.group;
      const int64_t first = a.nr.cu ? a.nr.cu[cur.b] : 0;
      const char* qb = a.q + (a.nr.cu ? 0 : cur.b * a.q_sb);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int pr = cur.qb * C::M + mt * 16 + g + 8 * hh;
          const bool ok = pr < R;
          const int t = ok ? pr / a.group : 0;
          const int h = cur.kvh * a.group + (ok ? pr - t * a.group : 0);
          const int pos = cur.s.P + (a.parents ? (ok ? s_depth[t - cur.t0] : 0) : t);
          hi[mt][hh] = !ok ? -2 : a.parents ? cur.s.P - 1 : pos;
          lo[mt][hh] = a.window ? max(0, pos - a.window + 1) : 0;
          const char* row = qb + (first + t) * a.q_sn + static_cast<int64_t>(h) * a.q_sh;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            if constexpr (C::kWide) {
              const uint32_t* w = reinterpret_cast<const uint32_t*>(row + ks * 32) + c;
              qf[mt][ks][hh] = ok ? __ldg(w) : 0u;
              qf[mt][ks][hh + 2] = ok ? __ldg(w + 4) : 0u;
            } else {
              const int d = (c + 4 * (ks >> 2)) * 16 + (ks & 3) * 4;
              const uint2 w = ok ? __ldg(reinterpret_cast<const uint2*>(row + d * 2)) : make_uint2(0u, 0u);
              qf[mt][ks][hh] = w.x;
              qf[mt][ks][hh + 2] = w.y;
            }
          }
          m[mt][hh] = -INFINITY;
          l[mt][hh] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < D / 8; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][t][e] = 0.f;
      }
      unit_exp = -116;
      all_hi = a.parents ? cur.s.P - 1 : cur.s.P + cur.t0;
      // the largest position of the unit's rows, at most: a tree row's depth is below c
      const int last = cur.s.P + (a.parents ? cur.s.c : cur.t1) - 1;
      all_lo = a.window ? max(0, last - a.window + 1) : 0;
    }

    cp_wait<kStages - 1>();
    __syncwarp();
    uint8_t* st = ring + stage * C::kStage;
    const uint32_t st_s = ring_s + stage * C::kStage;
    const uint32_t valid = *reinterpret_cast<const uint32_t*>(st + 2 * C::kHalf);
    if (valid) {
      const int j0 = cur.tile() * C::BN + warp * C::G;
      const bool plain = valid == (C::G == 32 ? 0xffffffffu : (1u << (C::G & 31)) - 1u) && j0 + C::G - 1 <= all_hi &&
                         (j0 >= all_lo || j0 + C::G <= a.sinks);
      float x[MT][C::G / 8][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < C::G / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[mt][n][e] = 0.f;
      // ---- scores
      if constexpr (C::kWide) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int n2 = 0; n2 < C::G / 16; ++n2) {
            uint32_t b[4];
            ldsm4(b, st_s + piece_at<C::kCpr>(n2 * 16 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma(x[mt][2 * n2], qf[mt][ks], b[0], b[1], T{});
              mma(x[mt][2 * n2 + 1], qf[mt][ks], b[2], b[3], T{});
            }
          }
      } else {
#pragma unroll
        for (int n = 0; n < C::G / 8; ++n)
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(st + piece_at<C::kCpr>(n * 8 + g, c + 4 * i));
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const uint32_t b0 = widen<ST, sel_lo(0, 1), sel_lo(0, 1)>(ww[s], ww[s], T{});
              const uint32_t b1 = widen<ST, sel_lo(2, 3), sel_lo(2, 3)>(ww[s], ww[s], T{});
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) mma(x[mt][n], qf[mt][i * 4 + s], b0, b1, T{});
            }
          }
      }
      // ---- softmax
      const float* ksc = reinterpret_cast<const float*>(st + 2 * C::kHalf + 16);
#pragma unroll
      for (int n = 0; n < C::G / 8; ++n) {
        float f0 = a.scale_log2, f1 = a.scale_log2;
        if constexpr (!C::kWide) {
          const float2 f = *reinterpret_cast<const float2*>(ksc + n * 8 + 2 * c);
          f0 *= f.x;
          f1 *= f.y;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[mt][n][e] *= (e & 1) ? f1 : f0;
            if (!plain) {
              const int k = n * 8 + 2 * c + (e & 1);
              if (!((valid >> k) & 1u) || !sees(mt, e >> 1, j0 + k)) x[mt][n][e] = -INFINITY;
            }
          }
      }
      bool slow = false;
      float regrade = 1.f;
      if constexpr (kUnits<T, ST>) {
        float top = lane < C::G ? ksc[C::G + lane] : 0.f;  // 0 for keys that were not fetched
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const int e = (__float_as_int(top) >> 23) - 126;  // top < 2^e
        if (e > unit_exp) {
          regrade = pow2(unit_exp - e);
          unit_exp = e;
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float alpha[2];
        bool moved = regrade != 1.f;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float top = m[mt][hh];
#pragma unroll
          for (int n = 0; n < C::G / 8; ++n) top = fmaxf(top, fmaxf(x[mt][n][2 * hh], x[mt][n][2 * hh + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float base = top == -INFINITY ? 0.f : top;
          alpha[hh] = ex2(m[mt][hh] - base);
          moved |= top > m[mt][hh];
          m[mt][hh] = top;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < C::G / 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float p = ex2(x[mt][n][2 * hh + e] - base);
              x[mt][n][2 * hh + e] = p;
              sum += p;
            }
          l[mt][hh] = l[mt][hh] * alpha[hh] + sum;
          if constexpr (kUnits<T, ST>) alpha[hh] *= regrade;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int t = 0; t < D / 8; ++t) {
            o[mt][t][0] *= alpha[0];
            o[mt][t][1] *= alpha[0];
            o[mt][t][2] *= alpha[1];
            o[mt][t][3] *= alpha[1];
          }
        }
      }
      // ---- a partly hidden group of 16-bit rows: 0 * infinity must not reach a row that does not see it
      if constexpr (C::kWide) {
        if (!plain) {
          bool odd = false;
          for (int it = lane; it < C::G * C::kCpr; it += 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(st + C::kHalf + it * 16);
            constexpr uint32_t top = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= (ww[e] & top) == top || ((ww[e] >> 16) & top) == top;
          }
          slow = __any_sync(0xffffffffu, odd);
        }
      }
      // ---- output rows
      if (C::kWide && slow) {
        // One key at a time on the CUDA cores.  The weights go over the K rows, which are done with.
        float* w = reinterpret_cast<float*>(st);
        static_assert(!C::kWide || C::M * C::G * 4 <= C::kHalf, "weights fit the K block");
        __syncwarp();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < C::G / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = n * 8 + 2 * c + (e & 1);
              const bool on = ((valid >> k) & 1u) && sees(mt, e >> 1, j0 + k);
              w[(mt * 16 + g + 8 * (e >> 1)) * C::G + k] = on ? x[mt][n][e] : -1.f;
            }
        __syncwarp();
#pragma unroll 1
        for (int k = 0; k < C::G; ++k)
#pragma unroll
          for (int t = 0; t < D / 8; ++t) {
            const T* v = reinterpret_cast<const T*>(st + C::kHalf + piece_at<C::kCpr>(k, t)) + 2 * c;
            const float v0 = Cvt<T>::to_f(v[0]), v1 = Cvt<T>::to_f(v[1]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const float p = w[(mt * 16 + g + 8 * hh) * C::G + k];
                if (!(p < 0.f)) {
                  o[mt][t][2 * hh] = fmaf(p, v0, o[mt][t][2 * hh]);
                  o[mt][t][2 * hh + 1] = fmaf(p, v1, o[mt][t][2 * hh + 1]);
                }
              }
          }
      } else {
#pragma unroll
        for (int s = 0; s < C::G / 16; ++s) {
          uint32_t pf[MT][4];
          float f[4] = {1.f, 1.f, 1.f, 1.f};
          if constexpr (!C::kWide) {
            const float2 f0 = *reinterpret_cast<const float2*>(ksc + C::G + s * 16 + 2 * c);
            const float2 f1 = *reinterpret_cast<const float2*>(ksc + C::G + s * 16 + 8 + 2 * c);
            const float F = kUnits<T, ST> ? pow2(10 - unit_exp) : 1.f;
            f[0] = f0.x * F;
            f[1] = f0.y * F;
            f[2] = f1.x * F;
            f[3] = f1.y * F;
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                float p0 = x[mt][2 * s + q][2 * hh], p1 = x[mt][2 * s + q][2 * hh + 1];
                if constexpr (!C::kWide) {  // a hidden key's weight is 0 whatever its scale
                  p0 = p0 == 0.f ? 0.f : p0 * f[2 * q];
                  p1 = p1 == 0.f ? 0.f : p1 * f[2 * q + 1];
                }
                pf[mt][hh + 2 * q] = pack2(p0, p1, T{});
              }
          if constexpr (C::kWide) {
#pragma unroll
            for (int t2 = 0; t2 < D / 16; ++t2) {
              uint32_t b[4];
              ldsm4t(b, st_s + C::kHalf + piece_at<C::kCpr>(s * 16 + (lane & 15), t2 * 2 + (lane >> 4)));
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                mma(o[mt][2 * t2], pf[mt], b[0], b[1], T{});
                mma(o[mt][2 * t2 + 1], pf[mt], b[2], b[3], T{});
              }
            }
          } else {
            // this thread's four keys, D / 8 values of each from n = g on
            uint32_t w[4][D / 32];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int key = s * 16 + (k >> 1) * 8 + 2 * c + (k & 1);
              if constexpr (D == 128) {
                const uint4 r = *reinterpret_cast<const uint4*>(st + C::kHalf + piece_at<C::kCpr>(key, g));
                w[k][0] = r.x;
                w[k][1] = r.y;
                w[k][2] = r.z;
                w[k][3] = r.w;
              } else {
                const uint2 r = *reinterpret_cast<const uint2*>(st + C::kHalf + piece_at<C::kCpr>(key, g >> 1) + (g & 1) * 8);
                w[k][0] = r.x;
                w[k][1] = r.y;
              }
            }
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
              const uint32_t b[8] = {
                  widen<ST, sel_lo(0, 4), sel_lo(0, 4)>(w[0][q], w[1][q], T{}), widen<ST, sel_lo(0, 4), sel_lo(0, 4)>(w[2][q], w[3][q], T{}),
                  widen<ST, sel_lo(1, 5), sel_lo(1, 5)>(w[0][q], w[1][q], T{}), widen<ST, sel_lo(1, 5), sel_lo(1, 5)>(w[2][q], w[3][q], T{}),
                  widen<ST, sel_lo(2, 6), sel_lo(2, 6)>(w[0][q], w[1][q], T{}), widen<ST, sel_lo(2, 6), sel_lo(2, 6)>(w[2][q], w[3][q], T{}),
                  widen<ST, sel_lo(3, 7), sel_lo(3, 7)>(w[0][q], w[1][q], T{}), widen<ST, sel_lo(3, 7), sel_lo(3, 7)>(w[2][q], w[3][q], T{})};
#pragma unroll
              for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) mma(o[mt][4 * q + e], pf[mt], b[2 * e], b[2 * e + 1], T{});
            }
          }
        }
      }
    }
    __syncwarp();  // every lane is done with the stage
    issue(stage);
    stage = stage + 1 == kStages ? 0 : stage + 1;

    // ---- the end of the unit, or of the CTA's part of it
    const bool unit_done = cur.i + 1 == cur.u.tiles;
    if (unit_done || left == 1) {
      const int64_t done = share.g1 - left;  // this tile's number
      const int64_t start = done - cur.i;
      const bool whole = unit_done && start >= share.g0;
      const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (start <= share.g0 ? 0 : 1);
      const int R = cur.s.c * a.group;
      const int64_t first = a.nr.cu ? a.nr.cu[cur.b] : 0;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          l[mt][hh] += __shfl_xor_sync(0xffffffffu, l[mt][hh], 1);
          l[mt][hh] += __shfl_xor_sync(0xffffffffu, l[mt][hh], 2);
          if (c == 0) s_ml[warp * C::M + mt * 16 + g + 8 * hh] = make_float2(m[mt][hh], l[mt][hh]);
        }
      __syncthreads();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int rows = min(16, R - cur.qb * C::M - mt * 16);
        if (rows <= 0) break;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float top = -INFINITY;
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w * C::M + mt * 16 + g + 8 * hh].x);
          float f = m[mt][hh] == -INFINITY ? 0.f : ex2(m[mt][hh] - top);
          if constexpr (kUnits<T, ST>) f *= pow2(unit_exp - 10);
#pragma unroll
          for (int t = 0; t < D / 8; ++t) {
            o[mt][t][2 * hh] = m[mt][hh] == -INFINITY ? 0.f : o[mt][t][2 * hh] * f;
            o[mt][t][2 * hh + 1] = m[mt][hh] == -INFINITY ? 0.f : o[mt][t][2 * hh + 1] * f;
          }
        }
        // column tiles per pass, as many as fit the buffer for the rows in use
        const int rp = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
        const int tiles = min(D / 8, 64 / rp);
        const int pitch = tiles * 8 + 8;
        for (int p0 = 0; p0 < D / 8; p0 += tiles) {
#pragma unroll
          for (int t = 0; t < D / 8; ++t) {
            if (t < p0 || t >= p0 + tiles) continue;
            float* at = s_red + warp * rp * pitch + (t - p0) * 8 + 2 * c;
            if (g < rp) *reinterpret_cast<float2*>(at + g * pitch) = make_float2(o[mt][t][0], o[mt][t][1]);
            if (g + 8 < rp) *reinterpret_cast<float2*>(at + (g + 8) * pitch) = make_float2(o[mt][t][2], o[mt][t][3]);
          }
          __syncthreads();
          const int cols = tiles * 8;
          for (int e = threadIdx.x; e < rows * cols; e += kThreads) {
            const int r = e / cols, q = e - r * cols;  // q: the pass's column in output order
            const int per = cols / 8;
            const int v = C::kWide ? q : (q % per) * 8 + q / per;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) sum += s_red[(w * rp + r) * pitch + v];
            const int d = C::kWide ? p0 * 8 + q : (q / per) * (D / 8) + p0 + q % per;
            const int row = mt * 16 + r;
            if (whole) {
              float top = -INFINITY, L = 0.f;
              for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w * C::M + row].x);
              for (int w = 0; w < kWarps; ++w) {
                const float2 x = s_ml[w * C::M + row];
                L += x.x == -INFINITY ? x.y : x.y * ex2(x.x - top);
              }
              const int pr = cur.qb * C::M + row, t = pr / a.group, h = cur.kvh * a.group + pr - t * a.group;
              T* out = reinterpret_cast<T*>(a.out) + (a.nr.cu ? 0 : cur.b * a.o_sb) + h * a.o_sh + (first + t) * a.o_sn;
              out[d] = Cvt<T>::from_f(sum * (1.f / L));
              if (a.lse && d == 0)
                a.lse[(a.nr.cu ? 0 : cur.b * a.l_sb) + h * a.l_sh + (first + t) * a.l_sn] = (top + log2f(L)) * 0.6931471805599453f;
            } else {
              a.part_o[(slot * C::M + row) * D + d] = sum;
              if (d == 0) {
                float top = -INFINITY, L = 0.f;
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w * C::M + row].x);
                for (int w = 0; w < kWarps; ++w) {
                  const float2 x = s_ml[w * C::M + row];
                  L += x.x == -INFINITY ? x.y : x.y * ex2(x.x - top);
                }
                a.part_ml[slot * C::M + row] = make_float2(top, L);
              }
            }
          }
          __syncthreads();
        }
      }
      __syncthreads();  // s_ml is read by every warp before the next unit writes it
      fresh = true;
    }
    if (left > 1) cur.next(a);
  }
  cp_wait<0>();
}

template <typename T, int ST, int D, int MT>
int launch_t(const PagedAttn& a, cudaStream_t st) {
  using C = Cfg<T, ST, D, MT>;
  static_assert(C::kSmem <= 232448 - 512, "shared memory per block");
  auto kern = paged_mma_kernel<T, ST, D, MT>;
  int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem),
                      "gorgon_paged_attn smem attribute");
  if (rc) return rc;
  kern<<<a.grid, kThreads, C::kSmem, st>>>(a);
  return check_cuda(cudaGetLastError(), "gorgon_paged_attn launch");
}

template <typename T, int ST, int D>
int launch_m(const PagedAttn& a, cudaStream_t st) {
  return a.m == 16 ? launch_t<T, ST, D, 1>(a, st) : launch_t<T, ST, D, 2>(a, st);
}
template <typename T, int ST>
int launch_d(const PagedAttn& a, cudaStream_t st) {
  return a.pool.d == 128 ? launch_m<T, ST, 128>(a, st) : launch_m<T, ST, 64>(a, st);
}
template <typename T>
int launch_s(const PagedAttn& a, cudaStream_t st) {
  switch (a.pool.storage) {
    case GORGON_KV_NATIVE: return launch_d<T, GORGON_KV_NATIVE>(a, st);
    case GORGON_KV_INT8: return launch_d<T, GORGON_KV_INT8>(a, st);
    default: return launch_d<T, GORGON_KV_E4M3>(a, st);
  }
}

}  // namespace

bool paged_mma_supported(const PagedAttn& a) {
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  auto m16 = [](int64_t x, int64_t y, int64_t z) { return ((x | y | z) & 15) == 0; };
  return a.pool.dtype != GORGON_F32 && (a.pool.d == 64 || a.pool.d == 128) && al(a.pool.k) && al(a.pool.v) && al(a.q) &&
         m16(a.pool.k_sp, a.pool.k_sh, a.pool.k_ss) && m16(a.pool.v_sp, a.pool.v_sh, a.pool.v_ss) &&
         m16(a.q_sb, a.q_sh, a.q_sn);
}

void paged_mma_plan(PagedAttn* a) {
  const int64_t rows = static_cast<int64_t>(a->n) * a->group;
  a->m = rows <= 16 ? 16 : 32;
  const int row_bytes = a->pool.d * (a->pool.storage == GORGON_KV_NATIVE ? 2 : 1);
  a->bn = (row_bytes == 256 ? 16 : 32) * kWarps;
  a->qblocks = static_cast<int>(ceil_div(rows, a->m));
  // no more CTAs than there can be tiles
  const int64_t keys = static_cast<int64_t>(a->pool.table_cols) * a->pool.page_size;
  const int64_t tiles = static_cast<int64_t>(a->pool.batch) * a->pool.hkv * a->qblocks * std::max<int64_t>(1, ceil_div(keys, a->bn));
  a->grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count(), tiles)));
}

int launch_paged_mma(const PagedAttn& a, cudaStream_t st) {
  return a.pool.dtype == GORGON_BF16 ? launch_s<__nv_bfloat16>(a, st) : launch_s<__half>(a, st);
}

}  // namespace gorgon

// Paged attention on the CUDA cores: any dtype, head_dim up to 256, any
// alignment.  The tensor-core kernels take 16-bit rows of whole 16-byte pieces;
// this one takes the rest, and is the plainest statement of the operator.
//
// A CTA per (new row, query head): its warps take every eighth visible key,
// a lane the values lane, lane + 32, ... of a row; each warp keeps a running
// max, sum and output row in fp32, joined through shared memory at the end.
// Bound by the latency of one key at a time per warp.
#include <cuda_fp8.h>

#include <algorithm>

#include "paged_attn.cuh"

namespace gorgon {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxD = 256;

template <typename T, int ST>
__device__ __forceinline__ float page_value(const char* row, int d) {
  if constexpr (ST == GORGON_KV_NATIVE) return Cvt<T>::to_f(reinterpret_cast<const T*>(row)[d]);
  if constexpr (ST == GORGON_KV_INT8) return static_cast<float>(reinterpret_cast<const int8_t*>(row)[d]);
  __nv_fp8_e4m3 f;
  f.__x = reinterpret_cast<const uint8_t*>(row)[d];
  return static_cast<float>(f);
}

template <typename T, int ST>
__global__ void __launch_bounds__(kWarps * 32) paged_simt_kernel(const PagedAttn a) {
  __shared__ uint32_t s_bits[kPagedMaxNodes / 32];
  __shared__ int s_depth;
  __shared__ float s_m[kWarps], s_l[kWarps];
  __shared__ float s_o[kWarps][kMaxD];
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Seq s = sequence(a, b, threadIdx.x == 0 && t == 0 && h == 0);
  if (t >= s.c || !rows_inside(a, b, s.c)) return;
  const int64_t row = a.nr.cu ? a.nr.first(b) + t : t;
  T* out = reinterpret_cast<T*>(a.out) + (a.nr.cu ? 0 : b * a.o_sb) + h * a.o_sh + row * a.o_sn;
  float* lse = a.lse ? a.lse + (a.nr.cu ? 0 : b * a.l_sb) + h * a.l_sh + row * a.l_sn : nullptr;
  const int D = a.pool.d;
  if (!s.ok) {  // (it may bring more rows than the grid covers)
    for (int64_t k = 0; t + k < s.c; k += gridDim.x) {
      for (int d = threadIdx.x; d < D; d += blockDim.x) out[k * a.o_sn + d] = Cvt<T>::from_f(0.f);
      if (lse && threadIdx.x == 0) lse[k * a.l_sn] = -INFINITY;
    }
    return;
  }
  int pos = s.P + t;
  if (a.parents) {
    for (int k = threadIdx.x; k < (s.c + 31) / 32; k += blockDim.x) s_bits[k] = 0;
    __syncthreads();
    if (threadIdx.x == 0) s_depth = tree_bits(a, s, b, t, s_bits);
    __syncthreads();
    pos = s.P + s_depth;
  }
  int lo = a.window ? max(0, pos - a.window + 1) : 0;
  if (a.parents) lo = min(lo, s.P);  // tree rows go by their bits: an ancestor may stand anywhere among them
  const int s_end = min(a.sinks, lo);
  const int hi = a.parents ? s.L : pos + 1;
  const int kvh = h / a.group;
  const T* q = reinterpret_cast<const T*>(a.q + (a.nr.cu ? 0 : b * a.q_sb) + h * a.q_sh + row * a.q_sn);
  float qv[kMaxD / 32], o[kMaxD / 32];
#pragma unroll
  for (int k = 0; k < kMaxD / 32; ++k) {
    const int d = lane + 32 * k;
    qv[k] = d < D ? Cvt<T>::to_f(q[d]) * a.scale_log2 : 0.f;
    o[k] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int keys = s_end + max(0, hi - lo);  // sinks, then the window
  for (int i = warp; i < keys; i += kWarps) {
    const int j = i < s_end ? i : lo + (i - s_end);
    if (a.parents && j >= s.P && !((s_bits[(j - s.P) >> 5] >> ((j - s.P) & 31)) & 1u)) continue;
    int col, r;
    a.pool.split(j, col, r);
    const int page = a.pool.page(b, col);
    if (page < 0) continue;
    const char* kr = a.pool.k + page * a.pool.k_sp + kvh * a.pool.k_sh + r * a.pool.k_ss;
    const char* vr = a.pool.v + page * a.pool.v_sp + kvh * a.pool.v_sh + r * a.pool.v_ss;
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxD / 32; ++k) {
      const int d = lane + 32 * k;
      if (d < D) x = fmaf(qv[k], page_value<T, ST>(kr, d), x);
    }
    x = warp_sum(x);
    float vsc = 1.f;
    if constexpr (ST != GORGON_KV_NATIVE) {
      if (D > 0) x *= a.pool.ks[page * a.pool.ks_sp + kvh * a.pool.ks_sh + r * a.pool.ks_ss];
      vsc = a.pool.vs[page * a.pool.vs_sp + kvh * a.pool.vs_sh + r * a.pool.vs_ss];
    }
    const float mn = fmaxf(m, x);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = exp2f(m - base), p = exp2f(x - base);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int k = 0; k < kMaxD / 32; ++k) {
      const int d = lane + 32 * k;
      if (d < D) o[k] = fmaf(p * vsc, page_value<T, ST>(vr, d), o[k] * f);
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int k = 0; k < kMaxD / 32; ++k)
    if (lane + 32 * k < D) s_o[warp][lane + 32 * k] = o[k];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
  const float base = M == -INFINITY ? 0.f : M;
  for (int w = 0; w < kWarps; ++w) L += s_l[w] * exp2f(s_m[w] - base);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w) x = fmaf(s_o[w][d], exp2f(s_m[w] - base), x);
    out[d] = Cvt<T>::from_f(L == 0.f ? 0.f : x / L);
  }
  if (lse && threadIdx.x == 0) *lse = (M + log2f(L)) * 0.6931471805599453f;
}

template <typename T>
int launch_t(const PagedAttn& a, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(std::max(a.n, 1)), static_cast<unsigned>(a.hq), static_cast<unsigned>(a.pool.batch));
  switch (a.pool.storage) {
    case GORGON_KV_NATIVE: paged_simt_kernel<T, GORGON_KV_NATIVE><<<grid, kWarps * 32, 0, st>>>(a); break;
    case GORGON_KV_INT8: paged_simt_kernel<T, GORGON_KV_INT8><<<grid, kWarps * 32, 0, st>>>(a); break;
    default: paged_simt_kernel<T, GORGON_KV_E4M3><<<grid, kWarps * 32, 0, st>>>(a); break;
  }
  return check_cuda(cudaGetLastError(), "gorgon_paged_attn launch");
}

// Joins the pieces of one unit that the schedule cut (see CutUnit): out = sum_k
// 2^(m_k - M) o_k / sum_k 2^(m_k - M) l_k.  Grid (main grid, row blocks of 8).
// A warp per row, or several when fewer than 8 rows are in use: each takes its
// share of the pieces, eight loads in flight, and their sums meet in shared
// memory in a fixed order.  Launched to overlap the end of the main kernel,
// which it waits for before it reads anything.
constexpr int kMergeWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_merge_kernel(const __grid_constant__ PagedAttn a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float s_acc[kMergeWarps][D];
  __shared__ float s_l[kMergeWarps];
  const int c = blockIdx.x;
  const CutUnit n = a.cut[c];
  if (n.pieces == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int V = D / 32;  // columns per lane
  const Seq s = sequence(a, n.b, false);
  const int rows = min(8, min(a.m, s.c * a.group - n.qb * a.m) - static_cast<int>(blockIdx.y) * 8);
  if (rows <= 0) return;
  const int per = rows <= 1 ? 8 : rows <= 2 ? 4 : rows <= 4 ? 2 : 1;  // warps per row
  const int sub = warp % per, r8 = warp / per;
  const bool live = r8 < rows;
  const int row = blockIdx.y * 8 + (live ? r8 : 0);
  auto slot = [&](int p) -> int64_t { return static_cast<int64_t>(c - 1 + p) * 2 + (p == 0 ? n.first_slot : 0); };
  float M = -INFINITY;
  for (int p = lane; p < n.pieces; p += 32) M = fmaxf(M, __ldcg(&a.part_ml[slot(p) * a.m + row]).x);
  M = warp_max(M);
  const float base = M == -INFINITY ? 0.f : M;
  float L = 0.f, acc[V] = {};
  constexpr int kInFlight = 8;
#pragma unroll 1
  for (int p0 = sub; p0 < n.pieces; p0 += per * kInFlight) {
    float2 ml[kInFlight];
    float x[kInFlight][V];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const int p = p0 + k * per;
      ml[k] = make_float2(-INFINITY, 0.f);
      if (p < n.pieces) {
        ml[k] = __ldcg(&a.part_ml[slot(p) * a.m + row]);
        const float* o = a.part_o + (slot(p) * a.m + row) * D + lane * V;
        if constexpr (V == 4)
          *reinterpret_cast<float4*>(x[k]) = __ldcg(reinterpret_cast<const float4*>(o));
        else
          *reinterpret_cast<float2*>(x[k]) = __ldcg(reinterpret_cast<const float2*>(o));
      }
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      if (p0 + k * per >= n.pieces) break;
      const float f = exp2f(ml[k].x - base);
      L = fmaf(f, ml[k].y, L);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(f, x[k][v], acc[v]);
    }
  }
  if (per > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) s_acc[warp][lane * V + v] = acc[v];
    if (lane == 0) s_l[warp] = L;
    __syncthreads();
    if (sub != 0) return;
    for (int w = 1; w < per; ++w) {
      L += s_l[warp + w];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += s_acc[warp + w][lane * V + v];
    }
  }
  if (!live) return;
  const int pr = n.qb * a.m + row;
  const int t = pr / a.group, h = n.kvh * a.group + pr - t * a.group;
  const int64_t r = a.nr.cu ? a.nr.cu[n.b] + t : t;
  T* out = reinterpret_cast<T*>(a.out) + (a.nr.cu ? 0 : n.b * a.o_sb) + h * a.o_sh + r * a.o_sn + lane * V;
  const float inv = 1.f / L;
#pragma unroll
  for (int v = 0; v < V; ++v) out[v] = Cvt<T>::from_f(L == 0.f ? 0.f : acc[v] * inv);
  if (a.lse && lane == 0)
    a.lse[(a.nr.cu ? 0 : n.b * a.l_sb) + h * a.l_sh + r * a.l_sn] = (M + log2f(L)) * 0.6931471805599453f;
}

// The same for units of many rows, most of them cut in two or three: a warp
// takes eight rows, four pieces at a time; lane 4 r + p holds row r's max and
// sum of piece p, and the eight rows of a piece are in flight together.
constexpr int kRowsPerWarp = 8;
constexpr int kMergeRows = kMergeWarps * kRowsPerWarp;
template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_merge_rows_kernel(const __grid_constant__ PagedAttn a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const CutUnit n = a.cut[c];
  if (n.pieces == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int V = D / 32;
  const Seq s = sequence(a, n.b, false);
  const int r0 = blockIdx.y * kMergeRows + warp * kRowsPerWarp;
  const int rows = min(kRowsPerWarp, min(a.m, s.c * a.group - n.qb * a.m) - r0);
  if (rows <= 0) return;
  auto slot = [&](int p) -> int64_t { return static_cast<int64_t>(c - 1 + p) * 2 + (p == 0 ? n.first_slot : 0); };
  float acc[kRowsPerWarp][V] = {};
  float M = -INFINITY, L = 0.f;  // of row lane / 4, the same on its four lanes
  for (int p0 = 0; p0 < n.pieces; p0 += 4) {
    const int p = p0 + (lane & 3), r = lane >> 2;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (p < n.pieces && r < rows) ml = __ldcg(&a.part_ml[slot(p) * a.m + r0 + r]);
    float top = fmaxf(M, ml.x);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float base = top == -INFINITY ? 0.f : top;
    const float old = exp2f(M - base), f = exp2f(ml.x - base);
    float add = f * ml.y;
    add += __shfl_xor_sync(0xffffffffu, add, 1);
    add += __shfl_xor_sync(0xffffffffu, add, 2);
    L = L * old + add;
    M = top;
    const int np = min(4, n.pieces - p0);
    if (p0 > 0) {
#pragma unroll
      for (int k = 0; k < kRowsPerWarp; ++k) {
        const float g = __shfl_sync(0xffffffffu, old, 4 * k);
#pragma unroll
        for (int v = 0; v < V; ++v) acc[k][v] *= g;
      }
    }
    for (int q = 0; q < np; ++q) {
      const float* o = a.part_o + (slot(p0 + q) * a.m + r0) * D + lane * V;
      float x[kRowsPerWarp][V];
#pragma unroll
      for (int k = 0; k < kRowsPerWarp; ++k)
        if (k < rows) {
          if constexpr (V == 4)
            *reinterpret_cast<float4*>(x[k]) = __ldcg(reinterpret_cast<const float4*>(o + k * D));
          else
            *reinterpret_cast<float2*>(x[k]) = __ldcg(reinterpret_cast<const float2*>(o + k * D));
        }
#pragma unroll
      for (int k = 0; k < kRowsPerWarp; ++k) {
        const float g = __shfl_sync(0xffffffffu, f, 4 * k + q);
        if (k < rows) {
#pragma unroll
          for (int v = 0; v < V; ++v) acc[k][v] = fmaf(g, x[k][v], acc[k][v]);
        }
      }
    }
  }
  const int64_t first = a.nr.cu ? a.nr.cu[n.b] : 0;
#pragma unroll
  for (int k = 0; k < kRowsPerWarp; ++k) {
    const float Lk = __shfl_sync(0xffffffffu, L, 4 * k), Mk = __shfl_sync(0xffffffffu, M, 4 * k);
    if (k >= rows) continue;
    const int pr = n.qb * a.m + r0 + k;
    const int t = group_div(a, pr), h = n.kvh * a.group + pr - t * a.group;
    T* out = reinterpret_cast<T*>(a.out) + (a.nr.cu ? 0 : n.b * a.o_sb) + h * a.o_sh + (first + t) * a.o_sn + lane * V;
    const float inv = 1.f / Lk;
    T y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = Cvt<T>::from_f(Lk == 0.f ? 0.f : acc[k][v] * inv);
    if (reinterpret_cast<uintptr_t>(out) % (V * sizeof(T)) == 0) {
      if constexpr (V == 4) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
      else *reinterpret_cast<uint32_t*>(out) = *reinterpret_cast<const uint32_t*>(y);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) out[v] = y[v];
    }
    if (a.lse && lane == 0)
      a.lse[(a.nr.cu ? 0 : n.b * a.l_sb) + h * a.l_sh + (first + t) * a.l_sn] = (Mk + log2f(Lk)) * 0.6931471805599453f;
  }
}

}  // namespace

int launch_paged_merge(const PagedAttn& a, cudaStream_t st) {
  if (a.m >= kMergeRows) {
    const int rows = static_cast<int>(ceil_div(std::min<int64_t>(a.m, static_cast<int64_t>(a.n) * a.group), kMergeRows));
    if (a.pool.dtype == GORGON_BF16)
      return a.pool.d == 128 ? launch_early(paged_merge_rows_kernel<__nv_bfloat16, 128>, a, kMergeWarps * 32, 0, st, rows)
                             : launch_early(paged_merge_rows_kernel<__nv_bfloat16, 64>, a, kMergeWarps * 32, 0, st, rows);
    return a.pool.d == 128 ? launch_early(paged_merge_rows_kernel<__half, 128>, a, kMergeWarps * 32, 0, st, rows)
                           : launch_early(paged_merge_rows_kernel<__half, 64>, a, kMergeWarps * 32, 0, st, rows);
  }
  const int y = static_cast<int>(ceil_div(a.m, 8));
  if (a.pool.dtype == GORGON_BF16)
    return a.pool.d == 128 ? launch_early(paged_merge_kernel<__nv_bfloat16, 128>, a, kMergeWarps * 32, 0, st, y)
                           : launch_early(paged_merge_kernel<__nv_bfloat16, 64>, a, kMergeWarps * 32, 0, st, y);
  return a.pool.d == 128 ? launch_early(paged_merge_kernel<__half, 128>, a, kMergeWarps * 32, 0, st, y)
                         : launch_early(paged_merge_kernel<__half, 64>, a, kMergeWarps * 32, 0, st, y);
}

int launch_paged_simt(const PagedAttn& a, cudaStream_t st) {
  switch (a.pool.dtype) {
    case GORGON_F32: return launch_t<float>(a, st);
    case GORGON_BF16: return launch_t<__nv_bfloat16>(a, st);
    default: return launch_t<__half>(a, st);
  }
}

}  // namespace gorgon

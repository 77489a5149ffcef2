// The paged key/value cache's own operators: append (with quantisation), read
// back, and trim-on-reject over all layers.  Each is bound by the bytes it
// moves (or, for a decode step's few rows, by one round trip to memory), so
// each is one launch in which every thread holds 16-byte pieces of K and of V
// in flight.
#include <cuda_fp8.h>

#include <algorithm>

#include "paged.cuh"

namespace gorgon {

int make_pool(const gorgon_paged_kv* p, const char* who, PagedPool* o) {
  const std::string w(who);
  if (!dtype_ok(p->dtype)) return set_error(GORGON_ERR_INVALID, w + ": unknown dtype");
  if (p->storage < GORGON_KV_NATIVE || p->storage > GORGON_KV_E4M3)
    return set_error(GORGON_ERR_INVALID, w + ": unknown storage");
  if (p->num_pages < 0 || p->page_size < 1 || p->heads_kv < 1 || p->head_dim < 0 || p->batch < 0 || p->table_cols < 0)
    return set_error(GORGON_ERR_INVALID, w + ": bad pool size");
  if (p->head_dim > 256) return set_error(GORGON_ERR_UNSUPPORTED, w + ": head_dim > 256");
  if (p->batch > 65535 || p->heads_kv > 65535 || p->batch * p->heads_kv > (int64_t(1) << 24))
    return set_error(GORGON_ERR_UNSUPPORTED, w + ": batch or heads_kv too large");
  if (p->num_pages > INT32_MAX || p->page_size > (1 << 20) || p->table_cols > INT32_MAX ||
      p->table_cols * p->page_size > (int64_t(1) << 30))
    return set_error(GORGON_ERR_UNSUPPORTED, w + ": more than 2^30 positions in a sequence");
  if (p->batch > 0 && p->head_dim > 0 && (!p->k_pages || !p->v_pages || (!p->block_table && p->table_cols > 0)))
    return set_error(GORGON_ERR_INVALID, w + ": null pages or block table");
  if (p->storage != GORGON_KV_NATIVE && p->batch > 0 && (!p->k_scale || !p->v_scale))
    return set_error(GORGON_ERR_INVALID, w + ": 8-bit pages need k_scale and v_scale");
  const int64_t es = storage_bytes(p->storage, p->dtype);
  PagedPool& x = *o;
  x = PagedPool{};
  x.k = static_cast<char*>(p->k_pages);
  x.v = static_cast<char*>(p->v_pages);
  x.k_sp = p->k_stride_p * es; x.k_sh = p->k_stride_h * es; x.k_ss = p->k_stride_s * es;
  x.v_sp = p->v_stride_p * es; x.v_sh = p->v_stride_h * es; x.v_ss = p->v_stride_s * es;
  x.ks = p->k_scale; x.vs = p->v_scale;
  x.ks_sp = p->ks_stride_p; x.ks_sh = p->ks_stride_h; x.ks_ss = p->ks_stride_s;
  x.vs_sp = p->vs_stride_p; x.vs_sh = p->vs_stride_h; x.vs_ss = p->vs_stride_s;
  x.table = p->block_table;
  x.table_sb = p->table_stride_b;
  x.table_cols = static_cast<int>(p->table_cols);
  x.lens = p->seq_lens;
  x.num_pages = static_cast<int>(p->num_pages);
  x.page_size = static_cast<int>(p->page_size);
  x.page_shift = -1;
  for (int s = 0; s <= 20; ++s)
    if ((1 << s) == x.page_size) x.page_shift = s;
  x.batch = static_cast<int>(p->batch);
  x.hkv = static_cast<int>(p->heads_kv);
  x.d = static_cast<int>(p->head_dim);
  x.dtype = p->dtype;
  x.storage = p->storage;
  x.err = device_error_word();
  return GORGON_OK;
}

namespace {

constexpr int kThreads = 256;
constexpr int kCuCached = 1024;  // batches whose cumulative counts are searched in shared memory

template <int ST> struct Largest;
template <> struct Largest<GORGON_KV_INT8> { static constexpr float value = 127.f; };
template <> struct Largest<GORGON_KV_E4M3> { static constexpr float value = 448.f; };

// Row parameters from amax's bit pattern (|x| as an unsigned integer orders
// like |x|, with infinities and NaNs on top): scale to store, factor to apply.
template <int ST>
__device__ __forceinline__ void row_scale(uint32_t amax_bits, float& inv, float& scale) {
  if (amax_bits >= 0x7f800000u) {  // an infinity or a NaN in the row: it reads back as NaN
    inv = 0.f;
    scale = __int_as_float(0x7fc00000);
    return;
  }
  const float amax = fmaxf(__uint_as_float(amax_bits), 7.8886090522101181e-31f);  // 2^-100
  inv = __uint_as_float(__float_as_uint(Largest<ST>::value / amax) & 0xfffff000u);
  scale = 1.f / inv;
}

// inv == 0 marks the non-finite row: zeros, so that no stored byte depends on it.
template <int ST>
__device__ __forceinline__ uint8_t store8(float x, float inv) {
  const float y = inv == 0.f ? 0.f : x * inv;
  if constexpr (ST == GORGON_KV_INT8)
    return static_cast<uint8_t>(static_cast<int8_t>(__float2int_rn(y)));
  else
    return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

template <int ST>
__device__ __forceinline__ uint32_t store8x4(float a, float b, float c, float d, float inv) {
  if constexpr (ST == GORGON_KV_INT8) {
    return store8<ST>(a, inv) | store8<ST>(b, inv) << 8 | store8<ST>(c, inv) << 16 | static_cast<uint32_t>(store8<ST>(d, inv)) << 24;
  } else {
    const bool none = inv == 0.f;
    const float2 x = none ? make_float2(0.f, 0.f) : make_float2(a * inv, b * inv), y = none ? make_float2(0.f, 0.f) : make_float2(c * inv, d * inv);
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
}

template <int ST>
__device__ __forceinline__ float load8(uint8_t s) {
  if constexpr (ST == GORGON_KV_INT8) {
    return static_cast<float>(static_cast<int8_t>(s));
  } else {
    __nv_fp8_e4m3 f;
    f.__x = s;
    return static_cast<float>(f);
  }
}

// What a stored byte stands for.  inv is cut downwards, so the largest byte may
// stand for up to 2^-11 more than the value it came from: at the very top of a
// type that would round to an infinity, so results stop at the type's largest
// finite value (a row's NaN scale stays NaN).
__device__ __forceinline__ float stands_for(float stored, float scale, float top) {
  const float y = stored * scale;
  return scale == scale ? fminf(fmaxf(y, -top), top) : y;
}
template <typename T> __host__ __device__ constexpr float type_top() { return 3.402823466e38f; }
template <> __host__ __device__ constexpr float type_top<__half>() { return 65504.f; }
template <> __host__ __device__ constexpr float type_top<__nv_bfloat16>() { return 3.3895313892515355e38f; }

struct AppendArgs {
  PagedPool pool;
  const char* k;
  const char* v;
  int64_t k_sb, k_sh, k_sn;  // bytes
  int64_t v_sb, v_sh, v_sn;
  NewRows nr;
  int64_t items;  // (row, head) pairs
};

struct ReadArgs {
  PagedPool pool;
  char* k;
  char* v;
  int64_t k_sn, k_sh, v_sn, v_sh;  // bytes
  const int32_t* cu;
  const int32_t* starts;
  int out_dtype;
  int64_t items;
};

// Cumulative counts in shared memory (one load round trip instead of a chain
// of dependent ones in the search), or the global array for large batches.
__device__ __forceinline__ const int32_t* cached_cu(const int32_t* cu, int batch, int32_t* buf) {
  if (!cu || batch > kCuCached) return cu;
  for (int i = threadIdx.x; i <= batch; i += blockDim.x) buf[i] = cu[i];
  __syncthreads();
  return buf;
}

// Cumulative counts that fall, or begin below 0, are reported (by one CTA): rows
// are found by a search among them, so some of a call's rows may be left out.
__device__ __forceinline__ void report_counts(const int32_t* cu, int batch, uint32_t* err) {
  if (!cu || blockIdx.x != 0) return;
  bool bad = threadIdx.x == 0 && cu[0] < 0;
  for (int i = threadIdx.x; i < batch; i += blockDim.x) bad |= cu[i] > cu[i + 1];
  if (bad) raise_device_error(err, kErrBadSeqlen);
}

struct Place {
  int b, i;      // sequence, number among its new rows
  int page, row;
  bool ok;
};

__device__ __forceinline__ Place append_place(const AppendArgs& a, const int32_t* cu, int r, bool report) {
  Place p{};
  int c;
  if (cu) {
    if (r < cu[0] || r >= cu[a.pool.batch]) return p;  // padding behind the last sequence
    p.b = sequence_of(cu, a.pool.batch, r);
    if (cu[p.b] < 0) {
      if (report) raise_device_error(a.pool.err, kErrBadSeqlen);
      return p;
    }
    p.i = r - cu[p.b];
    c = cu[p.b + 1] - cu[p.b];
  } else {
    c = a.nr.n;
    p.b = r / c;
    p.i = r - p.b * c;
  }
  const int L = a.pool.lens[p.b];
  // (a row outside its sequence: cu is out of order)
  if (L < c || p.i < 0 || p.i >= c || L - c + p.i < 0) {
    if (L != 0 && report) raise_device_error(a.pool.err, kErrBadSeqlen);
    return p;
  }
  int col;
  a.pool.split(L - c + p.i, col, p.row);
  p.page = a.pool.page(p.b, col);
  p.ok = p.page >= 0;
  return p;
}

// 16-bit rows of D = 8 * LPR values: LPR threads hold a row's 16-byte pieces
// of K and of V, and find its largest magnitude by shuffles.  They take HP heads
// of a row: where a row goes (its sequence, length and page: three dependent
// loads) is found once for them, and their loads are in flight together.
template <typename T, int ST, int LPR, int HP>
__global__ void __launch_bounds__(kThreads) paged_append_vec_kernel(const AppendArgs a) {
  __shared__ int32_t s_cu[kCuCached + 1];
  const int32_t* cu = cached_cu(a.nr.cu, a.pool.batch, s_cu);
  report_counts(cu, a.pool.batch, a.pool.err);
  const int sub = threadIdx.x % LPR;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / LPR;
  const int per_row = (a.pool.hkv + HP - 1) / HP;
  const bool live = item < a.items;
  const int r = live ? static_cast<int>(item / per_row) : 0;
  const int h0 = live ? static_cast<int>(item - static_cast<int64_t>(r) * per_row) * HP : 0;
  Place p{};
  if (live) p = append_place(a, cu, r, sub == 0);
  const int64_t rn = cu ? r : p.i;
  const int64_t rb = cu ? 0 : p.b;
  uint4 raw[HP][2] = {};
#pragma unroll
  for (int k = 0; k < HP; ++k)
    if (p.ok && h0 + k < a.pool.hkv) {
      raw[k][0] = __ldcs(reinterpret_cast<const uint4*>(a.k + rb * a.k_sb + (h0 + k) * a.k_sh + rn * a.k_sn) + sub);
      raw[k][1] = __ldcs(reinterpret_cast<const uint4*>(a.v + rb * a.v_sb + (h0 + k) * a.v_sh + rn * a.v_sn) + sub);
    }
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = h0 + k;
    const bool ok = p.ok && h < a.pool.hkv;
    char* dst[2] = {a.pool.k + p.page * a.pool.k_sp + h * a.pool.k_sh + p.row * a.pool.k_ss,
                    a.pool.v + p.page * a.pool.v_sp + h * a.pool.v_sh + p.row * a.pool.v_ss};
    if constexpr (ST == GORGON_KV_NATIVE) {
      if (ok) {
        reinterpret_cast<uint4*>(dst[0])[sub] = raw[k][0];
        reinterpret_cast<uint4*>(dst[1])[sub] = raw[k][1];
      }
    } else {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        // |x| as 16-bit integers, two at a time, orders like |x| (infinities and NaN on top)
        const uint32_t* two = reinterpret_cast<const uint32_t*>(&raw[k][kv]);
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __vmaxu2(top, two[j] & 0x7fff7fffu);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint16_t most = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
        float inv, scale;
        row_scale<ST>(__float_as_uint(Cvt<T>::to_f(*reinterpret_cast<const T*>(&most))), inv, scale);
        const T* e = reinterpret_cast<const T*>(&raw[k][kv]);
        if (ok) {
          uint2 w;
          w.x = store8x4<ST>(Cvt<T>::to_f(e[0]), Cvt<T>::to_f(e[1]), Cvt<T>::to_f(e[2]), Cvt<T>::to_f(e[3]), inv);
          w.y = store8x4<ST>(Cvt<T>::to_f(e[4]), Cvt<T>::to_f(e[5]), Cvt<T>::to_f(e[6]), Cvt<T>::to_f(e[7]), inv);
          reinterpret_cast<uint2*>(dst[kv])[sub] = w;
          if (sub == 0) {
            float* sc = kv ? a.pool.vs + p.page * a.pool.vs_sp + h * a.pool.vs_sh + p.row * a.pool.vs_ss
                           : a.pool.ks + p.page * a.pool.ks_sp + h * a.pool.ks_sh + p.row * a.pool.ks_ss;
            *sc = scale;
          }
        }
      }
    }
  }
}

// Any dtype, head_dim and alignment: a warp per (row, head).
template <typename T, int ST>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const AppendArgs a) {
  __shared__ int32_t s_cu[kCuCached + 1];
  const int32_t* cu = cached_cu(a.nr.cu, a.pool.batch, s_cu);
  report_counts(cu, a.pool.batch, a.pool.err);
  const int lane = threadIdx.x & 31;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / 32;
  if (item >= a.items) return;
  const int r = static_cast<int>(item / a.pool.hkv);
  const int h = static_cast<int>(item - static_cast<int64_t>(r) * a.pool.hkv);
  const Place p = append_place(a, cu, r, lane == 0);
  if (!p.ok) return;
  const int64_t rn = cu ? r : p.i;
  const int64_t rb = cu ? 0 : p.b;
  for (int kv = 0; kv < 2; ++kv) {
    const T* src = reinterpret_cast<const T*>(kv ? a.v + rb * a.v_sb + h * a.v_sh + rn * a.v_sn
                                                 : a.k + rb * a.k_sb + h * a.k_sh + rn * a.k_sn);
    char* dst = kv ? a.pool.v + p.page * a.pool.v_sp + h * a.pool.v_sh + p.row * a.pool.v_ss
                   : a.pool.k + p.page * a.pool.k_sp + h * a.pool.k_sh + p.row * a.pool.k_ss;
    if constexpr (ST == GORGON_KV_NATIVE) {
      for (int d = lane; d < a.pool.d; d += 32) reinterpret_cast<T*>(dst)[d] = src[d];
    } else {
      uint32_t top = 0;
      for (int d = lane; d < a.pool.d; d += 32) top = max(top, __float_as_uint(Cvt<T>::to_f(src[d])) & 0x7fffffffu);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      float inv, scale;
      row_scale<ST>(top, inv, scale);
      for (int d = lane; d < a.pool.d; d += 32)
        reinterpret_cast<uint8_t*>(dst)[d] = store8<ST>(Cvt<T>::to_f(src[d]), inv);
      if (lane == 0) {
        if (kv) a.pool.vs[p.page * a.pool.vs_sp + h * a.pool.vs_sh + p.row * a.pool.vs_ss] = scale;
        else a.pool.ks[p.page * a.pool.ks_sp + h * a.pool.ks_sh + p.row * a.pool.ks_ss] = scale;
      }
    }
  }
}

__device__ __forceinline__ Place read_place(const ReadArgs& a, const int32_t* cu, int r) {
  Place p{};
  if (r < cu[0] || r >= cu[a.pool.batch]) return p;
  p.b = sequence_of(cu, a.pool.batch, r);
  p.i = cu[p.b] < 0 ? -1 : r - cu[p.b];
  const int64_t pos = static_cast<int64_t>(a.starts ? a.starts[p.b] : 0) + p.i;
  if (p.i < 0 || pos < 0 || pos > INT32_MAX) {
    raise_device_error(a.pool.err, kErrBadSeqlen);
    return p;
  }
  int col;
  a.pool.split(static_cast<int>(pos), col, p.row);
  p.page = a.pool.page(p.b, col);
  p.ok = p.page >= 0;
  return p;
}

__device__ __forceinline__ uint32_t pair16(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair16(float x, float y, __half) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Rows of 16 * LPR stored bytes to rows of T (the pages' own type when NATIVE),
// HP heads of a row for every LPR threads (as above).
template <typename T, int ST, int LPR, int HP>
__global__ void __launch_bounds__(kThreads) paged_read_vec_kernel(const ReadArgs a) {
  __shared__ int32_t s_cu[kCuCached + 1];
  const int32_t* cu = cached_cu(a.cu, a.pool.batch, s_cu);
  report_counts(cu, a.pool.batch, a.pool.err);
  const int sub = threadIdx.x % LPR;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / LPR;
  if (item >= a.items) return;
  const int per_row = (a.pool.hkv + HP - 1) / HP;
  const int r = static_cast<int>(item / per_row);
  const int h0 = static_cast<int>(item - static_cast<int64_t>(r) * per_row) * HP;
  const Place p = read_place(a, cu, r);
  if (!p.ok) return;
  const char* src[2] = {a.pool.k + p.page * a.pool.k_sp + p.row * a.pool.k_ss, a.pool.v + p.page * a.pool.v_sp + p.row * a.pool.v_ss};
  uint4 raw[HP][2] = {};
  float sc[HP][2] = {};
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = h0 + k;
    if (h >= a.pool.hkv) break;
    raw[k][0] = __ldcs(reinterpret_cast<const uint4*>(src[0] + h * a.pool.k_sh) + sub);
    raw[k][1] = __ldcs(reinterpret_cast<const uint4*>(src[1] + h * a.pool.v_sh) + sub);
    if constexpr (ST != GORGON_KV_NATIVE) {
      sc[k][0] = a.pool.ks[p.page * a.pool.ks_sp + h * a.pool.ks_sh + p.row * a.pool.ks_ss];
      sc[k][1] = a.pool.vs[p.page * a.pool.vs_sp + h * a.pool.vs_sh + p.row * a.pool.vs_ss];
    }
  }
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = h0 + k;
    if (h >= a.pool.hkv) break;
    uint4* out[2] = {reinterpret_cast<uint4*>(a.k + r * a.k_sn + h * a.k_sh),
                     reinterpret_cast<uint4*>(a.v + r * a.v_sn + h * a.v_sh)};
    if constexpr (ST == GORGON_KV_NATIVE) {
      __stcs(out[0] + sub, raw[k][0]);
      __stcs(out[1] + sub, raw[k][1]);
    } else {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* e = reinterpret_cast<const uint8_t*>(&raw[k][kv]);
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[j] = pair16(stands_for(load8<ST>(e[2 * j]), sc[k][kv], type_top<T>()),
                        stands_for(load8<ST>(e[2 * j + 1]), sc[k][kv], type_top<T>()), T{});
        __stcs(out[kv] + 2 * sub, make_uint4(w[0], w[1], w[2], w[3]));
        __stcs(out[kv] + 2 * sub + 1, make_uint4(w[4], w[5], w[6], w[7]));
      }
    }
  }
}

template <typename T, int ST>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const ReadArgs a) {
  __shared__ int32_t s_cu[kCuCached + 1];
  const int32_t* cu = cached_cu(a.cu, a.pool.batch, s_cu);
  report_counts(cu, a.pool.batch, a.pool.err);
  const int lane = threadIdx.x & 31;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / 32;
  if (item >= a.items) return;
  const int r = static_cast<int>(item / a.pool.hkv);
  const int h = static_cast<int>(item - static_cast<int64_t>(r) * a.pool.hkv);
  const Place p = read_place(a, cu, r);
  if (!p.ok) return;
  for (int kv = 0; kv < 2; ++kv) {
    const char* src = kv ? a.pool.v + p.page * a.pool.v_sp + h * a.pool.v_sh + p.row * a.pool.v_ss
                         : a.pool.k + p.page * a.pool.k_sp + h * a.pool.k_sh + p.row * a.pool.k_ss;
    char* out = kv ? a.v + r * a.v_sn + h * a.v_sh : a.k + r * a.k_sn + h * a.k_sh;
    float sc = 1.f;
    if constexpr (ST != GORGON_KV_NATIVE)
      sc = kv ? a.pool.vs[p.page * a.pool.vs_sp + h * a.pool.vs_sh + p.row * a.pool.vs_ss]
              : a.pool.ks[p.page * a.pool.ks_sp + h * a.pool.ks_sh + p.row * a.pool.ks_ss];
    for (int d = lane; d < a.pool.d; d += 32) {
      float x;
      if constexpr (ST == GORGON_KV_NATIVE) x = Cvt<T>::to_f(reinterpret_cast<const T*>(src)[d]);
      else x = stands_for(load8<ST>(reinterpret_cast<const uint8_t*>(src)[d]), sc,
                          a.out_dtype == GORGON_F16 ? type_top<__half>()
                                                    : a.out_dtype == GORGON_BF16 ? type_top<__nv_bfloat16>() : type_top<float>());
      store_as(out, a.out_dtype, d, x);
    }
  }
}

// ------------------------------------------------------------------- trim
struct TrimArgs {
  PagedPool pool;
  int64_t k_sl, v_sl;    // byte strides of a layer
  int64_t ks_sl, vs_sl;  // scales, element strides
  int layers;
  const int32_t* idx;
  int64_t idx_sb;
  int max_len;
  const int32_t* lens;
  const int32_t* dst_start;
  int row_bytes;
};

// Checks sequence b's trim with one warp's lanes over r = lane, lane + 32, ...
__device__ __forceinline__ bool trim_ok(const TrimArgs& a, int b, int len, int d0, int lane, bool report) {
  const int64_t cap = static_cast<int64_t>(a.pool.table_cols) * a.pool.page_size;
  bool bad = len < 0 || len > a.max_len || d0 < 0 || static_cast<int64_t>(d0) + max(len, 0) > cap;
  bool bad_page = false;
  if (!bad) {
    for (int r = lane; r < len; r += 32) {
      const int s = a.idx[b * a.idx_sb + r];
      if (s < 0 || s >= cap) {
        bad = true;
        continue;
      }
      int c0, c1, row;
      a.pool.split(s, c0, row);
      a.pool.split(d0 + r, c1, row);
      const int32_t* tb = a.pool.table + static_cast<int64_t>(b) * a.pool.table_sb;
      const int p0 = tb[c0], p1 = tb[c1];
      bad_page |= p0 < 0 || p0 >= a.pool.num_pages || p1 < 0 || p1 >= a.pool.num_pages;
    }
  }
  const bool any = __any_sync(0xffffffffu, bad), any_page = __any_sync(0xffffffffu, bad_page);
  if (lane == 0 && report) {
    if (any) raise_device_error(a.pool.err, kErrBadTrimIndex);
    else if (any_page) raise_device_error(a.pool.err, kErrBadPage);
  }
  return !any && !any_page;
}

// Aligned rows, at most 32 of them and kChunks * 32 16-byte chunks: a warp per
// (layer, sequence, head) moves its K and V rows (and scales) through
// registers, every load before any store, so rows may overlap.
constexpr int kTrimWarps = 8;
template <int kChunks>
__global__ void __launch_bounds__(kTrimWarps * 32) paged_trim_warp_kernel(const TrimArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x * kTrimWarps + warp;
  const int b = blockIdx.y, layer = blockIdx.z;
  if (h >= a.pool.hkv) return;
  const int len = a.lens[b];
  const int d0 = a.dst_start ? a.dst_start[b] : 0;
  if (!trim_ok(a, b, len, d0, lane, h == 0 && layer == 0)) return;
  if (len == 0) return;
  // lane r: byte offsets of source and destination row r
  int64_t ks = 0, kd = 0, vs = 0, vd = 0;
  int p0 = 0, r0 = 0, p1 = 0, r1 = 0;
  if (lane < len) {
    int c;
    a.pool.split(a.idx[b * a.idx_sb + lane], c, r0);
    p0 = a.pool.table[static_cast<int64_t>(b) * a.pool.table_sb + c];
    a.pool.split(d0 + lane, c, r1);
    p1 = a.pool.table[static_cast<int64_t>(b) * a.pool.table_sb + c];
    ks = p0 * a.pool.k_sp + r0 * a.pool.k_ss;
    kd = p1 * a.pool.k_sp + r1 * a.pool.k_ss;
    vs = p0 * a.pool.v_sp + r0 * a.pool.v_ss;
    vd = p1 * a.pool.v_sp + r1 * a.pool.v_ss;
  }
  char* kb = a.pool.k + layer * a.k_sl + h * a.pool.k_sh;
  char* vb = a.pool.v + layer * a.v_sl + h * a.pool.v_sh;
  const int vpr = a.row_bytes / 16;
  const int total = len * vpr;
  uint4 kx[kChunks], vx[kChunks];
#pragma unroll
  for (int q = 0; q < kChunks; ++q) {
    const int e = lane + 32 * q;
    const int r = e / vpr, c = e - r * vpr;
    const int64_t ko = __shfl_sync(0xffffffffu, ks, min(r, 31)), vo = __shfl_sync(0xffffffffu, vs, min(r, 31));
    if (e < total) {
      kx[q] = *reinterpret_cast<const uint4*>(kb + ko + c * 16);
      vx[q] = *reinterpret_cast<const uint4*>(vb + vo + c * 16);
    }
  }
  float ksc = 0.f, vsc = 0.f;
  const bool sc = a.pool.storage != GORGON_KV_NATIVE && lane < len;
  if (sc) {
    ksc = a.pool.ks[layer * a.ks_sl + p0 * a.pool.ks_sp + h * a.pool.ks_sh + r0 * a.pool.ks_ss];
    vsc = a.pool.vs[layer * a.vs_sl + p0 * a.pool.vs_sp + h * a.pool.vs_sh + r0 * a.pool.vs_ss];
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < kChunks; ++q) {
    const int e = lane + 32 * q;
    const int r = e / vpr, c = e - r * vpr;
    const int64_t ko = __shfl_sync(0xffffffffu, kd, min(r, 31)), vo = __shfl_sync(0xffffffffu, vd, min(r, 31));
    if (e < total) {
      *reinterpret_cast<uint4*>(kb + ko + c * 16) = kx[q];
      *reinterpret_cast<uint4*>(vb + vo + c * 16) = vx[q];
    }
  }
  if (sc) {
    a.pool.ks[layer * a.ks_sl + p1 * a.pool.ks_sp + h * a.pool.ks_sh + r1 * a.pool.ks_ss] = ksc;
    a.pool.vs[layer * a.vs_sl + p1 * a.pool.vs_sp + h * a.pool.vs_sh + r1 * a.pool.vs_ss] = vsc;
  }
}

// Any row size: a CTA per (layer, sequence, head) and K or V, through shared memory,
// as many bytes of every row at a time as the stage holds (a column of the rows
// depends on that column alone, so rows may overlap all the same).  The stage is one that every launch may have: a larger limit
// is an attribute of the kernel, which two host threads would set for each other.
constexpr int kTrimThreads = 128;
constexpr int kTrimRows = 256;
constexpr int kTrimStage = 44 * 1024;
__global__ void __launch_bounds__(kTrimThreads) paged_trim_kernel(const TrimArgs a, int stage_bytes) {
  extern __shared__ uint8_t stage[];
  __shared__ int64_t s_row[kTrimRows];  // byte offsets of the rows read, then of those written
  __shared__ float s_scale[kTrimRows];
  __shared__ int s_ok;
  const int h = blockIdx.x, b = blockIdx.y;
  const int layer = blockIdx.z >> 1, kv = blockIdx.z & 1;
  const int len = a.lens[b];
  const int d0 = a.dst_start ? a.dst_start[b] : 0;
  if (threadIdx.x < 32) {
    const bool ok = trim_ok(a, b, len, d0, threadIdx.x, h == 0 && blockIdx.z == 0);
    if (threadIdx.x == 0) s_ok = ok;
  }
  __syncthreads();
  if (!s_ok || len == 0) return;
  const int32_t* tb = a.pool.table + static_cast<int64_t>(b) * a.pool.table_sb;
  char* base = kv ? a.pool.v + layer * a.v_sl + h * a.pool.v_sh : a.pool.k + layer * a.k_sl + h * a.pool.k_sh;
  const int64_t sp = kv ? a.pool.v_sp : a.pool.k_sp, ss = kv ? a.pool.v_ss : a.pool.k_ss;
  const bool scaled = a.pool.storage != GORGON_KV_NATIVE;
  float* sbase = nullptr;
  int64_t ssp = 0, sss = 0;
  if (scaled) {
    sbase = kv ? a.pool.vs + layer * a.vs_sl + h * a.pool.vs_sh : a.pool.ks + layer * a.ks_sl + h * a.pool.ks_sh;
    ssp = kv ? a.pool.vs_sp : a.pool.ks_sp;
    sss = kv ? a.pool.vs_ss : a.pool.ks_ss;
  }
  auto at = [&](int pos, int& page, int& row) {
    int col;
    a.pool.split(pos, col, row);
    page = tb[col];
  };
  int page, row;
  auto look_up = [&](auto pos, bool scales) {
    for (int r = threadIdx.x; r < len; r += kTrimThreads) {
      at(pos(r), page, row);
      s_row[r] = page * sp + row * ss;
      if (scales) s_scale[r] = sbase[page * ssp + row * sss];
    }
    __syncthreads();
  };
  auto source = [&](int r) { return a.idx[b * a.idx_sb + r]; };
  auto target = [&](int r) { return d0 + r; };
  const int width = min(a.row_bytes, stage_bytes / len);
  for (int c0 = 0; c0 < a.row_bytes; c0 += width) {
    const int w = min(width, a.row_bytes - c0);
    // (four loads before their stores: the compiler keeps loads of offsets behind stores of bytes)
    auto move = [&](auto load, auto store) {
      for (int e0 = threadIdx.x; e0 < len * w; e0 += kTrimThreads * 4) {
        uint8_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = e0 + k * kTrimThreads, r = e / w;
          if (e < len * w) x[k] = load(e, r, c0 + e - r * w);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = e0 + k * kTrimThreads, r = e / w;
          if (e < len * w) store(e, r, c0 + e - r * w, x[k]);
        }
      }
    };
    look_up(source, scaled && c0 == 0);
    move([&](int, int r, int c) { return static_cast<uint8_t>(base[s_row[r] + c]); }, [&](int e, int, int, uint8_t x) { stage[e] = x; });
    __syncthreads();
    look_up(target, false);
    move([&](int e, int, int) { return stage[e]; }, [&](int, int r, int c, uint8_t x) { base[s_row[r] + c] = static_cast<char>(x); });
    __syncthreads();
  }
  if (scaled)
    for (int r = threadIdx.x; r < len; r += kTrimThreads) {
      at(target(r), page, row);
      sbase[page * ssp + row * sss] = s_scale[r];
    }
}

// ---------------------------------------------------------------- dispatch
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool m16(int64_t a, int64_t b, int64_t c) { return ((a | b | c) & 15) == 0; }

template <typename F>
int by_lpr(int lpr, F&& f) {
  switch (lpr) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 4: return f(std::integral_constant<int, 4>());
    case 8: return f(std::integral_constant<int, 8>());
    case 16: return f(std::integral_constant<int, 16>());
    default: return f(std::integral_constant<int, 32>());
  }
}
inline bool pow2_upto32(int x) { return x >= 1 && x <= 32 && (x & (x - 1)) == 0; }

// How many groups of LPR threads the (row, head) pairs take: `heads` heads each
// once the pairs alone would fill the SMs (2048 threads each) twice over, where
// the lookups' latency counts for every wave (a read of 16 sequences of up to
// 8192 int8 rows: 75 us a head each, 66 us with four, 5.9 TB/s; an append of 8000
// rows to e4m3: 18.1 us with four, 17.0 us with two, 2.9 TB/s, the issue slots 67 %
// busy); one head each below, where all run at once (64 single rows:
// 3.4 us either way, a launch).
int64_t groups(int64_t items, int hkv, int lpr, int heads) {
  if (items * lpr < int64_t(2) * 2048 * sm_count()) return items;
  return items / hkv * ceil_div(hkv, heads);
}

template <typename T, int ST>
int append_t(const AppendArgs& a, bool vec, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    const int lpr = a.pool.d / 8;
    if (vec && a.pool.d % 8 == 0 && pow2_upto32(lpr))
      return by_lpr(lpr, [&](auto l) {
        constexpr int LPR = decltype(l)::value;
        constexpr int kHeads = 2;
        AppendArgs x = a;
        x.items = groups(a.items, a.pool.hkv, LPR, kHeads);
        const unsigned blocks = static_cast<unsigned>(ceil_div(x.items * LPR, kThreads));
        if (x.items < a.items) paged_append_vec_kernel<T, ST, LPR, kHeads><<<blocks, kThreads, 0, st>>>(x);
        else paged_append_vec_kernel<T, ST, LPR, 1><<<blocks, kThreads, 0, st>>>(x);
        return check_cuda(cudaGetLastError(), "gorgon_paged_append launch");
      });
  }
  paged_append_kernel<T, ST><<<static_cast<unsigned>(ceil_div(a.items * 32, kThreads)), kThreads, 0, st>>>(a);
  return check_cuda(cudaGetLastError(), "gorgon_paged_append launch");
}

template <typename T>
int append_s(const AppendArgs& a, bool vec, cudaStream_t st) {
  switch (a.pool.storage) {
    case GORGON_KV_NATIVE: return append_t<T, GORGON_KV_NATIVE>(a, vec, st);
    case GORGON_KV_INT8: return append_t<T, GORGON_KV_INT8>(a, vec, st);
    default: return append_t<T, GORGON_KV_E4M3>(a, vec, st);
  }
}

template <typename T, int ST>
int read_t(const ReadArgs& a, bool vec, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    const int per = ST == GORGON_KV_NATIVE ? 8 : 16;
    const int lpr = a.pool.d / per;
    if (vec && a.pool.d % per == 0 && pow2_upto32(lpr))
      return by_lpr(lpr, [&](auto l) {
        constexpr int LPR = decltype(l)::value;
        constexpr int kHeads = 4;
        ReadArgs x = a;
        x.items = groups(a.items, a.pool.hkv, LPR, kHeads);
        const unsigned blocks = static_cast<unsigned>(ceil_div(x.items * LPR, kThreads));
        if (x.items < a.items) paged_read_vec_kernel<T, ST, LPR, kHeads><<<blocks, kThreads, 0, st>>>(x);
        else paged_read_vec_kernel<T, ST, LPR, 1><<<blocks, kThreads, 0, st>>>(x);
        return check_cuda(cudaGetLastError(), "gorgon_paged_read launch");
      });
  }
  paged_read_kernel<T, ST><<<static_cast<unsigned>(ceil_div(a.items * 32, kThreads)), kThreads, 0, st>>>(a);
  return check_cuda(cudaGetLastError(), "gorgon_paged_read launch");
}

}  // namespace
}  // namespace gorgon

extern "C" int gorgon_paged_append(const gorgon_paged_append_params* p, void* stream) {
  using namespace gorgon;
  if (!p) return set_error(GORGON_ERR_INVALID, "gorgon_paged_append: params is null");
  AppendArgs a{};
  int rc = make_pool(&p->kv, "gorgon_paged_append", &a.pool);
  if (rc) return rc;
  if (p->n < 0 || p->rows < 0 || p->n > INT32_MAX) return set_error(GORGON_ERR_INVALID, "gorgon_paged_append: negative size");
  const int64_t rows = p->cu_q ? p->rows : p->kv.batch * p->n;
  if (rows > INT32_MAX) return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_append: more than 2^31 rows");
  a.items = rows * a.pool.hkv;
  if (a.items == 0 || a.pool.d == 0 || a.pool.batch == 0) return GORGON_OK;
  if (!p->k || !p->v || !a.pool.lens) return set_error(GORGON_ERR_INVALID, "gorgon_paged_append: null pointer");
  if (a.items > (int64_t(1) << 34)) return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_append: too many rows");
  const int64_t es = static_cast<int64_t>(dtype_bytes(p->kv.dtype));
  a.k = static_cast<const char*>(p->k);
  a.v = static_cast<const char*>(p->v);
  a.k_sb = p->k_stride_b * es; a.k_sh = p->k_stride_h * es; a.k_sn = p->k_stride_n * es;
  a.v_sb = p->v_stride_b * es; a.v_sh = p->v_stride_h * es; a.v_sn = p->v_stride_n * es;
  a.nr = NewRows{p->cu_q, static_cast<int>(p->n)};
  bool vec = al16(a.k) && al16(a.v) && m16(a.k_sb, a.k_sh, a.k_sn) && m16(a.v_sb, a.v_sh, a.v_sn) && al16(a.pool.k) &&
             al16(a.pool.v) && m16(a.pool.k_sp, a.pool.k_sh, a.pool.k_ss) && m16(a.pool.v_sp, a.pool.v_sh, a.pool.v_ss);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (p->kv.dtype) {
    case GORGON_F32: return append_s<float>(a, vec, st);
    case GORGON_BF16: return append_s<__nv_bfloat16>(a, vec, st);
    default: return append_s<__half>(a, vec, st);
  }
}

extern "C" int gorgon_paged_read(const gorgon_paged_read_params* p, void* stream) {
  using namespace gorgon;
  if (!p) return set_error(GORGON_ERR_INVALID, "gorgon_paged_read: params is null");
  ReadArgs a{};
  int rc = make_pool(&p->kv, "gorgon_paged_read", &a.pool);
  if (rc) return rc;
  if (!dtype_ok(p->out_dtype)) return set_error(GORGON_ERR_INVALID, "gorgon_paged_read: unknown out_dtype");
  if (p->rows < 0) return set_error(GORGON_ERR_INVALID, "gorgon_paged_read: negative size");
  if (p->rows > INT32_MAX) return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_read: more than 2^31 rows");
  a.items = p->rows * a.pool.hkv;
  if (a.items == 0 || a.pool.d == 0 || a.pool.batch == 0) return GORGON_OK;
  if (!p->k || !p->v || !p->cu_rows) return set_error(GORGON_ERR_INVALID, "gorgon_paged_read: null pointer");
  if (a.items > (int64_t(1) << 34)) return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_read: too many rows");
  const int64_t es = static_cast<int64_t>(dtype_bytes(p->out_dtype));
  a.k = static_cast<char*>(p->k);
  a.v = static_cast<char*>(p->v);
  a.k_sn = p->k_stride_n * es; a.k_sh = p->k_stride_h * es;
  a.v_sn = p->v_stride_n * es; a.v_sh = p->v_stride_h * es;
  a.cu = p->cu_rows;
  a.starts = p->starts;
  a.out_dtype = p->out_dtype;
  const bool vec = al16(a.k) && al16(a.v) && m16(a.k_sn, a.k_sh, 0) && m16(a.v_sn, a.v_sh, 0) && al16(a.pool.k) &&
                   al16(a.pool.v) && m16(a.pool.k_sp, a.pool.k_sh, a.pool.k_ss) &&
                   m16(a.pool.v_sp, a.pool.v_sh, a.pool.v_ss);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->kv.storage == GORGON_KV_NATIVE) {
    const bool v = vec && p->out_dtype == p->kv.dtype;
    switch (p->kv.dtype) {
      case GORGON_F32: return read_t<float, GORGON_KV_NATIVE>(a, v, st);
      case GORGON_BF16: return read_t<__nv_bfloat16, GORGON_KV_NATIVE>(a, v, st);
      default: return read_t<__half, GORGON_KV_NATIVE>(a, v, st);
    }
  }
  const bool v = vec && p->out_dtype != GORGON_F32;
  const bool half_out = p->out_dtype == GORGON_F16;
  if (p->kv.storage == GORGON_KV_INT8)
    return half_out ? read_t<__half, GORGON_KV_INT8>(a, v, st) : read_t<__nv_bfloat16, GORGON_KV_INT8>(a, v, st);
  return half_out ? read_t<__half, GORGON_KV_E4M3>(a, v, st) : read_t<__nv_bfloat16, GORGON_KV_E4M3>(a, v, st);
}

extern "C" int gorgon_paged_trim(const gorgon_paged_trim_params* p, void* stream) {
  using namespace gorgon;
  if (!p) return set_error(GORGON_ERR_INVALID, "gorgon_paged_trim: params is null");
  TrimArgs a{};
  int rc = make_pool(&p->kv, "gorgon_paged_trim", &a.pool);
  if (rc) return rc;
  if (p->layers < 0 || p->max_len < 0) return set_error(GORGON_ERR_INVALID, "gorgon_paged_trim: negative size");
  if (p->max_len > kTrimRows) return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_trim: max_len > 256");
  if (p->layers > 32767) return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_trim: layers > 32767");
  if (p->layers == 0 || a.pool.batch == 0 || a.pool.d == 0 || p->max_len == 0) return GORGON_OK;
  if (!p->src_idx || !p->lens || !a.pool.table) return set_error(GORGON_ERR_INVALID, "gorgon_paged_trim: null pointer");
  // Rows that are one in memory would be read and written by several warps at once.
  auto repeats = [&](int64_t layer, int64_t page, int64_t head, int64_t row) {
    return (p->layers > 1 && layer == 0) || (p->kv.num_pages > 1 && page == 0) || (p->kv.heads_kv > 1 && head == 0) ||
           (p->kv.page_size > 1 && row == 0);
  };
  const gorgon_paged_kv& kv = p->kv;
  if (repeats(p->k_stride_l, kv.k_stride_p, kv.k_stride_h, kv.k_stride_s) || repeats(p->v_stride_l, kv.v_stride_p, kv.v_stride_h, kv.v_stride_s) ||
      (kv.storage != GORGON_KV_NATIVE && (repeats(p->ks_stride_l, kv.ks_stride_p, kv.ks_stride_h, kv.ks_stride_s) ||
                                          repeats(p->vs_stride_l, kv.vs_stride_p, kv.vs_stride_h, kv.vs_stride_s))))
    return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_trim: layers, pages, kv heads or rows repeated by a stride of 0");
  const int64_t es = storage_bytes(p->kv.storage, p->kv.dtype);
  a.k_sl = p->k_stride_l * es;
  a.v_sl = p->v_stride_l * es;
  a.ks_sl = p->ks_stride_l;
  a.vs_sl = p->vs_stride_l;
  a.layers = static_cast<int>(p->layers);
  a.idx = p->src_idx;
  a.idx_sb = p->idx_stride_b;
  a.max_len = static_cast<int>(p->max_len);
  a.lens = p->lens;
  a.dst_start = p->dst_start;
  a.row_bytes = static_cast<int>(a.pool.d * es);
  const bool vec = a.row_bytes % 16 == 0 && al16(a.pool.k) && al16(a.pool.v) &&
                   m16(a.pool.k_sp, a.pool.k_sh, a.pool.k_ss) && m16(a.pool.v_sp, a.pool.v_sh, a.pool.v_ss) &&
                   m16(a.k_sl, a.v_sl, 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t chunks = p->max_len * (a.row_bytes / 16);
  if (vec && p->max_len <= 32 && chunks <= 32 * 8) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.pool.hkv, kTrimWarps)), static_cast<unsigned>(a.pool.batch),
                    static_cast<unsigned>(p->layers));
    if (chunks <= 32 * 4) paged_trim_warp_kernel<4><<<grid, kTrimWarps * 32, 0, st>>>(a);
    else paged_trim_warp_kernel<8><<<grid, kTrimWarps * 32, 0, st>>>(a);
    return check_cuda(cudaGetLastError(), "gorgon_paged_trim launch");
  }
  static_assert(kTrimStage / kTrimRows > 0 && kTrimStage + kTrimRows * 12 + 64 <= 48 * 1024, "a stage for every launch");
  const int smem = static_cast<int>(std::min<int64_t>(p->max_len * a.row_bytes, kTrimStage));
  const dim3 grid(static_cast<unsigned>(a.pool.hkv), static_cast<unsigned>(a.pool.batch),
                  2u * static_cast<unsigned>(p->layers));
  paged_trim_kernel<<<grid, kTrimThreads, static_cast<size_t>(smem), st>>>(a, smem);
  return check_cuda(cudaGetLastError(), "gorgon_paged_trim launch");
}

// gorgon_paged_attn: argument checking and kernel choice.
#include <algorithm>
#include <string>

#include "paged_attn.cuh"

namespace gorgon {
namespace {

// Nothing to write.  (Packed rows are, even where no sequence may bring any: they
// are too many then.  Rows of no values have a log-sum-exp.)
bool empty(const PagedAttn& a) {
  return a.pool.batch == 0 || a.hq == 0 || (a.n == 0 && !(a.nr.cu && a.rows > 0)) || (a.pool.d == 0 && !a.lse);
}

int make_args(const gorgon_paged_attn_params* p, PagedAttn* a) {
  if (!p) return set_error(GORGON_ERR_INVALID, "gorgon_paged_attn: params is null");
  PagedAttn& x = *a;
  x = PagedAttn{};
  int rc = make_pool(&p->kv, "gorgon_paged_attn", &x.pool);
  if (rc) return rc;
  if (p->heads_q < 0 || p->n < 0 || p->window < 0 || p->sinks < 0)
    return set_error(GORGON_ERR_INVALID, "gorgon_paged_attn: negative size");
  if (p->heads_q % p->kv.heads_kv != 0)
    return set_error(GORGON_ERR_INVALID, "gorgon_paged_attn: heads_q must be a multiple of heads_kv");
  if (p->heads_q > 65535 || p->n > (int64_t(1) << 24) || p->n * (p->heads_q / p->kv.heads_kv) > (int64_t(1) << 28))
    return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_attn: too many query rows");
  if (p->parents && p->n > kPagedMaxNodes)
    return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_attn: trees above 1024 nodes");
  if (!(p->scale >= 0.f && p->scale < INFINITY))
    return set_error(GORGON_ERR_INVALID, "gorgon_paged_attn: scale must be positive and finite");
  if (p->cu_q && (p->rows < 0 || p->rows > INT32_MAX))
    return set_error(GORGON_ERR_INVALID, "gorgon_paged_attn: bad count of packed rows");
  if (p->backend < GORGON_PAGED_AUTO || p->backend > GORGON_PAGED_TCGEN05)
    return set_error(GORGON_ERR_INVALID, "gorgon_paged_attn: unknown backend");
  const int64_t es = static_cast<int64_t>(dtype_bytes(p->kv.dtype));
  x.nr = NewRows{p->cu_q, static_cast<int>(p->n)};
  x.q = static_cast<const char*>(p->q);
  x.q_sb = p->q_stride_b * es; x.q_sh = p->q_stride_h * es; x.q_sn = p->q_stride_n * es;
  x.out = static_cast<char*>(p->out);
  x.o_sb = p->o_stride_b; x.o_sh = p->o_stride_h; x.o_sn = p->o_stride_n;
  x.lse = p->lse;
  x.l_sb = p->lse_stride_b; x.l_sh = p->lse_stride_h; x.l_sn = p->lse_stride_n;
  x.parents = p->parents;
  x.par_sb = p->parents_stride_b;
  x.max_depth = p->max_depth < 0 ? INT32_MAX : p->max_depth;
  x.window = static_cast<int>(std::min<int64_t>(p->window, int64_t(1) << 30));
  x.sinks = static_cast<int>(std::min<int64_t>(p->sinks, int64_t(1) << 30));
  x.hq = static_cast<int>(p->heads_q);
  x.group = x.hq / x.pool.hkv;
  x.n = static_cast<int>(p->n);
  if (x.group > 0) set_group_div(&x);
  x.rows = p->cu_q ? static_cast<int>(p->rows) : 0;
  const float scale = p->scale != 0.f ? p->scale : (x.pool.d > 0 ? 1.f / std::sqrt(static_cast<float>(x.pool.d)) : 1.f);
  x.scale_log2 = scale * 1.4426950408889634f;
  x.wait_ns = wait_limit_ns();
  if (!empty(x) && (!p->kv.seq_lens || (x.pool.d > 0 && (!p->out || (x.n > 0 && !p->q))) || (!p->kv.block_table && p->kv.table_cols > 0)))
    return set_error(GORGON_ERR_INVALID, "gorgon_paged_attn: null q, out, seq_lens or block table");
  return GORGON_OK;
}

enum class Kernel { kSimt, kMma, kTc, kNone };

// The schedule's places fit 32 bits (it counts them per `m` packed rows and 64
// positions, or more).
bool short_list(const PagedAttn& a, int m) {
  const int64_t blocks = static_cast<int64_t>(a.n) * a.group / m + 1;
  const int64_t tiles = static_cast<int64_t>(a.pool.table_cols) * a.pool.page_size / 64 + 6;
  return blocks * tiles < (int64_t(1) << 31) / (static_cast<int64_t>(a.pool.batch) * a.pool.hkv + 1);
}

Kernel choose(const gorgon_paged_attn_params* p, const PagedAttn& a) {
  if (a.n == 0 || a.pool.d == 0) return Kernel::kSimt;
  const bool mma = paged_mma_supported(a) && short_list(a, 8), tc = paged_tc_supported(a) && short_list(a, 128);
  switch (p->backend) {
    case GORGON_PAGED_SIMT: return Kernel::kSimt;
    case GORGON_PAGED_MMA: return mma ? Kernel::kMma : Kernel::kNone;
    case GORGON_PAGED_TCGEN05: return tc ? Kernel::kTc : Kernel::kNone;
    default:
      // The warp-level kernel passes the cache once for every 16 packed rows, the
      // tcgen05 kernel once for 256, at a higher price a pass where rows are widened.
      // 16 sequences of 8192 rows, us, warp-level / tcgen05: 16-bit 104 / 125 for 16
      // packed rows, 183 / 126 for 32; int8 93 / 215 for 16, 164 / 216 for 32, 243 / 217
      // for 48.  One sequence turns later (4096 rows: 16-bit 20 / 27 for 20, 33 / 27 for
      // 96; int8 25 / 31 for 48, 32 / 31 for 96).
      if (static_cast<int64_t>(a.n) * a.group > (p->kv.storage == GORGON_KV_NATIVE ? 16 : 32) && tc) return Kernel::kTc;
      return mma ? Kernel::kMma : Kernel::kSimt;
  }
}

constexpr size_t kAlign = 256;
inline size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

size_t cut_workspace(const PagedAttn& a) {
  const size_t rows = static_cast<size_t>(a.grid) * 2 * a.m;
  return align_up(a.grid * sizeof(CutUnit)) + align_up(rows * sizeof(float2)) + rows * a.pool.d * sizeof(float);
}

void place_workspace(PagedAttn* a, void* ws) {
  const size_t rows = static_cast<size_t>(a->grid) * 2 * a->m;
  char* w = static_cast<char*>(ws);
  a->cut = reinterpret_cast<CutUnit*>(w);
  a->part_ml = reinterpret_cast<float2*>(w + align_up(a->grid * sizeof(CutUnit)));
  a->part_o = reinterpret_cast<float*>(w + align_up(a->grid * sizeof(CutUnit)) + align_up(rows * sizeof(float2)));
}

}  // namespace
}  // namespace gorgon

extern "C" size_t gorgon_paged_attn_workspace_size(const gorgon_paged_attn_params* p) {
  using namespace gorgon;
  PagedAttn a;
  if (make_args(p, &a) != GORGON_OK || empty(a)) return 0;
  switch (choose(p, a)) {
    case Kernel::kMma:
      paged_mma_plan(&a);
      return cut_workspace(a);
    case Kernel::kTc:
      paged_tc_plan(&a);
      return cut_workspace(a);
    default: return 0;
  }
}

extern "C" int gorgon_paged_attn(const gorgon_paged_attn_params* p, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  using namespace gorgon;
  PagedAttn a;
  int rc = make_args(p, &a);
  if (rc) return rc;
  if (empty(a)) return GORGON_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Kernel k = choose(p, a);
  switch (k) {
    case Kernel::kSimt: return launch_paged_simt(a, st);
    case Kernel::kMma: paged_mma_plan(&a); break;
    case Kernel::kTc: paged_tc_plan(&a); break;
    default:
      return set_error(GORGON_ERR_UNSUPPORTED, "gorgon_paged_attn: the requested kernel needs a 16-bit dtype, head_dim 64 or "
                                               "128, rows of whole 16-byte pieces and (tcgen05) trees of at most 256 rows");
  }
  if (!workspace || workspace_bytes < cut_workspace(a))
    return set_error(GORGON_ERR_WORKSPACE, "gorgon_paged_attn: workspace smaller than gorgon_paged_attn_workspace_size()");
  place_workspace(&a, workspace);
  rc = k == Kernel::kTc ? launch_paged_tc(a, st) : launch_paged_mma(a, st);
  if (rc) return rc;
  return launch_paged_merge(a, st);
}

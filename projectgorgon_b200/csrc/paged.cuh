// A key/value cache in pages, as the paged kernels see it: where a position of
// a sequence lies, and how an 8-bit row stands for its values.
//
// Pages are [num_pages, heads_kv, page_size, head_dim] (any strides, head_dim
// contiguous), K and V apart.  A sequence is a row of the block table: its
// position p lies in page block_table[b, p / page_size], row p % page_size.
// 8-bit pages carry one fp32 scale per (page, kv head, row), for K and for V:
// a stored byte s stands for s * scale.  The scale comes from
//   inv = (largest / amax) cut to 12 significant bits,  scale = 1 / inv,
//   s = round_to_nearest_even(x * inv)       (largest: 127 int8, 448 e4m3)
// Cutting inv (a relative change of at most 2^-11, always towards the safe
// side of `largest`) makes x * inv exact in fp32 for every 16-bit x (11 + 12
// significant bits), so the stored byte is the correctly rounded one.
#pragma once

#include "common.cuh"

namespace gorgon {

constexpr uint32_t kErrBadPage = 1u << 6;  // a block-table entry outside the pool, or a length past the table

struct PagedPool {
  char* k;
  char* v;
  int64_t k_sp, k_sh, k_ss;  // byte strides of page, kv head, row
  int64_t v_sp, v_sh, v_ss;
  float* ks;                 // fp32 scales (8-bit storage), element strides below
  float* vs;
  int64_t ks_sp, ks_sh, ks_ss;
  int64_t vs_sp, vs_sh, vs_ss;
  const int32_t* table;
  int64_t table_sb;
  int table_cols;
  const int32_t* lens;
  int num_pages, page_size, page_shift;  // page_shift: log2(page_size), or -1
  int batch, hkv, d;
  int dtype, storage;
  uint32_t* err;

  __device__ __forceinline__ void split(int pos, int& col, int& row) const {
    if (page_shift >= 0) {
      col = pos >> page_shift;
      row = pos & (page_size - 1);
    } else {
      col = pos / page_size;
      row = pos - col * page_size;
    }
  }
  // Page of table column `col` of sequence b, or -1 (and the error bit) when
  // the column or the entry is out of range.
  __device__ __forceinline__ int page(int b, int col) const {
    int pg = -1;
    if (col < table_cols) pg = __ldg(table + static_cast<int64_t>(b) * table_sb + col);
    if (pg < 0 || pg >= num_pages) {
      raise_device_error(err, kErrBadPage);
      pg = -1;
    }
    return pg;
  }
};

// Fills `o` from the public parameters; returns GORGON_OK or an error code.
int make_pool(const gorgon_paged_kv* p, const char* who, PagedPool* o);

inline int64_t storage_bytes(int storage, int dtype) {
  return storage == GORGON_KV_NATIVE ? static_cast<int64_t>(dtype_bytes(dtype)) : 1;
}

// New rows of sequence b: [first, first + count) of the packed rows, or
// count = n rows of a padded batch.
struct NewRows {
  const int32_t* cu;  // null: every sequence brings n rows
  int n;
  __device__ __forceinline__ int count(int b) const { return cu ? cu[b + 1] - cu[b] : n; }
  __device__ __forceinline__ int first(int b) const { return cu ? cu[b] : 0; }
};

// Sequence of packed row r: the largest b with cu[b] <= r (cu in shared or global memory).
__device__ __forceinline__ int sequence_of(const int32_t* cu, int batch, int r) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= r) lo = mid; else hi = mid - 1;
  }
  return lo;
}

}  // namespace gorgon

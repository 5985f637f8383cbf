// The paged cache's device view and the checks that its entry points share.
#pragma once

#include "common.hpp"

namespace tqkv {
namespace paged {

constexpr int kMaxBatch = 1024;

// What kernels need of a tqkv_paged_kv: row t of sequence b of KV head h is
// row t % R of the block (page, h), page = table[b * tstride + t / R].
struct Pool {
  const int32_t* table;
  const int32_t* lens;
  float* weights;
  int64_t tstride;
  int64_t wstride;  // weights of one (sequence, KV head): tstride * R
  int64_t num_pages;
  int batch, Hkv, shift;  // R = 1 << shift
  int cap;                // rows that a sequence's row of the table can name
};

// Rows that sequence b holds, within the table and `most`.
__device__ __forceinline__ int held(const Pool& p, int b, int most) {
  const int n = p.lens[b];
  return n < 0 ? 0 : n < most ? n : most;
}

__device__ __forceinline__ bool valid_page(const Pool& p, int page) {
  return page >= 0 && page < p.num_pages;
}

// Row index (in units of rows of the pool's buffers) of row r of a page.
__device__ __forceinline__ int64_t pool_row(const Pool& p, int page, int h, int r) {
  return ((int64_t(page) * p.Hkv + h) << p.shift) + r;
}

inline bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Checks a tqkv_paged_kv and fills the kernels' view. TQKV_OK or the failure.
int32_t check(const tqkv_paged_kv* kv, Pool* out);

}  // namespace paged
}  // namespace tqkv

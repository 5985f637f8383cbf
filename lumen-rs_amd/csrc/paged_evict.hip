// Paged cache: eviction by gathered attention weight.
//
// Two launches. (1) One workgroup per (sequence, KV head) finds the weight of
// the last row that still fits (a radix select over the weights' bits, 11, 11
// and 10 a pass, histograms in LDS), then goes over the rows once more in
// their order and writes the kept positions, ascending: forced rows (the
// first `sinks`, the last `recent`) and heavier rows all, rows of exactly that
// weight while there is room. Bound by latency and by LDS atomics: 4 bytes a
// row, read four times, from the caches after the first. (2) The gather moves
// the rows to their new pages, 16 bytes a thread, bound by HBM.
#include <cmath>

#include "paged.hpp"

namespace tqkv {
namespace paged {
namespace {

constexpr int kSel = 1024;   // threads of the selection
constexpr int kPer = 4;      // rows a thread an iteration of the last pass
constexpr int kBins = 2048;

// Bits that order like the weights: larger is heavier; NaN counts as -inf and
// -0 as 0.
__device__ __forceinline__ uint32_t order_bits(float w) {
  w = w != w ? -INFINITY : w + 0.0f;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sums x over the workgroup, exclusive, and the total. All threads call it.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* waves, uint64_t* total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  uint64_t incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  __syncthreads();  // the last call's sums are read
  if (lane == 63) waves[wave] = incl;
  __syncthreads();
  uint64_t base = 0, all = 0;
  for (int w = 0; w < kSel / 64; ++w) {
    const uint64_t y = waves[w];
    if (w < wave) base += y;
    all += y;
  }
  *total = all;
  return base + incl - x;
}

__global__ __launch_bounds__(kSel) void evict_select_kernel(const Pool p, int budget, int sinks,
                                                            int recent, int32_t* __restrict__ kept) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint64_t waves[kSel / 64];
  __shared__ uint32_t found[2];  // the digit, and the rows wanted within it
  const int unit = blockIdx.x, b = unit / p.Hkv, tid = threadIdx.x;
  const int n = held(p, b, p.cap);
  int32_t* out = kept + int64_t(unit) * budget;
  if (n <= budget) {
    for (int i = tid; i < budget; i += kSel) out[i] = i < n ? i : -1;
    return;
  }
  const float* w = p.weights + unit * p.wstride;
  const int lo = sinks, hi = n - recent;  // the rows that compete
  uint32_t room = uint32_t(budget - sinks - recent);
  // The threshold: the room-th heaviest of [lo, hi). With no room, above all.
  uint32_t prefix = 0xffffffffu, mask = 0;
  if (room > 0) {
    prefix = 0;
    const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
    for (int pass = 0; pass < 3; ++pass) {
      const int sh = shifts[pass], bins = 1 << widths[pass];
      for (int i = tid; i < bins; i += kSel) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSel) {
        const uint32_t u = order_bits(w[i]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> sh) & (bins - 1)], 1u);
      }
      __syncthreads();
      // Counts from the heaviest digit down: thread t takes the digits
      // bins - 1 - 2t and below it.
      const int d0 = bins - 1 - 2 * tid;
      const uint32_t c0 = d0 >= 0 ? hist[d0] : 0, c1 = d0 >= 1 ? hist[d0 - 1] : 0;
      uint64_t all;
      const uint32_t above = uint32_t(block_scan(c0 + c1, waves, &all));
      if (above < room && above + c0 >= room) {
        found[0] = uint32_t(d0);
        found[1] = room - above;
      } else if (above + c0 < room && above + c0 + c1 >= room) {
        found[0] = uint32_t(d0 - 1);
        found[1] = room - above - c0;
      }
      __syncthreads();
      prefix |= found[0] << sh;
      mask |= uint32_t(bins - 1) << sh;
      room = found[1];
      __syncthreads();
    }
  }
  // room: the rows of exactly the threshold's weight that stay.
  uint32_t sure0 = 0, ties0 = 0;  // before this iteration
  for (int base = 0; base < n; base += kSel * kPer) {
    const int i0 = base + tid * kPer;
    uint32_t kind[kPer], sure = 0, ties = 0;  // 2 stays, 1 ties, 0 goes
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = i0 + e;
      kind[e] = 0;
      if (i < n) {
        if (i < lo || i >= hi) {
          kind[e] = 2;
        } else if (mask) {
          const uint32_t u = order_bits(w[i]);
          kind[e] = u > prefix ? 2 : u == prefix ? 1 : 0;
        }
      }
      sure += kind[e] == 2;
      ties += kind[e] == 1;
    }
    uint64_t all;
    const uint64_t before = block_scan((uint64_t(sure) << 32) | ties, waves, &all);
    uint32_t s = sure0 + uint32_t(before >> 32), t = ties0 + uint32_t(before);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const uint32_t at = s + (t < room ? t : room);
      if (kind[e] == 2 || (kind[e] == 1 && t < room)) out[at] = i0 + e;
      s += kind[e] == 2;
      t += kind[e] == 1;
    }
    sure0 += uint32_t(all >> 32);
    ties0 += uint32_t(all);
  }
}

struct MoveArgs {
  Pool pool;
  const int32_t* kept;
  const int32_t* dst_table;
  int64_t dst_stride;
  int32_t* dst_lens;
  float* dst_weights;
  int budget;
  void* slot[6];
  int row_bytes[6];
  int n_slots;
};

constexpr int kThreads = 256;
constexpr int kRows = 64;  // kept rows a workgroup

__global__ __launch_bounds__(kThreads) void evict_move_kernel(const MoveArgs a) {
  __shared__ int64_t src[kRows], dst[kRows];
  const Pool& p = a.pool;
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int i0 = blockIdx.x * kRows, rmask = (1 << p.shift) - 1;
  const int64_t unit = int64_t(b) * p.Hkv + h;
  if (tid < kRows) {
    const int i = i0 + tid;
    const int r = i < a.budget ? a.kept[unit * a.budget + i] : -1;
    int64_t s = -1, d = -1;
    if (r >= 0) {
      const int ps = p.table[b * p.tstride + (r >> p.shift)];
      const int pd = a.dst_table[b * a.dst_stride + (i >> p.shift)];
      if (valid_page(p, ps) && valid_page(p, pd)) {
        s = pool_row(p, ps, h, r & rmask);
        d = pool_row(p, pd, h, i & rmask);
      }
      if (a.dst_weights)
        a.dst_weights[unit * (a.dst_stride << p.shift) + i] = p.weights[unit * p.wstride + r];
    }
    src[tid] = s;
    dst[tid] = d;
  }
  // The new length, by one thread that alone reads the old one (lens may be
  // dst_lens).
  if (blockIdx.x == 0 && h == 0 && tid == 0) {
    const int n = held(p, b, p.cap);
    a.dst_lens[b] = n < a.budget ? n : a.budget;
  }
  __syncthreads();
  for (int k = 0; k < a.n_slots; ++k) {
    const int bytes = a.row_bytes[k];
    char* buf = static_cast<char*>(a.slot[k]);
    if (bytes % 16 == 0) {
      const int per = bytes / 16;
      for (int i = tid; i < kRows * per; i += kThreads) {
        const int r = i / per, c = i % per;
        if (dst[r] >= 0)
          *reinterpret_cast<uint4*>(buf + dst[r] * bytes + c * 16) =
              *reinterpret_cast<const uint4*>(buf + src[r] * bytes + c * 16);
      }
    } else {
      const int per = bytes / 2;
      for (int i = tid; i < kRows * per; i += kThreads) {
        const int r = i / per, c = i % per;
        if (dst[r] >= 0)
          *reinterpret_cast<uint16_t*>(buf + dst[r] * bytes + c * 2) =
              *reinterpret_cast<const uint16_t*>(buf + src[r] * bytes + c * 2);
      }
    }
  }
}

}  // namespace
}  // namespace paged
}  // namespace tqkv

extern "C" size_t tqkv_paged_evict_workspace_size(const tqkv_paged_kv* kv, int64_t budget) {
  tqkv::paged::Pool p;
  if (tqkv::paged::check(kv, &p) != TQKV_OK || budget < 1 || budget > 0x7fffffffLL) return 0;
  return size_t(p.batch) * p.Hkv * size_t(budget) * sizeof(int32_t);
}

extern "C" int32_t tqkv_paged_evict(const tqkv_paged_kv* kv, int64_t budget, int64_t sinks,
                                    int64_t recent, const int32_t* dst_table, int64_t dst_stride,
                                    int32_t* dst_lens, float* dst_weights, int32_t* kept,
                                    void* workspace, size_t workspace_bytes, tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::paged;
  MoveArgs a{};
  if (int32_t rc = check(kv, &a.pool)) return rc;
  if (dst_stride < 1 || dst_stride > (int64_t(1) << 30) / kv->page_rows || budget < 1 || sinks < 0 ||
      recent < 0 || sinks > budget || recent > budget - sinks ||
      budget > dst_stride * kv->page_rows || budget > (int64_t(1) << 29))
    return fail(TQKV_EINVAL_SHAPE, "budget=%lld sinks=%lld recent=%lld of %lld new pages a sequence",
                (long long)budget, (long long)sinks, (long long)recent, (long long)dst_stride);
  if (!kv->weights || !dst_table || !dst_lens) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (dst_weights == kv->weights) return fail(TQKV_EINVAL_ARG, "dst_weights is the pool's weights");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const size_t need = tqkv_paged_evict_workspace_size(kv, budget);
  if (!kept) {
    if (!workspace) {
      if (int32_t rc = scratch_for_current_device(need, &workspace)) return rc;
    } else if (workspace_bytes < need || !aligned(workspace, 4)) {
      return fail(TQKV_EINVAL_ARG, "workspace of %zu bytes, need %zu", workspace_bytes, need);
    }
    kept = static_cast<int32_t*>(workspace);
  }
  hipLaunchKernelGGL(evict_select_kernel, dim3(unsigned(kv->batch) * unsigned(kv->kv_heads)),
                     dim3(kSel), 0, st, a.pool, int(budget), int(sinks), int(recent), kept);
  TQKV_LAUNCHED();
  a.kept = kept;
  a.dst_table = dst_table;
  a.dst_stride = dst_stride;
  a.dst_lens = dst_lens;
  a.dst_weights = dst_weights;
  a.budget = int(budget);
  const int D = kv->dim;
  if (kv->kind == TQKV_CACHE_BF16) {
    a.n_slots = 2;
    a.row_bytes[0] = a.row_bytes[1] = 2 * D;
  } else {
    a.n_slots = 6;
    for (int s = 0; s < 2; ++s) {
      a.row_bytes[3 * s] = D * (s ? kv->bits_v : kv->bits_k) / 8;
      a.row_bytes[3 * s + 1] = a.row_bytes[3 * s + 2] = D / kv->group_size * 2;
    }
  }
  for (int i = 0; i < a.n_slots; ++i) a.slot[i] = kv->slot[i];
  hipLaunchKernelGGL(evict_move_kernel,
                     dim3(unsigned((budget + kRows - 1) / kRows), unsigned(kv->kv_heads),
                          unsigned(kv->batch)),
                     dim3(kThreads), 0, st, a);
  TQKV_LAUNCHED();
  return ok();
}

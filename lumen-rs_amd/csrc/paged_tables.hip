// Paged cache: pages given to sequences and taken back, on the device.
//
// Reserve: with n rows held and a more asked, a sequence needs
// ceil((n + a) / R) - ceil(n / R) pages. One scan over the batch (at most
// 1,024 sequences) of what is asked decides who is served, a second one of what is
// granted places tokens and pages; every token then finds its sequence by a
// search in LDS. Bound by a launch's time for a decode step, and for prompts
// by the 16 bytes a token that the slots take.
// Release: the same scan over the pages that come back; one workgroup walks
// them in order, since entries that name no page are left out of the stack
// (8 entries a thread at a time, a wavefront's side by side).
//
// 256 sequences of up to 6,000 rows and one token each: a reserve and a release
// 17.5 us by the host's clock with the copy of the state that the case restores;
// 24 sequences, most of them ending, 40,000 tokens: 21.4.
#include "paged.hpp"

namespace tqkv {
namespace paged {
namespace {

struct Tables {
  int32_t* table;
  int32_t* lens;
  int32_t* free_pages;
  int32_t* free_count;
  int64_t tstride;
  int num_pages, batch, shift, cap;
};

__device__ __forceinline__ int clamp_to(int x, int most) { return x < 0 ? 0 : x < most ? x : most; }
__device__ __forceinline__ int pages_of(int64_t rows, int shift) {
  return int((rows + (1 << shift) - 1) >> shift);
}

// Sums that stop at 2^32 - 1 (wrong tables and counts can ask for more).
__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// Inclusive sums over the wavefront: within rows of 16 lanes, then across.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = plus(x, __builtin_amdgcn_update_dpp(0, int(x), 0x111, 0xf, 0xf, true));  // row_shr 1, 2, 4, 8
  x = plus(x, __builtin_amdgcn_update_dpp(0, int(x), 0x112, 0xf, 0xf, true));
  x = plus(x, __builtin_amdgcn_update_dpp(0, int(x), 0x114, 0xf, 0xf, true));
  x = plus(x, __builtin_amdgcn_update_dpp(0, int(x), 0x118, 0xf, 0xf, true));
  x = plus(x, __builtin_amdgcn_update_dpp(0, int(x), 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
  x = plus(x, __builtin_amdgcn_update_dpp(0, int(x), 0x143, 0xc, 0xf, false));
  return x;
}

// Sums of x and y over the threads before this one, and over all.
struct Sums {
  uint32_t x, y, all_x, all_y;
};
template <int Threads>
__device__ __forceinline__ Sums block_scan(uint32_t x, uint32_t y) {
  __shared__ uint2 sums[Threads / 64];
  const int wave = threadIdx.x / 64;
  const uint32_t u = wave_scan(x), v = wave_scan(y);
  __syncthreads();
  if (threadIdx.x % 64 == 63) sums[wave] = make_uint2(u, v);
  __syncthreads();
  // The lanes before: shifted, since a sum that stopped cannot be taken back.
  Sums s{uint32_t(__shfl_up(int(u), 1, 64)), uint32_t(__shfl_up(int(v), 1, 64)), 0, 0};
  if (threadIdx.x % 64 == 0) s.x = s.y = 0;
  uint32_t before_x = 0, before_y = 0;
#pragma unroll
  for (int w = 0; w < Threads / 64; ++w) {
    const uint2 t = sums[w];
    if (w == wave) before_x = s.all_x, before_y = s.all_y;
    s.all_x = plus(s.all_x, t.x);
    s.all_y = plus(s.all_y, t.y);
  }
  s.x = plus(s.x, before_x);
  s.y = plus(s.y, before_y);
  return s;
}

// The last of s[0, n] (ascending) that is not above i: s[b] <= i < s[b + 1].
__device__ __forceinline__ int find(const int32_t* s, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (i >= s[mid]) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct ReserveArgs {
  Tables t;
  const int32_t* counts;
  int32_t* starts;
  int32_t* granted;
  int4* slots;
  int tokens;
};

// Fill: tokens' slots and the new table entries; Finish: lengths, the stack's
// height, starts and granted, which other workgroups' decisions read. One
// workgroup does both; with many tokens a grid fills and a second launch of
// one workgroup finishes.
template <int Threads, bool Fill, bool Finish>
__global__ __launch_bounds__(Threads) void reserve_kernel(const ReserveArgs a) {
  constexpr int kPer = kMaxBatch / Threads;
  __shared__ int32_t start[kMaxBatch + 1], base[kMaxBatch + 1], rows[kMaxBatch];
  const Tables& t = a.t;
  const int avail = clamp_to(*t.free_count, t.num_pages);
  // Consecutive sequences a thread.
  int n[kPer], want[kPer], need[kPer];
  uint32_t pages = 0, places = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    n[i] = b < t.batch ? clamp_to(t.lens[b], t.cap) : 0;
    want[i] = b < t.batch ? max(a.counts[b], 0) : 0;
    const bool fits = int64_t(n[i]) + want[i] <= t.cap;
    need[i] = fits ? pages_of(int64_t(n[i]) + want[i], t.shift) - pages_of(n[i], t.shift) : -1;
    pages = plus(pages, fits ? need[i] : 0);
    places = plus(places, fits ? want[i] : 0);
  }
  Sums sum = block_scan<Threads>(pages, places);
  int got[kPer], take[kPer];
  uint32_t gots = 0, takes = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool fits = need[i] >= 0;
    sum.x = plus(sum.x, fits ? need[i] : 0);
    sum.y = plus(sum.y, fits ? want[i] : 0);
    const bool ok = fits && (need[i] == 0 || sum.x <= uint32_t(avail)) &&
                    (want[i] == 0 || sum.y <= uint32_t(a.tokens));
    got[i] = ok ? want[i] : -1;
    take[i] = ok ? need[i] : 0;
    gots += ok ? want[i] : 0;
    takes += take[i];
  }
  sum = block_scan<Threads>(takes, gots);
  int first = int(sum.y), page = int(sum.x);
  const int taken = int(sum.all_x), total = int(sum.all_y), top = avail - taken;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    start[b] = first;
    base[b] = page;
    rows[b] = n[i];
    first += max(got[i], 0);
    page += take[i];
    if (Finish && b < t.batch) {
      a.starts[b] = start[b];
      if (a.granted) a.granted[b] = got[i];
      t.lens[b] = n[i] + max(got[i], 0);
    }
  }
  if (threadIdx.x == 0) {
    start[kMaxBatch] = total;
    base[kMaxBatch] = taken;
    if (Finish) {
      a.starts[t.batch] = total;
      *t.free_count = top;  // every thread has read the old one: block_scan's barriers
    }
  }
  if constexpr (!Fill) return;
  __syncthreads();
  const int grid = int(gridDim.x) * Threads;
  for (int64_t j = int64_t(blockIdx.x) * Threads + threadIdx.x; j < taken; j += grid) {
    const int b = find(base, kMaxBatch, int(j));
    t.table[b * t.tstride + pages_of(rows[b], t.shift) + j - base[b]] = t.free_pages[top + j];
  }
  if (!a.slots) return;
  for (int64_t i = int64_t(blockIdx.x) * Threads + threadIdx.x; i < a.tokens; i += grid) {
    int4 s = make_int4(-1, 0, -1, -1);
    if (i < total) {
      const int b = find(start, kMaxBatch, int(i));
      const int row = rows[b] + int(i) - start[b], held = pages_of(rows[b], t.shift);
      const int p = row >> t.shift;
      // Pages taken are read from the stack: the table's entries may not be there yet.
      const int at = p < held ? t.table[b * t.tstride + p] : t.free_pages[top + base[b] + p - held];
      s = make_int4(at >= 0 && at < t.num_pages ? at : -1, row & ((1 << t.shift) - 1), row, b);
    }
    a.slots[i] = s;
  }
}

constexpr int kWalk = 1024, kEach = 8;

__global__ __launch_bounds__(kWalk) void release_kernel(const Tables t, const int32_t* keep,
                                                         const int32_t* shared) {
  __shared__ int32_t base[kMaxBatch + 1], from[kMaxBatch];
  __shared__ int32_t valid[kWalk / 64];
  const int b = threadIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int count = 0;
  const int height = clamp_to(*t.free_count, t.num_pages);
  if (b < t.batch) {
    const int n = clamp_to(t.lens[b], t.cap), k = clamp_to(keep[b], n);
    int lo = pages_of(k, t.shift);
    if (shared && shared[b] > lo) lo = shared[b];
    from[b] = lo;
    count = max(0, pages_of(n, t.shift) - lo);
    t.lens[b] = k;
  }
  const Sums sum = block_scan<kWalk>(count, 0);
  // A walk past 2^31 entries, which only wrong tables can ask for, is cut there.
  base[b] = int(min(sum.x, 0x7fffffffu));
  const int total = int(min(sum.all_x, 0x7fffffffu));
  if (threadIdx.x == 0) base[kMaxBatch] = total;
  __syncthreads();
  int64_t pushed = height;
  for (int64_t j0 = 0; j0 < total; j0 += kWalk * kEach) {
    // A wavefront's entries lie side by side.
    int page[kEach], s = -1;
    int64_t place[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t j = j0 + (wave * kEach + i) * 64 + lane;
      page[i] = -1;
      place[i] = -1;
      if (j < total) {
        if (s < 0 || j >= base[s + 1]) s = find(base, kMaxBatch, int(j));
        place[i] = s * t.tstride + from[s] + (j - base[s]);
        page[i] = t.table[place[i]];
      }
    }
    int mine = 0, at[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const unsigned long long mask = __ballot(page[i] >= 0 && page[i] < t.num_pages);
      at[i] = mine + __popcll(mask & ((1ull << lane) - 1));
      mine += __popcll(mask);
    }
    if (lane == 0) valid[wave] = mine;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWalk / 64; ++w) {
      if (w == wave) before = all;
      all += valid[w];
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (place[i] >= 0) t.table[place[i]] = -1;
      const int64_t to = pushed + before + at[i];
      if (page[i] >= 0 && page[i] < t.num_pages && to < t.num_pages) t.free_pages[to] = page[i];
    }
    pushed += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *t.free_count = int(pushed < t.num_pages ? pushed : t.num_pages);
}

int32_t check_tables(const tqkv_page_tables* p, Tables* out) {
  if (!p) return fail(TQKV_EINVAL_ARG, "null pointer");
  const int R = p->page_rows;
  if (p->batch < 1 || p->num_pages < 1 || p->table_stride < 1)
    return fail(TQKV_EINVAL_SHAPE, "batch=%d num_pages=%lld table_stride=%lld", p->batch,
                (long long)p->num_pages, (long long)p->table_stride);
  if (p->batch > kMaxBatch || !(R == 16 || R == 32 || R == 64 || R == 128 || R == 256))
    return fail(TQKV_EUNSUPPORTED, "batch=%d (at most %d) page_rows=%d", p->batch, kMaxBatch, R);
  if (p->num_pages > 0x7fffffffLL || p->table_stride > (int64_t(1) << 30) / R)
    return fail(TQKV_EINVAL_SHAPE, "num_pages=%lld table_stride=%lld page_rows=%d",
                (long long)p->num_pages, (long long)p->table_stride, R);
  if (!p->table || !p->lens || !p->free_pages || !p->free_count)
    return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!aligned(p->table, 4) || !aligned(p->lens, 4) || !aligned(p->free_pages, 4) ||
      !aligned(p->free_count, 4))
    return fail(TQKV_EINVAL_ARG, "table, lens, free_pages or free_count not 4-byte aligned");
  int shift = 4;
  while ((1 << shift) < R) ++shift;
  *out = Tables{p->table,         p->lens,  p->free_pages, p->free_count,
                p->table_stride, int(p->num_pages), p->batch, shift,
                int(p->table_stride * R)};
  return TQKV_OK;
}

}  // namespace
}  // namespace paged
}  // namespace tqkv

extern "C" int32_t tqkv_paged_reserve(const tqkv_page_tables* tables, const int32_t* counts,
                                      int64_t tokens, int32_t* starts, int32_t* granted,
                                      int32_t* slots, tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::paged;
  ReserveArgs a{};
  if (int32_t rc = check_tables(tables, &a.t)) return rc;
  if (tokens < 0 || tokens > 0x7fffffffLL)
    return fail(TQKV_EINVAL_SHAPE, "tokens=%lld", (long long)tokens);
  if (!counts || !starts) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!aligned(counts, 4) || !aligned(starts, 4) || !aligned(granted, 4) || !aligned(slots, 16))
    return fail(TQKV_EINVAL_ARG, "counts, starts or granted not 4-byte aligned, or slots not 16-byte");
  a.counts = counts;
  a.starts = starts;
  a.granted = granted;
  a.slots = reinterpret_cast<int4*>(slots);
  a.tokens = int(tokens);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // One workgroup fills 1,024 slots at a time, each with two searches and two reads
  // one after the other: from there on a second launch (2.6 us of the kernels' time)
  // is less than it.
  if (tokens < 1024) {
    hipLaunchKernelGGL((reserve_kernel<1024, true, true>), dim3(1), dim3(1024), 0, st, a);
    TQKV_LAUNCHED();
    return ok();
  }
  const int64_t blocks = (tokens + 255) / 256;
  hipLaunchKernelGGL((reserve_kernel<256, true, false>), dim3(unsigned(blocks < 2048 ? blocks : 2048)),
                     dim3(256), 0, st, a);
  TQKV_LAUNCHED();
  hipLaunchKernelGGL((reserve_kernel<1024, false, true>), dim3(1), dim3(1024), 0, st, a);
  TQKV_LAUNCHED();
  return ok();
}

extern "C" int32_t tqkv_paged_release(const tqkv_page_tables* tables, const int32_t* keep,
                                      const int32_t* shared, tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::paged;
  Tables t;
  if (int32_t rc = check_tables(tables, &t)) return rc;
  if (!keep) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!aligned(keep, 4) || !aligned(shared, 4))
    return fail(TQKV_EINVAL_ARG, "keep or shared not 4-byte aligned");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kWalk), 0, st, t, keep, shared);
  TQKV_LAUNCHED();
  return ok();
}

// Paged cache: eviction by gathered attention weight.
//
// Two launches. (1) One workgroup per (sequence, KV head) finds the weight of
// the last row that still fits: a radix select over the weights' bits, 11, 11
// and 10 a pass, histograms in LDS. Then it goes over the rows in their order
// and writes the kept positions, ascending: heavier rows all, rows of exactly
// that weight while there is room. The rows that stay anyhow (the first
// `sinks`, the last `recent`) take part as the heaviest of all. Up to 32,768
// rows stay in registers between the passes; more are read again, from the
// caches. Bound by one CU's vector units (every operation a row costs 16
// cycles a 1,024 rows) and the passes' barriers: 13 us for 16,384 rows to 2,048
// (8 workgroups), 16 for 16 sequences of up to 30,000 to 4,096 (128); the third
// pass, which most selections do not need, took 2. (2) The gather moves the rows
// to their new pages, bound by HBM: 16 sequences cut to 4,096 rows x 8 heads of
// 4 bits 22 us (28 with four wavefronts a workgroup), where a row's 64 bytes
// come in lines of 128.
#include <cmath>

#include "paged.hpp"

namespace tqkv {
namespace paged {
namespace {

constexpr int kSel = 1024;        // threads of the selection
constexpr int kWaves = kSel / 64;
constexpr int kQuads = 8;         // quads of rows a thread holds
constexpr int kChunk = kSel * 4 * kQuads;
constexpr int kBins = 2048;
constexpr int kCopies = 4;        // of the histogram, by lane: weights crowd few digits
constexpr int64_t kMostBudget = int64_t(1) << 29;

// Bits that order like the weights: larger is heavier; NaN counts as -inf and
// -0 as 0. Between 0x007fffff (-inf) and 0xff800000 (inf).
__device__ __forceinline__ uint32_t order_bits(float w) {
  w = w != w ? -INFINITY : w + 0.0f;
  const uint32_t u = __float_as_uint(w);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}

// Sums x over the workgroup, exclusive. All threads call it.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* waves) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  uint32_t incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  if (lane == 63) waves[wave] = incl;
  __syncthreads();
  uint32_t base = incl - x;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) base += w < wave ? waves[w] : 0;
  return base;
}

// A wavefront's rows of a chunk: quad k of lane l is the four rows from
// first + 256 k + 4 l.
struct Held {
  uint32_t u[4 * kQuads];
};
// Forced rows get all bits set, rows past the end none.
__device__ __forceinline__ void load_rows(Held& x, const float* w, int first, int quads, int n,
                                          int lo, int hi) {
  const int at = first + 4 * int(threadIdx.x % 64);
  float4 f[kQuads];
#pragma unroll
  for (int k = 0; k < kQuads; ++k) {
    f[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // A quad that starts before n ends within the weights: they are whole pages.
    if (k < quads && at + 256 * k < n) f[k] = *reinterpret_cast<const float4*>(w + at + 256 * k);
  }
#pragma unroll
  for (int k = 0; k < kQuads; ++k) {
    const float y[4] = {f[k].x, f[k].y, f[k].z, f[k].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = at + 256 * k + e;
      uint32_t u = order_bits(y[e]);
      u = i < lo || i >= hi ? 0xffffffffu : u;
      x.u[4 * k + e] = k < quads && i < n ? u : 0;
    }
  }
}

// Writes the kept rows of a wavefront's part of a chunk, from out[at] on; ties
// (rows of bits `edge`) while fewer than `room` came before.
template <bool kTies>
__device__ __forceinline__ void write_rows(const Held& x, int first, int quads, uint32_t edge,
                                           uint32_t room, uint32_t at, uint32_t ties,
                                           int32_t* out) {
  const int i0 = first + 4 * int(threadIdx.x % 64);
#pragma unroll
  for (int k = 0; k < kQuads; ++k) {
    if (k >= quads) break;
    uint64_t stay[4], tie[4];
    uint32_t s = at, t = ties;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      stay[e] = __ballot(x.u[4 * k + e] > edge);
      s = __builtin_amdgcn_mbcnt_hi(uint32_t(stay[e] >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(stay[e]), s));
      at += __popcll(stay[e]);
      if (kTies) {
        tie[e] = __ballot(x.u[4 * k + e] == edge);
        t = __builtin_amdgcn_mbcnt_hi(uint32_t(tie[e] >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(tie[e]), t));
        ties += __popcll(tie[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = x.u[4 * k + e];
      if (kTies) {
        if (u > edge || (u == edge && t < room)) out[s + (t < room ? t : room)] = i0 + 256 * k + e;
        t += u == edge;
      } else if (u > edge) {
        out[s] = i0 + 256 * k + e;
      }
      s += u > edge;
    }
  }
}

__global__ __launch_bounds__(kSel) void evict_select_kernel(const Pool p, int budget, int sinks,
                                                            int recent, int32_t* __restrict__ kept) {
  __shared__ uint32_t hist[kCopies][kBins + 1];
  __shared__ uint32_t waves[kWaves], counts[2][kWaves];
  __shared__ uint32_t found[3];  // the digit, the rows wanted within it, the rows it has
  const int unit = blockIdx.x, b = unit / p.Hkv, tid = threadIdx.x, lane = tid % 64;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int n = held(p, b, p.cap);
  int32_t* out = kept + int64_t(unit) * budget;
  if (n <= budget) {
    for (int i = tid; i < budget; i += kSel) out[i] = i < n ? i : -1;
    return;
  }
  const float* w = p.weights + unit * p.wstride;
  const int lo = sinks, hi = n - recent;  // the rows that compete
  // Quads a wavefront: the rows dealt evenly, or a chunk at a time.
  const bool one = n <= kChunk;
  const int quads = one ? (n + 256 * kWaves - 1) / (256 * kWaves) : kQuads;
  const int step = 256 * kWaves * quads, first = 256 * quads * wave;
  Held x;
  if (one) load_rows(x, w, first, quads, n, lo, hi);
  // The threshold: the budget-th heaviest.
  uint32_t edge = 0, mask = 0, room = uint32_t(budget), have = 0;
  for (int pass = 0; pass < 3; ++pass) {
    const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      hist[c][tid] = 0;
      hist[c][tid + kSel] = 0;
    }
    __syncthreads();
    for (int base = 0; base < n; base += step) {
      if (!one) load_rows(x, w, base + first, quads, n, lo, hi);
#pragma unroll
      for (int k = 0; k < kQuads; ++k) {
        if (k >= quads) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t u = x.u[4 * k + e];
          if ((u & mask) == edge) atomicAdd(&hist[tid % kCopies][(u >> sh) & (bins - 1)], 1u);
        }
      }
    }
    __syncthreads();
    // Counts from the heaviest digit down: thread t takes the digits
    // bins - 1 - 2t and below it.
    const int d0 = bins - 1 - 2 * tid;
    uint32_t c0 = 0, c1 = 0;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      c0 += d0 >= 0 ? hist[c][d0] : 0;
      c1 += d0 >= 1 ? hist[c][d0 - 1] : 0;
    }
    const uint32_t above = block_scan(c0 + c1, waves);
    if (above < room && above + c0 >= room) {
      found[0] = uint32_t(d0);
      found[1] = room - above;
      found[2] = c0;
    } else if (above + c0 < room && above + c0 + c1 >= room) {
      found[0] = uint32_t(d0 - 1);
      found[1] = room - above - c0;
      found[2] = c1;
    }
    __syncthreads();
    edge |= found[0] << sh;
    mask |= uint32_t(bins - 1) << sh;
    room = found[1];
    have = found[2];
    if (have == room) break;  // the digits below decide nothing
  }
  // Of the `have` rows at the edge, the first `room` stay. Where all do, they
  // count as above it (the edge is then the least of its digits, and not 0: the
  // lightest weight's bits are above).
  const bool ties = have > room;
  if (!ties) edge -= 1;
  uint32_t at = 0, tied = 0;  // before this chunk
  for (int base = 0; base < n; base += step) {
    if (!one) load_rows(x, w, base + first, quads, n, lo, hi);
    uint32_t s = 0, t = 0;
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      if (k >= quads) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s += __popcll(__ballot(x.u[4 * k + e] > edge));
        if (ties) t += __popcll(__ballot(x.u[4 * k + e] == edge));
      }
    }
    if (lane == 0) {
      counts[0][wave] = s;
      counts[1][wave] = t;
    }
    __syncthreads();
    uint32_t s0 = at, t0 = tied;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const uint32_t cs = counts[0][v], ct = counts[1][v];
      if (v < wave) {
        s0 += cs;
        t0 += ct;
      }
      at += cs;
      tied += ct;
    }
    if (ties)
      write_rows<true>(x, base + first, quads, edge, room, s0, t0, out);
    else
      write_rows<false>(x, base + first, quads, edge, 0, s0, 0, out);
    __syncthreads();
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
  int slots;  // buffers a side
  int rows;   // kept rows a workgroup: a power of two
  void* k[3];
  void* v[3];
  int k_shift[3], v_shift[3];  // log2 of a row's bytes: all are powers of two
};

typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));  // a 16-byte unit

int log2_of(int x) { return 31 - __builtin_clz(unsigned(x)); }

// A wavefront a workgroup, so that the most of them have their chains of loads
// (positions, pages, rows) going at once.
constexpr int kThreads = 64;
constexpr int kRows = 64;  // kept rows a workgroup at most, and threads that place them

// Rows of one buffer (2^ks units of type T each) and of another (2^vs), two
// loads of each in flight a thread. src is a row that can be read also where
// dst is -1.
template <typename T>
__device__ __forceinline__ void move_rows(T* kb, int ks, T* vb, int vs, const int64_t* src,
                                          const int64_t* dst, int rows) {
  const int items = rows << (ks > vs ? ks : vs);
  auto load = [&](const T* buf, int shift, int i) {
    return buf[(src[(i >> shift) & (rows - 1)] << shift) + (i & ((1 << shift) - 1))];
  };
  auto store = [&](T* buf, int shift, int i, T x) {
    const int r = i >> shift;
    if (r < rows && dst[r] >= 0) buf[(dst[r] << shift) + (i & ((1 << shift) - 1))] = x;
  };
  for (int i = threadIdx.x; i < items; i += 2 * kThreads) {
    const T x0 = load(kb, ks, i), x1 = load(kb, ks, i + kThreads);
    const T y0 = load(vb, vs, i), y1 = load(vb, vs, i + kThreads);
    store(kb, ks, i, x0);
    store(kb, ks, i + kThreads, x1);
    store(vb, vs, i, y0);
    store(vb, vs, i + kThreads, y1);
  }
}

__global__ __launch_bounds__(kThreads) void evict_move_kernel(const MoveArgs a) {
  __shared__ int64_t src[kRows], dst[kRows];
  const Pool& p = a.pool;
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int i0 = blockIdx.x * a.rows, rmask = (1 << p.shift) - 1;
  const int64_t unit = int64_t(b) * p.Hkv + h;
  if (tid < a.rows) {
    const int i = i0 + tid;
    const int r = i < a.budget ? a.kept[unit * a.budget + i] : -1;
    int64_t s = 0, d = -1;
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
  // Keys and values side by side, so that their loads are in flight together.
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (i >= a.slots) break;
    const int ks = a.k_shift[i], vs = a.v_shift[i];
    if (ks >= 4 && vs >= 4)
      move_rows(static_cast<uintx4*>(a.k[i]), ks - 4, static_cast<uintx4*>(a.v[i]), vs - 4, src, dst,
                a.rows);
    else if (ks >= 2)  // scales and biases: rows of one length
      move_rows(static_cast<uint32_t*>(a.k[i]), ks - 2, static_cast<uint32_t*>(a.v[i]), vs - 2, src,
                dst, a.rows);
    else
      move_rows(static_cast<uint16_t*>(a.k[i]), ks - 1, static_cast<uint16_t*>(a.v[i]), vs - 1, src,
                dst, a.rows);
  }
}

}  // namespace
}  // namespace paged
}  // namespace tqkv

extern "C" size_t tqkv_paged_evict_workspace_size(const tqkv_paged_kv* kv, int64_t budget) {
  using namespace tqkv::paged;
  Pool p;
  if (check(kv, &p) != TQKV_OK || budget < 1 || budget > kMostBudget) return 0;
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
      budget > dst_stride * kv->page_rows || budget > kMostBudget)
    return fail(TQKV_EINVAL_SHAPE, "budget=%lld sinks=%lld recent=%lld of %lld new pages a sequence",
                (long long)budget, (long long)sinks, (long long)recent, (long long)dst_stride);
  if (!kv->weights || !dst_table || !dst_lens) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!aligned(dst_table, 4) || !aligned(dst_lens, 4) || !aligned(dst_weights, 4) ||
      !aligned(kept, 4))
    return fail(TQKV_EINVAL_ARG, "dst_table, dst_lens, dst_weights or kept not 4-byte aligned");
  // Rows move while others' weights are still read.
  const uintptr_t old_at = reinterpret_cast<uintptr_t>(kv->weights), new_at = reinterpret_cast<uintptr_t>(dst_weights);
  const uint64_t units = uint64_t(kv->batch) * uint64_t(kv->kv_heads) * sizeof(float);
  if (dst_weights && new_at < old_at + units * uint64_t(a.pool.wstride) &&
      old_at < new_at + units * uint64_t(dst_stride * kv->page_rows))
    return fail(TQKV_EINVAL_ARG, "dst_weights overlaps the pool's weights");
  const int D = kv->dim;
  a.slots = kv->kind == TQKV_CACHE_BF16 ? 1 : 3;
  for (int i = 0; i < a.slots; ++i) {
    a.k[i] = kv->slot[i];
    a.v[i] = kv->slot[a.slots + i];
    const int scales = 2 * D / (i > 0 ? kv->group_size : 1);  // bf16 rows also
    a.k_shift[i] = log2_of(i > 0 || a.slots == 1 ? scales : D * kv->bits_k / 8);
    a.v_shift[i] = log2_of(i > 0 || a.slots == 1 ? scales : D * kv->bits_v / 8);
  }
  // Two 16-byte pieces of the wider rows a thread (2,048 bf16 rows x 8 heads and
  // a batch's 4-bit rows: 5.0 and 23.2 us; four 5.7 and 24.6, eight 5.9 and 24.1).
  const int wide = a.k_shift[0] > a.v_shift[0] ? a.k_shift[0] : a.v_shift[0];
  a.rows = 2 * kThreads >> (wide - 4);
  if (a.rows > kRows) a.rows = kRows;
  const int64_t blocks = (budget + a.rows - 1) / a.rows;
  if (blocks > 0xffffffffLL / kThreads)  // a grid: below 2^32 threads
    return fail(TQKV_EUNSUPPORTED, "budget=%lld", (long long)budget);
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
  hipLaunchKernelGGL(evict_move_kernel,
                     dim3(unsigned(blocks), unsigned(kv->kv_heads), unsigned(kv->batch)),
                     dim3(kThreads), 0, st, a);
  TQKV_LAUNCHED();
  return ok();
}

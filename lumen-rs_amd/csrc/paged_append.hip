// Paged cache: the checks of a pool, and the append.
//
// Append: row lens[b] - count[b] + j of sequence b takes token starts[b] + j.
// Each workgroup finds the destinations of its tokens once (a search of
// `starts` in LDS, then the table), then moves rows. Bound by HBM: 4 D bytes
// read a (token, KV head) and the stored row written.
// Measured at D = 128, 8 heads: 12 bf16 prompts of up to 4,096 tokens, 158 MB,
// 33 us (4.8 TB/s, a large copy's rate); 13,548 tokens into 4 bits, 71 MB, 24
// us (the quantizer's operations). A decode step's 64 tokens take 3.7 us, a
// launch's time.
#include "affine_quantize.hpp"
#include "paged.hpp"

namespace tqkv {
namespace paged {

int32_t check(const tqkv_paged_kv* kv, Pool* out) {
  if (!kv) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (kv->kind != TQKV_CACHE_BF16 && kv->kind != TQKV_CACHE_AFFINE)
    return fail(TQKV_EUNSUPPORTED, "paged cache of kind %d", kv->kind);
  if (kv->batch < 1 || kv->kv_heads < 1 || kv->num_pages < 1 || kv->table_stride < 1)
    return fail(TQKV_EINVAL_SHAPE, "batch=%d kv_heads=%d num_pages=%lld table_stride=%lld",
                kv->batch, kv->kv_heads, (long long)kv->num_pages, (long long)kv->table_stride);
  if (kv->batch > kMaxBatch || kv->kv_heads > 1024)
    return fail(TQKV_EUNSUPPORTED, "batch=%d (at most %d) kv_heads=%d (at most 1024)", kv->batch,
                kMaxBatch, kv->kv_heads);
  const int D = kv->dim, R = kv->page_rows;
  if (!(D == 64 || D == 128 || D == 256 || D == 512) ||
      !(R == 16 || R == 32 || R == 64 || R == 128 || R == 256))
    return fail(TQKV_EUNSUPPORTED, "dim=%d page_rows=%d", D, R);
  // Page numbers are 32-bit in the kernels, and row numbers with room for a
  // tile past the end.
  if (kv->num_pages > 0x7fffffffLL || kv->table_stride > (int64_t(1) << 30) / R)
    return fail(TQKV_EINVAL_SHAPE, "num_pages=%lld table_stride=%lld page_rows=%d",
                (long long)kv->num_pages, (long long)kv->table_stride, R);
  const bool affine = kv->kind == TQKV_CACHE_AFFINE;
  if (affine) {
    const int gs = kv->group_size;
    if (!(gs == 32 || gs == 64 || gs == 128) || D % gs != 0)
      return fail(TQKV_EUNSUPPORTED, "dim=%d group_size=%d", D, gs);
    if (!(kv->bits_k == 4 || kv->bits_k == 8) || !(kv->bits_v == 4 || kv->bits_v == 8))
      return fail(TQKV_EUNSUPPORTED, "bits_k=%d bits_v=%d", kv->bits_k, kv->bits_v);
  }
  if (!kv->table || !kv->lens) return fail(TQKV_EINVAL_ARG, "null pointer");
  for (int i = 0; i < (affine ? 6 : 2); ++i)
    if (!kv->slot[i] || !aligned(kv->slot[i], 16))
      return fail(TQKV_EINVAL_ARG, "slot %d is null or not 16-byte aligned", i);
  if (!aligned(kv->table, 4) || !aligned(kv->lens, 4) || !aligned(kv->weights, 16))
    return fail(TQKV_EINVAL_ARG, "table or lens not 4-byte aligned, or weights not 16-byte");
  int shift = 4;
  while ((1 << shift) < R) ++shift;
  *out = Pool{kv->table,   kv->lens,        kv->weights,
              kv->table_stride, kv->table_stride * R, kv->num_pages,
              kv->batch,   kv->kv_heads,    shift,
              int(kv->table_stride * R)};
  return TQKV_OK;
}

namespace {

constexpr int kThreads = 256;

// Where a token's rows go: the page's first pool row of head 0 plus the row
// in the page (head h adds h << shift), and its place in the weights.
struct Dest {
  int64_t row;  // -1: not written
  int64_t weight;
};

// Destination of token i. starts: LDS copy of batch + 1 starts, or NULL.
__device__ __forceinline__ Dest dest_of(const Pool& p, const int32_t* starts, int64_t i) {
  int b = int(i), count = 1, j = 0;
  if (starts) {
    if (i < starts[0] || i >= starts[p.batch]) return {-1, 0};
    int lo = 0, hi = p.batch;  // starts[lo] <= i < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (i >= starts[mid]) lo = mid;
      else hi = mid;
    }
    b = lo;
    count = starts[b + 1] - starts[b];
    j = int(i) - starts[b];
  }
  const int64_t row = int64_t(p.lens[b]) - count + j;
  if (row < 0 || row >= p.cap) return {-1, 0};
  const int page = p.table[b * p.tstride + (row >> p.shift)];
  if (!valid_page(p, page)) return {-1, 0};
  return {pool_row(p, page, 0, int(row) & ((1 << p.shift) - 1)), int64_t(b) * p.Hkv * p.wstride + row};
}

// The destinations of tokens [t0, t0 + n) into LDS. All threads call it.
__device__ __forceinline__ void find_dests(const Pool& p, const int32_t* starts, int64_t t0, int n,
                                           int32_t* sstarts, Dest* dest) {
  if (starts) {
    for (int b = threadIdx.x; b <= p.batch; b += kThreads) sstarts[b] = starts[b];
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kThreads)
    dest[i] = dest_of(p, starts ? sstarts : nullptr, t0 + i);
  __syncthreads();
}

struct AppendArgs {
  Pool pool;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* starts;
  int64_t tokens, ts, hs;
  void* slot[6];
  int gs;
};

// Zeroes the written rows' weights: token x head items of the workgroup.
__device__ __forceinline__ void clear_weights(const Pool& p, const Dest* dest, int n) {
  if (!p.weights) return;
  for (int i = threadIdx.x; i < n * p.Hkv; i += kThreads) {
    const int t = i / p.Hkv, h = i % p.Hkv;
    if (dest[t].row >= 0) p.weights[dest[t].weight + h * p.wstride] = 0.0f;
  }
}

// bf16 rows: a thread moves 16 bytes of K and of V; a row is D / 8 threads.
// kTokens tokens a workgroup.
constexpr int kTokens = 4;
// Quantized prompts: a workgroup's rows of a head lie side by side in a page
// (13,548 tokens of 8 heads, 4 bits: 27 us at 4 tokens a workgroup, 24 at 8,
// 25 at 16, 28 at 32); few tokens keep the smaller workgroups, for latency. With
// 4 and 8 tokens a workgroup, D = 128, 8 heads: 1,024 tokens 4.6 and 5.1 us, 2,048
// 5.9 and 6.0, 4,096 11.2 and 10.0. The line lies lower for shorter rows (D = 64:
// 2,048 tokens 5.3 and 4.5) and higher for longer ones (D = 256: 4,096 15.7 and
// 15.9).
constexpr int kMany = 8, kManyTokens = 2048;

template <int D>
__global__ __launch_bounds__(kThreads) void append_bf16_kernel(const AppendArgs a) {
  __shared__ int32_t sstarts[kMaxBatch + 1];
  __shared__ Dest dest[kTokens];
  const Pool& p = a.pool;
  const int64_t t0 = int64_t(blockIdx.x) * kTokens;
  const int n = a.tokens - t0 < kTokens ? int(a.tokens - t0) : kTokens;
  constexpr int LPR = D / 8;
  const int c = threadIdx.x % LPR;
  // Rows are heads within tokens: a token's heads lie side by side where they
  // are read.
  auto source = [&](int row) {
    row = row < n * p.Hkv ? row : n * p.Hkv - 1;
    return (t0 + row / p.Hkv) * a.ts + (row % p.Hkv) * a.hs + c * 8;
  };
  // The first rows are on their way while their places are found.
  const int64_t first = source(threadIdx.x / LPR);
  uint4 x = *reinterpret_cast<const uint4*>(a.k + first);
  uint4 y = *reinterpret_cast<const uint4*>(a.v + first);
  find_dests(p, a.starts, t0, n, sstarts, dest);
  for (int r = threadIdx.x / LPR; r < n * p.Hkv; r += kThreads / LPR) {
    const int t = r / p.Hkv, h = r % p.Hkv;
    const uint4 xs = x, ys = y;
    if (r + kThreads / LPR < n * p.Hkv) {
      const int64_t next = source(r + kThreads / LPR);
      x = *reinterpret_cast<const uint4*>(a.k + next);
      y = *reinterpret_cast<const uint4*>(a.v + next);
    }
    if (dest[t].row < 0) continue;
    const int64_t dst = (dest[t].row + (int64_t(h) << p.shift)) * D + c * 8;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.slot[0]) + dst) = xs;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.slot[1]) + dst) = ys;
  }
  clear_weights(p, dest, n);
}

// Affine rows: a lane quantizes 16 elements (the bits of
// tqkv_affine_quantize), whose 4- or 8-bit codes are whole words, so they are
// stored from registers. blockIdx.y: K or V.
template <int D, int BK, int BV, int kTokens>
__global__ __launch_bounds__(kThreads) void append_affine_kernel(const AppendArgs a) {
  __shared__ int32_t sstarts[kMaxBatch + 1];
  __shared__ Dest dest[kTokens];
  const Pool& p = a.pool;
  const int64_t t0 = int64_t(blockIdx.x) * kTokens;
  const int n = a.tokens - t0 < kTokens ? int(a.tokens - t0) : kTokens;
  constexpr int LPR = D / aq::kLaneElems;
  const int side = blockIdx.y, bits = side ? BV : BK;
  const uint16_t* x = side ? a.v : a.k;
  uint32_t* packed = static_cast<uint32_t*>(a.slot[3 * side]);
  uint16_t* scales = static_cast<uint16_t*>(a.slot[3 * side + 1]);
  uint16_t* biases = static_cast<uint16_t*>(a.slot[3 * side + 2]);
  const int lpg = a.gs / aq::kLaneElems, groups = D / a.gs;
  // Lane c of a row; rows are tokens within heads, so that a wavefront's rows
  // lie side by side in a page.
  const int c = threadIdx.x % LPR, rows = p.Hkv * kTokens;
  auto load = [&](int row, float (&v)[aq::kLaneElems]) {
    // Whole wavefronts go round (the groups' butterflies exchange across
    // lanes): rows past the end load the last ones and are not stored.
    row = row < rows ? row : rows - 1;
    const int t = row % kTokens < n ? row % kTokens : n - 1;
    aq::load_lane(x + (t0 + t) * a.ts + (row / kTokens) * a.hs + c * aq::kLaneElems, v);
  };
  // The first rows are on their way while their places are found.
  float v[aq::kLaneElems];
  load(threadIdx.x / LPR, v);
  find_dests(p, a.starts, t0, n, sstarts, dest);
  for (int row0 = 0; row0 < rows; row0 += kThreads / LPR) {
    const int r = row0 + threadIdx.x / LPR, t = r % kTokens, h = r / kTokens;
    const aq::LaneCodes q = aq::quantize_lane_refined(v, a.gs, bits);
    if (row0 + kThreads / LPR < rows) load(r + kThreads / LPR, v);
    if (r >= rows || t >= n || dest[t].row < 0) continue;
    const int64_t row = dest[t].row + (int64_t(h) << p.shift);
    uint32_t* out = packed + row * (D * bits / 32) + c * (bits / 2);
    if (bits == 4)
      *reinterpret_cast<uint2*>(out) = make_uint2(uint32_t(q.chunk[0]), uint32_t(q.chunk[1]));
    else
      *reinterpret_cast<uint4*>(out) = make_uint4(uint32_t(q.chunk[0]), uint32_t(q.chunk[0] >> 32),
                                                  uint32_t(q.chunk[1]), uint32_t(q.chunk[1] >> 32));
    if (c % lpg == 0) {
      scales[row * groups + c / lpg] = f32_to_bf16(q.scale);
      biases[row * groups + c / lpg] = f32_to_bf16(q.bias);
    }
  }
  if (side == 0) clear_weights(p, dest, n);
}

template <int D, int kTokens>
void launch_affine(const tqkv_paged_kv* kv, const AppendArgs& a, hipStream_t st) {
  const unsigned blocks = unsigned((a.tokens + kTokens - 1) / kTokens);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks, 2), dim3(kThreads), 0, st, a);
  };
  if (kv->bits_k == 4 && kv->bits_v == 4) go(append_affine_kernel<D, 4, 4, kTokens>);
  else if (kv->bits_k == 4) go(append_affine_kernel<D, 4, 8, kTokens>);
  else if (kv->bits_v == 4) go(append_affine_kernel<D, 8, 4, kTokens>);
  else go(append_affine_kernel<D, 8, 8, kTokens>);
}

template <int D>
void launch_append(const tqkv_paged_kv* kv, const AppendArgs& a, hipStream_t st) {
  if (kv->kind == TQKV_CACHE_BF16)
    hipLaunchKernelGGL(append_bf16_kernel<D>, dim3(unsigned((a.tokens + kTokens - 1) / kTokens)),
                       dim3(kThreads), 0, st, a);
  else if (a.tokens >= kManyTokens)
    launch_affine<D, kMany>(kv, a, st);
  else
    launch_affine<D, kTokens>(kv, a, st);
}

}  // namespace
}  // namespace paged
}  // namespace tqkv

extern "C" int32_t tqkv_paged_append(const tqkv_paged_kv* kv, const uint16_t* k, const uint16_t* v,
                                     const int32_t* starts, int64_t tokens, int64_t token_stride,
                                     int64_t head_stride, tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::paged;
  AppendArgs a{};
  if (int32_t rc = check(kv, &a.pool)) return rc;
  if (tokens < 0 || tokens > 0xffffffffLL / kThreads * kTokens)  // a grid: below 2^32 threads
    return fail(TQKV_EINVAL_SHAPE, "tokens=%lld", (long long)tokens);
  if (!starts && tokens != kv->batch)
    return fail(TQKV_EINVAL_SHAPE, "no starts: tokens=%lld, batch=%d", (long long)tokens, kv->batch);
  if (tokens == 0) return ok();
  if (!k || !v) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(starts, 4) || token_stride % 8 != 0 ||
      head_stride % 8 != 0)
    return fail(TQKV_EINVAL_ARG,
                "k and v are 16-byte aligned, strides multiples of 8 elements (token %lld, head %lld)",
                (long long)token_stride, (long long)head_stride);
  a.k = k;
  a.v = v;
  a.starts = starts;
  a.tokens = tokens;
  a.ts = token_stride;
  a.hs = head_stride;
  a.gs = kv->group_size;
  for (int i = 0; i < 6; ++i) a.slot[i] = kv->slot[i];
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (kv->dim) {
    case 64: launch_append<64>(kv, a, st); break;
    case 128: launch_append<128>(kv, a, st); break;
    case 256: launch_append<256>(kv, a, st); break;
    default: launch_append<512>(kv, a, st); break;
  }
  TQKV_LAUNCHED();
  return ok();
}

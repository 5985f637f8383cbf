// Paged decode attention: the join of the segments, the gathered weights, and
// the host side. The attention kernel is in paged_decode.hpp.
#include "paged_decode.hpp"

namespace tqkv {
namespace paged {

extern template int launch_affine<64>(const DecodeArgs&, int, int, int, dim3, hipStream_t, bool);
extern template int launch_affine<128>(const DecodeArgs&, int, int, int, dim3, hipStream_t, bool);
extern template int launch_affine<256>(const DecodeArgs&, int, int, int, dim3, hipStream_t, bool);
extern template int launch_affine<512>(const DecodeArgs&, int, int, int, dim3, hipStream_t, bool);

namespace {

constexpr int kJoinThreads = 256;
constexpr int kWeightRows = 4 * kJoinThreads;  // rows whose weights a workgroup adds
constexpr float kPartDown = 0x1p-40f;  // parts hold weights and their sums times it
static_assert(Bf16Rows<128>::kDown == 40, "as the parts are");
static_assert(AffineRows<128, 4, 4, 64>::kLast == 0x1p-47f && AffineRows<128, 4, 4, 64>::kDown == 40 - 47,
              "as the parts are");
constexpr int kMaxSegments = 1024;  // of one sequence: the workgroups of a KV head

// 2^(m_s - m) of every segment s of one (sequence, head) into LDS, and the sum
// of the segments' sums by those. All threads call it.
__device__ __forceinline__ float segment_weights(const DecodeArgs& a, int64_t slot0, int n, int h,
                                                 float* weight, float* red, float* top) {
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  float pm[kMaxSegments / kJoinThreads], pl[kMaxSegments / kJoinThreads], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxSegments / kJoinThreads; ++i) {
    const int s = tid + i * kJoinThreads;
    pm[i] = s < n ? a.part_m[(slot0 + s) * a.H + h] : -INFINITY;
    pl[i] = s < n ? a.part_l[(slot0 + s) * a.H + h] : 0.0f;
    m = fmaxf(m, pm[i]);
  }
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  __syncthreads();
  if (lane == 0) red[wave] = m;
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 64; ++w) m = fmaxf(m, red[w]);
  float l = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxSegments / kJoinThreads; ++i) {
    const int s = tid + i * kJoinThreads;
    const float w = pm[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[i] - m);
    if (s < n) weight[s] = w;
    l += w * pl[i];  // a NaN sum stays one
  }
  for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
  __syncthreads();
  if (lane == 0) red[wave] = l;
  __syncthreads();
  l = 0.0f;
  for (int w = 0; w < kJoinThreads / 64; ++w) l += red[w];
  *top = m;
  return l;
}

// Channels that a workgroup joins, a quad a thread, and the threads that the
// segments are dealt over.
template <int D>
struct JoinShape {
  static constexpr int kPart = D < 128 ? D : 128, kParts = D / kPart;
  static constexpr int kQuads = kPart / 4, kDeal = kJoinThreads / kQuads;
};
// Segments whose weights a wavefront holds, one a lane.
constexpr int kFew = 64;

// Workgroups [0, batch x H x parts): channels of the output of one (sequence,
// head) from its segments. The others: kWeightRows rows of one (sequence, KV
// head), weights[row] += sum over the group's heads of 2^(s - m) / l. Bound by
// a chain of loads: the starts, then all that depends on them at once.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(const DecodeArgs a,
                                                                  int row_blocks) {
  using J = JoinShape<D>;
  constexpr int kQuads = J::kQuads, kDeal = J::kDeal;
  __shared__ float red[kJoinThreads / 64], weight[kMaxSegments], head_m[32], head_r[32];
  __shared__ float4 sums[kJoinThreads];
  const int tid = threadIdx.x, lane = tid % 64, outs = a.pool.batch * a.H * J::kParts;
  const bool joins = int(blockIdx.x) < outs;
  int b, h = 0, kvh = 0, block = 0, part = 0;
  if (joins) {
    part = blockIdx.x % J::kParts;
    h = blockIdx.x / J::kParts % a.H;
    b = blockIdx.x / J::kParts / a.H;
  } else {
    const int i = blockIdx.x - outs;
    block = i % row_blocks;
    kvh = i / row_blocks % a.pool.Hkv;
    b = i / row_blocks / a.pool.Hkv;
  }
  const int first = a.starts[b], next = a.starts[b + 1], total = a.starts[a.pool.batch];
  const int per = units_per_wg(a, total);
  const int w0 = (first + a.over) / per, n = (next - 1) / per - w0 + 1;
  const int64_t slot0 = w0 + b;
  float m;
  if (joins) {
    const int quad = tid % kQuads, deal = tid / kQuads, d = part * J::kPart + 4 * quad;
    uint16_t* out = a.out + (int64_t(b) * a.H + h) * D + d;
    if (next == first) {  // no rows
      if (deal == 0)
        for (int i = 0; i < 4; ++i) out[i] = 0;
      return;
    }
    if (n == 1) return;  // written by the attention kernel
    const float* po = a.part_o + (slot0 * a.H + h) * D + d;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l;
    auto add = [&](float w, const float4& y) {
      o.x = fmaf(w, y.x, o.x);
      o.y = fmaf(w, y.y, o.y);
      o.z = fmaf(w, y.z, o.z);
      o.w = fmaf(w, y.w, o.w);
    };
    if (n <= kFew) {
      const int seg = lane < n ? lane : n - 1;
      const float pm = a.part_m[(slot0 + seg) * a.H + h], pl = a.part_l[(slot0 + seg) * a.H + h];
      float4 y[kFew / kDeal];
#pragma unroll
      for (int i = 0; i < kFew / kDeal; ++i) {
        const int s = deal + i * kDeal < n ? deal + i * kDeal : n - 1;
        y[i] = *reinterpret_cast<const float4*>(po + int64_t(s) * a.H * D);
      }
      m = pm;
      for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
      const float w = pm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm - m);
      l = lane < n ? w * pl : 0.0f;  // a NaN sum stays one
      for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
#pragma unroll
      for (int i = 0; i < kFew / kDeal; ++i) {
        const float ws = __shfl(w, deal + i * kDeal, 64);
        if (deal + i * kDeal < n) add(ws, y[i]);
      }
    } else {
      l = segment_weights(a, slot0, n, h, weight, red, &m);
#pragma unroll 8
      for (int s = deal; s < n; s += kDeal)
        add(weight[s], *reinterpret_cast<const float4*>(po + int64_t(s) * a.H * D));
    }
    sums[tid] = o;
    __syncthreads();
    if (deal == 0) {
#pragma unroll
      for (int i = 1; i < kDeal; ++i) {
        const float4 y = sums[i * kQuads + quad];
        o.x += y.x;
        o.y += y.y;
        o.z += y.z;
        o.w += y.w;
      }
      const float v[4] = {o.x / l, o.y / l, o.z / l, o.w / l};
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = f32_to_bf16(l == 0.0f ? 0.0f : v[i]);
    }
    return;
  }
  const Span span = span_of(a, b);
  const int row0 = span.lo / 4 * 4 + block * kWeightRows, row = row0 + 4 * tid;
  if (row0 >= span.n) return;
  float* weights = a.pool.weights + (int64_t(b) * a.pool.Hkv + kvh) * a.pool.wstride;
  const float* scores = a.scores + (int64_t(b) * a.H + kvh * a.G) * a.srows;
  // Four rows a thread; the scores of rows outside the span are -inf or unset.
  // The first heads' are on their way while the heads' sums are found; rows
  // past the end load the first ones.
  const int at = row < span.n ? row : row0;
  const float4 old = *reinterpret_cast<const float4*>(weights + at);
  constexpr int kAhead = 4;
  float4 x[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    x[i] = *reinterpret_cast<const float4*>(scores + (i < a.G ? i : 0) * a.srows + at);
  // A wavefront a head.
  for (int i = tid / 64; i < a.G; i += kJoinThreads / 64) {
    const int head = kvh * a.G + i;
    float top = -INFINITY, l = 0.0f;
    for (int s = lane; s < n; s += 64) {  // the running maximum and sum of the lane's segments
      const float pm = a.part_m[(slot0 + s) * a.H + head], pl = a.part_l[(slot0 + s) * a.H + head];
      const float next = fmaxf(top, pm);
      if (next > -INFINITY)
        l = l * __builtin_amdgcn_exp2f(top - next) + pl * __builtin_amdgcn_exp2f(pm - next);
      else
        l += pl;  // a NaN sum stays one
      top = next;
    }
    m = top;
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    l = top == -INFINITY ? 0.0f * l : l * __builtin_amdgcn_exp2f(top - m);
    for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
    if (lane == 0) {
      head_m[i] = m == -INFINITY ? 0.0f : m;
      head_r[i] = l == 0.0f ? 0.0f : kPartDown / l;
    }
  }
  __syncthreads();
  if (row >= span.n) return;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](const float4& y, int i) {
    const float hm = head_m[i], hr = head_r[i];
    sum[0] += __builtin_amdgcn_exp2f(y.x - hm) * hr;
    sum[1] += __builtin_amdgcn_exp2f(y.y - hm) * hr;
    sum[2] += __builtin_amdgcn_exp2f(y.z - hm) * hr;
    sum[3] += __builtin_amdgcn_exp2f(y.w - hm) * hr;
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (i < a.G) add(x[i], i);
#pragma unroll 4
  for (int i = kAhead; i < a.G; ++i)
    add(*reinterpret_cast<const float4*>(scores + i * a.srows + row), i);
  const float v[4] = {old.x + sum[0], old.y + sum[1], old.z + sum[2], old.w + sum[3]};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (row + e >= span.lo && row + e < span.n) weights[row + e] = v[e];
}

// The attention kernel of a layout, launched; or only its wavefronts a SIMD.
int launch(const tqkv_paged_kv* kv, const DecodeArgs& a, dim3 grid, hipStream_t st,
           bool occupancy) {
  if (kv->kind == TQKV_CACHE_BF16) {
    switch (kv->dim) {
      case 64: return launch_rows<Bf16Rows<64>>(a, grid, st, occupancy);
      case 128: return launch_rows<Bf16Rows<128>>(a, grid, st, occupancy);
      case 256: return launch_rows<Bf16Rows<256>>(a, grid, st, occupancy);
      default: return launch_rows<Bf16Rows<512>>(a, grid, st, occupancy);
    }
  }
  const int bk = kv->bits_k, bv = kv->bits_v, gs = kv->group_size;
  switch (kv->dim) {
    case 64: return launch_affine<64>(a, bk, bv, gs, grid, st, occupancy);
    case 128: return launch_affine<128>(a, bk, bv, gs, grid, st, occupancy);
    case 256: return launch_affine<256>(a, bk, bv, gs, grid, st, occupancy);
    default: return launch_affine<512>(a, bk, bv, gs, grid, st, occupancy);
  }
}

// Workgroups a CU: as many as fit at once for affine rows, whose loads leave
// little in flight (16 x 16,384 4-bit rows at D = 128: 94 us with one, 75 with
// two, 76 with three, 91 with six); one for bf16 rows, which fill the memory
// system with it (131,071 rows at D = 128: 90 us, 102 with two, 110 with
// three; 4 x 8,179 at D = 512: 35 and 45).
int workgroups_a_cu(const tqkv_paged_kv* kv) {
  if (kv->kind == TQKV_CACHE_BF16) return 1;
  return launch(kv, DecodeArgs{}, dim3(1), nullptr, true);
}

// Workgroups wanted over all KV heads: one round of them on 256 CUs.
constexpr int kCus = 256;
// Units that a sequence's start counts as: its segment's own latencies. 32
// sequences of 17 to 16,000 4-bit rows: 49 us at 0, 40 at 8, 36 at 16, 33 at
// 32; 16 of 17 to 8,192 bf16 rows: 26, 21, 19, 20; 8 windows of 1,024 8-bit
// rows: 16, 18, 18, 20.
constexpr int kOver = 16;
static_assert(4 * kCus <= kMaxSegments, "a join holds a sequence's segments");

constexpr int64_t kKeptBytes = int64_t(192) << 20;  // of the 256 MB memory-side cache

// Units a workgroup takes at least: a step of each of its wavefronts, of 32 rows,
// or 16 for wide ones (2 x 600 bf16 rows at D = 256: 9.7 us with 8 units, 8.4 with
// 4; 5 x 300 8- and 4-bit rows at D = 512: 18.5 and 17.8).
int least_units(const tqkv_paged_kv* kv) { return kv->dim <= 128 ? 8 : 4; }

struct HostPlan {
  int groups16, W, least;
  int64_t srows;
  size_t slots, bytes;
};

// Host plan of a call that check() accepted. False where H or max_rows is out
// of range.
bool plan_of(const tqkv_paged_kv* kv, int32_t H, int64_t max_rows, HostPlan* out) {
  if (H < 1 || H % kv->kv_heads != 0 || H / kv->kv_heads > 32 || max_rows < 1 ||
      max_rows > kv->table_stride * kv->page_rows)
    return false;
  HostPlan p;
  p.groups16 = (H / kv->kv_heads + 15) / 16;
  p.srows = (max_rows + kUnit - 1) / kUnit * kUnit;
  const int64_t units = int64_t(kv->kv_heads) * p.groups16;
  int64_t W = (workgroups_a_cu(kv) * kCus + units - 1) / units;
  // No more than the longest possible batch fills.
  const int64_t most = int64_t(kv->batch) * (p.srows / kUnit + kOver);
  p.least = least_units(kv);
  if (W > (most + p.least - 1) / p.least) W = (most + p.least - 1) / p.least;
  p.W = int(W);
  p.slots = size_t(p.W) + kv->batch;
  size_t floats = p.slots * H * (size_t(kv->dim) + 2);
  floats = (floats + 3) / 4 * 4 + (size_t(kv->batch) + 4) / 4 * 4;
  if (kv->weights) floats += size_t(kv->batch) * H * size_t(p.srows);
  p.bytes = floats * sizeof(float);
  *out = p;
  return true;
}

// Workgroups of the join a sequence and KV head whose weights it adds: `seen` rows.
int row_blocks_of(const tqkv_paged_kv* kv, int64_t seen) {
  return kv->weights ? int((seen + kWeightRows - 1) / kWeightRows) : 0;
}
int64_t join_blocks(const tqkv_paged_kv* kv, int32_t H, int row_blocks) {
  const int parts = kv->dim > 128 ? kv->dim / 128 : 1;  // JoinShape's
  return int64_t(kv->batch) * H * parts + int64_t(kv->batch) * kv->kv_heads * row_blocks;
}
// Units over the whole batch are 32-bit in the kernels, and a grid holds below
// 2^32 threads.
bool fits(const tqkv_paged_kv* kv, const HostPlan& plan, int64_t blocks) {
  return int64_t(kv->batch) * (plan.srows / kUnit + kOver + 1) <= 0x7fffffffLL &&
         blocks <= 0xffffffffLL / kJoinThreads;
}

}  // namespace
}  // namespace paged
}  // namespace tqkv

extern "C" size_t tqkv_paged_decode_workspace_size(const tqkv_paged_kv* kv, int32_t H,
                                                   int64_t max_rows) {
  using namespace tqkv::paged;
  Pool pool;
  HostPlan plan;
  if (check(kv, &pool) != TQKV_OK || !plan_of(kv, H, max_rows, &plan)) return 0;
  // The least that a window leaves of the weights' rows.
  return fits(kv, plan, join_blocks(kv, H, row_blocks_of(kv, 1))) ? plan.bytes : 0;
}

extern "C" int32_t tqkv_paged_decode_attend(const tqkv_paged_kv* kv, const uint16_t* q,
                                            int64_t q_stride, int32_t H, float scale,
                                            int64_t window, int64_t max_rows, uint16_t* out,
                                            void* workspace, size_t workspace_bytes,
                                            tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::paged;
  DecodeArgs a{};
  if (int32_t rc = check(kv, &a.pool)) return rc;
  if (!q || !out) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!aligned(q, 16) || !aligned(out, 2) || q_stride % 8 != 0)
    return fail(TQKV_EINVAL_ARG, "q is 16-byte aligned and q_stride (%lld) a multiple of 8",
                (long long)q_stride);
  HostPlan plan;
  if (H >= 1 && H % kv->kv_heads == 0 && H / kv->kv_heads > 32)
    return fail(TQKV_EUNSUPPORTED, "%d query heads a KV head", H / kv->kv_heads);
  if (!plan_of(kv, H, max_rows, &plan))
    return fail(TQKV_EINVAL_SHAPE, "H=%d kv_heads=%d max_rows=%lld", H, kv->kv_heads,
                (long long)max_rows);
  a.window = window > 0 && window < max_rows ? int(window) : 0;
  const int64_t seen = a.window > 0 ? a.window + 3 : max_rows;  // from a row of four
  const int row_blocks = row_blocks_of(kv, seen);
  const int64_t blocks = join_blocks(kv, H, row_blocks);
  if (!fits(kv, plan, blocks))
    return fail(TQKV_EUNSUPPORTED, "batch=%d max_rows=%lld", kv->batch, (long long)max_rows);
  if (!workspace) {
    if (int32_t rc = scratch_for_current_device(plan.bytes, &workspace)) return rc;
  } else if (workspace_bytes < plan.bytes || !aligned(workspace, 16)) {
    return fail(TQKV_EINVAL_ARG, "workspace of %zu bytes (16-byte aligned), need %zu",
                workspace_bytes, plan.bytes);
  }
  const int D = kv->dim;
  for (int i = 0; i < 6; ++i) a.slot[i] = kv->slot[i];
  a.q = q;
  a.qstride = q_stride;
  a.out = out;
  a.H = H;
  a.G = H / kv->kv_heads;
  a.groups16 = plan.groups16;
  a.max_rows = int(max_rows);
  a.W = plan.W;
  a.over = kOver;
  a.least = plan.least;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.part_o = static_cast<float*>(workspace);
  a.part_m = a.part_o + plan.slots * H * D;
  a.part_l = a.part_m + plan.slots * H;
  a.srows = plan.srows;
  a.kept_units = int(kKeptBytes / (int64_t(kUnit) * kv->kv_heads * 4 * D));
  a.starts = reinterpret_cast<int32_t*>(static_cast<float*>(workspace) +
                                        (plan.slots * H * (size_t(D) + 2) + 3) / 4 * 4);
  if (kv->weights)
    a.scores = reinterpret_cast<float*>(a.starts) + (kv->batch + 4) / 4 * 4;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(unsigned(a.W), unsigned(kv->kv_heads * a.groups16));
  launch(kv, a, grid, st, false);
  TQKV_LAUNCHED();
  auto join = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kJoinThreads), 0, st, a, row_blocks);
  };
  switch (D) {
    case 64: join(paged_join_kernel<64>); break;
    case 128: join(paged_join_kernel<128>); break;
    case 256: join(paged_join_kernel<256>); break;
    default: join(paged_join_kernel<512>); break;
  }
  TQKV_LAUNCHED();
  return ok();
}

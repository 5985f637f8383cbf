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
constexpr float kPartDown = 40.0f;  // log2 by which parts hold weights and their sums lower
static_assert(Bf16Rows<128>::kDown == kPartDown, "as the parts are");
static_assert(AffineRows<128, 4, 4, 64>::kLast == 0x1p-47f && AffineRows<128, 4, 4, 64>::kDown == kPartDown - 47,
              "as the parts are");
constexpr int kMaxSegments = 1024;  // of one sequence: the workgroups of a KV head

// Where sequence b's segments lie: its first unit of all, and the total.
__device__ __forceinline__ void place(const DecodeArgs& a, int b, int64_t* red, int* first,
                                      int* total) {
  int64_t mine = 0;  // units before b in the high half, all in the low
  for (int i = threadIdx.x; i < a.pool.batch; i += kJoinThreads) {
    const int64_t t = span_of(a, i).units;
    mine += t + (i < b ? t << 32 : 0);
  }
  for (int off = 32; off > 0; off >>= 1) mine += __shfl_xor(mine, off, 64);
  __syncthreads();
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = mine;
  __syncthreads();
  mine = 0;
  for (int w = 0; w < kJoinThreads / 64; ++w) mine += red[w];
  *first = int(mine >> 32);
  *total = int(mine & 0xffffffff);
}

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

// Workgroups [0, batch x H): the output of one (sequence, head) from its
// segments, a quad of channels a thread, the segments dealt over the rows of
// threads, then the rows in order. The others: kWeightRows rows of one
// (sequence, KV head), weights[row] += sum over the group's heads of
// 2^(s - m) / l.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(const DecodeArgs a,
                                                                  int row_blocks) {
  constexpr int kQuads = D / 4, kDeal = kJoinThreads / kQuads;
  __shared__ int64_t red64[kJoinThreads / 64];
  __shared__ float red[kJoinThreads / 64], weight[kMaxSegments], head_m[32], head_r[32];
  __shared__ float4 sums[kJoinThreads];
  const int tid = threadIdx.x, outs = a.pool.batch * a.H;
  const bool joins = int(blockIdx.x) < outs;
  int b, h = 0, kvh = 0, block = 0;
  if (joins) {
    b = blockIdx.x / a.H;
    h = blockIdx.x % a.H;
  } else {
    const int i = blockIdx.x - outs;
    block = i % row_blocks;
    kvh = i / row_blocks % a.pool.Hkv;
    b = i / row_blocks / a.pool.Hkv;
  }
  const Span span = span_of(a, b);
  if (joins && span.n == 0) {
    for (int d = tid; d < D; d += kJoinThreads) a.out[int64_t(blockIdx.x) * D + d] = 0;
    return;
  }
  const int row0 = span.lo / 4 * 4 + block * kWeightRows;
  if (!joins && row0 >= span.n) return;
  int first, total;
  place(a, b, red64, &first, &total);
  const int per = units_per_wg(total, a.W);
  const int w0 = (first + a.over) / per, n = (first + span.units - 1) / per - w0 + 1;
  const int64_t slot0 = w0 + b;
  float m;
  if (joins) {
    if (n == 1) return;  // written by the attention kernel
    const float l = segment_weights(a, slot0, n, h, weight, red, &m);
    const int quad = tid % kQuads, deal = tid / kQuads;
    const float* po = a.part_o + (slot0 * a.H + h) * D + 4 * quad;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int s = deal; s < n; s += kDeal) {
      const float w = weight[s];
      const float4 y = *reinterpret_cast<const float4*>(po + int64_t(s) * a.H * D);
      o.x = fmaf(w, y.x, o.x);
      o.y = fmaf(w, y.y, o.y);
      o.z = fmaf(w, y.z, o.z);
      o.w = fmaf(w, y.w, o.w);
    }
    sums[tid] = o;
    __syncthreads();
    if (deal == 0) {
      for (int i = 1; i < kDeal; ++i) {
        const float4 y = sums[i * kQuads + quad];
        o.x += y.x;
        o.y += y.y;
        o.z += y.z;
        o.w += y.w;
      }
      const float v[4] = {o.x / l, o.y / l, o.z / l, o.w / l};
      uint16_t* out = a.out + int64_t(blockIdx.x) * D + 4 * quad;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = f32_to_bf16(l == 0.0f ? 0.0f : v[i]);
    }
    return;
  }
  // A wavefront a head.
  for (int i = tid / 64; i < a.G; i += kJoinThreads / 64) {
    const int at = kvh * a.G + i, lane = tid % 64;
    float top = -INFINITY, l = 0.0f;
    for (int s = lane; s < n; s += 64) {  // the running maximum and sum of the lane's segments
      const float pm = a.part_m[(slot0 + s) * a.H + at], pl = a.part_l[(slot0 + s) * a.H + at];
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
      head_m[i] = m == -INFINITY ? 0.0f : m + kPartDown;
      head_r[i] = l == 0.0f ? 0.0f : 1.0f / l;
    }
  }
  __syncthreads();
  float* weights = a.pool.weights + (int64_t(b) * a.pool.Hkv + kvh) * a.pool.wstride;
  const float* scores = a.scores + (int64_t(b) * a.H + kvh * a.G) * a.srows;
  const int row = row0 + 4 * tid;
  if (row >= span.n) return;
  // Four rows a thread; the scores of rows outside the span are -inf or unset.
  const float4 old = *reinterpret_cast<const float4*>(weights + row);
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = 0; i < a.G; ++i) {
    const float4 x = *reinterpret_cast<const float4*>(scores + i * a.srows + row);
    const float hm = head_m[i], hr = head_r[i];
    sum[0] += __builtin_amdgcn_exp2f(x.x - hm) * hr;
    sum[1] += __builtin_amdgcn_exp2f(x.y - hm) * hr;
    sum[2] += __builtin_amdgcn_exp2f(x.z - hm) * hr;
    sum[3] += __builtin_amdgcn_exp2f(x.w - hm) * hr;
  }
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

struct HostPlan {
  int groups16, W;
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
  if (W > (most + kMinUnits - 1) / kMinUnits) W = (most + kMinUnits - 1) / kMinUnits;
  p.W = int(W);
  p.slots = size_t(p.W) + kv->batch;
  size_t floats = p.slots * H * (size_t(kv->dim) + 2);
  floats = (floats + 3) / 4 * 4;
  if (kv->weights) floats += size_t(kv->batch) * H * size_t(p.srows);
  p.bytes = floats * sizeof(float);
  *out = p;
  return true;
}

}  // namespace
}  // namespace paged
}  // namespace tqkv

extern "C" size_t tqkv_paged_decode_workspace_size(const tqkv_paged_kv* kv, int32_t H,
                                                   int64_t max_rows) {
  tqkv::paged::Pool pool;
  tqkv::paged::HostPlan plan;
  if (tqkv::paged::check(kv, &pool) != TQKV_OK || !tqkv::paged::plan_of(kv, H, max_rows, &plan))
    return 0;
  return plan.bytes;
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
  const int row_blocks = kv->weights ? int((seen + kWeightRows - 1) / kWeightRows) : 0;
  const int64_t blocks = int64_t(kv->batch) * H + int64_t(kv->batch) * kv->kv_heads * row_blocks;
  // Units over the whole batch are 32-bit in the kernels, and a grid
  // holds below 2^32 threads.
  if (int64_t(kv->batch) * (plan.srows / kUnit + kOver + 1) > 0x7fffffffLL ||
      blocks > 0xffffffffLL / kJoinThreads)
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
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.part_o = static_cast<float*>(workspace);
  a.part_m = a.part_o + plan.slots * H * D;
  a.part_l = a.part_m + plan.slots * H;
  a.srows = plan.srows;
  a.kept_units = int(kKeptBytes / (int64_t(kUnit) * kv->kv_heads * 4 * D));
  if (kv->weights)
    a.scores = static_cast<float*>(workspace) + (plan.slots * H * (size_t(D) + 2) + 3) / 4 * 4;
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

// Attention of packed sequences, over their own tokens or the paged cache.
#include "prompt_attend.hpp"

namespace tqkv {
namespace prompt {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// Channel c of a stored row as a bf16 value in f32; rows of `bits` codes are
// dequantized to bf16, one rounding.
template <Source S>
__device__ __forceinline__ float value_at(const Args& a, bool key, int64_t row, int D, int c) {
  if constexpr (S == kPacked) {
    return bf16_to_f32((key ? a.k : a.v)[row + c]);
  } else if constexpr (S == kPagedBf16) {
    return bf16_to_f32(static_cast<const uint16_t*>(a.slot[key ? 0 : 1])[row * D + c]);
  } else {
    const int at = key ? 0 : 3, bits = key ? a.bits_k : a.bits_v;
    const uint32_t w = static_cast<const uint32_t*>(a.slot[at])[row * (D * bits / 32) + c * bits / 32];
    const uint32_t code = (w >> (c * bits % 32)) & ((1u << bits) - 1u);
    const int64_t g = row * (D / a.gs) + c / a.gs;
    const float s = bf16_to_f32(static_cast<const uint16_t*>(a.slot[at + 1])[g]);
    const float b = bf16_to_f32(static_cast<const uint16_t*>(a.slot[at + 2])[g]);
    return bf16_to_f32(f32_to_bf16(fmaf(s, float(code), b)));
  }
}

// The row of key t: an element offset (packed) or a pool row; -1: none.
template <Source S>
__device__ __forceinline__ int64_t row_of(const Args& a, int b, int64_t first, int h, int t) {
  if constexpr (S == kPacked) {
    return (first + t) * a.ts + h * a.hs;
  } else {
    const int page = a.pool.table[b * a.pool.tstride + (t >> a.pool.shift)];
    if (!paged::valid_page(a.pool, page)) return -1;
    return paged::pool_row(a.pool, page, h, t & ((1 << a.pool.shift) - 1));
  }
}

// One query row by one wavefront: a lane a key for the scores, channels for
// the values. Hidden keys are left out, not multiplied by zero.
template <int D, Source S>
__device__ void attend_row(const Args& a, int b, const Sequence& s, int64_t token, int head) {
  const int lane = threadIdx.x % 64, h = head / a.G;
  const int64_t p = int64_t(s.keys) - s.count + (token - s.first);
  const Range see = visible(a, p, s.keys);
  const uint16_t* q = a.q + token * a.qs + int64_t(head) * D;
  constexpr int C = D / 64;
  float o[C], m = -INFINITY, l = 0.0f;
  bool any = false;
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.0f;
  for (int t0 = see.lo; t0 < see.hi; t0 += 64) {
    const int t = t0 + lane;
    const int64_t row = t < see.hi ? row_of<S>(a, b, s.first, h, t) : -1;
    const bool on = t < see.hi && !(S != kPacked && row < 0);
    float x = 0.0f;
    if (on)
      for (int c = 0; c < D; ++c) x = fmaf(bf16_to_f32(q[c]), value_at<S>(a, true, row, D, c), x);
    x = on ? x * a.scale * kLog2e : -INFINITY;
    const unsigned long long live = __ballot(on);
    if (!live) continue;
    any = true;
    float top = x;
#pragma unroll
    for (int d = 32; d > 0; d /= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
    const float alpha = m == -INFINITY ? 0.0f : exp2f(m - base);
    m = mn;
    const float w = on ? exp2f(x - base) : 0.0f;
    float sum = w;
#pragma unroll
    for (int d = 32; d > 0; d /= 2) sum += __shfl_xor(sum, d, 64);
    l = l * alpha + sum;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= alpha;
    for (int i = 0; i < 64; ++i) {
      if (!((live >> i) & 1)) continue;
      const float wi = __shfl(w, i, 64);
      const int64_t ri = __shfl(row, i, 64);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(wi, value_at<S>(a, false, ri, D, c * 64 + lane), o[c]);
    }
  }
  uint16_t* out = a.out + (token * a.H + head) * D;
  const float inv = any ? 1.0f / l : 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) out[c * 64 + lane] = f32_to_bf16(any ? o[c] * inv : 0.0f);
}

template <int D, Source S>
__global__ __launch_bounds__(256) void row_kernel(const Args a) {
  const int64_t unit = int64_t(blockIdx.x) * 4 + threadIdx.x / 64;
  const int64_t token = unit / a.H;
  if (token >= a.tokens || token < a.starts[0] || token >= a.starts[a.batch]) return;
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (token >= a.starts[mid]) lo = mid;
    else hi = mid;
  }
  attend_row<D, S>(a, lo, sequence<S>(a, lo), token, int(unit % a.H));
}

template <Source S>
int32_t launch(const Args& a, int D, hipStream_t st) {
  const int64_t blocks = (a.tokens * a.H + 3) / 4;
  if (blocks > 0xffffffffLL / 256) return fail(TQKV_EUNSUPPORTED, "tokens=%lld", (long long)a.tokens);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, st, a);
  };
  switch (D) {
    case 64: go(row_kernel<64, S>); break;
    case 128: go(row_kernel<128, S>); break;
    case 256: go(row_kernel<256, S>); break;
    default: go(row_kernel<512, S>); break;
  }
  TQKV_LAUNCHED();
  return ok();
}

int32_t check_queries(const uint16_t* q, int64_t q_stride, int H, int H_kv, const int32_t* starts,
                      int64_t tokens, const uint16_t* out) {
  if (H < 1 || H_kv < 1 || H % H_kv != 0 || tokens < 0 || tokens > 0x7fffffffLL)
    return fail(TQKV_EINVAL_SHAPE, "H=%d H_kv=%d tokens=%lld", H, H_kv, (long long)tokens);
  if (H / H_kv > 32) return fail(TQKV_EUNSUPPORTED, "%d query heads a KV head", H / H_kv);
  if (tokens == 0) return TQKV_OK;
  if (!q || !out || !starts) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!paged::aligned(q, 16) || !paged::aligned(out, 16) || !paged::aligned(starts, 4) ||
      q_stride % 8 != 0)
    return fail(TQKV_EINVAL_ARG, "q and out are 16-byte aligned, q_stride (%lld) a multiple of 8",
                (long long)q_stride);
  return TQKV_OK;
}

}  // namespace
}  // namespace prompt
}  // namespace tqkv

extern "C" size_t tqkv_packed_attend_workspace_size(int32_t batch, int32_t H, int32_t H_kv,
                                                    int32_t D, int64_t tokens) {
  return 0;
}

extern "C" int32_t tqkv_packed_attend(const uint16_t* q, int64_t q_stride, const uint16_t* k,
                                      const uint16_t* v, int64_t token_stride, int64_t head_stride,
                                      int32_t batch, int32_t H, int32_t H_kv, int32_t D,
                                      const int32_t* starts, int64_t tokens, float scale,
                                      int32_t causal, int64_t window, uint16_t* out,
                                      void* workspace, size_t workspace_bytes,
                                      tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::prompt;
  if (batch < 1) return fail(TQKV_EINVAL_SHAPE, "batch=%d", batch);
  if (batch > paged::kMaxBatch || !(D == 64 || D == 128 || D == 256 || D == 512))
    return fail(TQKV_EUNSUPPORTED, "batch=%d (at most %d) D=%d", batch, paged::kMaxBatch, D);
  if (int32_t rc = check_queries(q, q_stride, H, H_kv, starts, tokens, out)) return rc;
  if (window > 0 && !causal) return fail(TQKV_EINVAL_ARG, "window=%lld without causal", (long long)window);
  if (tokens == 0) return ok();
  if (!k || !v) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!paged::aligned(k, 16) || !paged::aligned(v, 16) || token_stride % 8 != 0 || head_stride % 8 != 0)
    return fail(TQKV_EINVAL_ARG,
                "k and v are 16-byte aligned, strides multiples of 8 elements (token %lld, head %lld)",
                (long long)token_stride, (long long)head_stride);
  Args a{};
  a.q = q;
  a.qs = q_stride;
  a.out = out;
  a.starts = starts;
  a.tokens = tokens;
  a.batch = batch;
  a.H = H;
  a.Hkv = H_kv;
  a.G = H / H_kv;
  a.scale = scale;
  a.causal = causal != 0;
  a.window = window > 0 ? window : 0;
  a.k = k;
  a.v = v;
  a.ts = token_stride;
  a.hs = head_stride;
  return launch<kPacked>(a, D, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t tqkv_paged_prefill_workspace_size(const tqkv_paged_kv* kv, int32_t H,
                                                    int64_t tokens, int64_t max_rows) {
  return 0;
}

extern "C" int32_t tqkv_paged_prefill_attend(const tqkv_paged_kv* kv, const uint16_t* q,
                                             int64_t q_stride, int32_t H, const int32_t* starts,
                                             int64_t tokens, float scale, int64_t window,
                                             int64_t max_rows, uint16_t* out, void* workspace,
                                             size_t workspace_bytes, tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::prompt;
  Args a{};
  if (int32_t rc = paged::check(kv, &a.pool)) return rc;
  if (int32_t rc = check_queries(q, q_stride, H, kv->kv_heads, starts, tokens, out)) return rc;
  if (max_rows < 1 || max_rows > a.pool.cap)
    return fail(TQKV_EINVAL_SHAPE, "max_rows=%lld of a table of %d", (long long)max_rows, a.pool.cap);
  if (tokens == 0) return ok();
  a.q = q;
  a.qs = q_stride;
  a.out = out;
  a.starts = starts;
  a.tokens = tokens;
  a.batch = kv->batch;
  a.H = H;
  a.Hkv = kv->kv_heads;
  a.G = H / kv->kv_heads;
  a.scale = scale;
  a.causal = 1;
  a.window = window > 0 ? window : 0;
  for (int i = 0; i < 6; ++i) a.slot[i] = kv->slot[i];
  a.gs = kv->group_size;
  a.bits_k = kv->bits_k;
  a.bits_v = kv->bits_v;
  a.max_rows = int(max_rows);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return kv->kind == TQKV_CACHE_BF16 ? launch<kPagedBf16>(a, kv->dim, st)
                                     : launch<kPagedAffine>(a, kv->dim, st);
}

// Paged cache: queries rotated, keys rotated and written with the values into
// the slots that a plan gave their tokens. Every row is read once and written
// once: bound by HBM, for a decode step by a launch's time. One kernel, as
// parts (keys, values, queries) on the grid's second axis, so that a step's
// few tokens meet many CUs. A token's slot says all that its rows need, so
// nothing is searched for in every layer. 23,100 tokens of 10 prompts, 48 heads of 128: 140 us
// for 569 MB (4.1 TB/s; 162 with one job a thread on its way); 64 tokens of a
// decode step: 3.9 us on the device, 11.6 with the host's call.
#include "affine_quantize.hpp"
#include "paged.hpp"
#include "rope.hpp"

namespace tqkv {
namespace paged {
namespace {

constexpr int kThreads = 256;
using rope::kMostTokens;

struct EnterArgs {
  Pool pool;
  rope::Rope rope;
  const uint16_t* q;
  uint16_t* q_out;
  const uint16_t* k;
  const uint16_t* v;
  int64_t qs, qos, ts, hs, tokens, pstride;
  const int4* slots;
  const int32_t* positions;
  void* slot[6];
  int H, gs, per_block;
  rope::Jobs q_jobs, k_jobs;
  rope::Divisor heads;  // KV heads
};

// A token's place in the workgroup: its rotary position, and its pool row of
// head 0 (-1: none).
struct Place {
  int32_t position;
  int64_t row;
};

enum Part { kKeys, kValues, kQueries };

// Places of the workgroup's tokens, and their angles where `turn`.
__device__ __forceinline__ void find_places(const EnterArgs& a, int64_t t0, int n, bool turn,
                                            Place* place, rope::Angle* angles) {
  const Pool& p = a.pool;
  for (int t = threadIdx.x; t < n; t += kThreads) {
    const int4 s = a.slots[t0 + t];
    const int position = a.positions ? a.positions[(t0 + t) * a.pstride] : s.z;
    const bool row = position >= 0 && valid_page(p, s.x) && s.y >= 0 && s.y < (1 << p.shift);
    place[t] = Place{position, row ? pool_row(p, s.x, 0, s.y) : -1};
  }
  if (turn)
    for (int t = 0; t < n; ++t) {
      const int position = a.positions ? a.positions[(t0 + t) * a.pstride] : a.slots[t0 + t].z;
      for (int pair = threadIdx.x; pair < a.rope.pairs; pair += kThreads)
        angles[t * a.rope.pairs + pair] = rope::angle_of(a.rope, position, pair);
    }
  __syncthreads();
}

// The written rows' gathered weights.
__device__ __forceinline__ void clear_weights(const EnterArgs& a, int64_t t0, int n,
                                              const Place* place) {
  const Pool& p = a.pool;
  if (!p.weights) return;
  for (int i = threadIdx.x; i < n * p.Hkv; i += kThreads) {
    const int t = i / p.Hkv, h = i % p.Hkv;
    const int4 s = a.slots[t0 + t];
    if (place[t].row >= 0 && s.w >= 0 && s.w < p.batch && s.z >= 0 && s.z < p.cap)
      p.weights[(int64_t(s.w) * p.Hkv + h) * p.wstride + s.z] = 0.0f;
  }
}

__device__ __forceinline__ void enter_queries(const EnterArgs& a, int64_t t0, int n, int dim,
                                              Place* place, rope::Angle* angles) {
  rope::turn_rows<kThreads>(
      a.rope, a.q_jobs, angles, n, dim,
      [&](int t, int h) { return a.q + (t0 + t) * a.qs + h * dim; },
      [&](int t, int h) -> uint16_t* {
        return place[t].position < 0 ? nullptr : a.q_out + (t0 + t) * a.qos + h * dim;
      },
      [&]() { find_places(a, t0, n, true, place, angles); });
}

template <int D>
__global__ __launch_bounds__(kThreads) void enter_bf16_kernel(const EnterArgs a) {
  __shared__ Place place[kMostTokens];
  extern __shared__ rope::Angle angles[];  // [per_block][pairs]
  const Pool& p = a.pool;
  const int64_t t0 = int64_t(blockIdx.x) * a.per_block;
  const int n = a.tokens - t0 < a.per_block ? int(a.tokens - t0) : a.per_block;
  const int part = blockIdx.y;
  if (part == kQueries) return enter_queries(a, t0, n, D, place, angles);
  const uint16_t* x = part == kKeys ? a.k : a.v;
  uint16_t* out = static_cast<uint16_t*>(a.slot[part]);
  const auto from = [&](int t, int h) { return x + (t0 + t) * a.ts + h * a.hs; };
  const auto to = [&](int t, int h) -> uint16_t* {
    return place[t].row < 0 ? nullptr : out + (place[t].row + (int64_t(h) << p.shift)) * D;
  };
  if (part == kKeys) {
    rope::turn_rows<kThreads>(a.rope, a.k_jobs, angles, n, D, from, to,
                              [&]() { find_places(a, t0, n, true, place, angles); });
    clear_weights(a, t0, n, place);
    return;
  }
  find_places(a, t0, n, false, place, angles);
  // Values: 16 bytes a thread, kDeep of them on their way.
  constexpr int LPR = D / 8, kDeep = rope::kDeep;
  const int all = n * p.Hkv * LPR;
  for (int i0 = threadIdx.x; i0 < all; i0 += kThreads * kDeep) {
    uint4 y[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int i = min(i0 + k * kThreads, all - 1), r = i / LPR;
      const int t = rope::quotient(r, a.heads), h = r - t * p.Hkv;
      y[k] = *reinterpret_cast<const uint4*>(from(t, h) + i % LPR * 8);
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int i = i0 + k * kThreads, r = i / LPR;
      if (i >= all) break;
      const int t = rope::quotient(r, a.heads), h = r - t * p.Hkv;
      uint16_t* dst = to(t, h);
      if (dst) *reinterpret_cast<uint4*>(dst + i % LPR * 8) = y[k];
    }
  }
}

// The 16 channels from c on of a key row, turned and rounded to bf16.
__device__ __forceinline__ void load_turned(const rope::Rope& r, const rope::Angle* a,
                                            const uint16_t* row, int c,
                                            float (&v)[aq::kLaneElems]) {
  const int rd = 2 * r.pairs;
  aq::load_lane(row + c, v);
  if (r.interleaved) {
#pragma unroll
    for (int e = 0; e < aq::kLaneElems; e += 2)
      if (c + e < rd) {
        const rope::Angle t = a[(c + e) / 2];
        const float x = v[e], y = v[e + 1];
        v[e] = bf16_to_f32(f32_to_bf16(rope::turned_x(x, y, t)));
        v[e + 1] = bf16_to_f32(f32_to_bf16(rope::turned_y(x, y, t)));
      }
    return;
  }
#pragma unroll
  for (int e = 0; e < aq::kLaneElems; ++e)
    if (c + e < rd) {
      const int pair = c + e < r.pairs ? c + e : c + e - r.pairs;
      const rope::Angle t = a[pair];
      const float other = bf16_to_f32(row[c + e < r.pairs ? c + e + r.pairs : pair]);
      const float y = c + e < r.pairs ? rope::turned_x(v[e], other, t) : rope::turned_y(other, v[e], t);
      v[e] = bf16_to_f32(f32_to_bf16(y));
    }
}

template <int D, int BK, int BV>
__global__ __launch_bounds__(kThreads) void enter_affine_kernel(const EnterArgs a) {
  __shared__ Place place[kMostTokens];
  extern __shared__ rope::Angle angles[];  // [per_block][pairs]
  const Pool& p = a.pool;
  const int64_t t0 = int64_t(blockIdx.x) * a.per_block;
  const int n = a.tokens - t0 < a.per_block ? int(a.tokens - t0) : a.per_block;
  const int part = blockIdx.y;
  if (part == kQueries) return enter_queries(a, t0, n, D, place, angles);
  find_places(a, t0, n, part != kValues, place, angles);
  constexpr int LPR = D / aq::kLaneElems;
  const int bits = part == kKeys ? BK : BV;
  const uint16_t* x = part == kKeys ? a.k : a.v;
  uint32_t* packed = static_cast<uint32_t*>(a.slot[3 * part]);
  uint16_t* scales = static_cast<uint16_t*>(a.slot[3 * part + 1]);
  uint16_t* biases = static_cast<uint16_t*>(a.slot[3 * part + 2]);
  const int lpg = a.gs / aq::kLaneElems, groups = D / a.gs;
  // Rows are tokens within heads, so that neighbours in a page are written
  // together.
  const int c = threadIdx.x % LPR, rows = p.Hkv * n;
  for (int row0 = 0; row0 < rows; row0 += kThreads / LPR) {
    // Whole wavefronts go round (the groups' butterflies exchange across
    // lanes): rows past the end take the last one and are not stored.
    const int at = row0 + threadIdx.x / LPR, r = at < rows ? at : rows - 1;
    const int t = r % n, h = r / n;
    const uint16_t* src = x + (t0 + t) * a.ts + h * a.hs;
    float v[aq::kLaneElems];
    if (part == kKeys)
      load_turned(a.rope, angles + t * a.rope.pairs, src, c * aq::kLaneElems, v);
    else
      aq::load_lane(src + c * aq::kLaneElems, v);
    const aq::LaneCodes q = aq::quantize_lane_refined(v, a.gs, bits);
    if (at >= rows || place[t].row < 0) continue;
    const int64_t row = place[t].row + (int64_t(h) << p.shift);
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
  if (part == kKeys) clear_weights(a, t0, n, place);
}

template <int D>
void launch(const tqkv_paged_kv* kv, const EnterArgs& a, hipStream_t st) {
  const unsigned blocks = unsigned((a.tokens + a.per_block - 1) / a.per_block);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks, a.H > 0 ? 3 : 2), dim3(kThreads),
                       a.per_block * a.rope.pairs * sizeof(rope::Angle), st, a);
  };
  if (kv->kind == TQKV_CACHE_BF16) go(enter_bf16_kernel<D>);
  else if (kv->bits_k == 4 && kv->bits_v == 4) go(enter_affine_kernel<D, 4, 4>);
  else if (kv->bits_k == 4) go(enter_affine_kernel<D, 4, 8>);
  else if (kv->bits_v == 4) go(enter_affine_kernel<D, 8, 4>);
  else go(enter_affine_kernel<D, 8, 8>);
}

}  // namespace
}  // namespace paged
}  // namespace tqkv

extern "C" int32_t tqkv_paged_append_rope(const tqkv_paged_kv* kv, const tqkv_rope* rope,
                                          const uint16_t* q, int32_t H, int64_t q_stride,
                                          uint16_t* q_out, int64_t q_out_stride,
                                          const uint16_t* k, const uint16_t* v,
                                          int64_t token_stride, int64_t head_stride,
                                          const int32_t* slots, int64_t tokens,
                                          const int32_t* positions, int64_t position_stride,
                                          tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::paged;
  EnterArgs a{};
  if (int32_t rc = check(kv, &a.pool)) return rc;
  if (int32_t rc = rope::check(rope, kv->dim, &a.rope)) return rc;
  if (H < 0 || tokens < 0 || tokens > 0xffffffffLL / kThreads)  // a grid: below 2^32 threads
    return fail(TQKV_EINVAL_SHAPE, "H=%d tokens=%lld", H, (long long)tokens);
  if (H > 1024) return fail(TQKV_EUNSUPPORTED, "H=%d (at most 1024)", H);
  if (tokens == 0) return ok();
  if (!k || !v || !slots || (H > 0 && (!q || !q_out))) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 16) || !aligned(positions, 4) ||
      token_stride % 8 != 0 || head_stride % 8 != 0)
    return fail(TQKV_EINVAL_ARG,
                "k, v and slots are 16-byte aligned, strides multiples of 8 elements (token %lld, head %lld)",
                (long long)token_stride, (long long)head_stride);
  if (H > 0 && (!aligned(q, 16) || !aligned(q_out, 16) || q_stride % 8 != 0 || q_out_stride % 8 != 0 ||
                (q == q_out && q_stride != q_out_stride)))
    return fail(TQKV_EINVAL_ARG, "q and q_out are 16-byte aligned, strides multiples of 8 (%lld, %lld)",
                (long long)q_stride, (long long)q_out_stride);
  a.q = q;
  a.q_out = q_out;
  a.k = k;
  a.v = v;
  a.qs = q_stride;
  a.qos = q_out_stride;
  a.ts = token_stride;
  a.hs = head_stride;
  a.tokens = tokens;
  a.positions = positions;
  a.pstride = position_stride;
  a.slots = reinterpret_cast<const int4*>(slots);
  for (int i = 0; i < 6; ++i) a.slot[i] = kv->slot[i];
  a.H = H;
  a.gs = kv->group_size;
  a.q_jobs = rope::jobs_of(a.rope, H, kv->dim, q != q_out);
  a.k_jobs = rope::jobs_of(a.rope, kv->kv_heads, kv->dim, true);
  a.heads = rope::divisor(kv->kv_heads);
  a.per_block = rope::tokens_of(a.k_jobs, tokens);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (kv->dim) {
    case 64: launch<64>(kv, a, st); break;
    case 128: launch<128>(kv, a, st); break;
    case 256: launch<256>(kv, a, st); break;
    default: launch<512>(kv, a, st); break;
  }
  TQKV_LAUNCHED();
  return ok();
}

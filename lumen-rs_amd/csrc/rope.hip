// Rotary positions: the table of turns (host), and heads rotated in place or
// on their way elsewhere. Bound by HBM (each channel read and written once);
// a decode step by a launch's time. 20,011 tokens of 24 heads of 256 channels:
// 109 us for 492 MB (4.5 TB/s, a large copy runs at 4.9); 64 tokens of a decode
// step: 4.0 us on the device, 7.7 with the host's call.
#include "rope.hpp"

#include <cmath>

#include "paged.hpp"

namespace tqkv {
namespace rope {

int32_t check(const tqkv_rope* rope, int32_t dim, Rope* out) {
  if (!rope) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (rope->rotary_dim < 2 || rope->rotary_dim % 2 != 0 || rope->rotary_dim > dim)
    return fail(TQKV_EINVAL_SHAPE, "rotary_dim=%d of dim=%d", rope->rotary_dim, dim);
  if (!(rope->interleaved == 0 || rope->interleaved == 1) || rope->reserved != 0)
    return fail(TQKV_EINVAL_ARG, "interleaved=%d reserved=%d", rope->interleaved, rope->reserved);
  if (!rope->turns || !paged::aligned(rope->turns, 8))
    return fail(TQKV_EINVAL_ARG, "turns is null or not 8-byte aligned");
  *out = Rope{rope->turns, rope->magnitude, rope->rotary_dim / 2, rope->interleaved};
  return TQKV_OK;
}

namespace {

constexpr int kThreads = 256;

struct ApplyArgs {
  Rope rope;
  const int32_t* positions;
  int64_t pstride, tokens, xts, xhs, ots, ohs;
  const uint16_t* x;
  uint16_t* out;
  int dim, per_block;
  Jobs jobs;
};

__global__ __launch_bounds__(kThreads) void rope_kernel(const ApplyArgs a) {
  extern __shared__ Angle angles[];  // [per_block][pairs]
  __shared__ int32_t positions[kMostTokens];
  const int64_t t0 = int64_t(blockIdx.x) * a.per_block;
  const int n = a.tokens - t0 < a.per_block ? int(a.tokens - t0) : a.per_block;
  turn_rows<kThreads>(
      a.rope, a.jobs, angles, n, a.dim,
      [&](int t, int h) { return a.x + (t0 + t) * a.xts + h * a.xhs; },
      [&](int t, int h) -> uint16_t* {
        return positions[t] < 0 ? nullptr : a.out + (t0 + t) * a.ots + h * a.ohs;
      },
      [&]() {
        for (int t = 0; t < n; ++t) {
          const int position = a.positions[(t0 + t) * a.pstride];
          if (threadIdx.x == 0) positions[t] = position;
          for (int pair = threadIdx.x; pair < a.rope.pairs; pair += kThreads)
            angles[t * a.rope.pairs + pair] = angle_of(a.rope, position, pair);
        }
        __syncthreads();
      });
}

}  // namespace
}  // namespace rope
}  // namespace tqkv

extern "C" int32_t tqkv_rope_turns(const tqkv_rope_config* c, uint64_t* turns, float* magnitude) {
  using namespace tqkv;
  if (!c || !turns || !magnitude) return fail(TQKV_EINVAL_ARG, "null pointer");
  const int rd = c->rotary_dim;
  if (rd < 2 || rd % 2 != 0 || rd > 2 * rope::kMostPairs)
    return fail(TQKV_EINVAL_SHAPE, "rotary_dim=%d", rd);
  if (c->scaling < TQKV_ROPE_PLAIN || c->scaling > TQKV_ROPE_RAMP)
    return fail(TQKV_EUNSUPPORTED, "scaling=%d", c->scaling);
  if (!(c->base > 1.0) || !std::isfinite(c->base))
    return fail(TQKV_EINVAL_ARG, "base=%g", c->base);
  const bool ends = c->scaling == TQKV_ROPE_BANDS || c->scaling == TQKV_ROPE_RAMP;
  if (c->scaling != TQKV_ROPE_PLAIN && (!(c->factor > 0.0) || !std::isfinite(c->factor)))
    return fail(TQKV_EINVAL_ARG, "factor=%g", c->factor);
  if (ends && (!(c->original > 0.0) || !std::isfinite(c->original) || !(c->low > 0.0) ||
               !(c->high > c->low) || !std::isfinite(c->high)))
    return fail(TQKV_EINVAL_ARG, "original=%g low=%g high=%g", c->original, c->low, c->high);
  // 80-bit arithmetic: the turns carry 64 bits.
  typedef long double real;
  const real pi2 = 6.283185307179586476925286766559005768L;
  const real factor = c->factor;
  real base = c->base;
  if (c->scaling == TQKV_ROPE_BASE && rd > 2) {
    base *= powl(factor, real(rd) / (rd - 2));
    if (!(base > 1.0L) || !std::isfinite(base))
      return fail(TQKV_EINVAL_ARG, "base=%g factor=%g", c->base, c->factor);
  }
  const auto channel = [&](real t) { return rd * logl(c->original / (pi2 * t)) / (2.0L * logl(base)); };
  real first = 0.0L, last = 0.0L;
  if (c->scaling == TQKV_ROPE_RAMP) {
    first = fmaxl(floorl(channel(c->high)), 0.0L);
    last = fminl(ceill(channel(c->low)), real(rd - 1));
  }
  for (int i = 0; i < rd / 2; ++i) {
    real theta = powl(base, -2.0L * i / rd);
    real stays = 1.0L;  // share of the unscaled turn
    if (c->scaling == TQKV_ROPE_LINEAR) stays = 0.0L;
    if (c->scaling == TQKV_ROPE_BANDS)
      stays = (theta * c->original / pi2 - c->low) / (real(c->high) - c->low);
    if (c->scaling == TQKV_ROPE_RAMP) stays = 1.0L - (i - first) / fmaxl(last - first, 0.001L);
    stays = fminl(fmaxl(stays, 0.0L), 1.0L);
    if (stays < 1.0L) theta = theta * stays + theta / factor * (1.0L - stays);
    const real turn = fmodl(theta / pi2, 1.0L) * 18446744073709551616.0L;
    turns[i] = turn < 18446744073709551615.0L ? uint64_t(turn + 0.5L) : 0;
  }
  *magnitude = c->scaling == TQKV_ROPE_RAMP ? float(0.1L * logl(factor) + 1.0L) : 1.0f;
  return ok();
}

extern "C" int32_t tqkv_rope_apply(const tqkv_rope* rope, const int32_t* positions,
                                   int64_t position_stride, int64_t tokens, const uint16_t* x,
                                   int32_t heads, int32_t dim, int64_t x_token_stride,
                                   int64_t x_head_stride, uint16_t* out, int64_t out_token_stride,
                                   int64_t out_head_stride, tqkv_stream stream) {
  using namespace tqkv;
  using namespace tqkv::rope;
  if (dim < 8 || dim % 8 != 0 || dim > 2 * kMostPairs)
    return fail(TQKV_EUNSUPPORTED, "dim=%d", dim);
  ApplyArgs a{};
  if (int32_t rc = check(rope, dim, &a.rope)) return rc;
  if (heads < 1 || tokens < 0 || tokens > 0xffffffffLL / kThreads)  // a grid: below 2^32 threads
    return fail(TQKV_EINVAL_SHAPE, "heads=%d tokens=%lld", heads, (long long)tokens);
  if (heads > 1024) return fail(TQKV_EUNSUPPORTED, "heads=%d (at most 1024)", heads);
  if (tokens == 0) return ok();
  if (!positions || !x || !out) return fail(TQKV_EINVAL_ARG, "null pointer");
  if (!paged::aligned(positions, 4) || !paged::aligned(x, 16) || !paged::aligned(out, 16) ||
      x_token_stride % 8 != 0 || x_head_stride % 8 != 0 || out_token_stride % 8 != 0 ||
      out_head_stride % 8 != 0)
    return fail(TQKV_EINVAL_ARG, "x and out are 16-byte aligned, strides multiples of 8 elements");
  const bool same = x == out;
  if (same && (x_token_stride != out_token_stride || x_head_stride != out_head_stride))
    return fail(TQKV_EINVAL_ARG, "in place with other strides");
  a.positions = positions;
  a.pstride = position_stride;
  a.tokens = tokens;
  a.xts = x_token_stride;
  a.xhs = x_head_stride;
  a.ots = out_token_stride;
  a.ohs = out_head_stride;
  a.x = x;
  a.out = out;
  a.dim = dim;
  a.jobs = jobs_of(a.rope, heads, dim, !same);
  a.per_block = tokens_of(a.jobs, tokens);
  const int64_t blocks = (tokens + a.per_block - 1) / a.per_block;
  hipLaunchKernelGGL(rope_kernel, dim3(unsigned(blocks)), dim3(kThreads),
                     a.per_block * a.rope.pairs * sizeof(Angle), reinterpret_cast<hipStream_t>(stream), a);
  TQKV_LAUNCHED();
  return ok();
}

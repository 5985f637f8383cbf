// Attention of packed sequences, over their own tokens or the paged cache.
#include "prompt_few.hpp"

namespace tqkv {
namespace prompt {
// Each in a file of its own.
extern template void launch_prompt<64>(const Args&, Source, hipStream_t);
extern template void launch_few<64>(const Args&, Source, hipStream_t);
extern template void launch_prompt<128>(const Args&, Source, hipStream_t);
extern template void launch_few<128>(const Args&, Source, hipStream_t);
extern template void launch_prompt<256>(const Args&, Source, hipStream_t);
extern template void launch_few<256>(const Args&, Source, hipStream_t);
extern template void launch_prompt<512>(const Args&, Source, hipStream_t);
extern template void launch_few<512>(const Args&, Source, hipStream_t);
namespace {

// Affine rows of the sequences that have queries, dequantized once a KV head, as
// f16 (11 bits where bf16 keeps 8) times powers of two that bring the head's
// largest K and V below 2^15; V as bf16 where its groups' largest values lie too
// far apart for f16, since a query may see the small ones alone (K's are met by
// kCoarse). First what a head's scales and biases allow: (largest finite |K|,
// largest |V|, smallest |V| of a group's largest but zero).
constexpr int kRangeParts = 32;

struct Rows {
  int lo, n;  // rows [lo, n) are seen by some query
};
__device__ __forceinline__ Rows seen_rows(const Args& a, int b) {
  const Sequence s = sequence<kPagedAffine>(a, b);
  return Rows{first_seen(a, s.keys - s.count), s.count > 0 ? s.keys : 0};
}

__global__ __launch_bounds__(256) void range_kernel(const Args a, int D, float4* part) {
  __shared__ float4 tops[4];
  const int h = blockIdx.y, b = blockIdx.z, groups = D / a.gs;
  const Rows rows = seen_rows(a, b);
  const int span = max(0, rows.n - rows.lo), each = (span + kRangeParts - 1) / kRangeParts;
  const int from = rows.lo + int(blockIdx.x) * each, to = min(from + each, rows.n);
  const int words = a.gs * a.bits_v / 32;  // of a group
  const float most_k = float((1 << a.bits_k) - 1), most_v = float((1 << a.bits_v) - 1);
  const auto bound = [&](int side, int64_t g, float most) {
    const float s = bf16_to_f32(static_cast<const uint16_t*>(a.slot[3 * side + 1])[g]);
    const float z = bf16_to_f32(static_cast<const uint16_t*>(a.slot[3 * side + 2])[g]);
    const float x = fabsf(z), y = fabsf(fmaf(s, most, z));
    return x < INFINITY && y < INFINITY ? fmaxf(x, y) : INFINITY;  // NaN too
  };
  float k = 0.0f, v = 0.0f, low = INFINITY;
  for (int i = threadIdx.x; i < (to - from) * groups; i += 256) {
    const int64_t row = row_of<kPagedAffine>(a, b, 0, h, from + i / groups);
    if (row < 0) continue;
    const int64_t g = row * groups + i % groups;
    const float y = bound(0, g, most_k);
    if (y < INFINITY) k = fmaxf(k, y);
    const float x = bound(1, g, most_v);
    // A quantizer stores zeros as codes of zero times its least scale: those are
    // no small values.
    if (x > 0.0f && x < INFINITY && !(static_cast<const uint16_t*>(a.slot[5])[g] & 0x7fff)) {
      const uint32_t* codes = static_cast<const uint32_t*>(a.slot[3]) + g * words;
      uint32_t any = 0;
      for (int e = 0; e < words; ++e) any |= codes[e];
      if (!any) continue;
    }
    v = fmaxf(v, x);
    if (x > 0.0f) low = fminf(low, x);
  }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    k = fmaxf(k, __shfl_xor(k, d, 64));
    v = fmaxf(v, __shfl_xor(v, d, 64));
    low = fminf(low, __shfl_xor(low, d, 64));
  }
  if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = make_float4(k, v, low, 0.0f);
  __syncthreads();
  if (threadIdx.x == 0) {
    float4 x = tops[0];
    for (int i = 1; i < 4; ++i)
      x = make_float4(fmaxf(x.x, tops[i].x), fmaxf(x.y, tops[i].y), fminf(x.z, tops[i].z), 0.0f);
    part[(int64_t(b) * a.Hkv + h) * kRangeParts + blockIdx.x] = x;
  }
}

// 32 codes of `bits` from w as f32.
__device__ __forceinline__ void codes_of(const uint32_t* w, int bits, float (&f)[32]) {
  if (bits == 8) {
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = float((w[i / 4] >> (8 * (i % 4))) & 0xffu);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t e = w[k] & 0x0f0f0f0fu, o = (w[k] >> 4) & 0x0f0f0f0fu;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[8 * k + 2 * j] = float((e >> (8 * j)) & 0xffu);
        f[8 * k + 2 * j + 1] = float((o >> (8 * j)) & 0xffu);
      }
    }
  }
}

template <int D>
__global__ __launch_bounds__(256) void slab_kernel(const Args a, const float4* part, uint16_t* slab_k,
                                                   uint16_t* slab_v, int32_t* exponent) {
  constexpr int kRuns = D / 32;
  const int h = blockIdx.y, b = blockIdx.z;
  const Rows rows = seen_rows(a, b);
  const int t0 = int(blockIdx.x) * 64;
  if (t0 + 64 <= rows.lo || t0 >= rows.n) return;
  const int64_t unit = int64_t(b) * a.Hkv + h;
  float k_top = 0.0f, v_top = 0.0f, v_low = INFINITY;
#pragma unroll
  for (int i = 0; i < kRangeParts; ++i) {
    const float4 x = part[unit * kRangeParts + i];
    k_top = fmaxf(k_top, x.x);
    v_top = fmaxf(v_top, x.y);
    v_low = fminf(v_low, x.z);
  }
  const auto up_of = [](float top) {
    return top > 0.0f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
  };
  const int k_up = up_of(k_top), v_up = up_of(v_top);
  // A group whose largest is 2^-14 keeps 11 bits of that: f16's least step is 2^-24.
  const bool halves = v_top < INFINITY && (v_top == 0.0f || ldexpf(v_low, v_up) >= 0x1p-14f);
  if (threadIdx.x == 0) {  // every block of the head writes the same
    exponent[2 * unit] = -k_up;
    exponent[2 * unit + 1] = halves ? -v_up : kBf16;
  }
  for (int i = threadIdx.x; i < 64 * kRuns; i += 256) {
    const int t = t0 + i / kRuns, run = i % kRuns;
    if (t >= rows.n) break;
    const int64_t row = row_of<kPagedAffine>(a, b, 0, h, t);
    uint32_t k[16] = {}, v[16] = {};
    if (row >= 0) {
      uint32_t w[8];
      float f[32];
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const int bits = side ? a.bits_v : a.bits_k, at = 3 * side;
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(a.slot[at]) + row * (D * bits / 32) + run * bits);
        const uint4 x = src[0], y = bits == 8 ? src[1] : make_uint4(0, 0, 0, 0);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
        codes_of(w, bits, f);
        const int64_t g = row * (D / a.gs) + 32 * run / a.gs;
        const float s = bf16_to_f32(static_cast<const uint16_t*>(a.slot[at + 1])[g]);
        const float z = bf16_to_f32(static_cast<const uint16_t*>(a.slot[at + 2])[g]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = fmaf(s, f[2 * e], z), q = fmaf(s, f[2 * e + 1], z);
          if (!side) k[e] = pack_f16(ldexpf(p, k_up), ldexpf(q, k_up));
          else if (halves) v[e] = pack_f16(ldexpf(p, v_up), ldexpf(q, v_up));
          else v[e] = pack_bf16(p, q);
        }
      }
    }
    uint4* kd = reinterpret_cast<uint4*>(slab_k + (unit * a.slab_rows + t) * D + 32 * run);
    uint4* vd = reinterpret_cast<uint4*>(slab_v + (unit * a.slab_rows + t) * D + 32 * run);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      kd[e] = make_uint4(k[4 * e], k[4 * e + 1], k[4 * e + 2], k[4 * e + 3]);
      vd[e] = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
    }
  }
}

// What a call launches, and its workspace; false for what it refuses.
struct Plan {
  bool few;  // few_kernel
  int ids, splits, split_keys;
  int64_t slab_rows;                     // 0: no slab
  size_t slab, exponents, parts, bytes;  // bytes: of all
};
// Workgroups that splits make up to, and keys that a split holds at least. A
// prompt's blocks are split where they would not fill the CUs once and a half (two
// chunks of 2,048 tokens with 30,011 keys, 512 blocks: 1,950 us unsplit, 2,030 and
// 2,115 in two and three); few rows' small blocks up to 8 a CU, since their
// wavefronts wait for loads (32 sequences of up to 24,000 rows, D = 128, an earlier
// step of the kernel: 175 us, 305 unsplit).
constexpr int64_t kWanted = 384, kWantedFew = 2048;
constexpr int64_t kLeastKeys = 512, kLeastFew = 512;

bool plan_of(int batch, int H, int Hkv, int D, int64_t tokens, int64_t keys, Source source, Plan* out) {
  const int G = H / Hkv;
  const int64_t sequences = tokens < batch ? tokens : batch, rows = tokens * G;
  Plan p{};
  // Rows of a sequence on the average: the host knows no more. Up to a block of
  // few_kernel's: 6 drafted tokens of 4 heads a KV head take 117 us there, 568 in
  // the prompt kernel, whose 256-row blocks are nearly empty.
  const int64_t few_rows = D >= 256 ? Few<256, false>::kRows : Few<128, false>::kRows;
  p.few = source != kPacked && rows <= sequences * few_rows;
  const int64_t block = p.few ? few_rows
                        : D <= 128 ? Shape<128>::kRows
                        : D == 256 ? Shape<256>::kRows
                                   : Shape<512>::kRows;
  const int64_t ids = rows / block + batch;
  if (units_of(Hkv, ids) > 0xffffffffLL / 512) return false;  // a grid: below 2^32 threads
  p.ids = int(ids);
  const int64_t units = (rows / block + sequences) * Hkv;
  // A split writes and reads its block's partials: 16 keys a row pay for them.
  const int64_t live = rows / sequences < block ? rows / sequences : block;
  int64_t least = p.few ? kLeastFew : kLeastKeys;
  if (least < 16 * live) least = 16 * live;
  int64_t n = p.few ? (kWantedFew + units - 1) / units : kWanted / units;
  if (n > keys / least) n = keys / least;
  if (n < 1) n = 1;
  const int64_t len = ((keys + n - 1) / n + 63) / 64 * 64;
  p.splits = int((keys + len - 1) / len);
  p.split_keys = int(len);
  if (p.splits < 1) p.splits = 1;
  const auto whole = [](size_t x) { return (x + 255) / 256 * 256; };
  if (source == kPagedAffine && !p.few) {
    p.slab_rows = keys;
    p.slab = whole(size_t(batch) * Hkv * size_t(keys) * D * 2);
    p.exponents = whole(size_t(batch) * Hkv * 8) + whole(size_t(batch) * Hkv * kRangeParts * 16);
  }
  if (p.splits > 1) p.parts = whole(size_t(tokens) * H * p.splits * (D + 2) * 4);
  p.bytes = 2 * p.slab + p.exponents + p.parts;
  *out = p;
  return true;
}

int32_t attend(Args& a, int D, Source source, const Plan& p, void* workspace, size_t workspace_bytes,
               hipStream_t st) {
  if (p.bytes) {
    if (!workspace) {
      if (int32_t rc = scratch_for_current_device(p.bytes, &workspace)) return rc;
    } else if (workspace_bytes < p.bytes || !paged::aligned(workspace, 16)) {
      return fail(TQKV_EINVAL_ARG, "workspace of %zu bytes (16-byte aligned), need %zu",
                  workspace_bytes, p.bytes);
    }
  }
  a.ids = p.ids;
  a.splits = p.splits;
  a.split_keys = p.split_keys;
  char* at = static_cast<char*>(workspace);
  if (p.slab_rows) {
    uint16_t* k = reinterpret_cast<uint16_t*>(at);
    uint16_t* v = reinterpret_cast<uint16_t*>(at + p.slab);
    at += 2 * p.slab;
    int32_t* exponent = reinterpret_cast<int32_t*>(at);
    float4* part = reinterpret_cast<float4*>(at + (size_t(a.batch) * a.Hkv * 8 + 255) / 256 * 256);
    at += p.exponents;
    a.slab_k = k;
    a.slab_v = v;
    a.exponent = exponent;
    a.slab_rows = p.slab_rows;
    hipLaunchKernelGGL(range_kernel, dim3(kRangeParts, a.Hkv, a.batch), dim3(256), 0, st, a, D, part);
    TQKV_LAUNCHED();
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(unsigned((p.slab_rows + 63) / 64), a.Hkv, a.batch), dim3(256), 0,
                         st, a, part, k, v, exponent);
    };
    switch (D) {
      case 64: go(slab_kernel<64>); break;
      case 128: go(slab_kernel<128>); break;
      case 256: go(slab_kernel<256>); break;
      default: go(slab_kernel<512>); break;
    }
    TQKV_LAUNCHED();
  }
  if (p.splits > 1) {
    const size_t slots = size_t(a.tokens) * a.H * p.splits;
    a.part_o = reinterpret_cast<float*>(at);
    a.part_m = a.part_o + slots * D;
    a.part_l = a.part_m + slots;
  }
  switch (D) {
    case 64: (p.few ? launch_few<64> : launch_prompt<64>)(a, source, st); break;
    case 128: (p.few ? launch_few<128> : launch_prompt<128>)(a, source, st); break;
    case 256: (p.few ? launch_few<256> : launch_prompt<256>)(a, source, st); break;
    default: (p.few ? launch_few<512> : launch_prompt<512>)(a, source, st); break;
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
  // Rows that end with what is not finite are done again from their queries.
  if (q == out) return fail(TQKV_EINVAL_ARG, "out is q");
  return TQKV_OK;
}

}  // namespace
}  // namespace prompt
}  // namespace tqkv

extern "C" size_t tqkv_packed_attend_workspace_size(int32_t batch, int32_t H, int32_t H_kv,
                                                    int32_t D, int64_t tokens) {
  using namespace tqkv::prompt;
  Plan p;
  if (batch < 1 || batch > tqkv::paged::kMaxBatch || !(D == 64 || D == 128 || D == 256 || D == 512) ||
      H < 1 || H_kv < 1 || H % H_kv != 0 || H / H_kv > 32 || tokens < 1 || tokens > 0x7fffffffLL ||
      !plan_of(batch, H, H_kv, D, tokens, tokens, kPacked, &p))
    return 0;
  return p.bytes;
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
  if (token_stride < 0 || token_stride >= (int64_t(1) << 27))  // a lane's offset is 32-bit
    return fail(TQKV_EUNSUPPORTED, "token_stride=%lld (below 2^27)", (long long)token_stride);
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
  a.window = window > 0 && window < 0x7fffffff ? int(window) : 0;
  a.k = k;
  a.v = v;
  a.ts = token_stride;
  a.hs = head_stride;
  Plan p;
  if (!plan_of(batch, H, H_kv, D, tokens, tokens, kPacked, &p))
    return fail(TQKV_EUNSUPPORTED, "tokens=%lld", (long long)tokens);
  return attend(a, D, kPacked, p, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t tqkv_paged_prefill_workspace_size(const tqkv_paged_kv* kv, int32_t H,
                                                    int64_t tokens, int64_t max_rows) {
  using namespace tqkv::prompt;
  tqkv::paged::Pool pool;
  Plan p;
  if (tqkv::paged::check(kv, &pool) != TQKV_OK || H < 1 || H % kv->kv_heads != 0 ||
      H / kv->kv_heads > 32 || tokens < 1 || tokens > 0x7fffffffLL || max_rows < 1 ||
      max_rows > pool.cap ||
      !plan_of(kv->batch, H, kv->kv_heads, kv->dim, tokens, max_rows,
               kv->kind == TQKV_CACHE_AFFINE ? kPagedAffine : kPagedBf16, &p))
    return 0;
  return p.bytes;
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
  a.window = window > 0 && window < 0x7fffffff ? int(window) : 0;
  for (int i = 0; i < 6; ++i) a.slot[i] = kv->slot[i];
  a.gs = kv->group_size;
  a.bits_k = kv->bits_k;
  a.bits_v = kv->bits_v;
  a.max_rows = int(max_rows);
  const Source source = kv->kind == TQKV_CACHE_AFFINE ? kPagedAffine : kPagedBf16;
  Plan p;
  if (!plan_of(kv->batch, H, kv->kv_heads, kv->dim, tokens, max_rows, source, &p))
    return fail(TQKV_EUNSUPPORTED, "tokens=%lld max_rows=%lld", (long long)tokens, (long long)max_rows);
  return attend(a, kv->dim, p.slab_rows ? kSlab : source, p, workspace, workspace_bytes,
                reinterpret_cast<hipStream_t>(stream));
}

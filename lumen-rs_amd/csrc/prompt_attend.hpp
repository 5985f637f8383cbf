// Attention of packed sequences: what its kernels share. Keys and values are
// rows of the same packed tokens, or of the paged cache.
#pragma once

#include "paged.hpp"

namespace tqkv {
namespace prompt {

// Where keys and values lie.
enum Source { kPacked, kPagedBf16, kPagedAffine };

struct Args {
  const uint16_t* q;  // head h of token i at q + i * qs + h * D
  int64_t qs;
  uint16_t* out;  // [tokens, H, D]
  const int32_t* starts;
  int64_t tokens;
  int batch, H, Hkv, G;
  float scale;
  int causal;
  int64_t window;  // 0: none
  // kPacked: head h of token i at i * ts + h * hs.
  const uint16_t* k;
  const uint16_t* v;
  int64_t ts, hs;
  // Pages.
  paged::Pool pool;
  const void* slot[6];
  int gs, bits_k, bits_v, max_rows;
};

// A sequence's queries [first, first + count) and the keys that it has.
struct Sequence {
  int64_t first;
  int count, keys;
};
// starts is taken as ascending within [0, tokens]; what is not stays in bounds.
template <Source S>
__device__ __forceinline__ Sequence sequence(const Args& a, int b) {
  int64_t lo = a.starts[b], hi = a.starts[b + 1];
  lo = lo < 0 ? 0 : lo < a.tokens ? lo : a.tokens;
  hi = hi < lo ? lo : hi < a.tokens ? hi : a.tokens;
  const int count = int(hi - lo);
  if constexpr (S == kPacked) return Sequence{lo, count, count};
  return Sequence{lo, count, paged::held(a.pool, b, a.max_rows)};
}

// The keys [lo, hi) that the query at position p sees of n.
struct Range {
  int lo, hi;
};
__device__ __forceinline__ Range visible(const Args& a, int64_t p, int n) {
  int64_t lo = 0, hi = n;
  if (a.causal) {
    if (p + 1 < hi) hi = p + 1;
    if (a.window > 0 && p - a.window + 1 > lo) lo = p - a.window + 1;
  }
  if (hi < 0) hi = 0;
  return Range{int(lo < hi ? lo : hi), int(hi)};
}

}  // namespace prompt
}  // namespace tqkv

// Rotary positions: the device side that rope.hip and paged_append_rope.hip
// share.
//
// The angle of (position p, pair i) is p * turns[i] modulo 2^64 in units of
// 2^-64 turn: integer arithmetic wraps where the angle does, so nothing is
// lost at far positions (f32 angles are off by 2^-8 rad at position 65,536).
// Its upper 32 bits, signed, are a fraction of a turn in [-1/2, 1/2) to 2^-33;
// the cosine and sine of that in f32 are off by a few 2^-24, less than the
// products' own rounding. A workgroup takes its tokens' cosines and sines
// once into LDS, for all heads.
#pragma once

#include "common.hpp"

namespace tqkv {
namespace rope {

struct Rope {
  const uint64_t* turns;
  float magnitude;
  int pairs;  // rotary_dim / 2
  int interleaved;
};

constexpr int kMostPairs = 512;

struct Angle {
  float c, s;
};

__device__ __forceinline__ Angle angle_of(const Rope& r, int position, int pair) {
  const uint64_t turn = uint64_t(int64_t(position)) * r.turns[pair] + 0x80000000ull;
  const float half = float(int32_t(turn >> 32)) * 4.656612873077393e-10f;  // 2^-31: half turns
  float s, c;
  sincospif(half, &s, &c);
  return Angle{c * r.magnitude, s * r.magnitude};
}

// Pair (x, y) turned.
__device__ __forceinline__ float turned_x(float x, float y, Angle a) { return fmaf(x, a.c, -(y * a.s)); }
__device__ __forceinline__ float turned_y(float x, float y, Angle a) { return fmaf(x, a.s, y * a.c); }

__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t two(float x, float y) {
  return uint32_t(f32_to_bf16(x)) | (uint32_t(f32_to_bf16(y)) << 16);
}

// Eight channels as four neighbouring pairs from pair `first` on; those at or
// past `pairs` stay.
__device__ __forceinline__ uint4 turn_neighbours(uint4 x, const Angle* a, int first, int pairs) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (first + i < pairs) {
      const Angle t = a[first + i];
      const float u = low(w[i]), v = high(w[i]);
      w[i] = two(turned_x(u, v, t), turned_y(u, v, t));
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight pairs whose first and second channels are x's and y's.
__device__ __forceinline__ void turn_halves(uint4& x, uint4& y, const Angle* a) {
  uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Angle t0 = a[2 * i], t1 = a[2 * i + 1];
    const float x0 = low(u[i]), y0 = low(v[i]), x1 = high(u[i]), y1 = high(v[i]);
    u[i] = two(turned_x(x0, y0, t0), turned_x(x1, y1, t1));
    v[i] = two(turned_y(x0, y0, t0), turned_y(x1, y1, t1));
  }
  x = make_uint4(u[0], u[1], u[2], u[3]);
  y = make_uint4(v[0], v[1], v[2], v[3]);
}

// A quotient by a number fixed for a launch. m is 2^32 / d rounded up, less
// than one too much: the product's upper half is x / d or, from x * d = 2^32
// on, at times one more.
struct Divisor {
  uint32_t d, m;
};
inline Divisor divisor(int d) { return Divisor{uint32_t(d), uint32_t(((uint64_t(1) << 32) + d - 1) / d)}; }
__device__ __forceinline__ uint32_t quotient(uint32_t x, Divisor d) {
  const uint32_t q = d.d == 1 ? x : __umulhi(x, d.m);
  return q * d.d > x ? q - 1 : q;
}

// The heads of a workgroup's tokens as jobs, what one thread turns or copies at
// once: eight channels (neighbours, and channels behind the rotated ones),
// twice eight (halves that are whole pieces of eight) or single pairs and
// channels (other halves). A pair's two channels are read and written by one
// thread, so rows may turn in place.
struct Jobs {
  Divisor a_head, a_token;  // jobs
  int turning;              // of a head; the others copy
  int singles;
};
inline Jobs jobs_of(const Rope& r, int heads, int dim, bool copy) {
  const int rd = 2 * r.pairs;
  Jobs j;
  j.singles = !r.interleaved && r.pairs % 8 != 0;
  j.turning = j.singles ? r.pairs : r.interleaved ? (rd + 7) / 8 : r.pairs / 8;
  const int behind = j.singles ? dim - rd : (dim - (r.interleaved ? j.turning * 8 : rd)) / 8;
  const int each = j.turning + (copy ? behind : 0);
  j.a_head = divisor(each);
  j.a_token = divisor(each * (heads > 0 ? heads : 1));
  return j;
}
// Tokens a workgroup: enough jobs for every thread to have kDeep on their way, as
// long as there is a workgroup or two for every CU. Prompts' appends: 145 us with up
// to 8 tokens, 149 with 4, 162 with 2, 180 with 1.
constexpr int kDeep = 4, kMostTokens = 8;
inline int tokens_of(const Jobs& j, int64_t tokens) {
  int n = 1;
  while (n < kMostTokens && n * int(j.a_token.d) < 1024 && tokens >= 512 * n) n *= 2;
  return n;
}

// from(t, h) and to(t, h): rows of token t and head h; to gives NULL where
// nothing is written. ready() makes the angles, [tokens][pairs] in LDS, and
// what `to` needs, barrier included: the first jobs' channels are on their way
// meanwhile.
template <int Threads, typename From, typename To, typename Ready>
__device__ __forceinline__ void turn_rows(const Rope& r, const Jobs& jobs, const Angle* angles,
                                          int tokens, int dim, From from, To to, Ready ready) {
  const uint32_t all = jobs.a_token.d * tokens;
  const int rd = 2 * r.pairs;
  if (jobs.singles) {
    ready();
    for (uint32_t i = threadIdx.x; i < all; i += Threads) {
      const int t = quotient(i, jobs.a_token), in = i - t * jobs.a_token.d;
      const int h = quotient(in, jobs.a_head), j = in - h * jobs.a_head.d;
      uint16_t* dst = to(t, h);
      if (!dst) continue;
      const uint16_t* src = from(t, h);
      if (j < jobs.turning) {
        const Angle a = angles[t * r.pairs + j];
        const float x = bf16_to_f32(src[j]), y = bf16_to_f32(src[j + r.pairs]);
        dst[j] = f32_to_bf16(turned_x(x, y, a));
        dst[j + r.pairs] = f32_to_bf16(turned_y(x, y, a));
      } else {
        dst[rd + j - jobs.turning] = src[rd + j - jobs.turning];
      }
    }
    return;
  }
  bool first = true;
  for (uint32_t i0 = 0; i0 < all || first; i0 += Threads * kDeep) {
    uint4 x[kDeep], y[kDeep];
    int t[kDeep], h[kDeep], j[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const uint32_t i = i0 + k * Threads + threadIdx.x;
      t[k] = -1;
      if (i < all) {
        t[k] = quotient(i, jobs.a_token);
        const uint32_t in = i - t[k] * jobs.a_token.d;
        h[k] = quotient(in, jobs.a_head);
        j[k] = in - h[k] * jobs.a_head.d;
        const bool copied = j[k] >= jobs.turning;
        const uint16_t* src = from(t[k], h[k]);
        x[k] = *reinterpret_cast<const uint4*>(src + (copied ? dim - 8 * (int(jobs.a_head.d) - j[k]) : 8 * j[k]));
        if (!copied && !r.interleaved) y[k] = *reinterpret_cast<const uint4*>(src + 8 * j[k] + r.pairs);
      }
    }
    if (first) ready();
    first = false;
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      if (t[k] < 0) continue;
      uint16_t* dst = to(t[k], h[k]);
      if (!dst) continue;
      const Angle* a = angles + t[k] * r.pairs;
      if (j[k] >= jobs.turning) {
        *reinterpret_cast<uint4*>(dst + dim - 8 * (int(jobs.a_head.d) - j[k])) = x[k];
      } else if (r.interleaved) {
        *reinterpret_cast<uint4*>(dst + 8 * j[k]) = turn_neighbours(x[k], a, 4 * j[k], r.pairs);
      } else {
        turn_halves(x[k], y[k], a + 8 * j[k]);
        *reinterpret_cast<uint4*>(dst + 8 * j[k]) = x[k];
        *reinterpret_cast<uint4*>(dst + 8 * j[k] + r.pairs) = y[k];
      }
    }
  }
}

// Checks a tqkv_rope for heads of `dim` channels. TQKV_OK or the failure.
int32_t check(const tqkv_rope* rope, int32_t dim, Rope* out);

}  // namespace rope
}  // namespace tqkv

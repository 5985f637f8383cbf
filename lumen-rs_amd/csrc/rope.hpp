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

// The heads of a workgroup's tokens. A job is what one thread turns or copies
// at once: eight channels (neighbours, and channels behind the rotated ones),
// twice eight (halves that are whole pieces of eight) or single pairs and
// channels (other halves). from(t, h) and to(t, h): rows of token t and head
// h; to gives NULL where nothing is written. angles: [tokens][pairs] in LDS.
// A pair's two channels are read and written by one thread, so rows may turn
// in place.
template <int Threads, typename From, typename To>
__device__ __forceinline__ void turn_rows(const Rope& r, const Angle* angles, int tokens, int heads,
                                          int dim, bool copy, From from, To to) {
  const int rd = 2 * r.pairs;
  const bool singles = !r.interleaved && r.pairs % 8 != 0;
  const int turning = singles ? r.pairs : r.interleaved ? (rd + 7) / 8 : r.pairs / 8;
  const int behind = singles ? dim - rd : (dim - (r.interleaved ? turning * 8 : rd)) / 8;
  const int jobs = turning + (copy ? behind : 0);
  const int per_token = jobs * heads, all = per_token * tokens;
  for (int i = threadIdx.x; i < all; i += Threads) {
    const int t = i / per_token, h = i % per_token / jobs, j = i % jobs;
    uint16_t* dst = to(t, h);
    if (!dst) continue;
    const uint16_t* src = from(t, h);
    const Angle* a = angles + t * r.pairs;
    if (singles) {
      if (j < turning) {
        const float x = bf16_to_f32(src[j]), y = bf16_to_f32(src[j + r.pairs]);
        dst[j] = f32_to_bf16(turned_x(x, y, a[j]));
        dst[j + r.pairs] = f32_to_bf16(turned_y(x, y, a[j]));
      } else {
        dst[rd + j - turning] = src[rd + j - turning];
      }
    } else if (j >= turning) {
      const int c = dim - 8 * (jobs - j);
      *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
    } else if (r.interleaved) {
      const uint4 x = *reinterpret_cast<const uint4*>(src + 8 * j);
      *reinterpret_cast<uint4*>(dst + 8 * j) = turn_neighbours(x, a, 4 * j, r.pairs);
    } else {
      uint4 x = *reinterpret_cast<const uint4*>(src + 8 * j);
      uint4 y = *reinterpret_cast<const uint4*>(src + 8 * j + r.pairs);
      turn_halves(x, y, a + 8 * j);
      *reinterpret_cast<uint4*>(dst + 8 * j) = x;
      *reinterpret_cast<uint4*>(dst + 8 * j + r.pairs) = y;
    }
  }
}

// Checks a tqkv_rope for heads of `dim` channels. TQKV_OK or the failure.
int32_t check(const tqkv_rope* rope, int32_t dim, Rope* out);

}  // namespace rope
}  // namespace tqkv

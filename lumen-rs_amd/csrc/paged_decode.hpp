// Decode attention over a paged cache: one new token a sequence.
//
// o = sum_t p_t v_t with p = softmax(scale q.k_t): one pass over the rows with
// a running maximum and sum. The rows of the whole batch, in blocks of 16, are
// laid end to end and divided evenly among the W workgroups of a KV head, from
// lens on the device: a long sequence spreads over many
// workgroups and a workgroup may take several short ones. A workgroup's part
// of one sequence is a segment; it leaves the segment's output, maximum and
// sum in slot (workgroup + sequence), which no other segment shares (along
// the row order both only grow and one always does), unless the segment is
// the whole sequence. The second launch joins the slots.
//
// A wavefront takes every fourth step (32 rows, or 16 for wide rows) of the
// segment, on the matrix cores with the query heads of the KV head as the 16 columns:
//   S[row][head] = K Q^T  (A: lane l holds row l % 16 and 8 channels of
//     quarter l / 16; a product a 16 rows), so lane l ends up with head
//     l % 16 and rows 4 (l / 16) + i of each half;
//   O^T[channel][head] += V^T P^T: the eight weights that lane l just
//     computed are the operand it has to supply (rows as the contraction, in
//     an order that V's loads follow), so P never leaves the lane, and the
//     running maximum, sum and rescaling are the lane's own.
// V's operand is a channel's eight rows: a lane loads 8 (4 at D = 64)
// consecutive channels of its eight rows and pairs rows by byte permutes.
// bf16 rows take the weights as a bf16 pair hi + lo, 16 bits, so their rounding
// stays below the bf16 output's; the softmax sum is of the unrounded f32
// weights.
//
// Affine rows: scores use the codes themselves as f16 subnormals (one AND a
// pair; the queries enter as f16 in a unit of their own), one product a group,
// s = sum_g scale_g (q.c)_g + bias_g sum(q_g), and the bias part of all groups
// is one more product, of the biases as they lie and the query sums in three
// bf16 parts. Values are dequantized by one mixed multiply-add a code, f32 to
// f16 in a unit of the wavefront's, and weights enter as f16 too (each
// rounded by at most 2^-11 of itself, an eighth of the output's own rounding).
// Where a wavefront's values are of magnitudes too far apart for f16, it goes
// over its rows once more and takes values and weights as bf16 pairs.
//
// Bound by HBM: the live rows once. At G heads of 16 the matrix cores do
// 16 / G times the work that is needed and are still far from busy (4 to 20%).
// Measured, with the join: bf16, 131,071 rows x 8 KV heads at D = 128 (537 MB)
// 86 us, 6.2 TB/s; 4 bits, 16 x 32,768 x 8 at D = 256 (1.21 GB) 244 us, 5.0
// TB/s, where unpacking keeps the vector units 74% busy. Short calls are bound
// by latencies: 777 rows take 7.2 us and the join's 2.8.
#pragma once

#include <type_traits>

#include "paged.hpp"

namespace tqkv {
namespace paged {

constexpr int kWaves = 4;
constexpr int kUnit = 16;     // rows by which the batch is divided

struct DecodeArgs {
  Pool pool;
  const void* slot[6];
  const uint16_t* q;
  int64_t qstride;
  uint16_t* out;
  int H, G, groups16;  // query heads, of a KV head, 16-head sets of those
  int max_rows, window;
  int W;               // workgroups a (KV head, set)
  int over;            // units that a sequence's start counts as
  int least;           // units of a workgroup
  int kept_units;      // bf16 rows beyond these are streamed
  float scale_log2;
  float* part_o;  // [W + batch, H, D]
  float* part_m;  // [W + batch, H]: log2 units
  float* part_l;
  int32_t* starts;  // [batch + 1]: units before each sequence, all; for the join
  float* scores;  // [batch, H, srows] log2 units, or NULL
  int64_t srows;
};

// The rows of sequence b: n held, attended from the window's first, and its
// units, which the batch is divided by: 16-row blocks and `over` for starting
// on it.
struct Span {
  int n, lo, blocks, units;
};
__device__ __forceinline__ Span span_of_rows(const DecodeArgs& a, int n) {
  const int lo = a.window > 0 && n > a.window ? n - a.window : 0;
  const int blocks = n > 0 ? (n + kUnit - 1) / kUnit - lo / kUnit : 0;
  return {n, lo, blocks, n > 0 ? blocks + a.over : 0};
}
__device__ __forceinline__ Span span_of(const DecodeArgs& a, int b) {
  return span_of_rows(a, held(a.pool, b, a.max_rows < a.pool.cap ? a.max_rows : a.pool.cap));
}

// Units a workgroup takes of `total`.
__device__ __forceinline__ int units_per_wg(const DecodeArgs& a, int total) {
  const int per = (total + a.W - 1) / a.W;
  return per < a.least ? a.least : per;
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bf16x8 as_bf16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint4 x = make_uint4(a, b, c, d);
  return __builtin_bit_cast(bf16x8, x);
}
__device__ __forceinline__ floatx4 mfma(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// (lo half of a, lo half of b) and (hi half of a, hi half of b).
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
// bf16 of two f32, to nearest even, as a word (a in the low half).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const floatx2 x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}
__device__ __forceinline__ float low_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_f32(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Loads of the stream are buffer loads at a wavefront-uniform base (scalar
// registers) plus a 32-bit lane offset plus a constant. With plain pointers the
// compiler keeps a 64-bit lane address a load across the loop, tens of
// registers.
typedef __amdgpu_buffer_rsrc_t rsrc;
__device__ __forceinline__ rsrc uniform(const void* p, int64_t offset) {
  uint64_t x = reinterpret_cast<uint64_t>(p) + uint64_t(offset);
  x = uint32_t(__builtin_amdgcn_readfirstlane(int(x))) |
      uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(x >> 32)))) << 32;
  asm("" : "+s"(x));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(x), 0, 0x40000000, 0x00027000);
}

// Cache policies. Streaming past the caches pays where one load takes whole
// 64-byte pieces; with 4-bit codes several loads share a line (16 x 32,768
// rows at D = 256: 240 us kept, 308 streamed).
constexpr int kKeep = 0, kStream = 2;
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

// A load of N bytes (4, 8 or a multiple of 16) into words.
template <int N, int kPolicy = kKeep>
__device__ __forceinline__ void load_words(rsrc base, uint32_t off, uint32_t* w) {
  if constexpr (N == 4) {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(base, off, 0, kPolicy);
  } else if constexpr (N == 8) {
    const uintx2 x = __builtin_amdgcn_raw_buffer_load_b64(base, off, 0, kPolicy);
    w[0] = x.x;
    w[1] = x.y;
  } else {
    static_assert(N % 16 == 0, "whole 16-byte loads");
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const uintx4 x = __builtin_amdgcn_raw_buffer_load_b128(base, off + 16 * i, 0, kPolicy);
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  }
}

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ halfx8 as_halfx8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint4 x = make_uint4(a, b, c, d);
  return __builtin_bit_cast(halfx8, x);
}

// Output += V^T P^T over a step's rows, 8 rows a lane (two halves) or 4, of
// bf16 or f16 operands.
template <int HALVES, bool F16>
__device__ __forceinline__ floatx4 mfma_pv(const uint32_t (&v)[2 * HALVES],
                                           const uint32_t (&p)[2 * HALVES], floatx4 c) {
  if constexpr (HALVES == 2 && F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(as_halfx8(v[0], v[1], v[2], v[3]),
                                                  as_halfx8(p[0], p[1], p[2], p[3]), c, 0, 0, 0);
  } else if constexpr (HALVES == 2) {
    return mfma(as_bf16x8(v[0], v[1], v[2], v[3]), as_bf16x8(p[0], p[1], p[2], p[3]), c);
  } else {
    const uint2 x = make_uint2(v[0], v[1]), y = make_uint2(p[0], p[1]);
    if constexpr (F16)
      return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(halfx4, x),
                                                   __builtin_bit_cast(halfx4, y), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(shortx4, x),
                                                       __builtin_bit_cast(shortx4, y), c, 0, 0, 0);
  }
}

// The lane, counted anew: a thread index kept for its rare uses would be spilled,
// and every reload waits for the loads before it.
__device__ __forceinline__ int lane_anew() {
  uint32_t all = ~0u;
  asm volatile("" : "+s"(all));
  return int(__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0)));
}

// The pages of a wavefront's coming steps: a block of table entries in LDS,
// its own, filled when a step asks for an entry behind it. (An entry loaded
// when its step needs it, or one block in registers ahead of the next, makes
// the step wait for every load before it, its own values' too.)
constexpr int kBlock = 256;
struct Pages {
  const int32_t* table;
  int32_t* block;  // LDS, kBlock entries of the wavefront's
  int most;        // entries that may be read
  int first;       // entry of block[0]
  __device__ __forceinline__ void fill(int at) {
    first = at;
    const int me = lane_anew();
#pragma unroll
    for (int i = 0; i < kBlock / 64; ++i) {
      const int lane = 64 * i + me;
      block[lane] = at + lane < most ? table[at + lane] : -1;
    }
    __builtin_amdgcn_wave_barrier();
  }
  __device__ __forceinline__ void start(int32_t* lds, const int32_t* t, int n, int at) {
    table = t;
    block = lds;
    most = n;
    fill(at);
  }
  // Entry i, not below those asked for before.
  __device__ __forceinline__ int entry(int i) {
    if (i >= first + kBlock) fill(i);
    return __builtin_amdgcn_readfirstlane(block[i - first]);
  }
};

// The pool rows of a step's 16-row halves (uniform over the wavefront).
template <int HALVES>
struct Step {
  int64_t row[HALVES];  // pool row of the half's first row
  bool ok[HALVES];
};
template <int HALVES>
__device__ __forceinline__ Step<HALVES> step_of(const Pool& p, Pages& pages, int kvh, int row,
                                                int end) {
  Step<HALVES> h;
#pragma unroll
  for (int s = 0; s < HALVES; ++s) {
    const int r = row + s * 16;
    const int page = r < end ? pages.entry(r >> p.shift) : -1;
    h.ok[s] = page >= 0 && page < p.num_pages;
    h.row[s] = pool_row(p, h.ok[s] ? page : 0, kvh, h.ok[s] ? r & ((1 << p.shift) - 1) : 0);
  }
  return h;
}

// Two weights as bf16 words hi + lo, 16 bits of each: hi the upper bits, and
// lo the rest and 2^-23 of the weight. Both parts of a weight above 0 are above
// 0, so that an infinite value times each is infinite and not NaN.
__device__ __forceinline__ void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  hi = highs(__float_as_uint(p0), __float_as_uint(p1));
  lo = pack_bf16(fmaf(p0, 1.0f + 0x1p-23f, -low_f32(hi)), fmaf(p1, 1.0f + 0x1p-23f, -high_f32(hi)));
}

// Channel layout of the values: product j's output row r is channel
// (j / kCpl) * 16 kCpl + r * kCpl + j % kCpl.
template <int D>
struct Chan {
  static constexpr int kCpl = D >= 128 ? 8 : 4;      // consecutive channels a lane and piece
  static constexpr int kPieces = D / (16 * kCpl);
  static constexpr int kJ = D / 16;                  // products (and accumulators)
};

// ---------------------------------------------------------------- bf16 rows
// POLICY: of the rows' loads; the launched kernel holds both and chooses.
template <int D, int POLICY = kStream>
struct Bf16Rows {
  static constexpr int kD = D;
  static constexpr bool kChooses = true;
  typedef Bf16Rows<D, kKeep> Kept;
  static constexpr int kHalves = D <= 128 ? 2 : 1;
  static constexpr int kOcc = 2;  // wavefronts a SIMD that there are registers for
  using C = Chan<D>;
  using S = Step<kHalves>;
  static constexpr int kChunks = D / 32;
  static constexpr int kVWords = C::kPieces * C::kCpl / 2;
  typedef bf16x8 Operand;
  static constexpr int kOperands = kChunks;
  struct Rest {   // of the queries, beside their operands
    float mul;    // of a score: positive
  };
  struct K {
    uint32_t w[kHalves][kChunks * 4];
  };
  struct V {
    uint32_t w[4 * kHalves][kVWords];
  };

  // Channels of (chunk, quarter): 32 chunk + 8 quarter.
  // A head's queries: lanes without a head load the first one's (no branch
  // between the loads), and prepare() clears them.
  static __device__ __forceinline__ void load_q(uint32_t (&w)[D / 32][4], rsrc p, bool live, int r,
                                                int g) {
    const uint32_t off = (live ? r : 0) * (2 * D) + g * 16;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) load_words<16>(p, off + c * 64, w[c]);
  }
  static __device__ __forceinline__ void prepare(Operand (&op)[kOperands], Rest& q,
                                                 const uint32_t (&w)[D / 32][4], bool live, int,
                                                 float scale_log2) {
    // The scale's sign goes into the queries, and its power of two if it makes
    // them smaller (both exact): products stay within f32 where scores do.
    const uint32_t keep = live && scale_log2 != 0.0f ? 0xffffffffu : 0u;
    int e = int(__float_as_uint(scale_log2) >> 23 & 255) - 127;
    e = e > 0 ? 0 : e < -64 ? -64 : e;
    const float times = ldexpf(scale_log2 < 0.0f ? -1.0f : 1.0f, e);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      uint32_t x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t y = w[c][i] & keep;
        x[i] = highs(__float_as_uint(low_f32(y) * times), __float_as_uint(high_f32(y) * times));
      }
      op[c] = as_bf16x8(x[0], x[1], x[2], x[3]);
    }
    q.mul = scale_log2 != 0.0f ? ldexpf(fabsf(scale_log2), -e) : 1.0f;
  }
  static __device__ __forceinline__ void load_k(K& k, const DecodeArgs& a, const S& h, int r,
                                                int g) {
    const uint32_t off = r * (2 * D) + g * 16;
#pragma unroll
    for (int s = 0; s < kHalves; ++s) {
      const rsrc p = uniform(a.slot[0], h.row[s] * (2 * D));
#pragma unroll
      for (int c = 0; c < kChunks; ++c) load_words<16, POLICY>(p, off + c * 64, k.w[s] + 4 * c);
    }
  }
  static __device__ __forceinline__ void load_v(V& v, const DecodeArgs& a, const S& h, int r,
                                                int g) {
    const uint32_t off = 4 * g * (2 * D) + r * (2 * C::kCpl);
#pragma unroll
    for (int s = 0; s < kHalves; ++s) {
      const rsrc p = uniform(a.slot[1], h.row[s] * (2 * D));
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < C::kPieces; ++x)
          load_words<2 * C::kCpl, POLICY>(p, off + e * (2 * D) + x * 256, v.w[4 * s + e] + x * (C::kCpl / 2));
    }
  }
  // Scores of half s, to be multiplied by q.mul.
  // op(c): the queries' operand of product c.
  template <typename Op>
  static __device__ __forceinline__ floatx4 scores(Op&& op, const Rest&, const K& k, int s) {
    floatx4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      acc = mfma(as_bf16x8(k.w[s][4 * c], k.w[s][4 * c + 1], k.w[s][4 * c + 2], k.w[s][4 * c + 3]),
                 op(c), acc);
    return acc;
  }
  // The rows for which dead is set hold nothing: zero, whatever lies there.
  static __device__ __forceinline__ void clear(V& v, uint32_t dead, uint32_t) {
#pragma unroll
    for (int e = 0; e < 4 * kHalves; ++e)
#pragma unroll
      for (int i = 0; i < kVWords; ++i) v.w[e][i] = dead >> e & 1 ? 0 : v.w[e][i];
  }
  // Weights are held times 2^-40 (their sum too, so it cancels): 2^30 rows of
  // weight 2^kTau and values of bf16's largest magnitude stay within f32.
  // Weights below 2^-86 of the largest vanish.
  static constexpr float kDown = 40.0f, kLast = 1.0f;
  static constexpr bool kPairs = false;  // values are exact: no second pass
  struct Unit {  // of the accumulators
    __device__ __forceinline__ float of() const { return 1.0f; }
    __device__ __forceinline__ uint32_t filler() const { return 0; }
  };
  static __device__ __forceinline__ void accumulate(const V& v, const float (&p)[4 * kHalves],
                                                    floatx4 (&acc)[C::kJ], Unit&, int) {
    uint32_t hi[2 * kHalves], lw[2 * kHalves];
#pragma unroll
    for (int e = 0; e < 2 * kHalves; ++e) split(p[2 * e], p[2 * e + 1], hi[e], lw[e]);
#pragma unroll
    for (int i = 0; i < kVWords; ++i) {
      uint32_t x[2 * kHalves], y[2 * kHalves];
#pragma unroll
      for (int e = 0; e < 2 * kHalves; ++e) {
        x[e] = lows(v.w[2 * e][i], v.w[2 * e + 1][i]);
        y[e] = highs(v.w[2 * e][i], v.w[2 * e + 1][i]);
      }
      acc[2 * i] = mfma_pv<kHalves, false>(x, hi, acc[2 * i]);
      acc[2 * i] = mfma_pv<kHalves, false>(x, lw, acc[2 * i]);
      acc[2 * i + 1] = mfma_pv<kHalves, false>(y, hi, acc[2 * i + 1]);
      acc[2 * i + 1] = mfma_pv<kHalves, false>(y, lw, acc[2 * i + 1]);
    }
  }
  // The wide kernel's share of the values: the lane's 16 rows of a 64-row tile
  // at eight channels of the wavefront's 128.
  static constexpr int kWideOcc = 1;
  struct Wide {
    uint32_t w[16][4];
  };
  static __device__ __forceinline__ void load_wide(Wide& v, const DecodeArgs& a, const Step<4>& h,
                                                   int wave, int r, int g) {
    const uint32_t off = 4 * g * (2 * D) + wave * 256 + r * 16;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const rsrc p = uniform(a.slot[1], h.row[s] * (2 * D));
#pragma unroll
      for (int e = 0; e < 4; ++e) load_words<16, POLICY>(p, off + e * (2 * D), v.w[4 * s + e]);
    }
  }
  static __device__ __forceinline__ void clear_wide(Wide& v, uint32_t dead, uint32_t) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) v.w[e][i] = dead >> e & 1 ? 0 : v.w[e][i];
  }
  static __device__ __forceinline__ void accumulate_wide(const Wide& v, const float (&p)[16],
                                                         floatx4 (&acc)[8], Unit&, int, int) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t hi[4], lw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) split(p[8 * k + 2 * e], p[8 * k + 2 * e + 1], hi[e], lw[e]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = lows(v.w[8 * k + 2 * e][i], v.w[8 * k + 2 * e + 1][i]);
          y[e] = highs(v.w[8 * k + 2 * e][i], v.w[8 * k + 2 * e + 1][i]);
        }
        acc[2 * i] = mfma_pv<2, false>(x, hi, acc[2 * i]);
        acc[2 * i] = mfma_pv<2, false>(x, lw, acc[2 * i]);
        acc[2 * i + 1] = mfma_pv<2, false>(y, hi, acc[2 * i + 1]);
        acc[2 * i + 1] = mfma_pv<2, false>(y, lw, acc[2 * i + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// -------------------------------------------------------------- affine rows
template <int D, int BK, int BV, int GS>
struct AffineRows {
  static constexpr int kD = D;
  static constexpr bool kChooses = false;
  typedef AffineRows Kept;
  static constexpr int kHalves = D <= 128 ? 2 : 1;
  using C = Chan<D>;
  using S = Step<kHalves>;
  static constexpr int NG = D / GS;          // groups a row
  static constexpr int CPG = GS / 32;        // products a group
  static constexpr int kGroupBytes = GS / 4 * BK / 8;  // a lane's codes of a group
  static constexpr int kGroupWords = kGroupBytes / 4;
  static constexpr int kPieceBytes = C::kCpl * BV / 8;
  static constexpr int kPieceWords = (kPieceBytes + 3) / 4;
  static constexpr int kPieceLoad = kPieceBytes < 4 ? 4 : kPieceBytes;  // of two lanes at D = 64, 4 bits
  static constexpr int kKeyPolicy = kGroupBytes >= 16 ? kStream : kKeep;
  static constexpr int kValuePolicy = kPieceBytes >= 4 ? kStream : kKeep;
  static constexpr int kGpp = 16 * C::kCpl > GS ? 16 * C::kCpl / GS : 1;  // groups a piece
  static constexpr int kSets = (NG + 7) / 8;           // bias products
  // Loaded as whole words: two 16-bit loads would be packed into a register as
  // they arrive, a wait in the middle of the loads.
  static constexpr int kBiasBytes = NG == 1 ? 4 : 2 * NG < 16 ? 2 * NG : 16;
  typedef halfx8 Operand;
  static constexpr int kOperands = D / 32;
  struct Rest {
    bf16x8 sum[kSets];
    float mul;
  };
  struct K {
    uint32_t w[kHalves][NG * kGroupWords];
    uint32_t s[kHalves][2 * NG];     // scales of rows [4 g, 4 g + 4)
    uint32_t b[kHalves][kSets * 4];  // biases of row r
  };
  struct V {
    uint32_t w[4 * kHalves][C::kPieces * kPieceWords];
    uint32_t s[kHalves][2 * NG], b[kHalves][2 * NG];  // of rows [4 g, 4 g + 4)
  };

  // Wavefronts a SIMD: by the registers that live across a step, so that none
  // of them spill in the loop.
  static constexpr int kLive = kHalves * (NG * kGroupWords + 2 * NG + (NG + 1) / 2) +
                               4 * kHalves * C::kPieces * kPieceWords + kHalves * 4 * NG + 4 * C::kJ +
                               D / 8 + 4 * kSets + 1;
  static constexpr int kOcc = kLive <= 64 ? 4 : kLive <= 100 ? 3 : kLive <= 165 ? 2 : 1;

  // The f16 pairs of eight codes, as subnormals c 2^-24 (4-bit codes with an
  // odd place in their half word: c 2^-20): one AND a pair. 4 bits: codes
  // (0,4) (1,5)* (2,6) (3,7)*; 8 bits: (0,2) (1,3) (4,6) (5,7).
  static __device__ __forceinline__ halfx8 unpack(const uint32_t* w) {
    if constexpr (BK == 4) {
      const uint32_t x = w[0], y = x >> 8;
      return as_halfx8(x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u);
    } else {
      return as_halfx8(w[0] & 0x00ff00ffu, (w[0] >> 8) & 0x00ff00ffu, w[1] & 0x00ff00ffu,
                       (w[1] >> 8) & 0x00ff00ffu);
    }
  }
  // Queries as f16 times 2^(14 - E), E the head's largest exponent (so they
  // lie below 2^15; channels below 2^-27 of the largest lose bits), in unpack's
  // order; the sums of the groups in the same unit as three bf16 parts, which
  // hold all bits of an f32, one a quarter. Channels of (group, quarter):
  // group GS + quarter GS / 4, then in order.
  static __device__ __forceinline__ void load_q(uint32_t (&w)[D / 32][4], rsrc p, bool live, int r,
                                                int g) {
    const uint32_t off = (live ? r : 0) * (2 * D) + g * (GS / 2);
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
      load_words<16>(p, off + c / CPG * (2 * GS) + c % CPG * 16, w[c]);
  }
  static __device__ __forceinline__ void prepare(Operand (&op)[kOperands], Rest& q,
                                                 uint32_t (&w)[D / 32][4], bool live, int g,
                                                 float scale_log2) {
    const uint32_t keep = live && scale_log2 != 0.0f ? 0xffffffffu : 0u;
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[c][i] &= keep;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top = fmaxf(top, fmaxf(fabsf(low_f32(w[c][i])), fabsf(high_f32(w[c][i]))));
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int E = int(__float_as_uint(top) >> 23) - 127;
    E = E < -100 ? -100 : E;
    // The scale's sign goes into the queries.
    const float up = __uint_as_float(uint32_t(127 + 14 - E) << 23) * (scale_log2 < 0.0f ? -1.0f : 1.0f);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = low_f32(w[c][i]) * up;
        x[2 * i + 1] = high_f32(w[c][i]) * up;
      }
      halfx8 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int lo = BK == 4 ? i : i / 2 * 4 + i % 2, hi = lo + (BK == 4 ? 4 : 2);
        const float down = BK == 4 && i % 2 ? 0x1p-4f : 1.0f;
        o[2 * i] = _Float16(x[lo] * down);
        o[2 * i + 1] = _Float16(x[hi] * down);
      }
      op[c] = o;
    }
#pragma unroll
    for (int n = 0; n < 8 * kSets; ++n) {
      float sum = 0.0f;
      if (n < NG) {
#pragma unroll
        for (int c = n * CPG; c < (n + 1) * CPG; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += low_f32(w[c][i]) + high_f32(w[c][i]);
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        sum *= up * 0x1p-24f;
      }
      const float hi = __bf16(sum), mid = __bf16(sum - hi), lo = __bf16(sum - hi - mid);
      q.sum[n / 8][n % 8] = __bf16(g == 0 ? hi : g == 1 ? mid : g == 2 ? lo : 0.0f);
    }
    // Above 0: masked scores are -inf times it. Finite: queries above 2^90 only
    // have their scores' differences understated, and these decide at 2^100 too.
    q.mul = scale_log2 != 0.0f
                ? fminf(fmaxf(ldexpf(fabsf(scale_log2), E + 10), 0x1p-126f), 0x1p100f)
                : 1.0f;
  }
  static __device__ __forceinline__ void load_k(K& k, const DecodeArgs& a, const S& h, int r,
                                                int g) {
    const uint32_t off = r * (D * BK / 8) + g * kGroupBytes;
    const uint32_t soff = g * (8 * NG), boff = r * (2 * NG) & ~3u;
#pragma unroll
    for (int s = 0; s < kHalves; ++s) {
      const rsrc p = uniform(a.slot[0], h.row[s] * (D * BK / 8));
#pragma unroll
      for (int n = 0; n < NG; ++n)
        load_words<kGroupBytes, kKeyPolicy>(p, off + n * (GS * BK / 8), k.w[s] + n * kGroupWords);
      load_words<8 * NG>(uniform(a.slot[1], h.row[s] * (2 * NG)), soff, k.s[s]);
      const rsrc b = uniform(a.slot[2], h.row[s] * (2 * NG));
#pragma unroll
      for (int i = 0; i < kSets; ++i) load_words<kBiasBytes>(b, boff + 16 * i, k.b[s] + 4 * i);
    }
  }
  static __device__ __forceinline__ void load_v(V& v, const DecodeArgs& a, const S& h, int r,
                                                int g) {
    const uint32_t off = 4 * g * (D * BV / 8) + (r * kPieceBytes & ~3), soff = g * (8 * NG);
#pragma unroll
    for (int s = 0; s < kHalves; ++s) {
      const rsrc p = uniform(a.slot[3], h.row[s] * (D * BV / 8));
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < C::kPieces; ++x)
          load_words<kPieceLoad, kValuePolicy>(p, off + e * (D * BV / 8) + x * (16 * kPieceBytes),
                                  v.w[4 * s + e] + x * kPieceWords);
      load_words<8 * NG>(uniform(a.slot[4], h.row[s] * (2 * NG)), soff, v.s[s]);
      load_words<8 * NG>(uniform(a.slot[5], h.row[s] * (2 * NG)), soff, v.b[s]);
    }
  }
  // The f32 of entry (row i of four, group n) of four rows' scales.
  static __device__ __forceinline__ float entry(const uint32_t* w, int i, int n) {
    const int at = i * NG + n;
    return at % 2 ? high_f32(w[at / 2]) : low_f32(w[at / 2]);
  }
  // The biases' part of all groups in a product, then a scale a group.
  template <typename Op>
  static __device__ __forceinline__ floatx4 scores(Op&& op, const Rest& q, const K& k, int s) {
    floatx4 out = {0, 0, 0, 0};
    const int odd = NG == 1 ? threadIdx.x & 1 : 0;  // row r's half of a word of two rows
#pragma unroll
    for (int i = 0; i < kSets; ++i) {
      uint32_t b[4] = {0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < kBiasBytes / 4; ++x) b[x] = k.b[s][4 * i + x];
      if (NG == 1) b[0] = (b[0] >> (16 * odd)) & 0xffffu;
      out = mfma(as_bf16x8(b[0], b[1], b[2], b[3]), q.sum[i], out);
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      floatx4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < CPG; ++c)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(unpack(k.w[s] + n * kGroupWords + c * (BK / 4)),
                                                     op(n * CPG + c), acc, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = fmaf(entry(k.s[s], i, n), acc[i], out[i]);
    }
    return out;
  }
  // Dead rows: a scale of 0, and the unit's filler for a bias (their weights
  // are 0).
  static __device__ __forceinline__ void clear(V& v, uint32_t dead, uint32_t filler) {
#pragma unroll
    for (int e = 0; e < 4 * kHalves; ++e) {
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const int at = e % 4 * NG + n;
        const uint32_t keep = dead >> e & 1 ? (at % 2 ? 0x0000ffffu : 0xffff0000u) : 0xffffffffu;
        v.s[e / 4][at / 2] &= keep;
        v.b[e / 4][at / 2] = (v.b[e / 4][at / 2] & keep) | (filler & ~keep);
      }
    }
  }
  // The f32 of (row e, the lane's group of piece x): sel picks the lane's
  // half word of the piece's (at most four groups) by one byte permute.
  static __device__ __forceinline__ float lane_entry(const uint32_t* w, int e, int x, uint32_t sel) {
    const int first = e % 4 * NG + x * (16 * C::kCpl) / GS;
    if constexpr (kGpp == 1) {
      return first % 2 ? high_f32(w[first / 2]) : low_f32(w[first / 2]);
    } else if constexpr (kGpp == 2) {
      return __uint_as_float(__builtin_amdgcn_perm(0u, w[first / 2], sel));
    } else {
      return __uint_as_float(__builtin_amdgcn_perm(w[first / 2 + 1], w[first / 2], sel));
    }
  }
  // Channel j of a row's piece: scale * code + bias, as f16 one mixed
  // multiply-add. s24: the scale times 2^24 (2^20 for a code with an odd place
  // in its half word).
  static __device__ __forceinline__ _Float16 value(const uint32_t* w, int shift, int j, float s24,
                                                   float s20, float b) {
    uint32_t x;
    int half;
    if constexpr (BV == 4) {
      x = ((w[j / 8] >> shift) >> (j & 2 ? 8 : 0)) & (j & 1 ? 0x00f000f0u : 0x000f000fu);
      half = j % 8 / 4;
    } else {
      x = (w[j / 4] >> (j & 1 ? 8 : 0)) & 0x00ff00ffu;
      half = j % 4 / 2;
    }
    return _Float16(fmaf(float(__builtin_bit_cast(halfx2, x)[half]), BV == 4 && (j & 1) ? s20 : s24, b));
  }
  // The same in f32, of any magnitude.
  static __device__ __forceinline__ float plain_value(const uint32_t* w, int shift, int j, float s,
                                                      float b) {
    const uint32_t code = BV == 4 ? w[j / 8] >> (shift + 4 * (j % 8)) & 0xfu : w[j / 4] >> (8 * (j % 4)) & 0xffu;
    return fmaf(float(code), s, b);
  }
  // Weights are held times 2^7: they reach 2^(7 + kTau) in f16, and those that
  // f16 loses lie below 2^-32 of the largest, 2^-15 in all at 2^17 rows. At a
  // segment's end they and their sum go down by 2^-47, to bf16 rows' 2^-40.
  static constexpr float kDown = -7.0f, kLast = 0x1p-47f;
  // The accumulators hold values times `up`, a power of two, the wavefront's.
  // A bound on the values of a row's group is its scale times the largest code,
  // plus its bias. The unit puts a bound of the first rows that are not all 0 at
  // 2^4. As long as all bounds lie within 2^-4 and 2^12, each f16 value is off by
  // at most 2^-11 of itself or 2^-21 of its bound, none overflows, and no row is
  // so much larger than another that what f16 loses of its weight would matter
  // to the other's. Otherwise (infinite bounds too) the sums are given up, and
  // the second pass makes them: calls with such rows in every wavefront's part
  // take 1.5 to 2.3 times as long (16 x 16,384 rows of 4 bits at D = 128: 147 us
  // for 80). Pairs in the loop itself spilled, and cost every call (32 sequences
  // of 17 to 16,000 rows: 57 us for 39).
  static constexpr bool kPairs = true;
  struct Unit {
    float up = 1.0f;
    float low = INFINITY, high = 0.0f;  // 2^-4 and 2^12 in this unit; none yet
    int given_up = 0;
    __device__ __forceinline__ float of() const { return kLast / up; }
    // A scalar, and so a branch: in lanes masked off matrix products run all the
    // same.
    __device__ __forceinline__ bool gave_up() const {
      return __builtin_amdgcn_readfirstlane(given_up) != 0;
    }
    // Two bf16 of 1 in this unit (0 without one): biases of rows that hold
    // nothing, within the bounds.
    __device__ __forceinline__ uint32_t filler() const {
      const uint32_t one = __float_as_uint(low * 0x1p4f);
      return low == INFINITY ? 0 : one | one >> 16;
    }
    // The unit for a step's groups. (Without shuffles: the first rows of every
    // segment come through its second half. A NaN passes: it stays in its
    // channel.)
    template <int M, int N>
    __device__ __forceinline__ void admit(const float (&s)[M], const float (&b)[M],
                                          const floatx4 (&acc)[N]) {
      float bound[M], most = 0.0f, least = INFINITY;
#pragma unroll
      for (int e = 0; e < M; ++e) {
        bound[e] = fmaf(fabsf(s[e]), float((1 << BV) - 1), fabsf(b[e]));
        most = fmaxf(most, bound[e]);
        least = fminf(least, bound[e]);
      }
      if (__builtin_expect(!__any(least < low || most > high), 1)) return;
      const uint64_t some = __ballot(most > 0.0f);
      if (some == 0) return;  // rows of 0 alone
      bool empty = true;
      if (low < INFINITY) {  // rows of zeros, stored as steps of 1e-7, leave the choice open
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) empty &= acc[j][i] == 0.0f;
      }
      if (__all(empty)) {
        const uint32_t first = __builtin_amdgcn_readlane(__float_as_uint(most), __builtin_ctzll(some));
        int E = int(first >> 23) - 127 - 4;
        E = E < -94 ? -94 : E > 96 ? 96 : E;  // up * 2^24 and low stay normal
        up = __uint_as_float(uint32_t(127 - E) << 23);
        low = __uint_as_float(uint32_t(127 - 4 + E) << 23);
        high = __uint_as_float(uint32_t(127 + 12 + E) << 23);
      }
      bool out = most > high;
#pragma unroll
      for (int e = 0; e < M; ++e) out |= bound[e] > 0.0f && bound[e] < low;
      if (__any(out)) given_up = 1;
    }
  };
  static __device__ __forceinline__ void accumulate(const V& v, const float (&p)[4 * kHalves],
                                                    floatx4 (&acc)[C::kJ], Unit& unit, int r) {
    const int shift = kPieceBytes < 4 ? 16 * (r & 1) : 0;
    uint32_t pw[2 * kHalves];
#pragma unroll
    for (int e = 0; e < 2 * kHalves; ++e) {
      const floatx2 x = {p[2 * e], p[2 * e + 1]};
      pw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, halfx2));
    }
    const uint32_t grp = r * C::kCpl / GS;  // the lane's group of a piece
    const uint32_t sel = ((2 * grp + 1) << 24) | ((2 * grp) << 16) | 0x0c0cu;
#pragma unroll
    for (int x = 0; x < C::kPieces; ++x) {
      float s[4 * kHalves], b[4 * kHalves];
#pragma unroll
      for (int e = 0; e < 4 * kHalves; ++e) {
        s[e] = lane_entry(v.s[e / 4], e, x, sel);
        b[e] = lane_entry(v.b[e / 4], e, x, sel);
      }
      unit.admit(s, b, acc);
      const float up24 = unit.up * 0x1p24f;
      float s20[4 * kHalves];
#pragma unroll
      for (int e = 0; e < 4 * kHalves; ++e) {
        s[e] *= up24;
        s20[e] = s[e] * 0x1p-4f;
        b[e] *= unit.up;
      }
#pragma unroll
      for (int j = 0; j < C::kCpl; ++j) {
        uint32_t o[2 * kHalves];
#pragma unroll
        for (int e = 0; e < 2 * kHalves; ++e) {
          const halfx2 y = {
              value(v.w[2 * e] + x * kPieceWords, shift, j, s[2 * e], s20[2 * e], b[2 * e]),
              value(v.w[2 * e + 1] + x * kPieceWords, shift, j, s[2 * e + 1], s20[2 * e + 1],
                    b[2 * e + 1])};
          o[e] = __builtin_bit_cast(uint32_t, y);
        }
        acc[x * C::kCpl + j] = mfma_pv<kHalves, true>(o, pw, acc[x * C::kCpl + j]);
        if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // The second pass: values and weights as bf16 pairs, hi + lo, 16 bits of each
  // (an infinite value is its hi alone), in the unit of bf16 rows' sums.
  static __device__ __forceinline__ void split_values(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = highs(__float_as_uint(x), __float_as_uint(y));
    const float a = x - low_f32(hi), b = y - high_f32(hi);
    lo = pack_bf16(fabsf(x) < INFINITY ? a : 0.0f, fabsf(y) < INFINITY ? b : 0.0f);
  }
  template <int HALVES>
  struct Weights {
    uint32_t hi[2 * HALVES], lo[2 * HALVES];
  };
  template <int HALVES>
  static __device__ __forceinline__ Weights<HALVES> weights_of(const float* p) {
    Weights<HALVES> w;
#pragma unroll
    for (int e = 0; e < 2 * HALVES; ++e) split(p[2 * e] * kLast, p[2 * e + 1] * kLast, w.hi[e], w.lo[e]);
    return w;
  }
  template <int HALVES, typename Value>
  static __device__ __forceinline__ floatx4 pairs(Value&& value_of, const Weights<HALVES>& w, floatx4 acc) {
    uint32_t hi[2 * HALVES], lo[2 * HALVES];
#pragma unroll
    for (int e = 0; e < 2 * HALVES; ++e) split_values(value_of(2 * e), value_of(2 * e + 1), hi[e], lo[e]);
    acc = mfma_pv<HALVES, false>(hi, w.hi, acc);
    acc = mfma_pv<HALVES, false>(hi, w.lo, acc);
    return mfma_pv<HALVES, false>(lo, w.hi, acc);
  }
  static __device__ __forceinline__ void accumulate_pairs(const V& v, const float (&p)[4 * kHalves],
                                                          floatx4 (&acc)[C::kJ], int r) {
    const int shift = kPieceBytes < 4 ? 16 * (r & 1) : 0;
    const uint32_t grp = r * C::kCpl / GS;
    const uint32_t sel = ((2 * grp + 1) << 24) | ((2 * grp) << 16) | 0x0c0cu;
    const Weights<kHalves> w = weights_of<kHalves>(p);
#pragma unroll
    for (int x = 0; x < C::kPieces; ++x)
#pragma unroll
      for (int j = 0; j < C::kCpl; ++j) {
        acc[x * C::kCpl + j] = pairs<kHalves>(
            [&](int e) {
              const float s = lane_entry(v.s[e / 4], e, x, sel), b = lane_entry(v.b[e / 4], e, x, sel);
              return plain_value(v.w[e] + x * kPieceWords, shift, j, s, b);
            },
            w, acc[x * C::kCpl + j]);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  // The wide kernel's share of the values, as Bf16Rows': codes, and the scale
  // and bias of the lane's own group of each row.
  static constexpr int kWideOcc = NG <= 8 ? 2 : 1;  // groups of 32 would spill
  struct Wide {
    uint32_t w[16][kPieceWords];
    uint32_t s[16], b[16];  // words that hold the group's bf16
  };
  static __device__ __forceinline__ void load_wide(Wide& v, const DecodeArgs& a, const Step<4>& h,
                                                   int wave, int r, int g) {
    const uint32_t off = 4 * g * (D * BV / 8) + (16 * wave + r) * kPieceBytes;
    const uint32_t soff = 4 * g * (2 * NG) + ((128 * wave + 8 * r) / GS * 2 & ~3);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const rsrc p = uniform(a.slot[3], h.row[s] * (D * BV / 8));
      const rsrc ps = uniform(a.slot[4], h.row[s] * (2 * NG));
      const rsrc pb = uniform(a.slot[5], h.row[s] * (2 * NG));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        load_words<kPieceBytes, kValuePolicy>(p, off + e * (D * BV / 8), v.w[4 * s + e]);
        load_words<4>(ps, soff + e * (2 * NG), &v.s[4 * s + e]);
        load_words<4>(pb, soff + e * (2 * NG), &v.b[4 * s + e]);
      }
    }
  }
  static __device__ __forceinline__ void clear_wide(Wide& v, uint32_t dead, uint32_t filler) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      v.s[e] = dead >> e & 1 ? 0 : v.s[e];
      v.b[e] = dead >> e & 1 ? filler : v.b[e];
    }
  }
  static __device__ __forceinline__ void accumulate_wide(const Wide& v, const float (&p)[16],
                                                         floatx4 (&acc)[8], Unit& unit, int wave,
                                                         int r) {
    const uint32_t half = (128 * wave + 8 * r) / GS & 1;  // the group's place in its word
    const uint32_t sel = ((2 * half + 1) << 24) | ((2 * half) << 16) | 0x0c0cu;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t pw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const floatx2 x = {p[8 * k + 2 * e], p[8 * k + 2 * e + 1]};
        pw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, halfx2));
      }
      float s[8], s20[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[e] = __uint_as_float(__builtin_amdgcn_perm(0u, v.s[8 * k + e], sel));
        b[e] = __uint_as_float(__builtin_amdgcn_perm(0u, v.b[8 * k + e], sel));
      }
      unit.admit(s, b, acc);
      const float up24 = unit.up * 0x1p24f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[e] *= up24;
        s20[e] = s[e] * 0x1p-4f;
        b[e] *= unit.up;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const halfx2 y = {value(v.w[8 * k + 2 * e], 0, j, s[2 * e], s20[2 * e], b[2 * e]),
                            value(v.w[8 * k + 2 * e + 1], 0, j, s[2 * e + 1], s20[2 * e + 1],
                                  b[2 * e + 1])};
          o[e] = __builtin_bit_cast(uint32_t, y);
        }
        acc[j] = mfma_pv<2, true>(o, pw, acc[j]);
        if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  static __device__ __forceinline__ void accumulate_wide_pairs(const Wide& v, const float (&p)[16],
                                                               floatx4 (&acc)[8], int wave, int r) {
    const uint32_t half = (128 * wave + 8 * r) / GS & 1;
    const uint32_t sel = ((2 * half + 1) << 24) | ((2 * half) << 16) | 0x0c0cu;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Weights<2> w = weights_of<2>(p + 8 * k);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[j] = pairs<2>(
            [&](int e) {
              const float s = __uint_as_float(__builtin_amdgcn_perm(0u, v.s[8 * k + e], sel));
              const float b = __uint_as_float(__builtin_amdgcn_perm(0u, v.b[8 * k + e], sel));
              return plain_value(v.w[8 * k + e], 0, j, s, b);
            },
            w, acc[j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// ------------------------------------------------------------------- kernel
// What the workgroup takes, found from lens: the units of the sequences laid
// end to end.
struct Plan {
  int32_t start[kMaxBatch + 1];  // first unit of each sequence; [batch]: all
  int32_t rows[kMaxBatch];       // held
  int32_t waves[kWaves];
};

// Fills the plan in LDS, the first workgroup the join's copy too. All 64 kWaves
// threads call it.
__device__ __forceinline__ void lay_out(const DecodeArgs& a, Plan& plan) {
  constexpr int kThreads = 64 * kWaves, kMost = kMaxBatch / kThreads;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, B = a.pool.batch;
  const int per = (B + kThreads - 1) / kThreads;
  const bool writes = blockIdx.x == 0 && blockIdx.y == 0;
  int mine = 0, units[kMost];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int b = tid * per + i;
    units[i] = 0;
    if (i < per && b < B) {
      const Span s = span_of(a, b);
      plan.rows[b] = s.n;
      units[i] = s.units;
    }
    mine += units[i];
  }
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  if (lane == 63) plan.waves[wave] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int w = 0; w < wave; ++w) at += plan.waves[w];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int b = tid * per + i;
    if (i < per && b < B) {
      plan.start[b] = at;
      if (writes) a.starts[b] = at;
    }
    at += units[i];
  }
  if (tid == kThreads - 1) {
    plan.start[B] = at;
    if (writes) a.starts[B] = at;
  }
  __syncthreads();
}

// The workgroup's segments, one after the other (all values uniform).
struct Walk {
  int x, x1, b;          // next unit, the end, the sequence it is in
  int seq, n;            // the segment's sequence and the rows that it holds
  int row, lo, end;      // its rows: from a multiple of 16, those in [lo, end)
  bool whole;            // the whole sequence
  // Kept in scalar registers: the loops over it branch as one.
  static __device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
  __device__ __forceinline__ void start(const DecodeArgs& a, const Plan& plan) {
    const int batch = a.pool.batch, total = scalar(plan.start[batch]), per = units_per_wg(a, total);
    x = int(blockIdx.x) * per;
    x1 = x + per < total ? x + per : total;
    b = 0;
    int hi = batch;  // b: the last sequence that starts at or before x
    while (hi - b > 1) {
      const int mid = (b + hi) / 2;
      if (scalar(plan.start[mid]) <= x) b = mid;
      else hi = mid;
    }
  }
  __device__ __forceinline__ bool next(const DecodeArgs& a, const Plan& plan) {
    while (x < x1) {
      const int s0 = scalar(plan.start[b]), s1 = scalar(plan.start[b + 1]);
      seq = b++;
      if (s1 <= x) continue;
      const int stop = s1 < x1 ? s1 : x1;
      const int u0 = x - s0 - a.over, u1 = stop - s0 - a.over;
      x = stop;
      if (u1 <= 0) continue;  // only the units for starting on it
      const Span s = span_of_rows(a, scalar(plan.rows[seq]));
      n = s.n;
      lo = s.lo;
      row = ((u0 < 0 ? 0 : u0) + lo / kUnit) * kUnit;
      end = (u1 + lo / kUnit) * kUnit;
      end = end < n ? end : n;
      whole = u0 <= 0 && u1 == s.blocks;
      return true;
    }
    return false;
  }
};

constexpr float kTau = 8.0f;  // log2 by which a score may pass the running maximum

// What a workgroup keeps in LDS.
template <typename Rows>
struct Shared {
  static constexpr int kPiece = 16 * Chan<Rows::kD>::kCpl;  // channels joined at a time
  Plan plan;
  int32_t blocks[kWaves][kBlock];
  float ml[2][kWaves][16];
  __attribute__((aligned(16))) float joint[kWaves][16][kPiece + 4];
};

template <typename Rows>
__device__ __forceinline__ void attend(const DecodeArgs& a, Shared<Rows>& lds) {
  constexpr int D = Rows::kD, HALVES = Rows::kHalves, kRows = 16 * HALVES;  // rows a step
  using C = Chan<D>;
  constexpr int kPiece = Shared<Rows>::kPiece;
  auto& ml = lds.ml;
  auto& joint = lds.joint;
  const Pool& p = a.pool;
  const int tid = threadIdx.x, lane = tid % 64, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int kvh = blockIdx.y / a.groups16, set = blockIdx.y % a.groups16;
  const int live = a.G - 16 * set < 16 ? a.G - 16 * set : 16;  // heads here
  const int head0 = kvh * a.G + 16 * set;

  Walk walk;
  walk.start(a, lds.plan);
  while (walk.next(a, lds.plan)) {
    const int b = walk.seq, lo = walk.lo, end = walk.end;
    // A wavefront takes every fourth step of kRows rows.
    int row0 = walk.row + wave * kRows;
    // The queries and the table first, then the first step's rows, and the
    // queries' operands are prepared while these are on their way.
    uint32_t qw[D / 32][4];
    Rows::load_q(qw, uniform(a.q, 2 * (b * a.qstride + int64_t(head0) * D)), r < live, r, g);
    Pages pages;
    pages.start(lds.blocks[wave], p.table + b * p.tstride, (walk.n + (1 << p.shift) - 1) >> p.shift,
                row0 >> p.shift);
    typename Rows::K kr;
    typename Rows::V vr;
    Step<HALVES> h = step_of<HALVES>(p, pages, kvh, row0, end);
    Rows::load_k(kr, a, h, r, g);
    Rows::load_v(vr, a, h, r, g);
    typename Rows::Operand ops[Rows::kOperands];
    typename Rows::Rest q;
    Rows::prepare(ops, q, qw, r < live, g, a.scale_log2);
    floatx4 acc[C::kJ];
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) acc[j] = floatx4{0, 0, 0, 0};
    // The maximum of the scores before their factor: differences to it are exact
    // where they matter, however large the scores.
    float m = -INFINITY, l = 0.0f;
    typename Rows::Unit unit;
    for (; row0 < end; row0 += kWaves * kRows) {
      // The last step loads its own rows again: no branch between the loads.
      Step<HALVES> hn = h;
      if (row0 + kWaves * kRows < end)
        hn = step_of<HALVES>(p, pages, kvh, row0 + kWaves * kRows, end);
      float sc[4 * HALVES];
#pragma unroll
      for (int s = 0; s < HALVES; ++s) {
        const floatx4 y = Rows::scores([&](int c) { return ops[c]; }, q, kr, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[4 * s + i] = y[i];
        __builtin_amdgcn_sched_barrier(0);
      }
      Rows::load_k(kr, a, hn, r, g);
      __builtin_amdgcn_sched_barrier(0);
      if (!(row0 >= lo && row0 + kRows <= end && h.ok[0] && h.ok[HALVES - 1])) {
        uint32_t dead = 0;
#pragma unroll
        for (int e = 0; e < 4 * HALVES; ++e) {
          const int row = row0 + (e / 4) * 16 + 4 * g + e % 4;
          if (row < lo || row >= end || !h.ok[e / 4]) {
            dead |= 1u << e;
            sc[e] = -INFINITY;
          }
        }
        Rows::clear(vr, dead, unit.filler());
      }
      if (a.scores && r < live) {
        float* dst = a.scores + (int64_t(b) * a.H + head0 + r) * a.srows + row0 + 4 * g;
#pragma unroll
        for (int s = 0; s < HALVES; ++s)
          if (row0 + 16 * s < end)  // the rows behind are another segment's
            *reinterpret_cast<float4*>(dst + 16 * s) =
                make_float4(sc[4 * s] * q.mul, sc[4 * s + 1] * q.mul, sc[4 * s + 2] * q.mul,
                            sc[4 * s + 3] * q.mul);
      }
      float top = sc[0];
#pragma unroll
      for (int e = 1; e < 4 * HALVES; ++e) top = fmaxf(top, sc[e]);
      if (__any((top - m) * q.mul > kTau)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float next = fmaxf(m, top);
        const float scale = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - next) * q.mul);
        m = next;
        l *= scale;
#pragma unroll
        for (int j = 0; j < C::kJ; ++j) acc[j] *= scale;
      }
      const float base = m == -INFINITY ? 0.0f : m;
      float pr[4 * HALVES];
#pragma unroll
      for (int e = 0; e < 4 * HALVES; ++e) {
        pr[e] = __builtin_amdgcn_exp2f(fmaf(sc[e] - base, q.mul, -Rows::kDown));
        l += pr[e];
      }
      Rows::accumulate(vr, pr, acc, unit, r);
      __builtin_amdgcn_sched_barrier(0);
      Rows::load_v(vr, a, hn, r, g);
      __builtin_amdgcn_sched_barrier(0);
      h = hn;
    }

    float of = unit.of();
    if constexpr (Rows::kPairs) {
      if (__builtin_expect(unit.gave_up(), 0)) {  // again, with the maximum known
        of = 1.0f;
#pragma unroll
        for (int j = 0; j < C::kJ; ++j) acc[j] = floatx4{0, 0, 0, 0};
        const float base = m == -INFINITY ? 0.0f : m;
        row0 = walk.row + wave * kRows;
        pages.fill(row0 >> p.shift);
        for (; row0 < end; row0 += kWaves * kRows) {
          h = step_of<HALVES>(p, pages, kvh, row0, end);
          Rows::load_k(kr, a, h, r, g);
          Rows::load_v(vr, a, h, r, g);
          float pr[4 * HALVES];
          uint32_t dead = 0;
#pragma unroll
          for (int s = 0; s < HALVES; ++s) {
            const floatx4 y = Rows::scores([&](int c) { return ops[c]; }, q, kr, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = row0 + s * 16 + 4 * g + i;
              const bool none = row < lo || row >= end || !h.ok[s];
              dead |= uint32_t(none) << (4 * s + i);
              pr[4 * s + i] = none ? 0.0f : __builtin_amdgcn_exp2f(fmaf(y[i] - base, q.mul, -Rows::kDown));
            }
          }
          Rows::clear(vr, dead, 0);
          Rows::accumulate_pairs(vr, pr, acc, r);
        }
      }
    }

    // The four wavefronts' parts, joined in their order.
    m *= q.mul;
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    l *= Rows::kLast;
    if (lane < 16) {
      ml[0][wave][r] = m;
      ml[1][wave][r] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[0][w][r]);
    const float mine = m == -INFINITY ? 0.0f : exp2f(m - top) * of;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      sum += ml[0][w][r] == -INFINITY ? 0.0f * ml[1][w][r] : ml[1][w][r] * exp2f(ml[0][w][r] - top);
    const int64_t slot = int64_t(blockIdx.x) + b;
    if (tid < live) {
      a.part_m[slot * a.H + head0 + tid] = top;
      a.part_l[slot * a.H + head0 + tid] = sum;
    }
    __syncthreads();
    // Every thread keeps the sums of the heads it will write in LDS.
    if (wave == 0 && lane < 16) ml[1][0][r] = sum;
#pragma unroll
    for (int x0 = 0; x0 < C::kPieces; ++x0) {
      if (x0 > 0) __syncthreads();
      if (r < live) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* dst = &joint[wave][r][(4 * g + i) * C::kCpl];
#pragma unroll
          for (int j = 0; j < C::kCpl; j += 4) {
            const int at = x0 * C::kCpl + j;
            *reinterpret_cast<float4*>(dst + j) =
                make_float4(acc[at][i] * mine, acc[at + 1][i] * mine, acc[at + 2][i] * mine,
                            acc[at + 3][i] * mine);
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < live * kPiece; i += 64 * kWaves) {
        const int hd = i / kPiece, ch = i % kPiece;
        float o = joint[0][hd][ch];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) o += joint[w][hd][ch];
        const int d = x0 * kPiece + ch;
        if (walk.whole) {
          const float all = ml[1][0][hd];
          a.out[(int64_t(b) * a.H + head0 + hd) * D + d] = f32_to_bf16(all == 0.0f ? 0.0f : o / all);
        } else {
          a.part_o[(slot * a.H + head0 + hd) * D + d] = o;
        }
      }
    }
    __syncthreads();  // joint and ml are written again
  }
}

// Whether the batch's rows are more than the memory-side cache may still hold
// from an earlier call: then they are streamed. (16 ragged sequences, 70 MB in
// turn with two other pools: 17 us kept, 23 streamed; 131,071 rows, 537 MB:
// 95 us kept, 88 streamed; 268 MB: 50 and 46; 134 MB: 33 and 35.)
__device__ __forceinline__ bool streams(const DecodeArgs& a, const Plan& plan) {
  return __builtin_amdgcn_readfirstlane(plan.start[a.pool.batch]) > a.kept_units;
}

template <typename Rows>
__global__ __launch_bounds__(64 * kWaves, Rows::kOcc) void paged_decode_kernel(const DecodeArgs a) {
  __shared__ Shared<Rows> lds;
  lay_out(a, lds.plan);
  if constexpr (Rows::kChooses) {
    if (!streams(a, lds.plan)) {
      attend<typename Rows::Kept>(a, reinterpret_cast<Shared<typename Rows::Kept>&>(lds));
      return;
    }
  }
  attend<Rows>(a, lds);
}

// A workgroup barrier for LDS only: loads of the stream stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The 16 rows of a 64-row tile that a wavefront scores. By selects of values: an
// index would put the tile's rows into memory.
__device__ __forceinline__ Step<1> quarter_of(const Step<4>& h, int wave) {
  const int64_t r0 = h.row[0], r1 = h.row[1], r2 = h.row[2], r3 = h.row[3];
  const int64_t lo = wave & 1 ? r1 : r0, hi = wave & 1 ? r3 : r2;
  return Step<1>{{wave & 2 ? hi : lo}, {true}};
}

// Head dim 512. A wavefront of the kernel above would hold 128 accumulators
// beside 64 query and 64 key registers; here the four wavefronts of a
// workgroup share a 64-row tile: each scores 16 rows over all channels, the
// scores meet in LDS (two buffers, one barrier a tile), and each goes over the
// softmax of all 64 rows by itself and accumulates 128 output channels, which
// it also writes. The queries' operands lie in LDS: with them in registers the
// rows in flight went through accumulation registers, and each copy waited for
// its load.
constexpr int kWideTile = 16 * kWaves;

template <typename Rows>
struct SharedWide {
  Plan plan;
  int32_t blocks[kWaves][kBlock];
  float4 tiles[2][16][16];
  typename Rows::Operand queries[Rows::kOperands][64];
};

template <typename Rows>
__device__ __forceinline__ void attend_wide(const DecodeArgs& a, SharedWide<Rows>& lds) {
  constexpr int D = Rows::kD;
  static_assert(D == 128 * kWaves && Rows::kHalves == 1, "a wavefront takes 128 channels");
  auto& tiles = lds.tiles;
  auto& queries = lds.queries;
  const Pool& p = a.pool;
  const int tid = threadIdx.x, lane = tid % 64, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int kvh = blockIdx.y / a.groups16, set = blockIdx.y % a.groups16;
  const int live = a.G - 16 * set < 16 ? a.G - 16 * set : 16;
  const int head0 = kvh * a.G + 16 * set;
  Walk walk;
  walk.start(a, lds.plan);
  int buf = 0;
  while (walk.next(a, lds.plan)) {
    const int b = walk.seq, lo = walk.lo, end = walk.end;
    int row0 = walk.row;
    uint32_t qw[D / 32][4];
    Rows::load_q(qw, uniform(a.q, 2 * (b * a.qstride + int64_t(head0) * D)), r < live, r, g);
    Pages pages;
    pages.start(lds.blocks[wave], p.table + b * p.tstride, (walk.n + (1 << p.shift) - 1) >> p.shift,
                row0 >> p.shift);
    typename Rows::K kr;
    typename Rows::Wide vr;
    Step<4> h = step_of<4>(p, pages, kvh, row0, end);
    Rows::load_k(kr, a, quarter_of(h, wave), r, g);
    typename Rows::Rest q;
    {
      typename Rows::Operand ops[Rows::kOperands];
      Rows::prepare(ops, q, qw, r < live, g, a.scale_log2);
      // The last segment's reads are over: every wavefront passed a barrier
      // since its last (for scores, and of a second pass).
#pragma unroll
      for (int c = 0; c < Rows::kOperands; ++c)
        if (c % kWaves == wave) queries[c][lane] = ops[c];
      __builtin_amdgcn_sched_barrier(0);
      Rows::load_wide(vr, a, h, wave, r, g);  // after it: no registers for both
      lds_barrier();
    }
    floatx4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = floatx4{0, 0, 0, 0};
    // The maximum of the scores before their factor: differences to it are exact
    // where they matter, however large the scores.
    float m = -INFINITY, l = 0.0f;
    typename Rows::Unit unit;
    for (; row0 < end; row0 += kWideTile) {
      Step<4> hn = h;
      if (row0 + kWideTile < end) hn = step_of<4>(p, pages, kvh, row0 + kWideTile, end);
      const floatx4 y = Rows::scores([&](int c) { return queries[c][lane]; }, q, kr, 0);
      float4 mine = make_float4(y[0], y[1], y[2], y[3]);
      __builtin_amdgcn_sched_barrier(0);
      Rows::load_k(kr, a, quarter_of(hn, wave), r, g);
      __builtin_amdgcn_sched_barrier(0);
      const bool full = row0 >= lo && row0 + kWideTile <= end && h.ok[0] && h.ok[1] && h.ok[2] && h.ok[3];
      uint32_t dead = 0;  // of the lane's 16 rows
      if (!full) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int row = row0 + (e / 4) * 16 + 4 * g + e % 4;
          dead |= uint32_t(row < lo || row >= end || !h.ok[e / 4]) << e;
        }
        const uint32_t d = dead >> (4 * wave);
        mine.x = d & 1 ? -INFINITY : mine.x;
        mine.y = d & 2 ? -INFINITY : mine.y;
        mine.z = d & 4 ? -INFINITY : mine.z;
        mine.w = d & 8 ? -INFINITY : mine.w;
        Rows::clear_wide(vr, dead, unit.filler());
      }
      tiles[buf][4 * wave + g][r] = mine;
      if (a.scores && r < live && row0 + 16 * wave < end)
        *reinterpret_cast<float4*>(a.scores + (int64_t(b) * a.H + head0 + r) * a.srows + row0 +
                                   16 * wave + 4 * g) =
            make_float4(mine.x * q.mul, mine.y * q.mul, mine.z * q.mul, mine.w * q.mul);
      lds_barrier();
      float pr[16];
      float top = -INFINITY;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float4 x = tiles[buf][4 * s + g][r];
        pr[4 * s] = x.x;
        pr[4 * s + 1] = x.y;
        pr[4 * s + 2] = x.z;
        pr[4 * s + 3] = x.w;
        top = fmaxf(top, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)));
      }
      buf ^= 1;
      if (__any((top - m) * q.mul > kTau)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float next = fmaxf(m, top);
        const float scale = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - next) * q.mul);
        m = next;
        l *= scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] *= scale;
      }
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        pr[e] = __builtin_amdgcn_exp2f(fmaf(pr[e] - base, q.mul, -Rows::kDown));
        l += pr[e];
      }
      Rows::accumulate_wide(vr, pr, acc, unit, wave, r);
      __builtin_amdgcn_sched_barrier(0);
      Rows::load_wide(vr, a, hn, wave, r, g);
      __builtin_amdgcn_sched_barrier(0);
      h = hn;
    }
    float of = unit.of();
    if constexpr (Rows::kPairs) {
      if (__builtin_expect(unit.gave_up(), 0)) {  // again, with the maximum known, all scores its own
        of = 1.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = floatx4{0, 0, 0, 0};
        const float base = m == -INFINITY ? 0.0f : m;
        row0 = walk.row;
        pages.fill(row0 >> p.shift);
        for (; row0 < end; row0 += kWideTile) {
          h = step_of<4>(p, pages, kvh, row0, end);
          Rows::load_wide(vr, a, h, wave, r, g);
          float pr[16];
          uint32_t dead = 0;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            Rows::load_k(kr, a, quarter_of(h, s), r, g);
            const floatx4 y = Rows::scores([&](int c) { return queries[c][lane]; }, q, kr, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = row0 + s * 16 + 4 * g + i;
              const bool none = row < lo || row >= end || !h.ok[s];
              dead |= uint32_t(none) << (4 * s + i);
              pr[4 * s + i] = none ? 0.0f : __builtin_amdgcn_exp2f(fmaf(y[i] - base, q.mul, -Rows::kDown));
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          Rows::clear_wide(vr, dead, 0);
          Rows::accumulate_wide_pairs(vr, pr, acc, wave, r);
        }
      }
      lds_barrier();  // the queries are written again
    }
    // Every wavefront holds the same maximum and sum.
    m *= q.mul;
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    l *= Rows::kLast;
    const int64_t slot = int64_t(blockIdx.x) + b;
    if (tid < live) {
      a.part_m[slot * a.H + head0 + tid] = m;
      a.part_l[slot * a.H + head0 + tid] = l;
    }
    if (r < live) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 128 * wave + (4 * g + i) * 8;
        if (walk.whole) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = f32_to_bf16(l == 0.0f ? 0.0f : acc[2 * j][i] * of / l) |
                   uint32_t(f32_to_bf16(l == 0.0f ? 0.0f : acc[2 * j + 1][i] * of / l)) << 16;
          uint16_t* out = a.out + (int64_t(b) * a.H + head0 + r) * D + d;
#pragma unroll
          for (int j = 0; j < 8; ++j) out[j] = uint16_t(w[j / 2] >> (16 * (j % 2)));
        } else {
          float4* out = reinterpret_cast<float4*>(a.part_o + (slot * a.H + head0 + r) * D + d);
          out[0] = make_float4(acc[0][i] * of, acc[1][i] * of, acc[2][i] * of, acc[3][i] * of);
          out[1] = make_float4(acc[4][i] * of, acc[5][i] * of, acc[6][i] * of, acc[7][i] * of);
        }
      }
    }
  }
}

template <typename Rows>
__global__ __launch_bounds__(64 * kWaves, Rows::kWideOcc) void paged_wide_kernel(const DecodeArgs a) {
  __shared__ SharedWide<Rows> lds;
  lay_out(a, lds.plan);
  if constexpr (Rows::kChooses) {
    if (!streams(a, lds.plan)) {
      attend_wide<typename Rows::Kept>(a, reinterpret_cast<SharedWide<typename Rows::Kept>&>(lds));
      return;
    }
  }
  attend_wide<Rows>(a, lds);
}

// One affine layout's launch; a unit a head dim (paged_decode_d*.hip).
// occupancy: no launch, but the wavefronts a SIMD of the layout's kernel.
template <typename Rows>
int launch_rows(const DecodeArgs& a, dim3 grid, hipStream_t st, bool occupancy) {
  if constexpr (Rows::kD == 512) {
    if (!occupancy)
      hipLaunchKernelGGL(paged_wide_kernel<Rows>, grid, dim3(64 * kWaves), 0, st, a);
    return Rows::kWideOcc;
  } else {
    if (!occupancy)
      hipLaunchKernelGGL(paged_decode_kernel<Rows>, grid, dim3(64 * kWaves), 0, st, a);
    return Rows::kOcc;
  }
}

template <int D>
int launch_affine(const DecodeArgs& a, int bk, int bv, int gs, dim3 grid, hipStream_t st,
                  bool occupancy) {
  auto width = [&](auto group) {
    constexpr int GS = decltype(group)::value;
    if (bk == 4 && bv == 4) return launch_rows<AffineRows<D, 4, 4, GS>>(a, grid, st, occupancy);
    if (bk == 4) return launch_rows<AffineRows<D, 4, 8, GS>>(a, grid, st, occupancy);
    if (bv == 4) return launch_rows<AffineRows<D, 8, 4, GS>>(a, grid, st, occupancy);
    return launch_rows<AffineRows<D, 8, 8, GS>>(a, grid, st, occupancy);
  };
  if (gs == 32) return width(std::integral_constant<int, 32>{});
  if (gs == 64) return width(std::integral_constant<int, 64>{});
  if constexpr (D >= 128) return width(std::integral_constant<int, 128>{});
  return 1;
}

}  // namespace paged
}  // namespace tqkv

// Decode attention over a paged cache: one new token a sequence.
//
// o = sum_t p_t v_t with p = softmax(scale q.k_t): one pass over the rows with
// a running maximum and sum. The rows of the whole batch, cut into 32-row
// tiles, are laid end to end and divided evenly among the W workgroups of a
// KV head, from lens on the device: a long sequence spreads over many
// workgroups and a workgroup may take several short ones. A workgroup's part
// of one sequence is a segment; it leaves the segment's output, maximum and
// sum in slot (workgroup + sequence), which no other segment shares (along
// the row order both only grow and one always does), unless the segment is
// the whole sequence. The second launch joins the slots.
//
// A wavefront takes whole tiles, every fourth of the segment, on the matrix
// cores with the query heads of the KV head as the 16 columns:
//   S[row][head] = K Q^T  (A: lane l holds row l % 16 and 8 channels of
//     quarter l / 16; two 16-row products a tile), so lane l ends up with head
//     l % 16 and rows 4 (l / 16) + i of each half;
//   O^T[channel][head] += V^T P^T: the eight weights that lane l just
//     computed are the operand it has to supply (rows as the contraction, in
//     an order that V's loads follow), so P never leaves the lane, and the
//     running maximum, sum and rescaling are the lane's own.
// V's operand is a channel's eight rows: a lane loads 8 (4 at D = 64)
// consecutive channels of its eight rows and pairs rows by byte permutes.
// Weights enter as a bf16 pair hi + lo, 16 bits, so their rounding stays below
// the bf16 output's; the softmax sum is of the unrounded f32 weights.
//
// Affine rows: scores use the codes themselves, exact in bf16, one product a
// group: s = sum_g scale_g (q.c)_g + bias_g sum(q_g). 4-bit codes become
// bf16 128 + c by one AND-OR a pair, and the 128 goes into the bias. Values
// are dequantized in f32 and rounded once to bf16, the rows that
// tqkv_affine_dequantize gives.
//
// Bound by HBM: the live rows once. At G heads of 16 the matrix cores do
// 16 / G times the work that is needed and are still far from busy.
#pragma once

#include <type_traits>

#include "paged.hpp"

namespace tqkv {
namespace paged {

constexpr int kWaves = 4;
constexpr int kTile = 32;
constexpr int kMinTiles = 4;  // tiles a workgroup at least: one a wavefront

struct DecodeArgs {
  Pool pool;
  const void* slot[6];
  const uint16_t* q;
  int64_t qstride;
  uint16_t* out;
  int H, G, groups16;  // query heads, of a KV head, 16-head sets of those
  int max_rows, window;
  int W;               // workgroups a (KV head, set)
  float scale_log2;
  float* part_o;  // [W + batch, H, D]
  float* part_m;  // [W + batch, H]: log2 units
  float* part_l;
  float* scores;  // [batch, H, srows] log2 units, or NULL
  int64_t srows;
};

// The tiles of sequence b: n rows held, from the window's first.
struct Span {
  int n, lo, tiles;
};
__device__ __forceinline__ Span span_of(const DecodeArgs& a, int b) {
  const int most = a.max_rows < a.pool.cap ? a.max_rows : a.pool.cap;
  const int n = held(a.pool, b, most);
  const int lo = a.window > 0 && n > a.window ? n - a.window : 0;
  return {n, lo, n > 0 ? (n + kTile - 1) / kTile - lo / kTile : 0};
}

// Tiles a workgroup takes of `total`.
__device__ __forceinline__ int tiles_per_wg(int total, int W) {
  const int per = (total + W - 1) / W;
  return per < kMinTiles ? kMinTiles : per;
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

// A load of N bytes (2, 4, 8 or a multiple of 16) into words.
template <int N>
__device__ __forceinline__ void load_words(const char* p, uint32_t* w) {
  if constexpr (N == 2) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
    static_assert(N % 16 == 0, "whole 16-byte loads");
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(p + 16 * i);
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  }
}

// The two pool row blocks (page, KV head) of a tile's 16-row halves.
struct Halves {
  int64_t row[2];  // pool row of the half's first row
  bool ok[2];
};
__device__ __forceinline__ Halves halves_of(const Pool& p, const int32_t* table, int kvh, int tile,
                                            int n) {
  Halves h;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int r = tile * kTile + s * 16;
    int page = -1;
    if (r < n) page = table[r >> p.shift];
    h.ok[s] = page >= 0 && page < p.num_pages;
    h.row[s] = pool_row(p, h.ok[s] ? page : 0, kvh, h.ok[s] ? r & ((1 << p.shift) - 1) : 0);
  }
  return h;
}

// Channel layout of the values: MFMA j's output row r is channel_of(j, r).
template <int D>
struct Chan {
  static constexpr int kCpl = D >= 128 ? 8 : 4;      // consecutive channels a lane and piece
  static constexpr int kPieces = D / (16 * kCpl);
  static constexpr int kJ = D / 16;                  // products (and accumulators)
};

// ---------------------------------------------------------------- bf16 rows
template <int D>
struct Bf16Rows {
  static constexpr int kD = D;
  using C = Chan<D>;
  static constexpr int kChunks = D / 32;
  struct Q {
    bf16x8 op[kChunks];
  };
  struct K {
    uint32_t w[2][D / 32 * 4];
  };
  struct V {
    uint32_t w[8][C::kPieces * C::kCpl / 2];
  };

  // Channels of (chunk, quarter): 32 chunk + 8 quarter.
  static __device__ __forceinline__ void load_q(Q& q, const uint16_t* p, bool live, int g) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      uint32_t w[4] = {0, 0, 0, 0};
      if (live) load_words<16>(reinterpret_cast<const char*>(p + c * 32 + g * 8), w);
      q.op[c] = as_bf16x8(w[0], w[1], w[2], w[3]);
    }
  }
  static __device__ __forceinline__ void load_k(K& k, const DecodeArgs& a, const Halves& h, int r,
                                                int g) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p = static_cast<const char*>(a.slot[0]) + (h.row[s] + r) * (2 * D) + g * 16;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) load_words<16>(p + c * 64, k.w[s] + 4 * c);
    }
  }
  static __device__ __forceinline__ void load_v(V& v, const DecodeArgs& a, const Halves& h, int r,
                                                int g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const char* p = static_cast<const char*>(a.slot[1]) +
                      (h.row[e / 4] + 4 * g + e % 4) * (2 * D) + r * (2 * C::kCpl);
#pragma unroll
      for (int x = 0; x < C::kPieces; ++x)
        load_words<2 * C::kCpl>(p + x * 256, v.w[e] + x * (C::kCpl / 2));
    }
  }
  // Scores of half s, unscaled.
  static __device__ __forceinline__ floatx4 scores(const Q& q, const K& k, int s) {
    floatx4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      acc = mfma(as_bf16x8(k.w[s][4 * c], k.w[s][4 * c + 1], k.w[s][4 * c + 2], k.w[s][4 * c + 3]),
                 q.op[c], acc);
    return acc;
  }
  // The rows for which dead is set hold nothing: zero, whatever lies there.
  static __device__ __forceinline__ void clear(V& v, uint32_t dead) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < C::kPieces * C::kCpl / 2; ++i)
        if (dead >> e & 1) v.w[e][i] = 0;
  }
  template <typename F>
  static __device__ __forceinline__ void values(const V& v, int, F&& product) {
#pragma unroll
    for (int i = 0; i < C::kPieces * C::kCpl / 2; ++i) {
      product(2 * i, as_bf16x8(lows(v.w[0][i], v.w[1][i]), lows(v.w[2][i], v.w[3][i]),
                               lows(v.w[4][i], v.w[5][i]), lows(v.w[6][i], v.w[7][i])));
      product(2 * i + 1, as_bf16x8(highs(v.w[0][i], v.w[1][i]), highs(v.w[2][i], v.w[3][i]),
                                   highs(v.w[4][i], v.w[5][i]), highs(v.w[6][i], v.w[7][i])));
    }
  }
};

// -------------------------------------------------------------- affine rows
template <int D, int BK, int BV, int GS>
struct AffineRows {
  static constexpr int kD = D;
  using C = Chan<D>;
  static constexpr int NG = D / GS;          // groups a row
  static constexpr int CPG = GS / 32;        // products a group
  static constexpr int kGroupBytes = GS / 4 * BK / 8;  // a lane's codes of a group
  static constexpr int kGroupWords = (kGroupBytes + 3) / 4;
  static constexpr int kPieceBytes = C::kCpl * BV / 8;
  static constexpr int kPieceWords = (kPieceBytes + 3) / 4;
  static constexpr int kGpp = 16 * C::kCpl / GS > 0 ? 16 * C::kCpl / GS : 1;  // groups a piece
  struct Q {
    bf16x8 op[D / 32];
    float sum[NG];  // of a group's channels, log2-scaled later with the rest
  };
  struct K {
    uint32_t w[2][NG * kGroupWords];
    uint32_t s[2][2 * NG], b[2][2 * NG];  // 4 rows x NG scales and biases of each half
  };
  struct V {
    uint32_t w[8][C::kPieces * kPieceWords];
    uint32_t s[2][2 * NG], b[2][2 * NG];
  };

  // Channels of (group, quarter): group GS + quarter GS / 4, then in order; a
  // product's eight in the order that unpack() gives the codes.
  static __device__ __forceinline__ void load_q(Q& q, const uint16_t* p, bool live, int g) {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < CPG; ++c) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (live) load_words<16>(reinterpret_cast<const char*>(p + n * GS + g * (GS / 4) + c * 8), w);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += low_f32(w[i]) + high_f32(w[i]);
        if (BK == 4)  // (0,4) (1,5) (2,6) (3,7)
          q.op[n * CPG + c] = as_bf16x8(lows(w[0], w[2]), highs(w[0], w[2]), lows(w[1], w[3]),
                                        highs(w[1], w[3]));
        else
          q.op[n * CPG + c] = as_bf16x8(w[0], w[1], w[2], w[3]);
      }
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      q.sum[n] = sum;
    }
  }
  // Scales (or biases) of rows [4 g, 4 g + 4) of both halves.
  static __device__ __forceinline__ void load_scales(uint32_t (&w)[2][2 * NG], const void* slot,
                                                     const Halves& h, int g) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p = static_cast<const char*>(slot) + (h.row[s] + 4 * g) * (2 * NG);
      load_words<8 * NG>(p, w[s]);
    }
  }
  static __device__ __forceinline__ void load_k(K& k, const DecodeArgs& a, const Halves& h, int r,
                                                int g) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p = static_cast<const char*>(a.slot[0]) + (h.row[s] + r) * (D * BK / 8) +
                      g * kGroupBytes;
#pragma unroll
      for (int n = 0; n < NG; ++n)
        load_words<kGroupBytes>(p + n * (GS * BK / 8), k.w[s] + n * kGroupWords);
    }
    load_scales(k.s, a.slot[1], h, g);
    load_scales(k.b, a.slot[2], h, g);
  }
  static __device__ __forceinline__ void load_v(V& v, const DecodeArgs& a, const Halves& h, int r,
                                                int g) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const char* p = static_cast<const char*>(a.slot[3]) +
                      (h.row[e / 4] + 4 * g + e % 4) * (D * BV / 8) + r * kPieceBytes;
#pragma unroll
      for (int x = 0; x < C::kPieces; ++x)
        load_words<kPieceBytes>(p + x * (16 * kPieceBytes), v.w[e] + x * kPieceWords);
    }
    load_scales(v.s, a.slot[4], h, g);
    load_scales(v.b, a.slot[5], h, g);
  }
  // Eight codes as bf16: 4 bits, 128 + c of codes (0,4) (1,5) (2,6) (3,7);
  // 8 bits, the codes in order.
  static __device__ __forceinline__ bf16x8 unpack(const uint32_t* w) {
    if constexpr (BK == 4) {
      constexpr uint32_t m = 0x000f000fu, one = 0x43004300u;
      return as_bf16x8((w[0] & m) | one, ((w[0] >> 4) & m) | one, ((w[0] >> 8) & m) | one,
                       ((w[0] >> 12) & m) | one);
    } else {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = w[i / 2] >> (16 * (i % 2));
        o[i] = highs(__float_as_uint(float(x & 0xffu)), __float_as_uint(float((x >> 8) & 0xffu)));
      }
      return as_bf16x8(o[0], o[1], o[2], o[3]);
    }
  }
  // The f32 of entry (row i of four, group n) of four rows' scales.
  static __device__ __forceinline__ float entry(const uint32_t* w, int i, int n) {
    const int at = i * NG + n;
    return at % 2 ? high_f32(w[at / 2]) : low_f32(w[at / 2]);
  }
  static __device__ __forceinline__ floatx4 scores(const Q& q, const K& k, int s) {
    floatx4 out = {0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      floatx4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < CPG; ++c)
        acc = mfma(unpack(k.w[s] + n * kGroupWords + c * (BK / 4)), q.op[n * CPG + c], acc);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float sc = entry(k.s[s], i, n);
        float bi = entry(k.b[s], i, n);
        if (BK == 4) bi = fmaf(-128.0f, sc, bi);
        out[i] = fmaf(sc, acc[i], fmaf(bi, q.sum[n], out[i]));
      }
    }
    return out;
  }
  // Dead rows: codes of 0, a scale and a bias of 0.
  static __device__ __forceinline__ void clear(V& v, uint32_t dead) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!(dead >> e & 1)) continue;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const int at = e % 4 * NG + n;
        const uint32_t keep = at % 2 ? 0x0000ffffu : 0xffff0000u;
        v.s[e / 4][at / 2] &= keep;
        v.b[e / 4][at / 2] &= keep;
      }
    }
  }
  // The scale of (row e, the lane's group of piece x): of the kGpp
  // candidates, the one of lane row r.
  static __device__ __forceinline__ float lane_entry(const uint32_t (&w)[2][2 * NG], int e, int x,
                                                     int r) {
    const int first = x * (16 * C::kCpl) / GS;
    float f = entry(w[e / 4], e % 4, first);
#pragma unroll
    for (int c = 1; c < kGpp; ++c)
      f = r * C::kCpl / GS == c ? entry(w[e / 4], e % 4, first + c) : f;
    return f;
  }
  template <typename F>
  static __device__ __forceinline__ void values(const V& v, int r, F&& product) {
#pragma unroll
    for (int x = 0; x < C::kPieces; ++x) {
      uint32_t o[C::kCpl][4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float s0 = lane_entry(v.s, e, x, r), b0 = lane_entry(v.b, e, x, r);
        const float s1 = lane_entry(v.s, e + 1, x, r), b1 = lane_entry(v.b, e + 1, x, r);
#pragma unroll
        for (int j = 0; j < C::kCpl; ++j) {
          const int bit = j * BV;
          const uint32_t m = (1u << BV) - 1;
          const float c0 = float((v.w[e][x * kPieceWords + bit / 32] >> (bit % 32)) & m);
          const float c1 = float((v.w[e + 1][x * kPieceWords + bit / 32] >> (bit % 32)) & m);
          o[j][e / 2] = pack_bf16(fmaf(c0, s0, b0), fmaf(c1, s1, b1));
        }
      }
#pragma unroll
      for (int j = 0; j < C::kCpl; ++j)
        product(x * C::kCpl + j, as_bf16x8(o[j][0], o[j][1], o[j][2], o[j][3]));
    }
  }
};

// ------------------------------------------------------------------- kernel
// Exclusive prefix over the batch of the tiles of each sequence, into LDS:
// start[b], start[batch] = all. All threads call it; batch <= 4 kThreads.
template <int kThreads>
__device__ __forceinline__ void lay_out(const DecodeArgs& a, int32_t* start, int32_t* waves) {
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, B = a.pool.batch;
  const int per = (B + kThreads - 1) / kThreads;
  int mine = 0, t[kMaxBatch / kThreads];
#pragma unroll
  for (int i = 0; i < kMaxBatch / kThreads; ++i) {
    const int b = tid * per + i;
    t[i] = i < per && b < B ? span_of(a, b).tiles : 0;
    mine += t[i];
  }
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  if (lane == 63) waves[wave] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int w = 0; w < wave; ++w) at += waves[w];
#pragma unroll
  for (int i = 0; i < kMaxBatch / kThreads; ++i) {
    const int b = tid * per + i;
    if (i < per && b < B) start[b] = at;
    at += t[i];
  }
  if (tid == kThreads - 1) start[B] = at;
  __syncthreads();
}

constexpr float kTau = 8.0f;  // log2 by which a score may pass the running maximum
// Weights are held times 2^-40 (their sum too, so it cancels): 2^30 rows of
// weight 2^8 and values of bf16's largest magnitude stay within f32. Weights
// below 2^-86 of the largest vanish.
constexpr float kDown = 40.0f;

template <typename Rows>
__global__ __launch_bounds__(64 * kWaves) void paged_decode_kernel(const DecodeArgs a) {
  constexpr int D = Rows::kD;
  using C = Chan<D>;
  constexpr int kPiece = 16 * C::kCpl;      // channels the epilogue joins at a time
  constexpr int kStride = kPiece + 4;
  __shared__ int32_t start[kMaxBatch + 1];
  __shared__ int32_t wsum[kWaves];
  __shared__ float ml[2][kWaves][16];
  __shared__ __attribute__((aligned(16))) float joint[kWaves][16][kStride];
  const Pool& p = a.pool;
  const int tid = threadIdx.x, lane = tid % 64, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int kvh = blockIdx.y / a.groups16, set = blockIdx.y % a.groups16;
  const int live = a.G - 16 * set < 16 ? a.G - 16 * set : 16;  // heads here
  const int head0 = kvh * a.G + 16 * set;

  lay_out<64 * kWaves>(a, start, wsum);
  const int total = start[p.batch], per = tiles_per_wg(total, a.W);
  int x = int(blockIdx.x) * per;
  const int x1 = x + per < total ? x + per : total;
  if (x >= x1) return;
  int b = 0;
  {  // the last sequence that starts at or before x
    int hi = p.batch;
    while (hi - b > 1) {
      const int mid = (b + hi) / 2;
      if (start[mid] <= x) b = mid;
      else hi = mid;
    }
  }
  for (; x < x1; ++b) {
    b = __builtin_amdgcn_readfirstlane(b);
    const int s0 = start[b], s1 = start[b + 1];
    if (s1 <= x) continue;
    const int end = s1 < x1 ? s1 : x1;
    const bool whole = x == s0 && end == s1;
    const Span span = span_of(a, b);
    const int n = span.n, lo = span.lo;
    const int t1 = end - s0 + lo / kTile;
    int t = __builtin_amdgcn_readfirstlane(x - s0 + lo / kTile + wave);
    x = end;
    const int32_t* table = p.table + b * p.tstride;

    typename Rows::Q q;
    Rows::load_q(q, a.q + b * a.qstride + int64_t(head0 + r) * D, r < live, g);
    floatx4 acc[C::kJ];
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) acc[j] = floatx4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;

    typename Rows::K kr;
    typename Rows::V vr;
    Halves h{};
    if (t < t1) {
      h = halves_of(p, table, kvh, t, n);
      Rows::load_k(kr, a, h, r, g);
      Rows::load_v(vr, a, h, r, g);
    }
    for (; t < t1; t += kWaves) {
      const Halves hn = t + kWaves < t1 ? halves_of(p, table, kvh, t + kWaves, n) : h;
      float sc[8];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const floatx4 y = Rows::scores(q, kr, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[4 * s + i] = y[i] * a.scale_log2;
      }
      if (t + kWaves < t1) Rows::load_k(kr, a, hn, r, g);
      const int row0 = t * kTile;
      if (!(row0 >= lo && row0 + kTile <= n && h.ok[0] && h.ok[1])) {
        uint32_t dead = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = row0 + (e / 4) * 16 + 4 * g + e % 4;
          if (row < lo || row >= n || !h.ok[e / 4]) {
            dead |= 1u << e;
            sc[e] = -INFINITY;
          }
        }
        Rows::clear(vr, dead);
      }
      if (a.scores && r < live) {
        float* dst = a.scores + (int64_t(b) * a.H + head0 + r) * a.srows + row0 + 4 * g;
        *reinterpret_cast<float4*>(dst) = make_float4(sc[0], sc[1], sc[2], sc[3]);
        *reinterpret_cast<float4*>(dst + 16) = make_float4(sc[4], sc[5], sc[6], sc[7]);
      }
      float top = sc[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, sc[e]);
      if (__any(top > m + kTau)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float next = fmaxf(m, top);
        const float scale = m == -INFINITY ? 0.0f : exp2f(m - next);
        m = next;
        l *= scale;
#pragma unroll
        for (int j = 0; j < C::kJ; ++j) acc[j] *= scale;
      }
      const float base = m == -INFINITY ? 0.0f : m + kDown;
      uint32_t hi[4], lw[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(sc[e] - base);
        const float p1 = __builtin_amdgcn_exp2f(sc[e + 1] - base);
        l += p0 + p1;
        const uint32_t w = pack_bf16(p0, p1);
        hi[e / 2] = w;
        lw[e / 2] = pack_bf16(p0 - low_f32(w), p1 - high_f32(w));
      }
      const bf16x8 ph = as_bf16x8(hi[0], hi[1], hi[2], hi[3]);
      const bf16x8 pl = as_bf16x8(lw[0], lw[1], lw[2], lw[3]);
      Rows::values(vr, r, [&](int j, bf16x8 v) {
        acc[j] = mfma(v, ph, acc[j]);
        acc[j] = mfma(v, pl, acc[j]);
      });
      if (t + kWaves < t1) Rows::load_v(vr, a, hn, r, g);
      h = hn;
    }

    // The four wavefronts' parts, joined in their order.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < 16) {
      ml[0][wave][r] = m;
      ml[1][wave][r] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[0][w][r]);
    const float mine = m == -INFINITY ? 0.0f : exp2f(m - top);
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
        if (whole) {
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

// One affine layout's launch; a unit a head dim (paged_decode_d*.hip).
template <int D>
void launch_affine(const DecodeArgs& a, int bk, int bv, int gs, dim3 grid, hipStream_t st) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, st, a);
  };
  auto width = [&](auto group) {
    constexpr int GS = decltype(group)::value;
    if (bk == 4 && bv == 4) go(paged_decode_kernel<AffineRows<D, 4, 4, GS>>);
    else if (bk == 4) go(paged_decode_kernel<AffineRows<D, 4, 8, GS>>);
    else if (bv == 4) go(paged_decode_kernel<AffineRows<D, 8, 4, GS>>);
    else go(paged_decode_kernel<AffineRows<D, 8, 8, GS>>);
  };
  if (gs == 32) width(std::integral_constant<int, 32>{});
  else if (gs == 64) width(std::integral_constant<int, 64>{});
  else if constexpr (D >= 128) width(std::integral_constant<int, 128>{});
}

}  // namespace paged
}  // namespace tqkv

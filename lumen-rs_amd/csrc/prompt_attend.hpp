// Attention of packed sequences on the matrix cores: softmax(scale Q K^T +
// mask) V for the queries of many sequences, keys and values out of the same
// packed tokens, the pages of a bf16 pool, or a slab of dequantized rows.
//
// Work split: a block takes kRows rows of one (sequence, KV head); the G query
// heads of a KV head share its keys, so rows are (position, head) pairs, head
// fastest, and see nearly the same keys. Block ids count over the packed
// tokens: sequence b's begin at starts[b] G / kRows + b, which leaves each at
// least the ids that it needs (floor(x + y) - floor(x) + 1 >= ceil(y)), so a
// block finds its sequence from starts alone and the host needs no lengths.
// Later ids (later positions, more keys) run first, and the blocks of a KV
// head on as few XCDs as that allows, since they read the same rows.
//
// Per tile of kKeys keys: K and V rows go straight from HBM into LDS, two
// tiles ahead where LDS holds them, every 16-byte piece at a place of its row
// that leaves the operand reads free of bank conflicts. A wavefront owns kRW
// rows: S^T = K Q^T (Q in registers), online softmax per row, whose running
// maximum may lag by kTau so that the accumulators are seldom rescaled, then
// O^T += V^T P^T, the scores' registers being the operand's layout and V
// transposed by the LDS read. Weights are rounded to bf16 over bf16 rows (V
// keeps its range; f16 would keep three more bits of the weights and lose it),
// to f16 over affine rows as f16, and the row sum counts them as rounded.
//
// Bound by the matrix cores and what shares their issue slots. Eight ragged prompts
// up to 8,192 tokens, D = 128: 937 GF in 897 us where calls alternate with other work
// (1.04 PF/s; a matrix product of 8,192 cubed 1.24) and 940 to 1,060 one call after the
// other, when the clock falls (0.88 to 1.0 PF/s); the matrix pipes busy 47% of the CUs'
// cycles, vector operations (exp2 and the rounding of the weights) 49%. D = 256 with
// 16 rows a wavefront and D = 512 with one tile of K and V in LDS read LDS for every
// product: 400 and 665 TF/s over windows and prompts whose blocks do not divide evenly
// among the CUs.
//
// Weights of hidden keys are exact zeros, but zero times an infinite value is
// NaN (and sums of values next to f32's largest pass it): a row that ends with
// anything that is not finite is done again, one key at a time, by attend_row,
// which leaves hidden keys out.
#pragma once

#include <type_traits>
#include <utility>

#include "paged.hpp"

namespace tqkv {
namespace prompt {

// Where keys and values lie.
enum Source { kPacked, kPagedBf16, kPagedAffine, kSlab };

struct Args {
  const uint16_t* q;  // head h of token i at q + i * qs + h * D
  int64_t qs;
  uint16_t* out;  // [tokens, H, D]
  const int32_t* starts;
  int64_t tokens;
  int batch, H, Hkv, G;
  float scale;
  int causal;
  int window;  // 0: none
  // kPacked: head h of token i at i * ts + h * hs.
  const uint16_t* k;
  const uint16_t* v;
  int64_t ts, hs;
  // Pages.
  paged::Pool pool;
  const void* slot[6];
  int gs, bits_k, bits_v, max_rows;
  // kSlab: rows [batch, Hkv, slab_rows, D], K as f16 times 2^-exponent[2 u] of
  // unit u = (sequence, KV head), V alike by exponent[2 u + 1], or as bf16 where
  // that is kBf16.
  const uint16_t* slab_k;
  const uint16_t* slab_v;
  const int32_t* exponent;
  int64_t slab_rows;
  // Block ids a KV head. Key splits: split s covers keys [s * split_keys,
  // (s + 1) * split_keys); with part_o set a row's (o unnormalised, maximum in
  // log2 units, sum) go to slot (token * H + head) * splits + s.
  int ids, splits, split_keys;
  float* part_o;
  float* part_m;
  float* part_l;
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kBf16 = 0x7fffffff;
// The slab's keys share a power of two a (sequence, KV head): a channel is off by
// up to 2^-25, half of f16's least step, where the largest key is 2^14 or more, and
// a score by D 2^15 2^-25 of those units. A row whose unit makes that more than
// kCoarse (in log2 units; it may see none of the large keys) is done by attend_row:
// |q| |k| scale of 2^28 or so, far from where a softmax tells keys apart.
constexpr float kCoarse = 0x1p-10f;

// A sequence's queries [first, first + count) and the keys that it has.
struct Sequence {
  int64_t first;
  int count, keys;
};
// starts is taken as ascending within [0, tokens]; what is not stays in bounds.
__device__ __forceinline__ int64_t start_of(const Args& a, int b) {
  const int64_t s = a.starts[b];
  return s < 0 ? 0 : s < a.tokens ? s : a.tokens;
}
template <Source S>
__device__ __forceinline__ Sequence sequence(const Args& a, int b) {
  const int64_t lo = start_of(a, b), hi = start_of(a, b + 1);
  const int count = int(hi < lo ? 0 : hi - lo);
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

// The first of them. p may lie far before the first key, and the window be the
// largest that the type holds.
__device__ __forceinline__ int first_seen(const Args& a, int p) {
  return a.window > 0 && p >= a.window ? p - a.window + 1 : 0;
}

// Channel c of a stored row in f32.
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
    return fmaf(s, float(code), b);
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

// One query row by one wavefront, in f32: a lane a key for the scores,
// channels for the values. Hidden keys are left out, not multiplied by zero.
template <int D, Source S>
__device__ __forceinline__ void attend_row(const Args& a, int b, int64_t token, int head) {
  const Sequence s = sequence<S>(a, b);
  const int lane = threadIdx.x % 64, h = head / a.G;
  const int64_t p = int64_t(s.keys) - s.count + (token - s.first);
  const Range see = visible(a, p, s.keys);
  const uint16_t* q = a.q + token * a.qs + int64_t(head) * D;
  constexpr int C = D / 64;
  constexpr float kDown = 0x1p-16f;  // sums of values next to f32's largest stay finite
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
#pragma unroll 4
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
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
      if (!((live >> i) & 1)) continue;
      const float wi = __shfl(w, i, 64);
      const int64_t ri = __shfl(row, i, 64);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(wi, value_at<S>(a, false, ri, D, c * 64 + lane) * kDown, o[c]);
    }
  }
  uint16_t* out = a.out + (token * a.H + head) * D;
  const float inv = any ? 1.0f / l : 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) out[c * 64 + lane] = f32_to_bf16(any ? o[c] * inv / kDown : 0.0f);
}

// ------------------------------------------------------------- matrix cores
constexpr int kWave = 64;
constexpr int kXcds = 8;
constexpr float kTau = 8.0f;
// f16 weights are taken times 2^kLift: the largest, 2^kTau over the lagging
// maximum, is 2^15 there, and f16's least step, 2^-24, 2^-31 of a row's largest
// weight (of many keys 17 nats below a first one, times 1, all of the weight was
// lost). Sums and results are given without it.
constexpr int kLift = 7;
// A scale of zero as the least positive number: a hidden key's score, -infinity,
// times it stays that.
constexpr float kLeastScale = 0x1p-149f;

typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

// Launch shapes. Late: the second wavefront of each SIMD multiplies by V one
// tile late, so that one's softmax meets the other's products. At D = 512 LDS
// holds one tile of K and one of V: K's next is on its way while the weights
// multiply V, V's while K meets Q.
template <int D>
struct Shape {
  static constexpr int kWaves = 8;
  static constexpr int kRW = D <= 128 ? 32 : 16;  // rows a wavefront
  static constexpr int kKeys = 64;                // keys a tile
  static constexpr bool kLate = D <= 128;
  static constexpr int kAhead = D <= 128 ? 2 : D == 256 ? 1 : 0;  // tiles in flight
  static constexpr int kKBufs = kAhead + 1, kVBufs = kAhead + 1 + (kLate ? 1 : 0);
  static constexpr int kGroupK = 2, kGroupV = 2;  // operand reads in flight
  static constexpr int kRows = kWaves * kRW;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kPieces = kKeys * D * 2 / 1024 / kWaves;  // 1 KB pieces of K (of V) a wavefront
  static_assert(kPieces >= 1 && (kKBufs + kVBufs) * kKeys * D * 2 <= 160 * 1024, "LDS");
};

// The place of 16-byte piece c in row r of a tile is c ^ turn_of(r): rows that
// fall on the same 256 bytes of LDS banks are turned against each other by two
// pieces, so that 8 rows x 2 pieces, which K's and V's reads meet at once, lie on
// banks of their own (a probe of these reads alone: 246 and 220 bytes a cycle
// and CU, 126 where rows 2 i and 2 i + 1 are turned alike at D = 128).
template <int D>
__device__ __forceinline__ int turn_of(int r) {
  constexpr int n = D >= 128 ? 1 : 128 / D;
  return 2 * ((r / n) & (8 / n - 1));
}

// 16 bytes from each lane's src to LDS [lds + 16 lane, + 16). As assembly, so
// that the compiler does not make later LDS reads wait for it; the kernel
// waits (vmcnt) before the barrier that publishes a tile. M0 holds the LDS
// address, and its write needs a wait state before the load reads it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds)
               : "memory", "m0");
}
// The same from a uniform base and a lane's offset below 2^32.
__device__ __forceinline__ void to_lds_at(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}
// At most N of the wavefront's loads outstanding.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// Reads and writes at an LDS address.
template <typename T>
__device__ __forceinline__ T read_lds(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) T*>(at);
}
__device__ __forceinline__ void write_lds(uint32_t at, u4_t x) {
  *reinterpret_cast<__attribute__((address_space(3))) u4_t*>(at) = x;
}
__device__ __forceinline__ u2_t read_transposed(uint32_t at) {
  return __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                      reinterpret_cast<__attribute__((address_space(3))) s4_t*>(at)));
}
// Operand addresses, bytes from a tile's beginning. Tiles begin at multiples of
// 1 KB, so that the pieces' turns and the operands' numbers meet in one XOR:
// K, lane (row r, group g): row r + 16 i, piece (4 s + g) turned: k_lane ^ 64 s,
// plus the rows. V: row 4 g + r / 4 (+ 16, 32 u), piece (2 t + (r / 2) % 2)
// turned: v_lane ^ 32 t.
template <int D>
__device__ __forceinline__ uint32_t k_lane(int lane) {
  const int r = lane % 16, g = lane / 16;
  return uint32_t(r * D * 2 + (g ^ turn_of<D>(r)) * 16);
}
template <int D>
__device__ __forceinline__ uint32_t v_lane(int lane) {
  const int r = 4 * (lane / 16) + lane % 16 / 4;
  return uint32_t(r * D * 2 + ((lane % 4 / 2) ^ turn_of<D>(r)) * 16 + 8 * (lane % 2));
}
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  const f2_t f = {x, y};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf2_t));
}
__device__ __forceinline__ bf2_t as_bf2(uint32_t x) { return __builtin_bit_cast(bf2_t, x); }
// acc + both halves of a packed pair.
__device__ __forceinline__ float add_two(uint32_t w, float acc) {
  const bf2_t one = {__bf16(1.0f), __bf16(1.0f)};
  return __builtin_amdgcn_fdot2_f32_bf16(as_bf2(w), one, acc, false);
}
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ h2_t as_h2(uint32_t x) { return __builtin_bit_cast(h2_t, x); }
__device__ __forceinline__ uint32_t pack_f16(float x, float y) {
  const f2_t f = {x, y};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, h2_t));
}
// Two weights as the products take them, and acc plus both as rounded.
template <bool H>
__device__ __forceinline__ uint32_t pack_weights(float x, float y) {
  return H ? pack_f16(x, y) : pack_bf16(x, y);
}
template <bool H>
__device__ __forceinline__ float add_weights(uint32_t w, float acc) {
  if constexpr (!H) return add_two(w, acc);
  const h2_t one = {_Float16(1.0f), _Float16(1.0f)};
  return __builtin_amdgcn_fdot2(as_h2(w), one, acc, false);
}

// Lane l with lanes l ^ 16 and l ^ 32 (the lanes of one row).
__device__ __forceinline__ float max_of(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float row_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = max_of(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The lane's index, where D is large computed anew at each use: what depends
// on it (addresses) is then recomputed a tile and not held in registers that
// the accumulators need.
template <int D>
__device__ __forceinline__ int lane_now(int lane) {
  if constexpr (D < 256) return lane;
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}
// Keeps a block that few tiles take behind its branch.
__device__ __forceinline__ void rare() { asm volatile(""); }

// Products of `Count` operands out of LDS, `Group` at a time: a group's reads are
// issued before the products of the group before it, which cover their
// latency. (Left to itself the compiler reads each operand right before its
// products and waits for it; a list of scheduling groups over a whole tile's
// products is ignored.) read(i) gives operand i, use(i, x) multiplies it.
template <int Count, int Group, typename Op, typename Read, typename Use>
__device__ __forceinline__ void pipelined(Read read, Use use) {
  static_assert(Count % Group == 0, "whole groups");
  Op x[2][Group];
#pragma unroll
  for (int i = 0; i < Group; ++i) x[0][i] = read(i);
#pragma unroll
  for (int g = 0; g < Count / Group; ++g) {
    if (g + 1 < Count / Group)
#pragma unroll
      for (int i = 0; i < Group; ++i) x[(g + 1) % 2][i] = read((g + 1) * Group + i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < Group; ++i) use(g * Group + i, x[g % 2][i]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// What rows of pages that are none read instead.
__device__ const uint4 kZeroRow[64] = {};

// The id-th block of KV head h, of `ids`: later ids first, a KV head's blocks
// on 8 / Hkv XCDs (workgroup i runs on XCD i % 8), several heads on one where
// there are more.
struct Unit {
  int head, id;
};
__device__ __forceinline__ Unit unit_of(const Args& a, int i) {
  int h, t;
  if (a.Hkv % kXcds == 0) {
    const int j = i / kXcds;
    h = i % kXcds + kXcds * (j / a.ids);
    t = j % a.ids;
  } else if (kXcds % a.Hkv == 0) {
    const int f = kXcds / a.Hkv;
    h = i % kXcds / f;
    t = i / kXcds * f + i % f;
  } else {
    h = i % a.Hkv;
    t = i / a.Hkv;
  }
  return Unit{h, a.ids - 1 - t};
}
// Workgroups of that (host).
inline int64_t units_of(int Hkv, int64_t ids) {
  if (Hkv < kXcds && kXcds % Hkv == 0) {
    const int f = kXcds / Hkv;
    return (ids + f - 1) / f * kXcds;
  }
  return ids * Hkv;
}

// The block with this id, of `each` rows: its sequence and first row. All lanes
// call it and get the same; false for ids that no rows need.
struct Block {
  int b;
  Sequence seq;
  int64_t row0;
};
template <Source S>
__device__ __forceinline__ bool find_block(const Args& a, int id, int each, Block* out) {
  const int lane = threadIdx.x % kWave;
  int b = -1, begin = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kWave) {
    const int i = b0 + lane;
    const int64_t at = i < a.batch ? start_of(a, i) * a.G / each + i : 0;
    const unsigned long long on = __ballot(i < a.batch && at <= id);
    if (!on) break;
    const int last = 63 - __clzll(on);
    b = b0 + last;
    begin = __shfl(int(at), last, 64);  // ids are 32-bit
    if (last < kWave - 1) break;
  }
  // Said to be alike in every lane, so that what follows runs on scalars.
  b = __builtin_amdgcn_readfirstlane(b);
  begin = __builtin_amdgcn_readfirstlane(begin);
  if (b < 0) return false;
  const Sequence s = sequence<S>(a, b);
  out->b = b;
  out->seq.first = __builtin_amdgcn_readfirstlane(int(s.first));
  out->seq.count = __builtin_amdgcn_readfirstlane(s.count);
  out->seq.keys = __builtin_amdgcn_readfirstlane(s.keys);
  out->row0 = int64_t(id - begin) * each;
  return out->row0 < int64_t(out->seq.count) * a.G;
}

__device__ __forceinline__ bool finite(f4_t v) {
  return fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY && fabsf(v[2]) < INFINITY && fabsf(v[3]) < INFINITY;
}
__device__ __forceinline__ f4_t product(bf8_t x, bf8_t y, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
}
__device__ __forceinline__ f4_t product(h8_t x, h8_t y, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
}

// A query row as the products' operand (lane group g holds channels 32 s + 8 g
// + [0, 8)), its sign that of the scale; returns what takes its scores to log2
// units, which is not negative. As f16 the row is taken times a power of two
// that brings its largest channel into [2^14, 2^15): channels below 2^-28 of
// that lose bits.
template <int D, typename Op>
__device__ __forceinline__ float load_query(const Args& a, const uint16_t* src, int g, Op (&qf)[D / 32]) {
  const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
  float scale = fabsf(a.scale) * kLog2e;
  u4_t x[D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    x[s] = *reinterpret_cast<const u4_t*>(src + 32 * s + 8 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[s][e] ^= flip;
    if constexpr (std::is_same_v<Op, bf8_t>) qf[s] = __builtin_bit_cast(bf8_t, x[s]);
  }
  if constexpr (std::is_same_v<Op, h8_t>) {
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        top = fmaxf(top, fabsf(__uint_as_float(x[s][e] << 16)));
        top = fmaxf(top, fabsf(__uint_as_float(x[s][e] & 0xffff0000u)));
      }
    top = row_max(top);
    const int up = top > 0.0f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        qf[s][2 * e] = _Float16(ldexpf(__uint_as_float(x[s][e] << 16), up));
        qf[s][2 * e + 1] = _Float16(ldexpf(__uint_as_float(x[s][e] & 0xffff0000u), up));
      }
    scale = ldexpf(scale, -up);
  }
  return scale;
}

template <int D, Source S>
__global__ __launch_bounds__(Shape<D>::kThreads)
__attribute__((amdgpu_waves_per_eu(Shape<D>::kWaves / 4))) void prompt_kernel(const Args a) {
  typedef Shape<D> W;
  constexpr int kWaves = W::kWaves, RW = W::kRW, NR = RW / 16, KT = W::kKeys, NI = KT / 16;
  constexpr int ND = D / 32, NT = D / 16, NU = KT / 32, NP = W::kPieces;
  constexpr bool F16 = S == kSlab;
  __shared__ __attribute__((aligned(1024))) uint16_t tiles[W::kKBufs + W::kVBufs][KT * D];
  const int tid = threadIdx.x, lane = tid % kWave, lr = lane % 16, lg = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);

  // The block's sequence and rows.
  const Unit unit = unit_of(a, int(blockIdx.x));
  if (unit.id < 0) return;
  const int kvh = unit.head;
  Block blk;
  if (!find_block<S>(a, unit.id, W::kRows, &blk)) return;
  const int b = blk.b;
  const Sequence seq = blk.seq;
  const int64_t rows = int64_t(seq.count) * a.G, row0 = blk.row0;
  const int64_t row_end = row0 + W::kRows < rows ? row0 + W::kRows : rows;
  const int n = seq.keys, p0 = n - seq.count;  // p0: the first query's position
  const int pos_lo = p0 + int(row0 / a.G), pos_hi = p0 + int((row_end - 1) / a.G);
  const uint32_t in_position = uint32_t(row0 % a.G);  // the block's first row
  const int split = blockIdx.y;
  // Keys that some row of the block sees, within the split.
  int key_lo = split * a.split_keys, key_hi = n;
  if (n - key_lo > a.split_keys) key_hi = key_lo + a.split_keys;
  if (a.causal) {
    if (pos_hi + 1 < key_hi) key_hi = pos_hi + 1;
    if (first_seen(a, pos_lo) > key_lo) key_lo = first_seen(a, pos_lo);
  }
  if (a.part_o && key_lo >= key_hi) return;  // the join leaves such splits out

  using op_t = std::conditional_t<F16, h8_t, bf8_t>;
  op_t qf[NR][ND];
  float qscale[NR];  // scores to log2 units
  auto row_at = [&](int j) __attribute__((always_inline)) { return row0 + wave * RW + 16 * j + lr; };
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    const int64_t r = row_at(j) < rows ? row_at(j) : rows - 1;
    const uint16_t* src = a.q + (seq.first + r / a.G) * a.qs + (int64_t(kvh) * a.G + r % a.G) * D;
    qscale[j] = load_query<D>(a, src, lg, qf[j]);
    if constexpr (F16) qscale[j] = ldexpf(qscale[j], a.exponent[2 * (b * a.Hkv + kvh)]);
    qscale[j] = fmaxf(qscale[j], kLeastScale);
  }

  // Per row: the running maximum (log2 units) and the sum.
  float m[NR], lsum[NR];
  f4_t o[NT][NR];
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    m[j] = -INFINITY;
    lsum[j] = F16 && qscale[j] * (D * 0x1p-10f) > kCoarse ? NAN : 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // V as f16 (11 bits of the values and of the weights), where its range allows.
  int v_down = kBf16;
  if constexpr (F16) v_down = __builtin_amdgcn_readfirstlane(a.exponent[2 * (b * a.Hkv + kvh) + 1]);

  if (key_lo < key_hi) {
    const int t_lo = key_lo / KT, t_hi = (key_hi - 1) / KT;
    // A wavefront fetches kMine rows of each tile, which lie in one page (of
    // 16 rows or more), in pieces of 1 KB: lane l of piece i fills place l %
    // (D / 8) of row i 512 / D + l / (D / 8), which holds the piece of the row
    // that turn_of puts there.
    constexpr int kMine = KT / kWaves, kPieceRows = 512 / D, kRowPieces = D / 8;
    static_assert(kMine == NP * kPieceRows && 16 % kMine == 0, "a wavefront's rows lie in one page");
    const std::true_type kKey{};
    const std::false_type kValue{};
    auto page_of = [&](int t) __attribute__((always_inline)) {
      // The tables are written by no one while the kernel runs.
      typedef const __attribute__((address_space(4))) int32_t* constant;
      return ((constant)(a.pool.table + b * a.pool.tstride))[t >> a.pool.shift];
    };
    // Where row t of the sequence lies, and the bytes between rows; NULL for a
    // page that is none.
    auto row_bytes = [&]() __attribute__((always_inline)) { return S == kPacked ? uint32_t(a.ts) * 2 : uint32_t(D * 2); };
    auto row_from = [&](int t, auto key) __attribute__((always_inline)) -> const char* {
      constexpr bool KEY = decltype(key)::value;
      if constexpr (S == kPacked) {
        return reinterpret_cast<const char*>((KEY ? a.k : a.v) + (seq.first + t) * a.ts + kvh * a.hs);
      } else if constexpr (S == kSlab) {
        return reinterpret_cast<const char*>((KEY ? a.slab_k : a.slab_v) + ((int64_t(b) * a.Hkv + kvh) * a.slab_rows + t) * D);
      } else {
        const int page = page_of(t);
        if (!paged::valid_page(a.pool, page)) return nullptr;
        return static_cast<const char*>(a.slot[KEY ? 0 : 1]) +
               paged::pool_row(a.pool, page, kvh, t & ((1 << a.pool.shift) - 1)) * (D * 2);
      }
    };
    auto fetch = [&](int tile, auto key, int buf) __attribute__((always_inline)) {
      constexpr bool KEY = decltype(key)::value;
      const int tc = tile < t_hi ? tile : t_hi, ln = lane_now<D>(lane);
      const uint32_t lds = lds_address(tiles[KEY ? buf : W::kKBufs + buf]) + wave * NP * 1024;
      const int first = tc * KT + wave * kMine;
      const char* base = first + kMine <= n ? row_from(first, key) : nullptr;
      if (base) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int r = i * kPieceRows + ln / kRowPieces;
          const int c = (ln % kRowPieces) ^ turn_of<D>(wave * kMine + r);
          to_lds_at(base, uint32_t(r) * row_bytes() + 16 * c, lds + i * 1024);
        }
      } else {
        // Past the last key, which is read again (hidden, and finite where it
        // is), and in no page.
        rare();
#pragma unroll 1
        for (int i = 0; i < NP; ++i) {
          const int r = i * kPieceRows + ln / kRowPieces, t = min(first + r, n - 1);
          const int c = (ln % kRowPieces) ^ turn_of<D>(wave * kMine + r);
          const char* row = row_from(t, key);
          to_lds((row ? row : reinterpret_cast<const char*>(kZeroRow)) + 16 * c, lds + i * 1024);
        }
      }
    };
    // Pages that are none, in the range that the block reads: looked for once.
    bool holes = false;
    if constexpr (S == kPagedBf16 || S == kSlab) {
      const int32_t* table = a.pool.table + b * a.pool.tstride;
      for (int i = (key_lo >> a.pool.shift) + tid; i <= (key_hi - 1) >> a.pool.shift; i += W::kThreads)
        holes |= !paged::valid_page(a.pool, table[i]);
      holes = __syncthreads_or(holes);
    }
    // Which of the tile's groups of 16 keys lie in pages.
    auto held_groups = [&](int tile) __attribute__((always_inline)) {
      uint32_t on = 0;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (paged::valid_page(a.pool, page_of(min(tile * KT + 16 * i, n - 1)))) on |= 1u << i;
      return on;
    };
    const bool live = row0 + wave * RW < rows;

    auto rescale = [&](int j, bool up, float mx) __attribute__((always_inline)) {
      const float mn = up ? mx * qscale[j] : m[j];
      const float alpha = up ? __builtin_amdgcn_exp2f(m[j] - mn) : 1.0f;
      lsum[j] *= alpha;
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t][j] *= alpha;
      m[j] = mn;
    };
    auto scores = [&](uint32_t K, f4_t (&sc)[NI][NR]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NR; ++j) sc[i][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const uint32_t at = K + k_lane<D>(lane_now<D>(lane));
      pipelined<ND * NI, W::kGroupK, op_t>(
          [&](int x) __attribute__((always_inline)) { return read_lds<op_t>((at ^ (64 * (x / NI))) + 16 * (x % NI) * D * 2); },
          [&](int x, op_t ka) __attribute__((always_inline)) {
            const int s = x / NI, i = x % NI;
#pragma unroll
            for (int j = 0; j < NR; ++j) sc[i][j] = product(ka, qf[j][s], sc[i][j]);
          });
    };
    auto softmax = [&](int tile, f4_t (&sc)[NI][NR], u4_t (&pp)[NU][NR], auto halves) __attribute__((always_inline)) {
      constexpr bool H = decltype(halves)::value;
      const int kbase = tile * KT;
      // Hidden keys, where the block sees the tile in part.
      uint32_t on = (1u << NI) - 1u;
      if constexpr (S != kPacked)
        if (holes) {
          rare();
          on = held_groups(tile);
        }
      const bool whole = kbase >= key_lo && kbase + KT <= key_hi && on == (1u << NI) - 1u &&
                         (!a.causal || (kbase + KT - 1 <= pos_lo && first_seen(a, pos_hi) <= kbase));
      if (!whole) {
        rare();
        const int ln = lane_now<D>(lane), g4 = 4 * (ln / 16);
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          const int pos = pos_lo + int((in_position + uint32_t(wave * RW + 16 * j + ln % 16)) / uint32_t(a.G));
          int hi = key_hi - kbase, lo = key_lo - kbase;  // visible: [lo, hi)
          if (a.causal) {
            hi = min(hi, pos + 1 - kbase);
            lo = max(lo, first_seen(a, pos) - kbase);
          }
#pragma unroll
          for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int k = 16 * i + g4 + r;
              if (k < lo || k >= hi || !((on >> i) & 1)) sc[i][j][r] = -INFINITY;
            }
        }
      }
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[i][j][r]);
        // (In log2 units, for which nothing more is kept: registers.)
        if (__any(mx * qscale[j] > m[j] + kTau)) {
          rare();
          mx = row_max(mx);
          rescale(j, mx * qscale[j] > m[j] + kTau, mx);
        }
        const float nm = m[j] == -INFINITY ? 0.0f : (H ? kLift : 0.0f) - m[j];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          u4_t w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f4_t s = sc[2 * u + e / 2][j];
            const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * (e % 2)], qscale[j], nm));
            const float y = __builtin_amdgcn_exp2f(fmaf(s[2 * (e % 2) + 1], qscale[j], nm));
            w[e] = pack_weights<H>(x, y);
            lsum[j] = add_weights<H>(w[e], lsum[j]);
          }
          pp[u][j] = w;
        }
      }
    };
    auto values = [&](const u4_t (&pp)[NU][NR], uint32_t V, auto halves) __attribute__((always_inline)) {
      using v_t = std::conditional_t<decltype(halves)::value, h8_t, bf8_t>;
      const uint32_t at = V + v_lane<D>(lane_now<D>(lane));
      pipelined<NU * NT, W::kGroupV, v_t>(
          [&](int x) __attribute__((always_inline)) {
            const uint32_t src = (at ^ (32 * (x % NT))) + 32 * (x / NT) * D * 2;
            const u2_t y = read_transposed(src), z = read_transposed(src + 16 * D * 2);
            return __builtin_bit_cast(v_t, u4_t{y.x, y.y, z.x, z.y});
          },
          [&](int x, v_t va) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NR; ++j)
              o[x % NT][j] = product(va, __builtin_bit_cast(v_t, pp[x / NT][j]), o[x % NT][j]);
          });
    };

    auto run = [&](auto late, auto halves) __attribute__((always_inline)) {
      constexpr bool LATE = decltype(late)::value;
      wait_loads<0>();  // the queries
      fetch(t_lo, kKey, 0);
      if constexpr (W::kAhead > 0) fetch(t_lo, kValue, 0);
      if constexpr (W::kAhead == 2) {
        fetch(t_lo + 1, kKey, 1);
        fetch(t_lo + 1, kValue, 1);
      }
      wait_loads<(W::kAhead == 2 ? 2 : 0) * NP>();
      __syncthreads();
      u4_t pp[NU][NR];
      int kc = 0, vc = 0;
      const auto plus = [](int c, int d, int bufs) { return c + d >= bufs ? c + d - bufs : c + d; };
      for (int tile = t_lo; tile <= t_hi; ++tile) {
        // Into buffers last read before the barrier that ended the tile before.
        if constexpr (W::kAhead > 0) {
          fetch(tile + W::kAhead, kKey, plus(kc, W::kAhead, W::kKBufs));
          fetch(tile + W::kAhead, kValue, plus(vc, W::kAhead, W::kVBufs));
        } else {
          fetch(tile, kValue, 0);
        }
        if (live) {
          if constexpr (W::kLate) __builtin_amdgcn_s_setprio(1);
          if constexpr (LATE)
            if (tile > t_lo) values(pp, lds_address(tiles[W::kKBufs + plus(vc, W::kVBufs - 1, W::kVBufs)]), halves);
          f4_t sc[NI][NR];
          scores(lds_address(tiles[kc]), sc);
          if constexpr (W::kLate) __builtin_amdgcn_s_setprio(0);
          softmax(tile, sc, pp, halves);
        }
        if constexpr (W::kAhead == 0) {
          // V is here, and every wavefront is done with K.
          wait_loads<0>();
          __syncthreads();
          fetch(tile + 1, kKey, 0);
        }
        if (!LATE && live) {
          if constexpr (W::kLate) __builtin_amdgcn_s_setprio(1);
          values(pp, lds_address(tiles[W::kKBufs + vc]), halves);
          if constexpr (W::kLate) __builtin_amdgcn_s_setprio(0);
        }
        wait_loads<(W::kAhead == 2 ? 2 : 0) * NP>();
        __syncthreads();
        kc = plus(kc, 1, W::kKBufs);
        vc = plus(vc, 1, W::kVBufs);
      }
      if constexpr (LATE)
        if (live) values(pp, lds_address(tiles[W::kKBufs + plus(vc, W::kVBufs - 1, W::kVBufs)]), halves);
      wait_loads<0>();  // before the workgroup's LDS is given back
    };
    auto by_order = [&](auto halves) __attribute__((always_inline)) {
      if (W::kLate && wave >= kWaves / 2) run(std::bool_constant<W::kLate>{}, halves);
      else run(std::false_type{}, halves);
    };
    if (F16 && v_down != kBf16) by_order(std::bool_constant<F16>{});
    else by_order(std::false_type{});
  }

  bool bad = false;
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    float sum = row_sum(lsum[j]);
    const int64_t r = row_at(j);
    if (F16 && v_down != kBf16) {
      sum *= 1.0f / (1 << kLift);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][j][e] = ldexpf(o[t][j][e], v_down - kLift);
    }
    if (r >= rows) continue;
    const int64_t row = (seq.first + r / a.G) * a.H + int64_t(kvh) * a.G + r % a.G;
    if (a.part_o) {
      const int64_t slot = row * a.splits + split;
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<f4_t*>(a.part_o + slot * D + 16 * t + 4 * lg) = o[t][j];
      if (lg == 0) {
        a.part_m[slot] = m[j];
        a.part_l[slot] = sum;
      }
      continue;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    bad |= !(sum > 0.0f);  // no key, none of a score above -infinity, or kCoarse
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const f4_t v = o[t][j] * inv;
      bad |= !finite(v);
      *reinterpret_cast<u2_t*>(a.out + row * D + 16 * t + 4 * lg) = u2_t{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    }
  }
  if (__any(bad)) {
    rare();
    constexpr Source R = S == kSlab ? kPagedAffine : S;
#pragma unroll 1
    for (int i = 0; i < RW; ++i) {
      const int64_t r = row0 + wave * RW + i;
      if (r >= rows) break;
      attend_row<D, R>(a, b, seq.first + r / a.G, kvh * a.G + int(r % a.G));
    }
  }
}

// Joins the splits of one (token, head) row a wavefront: those that its own
// keys meet, which its block has written.
constexpr int kJoinThreads = 256;

template <int D, Source S>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const Args a) {
  const int lane = threadIdx.x % kWave;
  const int64_t unit = int64_t(blockIdx.x) * (kJoinThreads / kWave) + threadIdx.x / kWave;
  const int64_t token = unit / a.H;
  const int head = int(unit % a.H);
  if (token >= a.tokens || token < start_of(a, 0) || token >= start_of(a, a.batch)) return;
  int b = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kWave) {
    const unsigned long long on = __ballot(b0 + lane < a.batch && start_of(a, min(b0 + lane, a.batch - 1)) <= token);
    if (!on) break;
    b = b0 + 63 - __clzll(on);
  }
  const Sequence seq = sequence<S>(a, b);
  if (token >= seq.first + seq.count) return;  // starts that do not ascend
  const Range see = visible(a, int64_t(seq.keys) - seq.count + (token - seq.first), seq.keys);
  const int64_t slot0 = (token * a.H + head) * a.splits;
  constexpr int C = D / kWave;
  float o[C], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.0f;
  if (see.lo < see.hi) {
    const int s0 = see.lo / a.split_keys, s1 = (see.hi - 1) / a.split_keys;
    for (int s = s0 + lane; s <= s1; s += kWave) m = fmaxf(m, a.part_m[slot0 + s]);
#pragma unroll
    for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d, kWave));
    // 64 splits at a time: a lane a split for the factors, then channels.
    for (int s = s0; s <= s1; s += kWave) {
      float f = 0.0f;
      if (s + lane <= s1) {
        const float ms = a.part_m[slot0 + s + lane];
        f = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - m);
        l = fmaf(f, a.part_l[slot0 + s + lane], l);
      }
      const float* part = a.part_o + (slot0 + s) * D + lane;
      const int count = min(kWave, s1 + 1 - s);
#pragma unroll 8
      for (int i = 0; i < count; ++i) {
        const float fi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i));
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = fmaf(fi, part[i * D + c * kWave], o[c]);
      }
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) l += __shfl_xor(l, d, kWave);
  }
  const float inv = 1.0f / l;
  bool bad = !(l > 0.0f);
  uint16_t* out = a.out + (token * a.H + head) * D;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const float v = o[c] * inv;
    bad |= !(fabsf(v) < INFINITY);
    out[c * kWave + lane] = f32_to_bf16(v);
  }
  constexpr Source R = S == kSlab ? kPagedAffine : S;
  if (__any(bad)) attend_row<D, R>(a, b, token, head);
}

// Launches prompt_kernel<D, S> (few_kernel of prompt_few.hpp) and, for split
// keys, the join. Defined a head dim a file.
template <int D>
void launch_prompt(const Args& a, Source s, hipStream_t st);
template <int D>
void launch_few(const Args& a, Source s, hipStream_t st);

template <int D, Source S>
void launch_source(const Args& a, hipStream_t st) {
  hipLaunchKernelGGL((prompt_kernel<D, S>), dim3(unsigned(units_of(a.Hkv, a.ids)), unsigned(a.splits)),
                     dim3(Shape<D>::kThreads), 0, st, a);
  if (a.part_o)
    hipLaunchKernelGGL((join_kernel<D, S>), dim3(unsigned((a.tokens * a.H + 3) / 4)), dim3(kJoinThreads), 0, st, a);
}
template <int D>
void launch_prompt(const Args& a, Source s, hipStream_t st) {
  if (s == kPacked) launch_source<D, kPacked>(a, st);
  else if (s == kPagedBf16) launch_source<D, kPagedBf16>(a, st);
  else launch_source<D, kSlab>(a, st);
}

}  // namespace prompt
}  // namespace tqkv

// Attention of packed sequences with few rows each over the paged cache
// (drafted tokens, the ends of prompts): bound by reading keys and values.
//
// A block's rows are all of its wavefronts', which take every kWaves-th tile
// of 32 keys for themselves: no barrier in the loop, each wavefront's tile in
// LDS of its own (K's is on its way while the weights multiply V, and V's
// while K meets Q). What the wavefronts gathered meets in LDS at the end.
//
// Affine rows are dequantized on the way into LDS, out of registers that the
// next tile's codes have been loaded into meanwhile, to f16 (bf16 would cost the
// results three bits): every row of K times a power of two that brings the
// largest value its scales and biases allow below 2^15, which its scores take
// back (rows whose steps would be more than kCoarse in a score are attend_row's); V
// times one power of two for the wavefront's rows. Where V's groups' largest values
// lie 2^28 apart (a query may see the small ones alone), attend_row does the rows.
//
// 32 sequences of up to 24,000 bf16 rows, D = 128, 6 tokens each: 117 us for 453 MB
// (3.9 TB/s; a large copy 4.9). The same of 4-bit rows: 135 to 138 us for 134 MB, of
// 8-bit rows 144 for 180; 16 sequences of 8,000, D = 256, 3 tokens each, 168 us for 296
// MB and 208 for 559. No unit bounds the affine forms (vector 42% of the CUs' cycles at 4
// bits, matrix 7%, LDS conflicts 7 to 9%): a tile is one chain of conversion, LDS and
// products, K's and then V's, with one or two wavefronts a SIMD to cover it.
#pragma once

#include "prompt_attend.hpp"

namespace tqkv {
namespace prompt {

template <int D, bool AFFINE>
struct Few {
  // (bf16 tiles of 32 KB for K and for V at D = 512: two wavefronts.)
  static constexpr int kWaves = D == 512 && !AFFINE ? 2 : 4;
  static constexpr int kRW = D >= 256 ? 16 : 32;
  static constexpr int kRows = kRW;  // a block
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kKeys = 32;
  static constexpr int kPieces = kKeys * D * 2 / 1024;
  static constexpr int kGroup = D == 128 ? 8 : 4;  // operand reads in flight
  // Tiles in a wavefront's LDS: K's and V's, or one for both in turn.
  static constexpr int kBufs = AFFINE && D >= 256 ? 1 : 2;
  // Blocks that a CU's LDS (and registers) hold, as wavefronts a SIMD.
  static constexpr int kPerEu = D == 64 ? 3 : D == 128 || (D == 256 && AFFINE) ? 2 : 1;
};

// 16 codes of 4 or 8 bits out of w (2 or 4 words) as scale * code + bias in f16,
// rounded once, two an instruction: the bits 0x6400 | c are 1,024 + c exactly (a byte's upper code 1,024 + 16 c), one
// multiply-add takes the rest off exactly, one more scales.
template <int BITS>
__device__ __forceinline__ void halves16(const uint32_t* w, h2_t s, h2_t z, uint32_t (&x)[8]) {
  constexpr uint32_t k1024 = 0x64646464u;
  if constexpr (BITS == 8) {
    const h2_t one = {_Float16(1.0f), _Float16(1.0f)}, off = {_Float16(-1024.0f), _Float16(-1024.0f)};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t at = 2 * (i % 2);
      const h2_t c = __builtin_elementwise_fma(
          as_h2(__builtin_amdgcn_perm(w[i / 2], k1024, (4u + at) | ((5u + at) << 16))), one, off);
      x[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, s, z));
    }
  } else {
    const h2_t mul = {_Float16(1.0f), _Float16(0.0625f)}, off = {_Float16(-1024.0f), _Float16(-64.0f)};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t at = 4u + i % 4;
      const uint32_t y = __builtin_amdgcn_perm(w[i / 4], k1024, at | (at << 16)) & 0x64f0640fu;
      const h2_t c = __builtin_elementwise_fma(as_h2(y), mul, off);
      x[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, s, z));
    }
  }
}

// The same of s and z times 2^up, in units in which the results are below 2^15.
// Where f16 does not hold these (its least step is 2^-24, a scale may be a 255th
// of a group's largest) they are taken times a power of two more, up to what
// brings the group's largest there too, and the results, rounded to 11 bits,
// divided by it. So a value is off by its own rounding and half a step, whatever
// the others are (scales rounded to the steps cost 8-bit values 2^22 below the
// largest their bits).
template <int BITS, bool STEPS>
__device__ __forceinline__ void halves16(const uint32_t* w, float s, float z, int up, uint32_t (&x)[8]) {
  int lift = 0;
  if constexpr (STEPS) {
    const float most = fmaxf(fabsf(z), fabsf(fmaf(s, float((1 << BITS) - 1), z)));
    lift = min(15 - __builtin_amdgcn_frexp_expf(ldexpf(most, up)), 14);
  }
  const _Float16 sh = _Float16(ldexpf(s, up + lift)), zh = _Float16(ldexpf(z, up + lift));
  halves16<BITS>(w, h2_t{sh, sh}, h2_t{zh, zh}, x);
  if constexpr (STEPS) {
    const _Float16 down = _Float16(ldexpf(1.0f, -lift));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(uint32_t, as_h2(x[i]) * h2_t{down, down});
  }
}
// The least of them but zero: f16 holds bf16's 8 bits from 2^-17 on.
__device__ __forceinline__ float least_of(float least, float s, float z) {
  return fminf(least, fminf(s != 0.0f ? fabsf(s) : INFINITY, z != 0.0f ? fabsf(z) : INFINITY));
}
constexpr float kHeld = 0x1p-17f;

template <int D, Source S, int BK, int BV>
__global__ __launch_bounds__((Few<D, S == kPagedAffine>::kThreads))
__attribute__((amdgpu_waves_per_eu(Few<D, S == kPagedAffine>::kPerEu))) void few_kernel(const Args a) {
  typedef Few<D, S == kPagedAffine> W;
  constexpr int kWaves = W::kWaves, RW = W::kRW, NR = RW / 16, KT = W::kKeys, NI = KT / 16;
  constexpr int ND = D / 32, NT = D / 16, NP = W::kPieces;
  constexpr bool AFFINE = S == kPagedAffine;
  __shared__ __attribute__((aligned(1024))) uint16_t tiles[kWaves][W::kBufs][KT * D];
  __shared__ __attribute__((aligned(16))) int32_t shifts[AFFINE ? kWaves : 1][KT];
  __shared__ float part_m[kWaves][RW], part_l[kWaves][RW];
  static_assert(sizeof(tiles[0]) >= sizeof(float) * RW * D, "what a wavefront gathered fits its tiles");
  const int tid = threadIdx.x, lane = tid % kWave, lr = lane % 16, lg = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);

  const Unit unit = unit_of(a, int(blockIdx.x));
  if (unit.id < 0) return;
  const int kvh = unit.head;
  Block blk;
  if (!find_block<S>(a, unit.id, W::kRows, &blk)) return;
  const int b = blk.b;
  const Sequence seq = blk.seq;
  const int64_t rows = int64_t(seq.count) * a.G, row0 = blk.row0;
  const int64_t row_end = row0 + RW < rows ? row0 + RW : rows;
  const int n = seq.keys, p0 = n - seq.count;
  const int pos_lo = p0 + int(row0 / a.G), pos_hi = p0 + int((row_end - 1) / a.G);
  const int split = blockIdx.y;
  int key_lo = split * a.split_keys, key_hi = n;
  if (n - key_lo > a.split_keys) key_hi = key_lo + a.split_keys;
  if (pos_hi + 1 < key_hi) key_hi = pos_hi + 1;
  if (first_seen(a, pos_lo) > key_lo) key_lo = first_seen(a, pos_lo);
  if (a.part_o && key_lo >= key_hi) return;

  int v_up = 0;  // V as f16 is taken times 2^v_up
  const int t_lo = key_lo / KT, t_hi = (key_hi - 1) / KT;  // used where key_lo < key_hi
  const bool working = key_lo < key_hi && t_lo + wave <= t_hi;

  using op_t = std::conditional_t<AFFINE, h8_t, bf8_t>;
  op_t qf[NR][ND];
  int pos[NR];
  float qscale[NR];
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    const int64_t at = row0 + 16 * j + lr, r = at < rows ? at : rows - 1;
    pos[j] = p0 + int(r / a.G);
    qscale[j] = fmaxf(load_query<D>(a, a.q + (seq.first + r / a.G) * a.qs + (int64_t(kvh) * a.G + r % a.G) * D, lg, qf[j]),
                      kLeastScale);
  }
  // The largest exponent of a key row's units that leaves f16's steps kCoarse in
  // the scores of every row here.
  int most_units = 0;
  if constexpr (AFFINE) {
    float top = qscale[0];
    if constexpr (NR == 2) top = fmaxf(top, qscale[1]);
#pragma unroll
    for (int d = 32; d > 0; d /= 2) top = fmaxf(top, __shfl_xor(top, d, kWave));
    top = fmaxf(top, 0x1p-100f) * (D * 0x1p-10f);
    most_units = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(kCoarse / top) - 1);
  }
  float m[NR], nm[NR], thr[NR], lsum[NR];
  f4_t o[NT][NR];
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    m[j] = thr[j] = -INFINITY;
    nm[j] = lsum[j] = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  uint16_t* K = tiles[wave][0];
  uint16_t* V = tiles[wave][W::kBufs - 1];
  auto page_of = [&](int t) __attribute__((always_inline)) {
    typedef const __attribute__((address_space(4))) int32_t* constant;
    return ((constant)(a.pool.table + b * a.pool.tstride))[t >> a.pool.shift];
  };

  auto scores = [&](const uint16_t* from, f4_t (&sc)[NI][NR]) __attribute__((always_inline)) {
    const uint32_t at = lds_address(from) + k_lane<D>(lane_now<AFFINE ? 512 : D>(lane));
    pipelined<ND * NI, W::kGroup, op_t>(
        [&](int x) __attribute__((always_inline)) { return read_lds<op_t>((at ^ (64 * (x / NI))) + 16 * (x % NI) * D * 2); },
        [&](int x, op_t ka) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < NR; ++j) sc[x % NI][j] = product(ka, qf[j][x / NI], sc[x % NI][j]);
        });
  };
  auto softmax = [&](int tile, f4_t (&sc)[NI][NR], u4_t (&pp)[NR], auto h) __attribute__((always_inline)) {
    constexpr bool H16 = decltype(h)::value;
    const int kbase = tile * KT;
    uint32_t on = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (paged::valid_page(a.pool, page_of(min(kbase + 16 * i, n - 1)))) on |= 1u << i;
    const bool whole = kbase >= key_lo && kbase + KT <= key_hi && on == (1u << NI) - 1u &&
                       kbase + KT - 1 <= pos_lo && first_seen(a, pos_hi) <= kbase;
    if (!whole) {
      rare();
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        const int hi = min(key_hi, pos[j] + 1) - kbase;
        const int lo = max(key_lo, first_seen(a, pos[j])) - kbase;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int k = 16 * i + 4 * lg + r;
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
      if (__any(mx > thr[j])) {
        rare();
        mx = row_max(mx);
        const bool up = mx > thr[j];
        const float mn = up ? mx * qscale[j] : m[j];
        const float alpha = up ? __builtin_amdgcn_exp2f(m[j] - mn) : 1.0f;
        lsum[j] *= alpha;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][j] *= alpha;
        m[j] = mn;
        nm[j] = mn == -INFINITY ? 0.0f : (H16 ? kLift : 0.0f) - mn;
        thr[j] = (mn + kTau) * __builtin_amdgcn_rcpf(qscale[j]);
      }
      u4_t w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f4_t s = sc[e / 2][j];
        const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * (e % 2)], qscale[j], nm[j]));
        const float y = __builtin_amdgcn_exp2f(fmaf(s[2 * (e % 2) + 1], qscale[j], nm[j]));
        w[e] = pack_weights<H16>(x, y);
        lsum[j] = add_weights<H16>(w[e], lsum[j]);
      }
      pp[j] = w;
    }
  };
  auto values = [&](const u4_t (&pp)[NR], auto halves) __attribute__((always_inline)) {
    using v_t = std::conditional_t<decltype(halves)::value, h8_t, bf8_t>;
    const uint32_t at = lds_address(V) + v_lane<D>(lane_now<AFFINE ? 512 : D>(lane));
    pipelined<NT, W::kGroup, v_t>(
        [&](int t) __attribute__((always_inline)) {
          const u2_t x = read_transposed(at ^ (32 * t)), y = read_transposed((at ^ (32 * t)) + 16 * D * 2);
          return __builtin_bit_cast(v_t, u4_t{x.x, x.y, y.x, y.y});
        },
        [&](int t, v_t va) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < NR; ++j) o[t][j] = product(va, __builtin_bit_cast(v_t, pp[j]), o[t][j]);
        });
  };
  auto clear = [&](f4_t (&sc)[NI][NR]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NR; ++j) sc[i][j] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
  };

  if (working) {
    const int t0 = t_lo + wave;
    if constexpr (!AFFINE) {
      constexpr int kPieceRows = 512 / D, kRowPieces = D / 8;
      const int lrow = lane / kRowPieces;
      // One side of a tile, 16 bytes a lane and piece (as prompt_kernel's).
      auto fetch = [&](int tile, int side) __attribute__((always_inline)) {
        const int tc = tile < t_hi ? tile : t_hi;
        const uint32_t lds = __builtin_amdgcn_readfirstlane(lds_address(tiles[wave][side]));
        int page[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) page[i] = page_of(min(tc * KT + 16 * i, n - 1));
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int r = i * kPieceRows + lrow, t = min(tc * KT + r, n - 1);
          const int c = ((lane % kRowPieces) ^ turn_of<D>(r)) * 8;
          const int pg = page[i * kPieceRows / 16];
          const bool ok = paged::valid_page(a.pool, pg);
          const int64_t at = paged::pool_row(a.pool, ok ? pg : 0, kvh, t & ((1 << a.pool.shift) - 1)) * D + c;
          const uint16_t* zero = reinterpret_cast<const uint16_t*>(kZeroRow) + c;
          to_lds(ok ? static_cast<const uint16_t*>(a.slot[side]) + at : zero, lds + i * 1024);
        }
      };
      wait_loads<0>();  // the queries
      fetch(t0, 0);
      fetch(t0, 1);
      for (int tile = t0; tile <= t_hi; tile += kWaves) {
        f4_t sc[NI][NR];
        u4_t pp[NR];
        wait_loads<NP>();  // K
        clear(sc);
        scores(K, sc);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // K's reads are done (lgkmcnt 0)
        fetch(tile + kWaves, 0);
        softmax(tile, sc, pp, std::false_type{});
        wait_loads<NP>();  // V
        values(pp, std::false_type{});
        __builtin_amdgcn_s_waitcnt(0xC07F);
        fetch(tile + kWaves, 1);
      }
      wait_loads<0>();
    } else {
      // Lane l holds the codes of row l / 2, channels [l % 2 * D / 2, + D / 2).
      constexpr int H = D / 2, KW = H * BK / 32, VW = H * BV / 32;
      const int r = lane / 2, half = lane % 2;
      // Where the lane writes piece 2 i + e of its half row: a tile's address
      // plus this, XOR 16 (2 i + e). Made anew a tile (see lane_now).
      auto place = [&](const uint16_t* tile) __attribute__((always_inline)) {
        const int ln = lane_now<512>(lane), row = ln / 2;
        return lds_address(tile) + uint32_t(row * D * 2 + ((ln % 2 * (H / 8)) ^ turn_of<D>(row)) * 16);
      };
      constexpr int NRUN = H / 32;
      // The lane's pool row of a tile; not ok: in no page (row 0 of page 0).
      auto lane_row = [&](int tile, bool& ok) __attribute__((always_inline)) {
        const int tc = tile < t_hi ? tile : t_hi;
        const int t = min(tc * KT + r, n - 1);
        const int page = r < 16 ? page_of(min(tc * KT, n - 1)) : page_of(min(tc * KT + 16, n - 1));
        ok = paged::valid_page(a.pool, page);
        return paged::pool_row(a.pool, ok ? page : 0, kvh, t & ((1 << a.pool.shift) - 1));
      };
      auto load_scales = [&](int64_t row, bool ok, int side, float (&s)[NRUN], float (&z)[NRUN]) __attribute__((always_inline)) {
        const uint16_t* sc = static_cast<const uint16_t*>(a.slot[3 * side + 1]) + row * (D / a.gs);
        const uint16_t* bi = static_cast<const uint16_t*>(a.slot[3 * side + 2]) + row * (D / a.gs);
#pragma unroll
        for (int i = 0; i < NRUN; ++i) {
          const int g = (half * H + 32 * i) / a.gs;
          s[i] = bf16_to_f32(sc[g]);
          z[i] = bf16_to_f32(bi[g]);
          if (!ok) s[i] = z[i] = 0.0f;  // hidden, and finite
        }
      };
      // One side of a tile: codes, and the scales and biases of their runs of 32.
      auto load = [&](int tile, int side, auto& codes, float (&s)[NRUN], float (&z)[NRUN]) __attribute__((always_inline)) {
        constexpr int words = sizeof(codes) / 4;
        bool ok;
        const int64_t row = lane_row(tile, ok);
        const u4_t* src = reinterpret_cast<const u4_t*>(static_cast<const uint32_t*>(a.slot[3 * side]) + (2 * row + half) * words);
#pragma unroll
        for (int i = 0; i < words / 4; ++i) codes[i] = src[i];
        load_scales(row, ok, side, s, z);
      };
      // A side's codes into its tile. The rare form in a loop of its own: a branch
      // in each step cost the others 9% of a call's time at D = 128.
      auto convert = [&](const auto& codes, const float (&s)[NRUN], const float (&z)[NRUN], int up, bool steps,
                         const uint16_t* tile, auto width) __attribute__((always_inline)) {
        constexpr int BITS = decltype(width)::value;
        const uint32_t to = place(tile);
        auto run = [&](auto form) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < H / 16; ++i) {
            uint32_t w[BITS / 2], x[8];
#pragma unroll
            for (int e = 0; e < BITS / 2; ++e) {
              w[e] = codes[(i * BITS / 2 + e) / 4][(i * BITS / 2 + e) % 4];
              // Not to be taken apart before the branch, for both: registers.
              if constexpr (decltype(form)::value) asm volatile("" : "+v"(w[e]));
            }
            halves16<BITS, decltype(form)::value>(w, s[i / 2], z[i / 2], up, x);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              write_lds(to ^ (16 * (2 * i + e)), u4_t{x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]});
            __builtin_amdgcn_sched_barrier(0);  // few values at a time: registers
          }
        };
        if (steps) {
          rare();
          run(std::true_type{});
        } else {
          run(std::false_type{});
        }
      };
      // V's range in the wavefront's tiles, by the largest values that the runs'
      // scales and biases allow (a sixteenth of the rows' bytes, read again later),
      // and the least of these. A quantizer stores zeros as codes of zero times
      // its least scale, with a bias of zero: what such runs (`plain`) allow is no
      // value. Their codes are looked at only where they would decide something:
      // in a second pass, for the first one's loads are all on their way at once.
      float v_top = 0.0f, v_low = INFINITY, v_least = INFINITY, plain_top = 0.0f, plain_least = INFINITY;
      bool fine = true;
      auto range = [&](auto codes) __attribute__((always_inline)) {
#pragma unroll 4
        for (int tile = t0; tile <= t_hi; tile += kWaves) {
          bool ok;
          const int64_t row = lane_row(tile, ok);
          float s[NRUN], z[NRUN];
          load_scales(row, ok, 1, s, z);
#pragma unroll
          for (int i = 0; i < NRUN; ++i) {
            const float x = fabsf(z[i]), y = fabsf(fmaf(s[i], float((1 << BV) - 1), z[i])), most = fmaxf(x, y);
            bool out = z[i] == 0.0f;
            if constexpr (decltype(codes)::value) {
              if (!out || !(y > 0.0f)) continue;
              const uint32_t* src = static_cast<const uint32_t*>(a.slot[3]) + (2 * row + half) * VW + i * BV;
              uint32_t any = 0;
#pragma unroll
              for (int e = 0; e < BV; ++e) any |= src[e];
              out = !any;
            } else {  // no branches: loads of several tiles at once
              fine &= x < INFINITY && y < INFINITY;
              plain_top = fmaxf(plain_top, out ? y : 0.0f);
              plain_least = fminf(plain_least, out && y > 0.0f ? fabsf(s[i]) : INFINITY);
            }
            v_top = fmaxf(v_top, out ? 0.0f : most);
            v_low = fminf(v_low, out ? INFINITY : most);
            v_least = fminf(v_least, out ? INFINITY : least_of(INFINITY, s[i], z[i]));
          }
        }
#pragma unroll
        for (int d = 32; d > 0; d /= 2) {
          v_top = fmaxf(v_top, __shfl_xor(v_top, d, kWave));
          v_low = fminf(v_low, __shfl_xor(v_low, d, kWave));
          v_least = fminf(v_least, __shfl_xor(v_least, d, kWave));
        }
      };
      auto up_of = [&]() __attribute__((always_inline)) {
        return v_top > 0.0f && v_top < INFINITY ? __builtin_amdgcn_readfirstlane(15 - __builtin_amdgcn_frexp_expf(v_top)) : 0;
      };
      range(std::false_type{});
      v_up = up_of();
      // (Of scales that f16 holds there is nothing to know: 15 times one is 2^-14.)
      if (__any(plain_top > v_top || ldexpf(plain_least, v_up) < kHeld)) {
        rare();
        range(std::true_type{});
        v_up = up_of();
      }
      // Too far apart for f16: what is no number has attend_row do the rows.
      if (!__all(fine && (v_top == 0.0f || ldexpf(v_low, v_up) >= 0x1p-14f))) {
        rare();
#pragma unroll
        for (int j = 0; j < NR; ++j) lsum[j] = NAN;
      }
      const bool v_steps = __any(ldexpf(v_least, v_up) < kHeld);
      u4_t kc[KW / 4], vc[VW / 4];
      float ks[NRUN], kz[NRUN], vs[NRUN], vz[NRUN];
      load(t0, 0, kc, ks, kz);
      load(t0, 1, vc, vs, vz);
      for (int tile = t0; tile <= t_hi; tile += kWaves) {
        f4_t sc[NI][NR];
        u4_t pp[NR];
        float top = 0.0f;  // of the lane's half row, then of the row
#pragma unroll
        for (int i = 0; i < NRUN; ++i)
          top = fmaxf(top, fmaxf(fabsf(kz[i]), fabsf(fmaf(ks[i], float((1 << BK) - 1), kz[i]))));
        top = fmaxf(top, __shfl_xor(top, 1, kWave));
        const int up = top > 0.0f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
        if (half == 0) shifts[wave][r] = -up;
        float k_least = INFINITY;
#pragma unroll
        for (int i = 0; i < NRUN; ++i) k_least = least_of(k_least, ks[i], kz[i]);
        const bool k_steps = __any(ldexpf(k_least, up) < kHeld);
        const int t = tile * KT + r;
        const bool coarse = top > 0.0f && -up > most_units && t >= key_lo && t < key_hi;
        if (__any(coarse)) {
          rare();
          int units = coarse ? -up : most_units;
#pragma unroll
          for (int d = 32; d > 0; d /= 2) units = max(units, __shfl_xor(units, d, kWave));
#pragma unroll
          for (int j = 0; j < NR; ++j)
            if (ldexpf(qscale[j], units) * (D * 0x1p-10f) > kCoarse) lsum[j] = NAN;
        }
        convert(kc, ks, kz, up, k_steps, K, std::integral_constant<int, BK>{});
        load(tile + kWaves, 0, kc, ks, kz);
        clear(sc);
        scores(K, sc);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          typedef int i4_t __attribute__((ext_vector_type(4)));
          const i4_t down = *reinterpret_cast<const i4_t*>(&shifts[wave][16 * i + 4 * lg]);
#pragma unroll
          for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[i][j][e] = ldexpf(sc[i][j][e], down[e]);
        }
        softmax(tile, sc, pp, std::true_type{});
        convert(vc, vs, vz, v_up, v_steps, V, std::integral_constant<int, BV>{});
        load(tile + kWaves, 1, vc, vs, vz);
        values(pp, std::true_type{});
      }
    }
  }

  // The wavefronts' (m, l, o) meet.
  float* mine = reinterpret_cast<float*>(tiles[wave][0]);  // [RW][D]
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    const float sum = row_sum(lsum[j]);
    if (lg == 0) {
      part_m[wave][16 * j + lr] = m[j];
      part_l[wave][16 * j + lr] = AFFINE ? sum * (1.0f / (1 << kLift)) : sum;
    }
    if constexpr (AFFINE)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][j][e] = ldexpf(o[t][j][e], -v_up - kLift);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      *reinterpret_cast<f4_t*>(mine + (16 * j + lr) * D + ((4 * t + lg) ^ (lr & 7)) * 4) = o[t][j];
  }
  __syncthreads();
  bool bad = false;
  // A thread takes four channels of a row.
  for (int i = tid; i < RW * (D / 4); i += W::kThreads) {
    const int rr = i / (D / 4), c4 = i % (D / 4);
    const int64_t r = row0 + rr;
    if (r >= rows) break;
    float top = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, part_m[w][rr]);
    f4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = part_m[w][rr] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(part_m[w][rr] - top);
      l = fmaf(f, part_l[w][rr], l);
      const f4_t x = *reinterpret_cast<const f4_t*>(reinterpret_cast<const float*>(tiles[w][0]) + rr * D + (c4 ^ (rr & 7)) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, x[e], sum[e]);
    }
    const int64_t row = (seq.first + r / a.G) * a.H + int64_t(kvh) * a.G + r % a.G;
    if (a.part_o) {
      const int64_t slot = row * a.splits + split;
      *reinterpret_cast<f4_t*>(a.part_o + slot * D + 4 * c4) = sum;
      if (c4 == 0) {
        a.part_m[slot] = top;
        a.part_l[slot] = l;
      }
      continue;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const f4_t v = sum * inv;
    bad |= !(l > 0.0f) || !finite(v);
    *reinterpret_cast<u2_t*>(a.out + row * D + 4 * c4) = u2_t{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  }
  if (a.part_o) return;
  if (__syncthreads_or(bad)) {
    rare();
#pragma unroll 1
    for (int i = wave; i < RW; i += kWaves) {
      const int64_t r = row0 + i;
      if (r >= rows) break;
      attend_row<D, S>(a, b, seq.first + r / a.G, kvh * a.G + int(r % a.G));
    }
  }
}

template <int D>
void launch_few(const Args& a, Source s, hipStream_t st) {
  const unsigned threads = s == kPagedBf16 ? Few<D, false>::kThreads : Few<D, true>::kThreads;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(units_of(a.Hkv, a.ids)), unsigned(a.splits)), dim3(threads), 0, st, a);
  };
  if (s == kPagedBf16) go(few_kernel<D, kPagedBf16, 16, 16>);
  else if (a.bits_k == 4 && a.bits_v == 4) go(few_kernel<D, kPagedAffine, 4, 4>);
  else if (a.bits_k == 4) go(few_kernel<D, kPagedAffine, 4, 8>);
  else if (a.bits_v == 4) go(few_kernel<D, kPagedAffine, 8, 4>);
  else go(few_kernel<D, kPagedAffine, 8, 8>);
  auto join = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned((a.tokens * a.H + 3) / 4)), dim3(kJoinThreads), 0, st, a);
  };
  if (a.part_o && s == kPagedBf16) join(join_kernel<D, kPagedBf16>);
  else if (a.part_o) join(join_kernel<D, kPagedAffine>);
}

}  // namespace prompt
}  // namespace tqkv

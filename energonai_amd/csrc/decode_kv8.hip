// Decode attention over the 8-bit K/V cache: one query per sequence and head, queries of a key head together.
//
// What bounds it is reading the codes, 2 D bytes a position and key head, and the split of very different lengths over the chip:
//  - Work is dealt in tiles of 64 positions (four blocks).  The waves of the launch take equal, contiguous runs of all tiles of all (sequence,
//    key head) units in a row, whatever the lengths are; the lengths are read here, and all that the caches' capacity decides is whether few or
//    short units are dealt otherwise (kv8_deal).  A unit that one wave has whole is written by it; of others each wave leaves a partial result (at most two a wave: one at either end of its
//    run), and a second, small launch combines those.
//  - Scores are S^T = K Q^T on 16x16x32 matrix instructions: rows are positions, columns the up to 16 queries that share the key head.
//    Row i of key tile t is position 4t + i%4 of block i/4 of the four.  A lane's 16 scores (column l%16) are then the 16 positions of block
//    l/16 in order, which share their scales, and, packed to 16 bits, they are in place as the operand of O^T = V^T P^T: its other operand
//    is 16 consecutive positions of a channel, which is how the values are kept.  No transposition, no LDS.
//  - Codes become 16-bit numbers exactly; the key scale multiplies the score, the value scale the probability.
//  - The running maximum is raised only where a score passes it by 2^8: the sums are fp32, and probabilities of up to 2^8 are as exact
//    in 16 bits as those below 1.
// The probabilities, times their value scale, are rounded to the cache's 16-bit type for the second product (half a step, 2^-11 or 2^-8 of
// each; the first product's operands are exact): the matrix instructions take both operands in one type, and in fp32 they are a sixteenth as
// fast.  They are relative to a reference m_o that follows score + log2(value scale), so that they neither vanish nor overflow in fp16, and
// 2^7 below it there: a product of up to 2^(7 + 8) is an fp16 number, and the smallest one that is not rounded to zero is 2^-32 of the
// largest.  The sum of the softmax takes the probabilities in fp32, relative to the scores' own maximum m_s.
#include <type_traits>

#include "kv8_common.hip.h"

namespace en {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 4 * kBlk;               // positions of a tile
constexpr int kWaves = 1024;                  // of the launch: one a SIMD, whose loads of the next tile cover the latency by themselves.  Twice
                                              // as many leave twice the partial results: 32 of up to 2000, 32 / 8 x 128 19.9 -> 25.5 us, 128 of up to 4000 104 -> 107
constexpr int kQueries = 16;                  // columns of a tile: queries that share one pass
constexpr float kRaise = 8.f;                 // log2
// log2 that a value scale counts as at least: a block without values may have the highest scores by any margin, and what is a probability's
// factor there (below: ratio) is then 2^64 and not one that takes the other blocks' scales past the fp32 numbers.
constexpr float kLeastScale = -64.f;
constexpr float kLargestFactor = 3.402823466e38f;
// log2 that the largest probability stands above 1 for its product with the values (and up to kRaise more).
template <int DT> constexpr float kStand = DT == EN_F16 ? 7.f : 0.f;
constexpr int kTeam = 8;                      // waves of a workgroup that takes one unit
constexpr int kTeamCapacity = 1024, kTeamUnits = 512;
constexpr int kWholeCapacity = 256;
// How units are dealt: runs of tiles, equal whatever the lengths are, at the cost of a second launch; a workgroup a unit, where they are
// all resident at once and a unit is at most two tiles a wave; or whole units to the waves in turn, where units are many and lengths cannot
// differ by much.  us, pages of 64: runs / a workgroup a unit: 1 sequence of 100, 12 heads x 64 8.0 / 4.7; 32 of up to 500, 12 x 64 11.3 /
// 8.2; 32 of up to 1000, 32 / 8 x 128 15.5 / 13.4, of up to 2000 19.5 / 20.2; 8 of up to 1000 11.7 / 12.2 (where the rule gives up 0.5); 1
// of 2000 10.3 / 18.1; 64 of up to 250, 40 x 128 30.1 / 44.6.  Runs / whole units: 66 of 1, 128 / 8 x 80 9.3 / 6.6; 64 of up to 60, 40 x
// 128 19.7 / 17.0; 256 of up to 100, 8 x 128 22.8 / 16.5; 64 of up to 250, 40 x 128 31.3 / 30.5, of up to 500 42.9 / 47.3; 20 of up to 500,
// 32 x 128 18.3 / 20.3; 40 of up to 2000 64 / 96.
enum class Deal { kTeam, kWhole, kRuns };
inline Deal kv8_deal(int64_t units, int64_t capacity) {
  if (units <= kTeamUnits) return capacity <= kTeamCapacity ? Deal::kTeam : Deal::kRuns;
  return capacity <= kWholeCapacity ? Deal::kWhole : Deal::kRuns;
}

template <int DT> struct Mma;
template <> struct Mma<EN_F16> {
  __device__ static __forceinline__ f32x4 k32(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x4 k16(uint2 a, uint2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t two(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)lo, (_Float16)hi});
  }
};
template <> struct Mma<EN_BF16> {
  __device__ static __forceinline__ f32x4 k32(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x4 k16(uint2 a, uint2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a), __builtin_bit_cast(i16x4, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t two(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, b16x2{(__bf16)lo, (__bf16)hi});
  }
};

// Four codes as four 16-bit numbers.
template <int DT, int CODE> __device__ __forceinline__ uint2 widen(uint32_t w) {
  if constexpr (CODE == EN_KV8_E4M3 && DT == EN_F16) {
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)));
  } else if constexpr (CODE == EN_KV8_E4M3) {
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)));
  } else if constexpr (DT == EN_F16) {
    // code + 128 behind the exponent of 1024, less 1152
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)),
                hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
    const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
    return make_uint2(__builtin_bit_cast(uint32_t, lo - off), __builtin_bit_cast(uint32_t, hi - off));
  } else {
    // seven bits and a sign: the upper half of the fp32 number is the whole of it
    const uint32_t f0 = __float_as_uint((float)(int8_t)w), f1 = __float_as_uint((float)(int8_t)(w >> 8)),
                   f2 = __float_as_uint((float)(int8_t)(w >> 16)), f3 = __float_as_uint((float)(int8_t)(w >> 24));
    return make_uint2(__builtin_amdgcn_perm(f1, f0, 0x07060302u), __builtin_amdgcn_perm(f3, f2, 0x07060302u));
  }
}
// The 16 codes of a lane as its operands of two matrix instructions.
template <int DT, int CODE> __device__ __forceinline__ void widen16(const uint4 &w, uint4 &first, uint4 &second) {
  const uint2 a = widen<DT, CODE>(w.x), b = widen<DT, CODE>(w.y), c = widen<DT, CODE>(w.z), d = widen<DT, CODE>(w.w);
  first = make_uint4(a.x, a.y, b.x, b.y);
  second = make_uint4(c.x, c.y, d.x, d.y);
}

struct Kv8AttnArgs {
  Kv8 c;
  const void *q;
  void *ctx;
  const int32_t *lens;
  int G, chunks;                // queries of a key head, and the runs of kQueries they are taken in
  float c_exp;                  // scale * log2(e)
  uint32_t *first_tile;         // [B] of a sequence, in the row of all tiles; behind them the tiles of a wave's run
  float *part_o;                // [2 waves][rows][D]
  float2 *part_ml;              // [2 waves][rows]
  int rows;                     // min(G, kQueries)
  int whole;                    // waves take whole units, every kWaves-th
};

// The length of a sequence that the whole wave asks for, as a scalar load: as a vector load, waiting for it would be waiting for the
// keys and values that are on their way.
__device__ __forceinline__ int kv8_wave_len(const Kv8 &c, const int32_t *lens, int b) {
  typedef const __attribute__((address_space(4))) int32_t *scalar_t;
  const int n = *(scalar_t)(uintptr_t)(lens + __builtin_amdgcn_readfirstlane(b));
  return min(max(n, 0), (c.max_pages << c.lg_blocks) * kBlk);
}
// What a unit counts in the row of tiles beside its tiles: its tail, the softmax's end and the output.
constexpr int kUnitCost = 1;
__device__ __forceinline__ int kv8_tiles(int n) { return max(1, (n / kBlk + 3) / 4); }

// The tiles of all units in a row: per sequence its key heads' (and chunks'), one unit behind the other.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v, int lane) {
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) {
    const uint32_t up = (uint32_t)__shfl_up((int)v, m, kWave);
    v += lane >= m ? up : 0u;
  }
  return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }

__device__ __forceinline__ float over_blocks_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float over_blocks_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// What a wave carries through a unit's tiles; lane l: query l % 16.
template <int NT> struct Kv8State {
  float m_s, m_o, l;             // l: this lane's positions only
  f32x4 o[NT];                   // channel 16 t + 4 (l / 16) + i

  __device__ __forceinline__ void clear() {
    m_s = m_o = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Raises the references where a lane's largest score (log2) or score + lv (log2 of its value scale, less kStand) passes them by kRaise.
  __device__ __forceinline__ void raise(float top, float lv) {
    const float top_o = top + lv;
    if (__ballot(top > m_s + kRaise || top_o > m_o + kRaise) == 0) return;
    const float s = fmaxf(m_s, over_blocks_max(top)), t = fmaxf(m_o, over_blocks_max(top_o));
    const float keep_l = s > -INFINITY ? __builtin_amdgcn_exp2f(m_s - s) : 1.f, keep_o = t > -INFINITY ? __builtin_amdgcn_exp2f(m_o - t) : 1.f;
    l *= keep_l;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] *= keep_o;
    m_s = s;
    m_o = t;
  }
  __device__ __forceinline__ float base() const { return m_s > -INFINITY ? m_s : 0.f; }
  // What a probability relative to m_s is multiplied by, beside the value scale, to be one relative to m_o.
  __device__ __forceinline__ float ratio() const { return m_s > -INFINITY ? __builtin_amdgcn_exp2f(m_s - m_o) : 0.f; }
};

// What a partial result of maximum m and sum l is multiplied by where the largest maximum is `top`: 0 for one without positions, and for one
// whose sum is NaN a number, so that it stays.
__device__ __forceinline__ float share_weight(float m, float l, float top) {
  return m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : l == 0.f ? 0.f : 1.f;
}
// Four channels of a row of sum l; zeros where there was no position.
template <int DT> __device__ __forceinline__ void write_row(typename Elem<DT>::T *out, float l, const f32x4 &o) {
  typedef Elem<DT> E;
  const float by = l > 0.f ? 1.f / l : l;
  Pack<typename E::T, 4> y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y.v[e] = E::from_float(l == 0.f ? 0.f : o[e] * by);
  store_pack<typename E::T, 4>(out, y);
}

// A place in the row of all tiles: sequence, unit of it (key head and run of queries), tile.
struct Kv8At {
  int b, n, tiles, tile;
  int h, chunk;
  uint32_t x;                    // its place, in tiles and units' ends
  uint32_t u;                    // the unit's among all, where waves take whole units
};

// The keys of four rows (4t .. 4t + 3 of each of four blocks) a lane as the first product wants them: 16 channels of row l % 16, run c of 64.
// Rows of 128 codes are whole cache lines, and 16 lanes x 4 of 16 bytes take half of each of 16: both halves of eight rows in one
// load instead (lanes 8.. of 16 take the other half of rows 0..7, and the first half of rows 8..15 in the second load), and the
// halves back in place by a rotation in the registers.  (The loads alone, 1031 MB of 128 sequences: bytes as they lie 190 us, so 179.)
__device__ __forceinline__ uint32_t eight_away(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true); }
__device__ __forceinline__ void halves_in_place(uint4 &x, uint4 &y, bool low) {
  const uint4 a = x, b = y;
  x = make_uint4(low ? a.x : b.x, low ? a.y : b.y, low ? a.z : b.z, low ? a.w : b.w);
  y = make_uint4(eight_away(low ? b.x : a.x), eight_away(low ? b.y : a.y), eight_away(low ? b.z : a.z), eight_away(low ? b.w : a.w));
}

// Runs of 16 channels of which a team's results go through LDS at once: all, or four where they would be more than 64 KB.
__host__ __device__ constexpr int kv8_team_tiles(int rows, int nt) { return rows > 8 && nt > 4 ? 4 : nt; }

// TEAM 1: every wave by itself, a run of tiles or (a.whole) whole units.  TEAM 8: the waves of a workgroup take the tiles of one unit in turn and
// put their results together in LDS.
template <int DT, int CODE, int NT, int TEAM>
__global__ __launch_bounds__(TEAM == 1 ? kBlock : TEAM * kWave, TEAM == 1 ? 1 : 2) void decode_attn_kv8_kernel(Kv8AttnArgs a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  typedef Mma<DT> M;
  constexpr int D = NT * 16, NC = (D + 63) / 64;            // runs of 64 channels: 16 a lane
  constexpr bool kWholeLines = D == 128;
  const int lane = threadIdx.x % kWave, col = lane % 16, g = lane / 16;
  const uint32_t member = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // neighbouring runs, which read the same pages' other heads, on one XCD (its translations and its L2): 1 to 3 %
  const uint32_t block = TEAM == 1 ? blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds : blockIdx.x;
  const uint32_t wave = block * (kBlock / kWave) + member;
  const uint32_t units = a.c.H * a.chunks;
  uint32_t end = 0;              // of this wave's run
  Kv8At at;
  // The first tile of unit u of all.
  auto place = [&](Kv8At &c, uint32_t u) {
    c.u = u;
    c.b = (int)(u / units);
    const uint32_t unit = u - (uint32_t)c.b * units;
    c.h = (int)(unit / (uint32_t)a.chunks);
    c.chunk = (int)unit - c.h * a.chunks;
    c.n = kv8_wave_len(a.c, a.lens, c.b);
    c.tiles = kv8_tiles(c.n);
    c.tile = 0;
  };
  if (TEAM == 1 && a.whole) {
    if (wave >= units * a.c.B) return;
    end = 0xffffffffu;           // a place that none of its tiles has
    place(at, wave);
    at.x = 0;
  } else if constexpr (TEAM == 1) {
    // lengths of the first 64 sequences stay in a register: few batches have more
    const int len0 = lane < a.c.B ? kv8_len(a.c, a.lens, lane) : 0;
    const uint32_t incl0 = wave_prefix(lane < a.c.B ? (kv8_tiles(len0) + kUnitCost) * units : 0u, lane);
    uint32_t all = lane_value(incl0, kWave - 1);
    for (int b0 = kWave; b0 < a.c.B; b0 += kWave)
      all += lane_value(wave_prefix(b0 + lane < a.c.B ? (kv8_tiles(kv8_len(a.c, a.lens, b0 + lane)) + kUnitCost) * units : 0u, lane), kWave - 1);
    const uint32_t quota = (all + kWaves - 1) / kWaves, x0 = wave * quota;
    if (x0 >= all) return;
    end = min(x0 + quota, all);
    // the sequence of tile x0: the first whose tiles end past it
    int len = len0;
    uint32_t incl = incl0, before = 0;
    at.b = 0;
    while (true) {
      const uint64_t past = __ballot(before + incl > x0);
      if (past) {
        const int l = __builtin_ctzll(past);
        at.b += l;
        at.n = (int)lane_value((uint32_t)len, l);
        at.tiles = kv8_tiles(at.n);
        before += lane_value(incl, l) - (at.tiles + kUnitCost) * units;
        break;
      }
      before += lane_value(incl, kWave - 1);
      at.b += kWave;
      len = at.b + lane < a.c.B ? kv8_len(a.c, a.lens, at.b + lane) : 0;
      incl = wave_prefix(at.b + lane < a.c.B ? (kv8_tiles(len) + kUnitCost) * units : 0u, lane);
    }
    const uint32_t unit = (x0 - before) / (uint32_t)(at.tiles + kUnitCost);
    at.tile = (int)(x0 - before - unit * (at.tiles + kUnitCost));
    at.h = (int)(unit / (uint32_t)a.chunks);
    at.chunk = (int)unit - at.h * a.chunks;
    // for the combine launch: the run's length, and each sequence's first tile, from the wave that comes to it
    if (wave == 0 && lane == 0) a.first_tile[a.c.B] = quota;
    at.x = x0;
    at.u = 0;
  } else {
    place(at, blockIdx.x);
    at.tile = (int)member;
    at.x = 0;
  }
  auto past = [&](const Kv8At &c) { return TEAM == 1 ? c.x >= end : c.tile >= c.tiles; };
  // The next unit's first tile, where it is still this wave's.
  auto next_unit = [&](Kv8At &c) {
    if (a.whole) {
      if (c.u + kWaves >= units * a.c.B) c.x = end;
      else place(c, c.u + kWaves);
      return;
    }
    c.x += c.tiles + kUnitCost - c.tile;
    if (c.x >= end) return;
    c.tile = 0;
    if (++c.chunk < a.chunks) return;
    c.chunk = 0;
    if (++c.h < a.c.H) return;
    c.h = 0;
    ++c.b;
    c.n = kv8_wave_len(a.c, a.lens, c.b);
    c.tiles = kv8_tiles(c.n);
  };
  auto advance = [&](Kv8At &c) {
    if (past(c)) return;
    c.tile += TEAM;
    if constexpr (TEAM == 1) {
      ++c.x;
      if (c.tile == c.tiles) next_unit(c);
    }
  };
  if (TEAM == 1 && at.tile >= at.tiles) next_unit(at);      // the run begins with a unit's end
  // Pages of a tile: of the block whose rows this lane loads as keys, and of the one whose positions it loads as values.  As the table has
  // them: what depends on them comes a tile later, and nothing waits here for the loads of keys and values in between (the ids
  // looked at where they are loaded, every tile waited for all loads: 1 sequence of 130000, 8 heads x 128 50 us, so 44; 16 of up to 8000, 40 x 64 75, so 69).
  const int last_page = max(a.c.max_pages - 1, 0);
  auto pages = [&](const Kv8At &x, int &kid, int &vid) {
    const int32_t *row = a.c.table + (int64_t)x.b * a.c.max_pages;
    kid = row[min((4 * x.tile + (col >> 2)) >> a.c.lg_blocks, last_page)];
    vid = row[min((4 * x.tile + g) >> a.c.lg_blocks, last_page)];
  };
  // The id, or -1 for a block that is none of the sequence's or has no page.
  auto checked = [&](const Kv8At &x, int block, int id) {
    return 4 * x.tile + block < x.n / kBlk && (unsigned)id < (unsigned)a.c.num_pages ? id : -1;
  };
  // Lanes without a page load from the first one, and take zeros.
  uint4 kr[4][NC], vr[NT];
  float next_ks, next_vs;
  auto load_keys = [&](const Kv8At &x, int kid) {
    const uint8_t *p = kv8_k_block(a.c, max(kid, 0), x.h, kv8_block_in_page(a.c, 4 * x.tile + (col >> 2)), D) + (col & 3) * D + 16 * g;
    if constexpr (kWholeLines) {
      // rows of lanes 0..7 first, blocks 0 and 1; then those of lanes 8..15
      const int other = (int)eight_away((uint32_t)max(kid, 0));
      const uint8_t *p2 = kv8_k_block(a.c, other, x.h, kv8_block_in_page(a.c, 4 * x.tile + ((col ^ 8) >> 2)), D) + (col & 3) * D + 16 * g + 64;
      const uint8_t *first = col < 8 ? p : p2, *second = col < 8 ? p2 : p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kr[i][0] = load16<true>(first + 4 * i * D);
        kr[i][1] = load16<true>(second + 4 * i * D);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint8_t *pc = p + (64 * c + 16 * g < D ? 64 * c : -16 * g);      // past the head: any channels, their queries are zeros
#pragma unroll
        for (int i = 0; i < 4; ++i) kr[i][c] = load16<true>(pc + 4 * i * D);
      }
    }
  };
  auto load_scales = [&](const Kv8At &x, int vid) {
    const int blk = kv8_block_in_page(a.c, 4 * x.tile + g);
    next_ks = a.c.ks[kv8_k_scale(a.c, max(vid, 0), x.h, blk)];
    next_vs = a.c.vs[kv8_v_scale(a.c, max(vid, 0), x.h, blk)];
  };
  auto load_values = [&](const Kv8At &x, int vid) {
    const uint8_t *p = kv8_v_block(a.c, max(vid, 0), x.h, kv8_block_in_page(a.c, 4 * x.tile + g), D) + col * kBlk;
#pragma unroll
    for (int i = 0; i < NT; ++i) vr[i] = load16<true>(p + i * 16 * kBlk);
  };
  // The queries of a unit: column l % 16, channels 64 c + 16 g .. of run c.  Columns and channels that are none are zeros.
  uint4 q[NC][2], next_q[NC][2];
  auto load_queries = [&](const Kv8At &x) {
    const int queries = min(kQueries, a.G - x.chunk * kQueries);
    const T *row = reinterpret_cast<const T *>(a.q) + ((((int64_t)x.b * a.c.H + x.h) * a.G + x.chunk * kQueries) + min(col, queries - 1)) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int ch = 64 * c + 16 * g;
      const uint4 *p = reinterpret_cast<const uint4 *>(row + (ch < D ? ch : 0));
      next_q[c][0] = p[0];
      next_q[c][1] = p[1];
    }
  };
  auto take_queries = [&](const Kv8At &x) {
    const int queries = min(kQueries, a.G - x.chunk * kQueries);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bool in = col < queries && 64 * c + 16 * g < D;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      q[c][0] = in ? next_q[c][0] : zero;
      q[c][1] = in ? next_q[c][1] : zero;
    }
  };

  Kv8State<NT> st;
  st.clear();
  // One tile whose keys and values are on their way; `next` follows it, its loads are issued as registers become free
  // (without a branch around them: past one, the waits for what was loaded before no longer leave them out).
  auto step = [&](const Kv8At &x, int kid, int vid, const Kv8At &next, int next_kid, int next_vid, auto more) {
    if constexpr (kWholeLines) {
#pragma unroll
      for (int i = 0; i < 4; ++i) halves_in_place(kr[i][0], kr[i][1], col < 8);
    }
    const bool whole = __ballot(kid < 0 || vid < 0) == 0;      // uniform: most tiles have all their pages
    f32x4 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!whole && kid < 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) kr[i][c] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint4 lo, hi;
        widen16<DT, CODE>(kr[i][c], lo, hi);
        s[i] = M::k32(lo, q[c][0], s[i]);
        s[i] = M::k32(hi, q[c][1], s[i]);
      }
    float ks = next_ks, vs = next_vs;
    asm volatile("" : "+v"(ks), "+v"(vs));         // here, while the loads into their registers are still to come
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (more.value) {
      load_keys(next, next_kid);
      load_scales(next, next_vid);
    }
    __builtin_amdgcn_sched_barrier(0);

    if (!whole && vid < 0) {
      ks = vs = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) vr[i] = make_uint4(0, 0, 0, 0);
    }
    const float by = ks * a.c_exp;
    const bool in = 4 * x.tile + g < x.n / kBlk;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = in ? s[i][e] * by : -INFINITY;
        top = fmaxf(top, s[i][e]);
      }
    st.raise(top, fmaxf(__builtin_amdgcn_logf(fabsf(vs)), kLeastScale) - kStand<DT>);
    const float base = st.base();
    float f = vs * st.ratio();
    f = f > kLargestFactor ? kLargestFactor : f;             // scales of 2^57 and more; NaN stays what it is
    uint32_t p[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float e4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        e4[e] = __builtin_amdgcn_exp2f(s[i][e] - base);
        st.l += e4[e];
      }
      p[2 * i] = M::two(e4[0] * f, e4[1] * f);
      p[2 * i + 1] = M::two(e4[2] * f, e4[3] * f);
    }
    const uint4 p_lo = make_uint4(p[0], p[1], p[2], p[3]), p_hi = make_uint4(p[4], p[5], p[6], p[7]);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      uint4 lo, hi;
      widen16<DT, CODE>(vr[i], lo, hi);
      st.o[i] = M::k32(lo, p_lo, st.o[i]);
      st.o[i] = M::k32(hi, p_hi, st.o[i]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (more.value) load_values(next, next_vid);
    __builtin_amdgcn_sched_barrier(0);
  };
  // The positions behind the last full block, 16 bits as they are: row i of the one key tile is position i.  Where their page is none, zeros.
  uint4 tail_k[NC][2];
  uint2 tail_v[NT];
  int tail_id;
  auto load_tail = [&](const Kv8At &x) {
    tail_id = a.c.table[(int64_t)x.b * a.c.max_pages + ((x.n / kBlk) >> a.c.lg_blocks)];
    const int64_t from = ((int64_t)x.b * a.c.H + x.h) * kBlk * D;
    const T *kt = reinterpret_cast<const T *>(a.c.kt) + from + col * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint4 *p = reinterpret_cast<const uint4 *>(kt + (64 * c + 16 * g < D ? 64 * c + 16 * g : 0));
      tail_k[c][0] = p[0];
      tail_k[c][1] = p[1];
    }
    const uint16_t *vt = reinterpret_cast<const uint16_t *>(a.c.vt) + from + col * kBlk + 4 * g;
#pragma unroll
    for (int i = 0; i < NT; ++i) tail_v[i] = *reinterpret_cast<const uint2 *>(vt + i * 16 * kBlk);
  };
  auto tail = [&](const Kv8At &x) {
    const int in_tail = x.n % kBlk;
    if ((unsigned)tail_id >= (unsigned)a.c.num_pages) {
#pragma unroll
      for (int c = 0; c < NC; ++c) tail_k[c][0] = tail_k[c][1] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NT; ++i) tail_v[i] = make_uint2(0, 0);
    }
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      // past the head: no channels, and an infinity of another one in their place would not vanish
      if (D % 64 && 64 * c + 16 * g >= D) tail_k[c][0] = tail_k[c][1] = make_uint4(0, 0, 0, 0);
      s = M::k32(tail_k[c][0], q[c][0], s);
      s = M::k32(tail_k[c][1], q[c][1], s);
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = 4 * g + e < in_tail ? s[e] * a.c_exp : -INFINITY;
      top = fmaxf(top, s[e]);
    }
    st.raise(top, -kStand<DT>);
    const float base = st.base(), f = st.ratio();
    float e4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      e4[e] = __builtin_amdgcn_exp2f(s[e] - base);
      st.l += e4[e];
    }
    const uint2 pp = make_uint2(M::two(e4[0] * f, e4[1] * f), M::two(e4[2] * f, e4[3] * f));
    // rows behind the last position may hold anything
    const uint32_t m0 = (4 * g < in_tail ? 0xffffu : 0u) | (4 * g + 1 < in_tail ? 0xffff0000u : 0u),
                   m1 = (4 * g + 2 < in_tail ? 0xffffu : 0u) | (4 * g + 3 < in_tail ? 0xffff0000u : 0u);
#pragma unroll
    for (int i = 0; i < NT; ++i) st.o[i] = M::k16(make_uint2(tail_v[i].x & m0, tail_v[i].y & m1), pp, st.o[i]);
  };

  Kv8At next = at, later;
  int kid, vid, raw_kid, raw_vid;      // of the tile; of the next one, as the table has them
  if (!past(at)) {
    pages(at, kid, vid);
    advance(next);
    pages(next, raw_kid, raw_vid);
    kid = checked(at, col >> 2, kid);
    vid = checked(at, g, vid);
    load_keys(at, kid);
    load_scales(at, vid);
    load_values(at, vid);
    load_queries(at);
    take_queries(at);
  }
  int begin = at.tile;
  bool first_segment = true;
  // a sequence's first tile is where its first unit begins
  auto note = [&](const Kv8At &c) {
    if (TEAM == 1 && !a.whole && c.tile == 0 && c.h == 0 && c.chunk == 0 && lane == 0) a.first_tile[c.b] = c.x;
  };
  auto turn = [&](auto more) {
    later = next;
    advance(later);
    int next_kid = checked(next, col >> 2, raw_kid), next_vid = checked(next, g, raw_vid);
    asm volatile("" : "+v"(next_kid), "+v"(next_vid));
    __builtin_amdgcn_sched_barrier(0);
    pages(later, raw_kid, raw_vid);
    const bool done = TEAM == 1 && at.tile + 1 == at.tiles;
    if (done) {
      // what a unit's end and the next one's beginning need is sent for a tile before
      if (at.n % kBlk) load_tail(at);
      if constexpr (more.value) load_queries(next);
    }
    __builtin_amdgcn_sched_barrier(0);
    step(at, kid, vid, next, next_kid, next_vid, more);
    if constexpr (TEAM == 1) {
      if (!more.value || done) {
        // the end of the unit, or of this wave's part of it; the loads of the next unit's first tile are on their way
        if (done && at.n % kBlk) tail(at);
        const int queries = min(kQueries, a.G - at.chunk * kQueries);
        const int64_t q_row = ((int64_t)at.b * a.c.H + at.h) * a.G + at.chunk * kQueries;
        const float l = over_blocks_sum(st.l);
        const float back = st.m_s > -INFINITY ? __builtin_amdgcn_exp2f(st.m_o - st.m_s) : 0.f;
        if (begin == 0 && done) {
          const float by = l > 0.f ? back / l : (l == l ? 0.f : l);
          if (col < queries) {
            T *out = reinterpret_cast<T *>(a.ctx) + (q_row + col) * D + 4 * g;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              Pack<T, 4> w;
#pragma unroll
              for (int e = 0; e < 4; ++e) w.v[e] = E::from_float(l == 0.f ? 0.f : st.o[i][e] * by);
              store_pack<T, 4>(out + 16 * i, w);
            }
          }
        } else if (col < queries) {
          const int64_t slot = ((int64_t)wave * 2 + (first_segment ? 0 : 1)) * a.rows + col;
          float *out = a.part_o + slot * D + 4 * g;
#pragma unroll
          for (int i = 0; i < NT; ++i) *reinterpret_cast<f32x4 *>(out + 16 * i) = st.o[i] * back;
          if (g == 0) a.part_ml[slot] = make_float2(st.m_s, l);
        }
        st.clear();
        first_segment = false;
        begin = 0;
        if constexpr (more.value) {
          take_queries(next);
          note(next);
        }
      }
    }
    at = next;
    kid = next_kid;
    vid = next_vid;
    next = later;
  };
  if (!past(at)) {
    note(at);
    while (!past(next)) turn(std::true_type{});
    turn(std::false_type{});
  }

  if constexpr (TEAM > 1) {
    extern __shared__ __align__(16) float s_part[];          // m and l [TEAM][rows] each, then [TEAM][rows][16 tiles]
    const int rows = a.rows, queries = min(kQueries, a.G - at.chunk * kQueries);
    const int tiles = kv8_team_tiles(rows, NT), width = tiles * 16;      // channels of 16 that go through LDS at a time
    float *s_m = s_part, *s_l = s_m + TEAM * rows, *s_o = s_l + TEAM * rows;
    // the tail goes to the wave that has the fewest tiles, or no more than the others
    if (at.n % kBlk && member == (uint32_t)(at.tiles % TEAM)) {
      load_tail(at);
      load_queries(at);
      take_queries(at);
      tail(at);
    }
    const float l = over_blocks_sum(st.l);
    const float back = st.m_s > -INFINITY ? __builtin_amdgcn_exp2f(st.m_o - st.m_s) : 0.f;
    const int64_t q_row = ((int64_t)at.b * a.c.H + at.h) * a.G + at.chunk * kQueries;
    if (col < queries && g == 0) {
      s_m[member * rows + col] = st.m_s;
      s_l[member * rows + col] = l;
    }
    for (int t0 = 0; t0 < NT; t0 += tiles) {
      if (t0) __syncthreads();
      if (col < queries) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i >= t0 && i < t0 + tiles) *reinterpret_cast<f32x4 *>(s_o + (member * rows + col) * width + (i - t0) * 16 + 4 * g) = st.o[i] * back;
      }
      __syncthreads();
      const int per_row = min(tiles, NT - t0) * 4;
      for (int i = threadIdx.x; i < queries * per_row; i += TEAM * kWave) {
        const int r = i / per_row, d = i % per_row * 4;
        float m = -INFINITY, sum = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < TEAM; ++w) m = fmaxf(m, s_m[w * rows + r]);
#pragma unroll
        for (int w = 0; w < TEAM; ++w) {
          const float f = share_weight(s_m[w * rows + r], s_l[w * rows + r], m);
          sum += s_l[w * rows + r] * f;
          o += *reinterpret_cast<const f32x4 *>(s_o + (w * rows + r) * width + d) * f;
        }
        write_row<DT>(reinterpret_cast<T *>(a.ctx) + (q_row + r) * D + t0 * 16 + d, sum, o);
      }
    }
  }
}

// Combines the partial results of the units that several waves had tiles of.  A workgroup takes a unit's rows: 32 lanes four channels each,
// eight groups of lanes.  Few shares: a group takes a row.  Many (one sequence of 8 key heads: 256 each): the groups take every
// eighth share of a row, and their results go through LDS; what counts then is how many are on their way at once, eight a lane.
constexpr int kCombineLanes = 32, kCombineGroups = kBlock / kCombineLanes, kAhead = 8;

template <int DT>
__global__ __launch_bounds__(kBlock) void decode_attn_kv8_combine_kernel(Kv8AttnArgs a, int D) {
  typedef typename Elem<DT>::T T;
  __shared__ f32x4 s_o[kCombineGroups][kCombineLanes];
  __shared__ float s_m[kCombineGroups], s_l[kCombineGroups];
  const uint32_t units = a.c.H * a.chunks, b = blockIdx.x / units, unit = blockIdx.x - b * units, quota = a.first_tile[a.c.B];
  const uint32_t tiles = kv8_tiles(kv8_len(a.c, a.lens, (int)b)), x0 = a.first_tile[b] + unit * (tiles + kUnitCost), x1 = x0 + tiles;
  const uint32_t w0 = x0 / quota, w1 = (x1 - 1) / quota;
  if (w0 == w1) return;                                     // one wave had it whole
  const int h = (int)unit / a.chunks, chunk = (int)unit - h * a.chunks;
  const int queries = min(kQueries, a.G - chunk * kQueries);
  const bool from_start = x0 - w0 * quota <= kUnitCost;     // the first wave's run begins with this unit, or the end of the one before
  const int group = threadIdx.x / kCombineLanes, d = threadIdx.x % kCombineLanes * 4;
  T *out = reinterpret_cast<T *>(a.ctx) + (((int64_t)b * a.c.H + h) * a.G + chunk * kQueries) * D + d;
  // what the shares w, w + step, .. of row r combine to
  auto gather = [&](int r, uint32_t w, uint32_t step, float &m, float &l, f32x4 &o) {
    m = -INFINITY;
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (; w <= w1; w += kAhead * step) {
      float2 ml[kAhead];
      f32x4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t x = min(w + j * step, w1);
        const int64_t slot = ((int64_t)x * 2 + (x == w0 && !from_start ? 1 : 0)) * a.rows + r;
        ml[j] = a.part_ml[slot];
        v[j] = *reinterpret_cast<const f32x4 *>(a.part_o + slot * D + (d < D ? d : 0));
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (w + j * step <= w1) top = fmaxf(top, ml[j].x);
      const float keep = share_weight(m, l, top);
      l *= keep;
      o *= keep;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (w + j * step > w1) continue;
        const float f = share_weight(ml[j].x, ml[j].y, top);
        l += ml[j].y * f;
        o += v[j] * f;
      }
      m = top;
    }
  };
  float m, l;
  f32x4 o;
  if (w1 - w0 < 2 * kAhead) {
    const int r = blockIdx.y * kCombineGroups + group;
    if (r < queries && d < D) {
      gather(r, w0, 1, m, l, o);
      write_row<DT>(out + r * D, l, o);
    }
    return;
  }
  for (int r = blockIdx.y; r < queries; r += gridDim.y) {
    gather(r, w0 + group, kCombineGroups, m, l, o);
    if (r != (int)blockIdx.y) __syncthreads();              // the row before has been read
    s_o[group][threadIdx.x % kCombineLanes] = o;
    if (threadIdx.x % kCombineLanes == 0) {
      s_m[group] = m;
      s_l[group] = l;
    }
    __syncthreads();
    if (group == 0 && d < D) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < kCombineGroups; ++j) top = fmaxf(top, s_m[j]);
      l = 0.f;
      o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kCombineGroups; ++j) {
        const float f = share_weight(s_m[j], s_l[j], top);
        l += s_l[j] * f;
        o += s_o[j][d / 4] * f;
      }
      write_row<DT>(out + r * D, l, o);
    }
  }
}

static int64_t kv8_part_rows(int q_heads, int head_num) { return 2 * (int64_t)kWaves * (q_heads / head_num < kQueries ? q_heads / head_num : kQueries); }

}  // namespace en

using namespace en;

extern "C" int64_t en_decode_attn_kv8_workspace_bytes(int batch, int q_heads, int head_num, int capacity, int size_per_head) {
  if (batch < 1 || head_num < 1 || q_heads < head_num || q_heads % head_num || capacity < 0 || size_per_head < 1) return 0;
  if (kv8_deal((int64_t)batch * head_num * ceil_div(q_heads / head_num, kQueries), capacity) != Deal::kRuns) return 0;
  return kv8_part_rows(q_heads, head_num) * (4 * (int64_t)size_per_head + 8) + 4 * ((int64_t)batch + 1);
}

extern "C" int en_decode_attn_kv8(const void *q, void *ctx, const en_kv8_cache *cache, const int32_t *kv_lens, int q_heads, float scale,
                                  void *workspace, int64_t workspace_bytes, en_stream_t stream) {
  if (const int bad = check_kv8(cache)) return bad;
  if (q_heads < cache->head_num || q_heads % cache->head_num) return EN_ERR_SHAPE;
  if (cache->batch == 0) return EN_OK;
  if (!q || !ctx || !kv_lens) return EN_ERR_NULL;
  if (!aligned_to(q, 16) || !aligned_to(ctx, 16) || !aligned_to(workspace, 16)) return EN_ERR_ALIGN;
  const int64_t capacity = (int64_t)cache->max_pages_per_seq * cache->page_size;
  const Deal deal = kv8_deal((int64_t)cache->batch * cache->head_num * ceil_div(q_heads / cache->head_num, kQueries), capacity);
  const bool team = deal == Deal::kTeam;
  if (deal == Deal::kRuns && !workspace) return EN_ERR_NULL;
  if (workspace_bytes < en_decode_attn_kv8_workspace_bytes(cache->batch, q_heads, cache->head_num, (int)capacity, cache->size_per_head)) return EN_ERR_SHAPE;
  Kv8AttnArgs a{kv8_args(cache), q, ctx, kv_lens, q_heads / cache->head_num, 0, scale * 1.4426950408889634f, nullptr, nullptr, nullptr, 0, 0};
  if (capacity == 0) a.c.table = kv_lens;      // no row of the table to look at: any word, which names no position
  a.whole = deal == Deal::kWhole;
  a.chunks = (int)ceil_div(a.G, kQueries);
  a.rows = a.G < kQueries ? a.G : kQueries;
  const int64_t units = (int64_t)cache->batch * cache->head_num * a.chunks;
  if (units * (ceil_div(capacity + kTile, kTile) + kUnitCost) >= INT32_MAX) return EN_ERR_SHAPE;
  const int64_t rows = kv8_part_rows(q_heads, cache->head_num);
  a.part_o = reinterpret_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(a.part_o + rows * cache->size_per_head);
  a.first_tile = reinterpret_cast<uint32_t *>(a.part_ml + rows);
  const hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto dt, auto code, auto nt) {
    constexpr int DT = decltype(dt)::value, CODE = decltype(code)::value, NT = decltype(nt)::value;
    if (team) decode_attn_kv8_kernel<DT, CODE, NT, kTeam><<<(unsigned)units, kTeam * kWave, kTeam * a.rows * (kv8_team_tiles(a.rows, NT) * 16 + 2) * 4, s>>>(a);
    else decode_attn_kv8_kernel<DT, CODE, NT, 1><<<kWaves / (kBlock / kWave), kBlock, 0, s>>>(a);
  };
  auto heads = [&](auto dt, auto code) {
    switch (cache->size_per_head) {
      case 16: launch(dt, code, std::integral_constant<int, 1>{}); break;
      case 32: launch(dt, code, std::integral_constant<int, 2>{}); break;
      case 48: launch(dt, code, std::integral_constant<int, 3>{}); break;
      case 64: launch(dt, code, std::integral_constant<int, 4>{}); break;
      case 80: launch(dt, code, std::integral_constant<int, 5>{}); break;
      case 96: launch(dt, code, std::integral_constant<int, 6>{}); break;
      case 112: launch(dt, code, std::integral_constant<int, 7>{}); break;
      default: launch(dt, code, std::integral_constant<int, 8>{}); break;
    }
  };
  auto codes = [&](auto dt) {
    if (cache->code == EN_KV8_INT8) heads(dt, std::integral_constant<int, EN_KV8_INT8>{});
    else heads(dt, std::integral_constant<int, EN_KV8_E4M3>{});
  };
  if (cache->dtype == EN_F16) codes(std::integral_constant<int, EN_F16>{});
  else codes(std::integral_constant<int, EN_BF16>{});
  EN_RETURN_IF_LAUNCH_FAILED();
  if (deal != Deal::kRuns) return EN_OK;
  // rows of a unit in workgroups of their own where units are few; where units are many, each has few shares
  const dim3 shares((unsigned)units, units >= 512 ? (unsigned)ceil_div(a.rows, kCombineGroups) : (unsigned)a.rows);
  if (cache->dtype == EN_F16) decode_attn_kv8_combine_kernel<EN_F16><<<shares, kBlock, 0, s>>>(a, cache->size_per_head);
  else decode_attn_kv8_combine_kernel<EN_BF16><<<shares, kBlock, 0, s>>>(a, cache->size_per_head);
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

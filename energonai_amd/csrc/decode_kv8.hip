// Decode attention over the 8-bit K/V cache: one query per sequence and head, queries of a key head together.
//
// What bounds it is reading the codes, 2 D bytes a position and key head, and the split of very different lengths over the chip:
//  - Work is dealt in tiles of 64 positions (four blocks).  The waves of the launch take equal, contiguous runs of all tiles of all (sequence,
//    key head) units in a row, whatever the lengths are; the lengths are read here, so nothing depends on the caches' capacity.  A
//    unit that one wave has whole is written by it; of others each wave leaves a partial result (at most two a wave: one at either end of its
//    run), and a second, small launch combines those.
//  - Scores are S^T = K Q^T on 16x16x32 matrix instructions: rows are positions, columns the up to 16 queries that share the key head.
//    Row i of key tile t is position 4t + i%4 of block i/4 of the four.  A lane's 16 scores (column l%16) are then the 16 positions of block
//    l/16 in order, which share their scales, and, packed to 16 bits, they are in place as the operand of O^T = V^T P^T: its other operand
//    is 16 consecutive positions of a channel, which is how the values are kept.  No transposition, no LDS.
//  - Codes become 16-bit numbers exactly; the key scale multiplies the score, the value scale the probability.
//  - The running maximum is raised only where a score passes it by 2^8: the sums are fp32, and probabilities of up to 2^8 are as exact
//    in 16 bits as those below 1.
// The probabilities are rounded to the cache's 16-bit type for the second product (half a step, 2^-12 or 2^-9, each; the first product's operands
// are exact), relative to a reference m_o that follows score + log2(value scale), so that their products with the scale neither
// vanish nor overflow in fp16; the sum of the softmax takes them in fp32 relative to the scores' own maximum m_s.
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
constexpr int kWaves = 2048;                  // of the launch: two a SIMD, and what of the registers they leave holds loads in flight
constexpr int kQueries = 16;                  // columns of a tile: queries that share one pass
constexpr float kRaise = 8.f;                 // log2

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
  uint32_t waves;
  float *part_o;                // [2 waves][rows][D]
  float2 *part_ml;              // [2 waves][rows]
  int rows;                     // min(G, kQueries)
};

__device__ __forceinline__ int kv8_tiles(int n) { return max(1, (n / kBlk + 3) / 4); }

// The tiles of all units in a row: per sequence its key heads' (and chunks'), one unit behind the other.
struct Kv8Plan {
  uint32_t units, all, quota;    // units a sequence; tiles; tiles a wave
};
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) v += (uint32_t)__shfl_xor((int)v, m, kWave);
  return v;
}
__device__ __forceinline__ Kv8Plan kv8_plan(const Kv8AttnArgs &a, int lane) {
  uint32_t sum = 0;
  for (int b = lane; b < a.c.B; b += kWave) sum += kv8_tiles(kv8_len(a.c, a.lens, b));
  Kv8Plan p;
  p.units = a.c.H * a.chunks;
  p.all = __builtin_amdgcn_readfirstlane(wave_sum(sum)) * p.units;
  p.quota = (p.all + a.waves - 1) / a.waves;
  return p;
}
// Sequence that tile x belongs to, and the tiles before that sequence.
__device__ __forceinline__ void kv8_find(const Kv8AttnArgs &a, const Kv8Plan &p, uint32_t x, int lane, int &b, uint32_t &before) {
  before = 0;
  for (int b0 = 0;; b0 += kWave) {
    uint32_t incl = b0 + lane < a.c.B ? kv8_tiles(kv8_len(a.c, a.lens, b0 + lane)) * p.units : 0u;
    const uint32_t mine = incl;
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
      const uint32_t up = (uint32_t)__shfl_up((int)incl, m, kWave);
      incl += lane >= m ? up : 0u;
    }
    const uint64_t past = __ballot(before + incl > x);
    if (past || b0 + kWave >= a.c.B) {
      const int l = past ? __builtin_ctzll(past) : kWave - 1;
      b = b0 + l;
      before += (uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), l);
      return;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)incl, kWave - 1);
  }
}

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
  // Raises the references where a lane's largest score (log2) or score + log2 of its value scale passes them by kRaise.
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

template <int DT, int CODE, int NT>
__global__ __launch_bounds__(kBlock, 2) void decode_attn_kv8_kernel(Kv8AttnArgs a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  typedef Mma<DT> M;
  constexpr int D = NT * 16, NC = (D + 63) / 64;            // runs of 64 channels: 16 a lane
  const int lane = threadIdx.x % kWave, col = lane % 16, g = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave);
  const Kv8Plan plan = kv8_plan(a, lane);
  const uint32_t x0 = wave * plan.quota;
  if (x0 >= plan.all) return;
  uint32_t left = min(plan.quota, plan.all - x0);
  int b;
  uint32_t before;
  kv8_find(a, plan, x0, lane, b, before);
  b = __builtin_amdgcn_readfirstlane(b);
  before = __builtin_amdgcn_readfirstlane(before);
  int n = kv8_len(a.c, a.lens, b), tiles = kv8_tiles(n);
  uint32_t unit = (x0 - before) / (uint32_t)tiles;
  int tile = (int)(x0 - before - unit * tiles);
  bool first_segment = true;

  while (true) {
    const int h = (int)unit / a.chunks, chunk = (int)unit - h * a.chunks;
    const int queries = min(kQueries, a.G - chunk * kQueries);
    const int end = (int)min((uint32_t)tiles, tile + left);          // tiles [tile, end) of this unit are this wave's
    const int begin = tile, blocks = n / kBlk;
    const int64_t q_row = ((int64_t)b * a.c.H + h) * a.G + chunk * kQueries;

    // the queries: column l % 16, channels 64 c + 16 g .. of run c
    uint4 q[NC][2];
    {
      const T *row = reinterpret_cast<const T *>(a.q) + (q_row + min(col, queries - 1)) * D;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int ch = 64 * c + 16 * g;
        const bool in = col < queries && ch < D;
        const uint4 *p = reinterpret_cast<const uint4 *>(row + (ch < D ? ch : 0));
        const uint4 zero = make_uint4(0, 0, 0, 0), x = p[0], y = p[1];
        q[c][0] = in ? x : zero;
        q[c][1] = in ? y : zero;
      }
    }
    Kv8State<NT> st;
    st.clear();

    // Page ids of a tile: of the block whose rows this lane loads as keys, and of the one whose positions it loads as values.
    auto pages = [&](int t, int &kid, int &vid) {
      const int kb = 4 * t + (col >> 2), vb = 4 * t + g;
      kid = kb < blocks ? kv8_page(a.c, b, kb) : -1;
      vid = vb < blocks ? kv8_page(a.c, b, vb) : -1;
    };
    // Lanes without a page load what lies at the pool's start, and take zeros.
    uint4 kr[4][NC], vr[NT];
    float ks, vs;
    auto load_keys = [&](int t, int kid) {
      const int blk = kv8_block_in_page(a.c, 4 * t + (col >> 2));
      const uint8_t *p = kid >= 0 ? kv8_k_block(a.c, kid, h, blk, D) + (col & 3) * D : a.c.kp;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int ch = 64 * c + 16 * g < D ? 64 * c + 16 * g : 0;      // past the head: any channels, their queries are zeros
          kr[i][c] = load16<true>(kid >= 0 ? p + 4 * i * D + ch : p);
        }
    };
    auto load_values = [&](int t, int vid) {
      const int blk = kv8_block_in_page(a.c, 4 * t + g);
      const uint8_t *p = vid >= 0 ? kv8_v_block(a.c, vid, h, blk, D) + col * kBlk : a.c.vp;
#pragma unroll
      for (int i = 0; i < NT; ++i) vr[i] = load16<true>(vid >= 0 ? p + i * 16 * kBlk : p);
      ks = a.c.ks[vid >= 0 ? kv8_k_scale(a.c, vid, h, blk) : 0];
      vs = a.c.vs[vid >= 0 ? kv8_v_scale(a.c, vid, h, blk) : 0];
    };

    int kid, vid, next_kid, next_vid;
    pages(begin, kid, vid);
    load_keys(begin, kid);
    load_values(begin, vid);
    pages(begin + 1, next_kid, next_vid);
    for (int t = begin; t < end; ++t) {
      int after_kid, after_vid;
      pages(t + 2, after_kid, after_vid);
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
      __builtin_amdgcn_sched_barrier(0);
      if (t + 1 < end) load_keys(t + 1, next_kid);
      __builtin_amdgcn_sched_barrier(0);

      if (!whole && vid < 0) {
        ks = vs = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i) vr[i] = make_uint4(0, 0, 0, 0);
      }
      const float by = ks * a.c_exp;
      const bool in = 4 * t + g < blocks;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = in ? s[i][e] * by : -INFINITY;
          top = fmaxf(top, s[i][e]);
        }
      st.raise(top, fmaxf(__builtin_amdgcn_logf(fabsf(vs)), -126.f));
      const float base = st.base(), f = vs * st.ratio();
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
      if (t + 1 < end) load_values(t + 1, next_vid);
      __builtin_amdgcn_sched_barrier(0);
      kid = next_kid;
      vid = next_vid;
      next_kid = after_kid;
      next_vid = after_vid;
    }

    const int in_tail = n % kBlk;
    if (end == tiles && in_tail) {
      // the positions behind the last full block, 16 bits as they are: row i of the one key tile is position i
      const int64_t at = ((int64_t)b * a.c.H + h) * kBlk * D;
      const T *kt = reinterpret_cast<const T *>(a.c.kt) + at + col * D;
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int ch = 64 * c + 16 * g < D ? 64 * c + 16 * g : 0;
        const uint4 *p = reinterpret_cast<const uint4 *>(kt + ch);
        s = M::k32(p[0], q[c][0], s);
        s = M::k32(p[1], q[c][1], s);
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = 4 * g + e < in_tail ? s[e] * a.c_exp : -INFINITY;
        top = fmaxf(top, s[e]);
      }
      st.raise(top, 0.f);
      const float base = st.base(), f = st.ratio();
      float e4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        e4[e] = __builtin_amdgcn_exp2f(s[e] - base);
        st.l += e4[e];
      }
      const uint2 pp = make_uint2(M::two(e4[0] * f, e4[1] * f), M::two(e4[2] * f, e4[3] * f));
      const uint16_t *vt = reinterpret_cast<const uint16_t *>(a.c.vt) + at + col * kBlk + 4 * g;
      // rows behind the last position may hold anything
      const uint32_t m0 = (4 * g < in_tail ? 0xffffu : 0u) | (4 * g + 1 < in_tail ? 0xffff0000u : 0u),
                     m1 = (4 * g + 2 < in_tail ? 0xffffu : 0u) | (4 * g + 3 < in_tail ? 0xffff0000u : 0u);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint2 w = *reinterpret_cast<const uint2 *>(vt + i * 16 * kBlk);
        st.o[i] = M::k16(make_uint2(w.x & m0, w.y & m1), pp, st.o[i]);
      }
    }

    const float l = over_blocks_sum(st.l);
    const float back = st.m_s > -INFINITY ? __builtin_amdgcn_exp2f(st.m_o - st.m_s) : 0.f;
    if (begin == 0 && end == tiles) {
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

    left -= (uint32_t)(end - begin);
    if (left == 0) return;
    first_segment = false;
    tile = 0;
    if (++unit == plan.units) {
      unit = 0;
      ++b;
      n = kv8_len(a.c, a.lens, b);
      tiles = kv8_tiles(n);
    }
  }
}

// Combines the partial results of the units that several waves had tiles of: four channels a lane, the waves' shares in turn.
template <int DT>
__global__ __launch_bounds__(kBlock) void decode_attn_kv8_combine_kernel(Kv8AttnArgs a, int D) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  const int lane = threadIdx.x % kWave;
  const Kv8Plan plan = kv8_plan(a, lane);
  const int b = blockIdx.x / plan.units;
  const uint32_t unit = blockIdx.x - (uint32_t)b * plan.units;
  uint32_t sum = 0;
  for (int i = lane; i < b; i += kWave) sum += kv8_tiles(kv8_len(a.c, a.lens, i));
  const uint32_t tiles = kv8_tiles(kv8_len(a.c, a.lens, b));
  const uint32_t x0 = __builtin_amdgcn_readfirstlane(wave_sum(sum)) * plan.units + unit * tiles, x1 = x0 + tiles;
  const uint32_t w0 = x0 / plan.quota, w1 = (x1 - 1) / plan.quota;
  if (w0 == w1) return;                                     // one wave had it whole
  const int h = (int)unit / a.chunks, chunk = (int)unit - h * a.chunks;
  const int queries = min(kQueries, a.G - chunk * kQueries);
  const bool from_start = x0 == w0 * plan.quota;            // the first wave's run begins with this unit
  for (int i = threadIdx.x; i < queries * (D / 4); i += kBlock) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    constexpr int kAhead = 4;
    for (uint32_t w = w0; w <= w1; w += kAhead) {
      float2 ml[kAhead];
      f32x4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t x = min(w + j, w1);
        const int64_t slot = ((int64_t)x * 2 + (x == w0 && !from_start ? 1 : 0)) * a.rows + r;
        ml[j] = a.part_ml[slot];
        v[j] = *reinterpret_cast<const f32x4 *>(a.part_o + slot * D + d);
        if (w + j > w1) ml[j].x = -INFINITY;
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) top = fmaxf(top, ml[j].x);
      if (top == -INFINITY) continue;
      const float keep = __builtin_amdgcn_exp2f(m - top);
      l *= keep;
      o *= keep;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (w + j > w1) continue;
        const float f = __builtin_amdgcn_exp2f(ml[j].x - top);
        l += ml[j].y * f;
        o += v[j] * f;
      }
      m = top;
    }
    const float by = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    Pack<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = E::from_float(l == 0.f ? 0.f : o[e] * by);
    store_pack<T, 4>(reinterpret_cast<T *>(a.ctx) + (((int64_t)b * a.c.H + h) * a.G + chunk * kQueries + r) * D + d, y);
  }
}

static int64_t kv8_part_rows(int q_heads, int head_num) { return 2 * (int64_t)kWaves * (q_heads / head_num < kQueries ? q_heads / head_num : kQueries); }

}  // namespace en

using namespace en;

extern "C" int64_t en_decode_attn_kv8_workspace_bytes(int batch, int q_heads, int head_num, int capacity, int size_per_head) {
  if (batch < 1 || head_num < 1 || q_heads < head_num || q_heads % head_num || capacity < 0 || size_per_head < 1) return 0;
  return kv8_part_rows(q_heads, head_num) * (4 * (int64_t)size_per_head + 8);
}

extern "C" int en_decode_attn_kv8(const void *q, void *ctx, const en_kv8_cache *cache, const int32_t *kv_lens, int q_heads, float scale,
                                  void *workspace, int64_t workspace_bytes, en_stream_t stream) {
  if (const int bad = check_kv8(cache)) return bad;
  if (q_heads < cache->head_num || q_heads % cache->head_num) return EN_ERR_SHAPE;
  if (cache->batch == 0) return EN_OK;
  if (!q || !ctx || !kv_lens || !workspace) return EN_ERR_NULL;
  if (!aligned_to(q, 16) || !aligned_to(ctx, 16) || !aligned_to(workspace, 16)) return EN_ERR_ALIGN;
  const int64_t capacity = (int64_t)cache->max_pages_per_seq * cache->page_size;
  if (workspace_bytes < en_decode_attn_kv8_workspace_bytes(cache->batch, q_heads, cache->head_num, (int)capacity, cache->size_per_head)) return EN_ERR_SHAPE;
  Kv8AttnArgs a{kv8_args(cache), q, ctx, kv_lens, q_heads / cache->head_num, 0, scale * 1.4426950408889634f, kWaves, nullptr, nullptr, 0};
  a.chunks = (int)ceil_div(a.G, kQueries);
  a.rows = a.G < kQueries ? a.G : kQueries;
  const int64_t units = (int64_t)cache->batch * cache->head_num * a.chunks;
  if (units * ceil_div(capacity + kTile, kTile) >= INT32_MAX) return EN_ERR_SHAPE;
  const int64_t rows = kv8_part_rows(q_heads, cache->head_num);
  a.part_o = reinterpret_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(a.part_o + rows * cache->size_per_head);
  const hipStream_t s = (hipStream_t)stream;
  const unsigned grid = kWaves / (kBlock / kWave);
  auto heads = [&](auto dt, auto code) {
    constexpr int DT = decltype(dt)::value, CODE = decltype(code)::value;
    switch (cache->size_per_head) {
      case 16: decode_attn_kv8_kernel<DT, CODE, 1><<<grid, kBlock, 0, s>>>(a); break;
      case 32: decode_attn_kv8_kernel<DT, CODE, 2><<<grid, kBlock, 0, s>>>(a); break;
      case 48: decode_attn_kv8_kernel<DT, CODE, 3><<<grid, kBlock, 0, s>>>(a); break;
      case 64: decode_attn_kv8_kernel<DT, CODE, 4><<<grid, kBlock, 0, s>>>(a); break;
      case 80: decode_attn_kv8_kernel<DT, CODE, 5><<<grid, kBlock, 0, s>>>(a); break;
      case 96: decode_attn_kv8_kernel<DT, CODE, 6><<<grid, kBlock, 0, s>>>(a); break;
      case 112: decode_attn_kv8_kernel<DT, CODE, 7><<<grid, kBlock, 0, s>>>(a); break;
      default: decode_attn_kv8_kernel<DT, CODE, 8><<<grid, kBlock, 0, s>>>(a); break;
    }
  };
  auto codes = [&](auto dt) {
    if (cache->code == EN_KV8_INT8) heads(dt, std::integral_constant<int, EN_KV8_INT8>{});
    else heads(dt, std::integral_constant<int, EN_KV8_E4M3>{});
  };
  if (cache->dtype == EN_F16) codes(std::integral_constant<int, EN_F16>{});
  else codes(std::integral_constant<int, EN_BF16>{});
  EN_RETURN_IF_LAUNCH_FAILED();
  if (cache->dtype == EN_F16) decode_attn_kv8_combine_kernel<EN_F16><<<(unsigned)units, kBlock, 0, s>>>(a, cache->size_per_head);
  else decode_attn_kv8_combine_kernel<EN_BF16><<<(unsigned)units, kBlock, 0, s>>>(a, cache->size_per_head);
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

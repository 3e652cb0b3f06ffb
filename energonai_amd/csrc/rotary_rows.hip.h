// One head's row on its way from the projection: RMS norm over its channels and rotation by its position, in registers.
//
// A row of D channels is taken by LPR lanes, NP units each; a unit is two vectors of VEC channels, a and b, that hold both channels
// of every pair they have a part in, so that the rotation needs no other lane: channels u VEC .. and R/2 + u VEC .. of the rotated part; where
// pairs are neighbouring channels, and in the rest of the row, any two, and those are taken whose neighbours the neighbouring lanes take, so
// that a load fills cache lines (4 prompts of 8000, 80 heads x 128, neighbouring pairs: 357 us where a unit's vectors are neighbours, so 212).  Only the norm's sum crosses lanes.
// VEC is the largest of 8 (16-bit rows), 4, 2, 1 that divides R/2 and D (interleaved: R and D), a property of the head alone:
// loads and stores take any element's address.
#pragma once

#include <type_traits>

#include "common.hip.h"

namespace en {

constexpr int kRotaryMaxHead = 256;

typedef uint16_t u16_by2;
typedef uint32_t u32_by2 __attribute__((aligned(2)));
typedef uint32_t u32x2_by2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_by4 __attribute__((aligned(4)));
typedef uint32_t u32x2_by4 __attribute__((ext_vector_type(2), aligned(4)));
template <int SIZE, int BYTES> struct LooseType;
template <> struct LooseType<2, 2> { typedef u16_by2 type; };
template <> struct LooseType<2, 4> { typedef u32_by2 type; };
template <> struct LooseType<2, 8> { typedef u32x2_by2 type; };
template <> struct LooseType<2, 16> { typedef u32x4_by2 type; };
template <> struct LooseType<4, 4> { typedef u32_by4 type; };
template <> struct LooseType<4, 8> { typedef u32x2_by4 type; };
template <> struct LooseType<4, 16> { typedef u32x4_by4 type; };

// VEC elements at an address aligned to one of them.
template <typename T, int VEC, bool NT = false>
__device__ __forceinline__ Pack<T, VEC> load_loose(const T *p) {
  typedef typename LooseType<sizeof(T), sizeof(T) * VEC>::type W;
  const W w = NT ? __builtin_nontemporal_load(reinterpret_cast<const W *>(p)) : *reinterpret_cast<const W *>(p);
  Pack<T, VEC> r;
  __builtin_memcpy(&r, &w, sizeof(r));
  return r;
}
template <bool NT, typename T, int VEC>
__device__ __forceinline__ void store_loose(T *p, const Pack<T, VEC> &x) {
  typedef typename LooseType<sizeof(T), sizeof(T) * VEC>::type W;
  W w;
  __builtin_memcpy(&w, &x, sizeof(x));
  if constexpr (NT) __builtin_nontemporal_store(w, reinterpret_cast<W *>(p));
  else *reinterpret_cast<W *>(p) = w;
}

struct RotaryHow {
  const float *cos, *sin;
  const void *q_weight, *k_weight;
  int rows, R, D;
  int rest;             // half the vectors behind the rotated part, rounded up: how far apart the two of a unit there are
  float eps;
};

template <int DT, int VEC, int LPR, int NP, bool IL> struct RotaryRow {
  typedef Elem<DT> E;
  typedef typename E::T T;
  typedef Pack<T, VEC> P;
  P raw[NP][2];

  // First channel of vector `half` of unit u; D or more where the row has none.
  __device__ static __forceinline__ int channel(const RotaryHow &w, int u, int half) {
    if (IL) return VEC == 1 ? 2 * u + half : (u + half * LPR * NP) * VEC;
    const int turned = w.R / 2 / VEC;
    if (u < turned) return u * VEC + half * (w.R / 2);
    return u - turned < w.rest ? w.R + (u - turned + half * w.rest) * VEC : w.D;
  }
  template <bool NT = false> __device__ __forceinline__ void load(const RotaryHow &w, const T *row, int lane) {
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int c = channel(w, lane + i * LPR, half);
        raw[i][half] = load_loose<T, VEC, NT>(row + (c < w.D ? c : 0));
      }
  }
};

// The cos and sin of a lane's units at one position: f[0] cos, f[1] sin.  VEC pairs a unit; of neighbouring pairs, the first half of them
// is the first vector's.
template <int VEC, int LPR, int NP, bool IL> struct RotaryTurn {
  float f[NP][2][VEC];

  __device__ __forceinline__ void load(const RotaryHow &w, int64_t pos, int lane) {
    const bool in = (uint64_t)pos < (uint64_t)w.rows;
    const int half_dim = w.R / 2;
    const int64_t at = (in ? pos : 0) * half_dim;
    constexpr int PER = IL && VEC > 1 ? VEC / 2 : VEC, N = PER < 4 ? PER : 4;      // pairs a vector; R is made of vectors
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < VEC; e += N) {
        const int u = lane + i * LPR, first = PER == VEC ? u * VEC + e : (u + (e / PER) * LPR * NP) * PER + e % PER;
        const bool turned = first < half_dim;
        const Pack<float, N> c = turned ? load_loose<float, N>(w.cos + at + first) : Pack<float, N>{},
                             s = turned ? load_loose<float, N>(w.sin + at + first) : Pack<float, N>{};
#pragma unroll
        for (int j = 0; j < N; ++j) {
          f[i][0][e + j] = in ? c.v[j] : __builtin_nanf("");
          f[i][1][e + j] = in ? s.v[j] : __builtin_nanf("");
        }
      }
  }
};

__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }
template <int DT> __device__ __forceinline__ typename Elem<DT>::T round_to(float v) { return Elem<DT>::from_float(v); }
// From 64 bits by way of 32, rounded there to odd: the second rounding is then the only one.
template <int DT> __device__ __forceinline__ typename Elem<DT>::T round_to(double v) {
  const float f = (float)v;
  uint32_t u = __float_as_uint(f);
  const double back = (double)f;
  if (back != v && v == v && f != 0.f && !(u & 1)) u += (back < v) == (f > 0.f) ? 1 : -1;      // towards v, which lies between f and its odd neighbour
  return Elem<DT>::from_float(__uint_as_float(u));
}
template <int WIDTH> __device__ __forceinline__ float lanes_sum(float v) { return group_allreduce<OpSum, WIDTH>(v); }
template <int WIDTH> __device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
  for (int m = 1; m < WIDTH; m *= 2) v += __shfl_xor(v, m, kWave);
  return v;
}

// y of the row in `r`, in place, computed in A.  Called by all lanes of the wave.
template <typename A = float, int DT, int VEC, int LPR, int NP, bool IL>
__device__ __forceinline__ void norm_and_turn(const RotaryHow &w, RotaryRow<DT, VEC, LPR, NP, IL> &r, const RotaryTurn<VEC, LPR, NP, IL> &turn,
                                              const void *weight, int lane) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  typedef RotaryRow<DT, VEC, LPR, NP, IL> Row;
  A x[NP][2][VEC];
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[i][half][e] = E::to_float(r.raw[i][half].v[e]);
  if (weight) {
    A s = 0;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        if (Row::channel(w, lane + i * LPR, half) < w.D)
#pragma unroll
          for (int e = 0; e < VEC; ++e) s += x[i][half][e] * x[i][half][e];
    const A inv = A(1) / sqrt(lanes_sum<LPR>(s) / A(w.D) + A(w.eps));
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int c = Row::channel(w, lane + i * LPR, half);
        const Pack<T, VEC> g = load_loose<T, VEC>(reinterpret_cast<const T *>(weight) + (c < w.D ? c : 0));
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[i][half][e] = x[i][half][e] * inv * A(E::to_float(g.v[e]));
      }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if constexpr (IL && VEC > 1) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const bool turned = Row::channel(w, lane + i * LPR, half) < w.R;      // the others stay what they are, infinities too
          const A c = turn.f[i][0][(half * VEC + e) / 2], s = turn.f[i][1][(half * VEC + e) / 2];
          const A a = x[i][half][e], b = x[i][half][e + 1];
          x[i][half][e] = turned ? fused(a, c, -(b * s)) : a;
          x[i][half][e + 1] = turned ? fused(b, c, a * s) : b;
        }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool turned = (lane + i * LPR) * VEC < w.R / 2;
        const A a = x[i][0][e], b = x[i][1][e], c = turn.f[i][0][e], s = turn.f[i][1][e];
        x[i][0][e] = turned ? fused(a, c, -(b * s)) : a;
        x[i][1][e] = turned ? fused(b, c, a * s) : b;
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.raw[i][half].v[e] = round_to<DT>(x[i][half][e]);
  }
}

template <bool NT, int DT, int VEC, int LPR, int NP, bool IL>
__device__ __forceinline__ void store_row(const RotaryHow &w, const RotaryRow<DT, VEC, LPR, NP, IL> &r, typename Elem<DT>::T *row, int lane) {
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = RotaryRow<DT, VEC, LPR, NP, IL>::channel(w, lane + i * LPR, half);
      if (c < w.D) store_loose<NT, typename Elem<DT>::T, VEC>(row + c, r.raw[i][half]);
    }
}

// ---- host side: which form a head takes --------------------------------------------------------------------------------------------

// Vector width and lanes a row; every form the launches know.
struct RotaryForm { int vec, lpr; };
inline RotaryForm rotary_form(int D, int R, bool interleaved, int dtype) {
  int vec = dtype == EN_F32 ? 4 : 8;
  auto fits = [&](int v) { return D % v == 0 && (interleaved ? R % v == 0 : (R / 2) % v == 0); };
  while (vec > 1 && !fits(vec)) vec /= 2;
  const int turned = interleaved ? 0 : R / 2 / vec;
  const int units = turned + (int)ceil_div(D - 2 * turned * vec, 2 * vec);
  int lpr = 8;
  while (lpr < 64 && lpr < units) lpr *= 2;
  return {vec, vec == 1 ? 64 : lpr};
}

inline int check_rotary(const en_norm_rotary *how, int D) {
  if (!how) return EN_ERR_NULL;
  if (D < 1 || D > kRotaryMaxHead || how->rotary_dim < 0 || how->rotary_dim > D || how->rotary_dim % 2 || how->table_rows < 0) return EN_ERR_SHAPE;
  if (how->rotary_dim > 0 && how->table_rows > 0 && (!how->cos || !how->sin)) return EN_ERR_NULL;
  if (how->rotary_dim > 0 && how->table_rows == 0) return EN_ERR_SHAPE;
  if (!aligned_to(how->cos, 4) || !aligned_to(how->sin, 4)) return EN_ERR_ALIGN;
  return EN_OK;
}
// `vec`: the form's vector.
inline RotaryHow rotary_how(const en_norm_rotary *how, int D, int vec) {
  return RotaryHow{how->cos, how->sin, how->q_weight, how->k_weight, how->table_rows, how->rotary_dim, D,
                   (int)ceil_div(D - how->rotary_dim, 2 * vec), how->eps};
}

// Calls f(VEC, LPR, NP, interleaved) as integral constants for the form of this head; false where there is none.
template <int V> using Int = std::integral_constant<int, V>;
template <int DT, typename F>
static bool with_rotary_form(const RotaryForm &form, bool interleaved, F &&f) {
  auto lanes = [&](auto vec, auto il) {
    constexpr int VEC = decltype(vec)::value;
    if constexpr (VEC == 1) return f(vec, Int<64>{}, Int<2>{}, il), true;
    else if (form.lpr == 8 && VEC * 16 >= 64) return f(vec, Int<8>{}, Int<1>{}, il), true;
    else if (form.lpr <= 16 && VEC * 32 >= 64) return f(vec, Int<16>{}, Int<1>{}, il), true;
    else if constexpr (VEC <= 4) {
      if (form.lpr <= 32) return f(vec, Int<32>{}, Int<1>{}, il), true;
      if constexpr (VEC == 2) return f(vec, Int<64>{}, Int<1>{}, il), true;
      else return false;
    } else return false;
  };
  auto vecs = [&](auto il) {
    switch (form.vec) {
      case 8: if constexpr (DT != EN_F32) return lanes(Int<8>{}, il); else return false;
      case 4: return lanes(Int<4>{}, il);
      case 2: return lanes(Int<2>{}, il);
      default: return lanes(Int<1>{}, il);
    }
  };
  return interleaved ? vecs(std::true_type{}) : vecs(std::false_type{});
}

}  // namespace en

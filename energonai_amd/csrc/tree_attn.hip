// Attention of drafted tokens: the nodes of a tree behind each sequence's cached positions, over a paged cache and over one another.
//
// A sequence's up to 64 nodes times the G query heads that share a key head are the rows of one unit, and one pass over the unit's keys
// and values serves them all.  A workgroup takes a unit's rows, 16 QT QW of them at a time, and goes over its tiles of keys: the
// context's, in pages, and right behind its last position the nodes' own, of which a row sees what its mask says.
//  - Scores are S^T = K Q^T on 16x16x32 matrix instructions: rows are positions, columns queries.  A lane's scores of two neighbouring
//    key tiles (positions 4g .. 4g + 3 of each) are, packed to 16 bits, in place as the operand of O^T = V^T P^T when V^T is read from
//    LDS with the same order of positions, by its transposing read.
//  - Keys and values go through registers into LDS, a tile ahead: what lies behind a sequence's nodes or in no page arrives there as zeros,
//    so that nothing of another sequence, and no NaN of a page never written, meets a probability of zero.
//  - The running maximum is raised only where a score passes it by 2^8: the sums are fp32, and probabilities of up to 2^8 are as exact in
//    16 bits as those below 1.  In fp16 the maximum's own probability stands at 2^7, so that others count down to 2^-32 of it: from 1 on
//    they would end at 2^-25, and over the 10^5 positions of a long cache what is left out would pass half a step of the result.
// The probabilities are rounded to the cache's 16-bit type for the second product (half a step, 2^-11 or 2^-8 of each; the first product's
// operands are exact): the matrix instructions take both operands in one type, and in fp32 they are a sixteenth as fast.  The sum of the
// softmax takes them in fp32.
//
// Few rows a unit are bound by the stream of keys and values, many by exponents and matrix instructions in turn: 24 sequences of up to 4000, 32 / 8
// heads x 128, up to 64 rows (bf16) 46 us + 6 for the joining launch, 4.8 TB/s; 16 of 500 to 2000, 56 heads x 128, up to 64 rows (fp16) 150 + 15 us, 4.6
// TB/s; one of 130001, 64 / 8 heads x 128, 504 rows (bf16) 370 in all, 15 of them the joining launch, 0.72 PFLOP/s.
#include <type_traits>

#include "paged_common.hip.h"

namespace en {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kNodes = EN_DRAFT_MAX_NODES;
constexpr float kRaise = 8.f;                 // log2
template <int DT> constexpr float kTop = DT == EN_F16 ? 7.f : 0.f;      // log2 of the running maximum's probability: 2^(7 + 8) fits fp16

template <int DT> struct Mma;
template <> struct Mma<EN_F16> {
  __device__ static __forceinline__ f32x4 k32(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t two(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)lo, (_Float16)hi});
  }
};
template <> struct Mma<EN_BF16> {
  __device__ static __forceinline__ f32x4 k32(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t two(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, b16x2{(__bf16)lo, (__bf16)hi});
  }
};

// The halves of a word that are infinite or not a number, as a mask.
template <int DT> __device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  constexpr uint32_t kExp = DT == EN_F16 ? 0x7c00u : 0x7f80u;
  return ((w & kExp) == kExp ? 0xffffu : 0u) | ((w >> 16 & kExp) == kExp ? 0xffff0000u : 0u);
}

struct TreeArgs {
  const char *k_pool, *v_pool;                 // page, head and row strides in bytes
  int64_t k_page, k_head, v_page, v_head;
  uint32_t k_row, v_row;
  const int32_t *table, *lens, *cu;
  const int64_t *masks;
  const char *q, *k_new, *v_new;               // token and head strides in bytes
  int64_t q_token, q_head, kn_token, kn_head, vn_token, vn_head;
  void *ctx;                                   // [T, Hq, D]
  int num_pages, lg_page, max_pages, B, H, G, D;
  int chunks;                                  // runs of rows that a unit has at most
  int max_nodes;
  int total;                                   // rows of q
  float c_exp;                                 // scale * log2(e)
  int runs;                                    // workgroups take equal runs of all tiles, else a unit each
  uint32_t *first_tile;                        // [B] of a sequence, in the row of all tiles; behind them the tiles of a run
  float *part_o;                               // [2 workgroups][rows of a run of them][D]
  float2 *part_ml;                             // maximum and sum
};

__device__ __forceinline__ float over_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float over_groups_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v, int lane) {
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) {
    const uint32_t up = (uint32_t)__shfl_up((int)v, m, kWave);
    v += lane >= m ? up : 0u;
  }
  return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
// A word that the whole wave asks for, as a scalar load: a vector load would be waited for behind the keys and values on their way.
__device__ __forceinline__ int scalar_word(const int32_t *p) {
  typedef const __attribute__((address_space(4))) int32_t *scalar_t;
  return *(scalar_t)(uintptr_t)p;
}

// What a partial result of maximum m and sum l is multiplied by where the largest maximum is `top`: 0 for one without positions, and for one
// whose sum is NaN a number, so that it stays.
__device__ __forceinline__ float share_weight(float m, float l, float top) {
  return m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : l == 0.f ? 0.f : 1.f;
}

// A sequence's part in the row of all tiles: per key head, per run of rows, its tiles and the unit's end.
constexpr int kUnitCost = 1;
struct TreeSeq {
  int first, nodes, rows, len, chunks;
  int context, tiles;            // tiles of the context alone; all, the nodes following the context's last position
  __device__ __forceinline__ uint32_t per_unit() const { return tiles + kUnitCost; }
};
template <int TILE, int ROWS> __device__ __forceinline__ TreeSeq tree_seq(const TreeArgs &a, int first, int next, int len) {
  TreeSeq s;
  s.first = first;
  s.nodes = min(max(min(next, a.total) - first, 0), a.max_nodes);
  s.rows = s.nodes * a.G;
  s.len = min(max(len, 0), a.max_pages << a.lg_page);
  s.context = s.len / TILE;
  s.tiles = (s.len + s.nodes + TILE - 1) / TILE;
  s.chunks = (s.rows + ROWS - 1) / ROWS;
  return s;
}

// NT: runs of 16 channels the head is padded to.  QW waves take 16 QT rows each; KW waves share the positions of a tile.
template <int NT_, int QT_, int QW_, int KW_> struct TreeShape {
  static constexpr int NT = NT_, QT = QT_, QW = QW_, KW = KW_;
  static constexpr int kThreads = QW * KW * kWave, kTile = KW == 4 ? 128 : 64, kRows = 16 * QT * QW, kSub = kTile / 16 / KW, NC = NT / 2;
  static constexpr int kSlots = NT > 4 ? 16 : NT == 2 && QW == 8 ? 8 : 2 * NT;                     // lanes a row of a tile is moved by: whole rows a wave, and no more than 16
  static constexpr int kStep = kThreads / kSlots, kEach = kTile / kStep, kWaveRows = kWave / kSlots;
  static constexpr int kKeyPitch = NT * 32 + 16, kValuePitch = NT * 32 + 32;      // bytes: rows shifted by 4 and 8 banks
  static constexpr int kValues = kTile * kKeyPitch, kBytes = kValues + kTile * kValuePitch;
  static constexpr int kBuffers = KW == 1 ? 2 : 1;                        // of tiles in LDS, so that two workgroups fit a CU
  static constexpr int kMerge = (KW - 1) * QT * NT * 1024, kMergeBytes = kMerge + KW * QT * 128;
  static_assert(NT % 2 == 0 && kSub % 2 == 0 && kTile % kStep == 0 && kWaveRows <= 16 && kMergeBytes <= kBytes, "whole vectors, pairs of key tiles, rows of one page");
};

template <int DT, typename S>
__global__ __launch_bounds__(S::kThreads, 2) void tree_attn_kernel(TreeArgs a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  typedef Mma<DT> M;
  constexpr int NT = S::NT, QT = S::QT, QW = S::QW, KW = S::KW, NC = S::NC, kSub = S::kSub, kTile = S::kTile, kEach = S::kEach;
  __shared__ __align__(16) char s_mem[S::kBuffers * S::kBytes];
  __shared__ uint32_t s_odd[kNodes / 32];      // nodes with a value that is not a number, or infinite
  const int lane = threadIdx.x % kWave, col = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wq = wave % QW, wk = wave / QW;

  int b, h, chunk, tile;
  uint32_t x = 0, end = 0xffffffffu, group = blockIdx.x;
  TreeSeq s;
  auto seq_at = [&](int i) { return tree_seq<kTile, S::kRows>(a, scalar_word(a.cu + i), scalar_word(a.cu + i + 1), scalar_word(a.lens + i)); };
  if (!a.runs) {
    chunk = blockIdx.x % a.chunks;
    h = blockIdx.x / a.chunks % a.H;
    b = blockIdx.x / (a.chunks * a.H);
    s = seq_at(b);
    if (chunk >= s.chunks) return;
    tile = 0;
  } else {
    // neighbouring runs, which read neighbouring heads' rows of the same pages or the same rows, on one XCD
    group = blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds;
    uint32_t all = 0;
    auto cost = [&](int i) -> uint32_t {
      if (i >= a.B) return 0;
      const TreeSeq t = tree_seq<kTile, S::kRows>(a, a.cu[i], a.cu[i + 1], a.lens[i]);
      return (uint32_t)(a.H * t.chunks) * t.per_unit();
    };
    const uint32_t incl0 = wave_prefix(cost(lane), lane);
    all = lane_value(incl0, kWave - 1);
    for (int b0 = kWave; b0 < a.B; b0 += kWave) all += lane_value(wave_prefix(cost(b0 + lane), lane), kWave - 1);
    const uint32_t quota = (all + gridDim.x - 1) / gridDim.x, x0 = group * quota;
    if (x0 >= all) return;
    end = min(x0 + quota, all);
    if (group == 0 && threadIdx.x == 0) a.first_tile[a.B] = quota;
    // the sequence of tile x0: the first whose tiles end past it
    uint32_t incl = incl0, before = 0;
    b = 0;
    while (true) {
      const uint64_t past = __ballot(before + incl > x0);
      if (past) {
        const int l = __builtin_ctzll(past);
        if (l > 0) before += lane_value(incl, l - 1);
        b += l;
        break;
      }
      before += lane_value(incl, kWave - 1);
      b += kWave;
      incl = wave_prefix(cost(b + lane), lane);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    s = seq_at(b);
    const uint32_t unit = (x0 - before) / s.per_unit();
    tile = (int)(x0 - before - unit * s.per_unit());
    h = (int)(unit / (uint32_t)s.chunks);
    chunk = (int)unit - h * s.chunks;
    x = x0;
  }
  // The next unit that has rows.
  auto next_unit = [&] {
    x += s.per_unit() - tile;
    tile = 0;
    if (x >= end) return;
    if (++chunk < s.chunks) return;
    chunk = 0;
    if (++h < a.H) return;
    h = 0;
    do s = seq_at(++b);
    while (s.chunks == 0);
  };
  if (a.runs && tile >= s.tiles) {             // the run begins with a unit's end
    next_unit();
    if (x >= end) return;
  }

  uint4 kr[kEach], vr[kEach];
  int id[kEach];
  uint32_t valid = 0;
  const int slot = lane % S::kSlots, lane_row = lane / S::kSlots, ch = slot * 8;
  const uint32_t ch_bytes = ch < a.D ? ch * 2 : 0;
  // Pages of a tile: of the rows that this wave moves, which are in one page a step.
  auto pages = [&](int t) {
    const int32_t *names = a.table + (int64_t)b * a.max_pages;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      id[i] = scalar_word(names + min((t * kTile + i * S::kStep + wave * S::kWaveRows) >> a.lg_page, a.max_pages - 1));
  };
  // Rows of pages that are none are loaded from wherever there is memory, and taken for zeros.
  auto load_context = [&](int t) {
    valid = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int pos0 = t * kTile + i * S::kStep + wave * S::kWaveRows;
      const bool named = (unsigned)id[i] < (unsigned)a.num_pages;
      const int64_t page = named ? id[i] : 0;
      const char *kp = a.k_pool + page * a.k_page + h * a.k_head, *vp = a.v_pool + page * a.v_page + h * a.v_head;
      const uint32_t row = (pos0 & ((1 << a.lg_page) - 1)) + lane_row;
      kr[i] = *reinterpret_cast<const uint4 *>(kp + (row * a.k_row + ch_bytes));
      vr[i] = *reinterpret_cast<const uint4 *>(vp + (row * a.v_row + ch_bytes));
      if (named && ch < a.D) valid |= 1u << i;
    }
  };
  // A tile in which the context ends or that is behind it: the nodes follow its last position.
  auto load_end = [&](int t) {
    valid = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int pos0 = t * kTile + i * S::kStep + wave * S::kWaveRows, node = pos0 + lane_row - s.len;
      const bool named = pos0 < s.len && (unsigned)id[i] < (unsigned)a.num_pages;
      const int64_t page = named ? id[i] : 0, row = (pos0 & ((1 << a.lg_page) - 1)) + lane_row, from = s.first + min(max(node, 0), s.nodes - 1);
      const char *kp = node < 0 ? a.k_pool + page * a.k_page + h * a.k_head + row * a.k_row : a.k_new + from * a.kn_token + h * a.kn_head;
      const char *vp = node < 0 ? a.v_pool + page * a.v_page + h * a.v_head + row * a.v_row : a.v_new + from * a.vn_token + h * a.vn_head;
      kr[i] = *reinterpret_cast<const uint4 *>(kp + ch_bytes);
      vr[i] = *reinterpret_cast<const uint4 *>(vp + ch_bytes);
      if ((node < 0 ? named : node < s.nodes) && ch < a.D) valid |= 1u << i;
    }
  };
  auto load = [&](int t) {
    if (t < s.context) load_context(t);
    else load_end(t);
    if ((t + 1) * kTile < s.len) pages(t + 1);
  };
  // A node's value that is not a number, or infinite, may not meet the zeros of rows that do not see it: it is a zero here and
  // added where it is seen (below).
  auto put = [&](int t, int buf) {
    char *const s_k = s_mem + buf * S::kBytes, *const s_v = s_k + S::kValues;
    const bool whole = __ballot(valid != (1u << kEach) - 1) == 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int r = i * S::kStep + wave * S::kWaveRows + lane_row;
      if (!whole && !(valid >> i & 1)) kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      const int node = t * kTile + r - s.len;
      if (t >= s.context && node >= 0) {
        const uint4 odd = make_uint4(odd_halves<DT>(vr[i].x), odd_halves<DT>(vr[i].y), odd_halves<DT>(vr[i].z), odd_halves<DT>(vr[i].w));
        if (odd.x | odd.y | odd.z | odd.w) {
          vr[i] = make_uint4(vr[i].x & ~odd.x, vr[i].y & ~odd.y, vr[i].z & ~odd.z, vr[i].w & ~odd.w);
          atomicOr(&s_odd[node / 32], 1u << (node % 32));
        }
      }
      if (S::kSlots > 2 * NT && slot >= 2 * NT) continue;
      *reinterpret_cast<uint4 *>(s_k + r * S::kKeyPitch + slot * 16) = kr[i];
      *reinterpret_cast<uint4 *>(s_v + r * S::kValuePitch + slot * 16) = vr[i];
    }
  };

  bool first_segment = true;
  while (true) {
    // a unit, or this run's part of it
    lds_barrier();                             // the one before has been read
    const int begin = tile, stop = (int)min((uint32_t)s.tiles, tile + (end - x));
    if (a.runs && tile == 0 && h == 0 && chunk == 0 && threadIdx.x == 0) a.first_tile[b] = x;
    if (begin * kTile < s.len) pages(begin);
    load(begin);
    // queries: column l % 16 of tile t, channels 32 c + 8 g ..
    uint4 q[QT][NC];
    uint64_t mask[QT];
    int row[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      row[t] = chunk * S::kRows + (wq * QT + t) * 16 + col;
      const bool there = row[t] < s.rows;
      const int node = there ? row[t] / a.G : 0, head = there ? row[t] - node * a.G : 0;
      mask[t] = there ? (uint64_t)a.masks[s.first + node] & (s.nodes == kNodes ? ~0ull : (1ull << s.nodes) - 1) : 0;
      const char *p = a.q + (int64_t)(s.first + node) * a.q_token + (int64_t)(h * a.G + head) * a.q_head;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int from = 32 * c + 8 * g;
        q[t][c] = there && from < a.D ? *reinterpret_cast<const uint4 *>(p + from * 2) : make_uint4(0, 0, 0, 0);
      }
    }
    float m[QT], l[QT];
    f32x4 o[QT][NT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) o[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (threadIdx.x < kNodes / 32) s_odd[threadIdx.x] = 0;
    lds_barrier();
    put(tile, 0);
    if (tile + 1 < stop) load(tile + 1);
    lds_barrier();
    int buf = 0;
    for (; tile < stop; ++tile) {
      const bool own = tile >= s.context;
      const char *const s_k = s_mem + buf * S::kBytes, *const s_v = s_k + S::kValues;
      f32x4 sc[QT][kSub];
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        const char *kp = s_k + ((wk * kSub + u) * 16 + col) * S::kKeyPitch + g * 16;
#pragma unroll
        for (int t = 0; t < QT; ++t) sc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint4 k = *reinterpret_cast<const uint4 *>(kp + c * 64);
#pragma unroll
          for (int t = 0; t < QT; ++t) sc[t][u] = M::k32(k, q[t][c], sc[t][u]);
        }
      }
      if (S::kBuffers == 2 && tile + 1 < stop) {
        put(tile + 1, buf ^ 1);
        if (tile + 2 < stop) load(tile + 2);
      }
      if (own) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          // bit i: whether the lane's i-th position of this wave's tiles is seen
          uint32_t seen = 0;
#pragma unroll
          for (int u = 0; u < kSub; ++u) {
            const int node = tile * kTile + (wk * kSub + u) * 16 + 4 * g - s.len;      // of the first of four
            const uint32_t before = (1u << min(max(-node, 0), 4)) - 1;
            const uint32_t nodes = node >= kNodes || node <= -4 ? 0u : (uint32_t)(node >= 0 ? mask[t] >> node : mask[t] << -node) & 15u;
            seen |= (before | nodes) << (4 * u);
          }
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][u][e] = seen >> (4 * u + e) & 1 ? sc[t][u][e] : -INFINITY;
        }
      }
      uint32_t p[QT][kSub][2];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, sc[t][u][e]);
        top *= a.c_exp;
        if (__ballot(top > m[t] + kRaise)) {
          const float to = fmaxf(m[t], over_groups_max(top));
          const float keep = to > -INFINITY ? __builtin_amdgcn_exp2f(m[t] - to) : 1.f;
          l[t] *= keep;
#pragma unroll
          for (int n = 0; n < NT; ++n) o[t][n] *= keep;
          m[t] = to;
        }
        const float base = m[t] > -INFINITY ? m[t] - kTop<DT> : 0.f;
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          float e4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            e4[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][u][e], a.c_exp, -base));
            l[t] += e4[e];
          }
          p[t][u][0] = M::two(e4[0], e4[1]);
          p[t][u][1] = M::two(e4[2], e4[3]);
        }
      }
#pragma unroll
      for (int u = 0; u < kSub; u += 2)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const char *vp = s_v + ((wk * kSub + u) * 16 + 4 * g + col / 4) * S::kValuePitch + n * 32 + col % 4 * 8;
          const uint2 v0 = lds_read_tr16(vp), v1 = lds_read_tr16(vp + 16 * S::kValuePitch);
          const uint4 v = make_uint4(v0.x, v0.y, v1.x, v1.y);
#pragma unroll
          for (int t = 0; t < QT; ++t) o[t][n] = M::k32(v, make_uint4(p[t][u][0], p[t][u][1], p[t][u + 1][0], p[t][u + 1][1]), o[t][n]);
        }
      if (tile + 1 < stop) {
        lds_barrier();
        if constexpr (S::kBuffers == 1) {
          put(tile + 1, 0);
          if (tile + 2 < stop) load(tile + 2);
          lds_barrier();
        } else {
          buf ^= 1;
        }
      }
      if (!own || (s_odd[0] | s_odd[1]) == 0) continue;
      const uint64_t odd = (uint64_t)s_odd[1] << 32 | s_odd[0];
      for (int k = 0; k < kSub * 16; ++k) {
        const int node = tile * kTile + wk * kSub * 16 + k - s.len;
        if (node < 0 || node >= s.nodes || !(odd >> node & 1)) continue;
        const T *value = reinterpret_cast<const T *>(a.v_new + (int64_t)(s.first + node) * a.vn_token + h * a.vn_head) + 4 * g;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          uint32_t mine = 0;
#pragma unroll
          for (int u = 0; u < kSub; ++u) mine = u == k / 16 ? (k & 2 ? p[t][u][1] : p[t][u][0]) : mine;
          const uint32_t two = (uint32_t)__shfl((int)mine, k % 16 / 4 * 16 + col, kWave);
          const float by = E::to_float(__builtin_bit_cast(T, (uint16_t)(k & 1 ? two >> 16 : two)));
          if (!(mask[t] >> node & 1)) continue;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (16 * n + 4 * g >= a.D) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = E::to_float(value[16 * n + e]);
              if (!(fabsf(v) < INFINITY)) o[t][n][e] += by * v;
            }
          }
        }
      }
    }

#pragma unroll
    for (int t = 0; t < QT; ++t) l[t] = over_groups_sum(l[t]);
    if constexpr (KW > 1) {
      // what the waves that shared the positions have for the same rows meets in the tiles' place
      static_assert(QW == 1, "the waves have the same rows");
      float *s_o = reinterpret_cast<float *>(s_mem);
      float2 *s_ml = reinterpret_cast<float2 *>(s_mem + S::kMerge);
      lds_barrier();
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        if (g == 0) s_ml[(wk * QT + t) * 16 + col] = make_float2(m[t], l[t]);
        if (wk > 0) {
#pragma unroll
          for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4 *>(s_o + ((((wk - 1) * QT + t) * NT + n) * kWave + lane) * 4) = o[t][n];
        }
      }
      lds_barrier();
      if (wk == 0) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          float top = m[t];
#pragma unroll
          for (int w = 1; w < KW; ++w) top = fmaxf(top, s_ml[(w * QT + t) * 16 + col].x);
          const float keep = share_weight(m[t], l[t], top);
          l[t] *= keep;
#pragma unroll
          for (int n = 0; n < NT; ++n) o[t][n] *= keep;
#pragma unroll
          for (int w = 1; w < KW; ++w) {
            const float2 ml = s_ml[(w * QT + t) * 16 + col];
            const float f = share_weight(ml.x, ml.y, top);
            l[t] += ml.y * f;
#pragma unroll
            for (int n = 0; n < NT; ++n) o[t][n] += *reinterpret_cast<const f32x4 *>(s_o + ((((w - 1) * QT + t) * NT + n) * kWave + lane) * 4) * f;
          }
          m[t] = top;
        }
      }
    }
    if (wk == 0) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        if (row[t] >= s.rows) continue;
        if (begin == 0 && stop == s.tiles) {
          const float by = l[t] > 0.f ? 1.f / l[t] : l[t];
          const int node = row[t] / a.G, head = row[t] - node * a.G;
          T *out = reinterpret_cast<T *>(a.ctx) + ((int64_t)(s.first + node) * a.H * a.G + h * a.G + head) * a.D + 4 * g;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (16 * n + 4 * g >= a.D) continue;
            Pack<T, 4> w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w.v[e] = E::from_float(l[t] == 0.f ? 0.f : o[t][n][e] * by);
            store_pack<T, 4>(out + 16 * n, w);
          }
        } else {
          const int64_t part = ((int64_t)group * 2 + (first_segment ? 0 : 1)) * S::kRows + row[t] - chunk * S::kRows;
          float *out = a.part_o + part * a.D + 4 * g;
#pragma unroll
          for (int n = 0; n < NT; ++n)
            if (16 * n + 4 * g < a.D) *reinterpret_cast<f32x4 *>(out + 16 * n) = o[t][n];
          if (g == 0) a.part_ml[part] = make_float2(m[t], l[t]);
        }
      }
    }
    if (!a.runs) return;
    x += stop - begin;
    if (stop < s.tiles || x + kUnitCost >= end) return;
    next_unit();
    first_segment = false;
  }
}

// Combines the partial results of the units that several workgroups had tiles of: 32 lanes four channels each, eight groups of lanes.
// Few shares: a group takes a row.  Many: the groups take every eighth share of a row, and their results go through LDS.
constexpr int kCombineLanes = 32, kCombineGroups = kBlock / kCombineLanes, kAhead = 8;

template <int DT, int TILE, int ROWS>
__global__ __launch_bounds__(kBlock) void tree_combine_kernel(TreeArgs a) {
  typedef typename Elem<DT>::T T;
  __shared__ f32x4 s_o[kCombineGroups][kCombineLanes];
  __shared__ float2 s_ml[kCombineGroups];
  const int chunk = blockIdx.x % a.chunks, h = blockIdx.x / a.chunks % a.H, b = blockIdx.x / (a.chunks * a.H);
  const TreeSeq s = tree_seq<TILE, ROWS>(a, scalar_word(a.cu + b), scalar_word(a.cu + b + 1), scalar_word(a.lens + b));
  if (chunk >= s.chunks) return;
  const uint32_t quota = scalar_word(reinterpret_cast<const int32_t *>(a.first_tile) + a.B);
  const uint32_t x0 = scalar_word(reinterpret_cast<const int32_t *>(a.first_tile) + b) + (h * s.chunks + chunk) * s.per_unit(), x1 = x0 + s.tiles;
  const uint32_t w0 = x0 / quota, w1 = (x1 - 1) / quota;
  if (w0 == w1) return;                                     // one workgroup had it whole
  const bool from_start = x0 - w0 * quota <= kUnitCost;     // the first one's run begins with this unit, or the end of the one before
  const int rows = min(ROWS, s.rows - chunk * ROWS), group = threadIdx.x / kCombineLanes, part = threadIdx.x % kCombineLanes, d = part * 4;
  auto write = [&](int r, float l, const f32x4 &o) {
    const int at = chunk * ROWS + r, node = at / a.G, head = at - node * a.G;
    const float by = l > 0.f ? 1.f / l : l;
    Pack<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = Elem<DT>::from_float(l == 0.f ? 0.f : o[e] * by);
    store_pack<T, 4>(reinterpret_cast<T *>(a.ctx) + ((int64_t)(s.first + node) * a.H * a.G + h * a.G + head) * a.D + d, y);
  };
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
        const uint32_t at = min(w + j * step, w1);
        const int64_t slot = ((int64_t)at * 2 + (at == w0 && !from_start ? 1 : 0)) * ROWS + r;
        ml[j] = a.part_ml[slot];
        v[j] = *reinterpret_cast<const f32x4 *>(a.part_o + slot * a.D + (d < a.D ? d : 0));
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
    for (int r = blockIdx.y * kCombineGroups + group; r < rows; r += gridDim.y * kCombineGroups) {
      gather(r, w0, 1, m, l, o);
      if (d < a.D) write(r, l, o);
    }
    return;
  }
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    gather(r, w0 + group, kCombineGroups, m, l, o);
    if (r != (int)blockIdx.y) __syncthreads();              // the row before has been read
    s_o[group][part] = o;
    if (part == 0) s_ml[group] = make_float2(m, l);
    __syncthreads();
    if (group == 0 && d < a.D) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < kCombineGroups; ++j) top = fmaxf(top, s_ml[j].x);
      l = 0.f;
      o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kCombineGroups; ++j) {
        const float f = share_weight(s_ml[j].x, s_ml[j].y, top);
        l += s_ml[j].y * f;
        o += s_o[j][part] * f;
      }
      write(r, l, o);
    }
  }
}

// Rows a workgroup takes at a time, by the rows a unit may have: sixteen in four waves that share a tile's positions; else sixteen or
// thirty-two a wave.  us, 24 sequences of up to 4000, 32 / 8 x 128, rows 16 / 64 / 128 / 256 at a time: 16 rows a unit 43 / 47 / 59 / 88; 32 73 / 49 / 64 / 93;
// 64 130 / 53 / 68 / 97; 128 242 / 93 / 81 / 110; 8 sequences of up to 8000, 64 / 8 heads, 512 rows - / 280 / 186 / 178.
inline int tree_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256; }
// Workgroups that share all tiles: two of four waves a CU, or one of eight.
inline int tree_groups(int at_once) { return at_once == 256 ? 256 : 512; }
// Equal runs of tiles, whatever the lengths are, at the cost of a second launch, or a workgroup a unit where caches are short.  us, a
// workgroup a unit / runs: 1 sequence of 100, 12 x 64 8.2 / 13.6, of 1000 16.4 / 13.3; 4 of up to 1000, 32 / 8 x 128 40 / 22; 32 of up to 500, 12 x 64
// 13.5 / 18.8; 32 of up to 1000, 32 / 8 x 128 39.9 / 42.3; 64 of up to 250, 40 x 128 69 / 76; 128 of up to 200, 64 / 8 x 128 55 / 63; 8 of up to 2000 54 / 31.
inline bool tree_runs(int64_t units, int64_t capacity) { return capacity > (units >= 256 ? 1152 : 512); }

}  // namespace en

using namespace en;

extern "C" int64_t en_decode_attn_tree_workspace_bytes(int batch, int q_heads, int head_num, int capacity, int size_per_head, int max_nodes) {
  if (batch < 1 || head_num < 1 || q_heads < head_num || q_heads % head_num || capacity < 0 || size_per_head < 1 || max_nodes < 1) return 0;
  const int64_t rows = (int64_t)max_nodes * (q_heads / head_num), at_once = tree_rows(rows);
  if (!tree_runs((int64_t)batch * head_num * ceil_div(rows, at_once), capacity)) return 0;
  return 2 * tree_groups((int)at_once) * at_once * (4 * (int64_t)size_per_head + 8) + 4 * ((int64_t)batch + 1);
}

extern "C" int en_decode_attn_tree(const void *q, const void *k_new, const void *v_new, const int64_t *strides, void *ctx,
                                   const en_kv_pages *cache, const int32_t *kv_lens, const int32_t *cu_seqlens, const int64_t *masks, int64_t nodes,
                                   int max_nodes, int q_heads, float scale, void *workspace, int64_t workspace_bytes, en_stream_t stream) {
  if (!cache || !strides) return EN_ERR_NULL;
  const en_kv_pages &c = *cache;
  if (c.dtype != EN_F16 && c.dtype != EN_BF16) return EN_ERR_DTYPE;
  if (const int bad = check_kv_pages(c)) return bad;
  if (c.size_per_head % 8 || c.size_per_head > 128 || !(scale > 0.f)) return EN_ERR_UNSUPPORTED;
  if (q_heads < c.head_num || q_heads % c.head_num || max_nodes < 0 || max_nodes > kNodes || nodes < 0 || nodes > INT32_MAX) return EN_ERR_SHAPE;
  if (c.batch == 0 || nodes == 0 || max_nodes == 0) return EN_OK;
  if (!q || !k_new || !v_new || !ctx || !kv_lens || !cu_seqlens || !masks) return EN_ERR_NULL;
  for (const void *p : {q, k_new, v_new, (const void *)ctx, (const void *)c.k_pool, (const void *)c.v_pool, (const void *)workspace})
    if (!aligned_to(p, 16)) return EN_ERR_ALIGN;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 8 || c.strides[i] % 8) return EN_ERR_ALIGN;
  if (c.strides[2] > (1 << 30) / c.page_size || c.strides[5] > (1 << 30) / c.page_size) return EN_ERR_SHAPE;      // 32-bit offsets in a page
  const int64_t capacity = (int64_t)c.max_pages_per_seq * c.page_size, rows = (int64_t)max_nodes * (q_heads / c.head_num), at_once = tree_rows(rows);
  TreeArgs a{};
  a.chunks = (int)ceil_div(rows, at_once);
  const int64_t units = (int64_t)c.batch * c.head_num * a.chunks;
  a.runs = tree_runs(units, capacity);
  if (units * (ceil_div(capacity, 64) + 2) >= INT32_MAX) return EN_ERR_SHAPE;
  if (a.runs && !workspace) return EN_ERR_NULL;
  if (workspace_bytes < en_decode_attn_tree_workspace_bytes(c.batch, q_heads, c.head_num, (int)capacity, c.size_per_head, max_nodes)) return EN_ERR_SHAPE;
  a.k_pool = (const char *)c.k_pool; a.v_pool = (const char *)c.v_pool;
  a.k_page = 2 * c.strides[0]; a.k_head = 2 * c.strides[1]; a.k_row = (uint32_t)(2 * c.strides[2]);
  a.v_page = 2 * c.strides[3]; a.v_head = 2 * c.strides[4]; a.v_row = (uint32_t)(2 * c.strides[5]);
  a.table = c.page_table; a.lens = kv_lens; a.cu = cu_seqlens; a.masks = masks;
  a.q = (const char *)q; a.k_new = (const char *)k_new; a.v_new = (const char *)v_new;
  a.q_token = 2 * strides[0]; a.q_head = 2 * strides[1]; a.kn_token = 2 * strides[2]; a.kn_head = 2 * strides[3];
  a.vn_token = 2 * strides[4]; a.vn_head = 2 * strides[5];
  a.ctx = ctx;
  a.num_pages = c.num_pages; a.lg_page = page_log2(c.page_size); a.max_pages = c.max_pages_per_seq;
  a.B = c.batch; a.H = c.head_num; a.G = q_heads / c.head_num; a.D = c.size_per_head;
  a.max_nodes = max_nodes; a.total = (int)nodes;
  a.c_exp = scale * 1.4426950408889634f;
  a.part_o = reinterpret_cast<float *>(workspace);
  a.part_ml = reinterpret_cast<float2 *>(a.part_o + (int64_t)2 * tree_groups((int)at_once) * at_once * c.size_per_head);
  a.first_tile = reinterpret_cast<uint32_t *>(a.part_ml + (int64_t)2 * tree_groups((int)at_once) * at_once);
  const hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto dt, auto shape) {
    constexpr int DT = decltype(dt)::value;
    typedef decltype(shape) S;
    tree_attn_kernel<DT, S><<<a.runs ? tree_groups((int)at_once) : (unsigned)units, S::kThreads, 0, s>>>(a);
    if (!a.runs) return;
    // rows of a unit in workgroups of their own where units are few; where units are many, each has few shares
    const dim3 shares((unsigned)units, (unsigned)(units >= 64 ? ceil_div(at_once, kCombineGroups) : at_once));
    tree_combine_kernel<DT, S::kTile, S::kRows><<<shares, kBlock, 0, s>>>(a);
  };
  auto rows_of = [&](auto dt, auto nt) {
    constexpr int NT = decltype(nt)::value;
    if (at_once == 16) launch(dt, TreeShape<NT, 1, 1, 4>{});
    else if (at_once == 64) launch(dt, TreeShape<NT, 1, 4, 1>{});
    else if (at_once == 128) launch(dt, TreeShape<NT, 2, 4, 1>{});
    else launch(dt, TreeShape<NT, 2, 8, 1>{});
  };
  auto heads = [&](auto dt) {
    if (a.D <= 32) rows_of(dt, std::integral_constant<int, 2>{});
    else if (a.D <= 64) rows_of(dt, std::integral_constant<int, 4>{});
    else if (a.D <= 96) rows_of(dt, std::integral_constant<int, 6>{});
    else rows_of(dt, std::integral_constant<int, 8>{});
  };
  if (c.dtype == EN_F16) heads(std::integral_constant<int, EN_F16>{});
  else heads(std::integral_constant<int, EN_BF16>{});
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

// Attention of drafted tokens: the nodes of a tree behind each sequence's cached positions, over a paged cache and over one another.
//
// A sequence's up to 64 nodes times the G query heads that share a key head are the rows of one unit, and one pass over the unit's keys
// and values serves them all.  A workgroup takes a unit's rows, 16 QT QW of them at a time, and goes over its tiles of keys: those of the
// context in pages, and behind them one tile that holds the nodes' own keys, where a row sees what its mask says.
//  - Scores are S^T = K Q^T on 16x16x32 matrix instructions: rows are positions, columns queries.  A lane's scores of two neighbouring
//    key tiles (positions 4g .. 4g + 3 of each) are, packed to 16 bits, in place as the operand of O^T = V^T P^T when V^T is read from
//    LDS with the same order of positions, by its transposing read.
//  - Keys and values go through registers into LDS, a tile ahead: what lies behind a sequence's end or in no page arrives there as zeros,
//    so that nothing of another sequence, and no NaN of a page never written, meets a probability of zero.
//  - The running maximum is raised only where a score passes it by 2^8: the sums are fp32, and probabilities of up to 2^8 are as exact in
//    16 bits as those below 1.
// The probabilities are rounded to the cache's 16-bit type for the second product (half a step, 2^-11 or 2^-8 of each; the first product's
// operands are exact): the matrix instructions take both operands in one type, and in fp32 they are a sixteenth as fast.  The sum of the
// softmax takes them in fp32.
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
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
  const int32_t *table, *lens, *cu;
  const int64_t *masks;
  const char *q, *k_new, *v_new;               // token and head strides in bytes
  int64_t q_token, q_head, kn_token, kn_head, vn_token, vn_head;
  void *ctx;                                   // [T, Hq, D]
  int num_pages, lg_page, max_pages, B, H, G, D;
  int chunks;                                  // runs of a unit's rows
  int max_nodes;
  int total;                                   // rows of q
  float c_exp;                                 // scale * log2(e)
};

__device__ __forceinline__ float over_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float over_groups_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// NT: runs of 16 channels the head is padded to.  QW waves take 16 QT rows each; KW waves share the positions of a tile.
template <int DT, int NT, int QT, int QW, int KW>
__global__ __launch_bounds__(QW *KW *kWave) void tree_attn_kernel(TreeArgs a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  typedef Mma<DT> M;
  constexpr int kThreads = QW * KW * kWave, kTile = KW == 4 ? 128 : 64, kSub = kTile / 16 / KW, NC = NT / 2;
  constexpr int kPerRow = 2 * NT, kVectors = kTile * kPerRow, kEach = kVectors / kThreads;      // 16-byte vectors of a tile's keys
  constexpr int kKeyPitch = NT * 32 + 16, kValuePitch = NT * 32 + 32;                           // bytes: rows shifted by 4 and 8 banks
  static_assert(NT % 2 == 0 && kVectors % kThreads == 0 && kSub % 2 == 0, "whole vectors, pairs of key tiles");
  __shared__ __align__(16) char s_k[kTile * kKeyPitch];
  __shared__ __align__(16) char s_v[kTile * kValuePitch];
  __shared__ uint32_t s_odd[kNodes / 32];      // nodes with a value that is not a number, or infinite
  const int lane = threadIdx.x % kWave, col = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wq = wave % QW, wk = wave / QW;

  const int chunk = blockIdx.x % a.chunks, h = blockIdx.x / a.chunks % a.H, b = blockIdx.x / (a.chunks * a.H);
  const int first = a.cu[b], nodes = min(max(min(a.cu[b + 1], a.total) - first, 0), a.max_nodes);
  const int rows = nodes * a.G, row0 = chunk * 16 * QT * QW;
  if (row0 >= rows) return;
  const int len = min(max(a.lens[b], 0), a.max_pages << a.lg_page);
  const int context = (len + kTile - 1) / kTile, tiles = context + 1;

  // queries: column l % 16 of tile t, channels 32 c + 8 g ..
  uint4 q[QT][NC];
  uint64_t mask[QT];
  int row[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    row[t] = row0 + (wq * QT + t) * 16 + col;
    const bool there = row[t] < rows;
    const int node = there ? row[t] / a.G : 0, head = there ? row[t] - node * a.G : 0;
    mask[t] = there ? (uint64_t)a.masks[first + node] & (nodes == kNodes ? ~0ull : (1ull << nodes) - 1) : 0;
    const char *p = a.q + (int64_t)(first + node) * a.q_token + (int64_t)(h * a.G + head) * a.q_head;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int ch = 32 * c + 8 * g;
      q[t][c] = there && ch < a.D ? *reinterpret_cast<const uint4 *>(p + ch * 2) : make_uint4(0, 0, 0, 0);
    }
  }

  uint4 kr[kEach], vr[kEach];
  // The vectors of a tile that this thread moves: row i, channels 8 (i % kPerRow) ..
  auto load = [&](int tile) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int v = i * kThreads + threadIdx.x, r = v / kPerRow, ch = v % kPerRow * 8;
      const char *kp = a.k_pool, *vp = a.v_pool;
      bool ok = ch < a.D;
      if (tile < context) {
        const int pos = tile * kTile + r;
        ok = ok && pos < len;
        const int id = ok ? a.table[(int64_t)b * a.max_pages + (pos >> a.lg_page)] : -1;
        ok = ok && (unsigned)id < (unsigned)a.num_pages;
        const int64_t in_page = pos & ((1 << a.lg_page) - 1);
        kp += id * a.k_page + h * a.k_head + in_page * a.k_row + ch * 2;
        vp += id * a.v_page + h * a.v_head + in_page * a.v_row + ch * 2;
      } else {
        ok = ok && r < nodes;
        kp = a.k_new + (int64_t)(first + r) * a.kn_token + h * a.kn_head + ch * 2;
        vp = a.v_new + (int64_t)(first + r) * a.vn_token + h * a.vn_head + ch * 2;
      }
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      if (ok) {
        kr[i] = *reinterpret_cast<const uint4 *>(kp);
        vr[i] = *reinterpret_cast<const uint4 *>(vp);
      }
    }
  };
  // A node's value that is not a number, or infinite, may not meet the zeros of rows that do not see it: it is a zero here and
  // added where it is seen (below).
  auto put = [&](bool own) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int v = i * kThreads + threadIdx.x, r = v / kPerRow, c = v % kPerRow;
      if (own) {
        const uint4 odd = make_uint4(odd_halves<DT>(vr[i].x), odd_halves<DT>(vr[i].y), odd_halves<DT>(vr[i].z), odd_halves<DT>(vr[i].w));
        if (odd.x | odd.y | odd.z | odd.w) {
          vr[i] = make_uint4(vr[i].x & ~odd.x, vr[i].y & ~odd.y, vr[i].z & ~odd.z, vr[i].w & ~odd.w);
          atomicOr(&s_odd[r / 32], 1u << (r % 32));
        }
      }
      *reinterpret_cast<uint4 *>(s_k + r * kKeyPitch + c * 16) = kr[i];
      *reinterpret_cast<uint4 *>(s_v + r * kValuePitch + c * 16) = vr[i];
    }
  };

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
  load(0);
  for (int tile = 0; tile < tiles; ++tile) {
    lds_barrier();
    put(tile >= context);
    if (tile + 1 < tiles) load(tile + 1);
    lds_barrier();
    f32x4 s[QT][kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const char *kp = s_k + ((wk * kSub + u) * 16 + col) * kKeyPitch + g * 16;
#pragma unroll
      for (int t = 0; t < QT; ++t) s[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint4 k = *reinterpret_cast<const uint4 *>(kp + c * 64);
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t][u] = M::k32(k, q[t][c], s[t][u]);
      }
    }
    const int left = len - tile * kTile;       // of the context, from this tile on
    uint32_t p[QT][kSub][2];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pos = (wk * kSub + u) * 16 + 4 * g + e;
          const bool seen = tile < context ? pos < left : pos < kNodes && (mask[t] >> (pos & 63) & 1);
          s[t][u][e] = seen ? s[t][u][e] * a.c_exp : -INFINITY;
          top = fmaxf(top, s[t][u][e]);
        }
      if (__ballot(top > m[t] + kRaise)) {
        const float to = fmaxf(m[t], over_groups_max(top));
        const float keep = to > -INFINITY ? __builtin_amdgcn_exp2f(m[t] - to) : 1.f;
        l[t] *= keep;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[t][n] *= keep;
        m[t] = to;
      }
      const float base = m[t] > -INFINITY ? m[t] : 0.f;
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        float e4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          e4[e] = __builtin_amdgcn_exp2f(s[t][u][e] - base);
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
        const char *vp = s_v + ((wk * kSub + u) * 16 + 4 * g + col / 4) * kValuePitch + n * 32 + col % 4 * 8;
        const uint2 v0 = lds_read_tr16(vp), v1 = lds_read_tr16(vp + 16 * kValuePitch);
        const uint4 v = make_uint4(v0.x, v0.y, v1.x, v1.y);
#pragma unroll
        for (int t = 0; t < QT; ++t) o[t][n] = M::k32(v, make_uint4(p[t][u][0], p[t][u][1], p[t][u + 1][0], p[t][u + 1][1]), o[t][n]);
      }
    if (tile < context || (s_odd[0] | s_odd[1]) == 0) continue;
#pragma unroll
    for (int u = 0; u < kSub; ++u)
      for (int k = 0; k < 16; ++k) {
        const int node = (wk * kSub + u) * 16 + k;
        if (node >= nodes || !(s_odd[node / 32] >> (node % 32) & 1)) continue;
        const T *value = reinterpret_cast<const T *>(a.v_new + (int64_t)(first + node) * a.vn_token + h * a.vn_head) + 4 * g;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const uint32_t two = (uint32_t)__shfl((int)(k & 2 ? p[t][u][1] : p[t][u][0]), k / 4 * 16 + col, kWave);
          const float by = E::to_float(__builtin_bit_cast(T, (uint16_t)(k & 1 ? two >> 16 : two)));
          if (!(mask[t] >> node & 1)) continue;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (16 * n + 4 * g >= a.D) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = E::to_float(value[16 * n + e]);
              if (!(fabsf(x) < INFINITY)) o[t][n][e] += by * x;
            }
          }
        }
      }
  }

  if constexpr (KW > 1) {
    // what the waves that shared the positions have for the same rows meets in the tiles' place
    static_assert(QT == 1 && QW == 1, "one row tile");
    float *s_o = reinterpret_cast<float *>(s_k), *s_ml = reinterpret_cast<float *>(s_v);
    static_assert(sizeof(s_k) >= (KW - 1) * 16 * NT * 16 * 4 && sizeof(s_v) >= KW * 32 * 4, "room for the partial results");
    l[0] = over_groups_sum(l[0]);
    lds_barrier();
    if (g == 0) {
      s_ml[wk * 32 + col] = m[0];
      s_ml[wk * 32 + 16 + col] = l[0];
    }
    if (wk > 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4 *>(s_o + (((wk - 1) * NT + n) * kWave + lane) * 4) = o[0][n];
    }
    lds_barrier();
    if (wk > 0) return;
    float top = m[0];
#pragma unroll
    for (int w = 1; w < KW; ++w) top = fmaxf(top, s_ml[w * 32 + col]);
    auto weight = [&](float mw) { return mw > -INFINITY ? __builtin_amdgcn_exp2f(mw - top) : 1.f; };
    float keep = weight(m[0]);
    l[0] *= keep;
#pragma unroll
    for (int n = 0; n < NT; ++n) o[0][n] *= keep;
#pragma unroll
    for (int w = 1; w < KW; ++w) {
      keep = weight(s_ml[w * 32 + col]);
      l[0] += s_ml[w * 32 + 16 + col] * keep;
#pragma unroll
      for (int n = 0; n < NT; ++n) o[0][n] += *reinterpret_cast<const f32x4 *>(s_o + (((w - 1) * NT + n) * kWave + lane) * 4) * keep;
    }
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (row[t] >= rows) continue;
    const float sum = KW > 1 ? l[t] : over_groups_sum(l[t]);
    const float by = sum > 0.f ? 1.f / sum : sum;
    const int node = row[t] / a.G, head = row[t] - node * a.G;
    T *out = reinterpret_cast<T *>(a.ctx) + ((int64_t)(first + node) * a.H * a.G + h * a.G + head) * a.D + 4 * g;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (16 * n + 4 * g >= a.D) continue;
      Pack<T, 4> w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w.v[e] = E::from_float(sum == 0.f ? 0.f : o[t][n][e] * by);
      store_pack<T, 4>(out + 16 * n, w);
    }
  }
}

}  // namespace en

using namespace en;

extern "C" int64_t en_decode_attn_tree_workspace_bytes(int batch, int q_heads, int head_num, int capacity, int size_per_head, int max_nodes) {
  return 0;
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
  for (const void *p : {q, k_new, v_new, (const void *)ctx, (const void *)c.k_pool, (const void *)c.v_pool})
    if (!aligned_to(p, 16)) return EN_ERR_ALIGN;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 8 || c.strides[i] % 8) return EN_ERR_ALIGN;
  TreeArgs a{};
  a.k_pool = (const char *)c.k_pool; a.v_pool = (const char *)c.v_pool;
  a.k_page = 2 * c.strides[0]; a.k_head = 2 * c.strides[1]; a.k_row = 2 * c.strides[2];
  a.v_page = 2 * c.strides[3]; a.v_head = 2 * c.strides[4]; a.v_row = 2 * c.strides[5];
  a.table = c.page_table; a.lens = kv_lens; a.cu = cu_seqlens; a.masks = masks;
  a.q = (const char *)q; a.k_new = (const char *)k_new; a.v_new = (const char *)v_new;
  a.q_token = 2 * strides[0]; a.q_head = 2 * strides[1]; a.kn_token = 2 * strides[2]; a.kn_head = 2 * strides[3];
  a.vn_token = 2 * strides[4]; a.vn_head = 2 * strides[5];
  a.ctx = ctx;
  a.num_pages = c.num_pages; a.lg_page = page_log2(c.page_size); a.max_pages = c.max_pages_per_seq;
  a.B = c.batch; a.H = c.head_num; a.G = q_heads / c.head_num; a.D = c.size_per_head;
  a.max_nodes = max_nodes; a.total = (int)nodes;
  a.c_exp = scale * 1.4426950408889634f;
  const hipStream_t s = (hipStream_t)stream;
  const int64_t rows = (int64_t)max_nodes * a.G;
  int rc = EN_OK;
  auto launch = [&](auto dt, auto nt, auto qt, auto qw, auto kw) {
    constexpr int QT = decltype(qt)::value, QW = decltype(qw)::value, KW = decltype(kw)::value;
    a.chunks = (int)ceil_div(rows, 16 * QT * QW);
    const int64_t groups = (int64_t)a.B * a.H * a.chunks;
    if (groups > INT32_MAX) {
      rc = EN_ERR_SHAPE;
      return;
    }
    tree_attn_kernel<decltype(dt)::value, decltype(nt)::value, QT, QW, KW><<<(unsigned)groups, QW * KW * kWave, 0, s>>>(a);
  };
  auto shape = [&](auto dt, auto nt) {
    typedef std::integral_constant<int, 1> one;
    typedef std::integral_constant<int, 4> four;
    if (rows <= 16) launch(dt, nt, one{}, one{}, four{});
    else if (rows <= 64) launch(dt, nt, one{}, four{}, one{});
    else launch(dt, nt, std::integral_constant<int, 2>{}, four{}, one{});
  };
  auto heads = [&](auto dt) {
    if (a.D <= 32) shape(dt, std::integral_constant<int, 2>{});
    else if (a.D <= 64) shape(dt, std::integral_constant<int, 4>{});
    else if (a.D <= 96) shape(dt, std::integral_constant<int, 6>{});
    else shape(dt, std::integral_constant<int, 8>{});
  };
  if (c.dtype == EN_F16) heads(std::integral_constant<int, EN_F16>{});
  else heads(std::integral_constant<int, EN_BF16>{});
  if (rc) return rc;
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

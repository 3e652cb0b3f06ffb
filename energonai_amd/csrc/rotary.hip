// Norm and rotation of queries and keys: packed rows of a prompt, and a decode step's rows on their way into a paged cache.
//
// Both move each row once and compute a few operations an element, so what bounds them is memory (prompts) and the launch itself
// (decode steps).  rotary_rows.hip.h has the arithmetic.
#include "rotary_rows.hip.h"

namespace en {

// Rows from which a lane group takes several heads.  Fewer do not fill the chip, and what counts is that all of them are on their way at once;
// of more, each group's cos and sin are as much to load as a row, and several rows' loads are in flight together.  One head a group / four:
// 7 prompts of up to 2000, 32 + 8 heads x 128 38.5 / 36.4 us; a decode step's 256 x (64 + 8 + 8), one / two 6.8 / 6.6 us.
constexpr int64_t kManyRows = 16384;

struct RotaryRowsArgs {
  RotaryHow how;
  const void *in[2];            // q, k
  void *out[2];
  int64_t in_token[2], in_head[2], out_token[2], out_head[2];
  int heads[2];
  int parts[2];                 // lane groups a token's heads are dealt to
  const int32_t *cu, *positions;
  int batch;
  uint32_t tokens, groups;      // groups = tokens * (parts[0] + parts[1])
};

// Sequence of packed token t: the last one that starts at or before t and is not empty.  cu[0] = 0 <= t < cu[batch].
__device__ __forceinline__ int sequence_of(const int32_t *cu, int batch, int t) {
  int lo = 0, hi = batch;       // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// HPG heads of one token a lane group: its table rows are read once for them, and their loads are in flight together.
template <int DT, int VEC, int LPR, int NP, bool IL, int HPG, bool NT, bool NTL = false>
__global__ __launch_bounds__(kBlock) void qk_norm_rotary_kernel(RotaryRowsArgs a) {
  typedef typename Elem<DT>::T T;
  typedef RotaryRow<DT, VEC, LPR, NP, IL> Row;
  const int lane = threadIdx.x % LPR;
  const uint32_t group = blockIdx.x * (kBlock / LPR) + threadIdx.x / LPR;
  const uint32_t g = min(group, a.groups - 1);
  const uint32_t parts = a.parts[0] + a.parts[1];
  const uint32_t t = g / parts;
  int part = (int)(g - t * parts);
  const int which = part >= a.parts[0];
  part -= which ? a.parts[0] : 0;
  bool live = group < a.groups;
  int64_t pos = 0;
  if (a.positions) pos = a.positions[t];
  else if ((int64_t)t < a.cu[a.batch]) pos = (int)t - a.cu[sequence_of(a.cu, a.batch, (int)t)];
  else live = false;            // behind the last sequence
  const int first = part * HPG, heads = which ? a.heads[1] : a.heads[0];
  const T *in = reinterpret_cast<const T *>(which ? a.in[1] : a.in[0]) + (int64_t)t * (which ? a.in_token[1] : a.in_token[0]);
  T *out = reinterpret_cast<T *>(which ? a.out[1] : a.out[0]) + (int64_t)t * (which ? a.out_token[1] : a.out_token[0]);
  const int64_t in_head = which ? a.in_head[1] : a.in_head[0], out_head = which ? a.out_head[1] : a.out_head[0];
  Row rows[HPG];
#pragma unroll
  for (int h = 0; h < HPG; ++h) rows[h].template load<NTL>(a.how, in + min(first + h, heads - 1) * in_head, lane);
  RotaryTurn<VEC, LPR, NP, IL> turn;
  turn.load(a.how, pos, lane);
  const void *weight = which ? a.how.k_weight : a.how.q_weight;
#pragma unroll
  for (int h = 0; h < HPG; ++h) norm_and_turn(a.how, rows[h], turn, weight, lane);
  // behind all loads of the group: its heads may be written where they were read
#pragma unroll
  for (int h = 0; h < HPG; ++h)
    if (live && first + h < heads) store_row<NT>(a.how, rows[h], out + (first + h) * out_head, lane);
}

struct RotaryAppendArgs {
  RotaryHow how;
  const void *q, *k, *v;
  void *q_out, *k_pool, *v_pool;
  const int32_t *lens, *table;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, p_page, p_head, p_row;
  int B, Hq, Hk, max_pages, page, num_pages;
  int parts_q, parts_k;
  uint32_t groups;              // B * (parts_q + 2 parts_k)
  int32_t *overflow;
};

// HPG rows of one sequence and kind a lane group.
template <int DT, int VEC, int LPR, int NP, bool IL, int HPG>
__global__ __launch_bounds__(kBlock) void kv_append_paged_rotary_kernel(RotaryAppendArgs a) {
  typedef typename Elem<DT>::T T;
  typedef RotaryRow<DT, VEC, LPR, NP, IL> Row;
  const int lane = threadIdx.x % LPR;
  const uint32_t group = blockIdx.x * (kBlock / LPR) + threadIdx.x / LPR, g = min(group, a.groups - 1);
  const int per = a.parts_q + 2 * a.parts_k, b = (int)(g / per);
  int part = (int)(g - (uint32_t)b * per);
  const bool is_q = part < a.parts_q;
  part -= is_q ? 0 : a.parts_q;
  const bool is_v = !is_q && part >= a.parts_k;
  part -= is_v ? a.parts_k : 0;
  const int first = part * HPG, heads = is_q ? a.Hq : a.Hk;
  const T *in = is_q ? reinterpret_cast<const T *>(a.q) + b * a.q_sb : is_v ? reinterpret_cast<const T *>(a.v) + b * a.v_sb
                                                                           : reinterpret_cast<const T *>(a.k) + b * a.k_sb;
  const int64_t in_head = is_q ? a.q_sh : is_v ? a.v_sh : a.k_sh, out_head = is_q ? a.how.D : a.p_head;
  Row rows[HPG];
#pragma unroll
  for (int h = 0; h < HPG; ++h) rows[h].load(a.how, in + min(first + h, heads - 1) * in_head, lane);
  const int pos = a.lens[b];
  const void *weight = is_q ? a.how.q_weight : is_v ? nullptr : a.how.k_weight;
  T *out;
  bool live = group < a.groups;
  if (is_q) {
    out = reinterpret_cast<T *>(a.q_out) + (int64_t)b * a.Hq * a.how.D;
  } else {
    const int pi = pos >= 0 ? pos / a.page : a.max_pages;
    const int id = pi < a.max_pages ? a.table[(int64_t)b * a.max_pages + pi] : -1;
    if ((unsigned)id >= (unsigned)a.num_pages) {
      if (live && !is_v && first == 0 && lane == 0 && a.overflow) atomicAdd(a.overflow, 1);
      live = false;
    }
    out = reinterpret_cast<T *>(is_v ? a.v_pool : a.k_pool) + (live ? id * a.p_page + (pos - (int64_t)pi * a.page) * a.p_row : 0);
  }
  if (!is_v) {
    RotaryTurn<VEC, LPR, NP, IL> turn;
    turn.load(a.how, pos, lane);
#pragma unroll
    for (int h = 0; h < HPG; ++h) norm_and_turn(a.how, rows[h], turn, weight, lane);
  }
#pragma unroll
  for (int h = 0; h < HPG; ++h)
    if (live && first + h < heads) store_row<false>(a.how, rows[h], out + (first + h) * out_head, lane);
}

}  // namespace en

using namespace en;

extern "C" int en_qk_norm_rotary(const void *q, const void *k, void *q_out, void *k_out, const int32_t *cu_seqlens, const int32_t *positions,
                                 int batch, int64_t tokens, int q_heads, int k_heads, int size_per_head, const int64_t *strides,
                                 const en_norm_rotary *how, int dtype, en_stream_t stream) {
  const int es = dtype_size(dtype);
  if (!es) return EN_ERR_DTYPE;
  if (const int bad = check_rotary(how, size_per_head)) return bad;
  if (batch < 0 || tokens < 0 || q_heads < 1 || k_heads < 0) return EN_ERR_SHAPE;
  if (!strides || !q || !q_out || (k_heads && (!k || !k_out)) || (!cu_seqlens && !positions)) return EN_ERR_NULL;
  for (const void *p : {q, k, (const void *)q_out, (const void *)k_out, how->q_weight, how->k_weight})
    if (!aligned_to(p, es)) return EN_ERR_ALIGN;
  if (tokens == 0 || (!positions && batch == 0)) return EN_OK;
  const int64_t rows = tokens * (q_heads + k_heads);
  const bool many = rows >= kManyRows;
  const int hpg = many ? 4 : 1;
  const bool il = how->interleaved != 0;
  const RotaryForm form = rotary_form(size_per_head, how->rotary_dim, il, dtype);
  RotaryRowsArgs a{rotary_how(how, size_per_head, form.vec), {q, k}, {q_out, k_out}, {strides[0], strides[2]}, {strides[1], strides[3]},
                   {strides[4], strides[6]}, {strides[5], strides[7]}, {q_heads, k_heads},
                   {(int)ceil_div(q_heads, hpg), (int)ceil_div(k_heads, hpg)}, cu_seqlens, positions, batch, 0, 0};
  const int64_t groups = tokens * (a.parts[0] + a.parts[1]);
  if (groups > INT32_MAX) return EN_ERR_SHAPE;
  a.tokens = (uint32_t)tokens;
  a.groups = (uint32_t)groups;
  const int64_t bytes = tokens * (q_heads + k_heads) * size_per_head * es;
  const hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return with_rotary_form<DT>(form, il, [&](auto vec, auto lpr, auto np, auto inter) {
      constexpr int VEC = decltype(vec)::value, LPR = decltype(lpr)::value, NP = decltype(np)::value;
      constexpr bool IL = decltype(inter)::value;
      const unsigned grid = (unsigned)ceil_div(groups, kBlock / LPR);
      if (!many) qk_norm_rotary_kernel<DT, VEC, LPR, NP, IL, 1, false><<<grid, kBlock, 0, s>>>(a);
      else if (bytes < kStreamStoreBytes) qk_norm_rotary_kernel<DT, VEC, LPR, NP, IL, 4, false><<<grid, kBlock, 0, s>>>(a);
      else if (bytes < kStreamLoadBytes) qk_norm_rotary_kernel<DT, VEC, LPR, NP, IL, 4, true><<<grid, kBlock, 0, s>>>(a);
      else qk_norm_rotary_kernel<DT, VEC, LPR, NP, IL, 4, true, true><<<grid, kBlock, 0, s>>>(a);
    });
  };
  const bool known = dtype == EN_F32 ? launch(Int<EN_F32>{}) : dtype == EN_F16 ? launch(Int<EN_F16>{}) : launch(Int<EN_BF16>{});
  if (!known) return EN_ERR_UNSUPPORTED;
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

extern "C" int en_kv_append_paged_rotary(const void *q, const void *k_new, const void *v_new, void *q_out, void *k_pool, void *v_pool,
                                         const int32_t *kv_lens, const int32_t *page_table, int batch, int q_heads, int k_heads,
                                         int max_pages_per_seq, int page_size, int num_pages, int size_per_head, const int64_t *strides,
                                         const int64_t *pool_strides, const en_norm_rotary *how, int dtype, int32_t *overflow,
                                         en_stream_t stream) {
  const int es = dtype_size(dtype);
  if (!es) return EN_ERR_DTYPE;
  if (const int bad = check_rotary(how, size_per_head)) return bad;
  if (batch < 0 || q_heads < 1 || k_heads < 1 || max_pages_per_seq < 0 || num_pages < 0 || page_size < 16 || (page_size & (page_size - 1))) return EN_ERR_SHAPE;
  if (!q || !k_new || !v_new || !q_out || !k_pool || !v_pool || !kv_lens || !page_table || !strides || !pool_strides) return EN_ERR_NULL;
  for (const void *p : {q, k_new, v_new, (const void *)q_out, (const void *)k_pool, (const void *)v_pool, how->q_weight, how->k_weight})
    if (!aligned_to(p, es)) return EN_ERR_ALIGN;
  if (batch == 0) return EN_OK;
  const int64_t rows = (int64_t)batch * (q_heads + 2 * (int64_t)k_heads);
  if (rows > INT32_MAX) return EN_ERR_SHAPE;
  const bool il = how->interleaved != 0;
  const RotaryForm form = rotary_form(size_per_head, how->rotary_dim, il, dtype);
  const int hpg = rows >= kManyRows / 2 ? 2 : 1;
  RotaryAppendArgs a{rotary_how(how, size_per_head, form.vec), q, k_new, v_new, q_out, k_pool, v_pool, kv_lens, page_table,
                           strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], pool_strides[0], pool_strides[1],
                           pool_strides[2], batch, q_heads, k_heads, max_pages_per_seq, page_size, num_pages,
                           (int)ceil_div(q_heads, hpg), (int)ceil_div(k_heads, hpg), 0, overflow};
  const int64_t groups = batch * (a.parts_q + 2 * (int64_t)a.parts_k);
  a.groups = (uint32_t)groups;
  const hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return with_rotary_form<DT>(form, il, [&](auto vec, auto lpr, auto np, auto inter) {
      constexpr int LPR = decltype(lpr)::value;
      const unsigned grid = (unsigned)ceil_div(groups, kBlock / LPR);
      if (hpg == 1) kv_append_paged_rotary_kernel<DT, decltype(vec)::value, LPR, decltype(np)::value, decltype(inter)::value, 1><<<grid, kBlock, 0, s>>>(a);
      else kv_append_paged_rotary_kernel<DT, decltype(vec)::value, LPR, decltype(np)::value, decltype(inter)::value, 2><<<grid, kBlock, 0, s>>>(a);
    });
  };
  const bool known = dtype == EN_F32 ? launch(Int<EN_F32>{}) : dtype == EN_F16 ? launch(Int<EN_F16>{}) : launch(Int<EN_BF16>{});
  if (!known) return EN_ERR_UNSUPPORTED;
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

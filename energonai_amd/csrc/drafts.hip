// Drafted tokens around their attention: the tree's masks, which of them a greedy decoding accepts, and the accepted rows' way into the
// cache.
#include <type_traits>

#include "paged_common.hip.h"

namespace en {

constexpr int kNodes = EN_DRAFT_MAX_NODES;

__device__ __forceinline__ int draft_nodes(const int32_t *cu, int b, int max_nodes) { return min(max(cu[b + 1] - cu[b], 0), max_nodes); }

// One wave a sequence, lane i node i.  Every round doubles the way that is known: a mask takes in that of the node it has come to, and goes
// on from where that one has.
__global__ __launch_bounds__(kWave) void draft_tree_kernel(const int32_t *parents, const int32_t *cu, int64_t total, int64_t *masks, int32_t *depths) {
  const int b = blockIdx.x, lane = threadIdx.x, first = cu[b], nodes = draft_nodes(cu, b, INT32_MAX);
  int up = lane < min(nodes, kNodes) && (int64_t)first + lane < total ? parents[first + lane] : -1;
  if (up >= lane || up < 0) up = -1;
  uint64_t mask = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int from = max(up, 0);
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)mask, from, kWave), hi = (uint32_t)__shfl((int)(uint32_t)(mask >> 32), from, kWave);
    const int further = __shfl(up, from, kWave);
    if (up >= 0) {
      mask |= (uint64_t)hi << 32 | lo;
      up = further;
    }
  }
  for (int i = lane; i < nodes && first + (int64_t)i < total; i += kWave) {
    masks[first + i] = i < kNodes ? (int64_t)mask : 0;
    depths[first + i] = i < kNodes ? __popcll(mask) - 1 : 0;
  }
  // the rows behind the last sequence are no nodes either: all waves' work
  for (int64_t i = max(cu[gridDim.x], 0) + (int64_t)b * kWave + lane; i < total; i += (int64_t)gridDim.x * kWave) {
    masks[i] = 0;
    depths[i] = 0;
  }
}

// ---- acceptance ------------------------------------------------------------------------------------------------------------------

// What counts is how a row's largest logit is found: the rows on the way are read one after another, each by what the one before chose, and a
// compute unit that reads one by itself is bound by its instructions as much as by its loads.  So a lane takes vectors of 16 bytes, 16-bit
// logits two at a time as the integers that they are stored as, and remembers only which of its vectors holds the largest; the vector is read
// once more for the index.  As signed integers numbers from 0 up are in their order and above the negative ones, and NaN is above
// infinity; as unsigned ones a negative NaN is above all.  A row with NaN, or whose largest logit is 0 or negative, is gone over once more
// element by element.  (64 trees, 12 rows of 128000 on the longest way, bf16: 52 us, 4.4 a row, what a compute unit draws by itself: twice as
// many loads in flight change nothing; 71 us in the numbers' own order, sign and magnitude turned into it, 35 instructions a vector.)
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <int DT> struct Logits {
  static constexpr int kPer = 16 / Elem<DT>::kSize;
  static constexpr int kInf = DT == EN_F16 ? 0x7c00 : DT == EN_BF16 ? 0x7f80 : 0x7f800000;
  // The vector's largest as signed integers; `top` is raised to its largest as unsigned ones, half by half.
  __device__ static __forceinline__ int largest(const uint4 &v, uint32_t &top) {
    if constexpr (DT == EN_F32) {
      top = max(max(top, v.x), max(max(v.y, v.z), v.w));
      return max(max((int)v.x, (int)v.y), max((int)v.z, (int)v.w));
    } else {
      auto s = [](uint32_t x) { return __builtin_bit_cast(s16x2, x); };
      auto u = [](uint32_t x) { return __builtin_bit_cast(u16x2, x); };
      top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(u(top), __builtin_elementwise_max(__builtin_elementwise_max(u(v.x), u(v.y)), __builtin_elementwise_max(u(v.z), u(v.w)))));
      const s16x2 o = __builtin_elementwise_max(__builtin_elementwise_max(s(v.x), s(v.y)), __builtin_elementwise_max(s(v.z), s(v.w)));
      return max((int)o.x, (int)o.y);
    }
  }
  __device__ static __forceinline__ bool negative_nan(uint32_t top) {
    if constexpr (DT == EN_F32) return top > 0xff800000u;
    else return max(top & 0xffffu, top >> 16) > (0x8000u | (uint32_t)kInf);
  }
  // Index of the first element that is stored as `bits`.
  __device__ static __forceinline__ int first(const uint4 &v, uint32_t bits) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    int at = 0;
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i) at = (DT == EN_F32 ? w[i % 4] : w[i / 2 % 4] >> (16 * (i % 2)) & 0xffffu) == bits ? i : at;
    return at;
  }
};

// Logits in an order of whole numbers, NaN above all, zeros equal; 0 is below all of them.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0xffffffffu : x == 0.f ? 0x80000000u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint64_t w = (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), d, kWave) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, d, kWave);
    v = w > v ? w : v;
  }
  return v;
}
// Over a workgroup of W waves; every lane has the result.  Slots belong to one of two calls in turn.
template <int W> __device__ __forceinline__ uint64_t block_largest(uint64_t v, uint64_t *slots) {
  v = wave_largest(v);
  if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) v = max(v, slots[w]);
  return v;
}

// The largest of elements from .. to - 1 of a row, at least one: `ordered` above, the complement of its index below.
template <int DT, int W>
__device__ __forceinline__ uint64_t row_best(const typename Elem<DT>::T *row, int from, int to, uint64_t (*slots)[W]) {
  typedef Logits<DT> L;
  typedef typename Elem<DT>::T T;
  constexpr int kThreads = W * kWave, kPer = L::kPer, kAhead = 8;
  if (to - from >= kPer) {
    const int vectors = (to - from + kPer - 1) / kPer;
    auto start = [&](int v) { return min(from + v * kPer, to - kPer); };       // the last one overlaps the one before
    int best = INT32_MIN, at = 0;
    uint32_t above = 0;
    for (int v0 = threadIdx.x; v0 < vectors; v0 += kAhead * kThreads) {
      uint4 x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) x[i] = load16_at<false, sizeof(T)>(row + start(min(v0 + i * kThreads, vectors - 1)));
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int o = L::largest(x[i], above);
        if (o > best) {
          best = o;
          at = min(v0 + i * kThreads, vectors - 1);
        }
      }
    }
    // (a lane without vectors has INT32_MIN, which is 0 here)
    const uint64_t mine = (uint64_t)((uint32_t)best ^ 0x80000000u) << 32 | (uint32_t)~at;
    const uint64_t all = block_largest<W>(L::negative_nan(above) ? ~0ull : mine, slots[0]);
    const int largest = (int)((uint32_t)(all >> 32) ^ 0x80000000u);
    if (largest > 0 && largest <= L::kInf) {
      const int s = start((int)~(uint32_t)all);
      const int i = s + L::first(load16_at<false, sizeof(T)>(row + s), (uint32_t)largest);
      return (uint64_t)ordered(Elem<DT>::to_float(row[i])) << 32 | (uint32_t)~i;
    }
  }
  uint64_t best = 0;
  for (int i = from + threadIdx.x; i < to; i += kThreads) {
    const uint64_t v = (uint64_t)ordered(Elem<DT>::to_float(row[i])) << 32 | (uint32_t)~i;
    best = v > best ? v : best;
  }
  return block_largest<W>(best, slots[1]);
}

struct AcceptArgs {
  const void *logits;
  int64_t stride, total;
  int vocab;
  const void *tokens;
  int tokens_i64;
  const int32_t *parents, *cu;
  int max_nodes;
  int32_t *path, *counts;
  int64_t *next;
  uint64_t *best;                // [rows][slices] where all rows are looked at first
  int slices, slice;             // elements of a slice, a multiple of a vector
};

// The largest logit of every row, in slices.
constexpr int kBestWaves = 4;
template <int DT>
__global__ __launch_bounds__(kBestWaves *kWave) void accept_rows_kernel(AcceptArgs a) {
  __shared__ uint64_t s_best[2][kBestWaves];
  const int64_t row = blockIdx.x;
  const int from = blockIdx.y * a.slice;
  const uint64_t best = row_best<DT, kBestWaves>(reinterpret_cast<const typename Elem<DT>::T *>(a.logits) + row * a.stride, from, min(from + a.slice, a.vocab), s_best);
  if (threadIdx.x == 0) a.best[row * a.slices + blockIdx.y] = best;
}

// A workgroup walks a sequence's tree: W waves that read a row a round, or one wave where all rows have been looked at.
template <int DT, int W>
__global__ __launch_bounds__(W *kWave) void accept_walk_kernel(AcceptArgs a) {
  __shared__ uint64_t s_best[2][2][W];
  const int b = blockIdx.x, first = a.cu[b], lane = threadIdx.x % kWave;
  const int nodes = (int)min((int64_t)draft_nodes(a.cu, b, a.max_nodes), a.total - first);
  int32_t *path = a.path + (int64_t)b * a.max_nodes;
  // every wave has the whole tree, a node a lane
  const bool there = lane < nodes;
  const int parent = there ? a.parents[first + lane] : -2;
  const int64_t token = !there ? -1 : a.tokens_i64 ? reinterpret_cast<const int64_t *>(a.tokens)[first + lane] : reinterpret_cast<const int32_t *>(a.tokens)[first + lane];
  uint64_t mine = 0;
  if constexpr (W == 1)
    for (int i = 0; there && i < a.slices; ++i) mine = max(mine, a.best[(int64_t)(first + lane) * a.slices + i]);
  int cur = 0, count = 0;
  int64_t chosen = -1;
  while (cur < nodes) {
    uint32_t low;
    if constexpr (W == 1) {
      low = (uint32_t)__shfl((int)(uint32_t)mine, cur, kWave);
    } else {
      low = (uint32_t)row_best<DT, W>(reinterpret_cast<const typename Elem<DT>::T *>(a.logits) + (first + cur) * a.stride, 0, a.vocab, s_best[count & 1]);
    }
    chosen = (int64_t)(uint32_t)~low;
    if (threadIdx.x == 0) path[count] = cur;
    ++count;
    const uint64_t fits = __ballot(lane > cur && parent == cur && token == chosen);
    if (!fits) break;
    cur = __builtin_ctzll(fits);
  }
  for (int i = count + threadIdx.x; i < a.max_nodes; i += W * kWave) path[i] = -1;
  if (threadIdx.x == 0) {
    a.counts[b] = count;
    a.next[b] = chosen;
  }
}

constexpr int kWalkWaves = 16;
// us, a row at a time as the walk comes to it / all rows first: 4 trees of up to 32 nodes, vocabulary 128000 (23 MB) 17.0 / 11.0; 32 of 16, 50257 (49
// MB) 26.5 / 14.7; 8 of 32, 128000 (62 MB) 17.2 / 14.7; 64 of 16, 50257 (98 MB) 26.6 / 23.4; 16 of 32, 128000 (125 MB) 17.4 / 23.5.
constexpr int64_t kAllBytes = 96ll << 20, kSliceBytes = 32 << 10;
// Slices of a row where all rows are looked at first; 0: a row at a time, as the walk comes to it.
inline int accept_slices(int64_t nodes, int64_t vocab, int es) {
  if (nodes > kAllBytes / (vocab * es)) return 0;
  const int64_t n = ceil_div(vocab * es, kSliceBytes);
  return (int)(n < 1 ? 1 : n);
}

// ---- accepted rows into the pages --------------------------------------------------------------------------------------------------

struct ExtendArgs {
  const char *k_new, *v_new;
  char *k_pool, *v_pool;
  int64_t kn_token, kn_head, vn_token, vn_head, k_page, k_head, k_row, v_page, v_head, v_row;      // bytes
  const int32_t *table, *lens, *cu, *path, *counts;
  int64_t total;
  int width, max_nodes, num_pages, lg_page, max_pages, H;
  int row_bytes;
  int32_t *overflow;
};

// Keys and values of a sequence in workgroups of their own, which take what is accepted in vectors of W bytes, one by one: most sequences
// accept a few of the nodes that there is room for, and a workgroup for each node and head is mostly launches of nothing (256 sequences
// of up to 32 nodes, 8 heads x 128: 29.8 us, so 4.8).  Bound by the launch and the trip count, path, page, row.
template <int W>
__global__ __launch_bounds__(kBlock) void extend_kernel(ExtendArgs a) {
  typedef Pack<uint8_t, W> P;
  const int b = blockIdx.y, first = a.cu[b], count = min(a.counts[b], a.width), nodes = draft_nodes(a.cu, b, a.max_nodes), len = a.lens[b];
  const bool value = blockIdx.z;
  const char *from = value ? a.v_new : a.k_new;
  char *to = value ? a.v_pool : a.k_pool;
  const int64_t token = value ? a.vn_token : a.kn_token, from_head = value ? a.vn_head : a.kn_head, page = value ? a.v_page : a.k_page,
                to_head = value ? a.v_head : a.k_head, to_row = value ? a.v_row : a.k_row;
  const uint32_t vectors = a.row_bytes / W, each = vectors * a.H;
  for (uint32_t e = blockIdx.x * kBlock + threadIdx.x; count > 0 && e < each * count; e += gridDim.x * kBlock) {
    const uint32_t i = e / each, in = e - i * each, h = in / vectors, at = (in - h * vectors) * W;
    const int node = a.path[(int64_t)b * a.width + i];
    if (node < 0 || node >= nodes || (int64_t)first + node >= a.total) continue;
    const int64_t pos = (int64_t)len + i;
    const bool named = pos >= 0 && pos < ((int64_t)a.max_pages << a.lg_page);
    const int id = named ? a.table[(int64_t)b * a.max_pages + (pos >> a.lg_page)] : -1;
    if ((unsigned)id >= (unsigned)a.num_pages) {
      if (a.overflow && in == 0 && !value) atomicAdd(a.overflow, 1);
      continue;
    }
    const int64_t row = pos & ((1 << a.lg_page) - 1);
    *reinterpret_cast<P *>(to + id * page + h * to_head + row * to_row + at) = *reinterpret_cast<const P *>(from + ((int64_t)first + node) * token + h * from_head + at);
  }
}

}  // namespace en

using namespace en;

extern "C" {

int en_draft_tree(const int32_t *parents, const int32_t *cu_seqlens, int batch, int64_t nodes, int64_t *masks, int32_t *depths, en_stream_t stream) {
  if (batch < 0 || nodes < 0 || nodes > INT32_MAX) return EN_ERR_SHAPE;
  if (batch == 0 || nodes == 0) return EN_OK;
  if (!parents || !cu_seqlens || !masks || !depths) return EN_ERR_NULL;
  if (!aligned_to(masks, 8) || !aligned_to(parents, 4) || !aligned_to(cu_seqlens, 4) || !aligned_to(depths, 4)) return EN_ERR_ALIGN;
  draft_tree_kernel<<<(unsigned)batch, kWave, 0, (hipStream_t)stream>>>(parents, cu_seqlens, nodes, masks, depths);
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

int64_t en_accept_drafts_workspace_bytes(int64_t nodes, int vocab, int dtype) {
  const int es = dtype_size(dtype);
  if (es == 0 || nodes < 1 || nodes > INT32_MAX || vocab < 1) return 0;
  return nodes * accept_slices(nodes, vocab, es) * 8;
}

int en_accept_drafts(const void *logits, int64_t logits_stride, int vocab, const void *tokens, int tokens_are_i64, const int32_t *parents,
                     const int32_t *cu_seqlens, int batch, int64_t nodes, int max_nodes, int32_t *path, int32_t *counts, int64_t *next_tokens,
                     int dtype, void *workspace, int64_t workspace_bytes, en_stream_t stream) {
  const int es = dtype_size(dtype);
  if (es == 0) return EN_ERR_DTYPE;
  if (batch < 0 || nodes < 0 || nodes > INT32_MAX || max_nodes < 1 || max_nodes > kNodes || vocab < 1 || vocab > INT32_MAX - (1 << 20) || logits_stride < 0) return EN_ERR_SHAPE;
  if (batch == 0) return EN_OK;
  const int64_t need = en_accept_drafts_workspace_bytes(nodes, vocab, dtype);
  if (!cu_seqlens || !path || !counts || !next_tokens || (nodes > 0 && (!logits || !tokens || !parents)) || (need > 0 && !workspace)) return EN_ERR_NULL;
  if (workspace_bytes < need) return EN_ERR_SHAPE;
  if (!aligned_to(logits, es) || !aligned_to(tokens, tokens_are_i64 ? 8 : 4) || !aligned_to(next_tokens, 8) || !aligned_to(workspace, 8)) return EN_ERR_ALIGN;
  for (const void *p : {(const void *)parents, (const void *)cu_seqlens, (const void *)path, (const void *)counts})
    if (!aligned_to(p, 4)) return EN_ERR_ALIGN;
  AcceptArgs a{logits, logits_stride, nodes, vocab, tokens, tokens_are_i64, parents, cu_seqlens, max_nodes, path, counts, next_tokens, (uint64_t *)workspace,
               nodes > 0 ? accept_slices(nodes, vocab, es) : 1, 0};
  const hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.slices == 0) {
      accept_walk_kernel<DT, kWalkWaves><<<(unsigned)batch, kWalkWaves * kWave, 0, s>>>(a);
      return;
    }
    const int per = 16 / es;
    a.slice = (int)(ceil_div(ceil_div(vocab, a.slices), per) * per);
    a.slices = (int)ceil_div(vocab, a.slice);
    if (nodes > 0) accept_rows_kernel<DT><<<dim3((unsigned)nodes, (unsigned)a.slices), kBestWaves * kWave, 0, s>>>(a);
    accept_walk_kernel<DT, 1><<<(unsigned)batch, kWave, 0, s>>>(a);
  };
  if (dtype == EN_F32) launch(std::integral_constant<int, EN_F32>{});
  else if (dtype == EN_F16) launch(std::integral_constant<int, EN_F16>{});
  else launch(std::integral_constant<int, EN_BF16>{});
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

int en_kv_extend_paged_nodes(const void *k_new, const void *v_new, const int64_t *strides, const en_kv_pages *cache, const int32_t *kv_lens,
                             const int32_t *cu_seqlens, int64_t nodes, int max_nodes, const int32_t *path, int path_width, const int32_t *counts,
                             int32_t *overflow, en_stream_t stream) {
  if (!cache || !strides) return EN_ERR_NULL;
  const en_kv_pages &c = *cache;
  if (const int bad = check_kv_pages(c)) return bad;
  if (nodes < 0 || nodes > INT32_MAX || max_nodes < 0 || max_nodes > kNodes || path_width < 0 || path_width > kNodes || c.batch > 65535) return EN_ERR_SHAPE;
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0) return EN_ERR_SHAPE;
  if (c.batch == 0 || nodes == 0 || path_width == 0) return EN_OK;
  if (!k_new || !v_new || !kv_lens || !cu_seqlens || !path || !counts) return EN_ERR_NULL;
  const int64_t es = dtype_size(c.dtype);
  if (!aligned_to(k_new, es) || !aligned_to(v_new, es)) return EN_ERR_ALIGN;
  ExtendArgs a{};
  a.k_new = (const char *)k_new; a.v_new = (const char *)v_new; a.k_pool = (char *)c.k_pool; a.v_pool = (char *)c.v_pool;
  a.kn_token = es * strides[0]; a.kn_head = es * strides[1]; a.vn_token = es * strides[2]; a.vn_head = es * strides[3];
  a.k_page = es * c.strides[0]; a.k_head = es * c.strides[1]; a.k_row = es * c.strides[2];
  a.v_page = es * c.strides[3]; a.v_head = es * c.strides[4]; a.v_row = es * c.strides[5];
  a.table = c.page_table; a.lens = kv_lens; a.cu = cu_seqlens; a.path = path; a.counts = counts;
  a.total = nodes; a.width = path_width; a.max_nodes = max_nodes; a.num_pages = c.num_pages; a.lg_page = page_log2(c.page_size); a.max_pages = c.max_pages_per_seq; a.H = c.head_num;
  a.row_bytes = (int)(es * c.size_per_head);
  a.overflow = overflow;
  // the widest access that every row's address and length allow
  uint64_t all = (uint64_t)a.row_bytes | (uint64_t)(uintptr_t)k_new | (uint64_t)(uintptr_t)v_new | (uint64_t)(uintptr_t)c.k_pool | (uint64_t)(uintptr_t)c.v_pool;
  for (const int64_t v : {a.kn_token, a.kn_head, a.vn_token, a.vn_head, a.k_page, a.k_head, a.k_row, a.v_page, a.v_head, a.v_row}) all |= (uint64_t)v;
  const int width = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
  const int64_t vectors = (int64_t)path_width * c.head_num * (a.row_bytes / width);
  if (vectors > INT32_MAX) return EN_ERR_SHAPE;
  // eight vectors a lane where all nodes are accepted, in no more workgroups than are resident at once
  int64_t parts = ceil_div(vectors, 8 * kBlock);
  if (parts * c.batch > 1024) parts = ceil_div(1024, c.batch);
  const dim3 grid((unsigned)parts, (unsigned)c.batch, 2);
  const hipStream_t s = (hipStream_t)stream;
  if (width == 16) extend_kernel<16><<<grid, kBlock, 0, s>>>(a);
  else if (width == 4) extend_kernel<4><<<grid, kBlock, 0, s>>>(a);
  else extend_kernel<2><<<grid, kBlock, 0, s>>>(a);
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

int en_kv_extend_paged(const void *k_new, const void *v_new, const int64_t *strides, const en_kv_pages *cache, const int32_t *kv_lens,
                       const int32_t *cu_seqlens, int64_t nodes, const int32_t *path, int path_width, const int32_t *counts,
                       int32_t *overflow, en_stream_t stream) {
  return en_kv_extend_paged_nodes(k_new, v_new, strides, cache, kv_lens, cu_seqlens, nodes, kNodes, path, path_width, counts, overflow, stream);
}

}  // extern "C"

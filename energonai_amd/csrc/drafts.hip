// Drafted tokens around their attention: the tree's masks, which of them a greedy decoding accepts, and the accepted rows' way into the
// cache.
#include "paged_common.hip.h"

namespace en {

constexpr int kNodes = EN_DRAFT_MAX_NODES;

__device__ __forceinline__ int draft_nodes(const int32_t *cu, int b, int max_nodes) { return min(max(cu[b + 1] - cu[b], 0), max_nodes); }

// One wave a sequence, lane i node i.  Every round doubles the way that is known: a mask takes in that of the node it has come to, and goes
// on from where that one has.
__global__ __launch_bounds__(kWave) void draft_tree_kernel(const int32_t *parents, const int32_t *cu, int64_t total, int64_t *masks, int32_t *depths) {
  const int b = blockIdx.x, lane = threadIdx.x, first = cu[b], nodes = draft_nodes(cu, b, INT32_MAX);
  int up = lane < min(nodes, kNodes) && first + lane < total ? parents[first + lane] : -1;
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
}

// ---- acceptance ------------------------------------------------------------------------------------------------------------------

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
};

// Logits in an order of whole numbers, NaN above all; 0 is below all of them.
template <int DT> __device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0xffffffffu : x == 0.f ? 0x80000000u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kAcceptThreads = 1024;

// A workgroup walks a sequence's tree, a node a round.
template <int DT>
__global__ __launch_bounds__(kAcceptThreads) void accept_kernel(AcceptArgs a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  __shared__ uint64_t s_best[2][kAcceptThreads / kWave];
  const int b = blockIdx.x, first = a.cu[b], lane = threadIdx.x % kWave;
  const int nodes = (int)min((int64_t)draft_nodes(a.cu, b, a.max_nodes), a.total - first);
  int32_t *path = a.path + (int64_t)b * a.max_nodes;
  // every wave has the whole tree, a node a lane
  const int parent = lane < nodes ? a.parents[first + lane] : -2;
  const int64_t token = lane >= nodes ? -1 : a.tokens_i64 ? reinterpret_cast<const int64_t *>(a.tokens)[first + lane] : reinterpret_cast<const int32_t *>(a.tokens)[first + lane];
  int cur = 0, count = 0;
  int64_t chosen = -1;
  while (cur < nodes) {
    const T *row = reinterpret_cast<const T *>(a.logits) + (first + cur) * a.stride;
    uint64_t best = 0;           // the value's order above, the complement of its index below
    for (int i = threadIdx.x; i < a.vocab; i += kAcceptThreads) {
      const uint64_t v = (uint64_t)ordered<DT>(E::to_float(row[i])) << 32 | ~(uint32_t)i;
      best = v > best ? v : best;
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const uint64_t v = (uint64_t)(uint32_t)__shfl_xor((int)(best >> 32), d, kWave) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)best, d, kWave);
      best = v > best ? v : best;
    }
    if (lane == 0) s_best[count & 1][threadIdx.x / kWave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAcceptThreads / kWave; ++w) best = max(best, s_best[count & 1][w]);
    chosen = (int64_t)(~(uint32_t)best);
    if (threadIdx.x == 0) path[count] = cur;
    ++count;
    const uint64_t fits = __ballot(lane > cur && parent == cur && token == chosen);
    if (!fits) break;
    cur = __builtin_ctzll(fits);
  }
  for (int i = count + threadIdx.x; i < a.max_nodes; i += kAcceptThreads) path[i] = -1;
  if (threadIdx.x == 0) {
    a.counts[b] = count;
    a.next[b] = chosen;
  }
}

// ---- accepted rows into the pages --------------------------------------------------------------------------------------------------

struct ExtendArgs {
  const char *k_new, *v_new;
  char *k_pool, *v_pool;
  int64_t kn_token, kn_head, vn_token, vn_head, k_page, k_head, k_row, v_page, v_head, v_row;      // bytes
  const int32_t *table, *lens, *cu, *path, *counts;
  int64_t total;
  int width, num_pages, lg_page, max_pages, H;
  int row_bytes;
  int32_t *overflow;
};

// A wave a position and head; W bytes a lane and step.
template <int W>
__global__ __launch_bounds__(kWave) void extend_kernel(ExtendArgs a) {
  typedef Pack<uint8_t, W> P;
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  if (i >= a.counts[b]) return;
  const int first = a.cu[b], nodes = a.cu[b + 1] - first, node = a.path[(int64_t)b * a.width + i];
  if (node < 0 || node >= min(nodes, kNodes) || (int64_t)first + node >= a.total) return;
  const int64_t pos = (int64_t)a.lens[b] + i;
  const bool named = pos >= 0 && pos < ((int64_t)a.max_pages << a.lg_page);
  const int id = named ? a.table[(int64_t)b * a.max_pages + (pos >> a.lg_page)] : -1;
  if ((unsigned)id >= (unsigned)a.num_pages) {
    if (a.overflow && h == 0 && threadIdx.x == 0) atomicAdd(a.overflow, 1);
    return;
  }
  const int64_t row = pos & ((1 << a.lg_page) - 1), from = (int64_t)first + node;
  for (int at = threadIdx.x * W; at < a.row_bytes; at += kWave * W) {
    *reinterpret_cast<P *>(a.k_pool + id * a.k_page + h * a.k_head + row * a.k_row + at) = *reinterpret_cast<const P *>(a.k_new + from * a.kn_token + h * a.kn_head + at);
    *reinterpret_cast<P *>(a.v_pool + id * a.v_page + h * a.v_head + row * a.v_row + at) = *reinterpret_cast<const P *>(a.v_new + from * a.vn_token + h * a.vn_head + at);
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

int en_accept_drafts(const void *logits, int64_t logits_stride, int vocab, const void *tokens, int tokens_are_i64, const int32_t *parents,
                     const int32_t *cu_seqlens, int batch, int64_t nodes, int max_nodes, int32_t *path, int32_t *counts, int64_t *next_tokens,
                     int dtype, en_stream_t stream) {
  const int es = dtype_size(dtype);
  if (es == 0) return EN_ERR_DTYPE;
  if (batch < 0 || nodes < 0 || nodes > INT32_MAX || max_nodes < 1 || max_nodes > kNodes || vocab < 1 || logits_stride < 0) return EN_ERR_SHAPE;
  if (batch == 0) return EN_OK;
  if (!cu_seqlens || !path || !counts || !next_tokens || (nodes > 0 && (!logits || !tokens || !parents))) return EN_ERR_NULL;
  if (!aligned_to(logits, es) || !aligned_to(tokens, tokens_are_i64 ? 8 : 4) || !aligned_to(next_tokens, 8)) return EN_ERR_ALIGN;
  for (const void *p : {(const void *)parents, (const void *)cu_seqlens, (const void *)path, (const void *)counts})
    if (!aligned_to(p, 4)) return EN_ERR_ALIGN;
  const AcceptArgs a{logits, logits_stride, nodes, vocab, tokens, tokens_are_i64, parents, cu_seqlens, max_nodes, path, counts, next_tokens};
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == EN_F32) accept_kernel<EN_F32><<<(unsigned)batch, kAcceptThreads, 0, s>>>(a);
  else if (dtype == EN_F16) accept_kernel<EN_F16><<<(unsigned)batch, kAcceptThreads, 0, s>>>(a);
  else accept_kernel<EN_BF16><<<(unsigned)batch, kAcceptThreads, 0, s>>>(a);
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

int en_kv_extend_paged(const void *k_new, const void *v_new, const int64_t *strides, const en_kv_pages *cache, const int32_t *kv_lens,
                       const int32_t *cu_seqlens, int64_t nodes, const int32_t *path, int path_width, const int32_t *counts,
                       int32_t *overflow, en_stream_t stream) {
  if (!cache || !strides) return EN_ERR_NULL;
  const en_kv_pages &c = *cache;
  if (const int bad = check_kv_pages(c)) return bad;
  if (nodes < 0 || nodes > INT32_MAX || path_width < 0 || path_width > kNodes || c.batch > 65535) return EN_ERR_SHAPE;
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
  a.total = nodes; a.width = path_width; a.num_pages = c.num_pages; a.lg_page = page_log2(c.page_size); a.max_pages = c.max_pages_per_seq; a.H = c.head_num;
  a.row_bytes = (int)(es * c.size_per_head);
  a.overflow = overflow;
  // the widest access that every row's address and length allow
  uint64_t all = (uint64_t)a.row_bytes | (uint64_t)(uintptr_t)k_new | (uint64_t)(uintptr_t)v_new | (uint64_t)(uintptr_t)c.k_pool | (uint64_t)(uintptr_t)c.v_pool;
  for (const int64_t v : {a.kn_token, a.kn_head, a.vn_token, a.vn_head, a.k_page, a.k_head, a.k_row, a.v_page, a.v_head, a.v_row}) all |= (uint64_t)v;
  const dim3 grid((unsigned)c.head_num, (unsigned)path_width, (unsigned)c.batch);
  const hipStream_t s = (hipStream_t)stream;
  if (all % 16 == 0) extend_kernel<16><<<grid, kWave, 0, s>>>(a);
  else if (all % 4 == 0) extend_kernel<4><<<grid, kWave, 0, s>>>(a);
  else extend_kernel<2><<<grid, kWave, 0, s>>>(a);
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

}  // extern "C"

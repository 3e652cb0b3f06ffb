// The 8-bit K/V cache written and read back: prompts, a decode step's rows, and positions in 16 bits again.
//
// All three move bytes: a full block is 16 rows of 16-bit values in and a byte each out.  One wave takes a block of one head, keys or
// values; neighbouring waves take neighbouring heads, whose rows are neighbours in a projection's output.  Keys go through as they lie,
// 16 bytes a lane; values are read two channels a lane, so that a lane ends with all positions of its channels, which is how they are kept.
#include "kv8_common.hip.h"
#include "rotary_rows.hip.h"

namespace en {

// Two 16-bit elements as a word, at any element's address.
template <typename T, bool NT = false> __device__ __forceinline__ uint32_t load_two(const T *p) {
  return __builtin_bit_cast(uint32_t, load_loose<T, 2, NT>(p));
}
template <int DT> __device__ __forceinline__ float low_value(uint32_t w) {
  return Elem<DT>::to_float(__builtin_bit_cast(typename Elem<DT>::T, (uint16_t)w));
}
template <int DT> __device__ __forceinline__ float high_value(uint32_t w) {
  return Elem<DT>::to_float(__builtin_bit_cast(typename Elem<DT>::T, (uint16_t)(w >> 16)));
}
template <int DT> __device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The 16 rows of a block of keys: lane i holds vectors i, i + 64, .. of 8 channels, in row order.
template <int D> struct KeyBlock {
  static constexpr int kPerRow = D / 8, kVectors = kBlk * kPerRow, kEach = (kVectors + kWave - 1) / kWave;
  uint4 raw[kEach];
  __device__ static __forceinline__ bool has(int i, int lane) { return kVectors % kWave == 0 || i * kWave + lane < kVectors; }
  __device__ static __forceinline__ int row(int i, int lane) { return min(i * kWave + lane, kVectors - 1) / kPerRow; }
  __device__ static __forceinline__ int channel(int i, int lane) { return min(i * kWave + lane, kVectors - 1) % kPerRow * 8; }
};

template <int DT, int CODE, int D>
__device__ __forceinline__ void put_key_block(const KeyBlock<D> &k, uint8_t *codes, float *scale, int lane) {
  typedef KeyBlock<D> K;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < K::kEach; ++i) {
    const uint32_t w[4] = {k.raw[i].x, k.raw[i].y, k.raw[i].z, k.raw[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, max(magnitude<DT>(low_value<DT>(w[e])), magnitude<DT>(high_value<DT>(w[e]))));
  }
  const BlockScale s = block_scale<CODE>(wave_max_bits(top));
  if (lane == 0) *scale = s.scale;
  const bool none = s.inv == 0.f;                  // zeros, also for what is not finite
#pragma unroll
  for (int i = 0; i < K::kEach; ++i) {
    const uint32_t w[4] = {k.raw[i].x, k.raw[i].y, k.raw[i].z, k.raw[i].w};
    uint2 c;
    c.x = Codes<CODE>::four(low_value<DT>(w[0]), high_value<DT>(w[0]), low_value<DT>(w[1]), high_value<DT>(w[1]), s.inv);
    c.y = Codes<CODE>::four(low_value<DT>(w[2]), high_value<DT>(w[2]), low_value<DT>(w[3]), high_value<DT>(w[3]), s.inv);
    if (none) c = make_uint2(0, 0);
    if (K::has(i, lane)) *reinterpret_cast<uint2 *>(codes + (i * kWave + lane) * 8) = c;
  }
}

// The values of a block: lane l holds channels 2c, 2c + 1 (c = l % (D/2)) of positions first .. first + kEach - 1.  Heads of up to 64
// channels share the 16 positions between the wave's halves.
template <int D> struct ValueBlock {
  static constexpr int kHalves = D <= 64 ? 2 : 1, kEach = kBlk / kHalves, kLanes = kWave / kHalves;
  uint32_t raw[kEach];                             // position first + i: channel 2c low, 2c + 1 high
  __device__ static __forceinline__ int pair(int lane) { return min(lane % kLanes, D / 2 - 1); }
  __device__ static __forceinline__ bool has(int lane) { return lane % kLanes < D / 2; }
  __device__ static __forceinline__ int first(int lane) { return lane / kLanes * kEach; }
};

// The same of a tail, which has the positions of a channel side by side.
template <int D> __device__ __forceinline__ void value_rows(const uint16_t *tail, int lane, uint32_t (&raw)[ValueBlock<D>::kEach]) {
  typedef ValueBlock<D> V;
  const uint16_t *from = tail + 2 * V::pair(lane) * kBlk + V::first(lane);
#pragma unroll
  for (int i = 0; i < V::kEach; i += 8) {
    const uint4 lo = *reinterpret_cast<const uint4 *>(from + i), hi = *reinterpret_cast<const uint4 *>(from + kBlk + i);
    const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, u[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      raw[i + 2 * e] = (l[e] & 0xffffu) | u[e] << 16;
      raw[i + 2 * e + 1] = l[e] >> 16 | (u[e] & 0xffff0000u);
    }
  }
}

template <int DT, int CODE, int D>
__device__ __forceinline__ void put_value_block(const ValueBlock<D> &v, uint8_t *codes, float *scale, int lane) {
  typedef ValueBlock<D> V;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < V::kEach; ++i) top = max(top, max(magnitude<DT>(low_value<DT>(v.raw[i])), magnitude<DT>(high_value<DT>(v.raw[i]))));
  const BlockScale s = block_scale<CODE>(wave_max_bits(top));
  if (lane == 0) *scale = s.scale;
  const bool none = s.inv == 0.f;
  uint32_t c[2][V::kEach / 4];
#pragma unroll
  for (int j = 0; j < V::kEach / 4; ++j) {
    const uint32_t *w = v.raw + 4 * j;
    c[0][j] = Codes<CODE>::four(low_value<DT>(w[0]), low_value<DT>(w[1]), low_value<DT>(w[2]), low_value<DT>(w[3]), s.inv);
    c[1][j] = Codes<CODE>::four(high_value<DT>(w[0]), high_value<DT>(w[1]), high_value<DT>(w[2]), high_value<DT>(w[3]), s.inv);
    if (none) c[0][j] = c[1][j] = 0;
  }
  if (!V::has(lane)) return;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint8_t *to = codes + (2 * V::pair(lane) + half) * kBlk + V::first(lane);
    if constexpr (V::kEach == 16) *reinterpret_cast<uint4 *>(to) = make_uint4(c[half][0], c[half][1], c[half][2], c[half][3]);
    else *reinterpret_cast<uint2 *>(to) = make_uint2(c[half][0], c[half][1]);
  }
}

// ---- prompts ---------------------------------------------------------------------------------------------------------------------------

struct Kv8FillArgs {
  Kv8 c;
  const void *k, *v;
  int64_t k_token, k_head, v_token, v_head;
  const int32_t *cu;
  int max_seq_len;
  int64_t tokens;
  int32_t *overflow;
};

// Grid: blocks of the longest sequence (its last may be a tail) x 2 heads (keys, values) x sequences; four waves a workgroup.
template <int DT, int CODE, int D, bool NT>
__global__ __launch_bounds__(kBlock) void kv8_fill_kernel(Kv8FillArgs a) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x % kWave, unit = blockIdx.y * (kBlock / kWave) + threadIdx.x / kWave;
  const int b = blockIdx.z, j = blockIdx.x, H = a.c.H;
  const int start = a.cu[b], n = (int)min((int64_t)min(a.cu[b + 1] - start, a.max_seq_len), a.tokens - start);
  const int rows = min(n - j * kBlk, kBlk);
  if (unit >= 2 * H) return;
  const bool is_v = unit >= H;
  const int h = is_v ? unit - H : unit;
  if (rows <= 0) return;
  const T *src = is_v ? reinterpret_cast<const T *>(a.v) + (int64_t)h * a.v_head : reinterpret_cast<const T *>(a.k) + (int64_t)h * a.k_head;
  const int64_t step = is_v ? a.v_token : a.k_token;
  src += (int64_t)(start + j * kBlk) * step;
  const int64_t tail = ((int64_t)b * H + h) * kBlk * D;
  const int blk = kv8_block_in_page(a.c, j);
  int id;
  // the rows are on their way before the page is asked for
  auto no_page = [&]() {
    id = kv8_page(a.c, b, j);
    if (id < 0 && !is_v && h == 0 && lane == 0 && a.overflow) atomicAdd(a.overflow, rows);
    return id < 0;
  };
  if (!is_v) {
    typedef KeyBlock<D> K;
    K k;
#pragma unroll
    for (int i = 0; i < K::kEach; ++i)
      k.raw[i] = __builtin_bit_cast(uint4, load_loose<T, 8, NT>(src + min(K::row(i, lane), rows - 1) * step + K::channel(i, lane)));
    if (no_page()) return;
    if (rows == kBlk) {
      put_key_block<DT, CODE, D>(k, kv8_k_block(a.c, id, h, blk, D), a.c.ks + kv8_k_scale(a.c, id, h, blk), lane);
    } else {
#pragma unroll
      for (int i = 0; i < K::kEach; ++i)
        if (K::has(i, lane) && K::row(i, lane) < rows)
          *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.c.kt) + tail + (i * kWave + lane) * 8) = k.raw[i];
    }
  } else {
    typedef ValueBlock<D> V;
    V v;
#pragma unroll
    for (int i = 0; i < V::kEach; ++i) v.raw[i] = load_two<T, NT>(src + min(V::first(lane) + i, rows - 1) * step + 2 * V::pair(lane));
    if (no_page()) return;
    if (rows == kBlk) {
      put_value_block<DT, CODE, D>(v, kv8_v_block(a.c, id, h, blk, D), a.c.vs + kv8_v_scale(a.c, id, h, blk), lane);
    } else if (V::has(lane)) {
      uint16_t *to = reinterpret_cast<uint16_t *>(a.c.vt) + tail + 2 * V::pair(lane) * kBlk + V::first(lane);
#pragma unroll
      for (int i = 0; i < V::kEach; ++i)
        if (V::first(lane) + i < rows) {
          to[i] = (uint16_t)v.raw[i];
          to[kBlk + i] = (uint16_t)(v.raw[i] >> 16);
        }
    }
  }
}

// ---- a decode step's rows --------------------------------------------------------------------------------------------------------------

struct Kv8AppendArgs {
  Kv8 c;
  RotaryHow how;
  const void *q, *k, *v;
  void *q_out;
  const int32_t *lens;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh;
  int Hq, parts_q, interleaved;
  uint32_t units;                     // B * (parts_q + 2 H)
  int32_t *overflow;
};

// A row of up to 128 channels, a pair a lane.
template <int DT, bool IL> using PairRow = RotaryRow<DT, 1, kWave, 1, IL>;

// Up to kTurned heads of q of one sequence.
constexpr int kTurned = 4;
template <int DT, bool IL>
__device__ __forceinline__ void turn_queries(const Kv8AppendArgs &a, int b, int first, int pos, int lane) {
  typedef typename Elem<DT>::T T;
  PairRow<DT, IL> rows[kTurned];
#pragma unroll
  for (int h = 0; h < kTurned; ++h) rows[h].load(a.how, reinterpret_cast<const T *>(a.q) + b * a.q_sb + min(first + h, a.Hq - 1) * a.q_sh, lane);
  RotaryTurn<1, kWave, 1, IL> turn;
  turn.load(a.how, pos, lane);
#pragma unroll
  for (int h = 0; h < kTurned; ++h) norm_and_turn(a.how, rows[h], turn, a.how.q_weight, lane);
#pragma unroll
  for (int h = 0; h < kTurned; ++h)
    if (first + h < a.Hq) store_row<false>(a.how, rows[h], reinterpret_cast<T *>(a.q_out) + ((int64_t)b * a.Hq + first + h) * a.how.D, lane);
}
// A key head's new row, from `in` to the tail's row `out` and, if given, `copy`.  In 64 bits: a key that is held in 8 bits is rounded twice,
// and of a decode step's few rows the arithmetic is not what counts (64 sequences of 8 heads x 128: no difference to be seen).
// `has_page` is asked behind the loads.  False: nothing is written.
template <int DT, bool IL, typename T, typename F>
__device__ __forceinline__ bool turn_key(const RotaryHow &how, const T *in, int pos, T *out, T *copy, int lane, F &&has_page) {
  PairRow<DT, IL> row;
  RotaryTurn<1, kWave, 1, IL> turn;
  row.load(how, in, lane);
  turn.load(how, pos, lane);
  if (!has_page()) return false;
  norm_and_turn<double>(how, row, turn, how.k_weight, lane);
  store_row<false>(how, row, out, lane);
  if (copy) store_row<false>(how, row, copy, lane);
  return true;
}

// A wave takes a few rows of q, into q_out, or the row of a key or value head, into the tail and, where that completes the block, the block
// into its page.  (A few lanes a row, as for the 16-bit cache, and the blocks put one after another by the wave that completed them: 256
// sequences, 64 / 8 heads x 128 22.9 us, so 9.9.)
template <int DT, int CODE, int D>
__global__ __launch_bounds__(kBlock) void kv8_append_kernel(Kv8AppendArgs a) {
  typedef typename Elem<DT>::T T;
  __shared__ __align__(16) T s_row[kBlock / kWave][D];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, H = a.c.H;
  const uint32_t unit = blockIdx.x * (kBlock / kWave) + wave;
  if (unit >= a.units) return;
  const int per = a.parts_q + 2 * H, b = (int)(unit / per);
  int h = (int)(unit - (uint32_t)b * per);
  const int pos = a.lens[b];
  if (h < a.parts_q) {
    if (a.interleaved) turn_queries<DT, true>(a, b, h * kTurned, pos, lane);
    else turn_queries<DT, false>(a, b, h * kTurned, pos, lane);
    return;
  }
  h -= a.parts_q;
  const bool is_v = h >= H;
  h -= is_v ? H : 0;
  const int j = pos >> 4, slot = pos & (kBlk - 1);
  const int blk = kv8_block_in_page(a.c, j);
  int id = -1;
  auto has_page = [&]() {
    id = pos >= 0 ? kv8_page(a.c, b, j) : -1;
    if (id < 0 && !is_v && h == 0 && lane == 0 && a.overflow) atomicAdd(a.overflow, 1);
    return id >= 0;
  };
  const bool full = slot == kBlk - 1;
  const int64_t tail = ((int64_t)b * H + h) * kBlk * D;
  if (!is_v) {
    const T *in = reinterpret_cast<const T *>(a.k) + b * a.k_sb + h * a.k_sh;
    T *kt = reinterpret_cast<T *>(a.c.kt) + tail, *copy = full ? s_row[wave] : nullptr;
    if (!(a.interleaved ? turn_key<DT, true>(a.how, in, pos, kt + slot * D, copy, lane, has_page)
                        : turn_key<DT, false>(a.how, in, pos, kt + slot * D, copy, lane, has_page)) || !full)
      return;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();               // one wave: its LDS accesses are in order
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    typedef KeyBlock<D> K;
    K k;
#pragma unroll
    for (int i = 0; i < K::kEach; ++i) {
      const int r = K::row(i, lane), c = K::channel(i, lane);
      // the new row from LDS: its store to the tail may still be on its way
      k.raw[i] = *reinterpret_cast<const uint4 *>(kt + min(r, kBlk - 2) * D + c);
      if (r == kBlk - 1) k.raw[i] = *reinterpret_cast<const uint4 *>(s_row[wave] + c);
    }
    put_key_block<DT, CODE, D>(k, kv8_k_block(a.c, id, h, blk, D), a.c.ks + kv8_k_scale(a.c, id, h, blk), lane);
  } else {
    typedef ValueBlock<D> V;
    const uint32_t now = load_two<T>(reinterpret_cast<const T *>(a.v) + b * a.v_sb + h * a.v_sh + 2 * V::pair(lane));
    uint16_t *vt = reinterpret_cast<uint16_t *>(a.c.vt) + tail + 2 * V::pair(lane) * kBlk;
    if (!has_page()) return;
    V v;
    if (full) {
      value_rows<D>(reinterpret_cast<const uint16_t *>(a.c.vt) + tail, lane, v.raw);
      if (V::first(lane) + V::kEach == kBlk) v.raw[V::kEach - 1] = now;
    }
    if (V::has(lane) && V::first(lane) == 0) {
      vt[slot] = (uint16_t)now;
      vt[kBlk + slot] = (uint16_t)(now >> 16);
    }
    if (full) put_value_block<DT, CODE, D>(v, kv8_v_block(a.c, id, h, blk, D), a.c.vs + kv8_v_scale(a.c, id, h, blk), lane);
  }
}

// ---- read back -------------------------------------------------------------------------------------------------------------------------

struct Kv8ReadArgs {
  Kv8 c;
  const int32_t *lens, *first;
  int seq_len;
  void *k_out, *v_out;
};

// Grid: blocks that seq_len positions can touch x 2 heads x sequences; a wave a block, its rows written where they fall into the range.
template <int DT, int CODE, int D, bool NT>
__global__ __launch_bounds__(kBlock) void kv8_read_kernel(Kv8ReadArgs a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  const int lane = threadIdx.x % kWave, unit = blockIdx.y * (kBlock / kWave) + threadIdx.x / kWave;
  const int b = blockIdx.z, H = a.c.H;
  if (unit >= 2 * H) return;
  const int first = a.first ? max(a.first[b], 0) : 0;
  const int n = kv8_len(a.c, a.lens, b);
  const int64_t j64 = (int64_t)(first / kBlk) + blockIdx.x;
  const int64_t s0 = j64 * kBlk - first;                         // where the block's first position falls
  if (s0 >= a.seq_len) return;
  const int lo = s0 < 0 ? (int)-s0 : 0, hi = (int)min((int64_t)kBlk, a.seq_len - s0);      // rows lo .. hi - 1 are asked for
  const int there = (int)max((int64_t)0, min((int64_t)kBlk, n - j64 * kBlk));              // rows that are positions
  const int j = (int)min(j64, (int64_t)(INT32_MAX / kBlk));
  const bool is_v = unit >= H;
  const int h = is_v ? unit - H : unit;
  const int id = there > 0 ? kv8_page(a.c, b, j) : -1, blk = kv8_block_in_page(a.c, j);
  const bool codes_there = id >= 0 && there == kBlk, tail_there = id >= 0 && there < kBlk;
  const int64_t tail = ((int64_t)b * H + h) * kBlk * D;
  const int64_t to = (((int64_t)b * H + h) * a.seq_len + s0) * D;
  if (!is_v) {
    typedef KeyBlock<D> K;
    T *out = reinterpret_cast<T *>(a.k_out) + to;
    const float scale = codes_there ? a.c.ks[kv8_k_scale(a.c, id, h, blk)] : 0.f;
#pragma unroll
    for (int i = 0; i < K::kEach; ++i) {
      const int r = K::row(i, lane), c = K::channel(i, lane);
      uint4 w = make_uint4(0, 0, 0, 0);
      if (codes_there) {
        const uint2 codes = *reinterpret_cast<const uint2 *>(kv8_k_block(a.c, id, h, blk, D) + r * D + c);
        Pack<T, 8> p;
        p.v[0] = E::from_float(Codes<CODE>::template value<0>(codes.x) * scale);
        p.v[1] = E::from_float(Codes<CODE>::template value<1>(codes.x) * scale);
        p.v[2] = E::from_float(Codes<CODE>::template value<2>(codes.x) * scale);
        p.v[3] = E::from_float(Codes<CODE>::template value<3>(codes.x) * scale);
        p.v[4] = E::from_float(Codes<CODE>::template value<0>(codes.y) * scale);
        p.v[5] = E::from_float(Codes<CODE>::template value<1>(codes.y) * scale);
        p.v[6] = E::from_float(Codes<CODE>::template value<2>(codes.y) * scale);
        p.v[7] = E::from_float(Codes<CODE>::template value<3>(codes.y) * scale);
        w = __builtin_bit_cast(uint4, p);
      } else if (r < there && tail_there) {
        w = *reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.c.kt) + tail + r * D + c);
      }
      if (K::has(i, lane) && r >= lo && r < hi) store16<NT>(out + (int64_t)r * D + c, w);
    }
  } else {
    typedef ValueBlock<D> V;
    T *out = reinterpret_cast<T *>(a.v_out) + to;
    const int c = V::pair(lane), p0 = V::first(lane);
    uint32_t row[V::kEach];
    if (codes_there) {
      const float scale = a.c.vs[kv8_v_scale(a.c, id, h, blk)];
      const uint8_t *from = kv8_v_block(a.c, id, h, blk, D) + 2 * c * kBlk + p0;
#pragma unroll
      for (int i = 0; i < V::kEach; i += 4) {
        const uint32_t w0 = *reinterpret_cast<const uint32_t *>(from + i), w1 = *reinterpret_cast<const uint32_t *>(from + kBlk + i);
        auto two = [&](float x, float y) { return __builtin_bit_cast(uint32_t, Pack<T, 2>{{E::from_float(x * scale), E::from_float(y * scale)}}); };
        row[i] = two(Codes<CODE>::template value<0>(w0), Codes<CODE>::template value<0>(w1));
        row[i + 1] = two(Codes<CODE>::template value<1>(w0), Codes<CODE>::template value<1>(w1));
        row[i + 2] = two(Codes<CODE>::template value<2>(w0), Codes<CODE>::template value<2>(w1));
        row[i + 3] = two(Codes<CODE>::template value<3>(w0), Codes<CODE>::template value<3>(w1));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V::kEach; ++i) row[i] = 0;
      if (tail_there) {
        value_rows<D>(reinterpret_cast<const uint16_t *>(a.c.vt) + tail, lane, row);
#pragma unroll
        for (int i = 0; i < V::kEach; ++i) row[i] = p0 + i < there ? row[i] : 0u;
      }
    }
#pragma unroll
    for (int i = 0; i < V::kEach; ++i)
      if (V::has(lane) && p0 + i >= lo && p0 + i < hi) {
        uint32_t *to = reinterpret_cast<uint32_t *>(out + (int64_t)(p0 + i) * D + 2 * c);
        if constexpr (NT) __builtin_nontemporal_store(row[i], to);
        else *to = row[i];
      }
  }
}

// Calls f(dtype, code, D) as integral constants.
template <typename F> static void with_kv8_form(const en_kv8_cache *c, F &&f) {
  auto heads = [&](auto dt, auto code) {
    switch (c->size_per_head) {
      case 16: f(dt, code, Int<16>{}); break;
      case 32: f(dt, code, Int<32>{}); break;
      case 48: f(dt, code, Int<48>{}); break;
      case 64: f(dt, code, Int<64>{}); break;
      case 80: f(dt, code, Int<80>{}); break;
      case 96: f(dt, code, Int<96>{}); break;
      case 112: f(dt, code, Int<112>{}); break;
      default: f(dt, code, Int<128>{}); break;
    }
  };
  auto codes = [&](auto dt) {
    if (c->code == EN_KV8_INT8) heads(dt, Int<EN_KV8_INT8>{});
    else heads(dt, Int<EN_KV8_E4M3>{});
  };
  if (c->dtype == EN_F16) codes(Int<EN_F16>{});
  else codes(Int<EN_BF16>{});
}

}  // namespace en

using namespace en;

extern "C" int en_kv8_fill(const void *k, const void *v, const en_kv8_cache *cache, const int32_t *cu_seqlens, int64_t tokens, int max_seq_len,
                           const int64_t *strides, int32_t *overflow, en_stream_t stream) {
  if (const int bad = check_kv8(cache)) return bad;
  if (max_seq_len < 0 || tokens < 0 || cache->batch > 65535) return EN_ERR_SHAPE;
  if (cache->batch == 0 || max_seq_len == 0 || tokens == 0) return EN_OK;
  if (!k || !v || !cu_seqlens || !strides) return EN_ERR_NULL;
  if (!aligned_to(k, 2) || !aligned_to(v, 2)) return EN_ERR_ALIGN;
  const Kv8FillArgs a{kv8_args(cache), k, v, strides[0], strides[1], strides[2], strides[3], cu_seqlens, max_seq_len, tokens, overflow};
  const dim3 grid((unsigned)ceil_div(tokens < max_seq_len ? tokens : max_seq_len, kBlk), (unsigned)ceil_div(2 * (int64_t)cache->head_num, kBlock / kWave),
                  (unsigned)cache->batch);
  if (grid.y > 65535) return EN_ERR_SHAPE;
  with_kv8_form(cache, [&](auto dt, auto code, auto d) {
    constexpr int DT = decltype(dt)::value, CODE = decltype(code)::value, D = decltype(d)::value;
    if (4 * tokens * cache->head_num * D >= kStreamLoadBytes) kv8_fill_kernel<DT, CODE, D, true><<<grid, kBlock, 0, (hipStream_t)stream>>>(a);
    else kv8_fill_kernel<DT, CODE, D, false><<<grid, kBlock, 0, (hipStream_t)stream>>>(a);
  });
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

extern "C" int en_kv8_append(const void *q, const void *k_new, const void *v_new, void *q_out, const en_kv8_cache *cache,
                             const int32_t *kv_lens, int q_heads, const int64_t *strides, const en_norm_rotary *how, int32_t *overflow,
                             en_stream_t stream) {
  if (const int bad = check_kv8(cache)) return bad;
  if (const int bad = check_rotary(how, cache->size_per_head)) return bad;
  if (q_heads < 0) return EN_ERR_SHAPE;
  if (cache->batch == 0) return EN_OK;
  if (!k_new || !v_new || !kv_lens || !strides || (q_heads && (!q || !q_out))) return EN_ERR_NULL;
  for (const void *p : {q, k_new, v_new, (const void *)q_out, how->q_weight, how->k_weight})
    if (!aligned_to(p, 2)) return EN_ERR_ALIGN;
  const int parts_q = (int)ceil_div(q_heads, kTurned);
  const int64_t units = (int64_t)cache->batch * (parts_q + 2 * (int64_t)cache->head_num);
  if (units > INT32_MAX) return EN_ERR_SHAPE;
  const Kv8AppendArgs a{kv8_args(cache), rotary_how(how, cache->size_per_head, 1), q, k_new, v_new, q_out, kv_lens, strides[0], strides[1], strides[2],
                        strides[3], strides[4], strides[5], q_heads, parts_q, how->interleaved != 0, (uint32_t)units, overflow};
  with_kv8_form(cache, [&](auto dt, auto code, auto d) {
    kv8_append_kernel<decltype(dt)::value, decltype(code)::value, decltype(d)::value>
        <<<(unsigned)ceil_div(units, kBlock / kWave), kBlock, 0, (hipStream_t)stream>>>(a);
  });
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

extern "C" int en_kv8_read(const en_kv8_cache *cache, const int32_t *kv_lens, const int32_t *first, int seq_len, void *k_out, void *v_out,
                           en_stream_t stream) {
  if (const int bad = check_kv8(cache)) return bad;
  if (seq_len < 0 || cache->batch > 65535) return EN_ERR_SHAPE;
  if (cache->batch == 0 || seq_len == 0) return EN_OK;
  if (!kv_lens || !k_out || !v_out) return EN_ERR_NULL;
  if (!aligned_to(k_out, 16) || !aligned_to(v_out, 16)) return EN_ERR_ALIGN;
  const Kv8ReadArgs a{kv8_args(cache), kv_lens, first, seq_len, k_out, v_out};
  const dim3 grid((unsigned)(ceil_div(seq_len, kBlk) + (first ? 1 : 0)), (unsigned)ceil_div(2 * (int64_t)cache->head_num, kBlock / kWave),
                  (unsigned)cache->batch);
  if (grid.y > 65535) return EN_ERR_SHAPE;
  with_kv8_form(cache, [&](auto dt, auto code, auto d) {
    constexpr int DT = decltype(dt)::value, CODE = decltype(code)::value, D = decltype(d)::value;
    if (4ll * cache->batch * cache->head_num * seq_len * D >= kStreamStoreBytes) kv8_read_kernel<DT, CODE, D, true><<<grid, kBlock, 0, (hipStream_t)stream>>>(a);
    else kv8_read_kernel<DT, CODE, D, false><<<grid, kBlock, 0, (hipStream_t)stream>>>(a);
  });
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

// Products with weights in 4 bits: y = act(x W^T + b), W[n, k] = (code - zero) * scale with a scale and a zero point per group of channels.
//
// What bounds it for few rows is the stream of the codes, half a byte a weight.  They are laid out once in tiles of 16 rows of W and 128
// channels, 1 KB, so that a wave loads a tile with one 16-byte access a lane: word i of lane l holds channels 32 i + 8 (l / 16) .. + 7 of row
// l % 16, the operand of one 16x16x32 matrix instruction.  In a word, channel c < 4 is the low half of byte c, channel 4 + c its high half.
// A byte of 0 .. 15 is, read as e4m3, that number times 2^-9 (the subnormal numbers and the first binade go in equal steps), so two
// masks and four conversions with a scale of 2^9 make eight 16-bit numbers, exactly.
//
// The products are of codes as they are; a group's sum, in fp32, is then scale * (sum of code x - zero * sum of x), with the sums of x from a
// matrix instruction whose other operand is ones.  No weight is rounded.
#include <type_traits>
#include <utility>

#include "common.hip.h"

namespace en {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

constexpr int kTileRows = 16, kTileCols = 128;
constexpr int64_t kMostFeatures = 1 << 21;      // 256 rows of x stay within 2^30 bytes

template <int DT> __device__ __forceinline__ f32x4 mma(const uint4 &a, const uint4 &b, f32x4 c) {
  if constexpr (DT == EN_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}

// Two codes, bytes 0 and 1 or 2 and 3 of w, as 16-bit numbers.
template <int DT, bool HIGH> __device__ __forceinline__ uint32_t two_codes(uint32_t w) {
  if constexpr (DT == EN_F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 512.f, HIGH));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.f, HIGH));
}
template <int DT> __device__ __forceinline__ uint4 widen(uint32_t w) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = w >> 4 & 0x0f0f0f0fu;
  return make_uint4(two_codes<DT, false>(lo), two_codes<DT, true>(lo), two_codes<DT, false>(hi), two_codes<DT, true>(hi));
}

__device__ __forceinline__ float w4_activate(float v, int act) {
  switch (act) {
    case EN_ACT_RELU: return v < 0.f ? 0.f : v;      // NaN stays NaN
    case EN_ACT_GELU_TANH: return 0.5f * v * (1.f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
    case EN_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.7071067811865476f));
    default: return v;
  }
}

// Four neighbours of a row, `left` of them inside it, at any element's address.
template <typename T> __device__ __forceinline__ void w4_store(T *y, const Pack<T, 4> &v, int left) {
  typedef uint32_t u32x2_by2 __attribute__((ext_vector_type(2), aligned(2)));
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  if (left >= 4) {
    *reinterpret_cast<u32x2_by2 *>(y) = __builtin_bit_cast(u32x2, v);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) y[e] = v.v[e];
  }
}

// ---- layout ----------------------------------------------------------------------------------------------------------------------------

struct PackArgs {
  const uint8_t *codes;
  const uint16_t *scales;
  const uint8_t *zeros;
  uint32_t *codes_out;
  uint16_t *scales_out;
  uint8_t *zeros_out;
  int64_t N, K, groups, steps, per_step;    // per_step: groups of a tile
  int64_t words, scale_count;
};

__global__ __launch_bounds__(kBlock) void w4_pack_kernel(PackArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i < a.words) {
    const int word = (int)(i & 3), lane = (int)(i >> 2 & 63);
    const int64_t tile = i >> 8, step = tile % a.steps, n = tile / a.steps * kTileRows + lane % 16, k = step * kTileCols + word * 32 + lane / 16 * 8;
    uint32_t w = 0;
    if (n < a.N && k < a.K) {
      const uint8_t *p = a.codes + n * (a.K / 2) + k / 2;
      uint32_t c[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[2 * j] = p[j] & 15u;
        c[2 * j + 1] = p[j] >> 4;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= c[j] << (8 * j) | c[4 + j] << (8 * j + 4);
    }
    a.codes_out[i] = w;
  }
  if (i < a.scale_count) {
    // of a tile: its groups, row by row
    const int64_t tile = i / (16 * a.per_step), in = i % (16 * a.per_step), group = tile % a.steps * a.per_step + in % a.per_step, n = tile / a.steps * kTileRows + in / a.per_step;
    const bool there = n < a.N && group < a.groups;
    a.scales_out[i] = there ? a.scales[n * a.groups + group] : 0;
    if (a.zeros) a.zeros_out[i] = there ? a.zeros[n * a.groups + group] & 15 : 0;
  }
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------------

struct W4Args {
  const void *x;
  int64_t x_stride;
  int R, N, K, steps, tiles;      // steps of 128 channels, tiles of 16 rows of W
  const uint4 *codes;
  const void *scales;
  const uint8_t *zeros;
  const void *bias;
  int act;
  void *y;
};

// The NW waves of a workgroup share the channels of CT tiles of W and 16 RT rows of x.
template <int DT, int GROUP, int RT, int CT, int NW>
__global__ __launch_bounds__(NW *kWave) void w4_rows_kernel(W4Args a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  constexpr int kGroups = kTileCols / GROUP, kPer = GROUP / 32;       // groups of a step, matrix instructions of a group
  __shared__ __align__(16) float s_acc[NW][RT * CT][kWave][4];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, j = lane % 16, g = lane / 16;
  const int t0 = blockIdx.x * CT, r0 = blockIdx.y * 16 * RT;
  // rows past R and channels past K arrive as zeros
  const T *x0 = reinterpret_cast<const T *>(a.x) + r0 * a.x_stride;
  const int rows = min(16 * RT, a.R - r0);
  const rsrc_t x_rsrc = make_rsrc(x0, (uint32_t)(((rows - 1) * a.x_stride + a.K) * 2));
  uint32_t xrow[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) xrow[t] = t * 16 + j < rows ? (uint32_t)((t * 16 + j) * a.x_stride * 2) : kOutOfRange;
  const uint32_t one = DT == EN_F16 ? 0x3c003c00u : 0x3f803f80u;
  const uint4 ones = make_uint4(one, one, one, one);

  f32x4 acc[RT][CT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int step = wave; step < a.steps; step += NW) {
    uint4 w[CT], x[RT][4];
    Pack<T, 4 * kGroups> sc[CT];
    Pack<uint8_t, 4 * kGroups> ze[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int64_t tile = min(t0 + c, a.tiles - 1);
      w[c] = a.codes[(tile * a.steps + step) * kWave + lane];
      const int64_t at = ((tile * a.steps + step) * 16 + 4 * g) * kGroups;
      sc[c] = load_pack<T, 4 * kGroups>(reinterpret_cast<const T *>(a.scales) + at);
      if (a.zeros) ze[c] = load_pack<uint8_t, 4 * kGroups>(a.zeros + at);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = step * kTileCols + i * 32 + g * 8;
        x[t][i] = buffer_load16(x_rsrc, xrow[t] + (uint32_t)k * 2u | xrow[t] & kOutOfRange | (k < a.K ? 0u : kOutOfRange));
      }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      f32x4 sum[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kPer; ++k) sum[t] = mma<DT>(ones, x[t][i * kPer + k], sum[t]);
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        uint4 wide[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) wide[k] = widen<DT>((&w[c].x)[i * kPer + k]);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < kPer; ++k) p = mma<DT>(wide[k], x[t][i * kPer + k], p);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[t][c][e] += E::to_float(sc[c].v[e * kGroups + i]) * (p[e] - (a.zeros ? (float)ze[c].v[e * kGroups + i] : 8.f) * sum[t][e]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4 *>(s_acc[wave][t * CT + c][lane]) = acc[t][c];
  __syncthreads();
  // lane (j, g) has rows 4g .. 4g + 3 of W, which are neighbours in y, of row j of x
  for (int tc = wave; tc < RT * CT; tc += NW) {
    const int t = tc / CT, c = tc % CT, r = r0 + t * 16 + j, n = (t0 + c) * kTileRows + 4 * g;
    if (r >= a.R || n >= a.N) continue;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NW; ++k) v += *reinterpret_cast<const f32x4 *>(s_acc[k][tc][lane]);
    Pack<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float bias = a.bias && n + e < a.N ? E::to_float(reinterpret_cast<const T *>(a.bias)[n + e]) : 0.f;
      y.v[e] = E::from_float(w4_activate(v[e] + bias, a.act));
    }
    w4_store(reinterpret_cast<T *>(a.y) + (int64_t)r * a.N + n, y, a.N - n);
  }
}

// ---- many rows ---------------------------------------------------------------------------------------------------------------------------

// 256 rows of x times 256 rows of W a workgroup, 64 channels a stage; eight waves, 128 x 64 each.  Bound by the matrix instructions: x goes
// from memory into LDS as operands lie (a wave's load of 16 rows x 32 channels is one operand, 1 KB in lane order), and so do the
// weights, each turned into 16 bits once for the 256 rows: (code - zero) * scale in fp32, rounded as a weight kept in 16 bits would be
// (half a step of the activations' type; scaling sums of codes instead takes four multiplications for each four matrix instructions of a
// group of 32, as many cycles as those themselves).
constexpr int kManyRows = 256, kManyCols = 256, kManyWaves = 8;

template <int DT> __device__ __forceinline__ uint32_t pack_two(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_two<EN_F16>(float lo, float hi) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)lo, (_Float16)hi});
}
template <> __device__ __forceinline__ uint32_t pack_two<EN_BF16>(float lo, float hi) {
  typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, b16x2{(__bf16)lo, (__bf16)hi});
}
template <typename F, int... I> __device__ __forceinline__ void each(F &&f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }

// Codes 2 I and 2 I + 1 of a word times scale plus off.
template <int DT, int I> __device__ __forceinline__ uint32_t scaled_two(uint32_t w, float scale, float off) {
  const uint32_t b = I < 2 ? w & 0x0f0f0f0fu : w >> 4 & 0x0f0f0f0fu;
  constexpr int kShift = I % 2 * 16;
  return pack_two<DT>((float)(b >> kShift & 0xffu) * scale + off, (float)(b >> (kShift + 8) & 0xffu) * scale + off);
}

template <int DT, int GROUP>
__global__ __launch_bounds__(kManyWaves *kWave, 2) void w4_many_kernel(W4Args a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  constexpr int kGroups = kTileCols / GROUP, RT = 8, CT = 4;
  constexpr int kXStage = kManyRows * 64 * 2, kWStage = kManyCols * 64 * 2, kW = 3 * kXStage;
  __shared__ __align__(16) char s_mem[3 * kXStage + 2 * kWStage];      // x operands [row tile][half][lane] of three stages, W operands [tile][half][lane] of two
  const int lane = threadIdx.x % kWave, j = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wr = wave % 2, wc = wave / 2;
  // a column block's row blocks one after another: they read the same codes
  const int row_blocks = (a.R + kManyRows - 1) / kManyRows;
  const int rb = blockIdx.x % row_blocks, cb = blockIdx.x / row_blocks;
  const int r0 = rb * kManyRows, t0 = cb * (kManyCols / kTileRows);

  // x: this wave moves row tiles 2 wave, 2 wave + 1; channels past K and rows past R arrive as zeros
  const T *x0 = reinterpret_cast<const T *>(a.x) + (int64_t)r0 * a.x_stride;
  const int rows = min(kManyRows, a.R - r0);
  const uint32_t x_bytes = (uint32_t)(((int64_t)(rows - 1) * a.x_stride + a.K) * 2);
  const desc_t x_desc = make_desc(x0, x_bytes);
  uint32_t xrow[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = (2 * wave + t) * 16 + j;
    xrow[t] = r < rows ? (uint32_t)((int64_t)r * a.x_stride * 2) : kOutOfRange;
  }
  const uint32_t lds0 = lds_address(s_mem);
  auto load_x = [&](int stage, int buf) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = stage * 64 + half * 32 + g * 8;
        buffer_load16_to_lds(x_desc, lds0 + buf * kXStage + ((2 * wave + t) * 2 + half) * 1024,
                             (xrow[t] + (uint32_t)k * 2u) | (xrow[t] & kOutOfRange) | (k < a.K ? 0u : kOutOfRange));
      }
  };
  // W: this wave turns tiles 2 wave, 2 wave + 1 into 16 bits; a lane's row of W is l % 16
  uint4 codes[2], next_codes[2];
  Pack<T, kGroups> sc[2], next_sc[2];
  Pack<uint8_t, kGroups> ze[2], next_ze[2];
  rsrc_t code_rsrc[2], scale_rsrc[2], zero_rsrc[2];      // of a row of tiles
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int64_t tile = (int64_t)min(t0 + 2 * wave + t, a.tiles - 1) * a.steps;
    code_rsrc[t] = make_rsrc(a.codes + tile * kWave, a.steps * 1024);
    scale_rsrc[t] = make_rsrc(reinterpret_cast<const T *>(a.scales) + tile * 16 * kGroups, a.steps * 32 * kGroups);
    zero_rsrc[t] = make_rsrc(a.zeros + tile * 16 * kGroups, a.zeros ? a.steps * 16 * kGroups : 0);
  }
  auto load_codes = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) next_codes[t] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(code_rsrc[t], lane * 16, step * 1024, 0));
  };
  auto load_scales = [&](int step) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (kGroups == 4) {
        next_sc[t] = __builtin_bit_cast(Pack<T, 4>, __builtin_amdgcn_raw_buffer_load_b64(scale_rsrc[t], j * 8, step * 128, 0));
        next_ze[t] = __builtin_bit_cast(Pack<uint8_t, 4>, __builtin_amdgcn_raw_buffer_load_b32(zero_rsrc[t], j * 4, step * 64, 0));
      } else if constexpr (kGroups == 2) {
        next_sc[t] = __builtin_bit_cast(Pack<T, 2>, __builtin_amdgcn_raw_buffer_load_b32(scale_rsrc[t], j * 4, step * 64, 0));
        next_ze[t] = __builtin_bit_cast(Pack<uint8_t, 2>, __builtin_amdgcn_raw_buffer_load_b16(zero_rsrc[t], j * 2, step * 32, 0));
      } else {
        next_sc[t].v[0] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(scale_rsrc[t], j * 2, step * 32, 0));
        next_ze[t].v[0] = __builtin_amdgcn_raw_buffer_load_b8(zero_rsrc[t], j, step * 16, 0);
      }
    }
  };
  auto take_codes = [&] {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      codes[t] = next_codes[t];
      sc[t] = next_sc[t];
      ze[t] = next_ze[t];
    }
  };
  // Sixteen pieces of the weights of half a step: two codes a lane of operand piece / 4, which goes to LDS with its fourth.
  uint32_t piece4[4];
  float scale = 0.f, off = 0.f;
  auto put_w = [&](auto piece, int part, int buf) {
    constexpr int P = decltype(piece)::value, t = P / 8, half = P / 4 % 2;
    const int word = 2 * part + half, i = word * 32 / GROUP;
    const uint32_t w = word == 0 ? codes[t].x : word == 1 ? codes[t].y : word == 2 ? codes[t].z : codes[t].w;
    if constexpr (P % 4 == 0) {
      scale = E::to_float(sc[t].v[i]);
      off = -(a.zeros ? (float)ze[t].v[i] : 8.f) * scale;
      asm volatile("" : "+v"(scale), "+v"(off));         // here, not all operands' at once: sixteen registers more
    }
    piece4[P % 4] = scaled_two<DT, P % 4>(w, scale, off);
    if constexpr (P % 4 == 3)
      *reinterpret_cast<uint4 *>(s_mem + kW + buf * kWStage + ((2 * wave + t) * 2 + half) * 1024 + lane * 16) =
          make_uint4(piece4[0], piece4[1], piece4[2], piece4[3]);
  };
  auto put_all = [&](int part, int buf) {
    each([&](auto piece) { put_w(piece, part, buf); }, std::make_integer_sequence<int, 16>{});
  };

  f32x4 acc[RT][CT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  // A stage's products, and between them, while the matrix instructions run, the pieces of the next stage's weights.
  auto multiply = [&](int xbuf, int buf, auto more, int part) {
    const char *xs = s_mem + xbuf * kXStage + wr * RT * 2048 + lane * 16, *ws = s_mem + kW + buf * kWStage + wc * CT * 2048 + lane * 16;
    uint4 w[CT], x[2];
#pragma unroll
    for (int c = 0; c < CT; ++c) w[c] = *reinterpret_cast<const uint4 *>(ws + c * 2048);
    x[0] = *reinterpret_cast<const uint4 *>(xs);
    auto one = [&](auto index) {
      constexpr int I = decltype(index)::value, t = I % RT, half = I / RT;
      if constexpr (I + 1 < 2 * RT) x[(I + 1) % 2] = *reinterpret_cast<const uint4 *>(xs + (I + 1) % RT * 2048 + (I + 1) / RT * 1024);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        acc[t][c] = mma<DT>(w[c], x[I % 2], acc[t][c]);
        if constexpr (half == 0 && t == RT - 1) w[c] = *reinterpret_cast<const uint4 *>(ws + c * 2048 + 1024);
      }
      if constexpr (more.value) put_w(index, part, buf ^ 1);
      __builtin_amdgcn_sched_barrier(0);
    };
    each(one, std::make_integer_sequence<int, 2 * RT>{});
  };
  // All loads have arrived, those into LDS among them (as an instruction that the compiler counts with: it adds no wait of its own).
  auto arrived = [] {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __builtin_amdgcn_sched_barrier(0);
  };

  // Stage s has the first half of step s / 2 or the second.  In its first stage a step sends for x two stages ahead and waits for what was
  // sent before; in its second also for the codes of the step after next.  So x has one or two stages to arrive, codes have two.
  load_codes(0);
  load_scales(0);
  load_x(0, 0);
  load_x(1, 1);
  arrived();
  take_codes();
  load_codes(min(1, a.steps - 1));
  put_all(0, 0);
  lds_barrier();
  int xbuf = 0;                               // of the step's first stage
  auto ring = [](int b) { return b >= 3 ? b - 3 : b; };
  for (int step = 0; step + 1 < a.steps; ++step) {
    load_scales(step + 1);
    load_x(2 * step + 2, ring(xbuf + 2));
    multiply(xbuf, 0, std::true_type{}, 1);
    arrived();
    lds_barrier();
    take_codes();
    load_codes(min(step + 2, a.steps - 1));
    load_x(2 * step + 3, xbuf);
    multiply(ring(xbuf + 1), 1, std::true_type{}, 0);
    lds_barrier();
    xbuf = ring(xbuf + 2);
  }
  multiply(xbuf, 0, std::true_type{}, 1);
  arrived();
  lds_barrier();
  multiply(ring(xbuf + 1), 1, std::false_type{}, 0);
  auto finish = [&](auto act) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int n = (t0 + wc * CT + c) * kTileRows + 4 * g, left = a.N - n;
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = a.bias && e < left ? E::to_float(reinterpret_cast<const T *>(a.bias)[n + e]) : 0.f;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int r = r0 + (wr * RT + t) * 16 + j;
        Pack<T, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.v[e] = E::from_float(w4_activate(acc[t][c][e] + bias[e], act.value));
        if (r < a.R) w4_store(reinterpret_cast<T *>(a.y) + (int64_t)r * a.N + n, y, left);
      }
    }
  };
  switch (a.act) {
    case EN_ACT_RELU: finish(std::integral_constant<int, EN_ACT_RELU>{}); break;
    case EN_ACT_GELU_TANH: finish(std::integral_constant<int, EN_ACT_GELU_TANH>{}); break;
    case EN_ACT_GELU: finish(std::integral_constant<int, EN_ACT_GELU>{}); break;
    default: finish(std::integral_constant<int, EN_ACT_NONE>{});
  }
}

static int check_w4(const en_w4_weight *w) {
  if (!w) return EN_ERR_NULL;
  if (w->dtype != EN_F16 && w->dtype != EN_BF16) return EN_ERR_DTYPE;
  if (w->group != 32 && w->group != 64 && w->group != 128) return EN_ERR_UNSUPPORTED;
  if (w->out_features < 1 || w->in_features < 8 || w->in_features % 8 || w->out_features > kMostFeatures || w->in_features > kMostFeatures) return EN_ERR_SHAPE;
  if (!w->codes || !w->scales) return EN_ERR_NULL;
  if (!aligned_to(w->codes, 16) || !aligned_to(w->scales, 16) || !aligned_to(w->zeros, 16)) return EN_ERR_ALIGN;
  return EN_OK;
}

}  // namespace en

using namespace en;

extern "C" {

int64_t en_w4_codes_bytes(int64_t out_features, int64_t in_features) {
  if (out_features < 1 || in_features < 1) return 0;
  return ceil_div(out_features, kTileRows) * ceil_div(in_features, kTileCols) * (kTileRows * kTileCols / 2);
}

int64_t en_w4_groups(int64_t out_features, int64_t in_features, int group) {
  if (out_features < 1 || in_features < 1 || (group != 32 && group != 64 && group != 128)) return 0;
  return ceil_div(out_features, kTileRows) * ceil_div(in_features, kTileCols) * (kTileRows * kTileCols / group);
}

int en_w4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, const en_w4_weight *weight, en_stream_t stream) {
  if (const int bad = check_w4(weight)) return bad;
  if (!codes || !scales || (zeros != nullptr) != (weight->zeros != nullptr)) return EN_ERR_NULL;
  if (!aligned_to(scales, 2)) return EN_ERR_ALIGN;
  PackArgs a{codes, (const uint16_t *)scales, zeros, (uint32_t *)weight->codes, (uint16_t *)weight->scales, (uint8_t *)weight->zeros,
             weight->out_features, weight->in_features, ceil_div(weight->in_features, weight->group), ceil_div(weight->in_features, kTileCols), 0, 0, 0};
  a.per_step = kTileCols / weight->group;
  a.words = en_w4_codes_bytes(a.N, a.K) / 4;
  a.scale_count = en_w4_groups(a.N, a.K, weight->group);
  const int64_t blocks = ceil_div(a.words > a.scale_count ? a.words : a.scale_count, kBlock);
  if (blocks > INT32_MAX) return EN_ERR_SHAPE;
  w4_pack_kernel<<<(unsigned)blocks, kBlock, 0, (hipStream_t)stream>>>(a);
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

int en_linear_w4(const void *x, int64_t rows, int64_t x_stride, const en_w4_weight *weight, const void *bias, int activation, void *y,
                 en_stream_t stream) {
  if (const int bad = check_w4(weight)) return bad;
  const int64_t N = weight->out_features, K = weight->in_features;
  if (activation < EN_ACT_NONE || activation > EN_ACT_GELU) return EN_ERR_UNSUPPORTED;
  if (rows < 0 || rows > (1 << 20) || x_stride < 0 || (rows > 1 && x_stride < K) || x_stride > kMostFeatures) return EN_ERR_SHAPE;
  if (rows == 0) return EN_OK;
  if (!x || !y) return EN_ERR_NULL;
  if (!aligned_to(x, 16) || x_stride % 8 || !aligned_to(y, 2) || !aligned_to(bias, 2)) return EN_ERR_ALIGN;
  W4Args a{x, x_stride, (int)rows, (int)N, (int)K, (int)ceil_div(K, kTileCols), (int)ceil_div(N, kTileRows), (const uint4 *)weight->codes,
           weight->scales, (const uint8_t *)weight->zeros, bias, activation, y};
  const hipStream_t s = (hipStream_t)stream;
  auto launch = [&](auto dt, auto group, auto rt) {
    constexpr int RT = decltype(rt)::value, CT = 1, NW = 8;
    const dim3 grid((unsigned)ceil_div(a.tiles, CT), (unsigned)ceil_div(rows, 16 * RT));
    w4_rows_kernel<decltype(dt)::value, decltype(group)::value, RT, CT, NW><<<grid, NW * kWave, 0, s>>>(a);
  };
  auto many = [&](auto dt, auto group) {
    const int64_t blocks = ceil_div(rows, kManyRows) * ceil_div(N, kManyCols);
    w4_many_kernel<decltype(dt)::value, decltype(group)::value><<<(unsigned)blocks, kManyWaves * kWave, 0, s>>>(a);
  };
  auto shape = [&](auto dt, auto group) {
    if (rows > 128) return many(dt, group);
    if (rows <= 16) launch(dt, group, std::integral_constant<int, 1>{});
    else if (rows <= 32) launch(dt, group, std::integral_constant<int, 2>{});
    else launch(dt, group, std::integral_constant<int, 4>{});
  };
  auto groups = [&](auto dt) {
    if (weight->group == 32) shape(dt, std::integral_constant<int, 32>{});
    else if (weight->group == 64) shape(dt, std::integral_constant<int, 64>{});
    else shape(dt, std::integral_constant<int, 128>{});
  };
  if (weight->dtype == EN_F16) groups(std::integral_constant<int, EN_F16>{});
  else groups(std::integral_constant<int, EN_BF16>{});
  EN_RETURN_IF_LAUNCH_FAILED();
  return EN_OK;
}

}  // extern "C"

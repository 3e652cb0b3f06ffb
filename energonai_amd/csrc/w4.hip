// Products with weights in 4 bits: y = act(x W^T + b), W[n, k] = (code - zero) * scale with a scale and a zero point per group of channels.
//
// What bounds it for few rows is the stream of the codes, half a byte a weight.  They are laid out once in tiles of 16 rows of W and 128
// channels, 1 KB, so that a wave loads a tile with one 16-byte access a lane: word i of lane l holds channels 32 i + 8 (l / 16) .. + 7 of row
// l % 16, the operand of one 16x16x32 matrix instruction.  In a word, channel c < 4 is the low half of byte c, channel 4 + c its high half.
// A byte of 0 .. 15 is, read as e4m3, that number times 2^-9 (the subnormal numbers and the first binade go in equal steps), so two
// masks and four conversions with a scale of 2^9 make eight 16-bit numbers, exactly.
//
// Up to 64 rows the products are of codes as they are; a group's sum, in fp32, is then scale * (sum of code x - zero * sum of x), with the
// sums of x from a matrix instruction whose other operand is ones, and no weight is rounded.  For more rows, whose products are bound by the
// matrix instructions, weights are turned into 16 bits once for all rows of a workgroup (below).
//
// us, groups of 128, bf16, weights that no cache holds: 1 x 9216 -> 9216 16 (44 MB, 2.7 TB/s), 1 x 7168 -> 28672 25 (106 MB, 4.3 TB/s), 40 x 9216 ->
// 9216 26; 1000 x 9216 -> 9216 218 (0.78 PFLOP/s), 512 rows of the same 171 (0.51 PFLOP/s: 288 tiles on 256 compute units).
#include <type_traits>
#include <utility>

#include "common.hip.h"

namespace en {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

constexpr int kTileRows = 16, kTileCols = 128;
constexpr int kManyRows = 256, kManyCols = 256, kManyWaves = 8;
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
    if (a.zeros) a.zeros_out[i] = there ? a.zeros[n * a.groups + group] : 0;
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
  int per;                        // steps of a run
  float *part;                    // [runs][R][16 tiles] sums, or null
};

// Loads of `count` tiles of W that follow `tile`: codes, scales and zero points of a lane for matrix operands (all groups of four rows of W), by
// step.
template <typename T, int GROUPS> struct W4Tiles {
  rsrc_t codes, scales, zeros;
  __device__ __forceinline__ W4Tiles(const W4Args &a, int tile, int count) {
    const int64_t first = (int64_t)tile * a.steps;
    const uint32_t steps = count * a.steps;
    codes = make_rsrc(a.codes + first * kWave, steps * 1024);
    scales = make_rsrc(reinterpret_cast<const T *>(a.scales) + first * 16 * GROUPS, steps * 32 * GROUPS);
    zeros = make_rsrc(a.zeros + first * 16 * GROUPS, a.zeros ? steps * 16 * GROUPS : 0);
  }
};
// `base` is the same for the whole wave.
template <int BYTES, int AUX> __device__ __forceinline__ Pack<uint8_t, BYTES> w4_load(rsrc_t r, uint32_t at, uint32_t base = 0) {
  if constexpr (BYTES == 32) {
    Pack<uint8_t, 32> both;
    const uint4 lo = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, (int)base, AUX)),
                hi = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at + 16, (int)base, AUX));
    __builtin_memcpy(&both, &lo, 16);
    __builtin_memcpy(both.v + 16, &hi, 16);
    return both;
  } else if constexpr (BYTES == 16) return __builtin_bit_cast(Pack<uint8_t, 16>, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, (int)base, AUX));
  else if constexpr (BYTES == 8) return __builtin_bit_cast(Pack<uint8_t, 8>, __builtin_amdgcn_raw_buffer_load_b64(r, (int)at, (int)base, AUX));
  else if constexpr (BYTES == 4) return __builtin_bit_cast(Pack<uint8_t, 4>, __builtin_amdgcn_raw_buffer_load_b32(r, (int)at, (int)base, AUX));
  else if constexpr (BYTES == 2) return __builtin_bit_cast(Pack<uint8_t, 2>, __builtin_amdgcn_raw_buffer_load_b16(r, (int)at, (int)base, AUX));
  else return Pack<uint8_t, 1>{{__builtin_amdgcn_raw_buffer_load_b8(r, (int)at, (int)base, AUX)}};
}

// Sixteen rows of x by 32 channels, one matrix operand: lane l loads vector `operand_vector` of row l / 4, so that four neighbours read 64
// bytes of a row (a lane its own operand's 16 bytes, rows in turn, takes four times the accesses of the first-level cache: 40 x 9216 -> 9216 30 us, so 26), and the vectors
// lie in LDS in the lanes' order; a lane's operand, row l % 16 and vector l / 16, is at `operand_slot`.  Vectors go round by one every four
// rows, so that 16 lanes that read one vector of 16 rows meet all banks.
__device__ __forceinline__ int operand_vector(int lane) { return (lane + lane / 16) % 4; }
__device__ __forceinline__ int operand_slot(int lane) { return lane % 16 * 4 + (lane / 16 + 4 - lane % 16 / 4) % 4; }

// The NW waves of a workgroup share the channels of CT tiles of W and 16 RT rows of x, a step of 128 channels each in turn, and their sums
// meet in LDS in the end.  x goes through a wave's own part of LDS (see operand_vector); DIRECT: into registers as operands lie, for
// rows that are so few that most lanes of an operand load nothing.  The next step's x is on its way while this one is multiplied; its codes
// are asked for after that, which leaves the registers to a second wave a SIMD (codes ahead as well: 40 x 9216 -> 9216 26 -> 34 us).  With
// 64 rows two waves a SIMD are worth 20 registers in scratch (64 x 9216 -> 9216 42.1 -> 36.7 us; groups of 64 spill twice as many, 47 -> 56).
template <int DT, int GROUP, int RT, int CT, int NW, bool DIRECT>
__global__ __launch_bounds__(NW *kWave, RT == 4 && GROUP == 128 ? 2 : 1) void w4_rows_kernel(W4Args a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  constexpr int kGroups = kTileCols / GROUP, kPer = GROUP / 32;       // groups of a step, matrix instructions of a group
  constexpr int kAtOnce = CT < 4 ? CT : GROUP > 32 && RT == 1 ? 4 : GROUP > 32 || RT < 3 ? 2 : 1;      // tiles of W whose sums are under way
  constexpr int kMeet = CT < 4 ? CT : 4;                              // tiles of W whose sums meet in LDS at once
  constexpr int kWords = CT < 4 && RT > 1 ? 2 : 4;                    // operands of a step that are in LDS at once
  constexpr int kSlots = RT * (kMeet > kWords || DIRECT ? kMeet : kWords);
  __shared__ __align__(16) float s_mem[NW][kSlots][kWave][4];         // a wave's own: operands of x, in the end its sums
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), j = lane % 16, g = lane / 16;
  const int t0 = blockIdx.x * CT, r0 = blockIdx.y * 16 * RT;
  // rows past R and channels past K arrive as zeros
  const T *x0 = reinterpret_cast<const T *>(a.x) + r0 * a.x_stride;
  const int rows = min(16 * RT, a.R - r0);
  const rsrc_t x_rsrc = make_rsrc(x0, (uint32_t)(((rows - 1) * a.x_stride + a.K) * 2));
  uint32_t xrow[RT];
  const int x_row = DIRECT ? j : lane / 4, x_vector = DIRECT ? g : operand_vector(lane);
#pragma unroll
  for (int t = 0; t < RT; ++t) xrow[t] = t * 16 + x_row < rows ? (uint32_t)((t * 16 + x_row) * a.x_stride * 2) + x_vector * 16 : kOutOfRange;
  const uint32_t one = DT == EN_F16 ? 0x3c003c00u : 0x3f803f80u;
  const uint4 ones = make_uint4(one, one, one, one);
  typedef W4Tiles<T, kGroups> Tiles;
  const int begin = blockIdx.z * a.per, end = min(begin + a.per, a.steps), channels = min(a.K, end * kTileCols);
  const int last = min(CT, a.tiles - t0) - 1;  // tiles past the last one are the last one, and not stored
  const Tiles tile(a, t0, last + 1);

  uint4 w[CT], x[RT][4];
  Pack<T, 4 * kGroups> sc[CT];
  Pack<uint8_t, 4 * kGroups> ze[CT];
  auto fetch_w = [&](int step) {
    const uint32_t none = step < end ? 0u : kOutOfRange;      // nothing is read past the run
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const uint32_t from = min(c, last) * a.steps;
      w[c] = __builtin_bit_cast(uint4, w4_load<16, 2>(tile.codes, (step * kWave + lane) * 16 | none, from * 1024));
      sc[c] = __builtin_bit_cast(Pack<T, 4 * kGroups>, w4_load<8 * kGroups, 0>(tile.scales, (step * 4 + g) * 8 * kGroups | none, from * 32 * kGroups));
      ze[c] = w4_load<4 * kGroups, 0>(tile.zeros, (step * 4 + g) * 4 * kGroups | none, from * 16 * kGroups);
    }
  };
  auto fetch_x = [&](int step) {
    const int left = channels - step * kTileCols - x_vector * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < RT; ++t)
        x[t][i] = buffer_load16(x_rsrc, (xrow[t] + (uint32_t)(step * 256 + i * 64)) | (xrow[t] & kOutOfRange) | (i * 32 < left ? 0u : kOutOfRange));
  };
  auto own_lds = [] {                          // one wave: its LDS accesses are in order
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  auto put_x = [&](int from) {
    own_lds();
#pragma unroll
    for (int i = 0; i < kWords; ++i)
#pragma unroll
      for (int t = 0; t < RT; ++t) *reinterpret_cast<uint4 *>(s_mem[wave][t * kWords + i][lane]) = x[t][from + i];
    own_lds();
  };

  f32x4 acc[RT][CT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  fetch_x(begin + wave);
  fetch_w(begin + wave);
  const int slot = operand_slot(lane);
  for (int step = begin + wave; step < end; step += NW) {
    if constexpr (!DIRECT) {
      put_x(0);
      if (kWords == 4) fetch_x(step + NW);
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      // products of independent sums follow one another: each waits for the one before it of its own
      uint4 operand[RT][kPer];
      f32x4 sum[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c0 = 0; c0 < CT; c0 += kAtOnce) {
        f32x4 p[kAtOnce][RT];
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c)
#pragma unroll
          for (int t = 0; t < RT; ++t) p[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const int word = i * kPer + k;
          if (c0 == 0) {
            if (!DIRECT && kWords < 4 && word == kWords) {
              put_x(kWords);
              fetch_x(step + NW);
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              operand[t][k] = DIRECT ? x[t][word] : *reinterpret_cast<const uint4 *>(s_mem[wave][t * kWords + word % kWords][slot]);
              sum[t] = mma<DT>(ones, operand[t][k], sum[t]);
            }
          }
#pragma unroll
          for (int c = 0; c < kAtOnce; ++c) {
            const uint4 all = w[c0 + c], wide = widen<DT>(word == 0 ? all.x : word == 1 ? all.y : word == 2 ? all.z : all.w);
#pragma unroll
            for (int t = 0; t < RT; ++t) p[c][t] = mma<DT>(wide, operand[t][k], p[c][t]);
          }
        }
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float scale = E::to_float(sc[c0 + c].v[e * kGroups + i]), zero = a.zeros ? (float)ze[c0 + c].v[e * kGroups + i] : 8.f;
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t][c0 + c][e] += scale * (p[c][t][e] - zero * sum[t][e]);
          }
        if constexpr (GROUP == 32) __builtin_amdgcn_sched_barrier(0);      // a group's scales at a time in fp32
      }
    }
    if constexpr (DIRECT) fetch_x(step + NW);
    fetch_w(step + NW);
  }
#pragma unroll
  for (int c0 = 0; c0 < CT; c0 += kMeet) {
    if (c0 > 0) __syncthreads();               // those before have been read
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int c = 0; c < kMeet; ++c) *reinterpret_cast<f32x4 *>(s_mem[wave][t * kMeet + c][lane]) = acc[t][c0 + c];
    __syncthreads();
    // lane (j, g) has rows 4g .. 4g + 3 of W, which are neighbours in y, of row j of x
    for (int tc = wave; tc < RT * kMeet; tc += NW) {
      const int t = tc / kMeet, c = c0 + tc % kMeet, r = r0 + t * 16 + j, n = (t0 + c) * kTileRows + 4 * g;
      if (r >= a.R || n >= a.N) continue;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NW; ++k) v += *reinterpret_cast<const f32x4 *>(s_mem[k][tc][lane]);
      if (a.part) {
        *reinterpret_cast<f32x4 *>(a.part + ((int64_t)blockIdx.z * a.R + r) * (a.tiles * kTileRows) + n) = v;
        continue;
      }
      Pack<T, 4> y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float bias = a.bias && n + e < a.N ? E::to_float(reinterpret_cast<const T *>(a.bias)[n + e]) : 0.f;
        y.v[e] = E::from_float(w4_activate(v[e] + bias, a.act));
      }
      w4_store(reinterpret_cast<T *>(a.y) + (int64_t)r * a.N + n, y, a.N - n);
    }
  }
}

// The sums of the runs of steps, four neighbours of a row a lane.
template <int DT> __global__ __launch_bounds__(kBlock) void w4_join_kernel(W4Args a, int splits) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  const int n = (blockIdx.x * kBlock + threadIdx.x) * 4, r = blockIdx.y, pitch = a.tiles * kTileRows;
  if (n >= a.N) return;
  const float *p = a.part + (int64_t)r * pitch + n;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4 *>(p + (int64_t)s * a.R * pitch);
  Pack<T, 4> y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float bias = a.bias && n + e < a.N ? E::to_float(reinterpret_cast<const T *>(a.bias)[n + e]) : 0.f;
    y.v[e] = E::from_float(w4_activate(v[e] + bias, a.act));
  }
  w4_store(reinterpret_cast<T *>(a.y) + (int64_t)r * a.N + n, y, a.N - n);
}

// ---- more rows ---------------------------------------------------------------------------------------------------------------------------

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
  uint32_t b = I < 2 ? w & 0x0f0f0f0fu : w >> 4 & 0x0f0f0f0fu;
  asm("" : "+v"(b));             // bytes of a word, which a conversion takes by itself
  constexpr int kShift = I % 2 * 16;
  return pack_two<DT>((float)(b >> kShift & 0xffu) * scale + off, (float)(b >> (kShift + 8) & 0xffu) * scale + off);
}

// Bias, activation and the store of a wave's tiles.
template <int DT, int RT, int CT> __device__ __forceinline__ void w4_finish(const W4Args &a, const f32x4 (&acc)[RT][CT], int r0, int t0) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  const int lane = threadIdx.x % kWave, j = lane % 16, g = lane / 16;
  auto with = [&](auto act) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int n = (t0 + c) * kTileRows + 4 * g, left = a.N - n;
      float bias[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = a.bias && e < left ? E::to_float(reinterpret_cast<const T *>(a.bias)[n + e]) : 0.f;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int r = r0 + t * 16 + j;
        Pack<T, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.v[e] = E::from_float(w4_activate(acc[t][c][e] + bias[e], act.value));
        if (r < a.R) w4_store(reinterpret_cast<T *>(a.y) + (int64_t)r * a.N + n, y, left);
      }
    }
  };
  switch (a.act) {
    case EN_ACT_RELU: with(std::integral_constant<int, EN_ACT_RELU>{}); break;
    case EN_ACT_GELU_TANH: with(std::integral_constant<int, EN_ACT_GELU_TANH>{}); break;
    case EN_ACT_GELU: with(std::integral_constant<int, EN_ACT_GELU>{}); break;
    default: with(std::integral_constant<int, EN_ACT_NONE>{});
  }
}

// ROWS rows of x times COLS rows of W a workgroup, 64 channels a stage.  x and the codes come through registers, U steps of 128 channels ahead,
// into LDS, x as matrix operands (see operand_vector) and the weights too, each turned into 16 bits once for all rows: (code - zero) *
// scale in fp32, rounded as a weight kept in 16 bits would be (half a step of the activations' type; scaling sums of codes instead takes four
// multiplications for each four matrix instructions of a group of 32, as many cycles as those themselves).  Where the workgroups of all rows
// and columns are few, runs of steps are shared out too, and a second launch adds up.
template <int ROWS_, int COLS_, int WR_, int WC_, int U_> struct W4Shape {
  static constexpr int ROWS = ROWS_, COLS = COLS_, WR = WR_, WC = WC_, NW = WR * WC, U = U_;
  static constexpr int RT = ROWS / 16 / WR, CT = COLS / 16 / WC;       // row tiles and tiles of W that a wave multiplies
  static constexpr int XT = ROWS / 16 / NW, WT = COLS / 16 / NW;       // ... that it brings into LDS
  static constexpr int kXStage = ROWS * 128, kWStage = COLS * 128;
  static_assert(XT * NW * 16 == ROWS && WT * NW * 16 == COLS && 8 * WT % (2 * RT) == 0, "whole tiles, pieces a row tile");
};

template <int DT, int GROUP, typename S>
__global__ __launch_bounds__(S::NW *kWave, 2) void w4_tile_kernel(W4Args a) {
  typedef Elem<DT> E;
  typedef typename E::T T;
  constexpr int kGroups = kTileCols / GROUP, RT = S::RT, CT = S::CT, XT = S::XT, WT = S::WT, U = S::U, kPieces = 8 * WT / (2 * RT);
  constexpr int kXStage = S::kXStage, kWStage = S::kWStage, kW = 2 * kXStage;
  __shared__ __align__(16) char s_mem[2 * kXStage + 2 * kWStage];      // x operands [row tile][half][lane] of two stages, W operands [tile][half][lane]
  const int lane = threadIdx.x % kWave, j = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wr = wave % S::WR, wc = wave / S::WR;
  // a column block's row blocks one after another: they read the same codes
  const int row_blocks = (a.R + S::ROWS - 1) / S::ROWS;
  const int rb = blockIdx.x % row_blocks, cb = blockIdx.x / row_blocks;
  const int r0 = rb * S::ROWS, t0 = cb * (S::COLS / kTileRows);
  const int begin = blockIdx.y * a.per, end = min(begin + a.per, a.steps);      // one step at least

  // x: this wave moves row tiles XT wave ..; channels past K and rows past R arrive as zeros
  const T *x0 = reinterpret_cast<const T *>(a.x) + (int64_t)r0 * a.x_stride;
  const int rows = min(S::ROWS, a.R - r0);
  const rsrc_t x_rsrc = make_rsrc(x0, (uint32_t)(((int64_t)(rows - 1) * a.x_stride + a.K) * 2));
  uint32_t xrow[XT];
#pragma unroll
  for (int t = 0; t < XT; ++t) {
    const int r = (XT * wave + t) * 16 + lane / 4;
    xrow[t] = r < rows ? (uint32_t)((int64_t)r * a.x_stride * 2) + operand_vector(lane) * 16 : kOutOfRange;
  }
  // W: this wave turns tiles WT wave .. into 16 bits; a lane's row of W is l % 16
  rsrc_t code_rsrc[WT], scale_rsrc[WT], zero_rsrc[WT];
#pragma unroll
  for (int t = 0; t < WT; ++t) {
    const W4Tiles<T, kGroups> tiles(a, min(t0 + WT * wave + t, a.tiles - 1), 1);
    code_rsrc[t] = tiles.codes;
    scale_rsrc[t] = tiles.scales;
    zero_rsrc[t] = tiles.zeros;
  }
  uint4 xr[U][XT][4], codes[U][WT];
  Pack<T, kGroups> sc[U][WT];
  Pack<uint8_t, kGroups> ze[U][WT];
  auto fetch = [&](int u, int step) {
    const uint32_t none = step < end ? 0u : kOutOfRange;      // nothing is read past the run
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      codes[u][t] = __builtin_bit_cast(uint4, w4_load<16, 0>(code_rsrc[t], (step * kWave + lane) * 16 | none));
      sc[u][t] = __builtin_bit_cast(Pack<T, kGroups>, w4_load<2 * kGroups, 0>(scale_rsrc[t], (step * 16 + j) * 2 * kGroups | none));
      ze[u][t] = w4_load<kGroups, 0>(zero_rsrc[t], (step * 16 + j) * kGroups | none);
    }
    const int left = a.K - step * kTileCols - operand_vector(lane) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < XT; ++t)
        xr[u][t][i] = buffer_load16(x_rsrc, (xrow[t] + (uint32_t)(step * 256 + i * 64)) | (xrow[t] & kOutOfRange) | none | (i * 32 < left ? 0u : kOutOfRange));
  };
  // The pieces of the weights of half a step: two codes a lane of operand piece / 4, which goes to LDS with its fourth.
  uint32_t piece4[4];
  float scale = 0.f, off = 0.f;
  auto put_w = [&](auto piece, int u, int part, int buf) {
    constexpr int P = decltype(piece)::value, t = P / 8, half = P / 4 % 2;
    const int word = 2 * part + half, i = word * 32 / GROUP;
    const uint32_t w = word == 0 ? codes[u][t].x : word == 1 ? codes[u][t].y : word == 2 ? codes[u][t].z : codes[u][t].w;
    if constexpr (P % 4 == 0) {
      scale = E::to_float(sc[u][t].v[i]);
      off = -(a.zeros ? (float)ze[u][t].v[i] : 8.f) * scale;
      asm volatile("" : "+v"(scale), "+v"(off));         // here, not all operands' at once
    }
    piece4[P % 4] = scaled_two<DT, P % 4>(w, scale, off);
    if constexpr (P % 4 == 3)
      *reinterpret_cast<uint4 *>(s_mem + kW + buf * kWStage + ((WT * wave + t) * 2 + half) * 1024 + lane * 16) = make_uint4(piece4[0], piece4[1], piece4[2], piece4[3]);
  };
  auto put_x = [&](int u, int part, int buf) {
#pragma unroll
    for (int t = 0; t < XT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        *reinterpret_cast<uint4 *>(s_mem + buf * kXStage + ((XT * wave + t) * 2 + half) * 1024 + lane * 16) = xr[u][t][2 * part + half];
  };

  f32x4 acc[RT][CT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  // A stage's products from buffer `buf`, and between them the next stage's operands into the other one.
  auto multiply = [&](int buf, int u, int part) {
    const char *xs = s_mem + buf * kXStage + wr * RT * 2048 + operand_slot(lane) * 16, *ws = s_mem + kW + buf * kWStage + wc * CT * 2048 + lane * 16;
    uint4 w[CT], x[2];
#pragma unroll
    for (int c = 0; c < CT; ++c) w[c] = *reinterpret_cast<const uint4 *>(ws + c * 2048);
    x[0] = *reinterpret_cast<const uint4 *>(xs);
    put_x(u, part, buf ^ 1);
    auto one = [&](auto index) {
      constexpr int I = decltype(index)::value, t = I % RT, half = I / RT;
      if constexpr (I + 1 < 2 * RT) x[(I + 1) % 2] = *reinterpret_cast<const uint4 *>(xs + (I + 1) % RT * 2048 + (I + 1) / RT * 1024);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        acc[t][c] = mma<DT>(w[c], x[I % 2], acc[t][c]);
        if constexpr (half == 0 && t == RT - 1) w[c] = *reinterpret_cast<const uint4 *>(ws + c * 2048 + 1024);
      }
      each([&](auto p) { put_w(std::integral_constant<int, I * kPieces + decltype(p)::value>{}, u, part, buf ^ 1); }, std::make_integer_sequence<int, kPieces>{});
      __builtin_amdgcn_sched_barrier(0);
    };
    each(one, std::make_integer_sequence<int, 2 * RT>{});
  };
#pragma unroll
  for (int u = 0; u < U; ++u) fetch(u, begin + u);
  put_x(0, 0, 0);
  each([&](auto piece) { put_w(piece, 0, 0, 0); }, std::make_integer_sequence<int, 8 * WT>{});
  lds_barrier();
  // (steps past the run are zeros times zeros; their products are left out, and the barriers are the workgroup's)
  for (int step = begin; step < end; step += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (step + u < end) {
        multiply(0, u, 1);
        lds_barrier();
        fetch(u, step + u + U);
        multiply(1, (u + 1) % U, 0);
        lds_barrier();
      }
    }
  }
  if (a.part) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = r0 + (wr * RT + t) * 16 + j;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const int n = (t0 + wc * CT + c) * kTileRows + 4 * g;
        if (r < a.R && n < a.N) *reinterpret_cast<f32x4 *>(a.part + ((int64_t)blockIdx.y * a.R + r) * (a.tiles * kTileRows) + n) = acc[t][c];
      }
    }
    return;
  }
  w4_finish<DT, RT, CT>(a, acc, r0 + wr * RT * 16, t0 + wc * CT);
}

// 256 rows of x times 256 rows of W a workgroup, 64 channels a stage; eight waves, 128 x 64 each.  Bound by the matrix instructions: x goes
// straight from memory into LDS (a wave's load of 16 rows x 32 channels is one operand, 1 KB, its vectors in the order of operand_vector), and
// the weights through registers as operands lie, each turned into 16 bits once for the 256 rows: (code - zero) * scale in fp32, rounded as a weight kept in 16 bits would be
// (half a step of the activations' type; scaling sums of codes instead takes four multiplications for each four matrix instructions of a
// group of 32, as many cycles as those themselves).  2000 x 5120 -> 13841, bf16: groups of 128 267 us, 1.06 PFLOP/s, of 32 290, of 32 with zero
// points, bias and ReLU 298, 0.95 PFLOP/s, of 1.4 that a large product of 16-bit matrices reaches; the rest is the last round of tiles, 440 of them on 256 compute units.
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
    const int r = (2 * wave + t) * 16 + lane / 4;
    xrow[t] = r < rows ? (uint32_t)((int64_t)r * a.x_stride * 2) : kOutOfRange;
  }
  const uint32_t lds0 = lds_address(s_mem);
  auto load_x = [&](int stage, int buf) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = stage * 64 + half * 32 + operand_vector(lane) * 8;
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
    const char *xs = s_mem + xbuf * kXStage + wr * RT * 2048 + operand_slot(lane) * 16, *ws = s_mem + kW + buf * kWStage + wc * CT * 2048 + lane * 16;
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
  w4_finish<DT, RT, CT>(a, acc, r0 + wr * RT * 16, t0 + wc * CT);
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

// Which kernel, and in how many runs the channels are shared out (a launch more, and the sums through memory).  us, groups of 128, bf16, weights that no
// cache holds, calls in a graph:
//  - narrow / wide (one tile of W a workgroup, or four, which share the loads of x): 1 x 768 -> 2304 3.1 / 4.2, 64 x 768 -> 2304 5.2 / 9.7, 1 x 4096
//    -> 4096 5.7 / 8.8, 16 x 4096 -> 4096 6.6 / 9.2; 1 x 9216 -> 9216 19.5 / 16.2, 16 x 9216 -> 9216 24.2 / 17.0, 16 x 7168 -> 28672 42 / 28;
//  - wide, runs 1 / 3 or 4: 16 x 9216 -> 9216 17.0 / 17.8; 40 x 9216 -> 9216 45 / 26, 64 x 9216 -> 9216 55 / 36, 40 x 4096 -> 4096 21 / 11.7;
//    in more they are slower again: 40 x 9216 -> 9216 in 4, 5, 6 32.5, 29.8, 31.2;
//  - wide / tiles of 128 x 128, in the runs of each: 64 x 9216 -> 9216 36 / 38, 128 x 9216 -> 9216 63 / 46;
//  - tiles of 128 x 128 / of 256 x 256: 512 x 9216 -> 9216 171 / 218, 717 171 / 218, 200 x 7168 -> 28672 137 / 174; 1000 x 9216 -> 9216 256 / 218,
//    2000 x 5120 -> 13841 334 / 267, in groups of 32 344 / 290.
enum class W4Form { kNarrow, kWide, kTile, kMany };
struct W4Plan {
  W4Form form;
  int64_t runs;
};
inline W4Plan w4_plan(int64_t rows, int64_t tiles, int64_t steps) {
  auto share = [&](int64_t workgroups, int64_t enough, int64_t most) {
    int64_t runs = enough / workgroups;
    runs = runs > most ? most : runs;
    runs = runs > steps / 4 ? steps / 4 : runs;
    return runs < 1 ? 1 : runs;
  };
  if (rows > 64) {
    if (ceil_div(rows, kManyRows) * ceil_div(tiles, kManyCols / kTileRows) >= 128) return {W4Form::kMany, 1};
    return {W4Form::kTile, share(ceil_div(rows, 128) * ceil_div(tiles, 8), 512, 8)};
  }
  if (rows <= 16) return {tiles < 512 ? W4Form::kNarrow : W4Form::kWide, 1};
  if (tiles * steps < 2048) return {W4Form::kNarrow, 1};
  return {W4Form::kWide, share(ceil_div(tiles, 4), 448, 4)};
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

int64_t en_linear_w4_workspace_bytes(int64_t rows, int64_t out_features, int64_t in_features) {
  if (rows < 1 || out_features < 1 || in_features < 1) return 0;
  const W4Plan p = w4_plan(rows, ceil_div(out_features, kTileRows), ceil_div(in_features, kTileCols));
  return p.runs > 1 ? p.runs * rows * ceil_div(out_features, kTileRows) * kTileRows * 4 : 0;
}

int en_linear_w4(const void *x, int64_t rows, int64_t x_stride, const en_w4_weight *weight, const void *bias, int activation, void *y,
                 void *workspace, int64_t workspace_bytes, en_stream_t stream) {
  if (const int bad = check_w4(weight)) return bad;
  const int64_t N = weight->out_features, K = weight->in_features;
  if (activation < EN_ACT_NONE || activation > EN_ACT_GELU) return EN_ERR_UNSUPPORTED;
  if (rows < 0 || rows > (1 << 20) || x_stride < 0 || (rows > 1 && x_stride < K) || x_stride > kMostFeatures) return EN_ERR_SHAPE;
  if (rows == 0) return EN_OK;
  const int64_t need = en_linear_w4_workspace_bytes(rows, N, K);
  if (!x || !y || (need > 0 && !workspace)) return EN_ERR_NULL;
  if (workspace_bytes < need) return EN_ERR_SHAPE;
  if (!aligned_to(x, 16) || x_stride % 8 || !aligned_to(y, 2) || !aligned_to(bias, 2) || !aligned_to(workspace, 16)) return EN_ERR_ALIGN;
  W4Args a{x, x_stride, (int)rows, (int)N, (int)K, (int)ceil_div(K, kTileCols), (int)ceil_div(N, kTileRows), (const uint4 *)weight->codes,
           weight->scales, (const uint8_t *)weight->zeros, bias, activation, y, 0, nullptr};
  const W4Plan plan = w4_plan(rows, a.tiles, a.steps);
  a.per = (int)ceil_div(a.steps, plan.runs);
  if (plan.runs > 1) a.part = reinterpret_cast<float *>(workspace);
  const unsigned runs = (unsigned)ceil_div(a.steps, a.per);
  const hipStream_t s = (hipStream_t)stream;
  auto few = [&](auto dt, auto group, auto rt, auto ct, auto nw, auto direct) {
    constexpr int RT = decltype(rt)::value, CT = decltype(ct)::value, NW = decltype(nw)::value;
    const dim3 grid((unsigned)ceil_div(a.tiles, CT), (unsigned)ceil_div(rows, 16 * RT), runs);
    w4_rows_kernel<decltype(dt)::value, decltype(group)::value, RT, CT, NW, decltype(direct)::value><<<grid, NW * kWave, 0, s>>>(a);
  };
  auto shape = [&](auto dt, auto group) {
    constexpr int DT = decltype(dt)::value, GROUP = decltype(group)::value;
    typedef std::integral_constant<int, 1> i1;
    typedef std::integral_constant<int, 2> i2;
    typedef std::integral_constant<int, 3> i3;
    typedef std::integral_constant<int, 4> i4;
    typedef std::integral_constant<int, 8> i8;
    const int row_tiles = (int)ceil_div(rows, 16);
    const std::true_type yes;
    const std::false_type no;
    // us through LDS / direct: 1 x 9216 -> 9216 16.6 / 16.2, 8 16.4 / 16.0, 16 16.6 / 16.9; 8 x 7168 -> 28672 25.4 / 25.7, 16 27.3 / 28.3
    const bool few_rows = rows <= 8;
    if (plan.form == W4Form::kMany) {
      w4_many_kernel<DT, GROUP><<<(unsigned)(ceil_div(rows, kManyRows) * ceil_div(N, kManyCols)), kManyWaves * kWave, 0, s>>>(a);
    } else if (plan.form == W4Form::kTile) {
      typedef W4Shape<128, 128, 2, 2, 2> S;
      w4_tile_kernel<DT, GROUP, S><<<dim3((unsigned)(ceil_div(rows, S::ROWS) * ceil_div(N, S::COLS)), runs), S::NW * kWave, 0, s>>>(a);
    } else if (plan.form == W4Form::kNarrow) {
      if (few_rows) few(dt, group, i1{}, i1{}, i8{}, yes);
      else if (row_tiles == 1) few(dt, group, i1{}, i1{}, i8{}, no);
      else if (row_tiles == 2) few(dt, group, i2{}, i1{}, i8{}, no);
      else if (row_tiles == 3) few(dt, group, i3{}, i1{}, i8{}, no);
      else few(dt, group, i4{}, i1{}, i8{}, no);
    } else {
      if (few_rows) few(dt, group, i1{}, i4{}, i8{}, yes);
      else if (row_tiles == 1) few(dt, group, i1{}, i4{}, i8{}, no);
      else if (row_tiles == 2) few(dt, group, i2{}, i4{}, i4{}, no);
      else if (row_tiles == 3) few(dt, group, i3{}, i4{}, i4{}, no);
      else few(dt, group, i4{}, i4{}, i4{}, no);
    }
    if (a.part) w4_join_kernel<DT><<<dim3((unsigned)ceil_div(N, 4 * kBlock), (unsigned)rows), kBlock, 0, s>>>(a, (int)runs);
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

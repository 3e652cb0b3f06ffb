// What the kernels of the 8-bit K/V cache share: the cache as a kernel sees it, and codes.
//
// Why blocks of 16 positions, full ones only, and values transposed: the attention's matrix instructions take 16 positions (the rows of
// a key tile) and, for the values, consecutive positions of one channel in a lane.  A block that is quantized once, when it is full, can lie in
// whatever order its readers want, costs no second rounding when a later position is larger, and makes a cache filled by a prompt the
// same, bit for bit, as one filled position by position.  What is not full is at most 15 rows a sequence and head, in 16 bits.
#pragma once

#include "common.hip.h"

namespace en {

constexpr int kBlk = EN_KV8_BLOCK;

struct Kv8 {
  uint8_t *kp, *vp;
  float *ks, *vs;
  void *kt, *vt;
  const int32_t *table;
  uint32_t kp_page, kp_head, vp_page, vp_head;       // bytes
  uint32_t ks_page, ks_head, vs_page, vs_head;       // elements
  int num_pages, lg_blocks, max_pages, B, H;         // 1 << lg_blocks blocks a page
};

// Positions a sequence holds in its cache: no more than its row of the page table can name.
__device__ __forceinline__ int kv8_len(const Kv8 &c, const int32_t *lens, int b) {
  return min(max(lens[b], 0), (c.max_pages << c.lg_blocks) * kBlk);
}
// Page of block j of sequence b, or -1.
__device__ __forceinline__ int kv8_page(const Kv8 &c, int b, int j) {
  const int pi = j >> c.lg_blocks;
  const int id = pi < c.max_pages ? c.table[(int64_t)b * c.max_pages + pi] : -1;
  return (unsigned)id < (unsigned)c.num_pages ? id : -1;
}
__device__ __forceinline__ int kv8_block_in_page(const Kv8 &c, int j) { return j & ((1 << c.lg_blocks) - 1); }

__device__ __forceinline__ uint8_t *kv8_k_block(const Kv8 &c, int id, int h, int blk, int D) {
  return c.kp + (uint64_t)(uint32_t)id * c.kp_page + (uint64_t)(uint32_t)h * c.kp_head + (uint64_t)(uint32_t)blk * (kBlk * D);
}
__device__ __forceinline__ uint8_t *kv8_v_block(const Kv8 &c, int id, int h, int blk, int D) {
  return c.vp + (uint64_t)(uint32_t)id * c.vp_page + (uint64_t)(uint32_t)h * c.vp_head + (uint64_t)(uint32_t)blk * (kBlk * D);
}
__device__ __forceinline__ int64_t kv8_k_scale(const Kv8 &c, int id, int h, int blk) {
  return (int64_t)((uint64_t)(uint32_t)id * c.ks_page + (uint64_t)(uint32_t)h * c.ks_head) + blk;
}
__device__ __forceinline__ int64_t kv8_v_scale(const Kv8 &c, int id, int h, int blk) {
  return (int64_t)((uint64_t)(uint32_t)id * c.vs_page + (uint64_t)(uint32_t)h * c.vs_head) + blk;
}

template <int CODE> struct Codes;
template <> struct Codes<EN_KV8_INT8> {
  static constexpr float kLargest = 127.f;
  // Four codes of x * inv.  The product is rounded to fp32 and then, by the add, to a whole number, nearest even; |x * inv| is at most 127.
  __device__ static __forceinline__ uint32_t four(float a, float b, float c, float d, float inv) {
#pragma clang fp contract(off)
    const float magic = 12582912.f;      // 1.5 * 2^23
    const uint32_t u0 = __float_as_uint(a * inv + magic), u1 = __float_as_uint(b * inv + magic), u2 = __float_as_uint(c * inv + magic),
                   u3 = __float_as_uint(d * inv + magic);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u3, u2, 0x0c0c0400), __builtin_amdgcn_perm(u1, u0, 0x0c0c0400), 0x05040100);
  }
  template <int I> __device__ static __forceinline__ float value(uint32_t w) { return (float)(int8_t)(w >> (8 * I)); }
};
template <> struct Codes<EN_KV8_E4M3> {
  static constexpr float kLargest = 448.f;
  __device__ static __forceinline__ uint32_t four(float a, float b, float c, float d, float inv) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
    return (uint32_t)w;
  }
  template <int I> __device__ static __forceinline__ float value(uint32_t w) { return __builtin_amdgcn_cvt_f32_fp8((int)w, I); }
};

// Scale of a block whose largest magnitude has these fp32 bits (NaN above infinity above all numbers), and what its values are
// multiplied by.
struct BlockScale { float scale, inv; };
template <int CODE> __device__ __forceinline__ BlockScale block_scale(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  if (top_bits >= 0x7f800000u) return {__builtin_nanf(""), 0.f};
  if (top_bits < 0x0d800000u) return {0.f, 0.f};        // 2^-100: M / a has to stay a number
  return {top / Codes<CODE>::kLargest, Codes<CODE>::kLargest / top};
}

// Largest over the wave, of numbers compared as bits.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));
  v = max(v, (uint32_t)__shfl_xor((int)v, 16, kWave));
  v = max(v, (uint32_t)__shfl_xor((int)v, 32, kWave));
  return v;
}

// ---- host side -----------------------------------------------------------------------------------------------------------------------

inline int check_kv8(const en_kv8_cache *c) {
  if (!c) return EN_ERR_NULL;
  if (c->dtype != EN_F16 && c->dtype != EN_BF16) return EN_ERR_DTYPE;
  if (c->code != EN_KV8_INT8 && c->code != EN_KV8_E4M3) return EN_ERR_DTYPE;
  if (c->batch < 0 || c->head_num < 1 || c->num_pages < 1 || c->max_pages_per_seq < 0 || c->page_size < kBlk || (c->page_size & (c->page_size - 1)) ||
      c->size_per_head < 16 || c->size_per_head > 128 || c->size_per_head % 16 || (int64_t)c->max_pages_per_seq * c->page_size > INT32_MAX - kBlk)
    return EN_ERR_SHAPE;
  if (!c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales || !c->k_tail || !c->v_tail || (!c->page_table && c->max_pages_per_seq > 0 && c->batch > 0))
    return EN_ERR_NULL;
  for (const void *p : {(const void *)c->k_pages, (const void *)c->v_pages, (const void *)c->k_tail, (const void *)c->v_tail})
    if (!aligned_to(p, 16)) return EN_ERR_ALIGN;
  for (const void *p : {(const void *)c->k_scales, (const void *)c->v_scales, (const void *)c->page_table})
    if (!aligned_to(p, 4)) return EN_ERR_ALIGN;
  for (int i = 0; i < 4; ++i) {
    if (c->code_strides[i] < 0 || c->code_strides[i] > UINT32_MAX || c->scale_strides[i] < 0 || c->scale_strides[i] > UINT32_MAX) return EN_ERR_SHAPE;
    if (c->code_strides[i] % 16) return EN_ERR_ALIGN;
  }
  return EN_OK;
}
inline Kv8 kv8_args(const en_kv8_cache *c) {
  int lg = 0;
  while ((kBlk << lg) < c->page_size) ++lg;
  return Kv8{(uint8_t *)c->k_pages, (uint8_t *)c->v_pages, c->k_scales, c->v_scales, c->k_tail, c->v_tail, c->page_table,
             (uint32_t)c->code_strides[0], (uint32_t)c->code_strides[1], (uint32_t)c->code_strides[2], (uint32_t)c->code_strides[3],
             (uint32_t)c->scale_strides[0], (uint32_t)c->scale_strides[1], (uint32_t)c->scale_strides[2], (uint32_t)c->scale_strides[3],
             c->num_pages, lg, c->max_pages_per_seq, c->batch, c->head_num};
}

}  // namespace en

// Host checks of en_kv_pages, the pair of paged pools that a drafted step reads and writes.
#pragma once

#include "common.hip.h"

namespace en {

inline int page_log2(int page_size) {
  int lg = 0;
  while ((1 << lg) < page_size) ++lg;
  return lg;
}

inline int check_kv_pages(const en_kv_pages &c) {
  const int es = dtype_size(c.dtype);
  if (es == 0) return EN_ERR_DTYPE;
  if (c.batch < 0 || c.head_num < 1 || c.num_pages < 1 || c.max_pages_per_seq < 0 || c.size_per_head < 1) return EN_ERR_SHAPE;
  if (c.page_size < 16 || (c.page_size & (c.page_size - 1))) return EN_ERR_UNSUPPORTED;
  if ((int64_t)c.max_pages_per_seq * c.page_size > INT32_MAX - 256 || c.size_per_head > 65536) return EN_ERR_SHAPE;
  for (int i = 0; i < 6; ++i)
    if (c.strides[i] < 0) return EN_ERR_SHAPE;
  if (!c.k_pool || !c.v_pool || (!c.page_table && c.max_pages_per_seq > 0 && c.batch > 0)) return EN_ERR_NULL;
  if (!aligned_to(c.page_table, 4) || !aligned_to(c.k_pool, es) || !aligned_to(c.v_pool, es)) return EN_ERR_ALIGN;
  return EN_OK;
}

}  // namespace en

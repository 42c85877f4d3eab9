// What the entry points of the 8-bit KV cache share on the host.
#pragma once
#include "launch.cuh"

#include <cstdint>

namespace fa4 {

// Shape, strides and alignment of a cache.  Touches no CUDA API.
inline int validate_cache(const fa4_fp8_cache* c) {
  if (c == nullptr) return -FA4_E_NULL;
  if (c->struct_size != sizeof(fa4_fp8_cache)) return -FA4_E_STRUCT;
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return -FA4_E_NULL;
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return -FA4_E_SHAPE;
  if (c->num_pages <= 0 || c->page_size <= 0 || c->page_size % c->block != 0 || c->Hkv <= 0) return -FA4_E_SHAPE;
  if (c->D != 64 && c->D != 128) return -FA4_E_SHAPE;
  if (c->pages_per_seq <= 0 || (c->page_table == nullptr && c->pages_per_seq != 1)) return -FA4_E_SHAPE;
  // positions are 32-bit
  if ((int64_t)c->pages_per_seq * c->page_size > 0x7ffffc00ll) return -FA4_E_TOO_LARGE;
  const int64_t strides[] = {c->k_stride_page, c->k_stride_token, c->k_stride_head,
                             c->v_stride_page, c->v_stride_token, c->v_stride_head};
  for (int64_t s : strides)
    if (s <= 0 || (s & 15) != 0) return -FA4_E_STRIDE;
  if (!aligned16(c->k) || !aligned16(c->v)) return -FA4_E_ALIGN;
  return 0;
}

inline int log2_of(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

}  // namespace fa4

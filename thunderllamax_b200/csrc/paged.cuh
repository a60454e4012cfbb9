// The paged KV cache as the kernels see it (shared by the planning, append and
// attention kernels).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "tlx_internal.h"

namespace tlx {

enum : int { CT_F16 = 0, CT_BF16 = 1, CT_Q8 = 2 };   // element type of a cache

// host checks shared by every entry point that takes a cache
inline int check_paged_kv(const tlx_paged_kv* c) {
  if (!c || !c->k || !c->v) return TLX_ERR_NULL;
  const bool q8 = c->dtype == TLX_DT_Q8;
  if (c->dtype != TLX_DT_F16 && c->dtype != TLX_DT_BF16 && !q8) return TLX_ERR_DTYPE;
  if (q8 && (!c->k_scale || !c->v_scale)) return TLX_ERR_NULL;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return TLX_ERR_SHAPE;
  if (c->kv_heads < 1 || c->kv_heads > 1024 || c->pages < 1 || c->page_size < 8 || c->page_size > 1024 ||
      (c->page_size & (c->page_size - 1)) || c->pages * c->page_size > 0x7FFFFFFFll || c->pages > 0x7FFFFFFFll)
    return TLX_ERR_SHAPE;
  const int64_t esz = q8 ? 1 : 2;
  const int64_t sbytes = c->head_dim / 32 * 2;   // one row of scales
  if ((reinterpret_cast<uintptr_t>(c->k) & 15) || (reinterpret_cast<uintptr_t>(c->v) & 15)) return TLX_ERR_ALIGN;
  if (q8 && ((reinterpret_cast<uintptr_t>(c->k_scale) % sbytes) || (reinterpret_cast<uintptr_t>(c->v_scale) % sbytes)))
    return TLX_ERR_ALIGN;
  const int64_t count[3] = {c->pages, c->kv_heads, c->page_size};
  const int64_t most = (int64_t(1) << 40) / esz;   // a TMA stride's limit
  for (int i = 0; i < 3; ++i) {
    const int64_t least = count[i] > 1 ? 1 : 0;    // rows that share memory cannot be a cache
    if (c->k_stride[i] < least || c->v_stride[i] < least || c->k_stride[i] >= most || c->v_stride[i] >= most)
      return TLX_ERR_SHAPE;
    if (((c->k_stride[i] * esz) & 15) || ((c->v_stride[i] * esz) & 15)) return TLX_ERR_ALIGN;
    if (q8 && (c->ks_stride[i] < least || c->vs_stride[i] < least)) return TLX_ERR_SHAPE;
    if (q8 && ((c->ks_stride[i] * 2) % sbytes || (c->vs_stride[i] * 2) % sbytes)) return TLX_ERR_ALIGN;
  }
  return TLX_OK;
}

inline int cache_type(const tlx_paged_kv* c) {
  return c->dtype == TLX_DT_F16 ? CT_F16 : c->dtype == TLX_DT_BF16 ? CT_BF16 : CT_Q8;
}

inline int log2_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

}  // namespace tlx

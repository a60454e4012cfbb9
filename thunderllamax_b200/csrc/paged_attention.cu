// Attention of each request's new tokens over its paged KV cache.
//
// First form: one warp per (token, query head).  32 keys at a time, a lane per key for
// the scores, then the lanes share the head's dims for the sum over V; running maximum
// and sum in fp32.
#include <algorithm>

#include "paged.cuh"

namespace tlx {
namespace {

constexpr size_t kErrBytes = 256;   // the workspace starts with the device error word

struct AttnArgs {
  tlx_paged_kv c;
  const int32_t* table;
  int64_t table_ld;
  int width, shift;
  const int32_t *q_start, *kv_len;
  int n_req;
  const uint16_t* q;
  int64_t q_tok, q_head;
  int heads, group, n_tokens, max_new;
  float scale;
  const uint16_t* gate;
  int64_t g_tok, g_head;
  uint16_t* out;
  int64_t o_tok, o_head;
};

template <bool BF>
__device__ __forceinline__ float up16(uint16_t v) {
  if constexpr (BF) return __uint_as_float(static_cast<uint32_t>(v) << 16);
  else return __half2float(__ushort_as_half(v));
}
template <bool BF>
__device__ __forceinline__ uint16_t down16(float v) {
  if constexpr (BF) return __bfloat16_as_ushort(__float2bfloat16(v));
  else return __half_as_ushort(__float2half(v));
}

template <int CT, int HD>
__global__ void __launch_bounds__(128) paged_attn_simple_kernel(const AttnArgs a) {
  constexpr bool BF = CT == CT_BF16;
  constexpr int kPer = HD / 32;
  __shared__ float qs[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t unit = blockIdx.x * 4ll + warp;
  const int t = static_cast<int>(unit / a.heads), h = static_cast<int>(unit % a.heads), g = h / a.group;
  if (t >= a.n_tokens || t >= a.q_start[a.n_req]) return;
  int lo = 0, hi = a.n_req - 1;   // the request of row t: the last one that starts at or before it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.q_start[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  const int b = lo, n = a.q_start[b + 1] - a.q_start[b];
  if (t - a.q_start[b] >= a.max_new) return;
  const int total = static_cast<int>(min(static_cast<int64_t>(a.kv_len[b]), static_cast<int64_t>(a.width) << a.shift));
  const int lim = min(total, a.kv_len[b] - n + (t - a.q_start[b]) + 1);   // keys < lim
  for (int d = lane; d < HD; d += 32) qs[warp][d] = up16<BF>(a.q[t * a.q_tok + h * a.q_head + d]) * a.scale;
  __syncwarp();
  const int32_t* tab = a.table + b * a.table_ld;
  float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  auto value = [&](const void* base, const void* sbase, const int64_t* st, const int64_t* ss, int key, int d) -> float {
    const int page = tab[key >> a.shift];
    if (page < 0 || page >= a.c.pages) return 0.f;
    const int in = key & (a.c.page_size - 1);
    const int64_t at = page * st[0] + g * st[1] + in * st[2] + d;
    if constexpr (CT == CT_Q8) {
      const float s = __half2float(static_cast<const __half*>(sbase)[page * ss[0] + g * ss[1] + in * ss[2] + (d >> 5)]);
      const float v = static_cast<float>(static_cast<int>(static_cast<const uint8_t*>(base)[at]) - 128) * s;
      return __half2float(__float2half(v));
    } else {
      return up16<BF>(static_cast<const uint16_t*>(base)[at]);
    }
  };
  for (int k0 = 0; k0 < lim; k0 += 32) {
    const int key = k0 + lane;
    float s = -INFINITY;
    if (key < lim) {
      s = 0.f;
      for (int d = 0; d < HD; ++d) s = fmaf(qs[warp][d], value(a.c.k, a.c.k_scale, a.c.k_stride, a.c.ks_stride, key, d), s);
    }
    float mt = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
    const float mn = fmaxf(m, mt);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float cor = __expf(m - base), p = __expf(s - base);
    m = mn;
    l = l * cor + p;   // per lane; summed at the end
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] *= cor;
    for (int j = 0; j < min(32, lim - k0); ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        acc[i] = fmaf(pj, value(a.c.v, a.c.v_scale, a.c.v_stride, a.c.vs_stride, k0 + j, lane + 32 * i), acc[i]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 32 * i;
    float o = lim > 0 ? acc[i] / l : 0.f;
    if (a.gate) o /= 1.f + __expf(-up16<BF>(a.gate[t * a.g_tok + h * a.g_head + d]));
    a.out[t * a.o_tok + h * a.o_head + d] = down16<BF>(o);
  }
}

template <int CT>
int launch_simple(const AttnArgs& a, cudaStream_t s) {
  const int64_t units = static_cast<int64_t>(a.n_tokens) * a.heads;
  const unsigned grid = static_cast<unsigned>((units + 3) / 4);
  if (a.c.head_dim == 256) paged_attn_simple_kernel<CT, 256><<<grid, 128, 0, s>>>(a);
  else if (a.c.head_dim == 128) paged_attn_simple_kernel<CT, 128><<<grid, 128, 0, s>>>(a);
  else paged_attn_simple_kernel<CT, 64><<<grid, 128, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? TLX_OK : TLX_ERR_LAUNCH;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace tlx

using namespace tlx;

extern "C" {

size_t tlx_paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
  if (heads < 1 || kv_heads < 1 || kv_heads > 1024 || heads % kv_heads || heads / kv_heads > 128 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  return kErrBytes;
}

int tlx_paged_attention(const tlx_paged_kv* cache, const int32_t* block_table, int64_t table_stride, int table_width,
                        const int32_t* q_start, const int32_t* kv_len, int n_requests, const void* q, int q_dtype,
                        int64_t q_tok_stride, int64_t q_head_stride, int heads, int n_tokens, int max_new, float scale,
                        const void* gate, int64_t gate_tok_stride, int64_t gate_head_stride, void* out,
                        int64_t out_tok_stride, int64_t out_head_stride, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_paged_kv(cache);
  if (rc) return rc;
  if (n_tokens < 0 || n_tokens > (1 << 28) || n_requests < 1 || n_requests > (1 << 20) || max_new < 0 ||
      table_width < 1 || table_stride < table_width || !(scale == scale))
    return TLX_ERR_SHAPE;
  const size_t need = tlx_paged_attention_workspace_bytes(heads, cache->kv_heads, cache->head_dim);
  if (!need) return TLX_ERR_SHAPE;
  if (q_dtype != TLX_DT_F16 && q_dtype != TLX_DT_BF16) return TLX_ERR_DTYPE;
  if (q_dtype != (cache->dtype == TLX_DT_Q8 ? TLX_DT_F16 : cache->dtype)) return TLX_ERR_DTYPE;
  if (n_tokens == 0 || max_new == 0) return TLX_OK;
  if (!block_table || !q_start || !kv_len || !q || !out || !ws) return TLX_ERR_NULL;
  if (!al16(q) || !al16(out) || (q_tok_stride & 7) || (q_head_stride & 7) || (out_tok_stride & 7) ||
      (out_head_stride & 7) || (reinterpret_cast<uintptr_t>(ws) & 255))
    return TLX_ERR_ALIGN;
  if (gate && (!al16(gate) || (gate_tok_stride & 7) || (gate_head_stride & 7))) return TLX_ERR_ALIGN;
  if (ws_bytes < need) return TLX_ERR_WORKSPACE;
  AttnArgs a;
  a.c = *cache;
  a.table = block_table;
  a.table_ld = table_stride;
  a.width = table_width;
  a.shift = log2_of(cache->page_size);
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.n_req = n_requests;
  a.q = static_cast<const uint16_t*>(q);
  a.q_tok = q_tok_stride;
  a.q_head = q_head_stride;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.n_tokens = n_tokens;
  a.max_new = max_new;
  a.scale = scale;
  a.gate = static_cast<const uint16_t*>(gate);
  a.g_tok = gate_tok_stride;
  a.g_head = gate_head_stride;
  a.out = static_cast<uint16_t*>(out);
  a.o_tok = out_tok_stride;
  a.o_head = out_head_stride;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (cache_type(cache)) {
    case CT_F16: return launch_simple<CT_F16>(a, s);
    case CT_BF16: return launch_simple<CT_BF16>(a, s);
    default: return launch_simple<CT_Q8>(a, s);
  }
}

}  // extern "C"

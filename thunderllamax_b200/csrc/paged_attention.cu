// Attention of each request's new tokens over its paged KV cache.
//
//   o[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(z_j - m),  z_j = scale log2(e) q . k_j,
//   over the keys j <= kv_len - n + t of the request (times sigmoid(gate)).
//
// Work is cut into items (request, KV head[, query tile]) of units of kKeys keys each and
// the units, in one row, are dealt to the CTAs in equal contiguous ranges (shared by all
// forms): whatever the lengths, every SM streams the same number of keys, and an item
// split over CTAs leaves (max, sum, unnormalised rows) per piece, which
// paged_combine_kernel joins in piece order.  The lengths are read on the device.
//
// rows form (paged_rows_kernel)   requests with at most 16 query rows per KV head (single
//   tokens, a few drafts): bound by the cache's bytes, so a warp-level matrix product on
//   16 rows is enough and the decoded keys never leave registers.
// tiles form (paged_tiles_kernel)  the rest: tcgen05 on tiles of 128 query rows.
#include "paged_attention.cuh"

namespace tlx {
namespace {

// -------------------------------------------------------------------- combine
// Joins the pieces of the split items: the maxima give the pieces' weights, the weighted
// rows are added in piece order (with many pieces: eight shares in order, then the shares),
// so the result does not depend on when anything ran.  A warp takes a row of an item of up
// to kWarpPieces pieces, else a block does, a warp per share: a few pieces cost one trip to
// memory for their statistics and one for their rows, without a barrier.
constexpr int kWarpPieces = 16;

template <bool BF, int HD, int ROWS>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int VEC = HD / 32;   // values of a lane
  __shared__ float acc[8][HD];
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.by_item) {   // only the items of this launch have written their entry
    const Req r = get_req(a, blockIdx.x / a.c.kv_heads);
    if (r.n < 1 || r.n * static_cast<int64_t>(a.group) > a.rows_limit) return;
  }
  const int4 d = a.desc[blockIdx.x];   // {slot of the first piece, last CTA, request << 10 | KV head, tile}
  if (d.x < 0) return;
  const int b = d.z >> 10, head = d.z & 1023;
  const Req r = get_req(a, b);
  const int tt = 128 / a.group, t0 = d.w * tt, rows = min(tt, r.n - t0) * a.group;
  const int c0 = d.x >> 1, pieces = d.y - c0 + 1;
  auto slot_of = [&](int p) { return p == 0 ? d.x : 2 * (c0 + p); };
  const bool alone = pieces <= kWarpPieces;   // a warp for the row
  // pieces of this warp
  const int p0 = alone ? 0 : pieces * warp / 8, p1 = alone ? pieces : pieces * (warp + 1) / 8;
  for (int row = alone ? blockIdx.y * 8 + warp : blockIdx.y; row < rows; row += gridDim.y * (alone ? 8 : 1)) {
    float m = -INFINITY;
    for (int p = lane; p < pieces; p += 32) m = fmaxf(m, a.ml[slot_of(p) * ROWS + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int p = lane; p < pieces; p += 32) {
      const float2 x = a.ml[slot_of(p) * ROWS + row];
      l += x.y * ex2_approx(x.x - base);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = 0.f;
#pragma unroll 4
    for (int p = p0; p < p1; ++p) {
      const int slot = slot_of(p);
      const float w = ex2_approx(a.ml[slot * ROWS + row].x - base);
      const float2* v = reinterpret_cast<const float2*>(a.part + (static_cast<int64_t>(slot) * ROWS + row) * HD) + lane;
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {   // dims 64 (j / 2) + 2 lane, + 1
        const float2 y = v[j * 16];
        s[j] = fmaf(y.x, w, s[j]);
        s[j + 1] = fmaf(y.y, w, s[j + 1]);
      }
    }
    if (!alone) {
#pragma unroll
      for (int j = 0; j < VEC; j += 2) *reinterpret_cast<float2*>(&acc[warp][j * 32 + 2 * lane]) = make_float2(s[j], s[j + 1]);
      __syncthreads();
      if (warp == 0) {
        for (int w = 1; w < 8; ++w) {
#pragma unroll
          for (int j = 0; j < VEC; j += 2) {
            s[j] += acc[w][j * 32 + 2 * lane];
            s[j + 1] += acc[w][j * 32 + 2 * lane + 1];
          }
        }
      }
    }
    if (alone || warp == 0) {
      const int t = t0 + row / a.group, hq = head * a.group + row % a.group;
      const bool sees = min(r.keys, r.kv - r.n_all + t + 1) > 0;
      const int64_t tok = r.q0 + t;
      const float inv = 1.f / l;
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const int dim = j * 32 + 2 * lane;
        float v0 = sees ? s[j] * inv : 0.f, v1 = sees ? s[j + 1] * inv : 0.f;
        if (a.gate) {
          const float2 x = unpack2<BF>(*reinterpret_cast<const uint32_t*>(a.gate + tok * a.g_tok + hq * a.g_head + dim));
          v0 = gated(v0, x.x);
          v1 = gated(v1, x.y);
        }
        *reinterpret_cast<uint32_t*>(a.out + tok * a.o_tok + hq * a.o_head + dim) = pack2<BF>(v0, v1);
      }
    }
    if (!alone) __syncthreads();   // acc is free for the next row
  }
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

int launch_dependent(const void* kern, dim3 grid, dim3 block, cudaStream_t stream, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, kern, args) == cudaSuccess ? TLX_OK : TLX_ERR_LAUNCH;
}

template <bool BF, int HD>
const void* combine_kernel(int row_slots) {
  return row_slots == kRowsMax ? reinterpret_cast<const void*>(paged_combine_kernel<BF, HD, kRowsMax>)
                               : reinterpret_cast<const void*>(paged_combine_kernel<BF, HD, 128>);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int launch_combine(const AttnArgs& a, bool bf, int row_slots, int items, int rows, cudaStream_t stream) {
  const int hd = a.c.head_dim;
  const void* kern = bf ? (hd == 256 ? combine_kernel<true, 256>(row_slots) : hd == 128 ? combine_kernel<true, 128>(row_slots) : combine_kernel<true, 64>(row_slots))
                        : (hd == 256 ? combine_kernel<false, 256>(row_slots) : hd == 128 ? combine_kernel<false, 128>(row_slots) : combine_kernel<false, 64>(row_slots));
  AttnArgs copy = a;
  void* args[] = {&copy};
  return launch_dependent(kern, dim3(items, rows), dim3(256), stream, args);
}

}  // namespace tlx

using namespace tlx;

extern "C" {

size_t tlx_paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
  if (heads < 1 || kv_heads < 1 || kv_heads > 1024 || heads % kv_heads || heads / kv_heads > 128 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  const int sms = sm_count();
  return std::max(paged_rows_bytes(head_dim, sms), paged_tiles_bytes(head_dim, sms));
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
  a.max_new = std::min(max_new, n_tokens);
  a.rows_limit = kRowsMax;
  a.scale = scale;
  a.gate = static_cast<const uint16_t*>(gate);
  a.g_tok = gate_tok_stride;
  a.g_head = gate_head_stride;
  a.out = static_cast<uint16_t*>(out);
  a.o_tok = out_tok_stride;
  a.o_head = out_head_stride;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // the requests' lengths are on the device, so each form picks its own requests there
  const int ct = cache_type(cache), sms = sm_count();
  if (a.group <= kRowsMax) {
    const int rows_rc = launch_paged_rows(a, ct, ws, sms, s);
    if (rows_rc) return rows_rc;
  }
  if (static_cast<int64_t>(a.max_new) * a.group <= kRowsMax) return TLX_OK;
  return launch_paged_tiles(a, ct, ws, sms, s);
}

}  // extern "C"

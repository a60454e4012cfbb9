// Attention of each request's new tokens over its paged KV cache.
//
//   o[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(z_j - m),  z_j = scale log2(e) q . k_j,
//   over the keys j <= kv_len - n + t of the request (times sigmoid(gate)).
//
// Work is cut into items (request, KV head[, query tile]) of units of kKeys keys each and
// the units, in one row, are dealt to the CTAs in equal contiguous ranges (shared by all
// forms): whatever the lengths, every SM streams the same number of keys, and an item
// split over CTAs leaves (max, sum, unnormalised rows) per piece, which
// paged_combine_kernel joins in piece order.  An item's fixed cost counts as some units
// more (kItemCost).  The lengths are read on the device.
//
// rows form (paged_rows_kernel)   requests with at most 16 query rows per KV head (single
//   tokens, a few drafts): bound by the cache's bytes, so a warp-level matrix product on
//   16 rows is enough and the decoded keys never leave registers.
// tiles form (paged_tiles_kernel)  the rest: tcgen05 on tiles of 128 query rows.
#include <cmath>

#include "paged_attention.cuh"

namespace tlx {
namespace {

// -------------------------------------------------------------------- combine
// Joins the pieces of the split items: the maxima give the pieces' weights, the weighted
// rows are added in piece order (with many pieces: eight shares in order, then the shares),
// so the result does not depend on when anything ran.  A warp takes a row of an item of up
// to kWarpPieces pieces, else a block does, a warp per share: a few pieces cost one trip to
// memory for their statistics and one for their rows, without a barrier.  Bound by latency:
// about 6 us behind one decode row at 4097 keys (65 pieces a head).
constexpr int kWarpPieces = 16;

struct CombineArgs {
  AttnArgs a;
  SplitSet set[2];   // rows form, tiles form
};

template <bool BF, int HD>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ CombineArgs ca) {
  constexpr int VEC = HD / 32;   // values of a lane
  __shared__ float acc[8][HD];
  griddep_wait();
  const AttnArgs& a = ca.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool second = static_cast<int>(blockIdx.x) >= ca.set[0].items;
  const SplitSet& set = ca.set[second ? 1 : 0];
  const int index = blockIdx.x - (second ? ca.set[0].items : 0), slots = set.row_slots;
  const int4 d = set.desc[index];   // {slot of the first piece, last CTA, request << 10 | KV head, tile}
  int b = index / a.c.kv_heads;
  if (!set.by_item) {
    if (d.x < 0) return;
    b = d.z >> 10;
  }
  const Req r = get_req(a, b);
  // (an entry by item is this launch's only if the request has units in this form)
  if (set.by_item && (r.n < 1 || r.n * static_cast<int64_t>(a.group) > a.rows_limit || d.x < 0)) return;
  const int head = d.z & 1023;
  const int tt = 128 / a.group, t0 = d.w * tt, rows = min(tt, r.n - t0) * a.group;
  const int c0 = d.x >> 1, pieces = d.y - c0 + 1;
  auto slot_of = [&](int p) { return p == 0 ? d.x : 2 * (c0 + p); };
  const bool alone = pieces <= kWarpPieces;   // a warp for the row
  // pieces of this warp
  const int p0 = alone ? 0 : pieces * warp / 8, p1 = alone ? pieces : pieces * (warp + 1) / 8;
  for (int row = alone ? blockIdx.y * 8 + warp : blockIdx.y; row < rows; row += gridDim.y * (alone ? 8 : 1)) {
    // statistics of the first 64 pieces stay with their lane
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 x0 = lane < pieces ? set.ml[slot_of(lane) * slots + row] : none;
    const float2 x1 = 32 + lane < pieces ? set.ml[slot_of(32 + lane) * slots + row] : none;
    float m = fmaxf(x0.x, x1.x);
    for (int p = 64 + lane; p < pieces; p += 32) m = fmaxf(m, set.ml[slot_of(p) * slots + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    const float w0 = ex2_approx(x0.x - base), w1 = ex2_approx(x1.x - base);
    float l = x0.y * w0 + x1.y * w1;
    for (int p = 64 + lane; p < pieces; p += 32) {
      const float2 x = set.ml[slot_of(p) * slots + row];
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
      float w = __shfl_sync(0xffffffffu, p < 32 ? w0 : w1, p & 31);
      if (p >= 64) w = ex2_approx(set.ml[slot * slots + row].x - base);
      const float2* v = reinterpret_cast<const float2*>(set.part + (static_cast<int64_t>(slot) * slots + row) * HD) + lane;
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
#pragma unroll 1
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
  static int counts[64] = {};   // by device (asking takes as long as a launch)
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (counts[dev] == 0) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    counts[dev] = n > 0 ? n : 148;
  }
  return counts[dev];
}

template <bool BF>
const void* combine_kernel(int hd) {
  return hd == 256   ? reinterpret_cast<const void*>(paged_combine_kernel<BF, 256>)
         : hd == 128 ? reinterpret_cast<const void*>(paged_combine_kernel<BF, 128>)
                     : reinterpret_cast<const void*>(paged_combine_kernel<BF, 64>);
}

int launch_combine(CombineArgs& ca, bool bf, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  // rows of an item: one a block (many pieces), or eight; the tiles form's blocks walk theirs
  cfg.gridDim = dim3(ca.set[0].items + ca.set[1].items, std::max(ca.set[0].rows, std::min(32, ca.set[1].rows)));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&ca};
  return cudaLaunchKernelExC(&cfg, bf ? combine_kernel<true>(ca.a.c.head_dim) : combine_kernel<false>(ca.a.c.head_dim),
                             args) == cudaSuccess
             ? TLX_OK
             : TLX_ERR_LAUNCH;
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
  const int sms = sm_count();
  return kPagedErrBytes + paged_rows_bytes(head_dim, sms) + paged_tiles_bytes(head_dim, sms);
}

int tlx_paged_attention(const tlx_paged_kv* cache, const int32_t* block_table, int64_t table_stride, int table_width,
                        const int32_t* q_start, const int32_t* kv_len, int n_requests, const void* q, int q_dtype,
                        int64_t q_tok_stride, int64_t q_head_stride, int heads, int n_tokens, int max_new, float scale,
                        const void* gate, int64_t gate_tok_stride, int64_t gate_head_stride, void* out,
                        int64_t out_tok_stride, int64_t out_head_stride, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_paged_kv(cache);
  if (rc) return rc;
  if (n_tokens < 0 || n_tokens > (1 << 28) || n_requests < 1 || n_requests > (1 << 20) || max_new < 0 ||
      table_width < 1 || table_stride < table_width || !(scale > 0.f && scale < INFINITY))
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
  uint8_t* area = static_cast<uint8_t*>(ws) + kPagedErrBytes;
  CombineArgs ca;
  ca.a = a;
  ca.set[0] = ca.set[1] = SplitSet{nullptr, nullptr, nullptr, 0, 0, 0, 0};
  const bool rows = a.group <= kRowsMax, tiles = static_cast<int64_t>(a.max_new) * a.group > kRowsMax;
  if (rows) {
    const int rc_rows = launch_paged_rows(a, ct, area, sms, s, &ca.set[0]);
    if (rc_rows) return rc_rows;
  }
  if (tiles) {
    const int rc_tiles = launch_paged_tiles(a, ct, area + paged_rows_bytes(cache->head_dim, sms), static_cast<uint32_t*>(ws),
                                            sms, rows, s, &ca.set[1]);
    if (rc_tiles) return rc_tiles;
  }
  return launch_combine(ca, ct == CT_BF16, s);
}

}  // extern "C"

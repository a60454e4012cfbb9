// Paged KV cache: page planning on the device and the append of new rows.
//
// plan      For request b with c cached and n new tokens and h pages already held:
//             need = ceil((c + n) / page), take = max(0, need - h),
//             end  = inclusive prefix sum of take over the requests,
//             ok   = lengths valid, need <= table width, and take == 0 or end <= free pages.
//           The i-th page the batch takes (i = end - take + j) is free[n_free - 1 - i] and
//           becomes table entry h + j.  One launch: every CTA computes the same prefix
//           sums (they are a few loads and one block scan per 512 requests, cheaper than
//           a second launch) and writes its share of the tokens and pages, found by a
//           binary search in the prefix sums, so one long prompt spreads like many short
//           ones.  held and n_free may be updated in place: the last CTA to finish
//           writes them, when every CTA has read them.
//           Bound by the launch and a few dependent trips to memory: 4.1 us for 64 requests,
//           11.6 us for 1000 requests with 118 K new tokens.
// release   One CTA returns the pages of finished requests to the free stack.
// append    Copies or quantises the rows of the new tokens into their slots.  Bound by HBM: 8191
//           bf16 rows of 8 heads x 128 (67 MB) in 12.5 us, 5.4 TB/s (0.82 of the measured copy
//           rate); 64 int8 rows in 2.1 us (latency).
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace tlx {
namespace {

constexpr int kPlanThreads = 512;

struct Sums {
  int64_t tok, page;
};

// inclusive block scan of two counts; every thread calls it
__device__ __forceinline__ Sums block_scan(Sums v, Sums* warp_tot, Sums* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, v.tok, o), b = __shfl_up_sync(0xffffffffu, v.page, o);
    if (lane >= o) {
      v.tok += a;
      v.page += b;
    }
  }
  if (lane == 31) warp_tot[warp] = v;
  __syncthreads();
  if (warp == 0) {
    Sums w = lane < kPlanThreads / 32 ? warp_tot[lane] : Sums{0, 0};
#pragma unroll
    for (int o = 1; o < kPlanThreads / 32; o <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, w.tok, o), b = __shfl_up_sync(0xffffffffu, w.page, o);
      if (lane >= o) {
        w.tok += a;
        w.page += b;
      }
    }
    if (lane < kPlanThreads / 32) warp_tot[lane] = w;
  }
  __syncthreads();
  if (warp > 0) {
    v.tok += warp_tot[warp - 1].tok;
    v.page += warp_tot[warp - 1].page;
  }
  *total = warp_tot[kPlanThreads / 32 - 1];
  __syncthreads();   // warp_tot is free for the next call
  return v;
}

struct PlanArgs {
  const int32_t *cached, *fresh;
  int n_req, shift, page_mask, width;
  int64_t ld;
  int32_t* table;
  const int32_t* held_in;
  int32_t* held_out;
  const int32_t* free_pages;
  int64_t pages;
  const int32_t* n_free_in;
  int32_t* n_free_out;
  int n_tokens;
  int32_t *q_start, *kv_len, *slots, *positions, *status;
  uint32_t* arrivals;
};

struct PlanChunk {           // the requests of one chunk, in shared memory
  int64_t tok0[kPlanThreads + 1];   // first token of each request
  int64_t page0[kPlanThreads + 1];  // first page (of the batch's taken pages)
  int32_t cached[kPlanThreads], held[kPlanThreads], take[kPlanThreads];
  int32_t status[kPlanThreads];
  Sums warp_tot[kPlanThreads / 32];
};

__device__ __forceinline__ int last_at_most(const int64_t* a, int n, int64_t x) {   // largest i < n with a[i] <= x
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// loads requests [r0, r0 + cnt), leaves their prefix sums in sh and returns the sums
// after the chunk
__device__ __forceinline__ Sums plan_chunk(const PlanArgs& a, PlanChunk& sh, int r0, int cnt, Sums base, int64_t n_free) {
  const int i = threadIdx.x;
  int c = 0, n = 0, h = 0, st = 0;
  int64_t take = 0;
  if (i < cnt) {
    c = a.cached[r0 + i];
    n = a.fresh[r0 + i];
    h = a.held_in[r0 + i];
    if (c < 0 || n < 0 || h < 0 || n > a.n_tokens || c > 0x7FFFFFFF - n) {
      st = TLX_PAGED_BAD_LENGTH;
      n = n < 0 || n > a.n_tokens ? 0 : n;
      c = 0;
    } else {
      const int64_t need = (static_cast<int64_t>(c) + n + a.page_mask) >> a.shift;
      if (need > a.width || h > a.width) st = TLX_PAGED_TABLE_FULL;
      else take = need > h ? need - h : 0;
    }
  }
  Sums total;
  const Sums incl = block_scan(Sums{n, take}, sh.warp_tot, &total);
  if (i < cnt) {
    sh.tok0[i] = base.tok + incl.tok - n;
    sh.page0[i] = base.page + incl.page - take;
    if (st == 0 && base.tok + incl.tok > a.n_tokens) st = TLX_PAGED_BAD_LENGTH;
    if (st == 0 && take > 0 && base.page + incl.page > n_free) st = TLX_PAGED_NO_PAGES;
    sh.cached[i] = c;
    sh.held[i] = h;
    sh.take[i] = static_cast<int32_t>(take);
    sh.status[i] = st;
  }
  const Sums next{base.tok + total.tok, base.page + total.page};
  if (i == 0) {
    sh.tok0[cnt] = next.tok;
    sh.page0[cnt] = next.page;
  }
  __syncthreads();
  return next;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs a) {
  __shared__ PlanChunk sh;
  __shared__ int last;
  const int tid = threadIdx.x;
  const int64_t gsize = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid;
  const int64_t n_free = min(static_cast<int64_t>(max(a.n_free_in[0], 0)), a.pages);
  Sums base{0, 0};
  for (int r0 = 0; r0 < a.n_req; r0 += kPlanThreads) {
    const int cnt = min(kPlanThreads, a.n_req - r0);
    if (r0 > 0) __syncthreads();
    const Sums next = plan_chunk(a, sh, r0, cnt, base, n_free);
    if (blockIdx.x == 0) {
      for (int i = tid; i < cnt; i += kPlanThreads) {
        const int n = static_cast<int>(sh.tok0[i + 1] - sh.tok0[i]);
        a.q_start[r0 + i] = static_cast<int32_t>(min(sh.tok0[i], static_cast<int64_t>(a.n_tokens)));
        a.kv_len[r0 + i] = sh.status[i] == 0 ? sh.cached[i] + n : 0;
        a.status[r0 + i] = sh.status[i];
      }
      if (tid == 0 && r0 + cnt == a.n_req)
        a.q_start[a.n_req] = static_cast<int32_t>(min(next.tok, static_cast<int64_t>(a.n_tokens)));
    }
    // the table entries of the pages taken by this chunk
    for (int64_t p = base.page + gid; p < next.page && p < n_free; p += gsize) {
      const int i = last_at_most(sh.page0, cnt, p);
      const int64_t j = p - sh.page0[i];
      if (sh.status[i] == 0 && j < sh.take[i])
        a.table[(r0 + i) * a.ld + sh.held[i] + j] = a.free_pages[n_free - 1 - p];
    }
    // slots and positions of this chunk's tokens
    for (int64_t t = base.tok + gid; t < next.tok && t < a.n_tokens; t += gsize) {
      const int i = last_at_most(sh.tok0, cnt, t);
      const int pos = sh.cached[i] + static_cast<int>(t - sh.tok0[i]);
      int slot = -1;
      if (sh.status[i] == 0) {
        const int pg = pos >> a.shift;
        const int id = pg < sh.held[i] ? a.table[(r0 + i) * a.ld + pg]
                                       : a.free_pages[n_free - 1 - (sh.page0[i] + pg - sh.held[i])];
        if (id >= 0 && id < a.pages) slot = (id << a.shift) + (pos & a.page_mask);
      }
      a.slots[t] = slot;
      a.positions[t] = pos;
    }
    base = next;
  }
  // rows past the last request's tokens have no slot
  for (int64_t t = base.tok + gid; t < a.n_tokens; t += gsize) {
    a.slots[t] = -1;
    a.positions[t] = -1;
  }
  if (gridDim.x > 1) {
    __syncthreads();   // every thread of the CTA has read held and n_free
    if (tid == 0) {
      __threadfence();
      last = atomicAdd(a.arrivals, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
  } else {
    __syncthreads();
  }
  int64_t taken = 0;   // pages taken by the served requests: a prefix of the batch's, so the last one's end
  base = Sums{0, 0};
  for (int r0 = 0; r0 < a.n_req; r0 += kPlanThreads) {
    const int cnt = min(kPlanThreads, a.n_req - r0);
    Sums next = base;
    if (a.n_req > kPlanThreads) {
      __syncthreads();
      next = plan_chunk(a, sh, r0, cnt, base, n_free);
    }
    for (int i = tid; i < cnt; i += kPlanThreads) {
      if (sh.status[i] == 0 && sh.take[i] > 0) taken = sh.page0[i] + sh.take[i];
      a.held_out[r0 + i] = sh.held[i] + (sh.status[i] == 0 ? sh.take[i] : 0);
    }
    base = next;
  }
  __shared__ unsigned long long most;
  if (tid == 0) most = 0ull;
  __syncthreads();
  atomicMax(&most, static_cast<unsigned long long>(taken));
  __syncthreads();
  if (tid == 0) {
    a.n_free_out[0] = static_cast<int32_t>(n_free - static_cast<int64_t>(most));
    if (gridDim.x > 1) *a.arrivals = 0u;
  }
}

__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(const int32_t* __restrict__ done, int n_req,
                                                                     int32_t* __restrict__ table, int64_t ld, int width,
                                                                     int32_t* __restrict__ held,
                                                                     int32_t* __restrict__ free_pages, int64_t pages,
                                                                     int32_t* __restrict__ n_free) {
  __shared__ int64_t page0[kPlanThreads + 1];
  __shared__ Sums warp_tot[kPlanThreads / 32];
  int64_t top = max(n_free[0], 0);
  const int i = threadIdx.x;
  for (int r0 = 0; r0 < n_req; r0 += kPlanThreads) {
    const int cnt = min(kPlanThreads, n_req - r0);
    const int h = i < cnt && done[r0 + i] != 0 ? min(max(held[r0 + i], 0), width) : 0;
    Sums total;
    const Sums incl = block_scan(Sums{0, h}, warp_tot, &total);
    if (i < cnt) page0[i] = incl.page - h;
    __syncthreads();
    for (int64_t p = i; p < total.page; p += kPlanThreads) {
      const int r = last_at_most(page0, cnt, p);
      int32_t* e = table + (r0 + r) * ld + (p - page0[r]);
      if (top + p < pages) free_pages[top + p] = *e;
      *e = -1;
    }
    if (h > 0) held[r0 + i] = 0;
    top = min(top + total.page, pages);
    __syncthreads();
  }
  if (i == 0) n_free[0] = static_cast<int32_t>(top);
}

// ---------------------------------------------------------------------- append
struct AppendArgs {
  tlx_paged_kv c;
  const uint8_t* x[2];        // k, v rows
  int64_t tok_stride[2], head_stride[2];   // elements
  const int32_t* slots;
  int n_tokens, shift;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same_v<T, __half>) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
      } else {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
}

// A thread moves 8 dims of one row; four threads share a 32-dim group of the int8 cache.
// The int8 rule is the one of the contiguous cache: scale fp16(max|x| / 127), or 1e-8
// (0 in fp16) for an all-zero group, code rint(clamp(x / scale, +-127)) + 128 with the
// IEEE quotient; fmaxf / fminf turn the 0 / 0 of an all-zero group into code 1.
template <typename T, int CT, int HD>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs a) {
  constexpr int kUnits = HD / 8;
  const int64_t n = static_cast<int64_t>(a.n_tokens) * a.c.kv_heads * kUnits;   // per matrix
  const int which = blockIdx.y;
  const T* x = reinterpret_cast<const T*>(a.x[which]);
  uint8_t* cache = static_cast<uint8_t*>(which ? a.c.v : a.c.k);
  const int64_t* cs = which ? a.c.v_stride : a.c.k_stride;
  // a group's four threads are neighbours, and n is a multiple of 8, so a warp's
  // threads leave the loop together in groups of 8
  for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < n; u += gridDim.x * 256ll) {
    const int part = static_cast<int>(u % kUnits);
    const int64_t row = u / kUnits;
    const int head = static_cast<int>(row % a.c.kv_heads);
    const int64_t t = row / a.c.kv_heads;
    const int slot = a.slots[t];
    const bool ok = slot >= 0 && (slot >> a.shift) < a.c.pages;
    const int64_t page = slot >> a.shift, in_page = slot & (a.c.page_size - 1);
    const T* src = x + t * a.tok_stride[which] + head * a.head_stride[which] + part * 8;
    const int64_t dst = page * cs[0] + head * cs[1] + in_page * cs[2] + part * 8;
    if constexpr (CT != CT_Q8 && sizeof(T) == 2) {   // same type: the bytes themselves
      if (ok) *reinterpret_cast<uint4*>(cache + dst * 2) = *reinterpret_cast<const uint4*>(src);
    } else {
      float f[8];
      load8(src, f);
      if constexpr (CT == CT_F16) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = h2_bits(__floats2half2_rn(f[2 * j], f[2 * j + 1]));
        if (ok) *reinterpret_cast<uint4*>(cache + dst * 2) = make_uint4(w[0], w[1], w[2], w[3]);
      } else if constexpr (CT == CT_BF16) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        if (ok) *reinterpret_cast<uint4*>(cache + dst * 2) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(f[j]));
        const uint32_t peers = 0xFu << (threadIdx.x & 28);
        m = fmaxf(m, __shfl_xor_sync(peers, m, 1));
        m = fmaxf(m, __shfl_xor_sync(peers, m, 2));
        const __half s = __float2half(m > 0.f ? m * (1.f / 127.f) : 1e-8f);
        const float sf = __half2float(s);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int q = __float2int_rn(fminf(fmaxf(__fdiv_rn(f[j], sf), -127.f), 127.f));
          w[j >> 2] |= static_cast<uint32_t>(q + 128) << (8 * (j & 3));
        }
        if (ok) {
          *reinterpret_cast<uint2*>(cache + dst) = make_uint2(w[0], w[1]);
          if ((part & 3) == 0) {
            __half* sc = static_cast<__half*>(which ? a.c.v_scale : a.c.k_scale);
            const int64_t* ss = which ? a.c.vs_stride : a.c.ks_stride;
            sc[page * ss[0] + head * ss[1] + in_page * ss[2] + (part >> 2)] = s;
          }
        }
      }
    }
  }
}

template <typename T, int CT>
int launch_append(const AppendArgs& a, cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.n_tokens) * a.c.kv_heads * (a.c.head_dim / 8);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((units + 255) / 256, 148 * 32)), 2);
  if (a.c.head_dim == 256) paged_append_kernel<T, CT, 256><<<grid, 256, 0, stream>>>(a);
  else if (a.c.head_dim == 128) paged_append_kernel<T, CT, 128><<<grid, 256, 0, stream>>>(a);
  else paged_append_kernel<T, CT, 64><<<grid, 256, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? TLX_OK : TLX_ERR_LAUNCH;
}

bool al(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace tlx

using namespace tlx;

extern "C" {

size_t tlx_paged_plan_workspace_bytes(void) { return 256; }

int tlx_paged_plan(const int32_t* cached_len, const int32_t* new_len, int n_requests, int page_size,
                   int32_t* block_table, int64_t table_stride, int table_width, const int32_t* held_in,
                   int32_t* held_out, const int32_t* free_pages, int64_t pages, const int32_t* n_free_in,
                   int32_t* n_free_out, int n_tokens, int32_t* q_start, int32_t* kv_len, int32_t* slots,
                   int32_t* positions, int32_t* status, void* ws, size_t ws_bytes, void* stream) {
  if (!cached_len || !new_len || !block_table || !held_in || !held_out || !free_pages || !n_free_in || !n_free_out ||
      !q_start || !kv_len || !status || !ws || (n_tokens > 0 && (!slots || !positions)))
    return TLX_ERR_NULL;
  if (n_requests < 1 || n_requests > (1 << 20) || page_size < 8 || page_size > 1024 || (page_size & (page_size - 1)) ||
      table_width < 1 || table_stride < table_width || pages < 1 || pages * page_size > 0x7FFFFFFFll ||
      pages > 0x7FFFFFFFll || n_tokens < 0 || n_tokens > (1 << 28))
    return TLX_ERR_SHAPE;
  if (!al(ws, 4)) return TLX_ERR_ALIGN;
  if (ws_bytes < tlx_paged_plan_workspace_bytes()) return TLX_ERR_WORKSPACE;
  PlanArgs a;
  a.cached = cached_len;
  a.fresh = new_len;
  a.n_req = n_requests;
  a.shift = log2_of(page_size);
  a.page_mask = page_size - 1;
  a.width = table_width;
  a.ld = table_stride;
  a.table = block_table;
  a.held_in = held_in;
  a.held_out = held_out;
  a.free_pages = free_pages;
  a.pages = pages;
  a.n_free_in = n_free_in;
  a.n_free_out = n_free_out;
  a.n_tokens = n_tokens;
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.slots = slots;
  a.positions = positions;
  a.status = status;
  a.arrivals = static_cast<uint32_t*>(ws);
  const int blocks = std::max(1, std::min(148, (n_tokens + 2 * kPlanThreads - 1) / (2 * kPlanThreads)));
  paged_plan_kernel<<<blocks, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? TLX_OK : TLX_ERR_LAUNCH;
}

int tlx_paged_release(const int32_t* done, int n_requests, int32_t* block_table, int64_t table_stride, int table_width,
                      int32_t* held, int32_t* free_pages, int64_t pages, int32_t* n_free, void* stream) {
  if (!done || !block_table || !held || !free_pages || !n_free) return TLX_ERR_NULL;
  if (n_requests < 1 || n_requests > (1 << 20) || table_width < 1 || table_stride < table_width || pages < 1 ||
      pages > 0x7FFFFFFFll)
    return TLX_ERR_SHAPE;
  paged_release_kernel<<<1, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(done, n_requests, block_table,
                                                                                  table_stride, table_width, held,
                                                                                  free_pages, pages, n_free);
  return cudaGetLastError() == cudaSuccess ? TLX_OK : TLX_ERR_LAUNCH;
}

int tlx_paged_append(const tlx_paged_kv* cache, const void* k, const void* v, int x_dtype, int64_t k_tok_stride,
                     int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride, const int32_t* slots,
                     int n_tokens, void* stream) {
  const int rc = check_paged_kv(cache);
  if (rc) return rc;
  if (n_tokens < 0 || n_tokens > (1 << 28)) return TLX_ERR_SHAPE;
  if (x_dtype != TLX_DT_F32 && x_dtype != TLX_DT_F16 && x_dtype != TLX_DT_BF16) return TLX_ERR_DTYPE;
  if (n_tokens == 0) return TLX_OK;
  if (!k || !v || !slots) return TLX_ERR_NULL;
  const int esz = x_dtype == TLX_DT_F32 ? 4 : 2;
  // a 16-bit cache takes its own type or fp32
  if (esz == 2 && cache->dtype != TLX_DT_Q8 && cache->dtype != x_dtype) return TLX_ERR_DTYPE;
  if (!al(k, 16) || !al(v, 16) || k_tok_stride * esz % 16 || k_head_stride * esz % 16 || v_tok_stride * esz % 16 ||
      v_head_stride * esz % 16)
    return TLX_ERR_ALIGN;
  AppendArgs a;
  a.c = *cache;
  a.x[0] = static_cast<const uint8_t*>(k);
  a.x[1] = static_cast<const uint8_t*>(v);
  a.tok_stride[0] = k_tok_stride;
  a.tok_stride[1] = v_tok_stride;
  a.head_stride[0] = k_head_stride;
  a.head_stride[1] = v_head_stride;
  a.slots = slots;
  a.n_tokens = n_tokens;
  a.shift = log2_of(cache->page_size);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (cache_type(cache)) {
    case CT_F16:
      return esz == 4 ? launch_append<float, CT_F16>(a, s) : launch_append<__half, CT_F16>(a, s);
    case CT_BF16:
      return esz == 4 ? launch_append<float, CT_BF16>(a, s) : launch_append<__nv_bfloat16, CT_BF16>(a, s);
    default:
      if (x_dtype == TLX_DT_F32) return launch_append<float, CT_Q8>(a, s);
      if (x_dtype == TLX_DT_F16) return launch_append<__half, CT_Q8>(a, s);
      return launch_append<__nv_bfloat16, CT_Q8>(a, s);
  }
}

}  // extern "C"

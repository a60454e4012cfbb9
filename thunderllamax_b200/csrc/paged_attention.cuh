// What the forms of the paged attention share: arguments, the schedule, small device helpers.
#pragma once
#include <algorithm>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace tlx {

constexpr size_t kPagedErrBytes = 256;   // the workspace starts with the device error word
constexpr int kRowsMax = 16;             // query rows per KV head of the rows form

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
  int rows_limit;        // requests with 1 .. rows_limit query rows per KV head: the rows form
  float* part;           // [2 CTAs][rows][head_dim] unnormalised rows of split items
  float2* ml;            // [2 CTAs][rows] (max, sum)
  int4* desc;            // split items: {slot of the first piece, last CTA, request << 10 | KV head, tile}
  int by_item;           // desc is indexed by item (request * kv_heads + head), else by first CTA
};

// ------------------------------------------------------------------- schedule
// A request as the kernels see it.
struct Req {
  int q0, n;       // first row, new tokens (at most max_new)
  int n_all;       // new tokens as planned: row t sees keys < kv - n_all + t + 1
  int kv;          // planned length
  int keys;        // keys the table can hold of it
};
__device__ __forceinline__ Req get_req(const AttnArgs& a, int b) {
  Req r;
  r.q0 = min(max(a.q_start[b], 0), a.n_tokens);
  const int e = min(max(a.q_start[b + 1], r.q0), a.n_tokens);
  r.n_all = e - r.q0;
  r.n = min(r.n_all, a.max_new);
  r.kv = a.kv_len[b];
  r.keys = static_cast<int>(min(static_cast<int64_t>(max(r.kv, 0)), static_cast<int64_t>(a.width) << a.shift));
  return r;
}

// Work is dealt in a row of positions in which every item takes kItemCost positions (its
// Q load, its rows' end) and then one for each unit.  A CTA has the units whose positions
// lie in its range; both neighbours of a boundary find the same one.
//
// units of an item of the rows form (an item without keys is one unit, which writes zeros)
template <int KT>
__device__ __forceinline__ int rows_units(const AttnArgs& a, const Req& r) {
  if (r.n < 1 || r.n * static_cast<int64_t>(a.group) > a.rows_limit) return 0;
  return max(1, (r.keys + KT - 1) / KT);
}

__device__ __forceinline__ int64_t range_start(int64_t units, int cta, int ctas) { return units * cta / ctas; }
// the CTA whose range holds unit u
__device__ __forceinline__ int range_of(int64_t units, int64_t u, int ctas) {
  int c = static_cast<int>(u * ctas / units);
  while (c + 1 < ctas && range_start(units, c + 1, ctas) <= u) ++c;
  return c;
}

// All positions, and the request (with the position inside it) at which this CTA's range starts.
// Every thread of the block calls it; THREADS = blockDim.x; scratch: 8-byte aligned shared
// memory of THREADS / 4 + 16 bytes, free again after the block's next barrier.
struct Start {
  int64_t units, u0, u1;   // all positions, this CTA's range
  int64_t local;           // its start inside request b
  int b;
  int ctas;                // CTAs that have a range
};
template <int THREADS, typename F>
__device__ __forceinline__ Start find_start(const AttnArgs& a, void* scratch, F units_of) {
  volatile int64_t* tot = static_cast<int64_t*>(scratch);
  volatile int64_t& s_local = tot[THREADS / 32];
  volatile int64_t& s_b = tot[THREADS / 32 + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t sum = 0;
  for (int b = tid; b < a.n_req; b += THREADS) sum += units_of(b);
  int64_t incl = sum;   // (units_of: positions of a request)
  if (tid == 0) s_b = -1;
  auto scan = [&](int64_t v, int64_t& all) -> int64_t {   // inclusive scan over the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    if (lane == 31) tot[warp] = v;
    __syncthreads();
    int64_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += tot[w];
      all += tot[w];
    }
    return v + before;
  };
  Start s;
  incl = scan(sum, s.units);
  s.ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), s.units));
  const bool works = static_cast<int>(blockIdx.x) < s.ctas;
  s.u0 = works ? range_start(s.units, blockIdx.x, s.ctas) : s.units;
  s.u1 = works ? range_start(s.units, blockIdx.x + 1, s.ctas) : s.units;
  if (a.n_req <= THREADS) {
    if (incl - sum <= s.u0 && s.u0 < incl) {
      s_b = tid;
      s_local = s.u0 - (incl - sum);
    }
  } else {
    int64_t base = 0;
    for (int r0 = 0; r0 < a.n_req; r0 += THREADS) {
      const int b = r0 + tid;
      const int64_t u = b < a.n_req ? units_of(b) : 0;
      int64_t all;
      __syncthreads();
      const int64_t i = base + scan(u, all);
      if (i - u <= s.u0 && s.u0 < i) {
        s_b = b;
        s_local = s.u0 - (i - u);
      }
      base += all;
      if (base > s.u0) break;   // the same for every thread
    }
  }
  __syncthreads();
  s.b = static_cast<int>(s_b);
  s.local = s_local;
  return s;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, bool ok) {
  if constexpr (N == 16) cp_async16(dst, src, ok);
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(N), "r"(ok ? N : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }

// shared loads from 32-bit addresses
__device__ __forceinline__ uint4 ls128(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p));
  return v;
}
__device__ __forceinline__ void st128(uint32_t p, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(p), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint2 ls64(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(p));
  return v;
}
__device__ __forceinline__ uint32_t ls32(uint32_t p) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(p));
  return v;
}
__device__ __forceinline__ uint32_t ls16(uint32_t p) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(v) : "r"(p));
  return v;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
  else
    mma16816(d, x, b0, b1);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return h2_bits(__floats2half2_rn(lo, hi));
  }
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  else return __half22float2(bits_h2(w));
}
// v * sigmoid(g).  The reciprocal keeps subnormal results (the fast division is 0, or NaN for an
// infinite v, where 1 + e^-g passes 2^126: g below -87.3).
__device__ __forceinline__ float gated(float v, float g) {
  float s;
  asm("rcp.approx.f32 %0, %1;\n" : "=f"(s) : "f"(1.f + __expf(-g)));
  return v * s;
}
// codes (q + 128) of bytes sel of w -> fp16x2 of fp16(q) * s, rounded once
__device__ __forceinline__ uint32_t dq2(uint32_t w, uint32_t sel, uint32_t s2) {
  return hmul2_u(h2_bits(__hsub2(bits_h2(prmt(w, 0x64646464u, sel)), __float2half2_rn(1152.f))), s2);
}
// a half of w is infinite or NaN
template <bool BF>
__device__ __forceinline__ bool bad16(uint32_t w) {
  constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

// takes infinite and NaN halves out of w; whether there was one
template <bool BF>
__device__ __forceinline__ bool drop_bad(uint32_t& w) {
  constexpr uint32_t e = BF ? 0x7F80u : 0x7C00u;
  const bool lo = (w & e) == e, hi = (w & (e << 16)) == (e << 16);
  w &= (lo ? 0xFFFF0000u : 0xFFFFFFFFu) & (hi ? 0x0000FFFFu : 0xFFFFFFFFu);
  return lo || hi;
}

// ---------------------------------------------------------------- host side
// Each form launches its kernel and says what it may have split: `items` descriptors in its
// area of the workspace, at most `rows` query rows of an item (row_slots in the buffers).
struct SplitSet {
  float* part;
  float2* ml;
  int4* desc;
  int by_item, row_slots, items, rows;
};
// split-item area: descriptors, (max, sum) and partial rows of `ctas` CTAs
struct Split {
  size_t ml, part, end;
};
inline Split split_area(int ctas, int rows, int hd) {
  Split s;
  s.ml = (static_cast<size_t>(ctas) * sizeof(int4) + 255) & ~size_t(255);
  s.part = s.ml + ((static_cast<size_t>(ctas) * 2 * rows * sizeof(float2) + 255) & ~size_t(255));
  s.end = s.part + static_cast<size_t>(ctas) * 2 * rows * hd * sizeof(float);
  return s;
}
inline SplitSet set_split(AttnArgs& a, void* area, int ctas, int row_slots) {
  const Split s = split_area(ctas, row_slots, a.c.head_dim);
  uint8_t* p = static_cast<uint8_t*>(area);
  a.desc = reinterpret_cast<int4*>(p);
  a.ml = reinterpret_cast<float2*>(p + s.ml);
  a.part = reinterpret_cast<float*>(p + s.part);
  return SplitSet{a.part, a.ml, a.desc, a.by_item, row_slots, 0, 0};
}
int launch_paged_rows(const AttnArgs& a, int ct, void* area, int sms, cudaStream_t stream, SplitSet* set);
// after_rows: the rows form's kernel was launched just before and may still run
int launch_paged_tiles(const AttnArgs& a, int ct, void* area, uint32_t* err, int sms, bool after_rows, cudaStream_t stream,
                       SplitSet* set);
size_t paged_rows_bytes(int hd, int sms);    // workspace of a form, a multiple of 256
size_t paged_tiles_bytes(int hd, int sms);

}  // namespace tlx

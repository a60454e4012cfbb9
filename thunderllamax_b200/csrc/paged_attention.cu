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
#include <cuda.h>

#include <algorithm>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace tlx {
namespace {

constexpr size_t kErrBytes = 256;   // the workspace starts with the device error word
constexpr int kRowsMax = 16;        // query rows per KV head of the rows form
constexpr int kMaxPieces = 1024;    // CTAs of a launch at most

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

// units of a request in the rows form: kv_heads items of the same keys (an item without
// keys is one unit, which writes zeros)
template <int KT>
__device__ __forceinline__ int rows_units(const AttnArgs& a, const Req& r) {
  if (r.n < 1 || r.n * static_cast<int64_t>(a.group) > a.rows_limit) return 0;
  return max(1, (r.keys + KT - 1) / KT) * a.c.kv_heads;
}

__device__ __forceinline__ int64_t range_start(int64_t units, int cta, int ctas) { return units * cta / ctas; }
// the CTA whose range holds unit u
__device__ __forceinline__ int range_of(int64_t units, int64_t u, int ctas) {
  int c = static_cast<int>(u * ctas / units);
  while (c + 1 < ctas && range_start(units, c + 1, ctas) <= u) ++c;
  return c;
}

// Total units and the request (with the unit inside it) at which this CTA's range starts.
// Every thread of the block calls it; THREADS = blockDim.x; scratch: 8-byte aligned shared
// memory of THREADS / 4 + 16 bytes, free again after the block's next barrier.
struct Start {
  int64_t units, u0, u1;
  int64_t local;   // unit inside request b
  int b;
  int ctas;        // CTAs that have a unit: an item's pieces are consecutive ones
};
template <int THREADS, typename F>
__device__ __forceinline__ Start find_start(const AttnArgs& a, void* scratch, F units_of) {
  volatile int64_t* tot = static_cast<int64_t*>(scratch);
  volatile int64_t& s_local = tot[THREADS / 32];
  volatile int64_t& s_b = tot[THREADS / 32 + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t sum = 0;
  for (int b = tid; b < a.n_req; b += THREADS) sum += units_of(b);
  int64_t incl = sum;
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

// ------------------------------------------------------------------ rows form
// A CTA of four warps takes a unit of KT keys at a time.  The keys are split over the
// warps for S = Q K^T (m16n8k16: 16 rows x 8 keys) and the dims for O += P V, so no sum
// crosses warps; per unit the row maxima and P go through shared memory (two barriers).
// K and V rows come in by 16-byte asynchronous copies, kStages units deep, each warp
// loading its own keys.  The k order of a matrix product is free, so a lane takes 16
// contiguous bytes of its key's row as the B fragments of 2 (16-bit) or 4 (int8) steps,
// and Q is loaded in the same order.  int8 codes become fp16(code - 128) * scale, rounded
// once, in registers.
template <int CT, int HD>
struct RowsCfg {
  static constexpr bool kQ8 = CT == CT_Q8;
  static constexpr int kKeys = (!kQ8 && HD == 256) ? 32 : 64;
  static constexpr int kRow = HD * (kQ8 ? 1 : 2);              // bytes of a cached row
  static constexpr int kScaleRow = kQ8 ? HD / 16 : 0;          // bytes of a row of scales
  static constexpr int kStage = kKeys * 2 * (kRow + kScaleRow);
  static constexpr int kStages = kStage >= 32768 ? 2 : 3;
  static constexpr int kPPitch = kKeys * 2 + 16;
  static constexpr int kSmem = kStages * kStage + 16 * kPPitch + 4 * 16 * 8;
  static constexpr int kCtas = 228 * 1024 / (kSmem + 1024) > 4 ? 4 : 228 * 1024 / (kSmem + 1024);
};

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

template <int CT, int HD>
__global__ void __launch_bounds__(128, RowsCfg<CT, HD>::kCtas) paged_rows_kernel(const __grid_constant__ AttnArgs a) {
  using C = RowsCfg<CT, HD>;
  constexpr bool BF = CT == CT_BF16, Q8 = C::kQ8;
  constexpr int KT = C::kKeys, KW = KT / 4, NB = KW / 8;   // keys of a unit, of a warp, its 8-key blocks
  constexpr int CPR = C::kRow / 16;                        // 16-byte chunks of a row
  constexpr int DW = HD / 4, DB = DW / 8;                  // dims of a warp, its 8-dim blocks
  constexpr int KS = HD / 16;                              // k steps of S
  constexpr uint32_t kOffV = KT * C::kRow, kOffKs = 2 * KT * C::kRow, kOffVs = kOffKs + KT * C::kScaleRow;
  extern __shared__ __align__(128) uint8_t sm[];
  uint8_t* psm = sm + C::kStages * C::kStage;
  float* smax = reinterpret_cast<float*>(psm + 16 * C::kPPitch);   // [4][16]
  float* ssum = smax + 64;                                          // [4][16]
  const uint32_t sbase = smem_u32(sm), pbase = smem_u32(psm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;

  griddep_launch_dependents();
  const Start st = find_start<128>(a, psm, [&](int b) { return static_cast<int64_t>(rows_units<KT>(a, get_req(a, b))); });
  if (!a.by_item && tid == 0) a.desc[blockIdx.x] = make_int4(-1, -1, 0, 0);
  const int n_units = static_cast<int>(st.u1 - st.u0);
  if (n_units == 0) return;

  // position in the row of units: request, KV head, unit of the item
  struct Pos {
    int b, head, u, of;
    Req r;
  };
  auto seek = [&](Pos& p, int b, int64_t local) {
    p.b = b;
    p.r = get_req(a, b);
    p.of = max(1, (p.r.keys + KT - 1) / KT);
    p.head = static_cast<int>(local / p.of);
    p.u = static_cast<int>(local % p.of);
  };
  auto advance = [&](Pos& p) {
    if (++p.u < p.of) return;
    p.u = 0;
    if (++p.head < a.c.kv_heads) return;
    p.head = 0;
    do {
      if (++p.b >= a.n_req) return;
      p.r = get_req(a, p.b);
    } while (rows_units<KT>(a, p.r) == 0);
    p.of = max(1, (p.r.keys + KT - 1) / KT);
  };

  const uint8_t* kbase = static_cast<const uint8_t*>(a.c.k);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.c.v);
  constexpr int ESZ = Q8 ? 1 : 2;
  auto load_unit = [&](const Pos& p, int stage) {
    // lane l < KW finds the rows of key l of this warp
    const int key = p.u * KT + warp * KW + (lane & (KW - 1));
    int64_t ko = 0, vo = 0, kso = 0, vso = 0;
    bool ok = key < p.r.keys;
    if (ok) {
      const int page = a.table[p.b * a.table_ld + (key >> a.shift)];
      ok = page >= 0 && page < a.c.pages;
      if (ok) {
        const int64_t in = key & (a.c.page_size - 1);
        ko = (page * a.c.k_stride[0] + p.head * a.c.k_stride[1] + in * a.c.k_stride[2]) * ESZ;
        vo = (page * a.c.v_stride[0] + p.head * a.c.v_stride[1] + in * a.c.v_stride[2]) * ESZ;
        if constexpr (Q8) {
          kso = (page * a.c.ks_stride[0] + p.head * a.c.ks_stride[1] + in * a.c.ks_stride[2]) * 2;
          vso = (page * a.c.vs_stride[0] + p.head * a.c.vs_stride[1] + in * a.c.vs_stride[2]) * 2;
        }
      }
    }
    const uint32_t okm = __ballot_sync(0xffffffffu, ok);
    const uint32_t sb = sbase + stage * C::kStage;
#pragma unroll
    for (int i = 0; i < KW * CPR / 32; ++i) {
      const int idx = lane + 32 * i, kk = idx / CPR, ch = idx % CPR;
      const int row = warp * KW + kk;
      const int64_t kro = __shfl_sync(0xffffffffu, ko, kk), vro = __shfl_sync(0xffffffffu, vo, kk);
      const bool valid = (okm >> kk) & 1;
      // swizzles: the reads below touch all banks once (see there)
      const int kch = (Q8 && HD == 64) ? ch : ch ^ ((row & 1) << 2);
      const int vch = Q8 ? (HD == 64 ? ch ^ ((row >> 1) & 3) : ch ^ (((row >> 1) & 3) << 1)) : ch ^ (row & 7);
      cp_async16(sb + row * C::kRow + kch * 16, kbase + kro + ch * 16, valid);
      cp_async16(sb + kOffV + row * C::kRow + vch * 16, vbase + vro + ch * 16, valid);
    }
    if constexpr (Q8) {
      if (lane < KW) {
        const int row = warp * KW + lane;
        cp_async_small<C::kScaleRow>(sb + kOffKs + row * C::kScaleRow, static_cast<const uint8_t*>(a.c.k_scale) + kso, ok);
        cp_async_small<C::kScaleRow>(sb + kOffVs + row * C::kScaleRow, static_cast<const uint8_t*>(a.c.v_scale) + vso, ok);
      }
    }
  };

  Pos load_at, at;
  seek(load_at, st.b, st.local);
  at = load_at;
  int loaded = 0;
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) {
    if (loaded < n_units) {
      load_unit(load_at, loaded % C::kStages);
      if (++loaded < n_units) advance(load_at);
    }
    cp_async_commit();
  }

  const float sc = a.scale * 1.4426950408889634f;
  uint32_t qf[KS][4];   // Q in fragment order
  float o[DB][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  int lim0 = 0, lim1 = 0;   // keys that rows g and g + 8 see
  bool first = true;        // the next unit starts an item (or this CTA's part of one)
  for (int i = 0; i < n_units; ++i) {
    const int stage = i % C::kStages;
    if (first) {
      first = false;
      const int rows = at.r.n * a.group, t0 = g / a.group, t1 = (g + 8) / a.group;
      const int lim = at.r.kv - at.r.n_all;
      lim0 = g < rows ? min(at.r.keys, lim + t0 + 1) : 0;
      lim1 = g + 8 < rows ? min(at.r.keys, lim + t1 + 1) : 0;
      const uint16_t* qh = a.q + at.head * a.group * a.q_head;
      const uint16_t* r0 = qh + (at.r.q0 + t0) * a.q_tok + (g - t0 * a.group) * a.q_head;
      const uint16_t* r1 = qh + (at.r.q0 + t1) * a.q_tok + (g + 8 - t1 * a.group) * a.q_head;
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int j = 0; j < KS / 2; ++j) {   // two k steps per 16 bytes
        const int d = Q8 ? (j >> 1) * 64 + 16 * q + (j & 1) * 8 : j * 32 + 8 * q;
        const uint4 x0 = g < rows ? __ldg(reinterpret_cast<const uint4*>(r0 + d)) : zero;
        const uint4 x1 = g + 8 < rows ? __ldg(reinterpret_cast<const uint4*>(r1 + d)) : zero;
        qf[2 * j][0] = x0.x; qf[2 * j][2] = x0.y; qf[2 * j + 1][0] = x0.z; qf[2 * j + 1][2] = x0.w;
        qf[2 * j][1] = x1.x; qf[2 * j][3] = x1.y; qf[2 * j + 1][1] = x1.z; qf[2 * j + 1][3] = x1.w;
      }
#pragma unroll
      for (int j = 0; j < DB; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
    }
    cp_async_wait<C::kStages - 2>();
    __syncwarp();
    const uint8_t* kb = sm + stage * C::kStage;
    // S of this warp's keys.  K reads: 8 lanes of a phase are 2 keys x 4 chunks, the
    // swizzle puts the second key's chunks in the other half of the banks.
    float s[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = warp * KW + nb * 8 + g;
      float e[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if constexpr (Q8) {
        uint32_t sw[HD / 64];   // the row's scales, two groups a word
        const uint8_t* sp = kb + kOffKs + row * C::kScaleRow;
        if constexpr (HD == 256) {
          const uint4 v = lds128(sp);
          sw[0] = v.x; sw[1] = v.y; sw[2] = v.z; sw[3] = v.w;
        } else if constexpr (HD == 128) {
          const uint2 v = lds64(sp);
          sw[0] = v.x; sw[1] = v.y;
        } else {
          sw[0] = lds32(sp);
        }
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          const int ch = HD == 64 ? q : (4 * j + q) ^ ((row & 1) << 2);
          const uint4 v = lds128(kb + row * C::kRow + ch * 16);
          const uint32_t s2 = prmt(sw[j], sw[j], q >= 2 ? 0x3232u : 0x1010u);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int t = 0; t < 4; ++t) mma16<false>(e[t & 1], qf[4 * j + t], dq2(w[t], 0x5140u, s2), dq2(w[t], 0x7362u, s2));
        }
      } else {
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const uint4 v = lds128(kb + row * C::kRow + (((4 * j + q) ^ ((row & 1) << 2)) * 16));
          mma16<BF>(e[0], qf[2 * j], v.x, v.y);
          mma16<BF>(e[1], qf[2 * j + 1], v.z, v.w);
        }
      }
      // z = scale log2(e) s, -inf where the row does not see the key
      const int key = at.u * KT + warp * KW + nb * 8 + 2 * q;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float z = (e[0][c] + e[1][c]) * sc;
        s[nb][c] = key + (c & 1) < (c < 2 ? lim0 : lim1) ? z : -INFINITY;
      }
    }
    float x0 = s[0][0], x1 = s[0][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      x0 = fmaxf(x0, fmaxf(s[nb][0], s[nb][1]));
      x1 = fmaxf(x1, fmaxf(s[nb][2], s[nb][3]));
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
    }
    if (q == 0) {
      smax[warp * 16 + g] = x0;
      smax[warp * 16 + g + 8] = x1;
    }
    __syncthreads();   // maxima are in; the unit before this one has been read by all warps
    if (loaded < n_units) {
      load_unit(load_at, loaded % C::kStages);
      if (++loaded < n_units) advance(load_at);
    }
    cp_async_commit();
    float n0 = m0, n1 = m1;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      n0 = fmaxf(n0, smax[w * 16 + g]);
      n1 = fmaxf(n1, smax[w * 16 + g + 8]);
    }
    const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
    const float f0 = ex2_approx(m0 - b0), f1 = ex2_approx(m1 - b1);   // 0 for the first unit
    m0 = n0;
    m1 = n1;
    l0 *= f0;
    l1 *= f1;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t p0 = pack2<BF>(ex2_approx(s[nb][0] - b0), ex2_approx(s[nb][1] - b0));
      const uint32_t p1 = pack2<BF>(ex2_approx(s[nb][2] - b1), ex2_approx(s[nb][3] - b1));
      // the sum is taken over the rounded probabilities: what rounding does to all of a
      // row's weights alike cancels in the quotient
      const float2 r0 = unpack2<BF>(p0), r1 = unpack2<BF>(p1);
      l0 += r0.x + r0.y;
      l1 += r1.x + r1.y;
      uint8_t* dst = psm + g * C::kPPitch + (warp * KW + nb * 8 + 2 * q) * 2;
      *reinterpret_cast<uint32_t*>(dst) = p0;
      *reinterpret_cast<uint32_t*>(dst + 8 * C::kPPitch) = p1;
    }
    if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f)) {
#pragma unroll
      for (int j = 0; j < DB; ++j) {
        o[j][0] *= f0;
        o[j][1] *= f0;
        o[j][2] *= f1;
        o[j][3] *= f1;
      }
    }
    __syncthreads();   // P is in
    // O of this warp's dims
    const uint8_t* vb = kb + kOffV;
    // a key that some rows do not see must not reach them through 0 * inf or 0 * NaN
    const bool edge = at.r.n > 1 && (at.u + 1) * KT > at.r.kv - at.r.n_all;
    auto product = [&](int j, const uint32_t (&pf)[4], uint32_t v0, uint32_t v1, int k16) {
      if (edge && __any_sync(0xffffffffu, bad16<BF>(v0) || bad16<BF>(v1))) {
        const int key = at.u * KT + k16 * 16 + 2 * q;
        for (int t = 0; t < at.r.n; ++t) {   // each token's rows with the keys it sees
          const int lim = at.r.kv - at.r.n_all + t + 1;
          const uint32_t w0 = v0 & ((key < lim ? 0xFFFFu : 0u) | (key + 1 < lim ? 0xFFFF0000u : 0u));
          const uint32_t w1 = v1 & ((key + 8 < lim ? 0xFFFFu : 0u) | (key + 9 < lim ? 0xFFFF0000u : 0u));
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma16<BF>(d, pf, w0, w1);
          if (g / a.group == t) {
            o[j][0] += d[0];
            o[j][1] += d[1];
          }
          if ((g + 8) / a.group == t) {
            o[j][2] += d[2];
            o[j][3] += d[3];
          }
        }
      } else {
        mma16<BF>(o[j], pf, v0, v1);
      }
    };
#pragma unroll
    for (int k = 0; k < KT / 16; ++k) {
      uint32_t pf[4];
      ldsm4(pf, pbase + ((lane & 7) + ((lane >> 3) & 1) * 8) * C::kPPitch + (2 * k + (lane >> 4)) * 16);
      if constexpr (Q8) {
        // lane (g, q): keys 2q, 2q+1, 2q+8, 2q+9 and DB contiguous dims from DB g on
        uint32_t w[4][DB > 4 ? 2 : 1];
        uint32_t sh[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = k * 16 + 2 * q + (e & 1) + (e >> 1) * 8;
          const int byte = warp * DW + DB * g;
          const int ch = HD == 64 ? (byte >> 4) ^ ((row >> 1) & 3) : (byte >> 4) ^ (((row >> 1) & 3) << 1);
          const uint8_t* p = vb + row * C::kRow + ch * 16 + (byte & 15);
          if constexpr (DB == 8) {
            const uint2 v = lds64(p);
            w[e][0] = v.x;
            w[e][1] = v.y;
          } else if constexpr (DB == 4) {
            w[e][0] = lds32(p);
          } else {
            w[e][0] = *reinterpret_cast<const uint16_t*>(p);
          }
          sh[e] = *reinterpret_cast<const uint16_t*>(kb + kOffVs + row * C::kScaleRow + (byte >> 5) * 2);
        }
        const uint32_t s01 = prmt(sh[0], sh[1], 0x5410u), s23 = prmt(sh[2], sh[3], 0x5410u);
#pragma unroll
        for (int h = 0; h < (DB > 4 ? 2 : 1); ++h) {
          // (key 2q, key 2q+1) byte pairs of four dims
          const uint32_t a01 = prmt(w[0][h], w[1][h], 0x5140u), a23 = prmt(w[0][h], w[1][h], 0x7362u);
          const uint32_t c01 = prmt(w[2][h], w[3][h], 0x5140u), c23 = prmt(w[2][h], w[3][h], 0x7362u);
          const int j = 4 * h;
          product(j, pf, dq2(a01, 0x5140u, s01), dq2(c01, 0x5140u, s23), k);
          product(j + 1, pf, dq2(a01, 0x7362u, s01), dq2(c01, 0x7362u, s23), k);
          if constexpr (DB >= 4) {
            product(j + 2, pf, dq2(a23, 0x5140u, s01), dq2(c23, 0x5140u, s23), k);
            product(j + 3, pf, dq2(a23, 0x7362u, s01), dq2(c23, 0x7362u, s23), k);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < DB; j += 2) {
          const int row = k * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
          const int ch = (warp * DB + j + (lane >> 4)) ^ (row & 7);
          uint32_t v[4];
          ldsm4t(v, smem_u32(vb) + row * C::kRow + ch * 16);
          product(j, pf, v[0], v[1], k);
          product(j + 1, pf, v[2], v[3], k);
        }
      }
    }
    // the end of the item, or of this CTA's part of it
    if (at.u + 1 == at.of || i + 1 == n_units) {
      first = true;
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
      }
      if (q == 0) {
        ssum[warp * 16 + g] = l0;
        ssum[warp * 16 + g + 8] = l1;
      }
      __syncthreads();
      l0 = l1 = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        l0 += ssum[w * 16 + g];
        l1 += ssum[w * 16 + g + 8];
      }
      const int64_t begin = st.u0 + i - at.u, end = begin + at.of;   // the item's units
      const bool whole = begin >= st.u0 && end <= st.u1;
      const int rows = at.r.n * a.group;
      const int slot = 2 * blockIdx.x + (begin > st.u0 ? 1 : 0);   // a part that the CTA's range starts in, or a later one
      if (tid == 0) {
        const int64_t item = static_cast<int64_t>(at.b) * a.c.kv_heads + at.head;
        if (begin >= st.u0) {   // the item starts here: where its pieces are, if it is split
          const int4 d = make_int4(whole ? -1 : slot, whole ? -1 : range_of(st.units, end - 1, st.ctas), at.b << 10 | at.head, 0);
          if (a.by_item) a.desc[item] = d;
          else if (!whole) a.desc[blockIdx.x] = d;
        }
      }
      // columns of a lane: 16-bit 8j + 2q + {0, 1}; int8 (2q + {0, 1}) DB + j
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = g + 8 * half, t = row / a.group, hl = row - t * a.group;
        if (row >= rows) continue;
        const float l = half ? l1 : l0, m = half ? m1 : m0;
        if (!whole) {
          float* dst = a.part + (static_cast<int64_t>(slot) * 16 + row) * HD + warp * DW;
          if constexpr (Q8) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int j = 0; j < DB; j += 2)
                *reinterpret_cast<float2*>(dst + (2 * q + c) * DB + j) = make_float2(o[j][2 * half + c], o[j + 1][2 * half + c]);
          } else {
#pragma unroll
            for (int j = 0; j < DB; ++j)
              *reinterpret_cast<float2*>(dst + 8 * j + 2 * q) = make_float2(o[j][2 * half], o[j][2 * half + 1]);
          }
          if (warp == 0 && q == 0) a.ml[slot * 16 + row] = make_float2(m, l);
          continue;
        }
        const bool sees = (half ? lim1 : lim0) > 0;
        const float inv = 1.f / l;
        const int64_t tok = at.r.q0 + t;
        const int head = at.head * a.group + hl;
        uint16_t* dst = a.out + tok * a.o_tok + head * a.o_head + warp * DW;
        const uint16_t* gp = a.gate ? a.gate + tok * a.g_tok + head * a.g_head + warp * DW : nullptr;
        auto put2 = [&](int d, float v0, float v1) {
          v0 = sees ? v0 * inv : 0.f;
          v1 = sees ? v1 * inv : 0.f;
          if (gp) {
            const float2 x = unpack2<BF>(*reinterpret_cast<const uint32_t*>(gp + d));
            v0 /= 1.f + __expf(-x.x);
            v1 /= 1.f + __expf(-x.y);
          }
          *reinterpret_cast<uint32_t*>(dst + d) = pack2<BF>(v0, v1);
        };
        if constexpr (Q8) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < DB; j += 2) put2((2 * q + c) * DB + j, o[j][2 * half + c], o[j + 1][2 * half + c]);
        } else {
#pragma unroll
          for (int j = 0; j < DB; ++j) put2(8 * j + 2 * q, o[j][2 * half], o[j][2 * half + 1]);
        }
      }
    }
    if (i + 1 < n_units) advance(at);
  }
}

// ----------------------------------------------------------------- tiles form
// The 128 rows of a tensor-core tile are the query heads of one KV head times as many
// tokens as fit (row = token * group + head), so every key read serves the whole group.
// A CTA walks its units (64 keys of one item) on tcgen05:
//   S(i) = Q K_i^T   M = 128, N = 64, K = head_dim; Q in tensor memory (head_dim 256) or
//                    shared memory, S double-buffered in tensor memory
//   O += P(i) V_i    M = 128, N = head_dim, K = 64; V is the MN-major operand as it lies
//                    in the cache, P (16 bit) in shared memory, double-buffered
//   warps 0..3   softmax, one thread per row; O is rescaled (in tensor memory) only when a
//                row's maximum grows by more than 2^8, which keeps P in range
//   warp 4       one thread issues the MMAs, S(i + 1) ahead of O += P(i) V(i)
//   warp 5       loads the K and V halves of the units, in the order the MMAs read them:
//                one TMA box per page (and 64 dims), so pages may lie anywhere and what is
//                outside the pool reads as 0
//   warps 6..    16-bit caches: on the MMA thread's request take out of V what must not
//                reach the product (rows past the last key, and infinite or NaN values where
//                some rows do not see the unit whole); int8 caches: turn every half into
//                fp16(code * scale)
// Every wait is bounded: a timeout raises the error word, all roles leave, issued MMAs
// and copies are drained and tensor memory is freed.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(b))
      : "memory");
}
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity) {
  const bool ok = tc_wait(b, parity);
  __syncwarp();   // what follows is for the whole warp
  return ok;
}

template <int CT, int HD>
struct TilesCfg {
  static constexpr bool kQ8 = CT == CT_Q8;
  static constexpr int kKeys = 64;
  static constexpr int kHalf = kKeys * HD * 2;                  // bytes of a K or V half
  static constexpr bool kQTmem = HD == 256;
  static constexpr int kQBytes = kQTmem ? 0 : 128 * HD * 2;
  static constexpr int kPBytes = 128 * kKeys * 2;
  static constexpr int kPBufs = HD == 128 || (kQ8 && HD == 256) ? 1 : 2;
  // 16-bit halves of K or V that the MMAs read, and (int8) halves as they lie in the cache
  static constexpr int kRing = kQ8 ? (HD == 128 ? 2 : 4) : HD == 128 ? 4 : 6;
  static constexpr int kRaw = !kQ8 ? 0 : HD == 128 ? 3 : 4;
  static constexpr int kRawHalf = kKeys * HD;                   // codes; the scales follow
  static constexpr int kRawBytes = kRawHalf + kKeys * (HD / 16);
  static constexpr int kThreads = HD == 256 ? 384 : 256;
  static constexpr int kHelpers = kThreads / 32 - 6;            // warps
  static constexpr int kCtas = HD == 256 ? 1 : 2;               // on an SM
  static constexpr int kOffP = kRing * kHalf;
  static constexpr int kOffQ = kOffP + kPBufs * kPBytes;
  static constexpr int kOffRaw = kOffQ + kQBytes;
  static constexpr int kOffBar = kOffRaw + kRaw * kRawBytes;
  static constexpr int kSmem = kOffBar + 512;
  static constexpr uint32_t kTmem = HD == 256 ? 512 : 256;
  static constexpr uint32_t kColS = 0, kColO = 128;
  static constexpr uint32_t kColQ = kQTmem ? 384 : 0;
  static constexpr uint32_t kFmt = CT == CT_BF16 ? (1u << 7) | (1u << 10) : 0u;   // A, B bf16
  static constexpr uint32_t kIdescQK = (1u << 4) | kFmt | (64u >> 3) << 17 | (128u >> 4) << 24;
  static constexpr uint32_t kIdescPV = (1u << 4) | kFmt | (1u << 16) | static_cast<uint32_t>(HD >> 3) << 17 | (128u >> 4) << 24;
};

// sum over i < n of floor((a i + b) / m): the Euclid-like recursion, as a loop
__device__ __forceinline__ int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  int64_t s = 0;
  while (n > 0) {
    if (a >= m) {
      s += (n - 1) * n / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      s += n * (b / m);
      b %= m;
    }
    const int64_t y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const int64_t t = m;
    m = a;
    a = t;
  }
  return s;
}

__device__ __forceinline__ int tile_tokens(const AttnArgs& a) { return 128 / a.group; }
__device__ __forceinline__ int tile_count(const AttnArgs& a, const Req& r) {
  if (r.n < 1 || r.n * static_cast<int64_t>(a.group) <= a.rows_limit) return 0;
  return (r.n + tile_tokens(a) - 1) / tile_tokens(a);
}
// keys that the last token of the tile sees
__device__ __forceinline__ int tile_keys(const AttnArgs& a, const Req& r, int tile) {
  const int64_t last = min(static_cast<int64_t>(tile + 1) * tile_tokens(a), static_cast<int64_t>(r.n));
  return static_cast<int>(min(max(static_cast<int64_t>(r.kv) - r.n_all + last, static_cast<int64_t>(0)),
                              static_cast<int64_t>(r.keys)));
}
__device__ __forceinline__ int tile_units(const AttnArgs& a, const Req& r, int tile) {
  return max(1, (tile_keys(a, r, tile) + 63) >> 6);
}
// units of one KV head in the tiles before `tile`
__device__ __forceinline__ int64_t units_before(const AttnArgs& a, const Req& r, int tile) {
  const int64_t tt = tile_tokens(a), c = static_cast<int64_t>(r.kv) - r.n_all;
  const int full = min(tile, r.n / static_cast<int>(tt));   // tiles with all their tokens
  int64_t s = 0;
  int i = 0;
  if (c >= 0 && r.keys == r.kv) {   // ceil((c + (i + 1) tt) / 64), at least 1 since tt >= 1
    s = floor_sum(full, 64, tt, c + tt + 63);
    i = full;
  }
  for (; i < tile; ++i) s += tile_units(a, r, i);
  return s;
}

// The helpers replace infinite and NaN values of V by 0 in the units that some rows do
// not see whole (0 * inf in the product would reach those rows); this adds weight * value
// of such keys to the rows that do see them.  Called by whole warps with O at rest; the
// weights are the rounded ones of the product, from P in shared memory.
template <int CT, int HD>
__device__ __noinline__ void restore_bad_values(const AttnArgs& a, int b, int head, int k0, int keys, int lim,
                                                const uint8_t* p_buf, int row, uint32_t o_tmem) {
  constexpr bool BF = CT == CT_BF16;
  for (int c = 0; c < HD / 32; ++c) {
    uint32_t r[32];
    tc_ld32(o_tmem + c * 32, r);
    tc_wait_ld();
    for (int j = 0; j < 64 && k0 + j < keys; ++j) {
      const int key = k0 + j;
      const int page = a.table[b * a.table_ld + (key >> a.shift)];
      if (page < 0 || page >= a.c.pages) continue;
      const int64_t in = key & (a.c.page_size - 1);
      const int64_t at = page * a.c.v_stride[0] + head * a.c.v_stride[1] + in * a.c.v_stride[2] + c * 32;
      const float p = unpack2<BF>(*reinterpret_cast<const uint16_t*>(p_buf + sw128(row, j >> 3) + (j & 7) * 2)).x;
#pragma unroll
      for (int x = 0; x < 32; ++x) {
        uint32_t v;
        if constexpr (CT == CT_Q8) {
          const uint32_t s = static_cast<const uint16_t*>(
              a.c.v_scale)[page * a.c.vs_stride[0] + head * a.c.vs_stride[1] + in * a.c.vs_stride[2] + c];
          v = dq2(static_cast<const uint8_t*>(a.c.v)[at + x], 0x4040u, s | s << 16) & 0xFFFFu;
        } else {
          v = static_cast<const uint16_t*>(a.c.v)[at + x];
        }
        if (bad16<BF>(v) && key < lim) r[x] = __float_as_uint(__uint_as_float(r[x]) + p * unpack2<BF>(v).x);
      }
    }
    __syncwarp();
    tc_st32(o_tmem + c * 32, r);
    tc_wait_st();
  }
}

template <int CT, int HD>
__global__ void __launch_bounds__(TilesCfg<CT, HD>::kThreads, TilesCfg<CT, HD>::kCtas)
    paged_tiles_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map, uint32_t* err) {
  using C = TilesCfg<CT, HD>;
  constexpr bool BF = CT == CT_BF16, Q8 = C::kQ8;
  static_assert(C::kColO + HD + (C::kQTmem ? C::kColQ - 384 + HD / 2 : 0) <= C::kTmem, "tensor memory");
  constexpr int NH = C::kHelpers, RING = C::kRing, PB = C::kPBufs;
  extern __shared__ __align__(1024) uint8_t sm_tiles[];
  uint8_t* const sm = sm_tiles;
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + C::kOffBar);
  uint64_t* landed = bar;               // [8] TMA -> MMA or helpers
  uint64_t* raw_free = landed + 8;      // [RAW] helpers -> loader
  uint64_t* full = raw_free + 8;        // [RING] helpers -> MMA
  uint64_t* empty = full + 8;           // [RING] MMA -> loader or helpers
  uint64_t* s_full = empty + 8;         // [2] MMA -> softmax
  uint64_t* s_free = s_full + 2;        // [2] softmax -> MMA
  uint64_t* p_full = s_free + 2;        // [2] softmax -> MMA
  uint64_t* pv_done = p_full + 2;       // [2] MMA -> softmax
  uint64_t* q_full = pv_done + 2;       // softmax -> MMA: Q of the next item is in
  uint64_t* o_free = q_full + 1;        // softmax -> MMA: O of the last item is read
  uint64_t* fix_req = o_free + 1;       // MMA -> helpers: a V half to clean
  uint64_t* fix_done = fix_req + 1;     // helpers -> MMA
  uint64_t* done = fix_done + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  // [8] by unit: unit + 1 if the helpers took a bad value out of its V (they are fewer than
  // 8 units ahead of the softmax)
  volatile int* bad = reinterpret_cast<int*>(tmem_holder + 2);
  struct First {
    int tile, head, u;
  };
  First* first_at = reinterpret_cast<First*>(tmem_holder + 10);
  struct Fix {
    int slot, valid, edge, unit;   // ring slot (-1: no more), keys of the unit that exist
  };
  Fix* fix = reinterpret_cast<Fix*>(tmem_holder + 14);
  static_assert((4 * 8 + 13) * 8 + 14 * 4 + sizeof(Fix) <= 512 && RING <= 8 && C::kRaw <= 8, "barrier area");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_launch_dependents();
  const Start st = find_start<C::kThreads>(a, sm + C::kOffP, [&](int b) -> int64_t {
    const Req r = get_req(a, b);
    const int tiles = tile_count(a, r);
    return tiles ? units_before(a, r, tiles) * a.c.kv_heads : 0;
  });
  if (tid == 0) a.desc[blockIdx.x] = make_int4(-1, -1, 0, 0);
  const int n = static_cast<int>(st.u1 - st.u0);
  if (n == 0) return;
  const uint32_t sbase = smem_u32(sm);
  if (sbase & 1023u) {   // the descriptors need the swizzle atoms' alignment
    if (tid == 0) atomicOr(err, ERR_BAD_PARAM);
    return;
  }
  if (warp == 0) {   // the tile, head and unit at which the range starts: a 32-way search
    const Req r = get_req(a, st.b);
    int lo = 0, hi = tile_count(a, r);   // units_before(lo) * heads <= local < units_before(hi) * heads
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, t = min(lo + lane * step, hi);
      const bool le = t < hi && units_before(a, r, t) * a.c.kv_heads <= st.local;
      const int k = 31 - __clz(__ballot_sync(0xffffffffu, le));   // lane 0 always holds
      const int nlo = lo + k * step;
      hi = min(hi, nlo + step);
      lo = nlo;
    }
    if (lane == 0) {
      const int64_t rest = st.local - units_before(a, r, lo) * a.c.kv_heads;
      const int of = tile_units(a, r, lo);
      *first_at = First{lo, static_cast<int>(rest / of), static_cast<int>(rest % of)};
    }
  }
  if (tid == 0) {
    for (int i = 0; i < 8; ++i) {
      mbar_init(&landed[i], Q8 ? 33 : 1);   // int8: 32 lanes' copies of the scales as well
      mbar_init(&raw_free[i], NH);
      mbar_init(&full[i], NH);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 8; ++i) bad[i] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, 4);
    mbar_init(o_free, 4);
    mbar_init(fix_req, 1);
    mbar_init(fix_done, NH);
    mbar_init(done, 1);
    *abort_flag = 0u;
    mbar_fence_init();
  }
  if (warp == 4) tc_alloc(tmem_holder, C::kTmem);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_holder;
  auto fail = [&]() {
    atomicOr(err, ERR_MBAR_TIMEOUT);
    *abort_flag = 1u;
  };

  struct Pos {
    int b, tile, head, u, of, tiles;
    Req r;
  };
  Pos at;
  at.b = st.b;
  at.r = get_req(a, st.b);
  at.tiles = tile_count(a, at.r);
  at.tile = first_at->tile;
  at.head = first_at->head;
  at.u = first_at->u;
  at.of = tile_units(a, at.r, at.tile);
  // the next item (not called past the last unit of the launch)
  auto next_item = [&](Pos& p) {
    p.u = 0;
    if (++p.head == a.c.kv_heads) {
      p.head = 0;
      if (++p.tile == p.tiles) {
        p.tile = 0;
        do {
          if (++p.b >= a.n_req) return;
          p.r = get_req(a, p.b);
          p.tiles = tile_count(a, p.r);
        } while (p.tiles == 0);
      }
      p.of = tile_units(a, p.r, p.tile);
    }
  };

  // V of a unit that some row of the tile does not see whole, and the keys it really has
  auto is_edge = [&](const Pos& p) {
    return max(0, min(p.r.keys, p.r.kv - p.r.n_all + p.tile * tile_tokens(a) + 1)) < min(p.u * 64 + 64, p.r.keys);
  };
  auto is_special = [&](const Pos& p) { return p.u * 64 + 64 > p.r.keys || is_edge(p); };

  if (warp == 4) {
    // --------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      int h = 0;               // ring halves consumed
      int fixes = 0;           // 16-bit: V halves the helpers were asked to clean
      int item = 0, left = min(at.of - at.u, n);   // units left of the current item
      auto issue_qk = [&](int i, bool starts, int it) -> bool {
        const int b = i & 1, slot = h % RING;
        if (starts && !tc_wait(q_full, it & 1)) return false;
        if (!tc_wait(Q8 ? &full[slot] : &landed[slot], (h / RING) & 1) || !tc_wait(&s_free[b], ((i >> 1) & 1) ^ 1))
          return false;
        tc_after();
        const uint32_t kb = sbase + slot * C::kHalf;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
          const uint64_t bd = sw128_desc(kb + (s >> 2) * 8192 + (s & 3) * 32);
          if constexpr (C::kQTmem)
            tc_mma_ts(tmem + C::kColS + b * 64, tmem + C::kColQ + s * 8, bd, C::kIdescQK, s > 0 ? 1u : 0u);
          else
            tc_mma(tmem + C::kColS + b * 64, sw128_desc(sbase + C::kOffQ + (s >> 2) * 16384 + (s & 3) * 32), bd,
                   C::kIdescQK, s > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[b]);
        tc_commit(&empty[slot]);
        ++h;
        return true;
      };
      auto issue_pv = [&](int i, bool starts, int it) -> bool {
        const int slot = h % RING, pb = PB == 2 ? i & 1 : 0;
        if (starts && it > 0 && !tc_wait(o_free, (it - 1) & 1)) return false;
        if (!tc_wait(Q8 ? &full[slot] : &landed[slot], (h / RING) & 1)) return false;
        if (!Q8 && is_special(at)) {
          *fix = Fix{slot, at.r.keys - at.u * 64, is_edge(at), i};
          mbar_arrive(fix_req);
          if (!tc_wait(fix_done, fixes++ & 1)) return false;
        }
        if (!tc_wait(&p_full[i & 1], (i >> 1) & 1)) return false;
        tc_after();
        const uint32_t vb = sbase + slot * C::kHalf;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          tc_mma(tmem + C::kColO, sw128_desc(sbase + C::kOffP + pb * C::kPBytes + kk * 32),
                 sw128_desc_mn(vb + kk * 2048, 8192), C::kIdescPV, (!starts || kk > 0) ? 1u : 0u);
        tc_commit(&pv_done[i & 1]);
        tc_commit(&empty[slot]);
        ++h;
        return true;
      };
      bool ok = issue_qk(0, true, 0), starts = true;
      for (int i = 0; i < n && ok && !*abort_flag; ++i) {
        const bool ends = --left == 0;
        if (!ends && i + 1 < n) ok = issue_qk(i + 1, false, item);
        ok = ok && issue_pv(i, starts, item);
        ++at.u;
        starts = ends;
        if (ends && i + 1 < n) {
          next_item(at);
          left = at.of;
          ++item;
          ok = ok && issue_qk(i + 1, true, item);
        }
      }
      if (!ok) fail();
      if constexpr (!Q8) {
        fix->slot = -1;
        mbar_arrive(fix_req);
      }
      tc_commit(done);   // every issued MMA has completed before tensor memory is released
      if (!tc_wait(done, 0)) fail();
    }
  } else if (warp < 4) {
    // ----------------------------------------------------------------- softmax
    const int row = warp * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const float sc = a.scale * 1.4426950408889634f;
    const int tt = tile_tokens(a), t_in = row / a.group, hl = row - t_in * a.group;
    bool ok = true;
    auto load_q = [&](const Pos& p) {   // this row of Q (zero past the last row)
      const int t = p.tile * tt + t_in;
      const bool valid = t_in < tt && t < p.r.n;
      const uint4* src = reinterpret_cast<const uint4*>(a.q + static_cast<int64_t>(p.r.q0 + t) * a.q_tok +
                                                        (p.head * a.group + hl) * a.q_head);
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 v = valid ? __ldg(src + c * 4 + j) : make_uint4(0u, 0u, 0u, 0u);
          if constexpr (C::kQTmem) {
            w[4 * j] = v.x;
            w[4 * j + 1] = v.y;
            w[4 * j + 2] = v.z;
            w[4 * j + 3] = v.w;
          } else {
            const int ch = c * 4 + j;
            *reinterpret_cast<uint4*>(sm + C::kOffQ + (ch >> 3) * 16384 + sw128(row, ch & 7)) = v;
          }
        }
        if constexpr (C::kQTmem) tc_st16(tmem + lanes + C::kColQ + c * 16, w);
      }
      if constexpr (C::kQTmem) {
        tc_wait_st();
        tc_before();
      } else {
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    };
    load_q(at);
    int i = 0;
    while (i < n && ok && !*abort_flag) {
      // one item, or this CTA's part of it
      const int count = min(at.of - at.u, n - i);
      const int t = at.tile * tt + t_in;
      const bool valid = t_in < tt && t < at.r.n;
      const int lim = valid ? max(0, min(at.r.keys, at.r.kv - at.r.n_all + t + 1)) : 0;   // keys < lim
      const int lim_first = max(0, min(at.r.keys, at.r.kv - at.r.n_all + at.tile * tt + 1));
      const bool any = __any_sync(0xffffffffu, valid);   // a warp without rows only keeps the barriers going
      float m_ref = -INFINITY, l_run = 0.f;
      Pos next = at;
      for (int k = 0; k < count && ok; ++k, ++i) {
        const int b = i & 1, pb = PB == 2 ? b : 0;
        if (!(ok = warp_wait(&s_full[b], (i >> 1) & 1))) break;
        tc_after();
        float s[64];
        if (any) {
          uint32_t r0[32], r1[32];
          tc_ld32(tmem + lanes + C::kColS + b * 64, r0);
          tc_ld32(tmem + lanes + C::kColS + b * 64 + 32, r1);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            s[j] = __uint_as_float(r0[j]) * sc;
            s[32 + j] = __uint_as_float(r1[j]) * sc;
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[b]);
        const int k0 = (at.u + k) * 64;
        float off = 0.f;
        if (any) {
          const int rem = lim - k0;
          if (__any_sync(0xffffffffu, rem < 64)) {
#pragma unroll
            for (int j = 0; j < 64; ++j) s[j] = j < rem ? s[j] : -INFINITY;
          }
          float mx[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) mx[j] = s[j];
#pragma unroll
          for (int j = 8; j < 64; ++j) mx[j & 7] = fmaxf(mx[j & 7], s[j]);
          const float mt = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                 fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
          const bool grows = mt > m_ref + 8.f || (m_ref == -INFINITY && mt > -INFINITY);
          if (__any_sync(0xffffffffu, grows)) {
            const float m_new = grows ? mt : m_ref;
            const float cor = m_ref == m_new ? 1.f : ex2_approx(m_ref - m_new);
            if (k > 0) {
              if (!(ok = warp_wait(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1))) break;   // O is at rest
              tc_after();
              l_run *= cor;
#pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t r[32];
                tc_ld32(tmem + lanes + C::kColO + c * 32, r);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * cor);
                tc_st32(tmem + lanes + C::kColO + c * 32, r);
              }
              tc_wait_st();
            }
            m_ref = m_new;
          }
          off = m_ref == -INFINITY ? 0.f : m_ref;
        }
        // the P buffer is free once the product that read it is done
        if (i >= PB && !(ok = warp_wait(&pv_done[(i - PB) & 1], ((i - PB) >> 1) & 1))) break;
        if (any) {
          float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              w[j] = pack2<BF>(ex2_approx(s[8 * c + 2 * j] - off), ex2_approx(s[8 * c + 2 * j + 1] - off));
              const float2 p = unpack2<BF>(w[j]);   // the rounded weights are summed: see the rows form
              sums[j] += p.x + p.y;
            }
            *reinterpret_cast<uint4*>(sm + C::kOffP + pb * C::kPBytes + sw128(row, c)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          l_run += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        }
        fence_proxy_async_smem();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
        // Q of the next item may follow once every S of this one is read
        if (k + 1 == count && i + 1 < n) {
          next_item(next);
          load_q(next);
        }
        // bad values that the producers took out of V, for the rows that see them
        if (any && lim_first < min(k0 + 64, at.r.keys)) {
          if (!(ok = warp_wait(&pv_done[b], (i >> 1) & 1))) break;
          tc_after();
          if (bad[i & 7] == i + 1)
            restore_bad_values<CT, HD>(a, at.b, at.head, k0, at.r.keys, lim, sm + C::kOffP + pb * C::kPBytes, row,
                                       tmem + lanes + C::kColO);
        }
      }
      if (!ok) break;
      // the item's rows, or this part's
      if (!(ok = warp_wait(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1))) break;
      tc_after();
      const int64_t begin = st.u0 + (i - count) - at.u, end = begin + at.of;   // the item's units
      const bool whole = begin >= st.u0 && end <= st.u1;
      const int slot = 2 * blockIdx.x + (begin > st.u0 ? 1 : 0);
      if (tid == 0 && begin >= st.u0 && !whole)
        a.desc[blockIdx.x] = make_int4(slot, range_of(st.units, end - 1, st.ctas), at.b << 10 | at.head, at.tile);
      if (any) {
        const bool sees = lim > 0;
        const float inv = 1.f / l_run;
        const int64_t tok = at.r.q0 + t;
        const int head = at.head * a.group + hl;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t r[32];
          tc_ld32(tmem + lanes + C::kColO + c * 32, r);
          tc_wait_ld();
          if (!valid) continue;
          if (!whole) {
            float4* dst = reinterpret_cast<float4*>(a.part + (static_cast<int64_t>(slot) * 128 + row) * HD + c * 32);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              dst[j] = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                                   __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
          } else {
            const uint4* gp = reinterpret_cast<const uint4*>(a.gate + tok * a.g_tok + head * a.g_head + c * 32);
            uint4* dst = reinterpret_cast<uint4*>(a.out + tok * a.o_tok + head * a.o_head + c * 32);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float v[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) v[x] = sees ? __uint_as_float(r[8 * j + x]) * inv : 0.f;
              if (a.gate) {
                const uint4 gv = __ldg(gp + j);
                const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const float2 y = unpack2<BF>(gw[x]);
                  v[2 * x] /= 1.f + __expf(-y.x);
                  v[2 * x + 1] /= 1.f + __expf(-y.y);
                }
              }
              dst[j] = make_uint4(pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3]), pack2<BF>(v[4], v[5]), pack2<BF>(v[6], v[7]));
            }
          }
        }
        if (!whole && valid) a.ml[slot * 128 + row] = make_float2(m_ref, l_run);
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      at = next;
    }
    if (!ok) fail();
  } else if (warp == 5) {
    // ------------------------------------------------------------------ loader
    // Halves in MMA order: per unit K(i) then V(i - 1), or V(i - 1) first where unit i
    // starts an item.  A lane owns one TMA box of a half: 64 dims (int8: all) of the keys
    // of one page.
    constexpr int ATOMS = Q8 ? 1 : HD / 64, LR = Q8 ? C::kRaw : RING;
    const int rows = min(a.c.page_size, 64), part = lane / ATOMS, atom = lane % ATOMS;
    const bool mine = part * rows < 64;
    auto page_of = [&](const Pos& p) -> int {   // -1: outside the pool, read as 0
      const int key = p.u * 64 + part * rows;
      return mine && key < p.r.keys ? a.table[p.b * a.table_ld + (key >> a.shift)] : -1;
    };
    int h = 0;
    bool ok = true;
    auto load = [&](bool v, int page, int u, int head, int keys) {
      const int slot = h % LR;
      if (!(ok = warp_wait(Q8 ? &raw_free[slot] : &empty[slot], ((h / LR) & 1) ^ 1))) return;
      if (lane == 0) mbar_arrive_expect_tx(&landed[slot], Q8 ? C::kRawHalf : C::kHalf);
      __syncwarp();
      const int in = (u * 64 + part * rows) & (a.c.page_size - 1);
      uint8_t* dst = Q8 ? sm + C::kOffRaw + slot * C::kRawBytes + part * rows * HD
                        : sm + slot * C::kHalf + atom * 8192 + part * rows * 128;
      if (mine) tma_load_4d(dst, v ? &v_map : &k_map, atom * 64, in, head, page, &landed[slot]);
      if constexpr (Q8) {
        const uint16_t* sc = static_cast<const uint16_t*>(v ? a.c.v_scale : a.c.k_scale);
        const int64_t* ss = v ? a.c.vs_stride : a.c.ks_stride;
        const uint32_t sb = sbase + C::kOffRaw + slot * C::kRawBytes + C::kRawHalf;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int k = x * 32 + lane, key = u * 64 + k;
          const int pg = __shfl_sync(0xffffffffu, page, k / rows);
          const bool in_pool = key < keys && pg >= 0 && pg < a.c.pages;
          const uint16_t* src = in_pool ? sc + pg * ss[0] + head * ss[1] + (key & (a.c.page_size - 1)) * ss[2] : sc;
          cp_async_small<HD / 16>(sb + k * (HD / 16), src, in_pool);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_u32(&landed[slot])) : "memory");
      }
      ++h;
    };
    int pk = page_of(at), pv = -1, u_v = 0, head_v = 0, keys_v = 0, left = min(at.of - at.u, n);
    bool starts = true;
    for (int i = 0; i <= n && ok && !*abort_flag; ++i) {
      if (i > 0 && (starts || i == n)) load(true, pv, u_v, head_v, keys_v);
      if (i == n || !ok) break;
      load(false, pk, at.u, at.head, at.r.keys);
      if (i > 0 && !starts && ok) load(true, pv, u_v, head_v, keys_v);
      pv = pk;
      u_v = at.u;
      head_v = at.head;
      keys_v = at.r.keys;
      starts = --left == 0;
      if (i + 1 < n) {
        if (starts) {
          next_item(at);
          left = at.of;
        } else {
          ++at.u;
        }
        pk = page_of(at);   // in flight while the ring is full
      }
    }
    if (!ok) fail();
    if (!ok || *abort_flag) {   // no copy may still be in flight when the CTA ends
      if constexpr (Q8) cp_async_wait_all();
      for (int f = max(0, h - LR); f < h; ++f) tc_wait(&landed[f % LR], (f / LR) & 1);
    }
  } else {
    // ----------------------------------------------------------------- helpers
    const int hw = warp - 6;
    bool ok = true;
    if constexpr (!Q8) {
      for (int k = 0; ok && !*abort_flag; ++k) {
        if (!(ok = warp_wait(fix_req, k & 1))) break;
        const Fix f = *fix;
        if (f.slot < 0) break;
        uint8_t* hb = sm + f.slot * C::kHalf;
        bool any_bad = false;
        for (int idx = hw * 32 + lane; idx < 64 * HD / 8; idx += NH * 32) {
          const int key = idx / (HD / 8), ch = idx % (HD / 8);
          uint4* p = reinterpret_cast<uint4*>(hb + (ch >> 3) * 8192 + sw128(key, ch & 7));
          if (key >= f.valid) {
            *p = make_uint4(0u, 0u, 0u, 0u);
          } else if (f.edge) {
            const uint4 x = *p;
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            if (drop_bad<BF>(w[0]) | drop_bad<BF>(w[1]) | drop_bad<BF>(w[2]) | drop_bad<BF>(w[3])) {
              *p = make_uint4(w[0], w[1], w[2], w[3]);
              any_bad = true;
            }
          }
        }
        if (any_bad) bad[f.unit & 7] = f.unit + 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(fix_done);
      }
    } else {
      constexpr int CPK = HD / 16;   // 16-byte chunks of a cached row
      int h = 0;
      auto convert = [&](bool v, int valid, bool edge, int unit) {
        const int slot = h % RING, rs = h % C::kRaw;
        if (!(ok = warp_wait(&landed[rs], (h / C::kRaw) & 1)) || !(ok = warp_wait(&empty[slot], ((h / RING) & 1) ^ 1))) return;
        const uint8_t* raw = sm + C::kOffRaw + rs * C::kRawBytes;
        bool any_bad = false;
#pragma unroll 4
        for (int idx = hw * 32 + lane; idx < 64 * CPK; idx += NH * 32) {
          const int key = idx / CPK, ch = idx % CPK;   // 16 dims: 16-bit chunks 2 ch and 2 ch + 1
          const uint4 x = lds128(raw + idx * 16);
          uint32_t sc = *reinterpret_cast<const uint16_t*>(raw + C::kRawHalf + key * (HD / 16) + (ch >> 1) * 2);
          if (key >= valid) sc = 0u;   // rows past the last key: +-0
          const uint32_t s2 = sc | sc << 16;
          const uint32_t in[4] = {x.x, x.y, x.z, x.w};
          uint32_t o[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            o[2 * y] = dq2(in[y], 0x5140u, s2);
            o[2 * y + 1] = dq2(in[y], 0x7362u, s2);
          }
          if (edge) {
#pragma unroll
            for (int y = 0; y < 8; ++y) any_bad |= drop_bad<false>(o[y]);
          }
          // lanes of neighbouring atoms write their two chunks in opposite order: all banks once
          const int first = (ch >> 2) & 1;
          uint8_t* hb = sm + slot * C::kHalf + (ch >> 2) * 8192;
          const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
          *reinterpret_cast<uint4*>(hb + sw128(key, ((2 * ch) & 7) + first)) = first ? hi : lo;
          *reinterpret_cast<uint4*>(hb + sw128(key, ((2 * ch) & 7) + (first ^ 1))) = first ? lo : hi;
        }
        if (any_bad) bad[unit & 7] = unit + 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[slot]);
          mbar_arrive(&raw_free[rs]);
        }
        ++h;
      };
      bool starts = true, edge_v = false;
      int valid_v = 0, left = min(at.of - at.u, n);
      for (int i = 0; i <= n && ok && !*abort_flag; ++i) {
        if (i > 0 && (starts || i == n)) convert(true, valid_v, edge_v, i - 1);
        if (i == n || !ok) break;
        convert(false, at.r.keys - at.u * 64, false, i);
        if (i > 0 && !starts && ok) convert(true, valid_v, edge_v, i - 1);
        valid_v = at.r.keys - at.u * 64;
        edge_v = is_edge(at);
        starts = --left == 0;
        if (i + 1 < n) {
          if (starts) {
            next_item(at);
            left = at.of;
          } else {
            ++at.u;
          }
        }
      }
    }
    if (!ok) fail();
  }

  tc_before();
  __syncthreads();
  if (warp == 4) {
    tc_after();
    tc_dealloc(tmem, C::kTmem);
  }
}

// -------------------------------------------------------------------- combine
// A block per split item and row (or every gridDim.y-th row).  The pieces' maxima give
// their weights; groups of threads sum a contiguous share of the pieces each, in piece
// order, and the groups' sums are added in order, so the result does not depend on when
// anything ran.
template <bool BF, int HD, int ROWS>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int kLanes = HD / 4, kGroups = 256 / kLanes;
  __shared__ float wgt[kMaxPieces];
  __shared__ float4 acc[256];
  __shared__ float red[8];
  griddep_wait();
  const int tid = threadIdx.x;
  if (a.by_item) {   // only the items of this launch have written their entry
    const Req r = get_req(a, blockIdx.x / a.c.kv_heads);
    if (r.n < 1 || r.n * static_cast<int64_t>(a.group) > a.rows_limit) return;
  }
  const int4 d = a.desc[blockIdx.x];   // {slot of the first piece, last CTA, request << 10 | KV head, tile}
  if (d.x < 0) return;
  const int b = d.z >> 10, head = d.z & 1023;
  const Req r = get_req(a, b);
  const int tt = 128 / a.group, t0 = d.w * tt, rows = min(tt, r.n - t0) * a.group;
  const int c0 = d.x >> 1, pieces = min(d.y - c0 + 1, kMaxPieces);
  auto slot_of = [&](int p) { return p == 0 ? d.x : 2 * (c0 + p); };
  auto block_reduce = [&](float v, bool is_max) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float w = __shfl_xor_sync(0xffffffffu, v, o);
      v = is_max ? fmaxf(v, w) : v + w;
    }
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) v = is_max ? fmaxf(v, red[w]) : v + red[w];
    return v;
  };
  const int lane = tid % kLanes, grp = tid / kLanes;
  const int p0 = pieces * grp / kGroups, p1 = pieces * (grp + 1) / kGroups;
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    float m = -INFINITY;
    for (int p = tid; p < pieces; p += 256) m = fmaxf(m, a.ml[slot_of(p) * ROWS + row].x);
    m = block_reduce(m, true);   // (its barriers also end the last row's use of wgt and acc)
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int p = tid; p < pieces; p += 256) {
      const float2 x = a.ml[slot_of(p) * ROWS + row];
      const float w = ex2_approx(x.x - base);
      wgt[p] = w;
      l += x.y * w;
    }
    l = block_reduce(l, false);   // (its barriers also publish wgt)
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = p0; p < p1; ++p) {
      const float4 v =
          *reinterpret_cast<const float4*>(a.part + (static_cast<int64_t>(slot_of(p)) * ROWS + row) * HD + 4 * lane);
      const float w = wgt[p];
      s.x = fmaf(v.x, w, s.x);
      s.y = fmaf(v.y, w, s.y);
      s.z = fmaf(v.z, w, s.z);
      s.w = fmaf(v.w, w, s.w);
    }
    acc[tid] = s;
    __syncthreads();
    if (grp == 0) {
      for (int k = 1; k < kGroups; ++k) {
        const float4 v = acc[k * kLanes + lane];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      const int t = t0 + row / a.group, hq = head * a.group + row % a.group;
      const bool sees = min(r.keys, r.kv - r.n_all + t + 1) > 0;
      float v[4] = {s.x / l, s.y / l, s.z / l, s.w / l};
      const int64_t tok = r.q0 + t;
      if (a.gate) {
        const uint2 x = *reinterpret_cast<const uint2*>(a.gate + tok * a.g_tok + hq * a.g_head + 4 * lane);
        const float2 x0 = unpack2<BF>(x.x), x1 = unpack2<BF>(x.y);
        v[0] /= 1.f + __expf(-x0.x);
        v[1] /= 1.f + __expf(-x0.y);
        v[2] /= 1.f + __expf(-x1.x);
        v[3] /= 1.f + __expf(-x1.y);
      }
      if (!sees) v[0] = v[1] = v[2] = v[3] = 0.f;
      *reinterpret_cast<uint2*>(a.out + tok * a.o_tok + hq * a.o_head + 4 * lane) =
          make_uint2(pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3]));
    }
  }
}

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// split-item area: descriptors, (max, sum) and partial rows of `ctas` CTAs
struct Split {
  size_t desc, ml, part, end;
};
Split split_area(int ctas, int rows, int hd) {
  Split s;
  s.desc = kErrBytes;
  s.ml = s.desc + ((static_cast<size_t>(ctas) * sizeof(int4) + 255) & ~size_t(255));
  s.part = s.ml + ((static_cast<size_t>(ctas) * 2 * rows * sizeof(float2) + 255) & ~size_t(255));
  s.end = s.part + static_cast<size_t>(ctas) * 2 * rows * hd * sizeof(float);
  return s;
}
void set_split(AttnArgs& a, void* ws, const Split& s) {
  uint8_t* p = static_cast<uint8_t*>(ws);
  a.desc = reinterpret_cast<int4*>(p + s.desc);
  a.ml = reinterpret_cast<float2*>(p + s.ml);
  a.part = reinterpret_cast<float*>(p + s.part);
}
// CTAs of the rows form: at most four on an SM (RowsCfg::kCtas)
constexpr int kRowsCtasPerSm = 4;

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

template <int CT, int HD>
int launch_rows(AttnArgs a, void* ws, int sms, cudaStream_t s) {
  using C = RowsCfg<CT, HD>;
  static bool configured = false;
  if (!configured) {
    if (cudaFuncSetAttribute(paged_rows_kernel<CT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
        cudaSuccess)
      return TLX_ERR_LAUNCH;
    configured = true;
  }
  const int ctas = sms * C::kCtas;
  set_split(a, ws, split_area(ctas, kRowsMax, HD));
  const int64_t items = static_cast<int64_t>(a.n_req) * a.c.kv_heads;
  a.by_item = items <= ctas;
  paged_rows_kernel<CT, HD><<<ctas, 128, C::kSmem, s>>>(a);
  if (cudaGetLastError() != cudaSuccess) return TLX_ERR_LAUNCH;
  const int most = std::min(kRowsMax, static_cast<int>(std::min<int64_t>(static_cast<int64_t>(a.max_new) * a.group, kRowsMax)));
  void* args[] = {&a};
  return launch_dependent(reinterpret_cast<const void*>(paged_combine_kernel<CT == CT_BF16, HD, kRowsMax>),
                          dim3(static_cast<unsigned>(std::min<int64_t>(items, ctas)), most), dim3(256), s, args);
}
// The pool as TMA sees it: [page][head][slot][dim], a box of 64 dims (int8: the row) of the
// keys of one page that fall in a unit of 64.  A dimension of one entry takes any stride.
bool page_map(CUtensorMap* map, const tlx_paged_kv& c, const void* base, const int64_t* stride) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode enc = nullptr;   // looked up through the runtime: the library does not link the driver's
  if (!enc) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return false;
    enc = reinterpret_cast<Encode>(fn);
  }
  const bool q8 = c.dtype == TLX_DT_Q8;
  const cuuint64_t esz = q8 ? 1 : 2;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_size),
                              static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.pages)};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i)
    strides[i] = dims[i + 1] > 1 ? static_cast<cuuint64_t>(stride[2 - i]) * esz : static_cast<cuuint64_t>(c.head_dim) * esz;
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(q8 ? c.head_dim : 64), static_cast<cuuint32_t>(std::min(c.page_size, 64)),
                             1u, 1u};
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  return enc(map, q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims,
             strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             q8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CT, int HD>
int launch_tiles(AttnArgs a, void* ws, int sms, cudaStream_t s) {
  using C = TilesCfg<CT, HD>;
  static bool configured = false;
  if (!configured) {
    if (cudaFuncSetAttribute(paged_tiles_kernel<CT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) !=
        cudaSuccess)
      return TLX_ERR_LAUNCH;
    configured = true;
  }
  const int ctas = sms * C::kCtas;
  set_split(a, ws, split_area(ctas, 128, HD));
  a.by_item = 0;
  CUtensorMap km, vm;
  if (!page_map(&km, a.c, a.c.k, a.c.k_stride) || !page_map(&vm, a.c, a.c.v, a.c.v_stride)) return TLX_ERR_LAUNCH;
  paged_tiles_kernel<CT, HD><<<ctas, C::kThreads, C::kSmem, s>>>(a, km, vm, static_cast<uint32_t*>(ws));
  if (cudaGetLastError() != cudaSuccess) return TLX_ERR_LAUNCH;
  void* args[] = {&a};
  return launch_dependent(reinterpret_cast<const void*>(paged_combine_kernel<CT == CT_BF16, HD, 128>),
                          dim3(ctas, 16), dim3(256), s, args);
}
template <int CT>
int launch_hd(const AttnArgs& a, bool tiles, void* ws, int sms, cudaStream_t s) {
  if (a.c.head_dim == 256) return tiles ? launch_tiles<CT, 256>(a, ws, sms, s) : launch_rows<CT, 256>(a, ws, sms, s);
  if (a.c.head_dim == 128) return tiles ? launch_tiles<CT, 128>(a, ws, sms, s) : launch_rows<CT, 128>(a, ws, sms, s);
  return tiles ? launch_tiles<CT, 64>(a, ws, sms, s) : launch_rows<CT, 64>(a, ws, sms, s);
}
int launch_form(const AttnArgs& a, int ct, bool tiles, void* ws, int sms, cudaStream_t s) {
  if (ct == CT_F16) return launch_hd<CT_F16>(a, tiles, ws, sms, s);
  if (ct == CT_BF16) return launch_hd<CT_BF16>(a, tiles, ws, sms, s);
  return launch_hd<CT_Q8>(a, tiles, ws, sms, s);
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
  return std::max(split_area(sms * kRowsCtasPerSm, kRowsMax, head_dim).end,
                  split_area(sms * (head_dim == 256 ? 1 : 2), 128, head_dim).end);
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
    const int rows_rc = launch_form(a, ct, false, ws, sms, s);
    if (rows_rc) return rows_rc;
  }
  if (static_cast<int64_t>(a.max_new) * a.group <= kRowsMax) return TLX_OK;
  return launch_form(a, ct, true, ws, sms, s);
}

}  // extern "C"

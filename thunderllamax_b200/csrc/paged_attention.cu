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
// simple form                     the rest.
#include <algorithm>

#include "paged.cuh"

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
  int4* desc;            // split items: {slot of the first piece, last CTA, request, KV head}
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
  if (r.n < 1 || r.n * a.group > a.rows_limit) return 0;
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
// Every thread of the block calls it; THREADS = blockDim.x.
struct Start {
  int64_t units, u0, u1;
  int64_t local;   // unit inside request b
  int b;
  int ctas;        // CTAs that have a unit: an item's pieces are consecutive ones
};
template <int THREADS, typename F>
__device__ __forceinline__ Start find_start(const AttnArgs& a, F units_of) {
  __shared__ int64_t tot[THREADS / 32];
  __shared__ int64_t s_local;
  __shared__ int s_b;
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
  s.b = s_b;
  s.local = s_local;
  return s;
}

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
// 2^x (ex2.approx: relative error about 2^-22; 2^-inf = 0)
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
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

template <int CT, int HD>
__global__ void __launch_bounds__(128, RowsCfg<CT, HD>::kCtas) paged_rows_kernel(const AttnArgs a) {
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
  const Start st = find_start<128>(a, [&](int b) { return static_cast<int64_t>(rows_units<KT>(a, get_req(a, b))); });
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
    const float f0 = pow2(m0 - b0), f1 = pow2(m1 - b1);   // 0 for the first unit
    m0 = n0;
    m1 = n1;
    l0 *= f0;
    l1 *= f1;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t p0 = pack2<BF>(pow2(s[nb][0] - b0), pow2(s[nb][1] - b0));
      const uint32_t p1 = pack2<BF>(pow2(s[nb][2] - b1), pow2(s[nb][3] - b1));
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
          const int4 d = make_int4(whole ? -1 : slot, whole ? -1 : range_of(st.units, end - 1, st.ctas), at.b, at.head);
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

// -------------------------------------------------------------------- combine
// One block per (split item, row).  The pieces' maxima give their weights; groups of
// threads sum a contiguous share of the pieces each, in piece order, and the groups' sums
// are added in order, so the result does not depend on when anything ran.
template <bool BF, int HD, int ROWS>
__global__ void __launch_bounds__(256) paged_combine_kernel(const AttnArgs a) {
  constexpr int kLanes = HD / 4, kGroups = 256 / kLanes;
  __shared__ float wgt[kMaxPieces];
  __shared__ float4 acc[256];
  __shared__ float red[8];
  griddep_wait();
  const int row = blockIdx.y, tid = threadIdx.x;
  int b = 0, head = 0;
  if (a.by_item) {   // only the items of this launch have written their entry
    b = blockIdx.x / a.c.kv_heads;
    head = blockIdx.x % a.c.kv_heads;
    const Req r = get_req(a, b);
    if (r.n < 1 || r.n * a.group > a.rows_limit) return;
  }
  const int4 d = a.desc[blockIdx.x];   // {slot of the first piece, last CTA, request, KV head}
  if (d.x < 0) return;
  if (!a.by_item) {
    b = d.z;
    head = d.w;
  }
  const Req r = get_req(a, b);
  if (row >= r.n * a.group) return;
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
  float m = -INFINITY;
  for (int p = tid; p < pieces; p += 256) m = fmaxf(m, a.ml[slot_of(p) * ROWS + row].x);
  m = block_reduce(m, true);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int p = tid; p < pieces; p += 256) {
    const float2 x = a.ml[slot_of(p) * ROWS + row];
    const float w = pow2(x.x - base);
    wgt[p] = w;
    l += x.y * w;
  }
  l = block_reduce(l, false);   // its barriers also publish wgt
  const int lane = tid % kLanes, grp = tid / kLanes;
  const int p0 = pieces * grp / kGroups, p1 = pieces * (grp + 1) / kGroups;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int p = p0; p < p1; ++p) {
    const float4 v = *reinterpret_cast<const float4*>(a.part + (static_cast<int64_t>(slot_of(p)) * ROWS + row) * HD + 4 * lane);
    const float w = wgt[p];
    s.x = fmaf(v.x, w, s.x);
    s.y = fmaf(v.y, w, s.y);
    s.z = fmaf(v.z, w, s.z);
    s.w = fmaf(v.w, w, s.w);
  }
  acc[tid] = s;
  __syncthreads();
  if (grp > 0) return;
  for (int k = 1; k < kGroups; ++k) {
    const float4 v = acc[k * kLanes + lane];
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  const int t = row / a.group, hq = head * a.group + row - t * a.group;
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

// ---------------------------------------------------------------- simple form
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
  if (min(n, a.max_new) * a.group <= a.rows_limit) return;
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
template <int CT>
int launch_rows_hd(const AttnArgs& a, void* ws, int sms, cudaStream_t s) {
  if (a.c.head_dim == 256) return launch_rows<CT, 256>(a, ws, sms, s);
  if (a.c.head_dim == 128) return launch_rows<CT, 128>(a, ws, sms, s);
  return launch_rows<CT, 64>(a, ws, sms, s);
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
  return split_area(sm_count() * kRowsCtasPerSm, kRowsMax, head_dim).end;
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
  const int ct = cache_type(cache);
  if (a.group <= kRowsMax) {   // the requests' lengths are on the device: the forms share them out there
    const int sms = sm_count();
    const int rr = ct == CT_F16    ? launch_rows_hd<CT_F16>(a, ws, sms, s)
                   : ct == CT_BF16 ? launch_rows_hd<CT_BF16>(a, ws, sms, s)
                                   : launch_rows_hd<CT_Q8>(a, ws, sms, s);
    if (rr) return rr;
  }
  if (static_cast<int64_t>(a.max_new) * a.group <= kRowsMax) return TLX_OK;
  if (ct == CT_F16) return launch_simple<CT_F16>(a, s);
  if (ct == CT_BF16) return launch_simple<CT_BF16>(a, s);
  return launch_simple<CT_Q8>(a, s);
}

}  // extern "C"

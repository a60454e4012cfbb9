// Rows form of the paged attention: requests with at most 16 query rows per KV head.
#include "kernel_setup.h"
#include "paged_attention.cuh"

namespace tlx {
namespace {

// ------------------------------------------------------------------ rows form
// A CTA of four warps takes a unit of KT keys at a time.  The keys are split over the
// warps for S = Q K^T (m16n8k16: 16 rows x 8 keys) and the dims for O += P V, so no sum
// crosses warps; per unit the row maxima and P go through shared memory (two barriers).
// K and V rows come in by 16-byte asynchronous copies, kStages units deep, each warp
// loading its own keys.  The k order of a matrix product is free, so a lane takes 16
// contiguous bytes of its key's row as the B fragments of 2 (16-bit) or 4 (int8) steps,
// and Q is loaded in the same order.  int8 codes become fp16(code - 128) * scale, rounded
// once, in registers.
//
// Bound by HBM in principle and by issue in practice for int8 caches: the kernel spends
// about 1250 instructions a warp on a unit of 64 keys, a third of them decoding codes (60 %
// of the issue slots, three warps a scheduler).  Measured: 64 requests of 300..16000 keys,
// 24 / 4 heads, dim 256, int8: 149 us, 4.0 TB/s (0.61 of the measured copy rate); the same
// lengths in bf16, 32 / 8 heads of 128: 173 us, 6.5 TB/s (0.99; 177 us a call); one request of
// 4097 int8 keys 15.8 us with the joining kernel.  32 keys a unit for 16-bit rows of
// 256 dims and two or three stages, so that two to four CTAs share an SM.
// Positions of an item besides its units (see the schedule): 64 requests take 179 us with
// none, 170 with one, 171 with three.
constexpr int kItemCost = 1;

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
  const Start st = find_start<128>(a, psm, [&](int b) -> int64_t {
    const int units = rows_units<KT>(a, get_req(a, b));
    return units ? static_cast<int64_t>(units + kItemCost) * a.c.kv_heads : 0;
  });
  if (!a.by_item && tid == 0) a.desc[blockIdx.x] = make_int4(-1, -1, 0, 0);
  if (st.u0 == st.u1) return;

  // position in the row of units: request, KV head, unit of the item
  struct Pos {
    int b, head, u, of;
    Req r;
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

  Pos load_at;
  load_at.b = st.b;
  load_at.r = get_req(a, st.b);
  load_at.of = rows_units<KT>(a, load_at.r);
  load_at.head = static_cast<int>(st.local / (load_at.of + kItemCost));
  const int into = static_cast<int>(st.local % (load_at.of + kItemCost));
  load_at.u = max(0, into - kItemCost);
  int64_t pos = st.u0 + max(0, kItemCost - into);   // of the part's first unit
  // the units of the range
  int n_units = 0;
  {
    int64_t x = pos;
    int head = load_at.head, of = load_at.of, b = load_at.b, u = load_at.u;
    while (x < st.u1) {
      const int k = static_cast<int>(min(static_cast<int64_t>(of - u), st.u1 - x));
      n_units += k;
      x += k + kItemCost;
      u = 0;
      if (++head < a.c.kv_heads) {   // the request's other heads are like this one
        const int span = of + kItemCost;
        const int skip = static_cast<int>(min(static_cast<int64_t>(a.c.kv_heads - head), max(st.u1 - x, static_cast<int64_t>(0)) / span));
        n_units += skip * of;
        x += static_cast<int64_t>(skip) * span;
        head += skip;
      }
      if (head == a.c.kv_heads) {
        head = 0;
        do {
          ++b;
        } while (b < a.n_req && (of = rows_units<KT>(a, get_req(a, b))) == 0);
        if (b >= a.n_req) break;
      }
    }
  }
  if (n_units == 0) return;
  Pos at = load_at;
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
  int part_i = 0;           // first unit of the part
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
    const uint32_t kb = sbase + stage * C::kStage;   // (32-bit shared addresses throughout)
    // chunk 4 j + q of a row lies at 4 (j ^ (row & 1)) + q, and row & 1 = g & 1: even and odd
    // j from one address each
    const uint32_t k_even = kb + (warp * KW + g) * C::kRow + q * 16 + ((Q8 && HD == 64) ? 0 : (g & 1) * 64);
    const uint32_t k_odd = kb + (warp * KW + g) * C::kRow + q * 16 + 64 - (g & 1) * 64;
    // S of this warp's keys.  K reads: 8 lanes of a phase are 2 keys x 4 chunks, the
    // swizzle puts the second key's chunks in the other half of the banks.
    float s[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = warp * KW + nb * 8 + g;
      float e[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if constexpr (Q8) {
        uint32_t sw[HD / 64];   // the row's scales, two groups a word
        const uint32_t sp = kb + kOffKs + row * C::kScaleRow;
        if constexpr (HD == 256) {
          const uint4 v = ls128(sp);
          sw[0] = v.x; sw[1] = v.y; sw[2] = v.z; sw[3] = v.w;
        } else if constexpr (HD == 128) {
          const uint2 v = ls64(sp);
          sw[0] = v.x; sw[1] = v.y;
        } else {
          sw[0] = ls32(sp);
        }
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          const uint4 v = ls128((j & 1 ? k_odd : k_even) + nb * 8 * C::kRow + (j >> 1) * 128);
          const uint32_t s2 = prmt(sw[j], sw[j], q >= 2 ? 0x3232u : 0x1010u);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int t = 0; t < 4; ++t) mma16<false>(e[t & 1], qf[4 * j + t], dq2(w[t], 0x5140u, s2), dq2(w[t], 0x7362u, s2));
        }
      } else {
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const uint4 v = ls128((j & 1 ? k_odd : k_even) + nb * 8 * C::kRow + (j >> 1) * 128);
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
    const uint32_t vb = kb + kOffV;
    // A key that some rows do not see must not reach them through 0 * inf or 0 * NaN: units
    // with such keys are looked over first.  (A request's only new token sees all its keys; of
    // several planned tokens even the only row that is asked for, max_new = 1, does not.)
    bool slow = false;
    if (at.r.n_all > 1 && (at.u + 1) * KT > at.r.kv - at.r.n_all + 1) {
      bool found = false;
      for (int key = max(0, at.r.kv - at.r.n_all + 1 - at.u * KT) + warp; key < KT; key += 4) {
        if constexpr (Q8) {   // (any product may overflow where the scale passes 65504 / 128)
          for (int x = lane; x < HD / 32; x += 32)
            found |= !(fabsf(__half2float(__ushort_as_half(static_cast<uint16_t>(ls16(kb + kOffVs + key * C::kScaleRow + 2 * x))))) < 511.f);
        } else {
          for (int x = lane; x < CPR; x += 32) {
            const uint4 v = ls128(vb + key * C::kRow + x * 16);
            found |= bad16<BF>(v.x) || bad16<BF>(v.y) || bad16<BF>(v.z) || bad16<BF>(v.w);
          }
        }
      }
      slow = __syncthreads_or(found);
    }
    auto product = [&](int j, const uint32_t (&pf)[4], uint32_t v0, uint32_t v1, int) { mma16<BF>(o[j], pf, v0, v1); };
    // the same token by token, each with the keys it sees
    auto careful = [&](int j, const uint32_t (&pf)[4], uint32_t v0, uint32_t v1, int k16) {
      const int key = at.u * KT + k16 * 16 + 2 * q;
#pragma unroll 1
      for (int t = 0; t < at.r.n; ++t) {
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
    };
    auto unit_product = [&](auto&& product) {
#pragma unroll 1
      for (int k = 0; k < KT / 16; ++k) {
        uint32_t pf[4];
        ldsm4(pf, pbase + ((lane & 7) + ((lane >> 3) & 1) * 8) * C::kPPitch + (2 * k + (lane >> 4)) * 16);
        if constexpr (Q8) {
          // lane (g, q): keys 2q, 2q+1, 2q+8, 2q+9 and DB contiguous dims from DB g on
          uint32_t w[4][DB > 4 ? 2 : 1];
          uint32_t sh[4];
          // (row >> 1) & 3 = q for all four rows: one address and immediates
          const int byte = warp * DW + DB * g;
          const int ch = HD == 64 ? (byte >> 4) ^ q : (byte >> 4) ^ (q << 1);
          const uint32_t v_at = vb + (k * 16 + 2 * q) * C::kRow + ch * 16 + (byte & 15);
          const uint32_t s_at = kb + kOffVs + (k * 16 + 2 * q) * C::kScaleRow + (byte >> 5) * 2;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = (e & 1) + (e >> 1) * 8;
            const uint32_t p = v_at + row * C::kRow;
            if constexpr (DB == 8) {
              const uint2 v = ls64(p);
              w[e][0] = v.x;
              w[e][1] = v.y;
            } else if constexpr (DB == 4) {
              w[e][0] = ls32(p);
            } else {
              w[e][0] = ls16(p);
            }
            sh[e] = ls16(s_at + row * C::kScaleRow);
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
            ldsm4t(v, vb + row * C::kRow + ch * 16);
            product(j, pf, v[0], v[1], k);
            product(j + 1, pf, v[2], v[3], k);
          }
        }
      }
    };
    if (slow) unit_product(careful);
    else unit_product(product);
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
      const int part = i + 1 - part_i, u_first = at.u + 1 - part;   // the units of this part
      const bool whole = u_first == 0 && part == at.of;
      const int rows = at.r.n * a.group;
      const int slot = 2 * blockIdx.x + (part_i > 0 ? 1 : 0);   // the CTA's first part, or a later one
      if (tid == 0) {
        const int64_t item = static_cast<int64_t>(at.b) * a.c.kv_heads + at.head;
        if (u_first == 0) {   // the item starts here: where its pieces are, if it is split
          const int4 d = make_int4(whole ? -1 : slot, whole ? -1 : range_of(st.units, pos + at.of - 1, st.ctas), at.b << 10 | at.head, 0);
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
            v0 = gated(v0, x.x);
            v1 = gated(v1, x.y);
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
    if (first) {
      pos += i + 1 - part_i + kItemCost;
      part_i = i + 1;
    }
    if (i + 1 < n_units) advance(at);
  }
}

// CTAs of the rows form: at most four on an SM (RowsCfg::kCtas)
constexpr int kRowsCtasPerSm = 4;

template <int CT, int HD>
int launch_rows(AttnArgs a, void* area, int sms, cudaStream_t s, SplitSet* set) {
  using C = RowsCfg<CT, HD>;
  static std::atomic<uint64_t> done{0};
  if (!setup_kernel(reinterpret_cast<const void*>(paged_rows_kernel<CT, HD>), C::kSmem, done)) return TLX_ERR_LAUNCH;
  const int ctas = sms * C::kCtas;
  const int64_t items = static_cast<int64_t>(a.n_req) * a.c.kv_heads;
  a.by_item = items <= ctas;
  *set = set_split(a, area, ctas, kRowsMax);
  set->items = static_cast<int>(std::min<int64_t>(items, ctas));
  set->rows = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(a.max_new) * a.group, kRowsMax));
  paged_rows_kernel<CT, HD><<<ctas, 128, C::kSmem, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? TLX_OK : TLX_ERR_LAUNCH;
}

}  // namespace

template <int CT>
static int launch_rows_hd(const AttnArgs& a, void* area, int sms, cudaStream_t stream, SplitSet* set) {
  if (a.c.head_dim == 256) return launch_rows<CT, 256>(a, area, sms, stream, set);
  if (a.c.head_dim == 128) return launch_rows<CT, 128>(a, area, sms, stream, set);
  return launch_rows<CT, 64>(a, area, sms, stream, set);
}

int launch_paged_rows(const AttnArgs& a, int ct, void* area, int sms, cudaStream_t stream, SplitSet* set) {
  if (ct == CT_F16) return launch_rows_hd<CT_F16>(a, area, sms, stream, set);
  if (ct == CT_BF16) return launch_rows_hd<CT_BF16>(a, area, sms, stream, set);
  return launch_rows_hd<CT_Q8>(a, area, sms, stream, set);
}

size_t paged_rows_bytes(int hd, int sms) { return (split_area(sms * kRowsCtasPerSm, kRowsMax, hd).end + 255) & ~size_t(255); }

}  // namespace tlx

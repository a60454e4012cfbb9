// Tiles form of the paged attention: requests with more than 16 query rows per KV head.
#include <cuda.h>

#include "kernel_setup.h"
#include "paged_attention.cuh"
#include "paged_schedule.h"

namespace tlx {
namespace {

// ----------------------------------------------------------------- tiles form
// The 128 rows of a tensor-core tile are the query heads of one KV head times as many
// tokens as fit (row = token * group + head), so every key read serves the whole group.
// A CTA walks its units (64 keys of one item) on tcgen05:
//   S(i) = Q K_i^T   M = 128, N = 64, K = head_dim; Q in tensor memory (head_dim 256) or
//                    shared memory, S double-buffered in tensor memory
//   O += P(i) V_i    M = 128, N = head_dim, K = 64; V is the MN-major operand as it lies
//                    in the cache, P (16 bit) in shared memory, double-buffered where it fits
//   softmax warpgroups   one thread per row; with two groups they take the units in turn,
//                so one group's exponentials run beside the other's loads and waits, and
//                hand on the row's reference maximum.  O is rescaled (in tensor memory) only
//                when a row's maximum grows by more than 2^8, which keeps P in range.
//   QK warps, PV warp    one thread each issues its MMAs: several issuers (two for S, the
//                units in turn), because the waits and commits of one would leave the tensor
//                pipe idle.  The PV warp also takes out of a 16-bit V what must not reach the
//                product (rows past the last key, and infinite or NaN values where some rows
//                do not see the unit whole).
//   loader warps         the K and V halves of the units: one TMA box per page (and 64 dims),
//                so pages may lie anywhere and what is outside the pool reads as 0; issuing a
//                box costs its warp about 100 cycles, so the warps share the boxes of a half
//   converter warps      (int8 caches) turn every half into fp16(code * scale)
// Every wait is bounded: a timeout raises the error word, all roles leave, issued MMAs
// and copies are drained and tensor memory is freed.
//
// Measured (24 / 4 heads, dim 256): 4096 new tokens over 8192 fp16 keys 0.64 ms in one launch,
// 0.77 ms in a row of calls under the power cap's clocks (0.80 PFLOP/s, 0.48 of the measured
// matrix rate); the MMAs alone would take 0.43 ms in this form (16 MMAs of N = 64 and 4 of
// N = 256 cost 1050 to 1430 cycles a unit from one or two issuers); 11 rows at 100011 int8 keys
// 114 us, 130 us a call (without the converters a call takes 114 us; what makes up the rest of
// the distance to the floor of 33 us has not been measured); 2000 rows over 4000 int8 keys
// 330 us a call; the mixed bf16 batch 212 us, 237 us a call.
//
// Code size: the roles' loops run side by side on each scheduler, one warp each, so what
// does not fit the instruction caches is fetched again for every unit.  Hence the loops
// that could be unrolled further and are not, and one call site for each large body.
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N));
}
// two fp32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;\n"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return d;
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(b))
      : "memory");
}
// A bounded wait, as little code as it can be.
__device__ __forceinline__ bool thread_wait(uint64_t* b, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 0; i < kMbarPollLimit; ++i)
    if (mbar_try_wait(b, parity)) return true;
  return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity) {
  const bool ok = thread_wait(b, parity);
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
  // One CTA of two softmax groups on an SM, or (16-bit caches of narrow heads, whose smaller
  // rings leave room) two CTAs of one group.
  static constexpr int kGroups = HD == 256 || kQ8 ? 2 : 1;
  static constexpr int kCtas = kGroups == 2 ? 1 : 2;
  static constexpr int kPBufs = HD == 128 && !kQ8 ? 1 : 2;
  // 16-bit halves that the MMAs read, one half of the ring for K and one for V (so that each
  // issuer waits for its slots in order), and (int8) halves as they lie in the cache
  static constexpr int kRing = kQ8 && HD == 256 ? 4 : HD == 128 && !kQ8 ? 4 : 6;
  static constexpr int kRaw = !kQ8 ? 0 : HD == 256 ? 3 : 6;
  static constexpr int kRawHalf = kKeys * HD;                   // codes; the scales follow
  static constexpr int kRawBytes = kRawHalf + kKeys * (HD / 16);
  static constexpr int kThreads = kGroups == 2 ? 512 : 256;
  static constexpr int kQkWarp = 4 * kGroups, kPvWarp = kQkWarp + kGroups, kLoadWarp = kPvWarp + 1;
  static constexpr int kLoaders = kQ8 ? 1 : kGroups == 2 ? 4 : 2;
  static constexpr int kConvWarp = kThreads / 32 - 4;           // int8: four converters
  // registers after the roles part (of the 128 of the launch)
  static constexpr int kRegsSoftmax = kGroups == 2 ? 168 : 184;
  static constexpr int kRegsOther = kGroups == 2 ? 88 : 72;
  static_assert(kGroups * kRegsSoftmax + (kThreads / 128 - kGroups) * kRegsOther <= kThreads, "register split");
  static constexpr int kOffP = kRing * kHalf;
  static constexpr int kOffQ = kOffP + kPBufs * kPBytes;
  static constexpr int kOffRaw = kOffQ + kQBytes;
  static constexpr int kOffX = kOffRaw + kRaw * kRawBytes;      // row maxima and sums the groups exchange
  static constexpr int kOffBar = kOffX + (kGroups == 2 ? 5 * 128 * 4 : 0);
  static constexpr int kSmem = kOffBar + 512;
  static_assert(kSmem <= 227 * 1024 / kCtas - (kCtas - 1) * 512, "shared memory");
  static constexpr uint32_t kTmem = HD == 256 || kCtas == 1 ? 512 : 256;
  static constexpr uint32_t kColS = 0, kColO = 128;
  static constexpr uint32_t kColQ = kQTmem ? 384 : 0;
  static constexpr uint32_t kFmt = CT == CT_BF16 ? (1u << 7) | (1u << 10) : 0u;   // A, B bf16
  static constexpr uint32_t kIdescQK = (1u << 4) | kFmt | (64u >> 3) << 17 | (128u >> 4) << 24;
  static constexpr uint32_t kIdescPV = (1u << 4) | kFmt | (1u << 16) | static_cast<uint32_t>(HD >> 3) << 17 | (128u >> 4) << 24;
};

// Barriers of the P V products, by unit.  A wait names a phase by its parity alone, so it is
// right only where the phase before (the product kPvRing units earlier) is known to be
// complete.  The furthest look ahead is the rescale of O: at unit i a group waits for product
// i - 1 when all it knows, from the other group's maximum of unit i - 1, is that product i - 5
// is complete (that group saw it before it wrote P of unit i - 3).  Hence four, not two.
constexpr int kPvRing = 4;

// Positions of an item besides its units (see the schedule): with 3 / 6 / 10 the mixed batch
// takes 309 / 250 / 246 us, with none 440.
constexpr int kItemCost = 8;

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
// positions of one KV head in the tiles before `tile`
__device__ __forceinline__ int64_t positions_before(const AttnArgs& a, const Req& r, int tile) {
  return units_before(static_cast<int64_t>(r.kv) - r.n_all, tile_tokens(a), r.n, r.keys, tile) +
         static_cast<int64_t>(tile) * kItemCost;
}

// Infinite and NaN values of V are replaced by 0 in shared memory in the units that some rows do
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

// An item (tile of a request's rows, KV head) and a unit of it.
struct Pos {
  int b, tile, head, u, of, tiles;
  Req r;
};
__device__ __forceinline__ Pos item_after(const AttnArgs& a, Pos p) {
  p.u = 0;
  if (++p.head == a.c.kv_heads) {
    p.head = 0;
    if (++p.tile == p.tiles) {
      p.tile = 0;
      do {
        if (++p.b >= a.n_req) return p;
        p.r = get_req(a, p.b);
        p.tiles = tile_count(a, p.r);
      } while (p.tiles == 0);
    }
    p.of = tile_units(a, p.r, p.tile);
  }
  return p;
}

// units in the positions [pos, end), from unit p.u (at pos) of item p on
__device__ __noinline__ int units_of_range(const AttnArgs& a, Pos p, int64_t pos, int64_t end) {
  int n = 0;
  while (pos < end) {
    const int k = static_cast<int>(min(static_cast<int64_t>(p.of - p.u), end - pos));
    n += k;
    pos += k + kItemCost;
    p.u = 0;
    if (p.head + 1 < a.c.kv_heads) {   // the tile's other heads are like this one
      const int span = p.of + kItemCost;
      const int skip = static_cast<int>(min(static_cast<int64_t>(a.c.kv_heads - 1 - p.head), max(end - pos, static_cast<int64_t>(0)) / span));
      n += skip * p.of;
      pos += static_cast<int64_t>(skip) * span;
      p.head += skip;
    }
    if (pos >= end) break;
    p = item_after(a, p);
    if (p.b >= a.n_req) break;
  }
  return n;
}

template <int CT, int HD>
__global__ void __launch_bounds__(TilesCfg<CT, HD>::kThreads, TilesCfg<CT, HD>::kCtas)
    paged_tiles_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map, uint32_t* err) {
  using C = TilesCfg<CT, HD>;
  constexpr bool BF = CT == CT_BF16, Q8 = C::kQ8;
  static_assert(C::kColO + HD + (C::kQTmem ? C::kColQ - 384 + HD / 2 : 0) <= C::kTmem, "tensor memory");
  constexpr int RING = C::kRing, RH = RING / 2, PB = C::kPBufs, NG = C::kGroups;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + C::kOffBar);
  uint64_t* landed = bar;               // [RING or RAW] TMA -> MMA or converters
  uint64_t* raw_free = landed + 6;      // [RAW] converters -> loader
  uint64_t* full = raw_free + 6;        // [RING] converters -> MMA
  uint64_t* empty = full + 6;           // [RING] MMA -> loaders or converters
  uint64_t* s_full = empty + 6;         // [2] QK -> softmax
  uint64_t* s_free = s_full + 2;        // [2] softmax -> QK
  uint64_t* p_full = s_free + 2;        // [2] softmax -> PV
  uint64_t* pv_done = p_full + 2;       // [kPvRing] PV -> softmax
  uint64_t* q_full = pv_done + kPvRing; // softmax -> QK: Q of the next item is in
  uint64_t* o_free = q_full + 1;        // softmax -> PV: O of the last item is read
  uint64_t* done = o_free + 1;
  uint64_t* turn = done + 1;            // [2] QK warp -> QK warp: S of unit i is issued
  uint64_t* m_full = turn + 2;          // [4][2] between the groups' warps of the same rows: maximum of unit i
  uint64_t* l_full = m_full + 8;        // [4] the same: both groups' sums of an item
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(l_full + 4);
  volatile uint32_t* abort_flag = tmem_holder + 1;
  // [8] by unit: unit + 1 if a bad value was taken out of its V (V is fewer than 8 units ahead
  // of the softmax)
  volatile int* bad = reinterpret_cast<int*>(tmem_holder + 2);
  struct First {
    int tile, head, u, skip, n;   // ..., positions before the first unit, units of the range
  };
  First* first_at = reinterpret_cast<First*>(tmem_holder + 10);
  volatile float* m_sh = reinterpret_cast<float*>(sm + C::kOffX);   // [128]
  volatile float* l_sh = m_sh + 128;                                 // [2 items][2 groups][128]
  static_assert((4 * 6 + 23 + kPvRing) * 8 + 15 * 4 <= 512 && RING <= 6 && C::kRaw <= 6, "barrier area");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_launch_dependents();
  const Start st = find_start<C::kThreads>(a, sm + C::kOffP, [&](int b) -> int64_t {
    const Req r = get_req(a, b);
    const int tiles = tile_count(a, r);
    return tiles ? positions_before(a, r, tiles) * a.c.kv_heads : 0;
  });
  if (tid == 0) a.desc[blockIdx.x] = make_int4(-1, -1, 0, 0);
  if (st.u0 == st.u1) {
    griddep_wait();
    return;
  }
  const uint32_t sbase = smem_u32(sm);
  if (sbase & 1023u) {   // the descriptors need the swizzle atoms' alignment
    if (tid == 0) atomicOr(err, ERR_BAD_PARAM);
    return;
  }
  if (warp == 0) {   // the tile, head and unit at which the range starts: a 32-way search
    const Req r = get_req(a, st.b);
    int lo = 0, hi = tile_count(a, r);   // positions_before(lo) * heads <= local < positions_before(hi) * heads
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, t = min(lo + lane * step, hi);
      const bool le = t < hi && positions_before(a, r, t) * a.c.kv_heads <= st.local;
      const int k = 31 - __clz(__ballot_sync(0xffffffffu, le));   // lane 0 always holds
      const int nlo = lo + k * step;
      hi = min(hi, nlo + step);
      lo = nlo;
    }
    if (lane == 0) {
      const int64_t rest = st.local - positions_before(a, r, lo) * a.c.kv_heads;
      Pos p;
      p.b = st.b;
      p.r = r;
      p.tiles = tile_count(a, r);
      p.tile = lo;
      p.of = tile_units(a, r, lo);
      p.head = static_cast<int>(rest / (p.of + kItemCost));
      const int into = static_cast<int>(rest % (p.of + kItemCost));
      p.u = max(0, into - kItemCost);
      const int64_t pos = st.u0 + max(0, kItemCost - into);
      *first_at = First{p.tile, p.head, p.u, static_cast<int>(pos - st.u0), units_of_range(a, p, pos, st.u1)};
    }
  }
  if (tid == 0) {
    for (int i = 0; i < 6; ++i) {
      mbar_init(&landed[i], Q8 ? 33 : C::kLoaders);   // int8: 32 lanes' copies of the scales as well
      mbar_init(&raw_free[i], 4);
      mbar_init(&full[i], 4);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 8; ++i) bad[i] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
    }
    for (int i = 0; i < kPvRing; ++i) mbar_init(&pv_done[i], 1);
    mbar_init(q_full, 4 * NG);
    mbar_init(o_free, 4 * NG);
    mbar_init(done, NG + 1);
    for (int i = 0; i < 2; ++i) mbar_init(&turn[i], 1);
    for (int i = 0; i < 8; ++i) mbar_init(&m_full[i], 1);
    for (int i = 0; i < 4; ++i) mbar_init(&l_full[i], 2);
    *abort_flag = 0u;
    mbar_fence_init();
  }
  if (warp == C::kQkWarp) tc_alloc(tmem_holder, C::kTmem);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_holder;
  auto pv_bar = [&](int unit) { return &pv_done[unit % kPvRing]; };
  auto pv_wait = [&](int unit) { return warp_wait(pv_bar(unit), (unit / kPvRing) & 1); };   // product of the unit
  auto fail = [&]() {
    atomicOr(err, ERR_MBAR_TIMEOUT);
    *abort_flag = 1u;
  };

  Pos at;
  at.b = st.b;
  at.r = get_req(a, st.b);
  at.tiles = tile_count(a, at.r);
  at.tile = first_at->tile;
  at.head = first_at->head;
  at.u = first_at->u;
  const int n = first_at->n;
  at.of = tile_units(a, at.r, at.tile);
  // the next item (not called past the last unit of the launch)
  auto next_item = [&](Pos& p) { p = item_after(a, p); };

  // keys that every row of the item's tile sees; a unit past them needs care (is not seen
  // whole by some row, or holds fewer than 64 keys)
  auto seen_by_all = [&](const Pos& p) {
    return max(0, min(p.r.keys, p.r.kv - p.r.n_all + p.tile * tile_tokens(a) + 1));
  };

  if (warp < 4 * NG) {
    reg_inc<C::kRegsSoftmax>();
    // ----------------------------------------------------------------- softmax
    const int grp = NG == 2 ? warp >> 2 : 0, qd = warp & 3, row = qd * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(qd * 32) << 16;
    const float sc = a.scale * 1.4426950408889634f;
    const int tt = tile_tokens(a), t_in = row / a.group, hl = row - t_in * a.group;
    bool ok = true;
    auto load_q = [&](const Pos& p) {   // this row of Q (zero past the last row)
      const int t = p.tile * tt + t_in;
      const bool valid = t_in < tt && t < p.r.n;
      const uint4* src = reinterpret_cast<const uint4*>(a.q + static_cast<int64_t>(p.r.q0 + t) * a.q_tok +
                                                        (p.head * a.group + hl) * a.q_head);
      constexpr int CH = HD / 8 / NG, FLY = CH < 8 ? CH : 8;   // 16-byte chunks of this group, FLY in flight
#pragma unroll 1
      for (int c0 = grp * CH; c0 < (grp + 1) * CH; c0 += FLY) {
        uint4 v[FLY];
#pragma unroll
        for (int j = 0; j < FLY; ++j) v[j] = valid ? __ldg(src + c0 + j) : make_uint4(0u, 0u, 0u, 0u);
        if constexpr (C::kQTmem) {
#pragma unroll
          for (int x = 0; x < FLY; x += 4) {
            const uint32_t w[16] = {v[x].x,     v[x].y,     v[x].z,     v[x].w,     v[x + 1].x, v[x + 1].y,
                                    v[x + 1].z, v[x + 1].w, v[x + 2].x, v[x + 2].y, v[x + 2].z, v[x + 2].w,
                                    v[x + 3].x, v[x + 3].y, v[x + 3].z, v[x + 3].w};
            tc_st16(tmem + lanes + C::kColQ + (c0 + x) * 4, w);
          }
        } else {
#pragma unroll
          for (int j = 0; j < FLY; ++j)
            *reinterpret_cast<uint4*>(sm + C::kOffQ + ((c0 + j) >> 3) * 16384 + sw128(row, (c0 + j) & 7)) = v[j];
        }
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
    int i = 0, item = -1, last = -1, begin_i = 0;
    int64_t pos = st.u0 + first_at->skip;   // of the part's first unit
    Pos next = at;
    float m_ref, l_run;
    for (;;) {
      // (one site each for the Q load, the item's units and its end: see the note on code size)
      const bool more = i < n;
      if (more) {   // Q of the next item may follow once the last S of this one is made
        // (S of last - 2 is complete: its group sent its maximum for this one's unit last - 1)
        if (NG == 2 && item >= 0 && (last & 1) != grp && !(ok = warp_wait(&s_full[last & 1], (last >> 1) & 1))) break;
        load_q(next);
      }
      const int t = at.tile * tt + t_in;
      const bool valid = t_in < tt && t < at.r.n;
      const int lim = valid ? max(0, min(at.r.keys, at.r.kv - at.r.n_all + t + 1)) : 0;   // keys < lim
      const bool any = __any_sync(0xffffffffu, valid);   // a warp without rows only keeps the barriers going
      if (item >= 0) {
        // the item's rows, or this part's; two groups take half of the columns each
        if (NG == 2) {
          if ((last & 1) != grp) {
            if (!(ok = warp_wait(&m_full[qd * 2 + (last & 1)], (last >> 1) & 1))) break;
            const float m_end = m_sh[row];
            if (m_ref != m_end) {
              l_run *= ex2_approx(m_ref - m_end);
              m_ref = m_end;
            }
          }
          volatile float* l2 = l_sh + (item & 1) * 256;
          l2[grp * 128 + row] = l_run;
          __syncwarp();
          if (lane == 0) mbar_arrive(&l_full[qd]);
          if (!(ok = warp_wait(&l_full[qd], item & 1))) break;
          l_run = l2[row] + l2[128 + row];
        }
        // (product last - 4 is complete: the group of unit `last` saw it at unit last - 2)
        if (!(ok = pv_wait(last))) break;
        tc_after();
        const bool whole = at.u == 0 && last + 1 - begin_i == at.of;
        const int slot = 2 * blockIdx.x + (begin_i > 0 ? 1 : 0);   // the CTA's first part, or a later one
        if (tid == 0 && at.u == 0 && !whole)
          a.desc[blockIdx.x] = make_int4(slot, range_of(st.units, pos + at.of - 1, st.ctas), at.b << 10 | at.head, at.tile);
        pos += last + 1 - begin_i + kItemCost;
        if (any) {
          const bool sees = lim > 0;
          const float inv = 1.f / l_run;
          const int64_t tok = at.r.q0 + t;
          const int head = at.head * a.group + hl;
          const uint16_t* g_row = a.gate + tok * a.g_tok + head * a.g_head;
          uint16_t* o_row = a.out + tok * a.o_tok + head * a.o_head;
          float* p_row = a.part + (static_cast<int64_t>(slot) * 128 + row) * HD;
          const bool gate = whole && a.gate && valid;
          uint4 g0, g1;   // the gate's next 16 dims, in flight
          constexpr int CN = HD / 16 / NG;
          if (gate) {
            g0 = __ldg(reinterpret_cast<const uint4*>(g_row + grp * CN * 16));
            g1 = __ldg(reinterpret_cast<const uint4*>(g_row + grp * CN * 16 + 8));
          }
#pragma unroll 1
          for (int c = grp * CN; c < (grp + 1) * CN; ++c) {
            const uint32_t gw[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
            if (gate && c + 1 < (grp + 1) * CN) {
              g0 = __ldg(reinterpret_cast<const uint4*>(g_row + c * 16 + 16));
              g1 = __ldg(reinterpret_cast<const uint4*>(g_row + c * 16 + 24));
            }
            uint32_t r[16];
            tc_ld16(tmem + lanes + C::kColO + c * 16, r);
            tc_wait_ld();
            if (!valid) continue;
            if (!whole) {
              uint4* dst = reinterpret_cast<uint4*>(p_row + c * 16);
#pragma unroll
              for (int j = 0; j < 4; ++j) dst[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
            } else {
              uint32_t w[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float v0 = sees ? __uint_as_float(r[2 * j]) * inv : 0.f, v1 = sees ? __uint_as_float(r[2 * j + 1]) * inv : 0.f;
                if (gate) {
                  const float2 y = unpack2<BF>(gw[j]);
                  v0 = gated(v0, y.x);
                  v1 = gated(v1, y.y);
                }
                w[j] = pack2<BF>(v0, v1);
              }
              uint4* dst = reinterpret_cast<uint4*>(o_row + c * 16);
              dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
              dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
          if (!whole && valid && grp == 0) a.ml[slot * 128 + row] = make_float2(m_ref, l_run);
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free);
      }
      if (!more || *abort_flag) break;
      at = next;
      ++item;
      // one item, or this CTA's part of it: units i .. last
      begin_i = i;
      last = i + min(at.of - at.u, n - i) - 1;
      const int tn = at.tile * tt + t_in;
      const bool here = t_in < tt && tn < at.r.n;
      const int lim_n = here ? max(0, min(at.r.keys, at.r.kv - at.r.n_all + tn + 1)) : 0;   // keys < lim_n
      const int all = seen_by_all(at);
      const bool run = __any_sync(0xffffffffu, here);
      // m_ref: the row's reference maximum as this group last knew it, its sum relative to it
      m_ref = -INFINITY;
      l_run = 0.f;
      if (last + 1 < n) next_item(next);
      for (; i <= last && ok; ++i) {
        if (NG == 2 && (i & 1) != grp) continue;
        const int b = i & 1, pb = PB == 2 ? b : 0, k0 = (at.u + i - begin_i) * 64;
        if (!(ok = warp_wait(&s_full[b], (i >> 1) & 1))) break;
        tc_after();
        const int rem = lim_n - k0;
        float mt = -INFINITY;
        uint32_t r0[32], r1[32];   // the unit's scores
        if (run) {
          if (k0 + 64 > all) {   // some row does not see the whole unit: -inf in place
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t r[16];
              tc_ld16(tmem + lanes + C::kColS + b * 64 + c * 16, r);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) r[j] = c * 16 + j < rem ? r[j] : 0xFF800000u;
              tc_st16(tmem + lanes + C::kColS + b * 64 + c * 16, r);
            }
            tc_wait_st();
          }
          tc_ld32(tmem + lanes + C::kColS + b * 64, r0);
          tc_ld32(tmem + lanes + C::kColS + b * 64 + 32, r1);
          tc_wait_ld();
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[b]);
        if (run) {
          float mx[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) mx[x] = fmaxf(__uint_as_float(r0[x]), __uint_as_float(r1[x]));
#pragma unroll
          for (int j = 4; j < 32; j += 4) {
#pragma unroll
            for (int x = 0; x < 4; ++x) mx[x] = fmaxf(mx[x], fmaxf(__uint_as_float(r0[j + x]), __uint_as_float(r1[j + x])));
          }
          mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        }
        // the row's reference maximum after the unit before this one (every unit waits for the
        // one before, so the phases come one at a time)
        float m_old = m_ref;
        if (NG == 2 && i > 0) {
          if (!(ok = warp_wait(&m_full[qd * 2 + (b ^ 1)], ((i - 1) >> 1) & 1))) break;
          if (i > begin_i) m_old = m_sh[row];
        }
        const bool grows = mt > m_old + 8.f || (m_old == -INFINITY && mt > -INFINITY);
        float m_new = m_old;
        if (__any_sync(0xffffffffu, grows)) {
          if (grows) m_new = mt;
          if (i > begin_i) {
            const float cor = m_old == m_new ? 1.f : ex2_approx(m_old - m_new);
            if (!(ok = pv_wait(i - 1))) break;   // O is at rest (product i - 5 is complete: see kPvRing)
            tc_after();
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t r[16];
              tc_ld16(tmem + lanes + C::kColO + c * 16, r);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * cor);
              tc_st16(tmem + lanes + C::kColO + c * 16, r);
            }
            tc_wait_st();
          }
        }
        const bool edge = run && all < min(k0 + 64, at.r.keys);   // some row does not see the unit whole
        if (NG == 2) {
          m_sh[row] = m_new;
          tc_before();
          __syncwarp();
          if (!edge && lane == 0) mbar_arrive(&m_full[qd * 2 + b]);   // (edge: below, when O is complete)
        }
        if (m_ref != m_new) {
          l_run *= ex2_approx(m_ref - m_new);
          m_ref = m_new;
        }
        const float off = m_ref == -INFINITY ? 0.f : -m_ref;
        // the P buffer is free once the product that read it is done (product i - PB - 4 is
        // complete: this group saw it at unit i - 4)
        if (i >= PB && !(ok = pv_wait(i - PB))) break;
        if (run) {
          float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 sc2 = make_float2(sc, sc), off2 = make_float2(off, off);
          auto weights = [&](const uint32_t (&r)[32], int c) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                // 2^(scale log2(e) s - m); a masked key's -inf gives 0
                const float2 z = fma2(make_float2(__uint_as_float(r[8 * x + 2 * j]), __uint_as_float(r[8 * x + 2 * j + 1])), sc2, off2);
                w[j] = pack2<BF>(ex2_approx(z.x), ex2_approx(z.y));
                // the sum is taken over the rounded weights: what rounding does to all of a row's
                // weights alike cancels in the quotient
                sums[j & 1] = add2(sums[j & 1], unpack2<BF>(w[j]));
              }
              *reinterpret_cast<uint4*>(sm + C::kOffP + pb * C::kPBytes + sw128(row, c * 4 + x)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          };
          weights(r0, 0);
          weights(r1, 1);
          const float2 t2 = add2(sums[0], sums[1]);
          l_run += t2.x + t2.y;
        }
        fence_proxy_async_smem();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
        if (edge) {
          // bad values that were taken out of V, for the rows that see them
          if (!(ok = pv_wait(i))) break;   // (product i - 4 is complete: seen at unit i - 4 + PB)
          tc_after();
          if (bad[i & 7] == i + 1)
            restore_bad_values<CT, HD>(a, at.b, at.head, k0, at.r.keys, lim_n, sm + C::kOffP + pb * C::kPBytes, row,
                                       tmem + lanes + C::kColO);
          tc_before();
          __syncwarp();
          if (NG == 2 && lane == 0) mbar_arrive(&m_full[qd * 2 + b]);
        }
      }
      if (!ok) break;
    }
    if (!ok) fail();
  } else {
    reg_dec<C::kRegsOther>();
    if (warp < C::kPvWarp) {
      // --------------------------------------------------------------- S = Q K^T
      if (lane == 0) {
        bool ok = true;
        int left = min(at.of - at.u, n), item = 0;
        bool starts = true;
        for (int i = 0; i < n && ok && !*abort_flag; ++i) {
          const int slot = i % RH, b = i & 1;
          if (NG == 1 || b == warp - C::kQkWarp) {   // (two warps: the units in turn)
            if (!(ok = thread_wait(&s_free[b], ((i >> 1) & 1) ^ 1))) break;
            if (!(ok = thread_wait(Q8 ? &full[slot] : &landed[slot], (i / RH) & 1))) break;
            // the turn first: it says that Q of the item before has come, so that the wait for this
            // item's Q is for the next phase
            if (NG == 2 && i > 0 && !(ok = thread_wait(&turn[b ^ 1], ((i - 1) >> 1) & 1))) break;
            if (starts && !(ok = thread_wait(q_full, item & 1))) break;
            tc_after();
            const uint64_t kd = sw128_desc(sbase + slot * C::kHalf);
            const uint64_t qd = C::kQTmem ? 0ull : sw128_desc(sbase + C::kOffQ);
#pragma unroll 1
            for (int x = 0; x < HD / 64; ++x) {   // (a loop over the atoms: see the note on code size)
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint64_t bd = kd + (x * 8192 + y * 32) / 16;   // the address field, in 16-byte units
                if constexpr (C::kQTmem)
                  tc_mma_ts(tmem + C::kColS + b * 64, tmem + C::kColQ + x * 32 + y * 8, bd, C::kIdescQK, x + y > 0 ? 1u : 0u);
                else
                  tc_mma(tmem + C::kColS + b * 64, qd + (x * 16384 + y * 32) / 16, bd, C::kIdescQK, x + y > 0 ? 1u : 0u);
              }
            }
            if (NG == 2) {
              tc_before();
              mbar_arrive(&turn[b]);
            }
            tc_commit(&s_full[b]);
            tc_commit(&empty[slot]);
          }
          starts = --left == 0;
          if (starts && i + 1 < n) {
            next_item(at);
            left = at.of;
            ++item;
          }
        }
        if (!ok) fail();
        tc_commit(done);   // every issued MMA has completed before tensor memory is released
        if (!thread_wait(done, 0)) fail();
      }
    } else if (warp == C::kPvWarp) {
      // ---------------------------------------------------------------- O += P V
      bool ok = true;
      int left = min(at.of - at.u, n), item = 0, all = seen_by_all(at);
      bool starts = true;
      for (int i = 0; i < n && ok && !*abort_flag; ++i) {
        const int slot = RH + i % RH, pb = PB == 2 ? i & 1 : 0;
        if (starts && item > 0 && !(ok = warp_wait(o_free, (item - 1) & 1))) break;
        if (!(ok = warp_wait(Q8 ? &full[slot] : &landed[slot], (i / RH) & 1))) break;
        if (!Q8 && at.u * 64 + 64 > all) {   // not seen whole by some row, or with fewer than 64 keys
          // from the first key that some row does not see; a lane owns one chunk of every row
          // (of every second or fourth row)
          constexpr int CH = HD / 8, STEP = 32 / CH;
          const int valid = at.r.keys - at.u * 64, from = max(0, all - at.u * 64), ch = lane % CH;
          uint8_t* hc = sm + slot * C::kHalf + (ch >> 3) * 8192;
          bool any_bad = false;
#pragma unroll 2
          for (int key = from / STEP * STEP + lane / CH; key < 64; key += STEP) {
            uint4* p = reinterpret_cast<uint4*>(hc + sw128(key, ch & 7));
            const uint4 x = *p;
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            if (key >= valid) {
              *p = make_uint4(0u, 0u, 0u, 0u);
            } else if ((drop_bad<BF>(w[0]) | drop_bad<BF>(w[1]) | drop_bad<BF>(w[2]) | drop_bad<BF>(w[3])) && key >= from) {
              *p = make_uint4(w[0], w[1], w[2], w[3]);
              any_bad = true;
            }
          }
          if (any_bad) bad[i & 7] = i + 1;
          fence_proxy_async_smem();
        }
        if (!(ok = warp_wait(&p_full[i & 1], (i >> 1) & 1))) break;
        tc_after();
        if (lane == 0) {
          const uint64_t pd = sw128_desc(sbase + C::kOffP + pb * C::kPBytes);
          const uint64_t vd = sw128_desc_mn(sbase + slot * C::kHalf, 8192);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc_mma(tmem + C::kColO, pd + k * 2, vd + k * 128, C::kIdescPV, (!starts || k > 0) ? 1u : 0u);
          tc_commit(pv_bar(i));
          tc_commit(&empty[slot]);
        }
        __syncwarp();
        ++at.u;
        starts = --left == 0;
        if (starts && i + 1 < n) {
          next_item(at);
          left = at.of;
          all = seen_by_all(at);
          ++item;
        }
      }
      if (!ok) fail();
      if (lane == 0) {
        tc_commit(done);
        if (!thread_wait(done, 0)) fail();
      }
    } else if (warp < C::kLoadWarp + C::kLoaders) {
      // ------------------------------------------------------------------ loader
      // Halves in MMA order: per unit K(i) then V(i - 1), or V(i - 1) first where unit i
      // starts an item.  A lane owns one TMA box of a half: 64 dims (int8: all) of the keys
      // of one page.
      constexpr int ATOMS = Q8 ? 1 : HD / 64, LR = Q8 ? C::kRaw : RING, NL = C::kLoaders;
      const int rows = min(a.c.page_size, 64), box = lane * NL + warp - C::kLoadWarp, part = box / ATOMS, atom = box % ATOMS;
      const bool mine = part * rows < 64;
      const int row_bits = min(a.shift, 6);   // log2(rows)
      // bytes of this warp's boxes
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * rows * (Q8 ? HD : 128);
      // Page ids come from two windows of 32 table entries, a lane holding one of each: the
      // second is in flight while the first is used.
      int w_req = -1, w0 = 0, cur = -1, nxt = -1;
      auto entry = [&](int b, int i) { return i < a.width ? a.table[b * a.table_ld + i] : -1; };
      auto page_of = [&](const Pos& p) -> int {   // of this lane's box; -1: outside the pool, read as 0
        const int first = (p.u * 64) >> a.shift, base = first & ~31;   // (a unit's pages share a window)
        if (p.b != w_req || base != w0) {
          if (p.b == w_req && base == w0 + 32) {
            cur = nxt;
          } else {
            cur = entry(p.b, base + lane);
          }
          w_req = p.b;
          w0 = base;
          nxt = entry(p.b, base + 32 + lane);
        }
        const int key = p.u * 64 + part * rows;
        const int page = __shfl_sync(0xffffffffu, cur, ((mine ? key : p.u * 64) >> a.shift) & 31);
        return mine && key < p.r.keys ? page : -1;
      };
      int h = 0;
      bool ok = true;
      auto load = [&](bool v, int unit, const auto& x) {
        const int page = x.page, u = x.u, head = x.head, keys = x.keys;
        const int slot = Q8 ? h % LR : (v ? RH : 0) + unit % RH, turn_of = Q8 ? h / LR : unit / RH;
        if (!(ok = warp_wait(Q8 ? &raw_free[slot] : &empty[slot], (turn_of & 1) ^ 1))) return;
        if (lane == 0) mbar_arrive_expect_tx(&landed[slot], bytes);
        __syncwarp();
        const int in = (u * 64 + part * rows) & (a.c.page_size - 1);
        uint8_t* dst = Q8 ? sm + C::kOffRaw + slot * C::kRawBytes + part * rows * HD
                          : sm + slot * C::kHalf + atom * 8192 + part * rows * 128;
        if (mine) tma_load_4d(dst, v ? &v_map : &k_map, atom * 64, in, head, page, &landed[slot]);
        if constexpr (Q8) {
          // one row of scales a lane and 32 keys: a page's address, then constants of the lane
          const uint16_t* sc = static_cast<const uint16_t*>(v ? a.c.v_scale : a.c.k_scale) +
                               head * (v ? a.c.vs_stride[1] : a.c.ks_stride[1]);
          const int64_t s_page = v ? a.c.vs_stride[0] : a.c.ks_stride[0], s_slot = v ? a.c.vs_stride[2] : a.c.ks_stride[2];
          const uint32_t sb = sbase + C::kOffRaw + slot * C::kRawBytes + C::kRawHalf + lane * (HD / 16);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int key = u * 64 + x * 32 + lane;
            const int pg = __shfl_sync(0xffffffffu, page, (x * 32 + lane) >> row_bits);
            const bool in_pool = key < keys && pg >= 0 && pg < a.c.pages;
            const int at_page = in_pool ? pg : 0;
            cp_async_small<HD / 16>(sb + x * 32 * (HD / 16), sc + at_page * s_page + (key & (a.c.page_size - 1)) * s_slot, in_pool);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_u32(&landed[slot])) : "memory");
        }
        ++h;
      };
      struct Half {
        int page, u, head, keys;
      };
      auto half_of = [&](const Pos& p) { return Half{page_of(p), p.u, p.head, p.r.keys}; };
      // i Ks are out and v Vs; K(i) is next unless two Vs are owed, or one and unit i starts an item
      Half k = half_of(at), v1{}, v2{};
      int i = 0, v = 0, left = min(at.of - at.u, n);
      bool starts = true;
      while (v < n && ok && !*abort_flag) {
        const bool is_v = i - v == 2 || (i - v == 1 && (starts || i == n));
        load(is_v, is_v ? v : i, is_v ? (i - v == 2 ? v2 : v1) : k);
        if (is_v) {
          ++v;
          continue;
        }
        ++i;
        v2 = v1;
        v1 = k;
        starts = --left == 0;
        if (i < n) {
          if (starts) {
            next_item(at);
            left = at.of;
          } else {
            ++at.u;
          }
          k = half_of(at);   // the page id is in flight while the ring is full
        }
      }
      if (!ok) fail();
      if (!ok || *abort_flag) {   // no copy may still be in flight when the CTA ends
        if constexpr (Q8) cp_async_wait_all();
        if constexpr (Q8) {
          for (int f = max(0, h - LR); f < h; ++f) thread_wait(&landed[f % LR], (f / LR) & 1);
        } else {
          for (int f = max(0, i - RH); f < i; ++f) thread_wait(&landed[f % RH], (f / RH) & 1);
          for (int f = max(0, v - RH); f < v; ++f) thread_wait(&landed[RH + f % RH], (f / RH) & 1);
        }
      }
    } else if (Q8 && warp >= C::kConvWarp) {
      // -------------------------------------------------------------- converters
      const int hw = warp - C::kConvWarp;
      bool ok = true;
      if constexpr (Q8) {
        constexpr int CPK = HD / 16;   // 16-byte chunks of a cached row
        int h = 0;
        auto convert = [&](bool v, int unit, int valid, bool edge) {
          const int slot = (v ? RH : 0) + unit % RH, rs = h % C::kRaw;
          if (!(ok = warp_wait(&landed[rs], (h / C::kRaw) & 1)) || !(ok = warp_wait(&empty[slot], ((unit / RH) & 1) ^ 1))) return;
          // A lane converts the same chunk of every KEYS-th key: KEYS is a multiple of 8, so the
          // swizzle is a constant of the lane and everything moves by constants.
          constexpr int PER = 64 * CPK / 128, KEYS = 128 / CPK;
          const int id = hw * 32 + lane, key0 = id / CPK, ch = id % CPK;   // 16 dims: 16-bit chunks 2 ch, 2 ch + 1
          const uint32_t raw = sbase + C::kOffRaw + rs * C::kRawBytes;
          uint32_t src = raw + id * 16, scl = raw + C::kRawHalf + key0 * (HD / 16) + (ch >> 1) * 2;
          const uint32_t base = sbase + slot * C::kHalf + (ch >> 2) * 8192;
          uint32_t lo = base + sw128(key0, (2 * ch) & 7), hi = base + sw128(key0, ((2 * ch) & 7) + 1);
#pragma unroll 2
          for (int x = 0; x < PER; ++x) {
            const uint4 w = ls128(src);
            uint32_t s2 = ls16(scl);
            s2 = key0 + x * KEYS < valid ? s2 | s2 << 16 : 0u;   // rows past the last key: +-0
            st128(lo, dq2(w.x, 0x5140u, s2), dq2(w.x, 0x7362u, s2), dq2(w.y, 0x5140u, s2), dq2(w.y, 0x7362u, s2));
            st128(hi, dq2(w.z, 0x5140u, s2), dq2(w.z, 0x7362u, s2), dq2(w.w, 0x5140u, s2), dq2(w.w, 0x7362u, s2));
            src += 128 * 16;
            scl += KEYS * (HD / 16);
            lo += KEYS * 128;
            hi += KEYS * 128;
          }
          bool any_bad = false;
          if (edge) {   // the same chunks again: what must not reach the product
#pragma unroll 1
            for (int x = 0; x < 2 * PER; ++x) {
              const uint32_t at_w = (x & 1 ? hi : lo) - (x / 2 + 1) * KEYS * 128;
              const uint4 v = ls128(at_w);
              uint32_t o[4] = {v.x, v.y, v.z, v.w};
              if (drop_bad<false>(o[0]) | drop_bad<false>(o[1]) | drop_bad<false>(o[2]) | drop_bad<false>(o[3])) {
                st128(at_w, o[0], o[1], o[2], o[3]);
                any_bad = true;
              }
            }
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
        struct Half {
          int valid, edge;
        };
        auto half_of = [&](const Pos& p) {
          return Half{p.r.keys - p.u * 64, seen_by_all(p) < min(p.u * 64 + 64, p.r.keys)};
        };
        Half k = half_of(at), v1{}, v2{};   // order of the halves: see the loader
        int i = 0, v = 0, left = min(at.of - at.u, n);
        bool starts = true;
        while (v < n && ok && !*abort_flag) {
          const bool is_v = i - v == 2 || (i - v == 1 && (starts || i == n));
          const Half x = is_v ? (i - v == 2 ? v2 : v1) : k;
          convert(is_v, is_v ? v : i, x.valid, is_v && x.edge);
          if (is_v) {
            ++v;
            continue;
          }
          ++i;
          v2 = v1;
          v1 = k;
          starts = --left == 0;
          if (i < n) {
            if (starts) {
              next_item(at);
              left = at.of;
            } else {
              ++at.u;
            }
            k = half_of(at);
          }
        }
      }
      if (!ok) fail();
    }
  }

  tc_before();
  __syncthreads();
  if (warp == C::kQkWarp) {
    tc_after();
    tc_dealloc(tmem, C::kTmem);
  }
  // The rows form's kernel may run beside this one; the joining kernel waits for this one
  // only, so this one does not end before it.
  griddep_wait();
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
int launch_tiles(AttnArgs a, void* area, uint32_t* err, int sms, bool after_rows, cudaStream_t stream, SplitSet* set) {
  using C = TilesCfg<CT, HD>;
  static std::atomic<uint64_t> done{0};
  if (!setup_kernel(reinterpret_cast<const void*>(paged_tiles_kernel<CT, HD>), C::kSmem, done)) return TLX_ERR_LAUNCH;
  const int ctas = sms * C::kCtas;
  a.by_item = 0;
  *set = set_split(a, area, ctas, 128);
  set->items = ctas;
  set->rows = 128;
  CUtensorMap km, vm;
  if (!page_map(&km, a.c, a.c.k, a.c.k_stride) || !page_map(&vm, a.c, a.c.v, a.c.v_stride)) return TLX_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_rows ? 1 : 0;
  void* args[] = {&a, &km, &vm, &err};
  return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(paged_tiles_kernel<CT, HD>), args) == cudaSuccess
             ? TLX_OK
             : TLX_ERR_LAUNCH;
}

}  // namespace

template <int CT>
static int launch_tiles_hd(const AttnArgs& a, void* area, uint32_t* err, int sms, bool after_rows, cudaStream_t stream,
                           SplitSet* set) {
  if (a.c.head_dim == 256) return launch_tiles<CT, 256>(a, area, err, sms, after_rows, stream, set);
  if (a.c.head_dim == 128) return launch_tiles<CT, 128>(a, area, err, sms, after_rows, stream, set);
  return launch_tiles<CT, 64>(a, area, err, sms, after_rows, stream, set);
}

int launch_paged_tiles(const AttnArgs& a, int ct, void* area, uint32_t* err, int sms, bool after_rows, cudaStream_t stream,
                       SplitSet* set) {
  if (ct == CT_F16) return launch_tiles_hd<CT_F16>(a, area, err, sms, after_rows, stream, set);
  if (ct == CT_BF16) return launch_tiles_hd<CT_BF16>(a, area, err, sms, after_rows, stream, set);
  return launch_tiles_hd<CT_Q8>(a, area, err, sms, after_rows, stream, set);
}

size_t paged_tiles_bytes(int hd, int sms) {
  return (split_area(sms * (hd == 256 ? 1 : 2), 128, hd).end + 255) & ~size_t(255);   // kCtas at most
}

}  // namespace tlx

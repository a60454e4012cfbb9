// Sums of the tiles form's schedule, for the device and for tests on the host.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define TLX_SCHED static __host__ __device__ __noinline__   // (64-bit arithmetic, kept out of the callers' code)
#else
#define TLX_SCHED static inline
#endif

namespace tlx {

// sum over i < n of floor((a i + b) / m): the Euclid-like recursion, as a loop
TLX_SCHED int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
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

// Units of 64 keys in the first `tiles` tiles of a request of n rows, tt rows a tile, whose row t
// sees min(c + t + 1, keys) keys (none below 0).  A tile has the units of its last row, at least 1.
TLX_SCHED int64_t units_before(int64_t c, int tt, int n, int keys, int tiles) {
  auto units = [&](int64_t last) -> int64_t {
    const int64_t seen = c + last < keys ? c + last : keys;
    return seen > 64 ? (seen + 63) / 64 : 1;
  };
  const int64_t full = tiles < n / tt ? tiles : n / tt;   // tiles with all their rows
  auto within = [&](int64_t x, int64_t lo) { return x < lo ? lo : x > full ? full : x; };
  int64_t one = 0, top = full;
  if (c < 0 || c + full * tt > keys) {
    // tiles [0, one) see at most 64 keys, tiles from top on all of them
    one = 64 > c ? within((64 - c) / tt, 0) : 0;
    top = keys > c ? within((keys - c + tt - 1) / tt - 1, one) : one;
  }
  int64_t s = one;
  if (top > one) s += floor_sum(top - one, 64, tt, c + (one + 1) * tt + 63);
  if (full > top) s += (full - top) * units(keys - c);
  if (tiles > full) s += units(n);   // the last tile, with fewer rows
  return s;
}

}  // namespace tlx

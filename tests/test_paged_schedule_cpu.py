"""The tiles form's schedule: the units of a request's first tiles in closed form, against tile
by tile, for every way in which the keys can run out (nothing cached, more new rows than keys,
a planned request that got no pages, a table too narrow for the length); and a prompt of many
tiles without keys, whose sum must not take time by the tile."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "thunderllamax_b200", "csrc")
PROGRAM = r"""
#include "paged_schedule.h"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
static int64_t tile_by_tile(int64_t c, int64_t tt, int64_t n, int64_t keys, int64_t tiles) {
  int64_t s = 0;
  for (int64_t i = 0; i < tiles; ++i) {
    const int64_t seen = std::min(std::max(c + std::min((i + 1) * tt, n), int64_t(0)), keys);
    s += std::max(int64_t(1), (seen + 63) / 64);
  }
  return s;
}
int main() {
  std::mt19937_64 rng(1);
  auto pick = [&](int64_t lo, int64_t hi) { return lo + int64_t(rng() % uint64_t(hi - lo + 1)); };
  const int tts[] = {1, 2, 4, 5, 10, 16, 21, 32, 42, 63, 64, 65, 100, 127, 128};
  for (int k = 0; k < 400000; ++k) {
    const int tt = tts[pick(0, 14)];
    const int n = int(pick(1, k % 3 ? 300 : 5000));
    const int n_all = n + (k % 5 ? 0 : int(pick(0, 200)));           // rows past max_new
    int64_t kv = n_all + pick(0, k % 2 ? 200 : 4000);
    if (k % 7 == 0) kv = pick(0, n_all);                             // more rows than keys
    if (k % 11 == 0) kv = 0;                                         // no pages
    const int64_t keys = k % 4 ? kv : pick(0, kv);                   // a narrow table
    const int tiles = int(pick(0, (n + tt - 1) / tt));
    const int64_t got = tlx::units_before(kv - n_all, tt, n, int(keys), tiles);
    const int64_t want = tile_by_tile(kv - n_all, tt, n, keys, tiles);
    if (got != want) {
      std::printf("kv %lld n_all %d n %d tt %d keys %lld tiles %d: %lld, not %lld\n", (long long)kv, n_all, n, tt,
                  (long long)keys, tiles, (long long)got, (long long)want);
      return 1;
    }
  }
  // the largest prompt, one row a tile: no keys, fewer keys than rows, a narrow table
  const int n = 1 << 28;
  int64_t sum = 0;
  for (int k = 0; k < 1000; ++k)
    sum += tlx::units_before(-int64_t(n), 1, n, 0, n - k) + tlx::units_before(-int64_t(n) / 2, 1, n, n / 2, n - k) +
           tlx::units_before(0, 1, n, 1000, n - k);
  std::printf("%lld\n", (long long)sum);
  const int64_t none = tlx::units_before(-int64_t(n), 1, n, 0, n);
  return none == n ? 0 : 2;
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="needs g++")
def test_units_in_closed_form(tmp_path):
    src = tmp_path / "schedule.cpp"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "schedule")
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{CSRC}", str(src), "-o", exe], check=True)
    got = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0, got.stdout

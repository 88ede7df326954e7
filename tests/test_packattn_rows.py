"""The rows that the gradient of a packed sequence's keys goes over: against a
count of them, and within 32 bits for every number of tokens that a call takes
(a constant expression that overflows does not compile)."""
import shutil
import subprocess

import pytest

from bindcraft2_amd import build

PROGRAM = r"""
#include "packrows.h"
using namespace bc2n;

constexpr int TILE = 64;
constexpr bool counted(bool causal, int lq, int lk, int G, int capacity) {
  for (int j0 = 0; j0 < capacity; j0 += 128) {
    const KeyRows r = rows_of_keys(causal, j0, lq, lk, G, TILE);
    if (j0 >= lk) {
      if (r.all || r.first || r.blind) return false;
      continue;
    }
    int first = lq * G, blind = 0;
    for (int row = lq * G - 1; row >= 0; --row) {
      const int last = causal ? row / G + lk - lq : lk - 1;
      if (last >= j0) first = row;
      if (last < 0) ++blind;
    }
    if (first_row(causal, j0, lq, lk, G) != first) return false;
    if (r.all != lq * G || r.blind != blind || r.first % TILE || r.first > first || r.first + TILE <= first)
      return false;
    for (int parts = 1; parts < 6; ++parts) {
      int at = r.first;
      for (int p = 0; p < parts; ++p) {
        const Part x = part_of_rows(r, parts, p, TILE);
        if (x.from != at || x.to < x.from) return false;
        at = x.to;
      }
      if (at != r.all) return false;
    }
  }
  return true;
}
static_assert(counted(true, 70, 70, 2, 300), "");
static_assert(counted(true, 100, 40, 3, 300), "");
static_assert(counted(true, 5, 300, 4, 500), "");
static_assert(counted(true, 0, 130, 4, 500), "");
static_assert(counted(true, 30, 0, 4, 500), "");
static_assert(counted(false, 90, 200, 3, 600), "");

// tokens * G below 2^31 - 2^14, of queries and of keys' capacity
constexpr bool fits(bool causal, int G, int lq, int lk, int capacity) {
  const int at[] = {0, lk / 2, lk - 1, lk, lk + 1, capacity / 2, capacity - 1};
  for (int j : at) {
    const int j0 = (j < 0 ? 0 : j) / 128 * 128;
    const KeyRows r = rows_of_keys(causal, j0, lq, lk, G, TILE);
    if (r.first < 0 || r.first > r.all + TILE || r.blind < 0) return false;
    for (int on : {0, 31, 127}) {
      const int x = first_row(causal, j0 + on, lq, lk, G);
      if (x < 0 || x > lq * G) return false;
    }
    for (int parts : {1, 2, 7, 64})
      for (int p = 0; p < parts; ++p) {
        const Part x = part_of_rows(r, parts, p, TILE);
        if (x.from < 0 || x.to < x.from || x.to > r.all) return false;
      }
  }
  return true;
}
constexpr int MOST = 0x7fffffff - (1 << 14);
constexpr bool every(bool causal) {
  for (int G : {1, 2, 3, 8, 32, 128}) {
    const int n = MOST / G;
    const int lengths[] = {0, 1, 100, n / 2, n - 1, n};
    for (int lq : lengths)
      for (int lk : lengths)
        if (!fits(causal, G, lq, lk, n)) return false;
  }
  return true;
}
static_assert(every(true), "");
static_assert(every(false), "");
"""


@pytest.mark.skipif(not shutil.which(build.HIPCC), reason="no hipcc")
def test_rows(tmp_path):
    src = tmp_path / "rows.hip"
    src.write_text(PROGRAM)
    r = subprocess.run([build.HIPCC, "-x", "hip", f"--offload-arch={build.ARCH}", "-std=c++17", "--cuda-host-only",
                        "-fsyntax-only", "-fconstexpr-steps=100000000", "-I", build.CSRC, str(src)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]

"""The search over the starts of packed sequences (``csrc/sequences.h``),
compiled for the host: a tile lies within the rows that there are whatever the
starts hold, and ascending starts have every row in one tile of its own
sequence."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / 'bevfusion-triton_amd' / 'csrc'

PROGRAM = r'''
#include <cstdio>
#include <random>
#include <vector>
#include "sequences.h"
using namespace sequences;

struct Wave {  // 64 lanes in turn
  template <typename Ok>
  int count(Ok ok) const {
    int n = 0;
    for (int lane = 0; lane < 64; ++lane) n += ok(lane);
    return n;
  }
  int uniform(int v) const { return v; }
};

static int bad = 0;
static void report(const char *what, const std::vector<int32_t> &q, int total, int group, int tile,
                   int index) {
  if (++bad > 20) return;
  std::printf("%s: starts", what);
  for (size_t i = 0; i < q.size() && i < 12; ++i) std::printf(" %d", q[i]);
  std::printf(" total %d group %d tile %d index %d\n", total, group, tile, index);
}

// Every tile of a call; with `exact` (starts ascend within the rows) every row
// in one tile, of the sequence that it belongs to.
static void check(const std::vector<int32_t> &q, const std::vector<int32_t> &k, int tq, int tk,
                  int group, int tile, bool causal, bool exact) {
  const int n = int(q.size()) - 1;
  const Starts s = {q.data(), k.data(), n, tq, tk};
  const Group g = make_group(group);
  std::vector<int> rows(size_t(tq) * group, 0), keys(tk, 0);
  const int row_tiles = int(int64_t(tq) * group / tile) + n + 1;
  for (int index = 0; index < row_tiles; ++index) {
    const RowTile t = row_tile(s, group, tile, index, Wave{});
    if (!t.on) continue;
    // (what the kernels form of it: the first row, the last, and their queries)
    const int last = (t.r0 + tile < t.rows ? t.r0 + tile : t.rows) - 1;
    if (t.r0 < 0 || last < t.r0 || t.seq.q0 < 0 || t.seq.q0 + g.div(t.r0) >= tq ||
        g.div(t.r0) < 0 || g.div(last) < 0 || t.seq.q0 + g.div(last) >= tq || t.seq.k0 < 0 ||
        t.seq.nk < 0 || t.seq.k0 + t.seq.nk > tk) {
      report("rows", q, tq, group, tile, index);
      continue;
    }
    for (int r = t.r0; r <= last; ++r) {
      if (g.div(r) != r / group) report("division", q, tq, group, tile, index);
      const size_t at = size_t(t.seq.q0 + r / group) * group + r % group;
      ++rows[at];
      if (!exact || r % 7) continue;
      int which = n;
      for (int i = 0; i < n; ++i)
        if (t.seq.q0 + r / group >= q[i] && t.seq.q0 + r / group < q[i + 1]) which = i;
      if (which < n ? t.seq.q0 != q[which] || t.seq.nk != k[which + 1] - k[which]
                    : t.seq.nk != 0 && t.seq.q0 != q[n])
        report("sequence", q, tq, group, tile, index);
    }
  }
  const int key_tiles = tk / tile + n + 1;
  for (int index = 0; index < key_tiles; ++index) {
    const KeyTile t = key_tile(s, group, causal, tile, 64, index, Wave{});
    if (!t.on) continue;
    const int last = (t.kb + tile < t.seq.nk ? t.kb + tile : t.seq.nk) - 1;
    if (t.kb < 0 || last < t.kb || t.seq.k0 < 0 || t.seq.k0 + last >= tk || t.begin < 0 ||
        t.begin > t.rows || t.begin % group || t.seq.q0 < 0 ||
        t.seq.q0 + t.seq.nq > tq || t.rows != t.seq.nq * group ||
        t.tiles != (t.rows - t.begin + 63) / 64) {
      report("keys", k, tk, group, tile, index);
      continue;
    }
    for (int j = t.kb; j <= last; ++j) ++keys[t.seq.k0 + j];
  }
  if (!exact) return;
  for (int c : rows)
    if (c != 1) return report("row not once", q, tq, group, tile, -1);
  for (int c : keys)
    if (c != 1) return report("key not once", k, tk, group, tile, -1);
}

int main() {
  // a start that clamping, or a caller, put out of order
  check({0, 5000, -5}, {0, 5000, -5}, 5000, 5000, 4, 128, true, false);
  check({0, 1000, 100, 2000}, {0, 1000, 100, 2000}, 2000, 2000, 1, 64, true, false);
  check({0, 1000, 100, 2000}, {0, 1000, 100, 2000}, 2000, 2000, 4, 64, false, false);
  std::mt19937 gen(1);
  auto up_to = [&](int n) { return int(gen() % (n + 1)); };
  const int groups[] = {1, 2, 3, 4, 7, 8, 21, 40, 64, 129};
  for (int round = 0; round < 400; ++round) {
    const int n = round % 3 == 0 ? up_to(300) : up_to(8), group = groups[up_to(9)];
    const int tile = up_to(1) ? 64 : 128;
    const bool causal = up_to(1);
    // ascending, the ends of both within the rows
    std::vector<int32_t> q(n + 1, 0), k(n + 1, 0);
    for (int i = 0; i < n; ++i) {
      q[i + 1] = q[i] + (up_to(3) ? up_to(4) : up_to(300));
      k[i + 1] = k[i] + (up_to(3) ? up_to(4) : up_to(300));
    }
    const int tq = q[n] + (up_to(1) ? up_to(200) : 0), tk = k[n] + (up_to(1) ? up_to(200) : 0);
    check(q, k, tq, tk, group, tile, causal, true);
    // anything at all
    for (auto *s : {&q, &k})
      for (int i = 0; i <= n; ++i)
        if (up_to(2) == 0) {
          const int kind = up_to(4);
          (*s)[i] = kind == 0 ? INT32_MIN : kind == 1 ? INT32_MAX : kind == 2 ? -up_to(5000)
                  : kind == 3 ? up_to(tq + tk + 10) : up_to(1 << 30);
        }
    check(q, k, tq, tk, group, tile, causal, false);
  }
  return bad ? 1 : 0;
}
'''


def test_tiles_lie_within_the_rows(tmp_path):
    cxx = shutil.which('g++') or shutil.which('c++')
    if cxx is None:
        pytest.skip('no host C++ compiler')
    src, exe = tmp_path / 'sequences.cpp', tmp_path / 'sequences'
    src.write_text(PROGRAM)
    subprocess.run([cxx, '-std=c++17', '-O2', '-Wall', '-Werror', '-fsanitize=undefined',
                    '-fno-sanitize-recover=all', f'-I{CSRC}', str(src), '-o', str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr

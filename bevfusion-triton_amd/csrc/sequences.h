// Packed sequences and their tiles: the arithmetic by which a block finds what
// it works on (constexpr, so host and device code share it).
//
// Sequence i has the tokens [starts[i], starts[i + 1]).  The starts are read on
// the device alone, so nothing checks them before a launch.  Whatever they
// hold, a tile found here lies within the rows that there are: each start is
// clamped to them, and a tile that the search does not find (the starts do not
// ascend) is off.
#pragma once

#include <stdint.h>

namespace sequences {

// n / size for 0 <= n < 2^32 / size.
struct Group {
  int size;
  uint32_t magic;  // ceil(2^32 / size); 0 for 1
  constexpr int div(int n) const {
    return magic ? int((uint64_t(uint32_t(n)) * magic) >> 32) : n;
  }
};

constexpr Group make_group(int size) {
  return {size, size == 1 ? 0u : uint32_t(((uint64_t(1) << 32) + size - 1) / size)};
}

// starts[i] kept within the rows there are, whatever the array holds.
constexpr int start_at(const int32_t *starts, int i, int total) {
  if (i <= 0) return 0;
  const int v = starts[i];
  return v < 0 ? 0 : v > total ? total : v;
}

struct Starts {
  const int32_t *q, *k;  // n + 1 each
  int n, q_total, k_total;
};

struct Sequence {
  int q0, nq, k0, nk;
};

constexpr Sequence sequence_at(const Starts &s, int i) {
  Sequence x = {start_at(s.q, i, s.q_total), 0, start_at(s.k, i, s.k_total), 0};
  x.nq = i < s.n ? start_at(s.q, i + 1, s.q_total) - x.q0 : 0;
  x.nk = i < s.n ? start_at(s.k, i + 1, s.k_total) - x.k0 : 0;
  if (x.nq < 0) x.nq = 0;
  if (x.nk < 0) x.nk = 0;
  return x;
}

// Tiles of `tile` rows over sequences of starts[i + 1] - starts[i] tokens of
// `per` rows each, without a plan: sequence i's tiles are numbered from
// starts[i] * per / tile + i.  No two sequences' numbers meet, since
// floor(a) + ceil(b) <= floor(a + b) + 1, and all are below
// total * per / tile + n + 1, which the host knows.  Sequence n stands for
// the rows after the last one, which belong to none.
constexpr int first_tile(const int32_t *starts, int i, int total, int per, int tile) {
  return int(int64_t(start_at(starts, i, total)) * per / tile) + i;
}

// The sequence whose numbers `index` is among.  Each round narrows the range
// 64 times, so that any number of sequences takes a few loads.  The whole wave
// calls it: wave.count(ok) is the number of lanes for which ok(lane) holds,
// wave.uniform(v) v, the same in all lanes.  The count is the place of the
// last lane that holds only if the starts ascend; otherwise the first number
// of the sequence found may be above index.
template <typename Wave>
constexpr int find_sequence(const int32_t *starts, int n, int total, int per, int tile, int index,
                            Wave wave) {
  int low = 0, count = n + 1;
  for (;;) {
    const int step = (count + 63) / 64;
    const int taken = wave.count([&](int lane) {
      return lane * step < count &&
             first_tile(starts, low + lane * step, total, per, tile) <= index;
    });
    const int i = taken > 0 ? taken - 1 : 0;
    low += i * step;
    count = count - i * step < step ? count - i * step : step;
    if (step == 1) break;
  }
  return wave.uniform(low);
}

// Rows [r0, r0 + tile) of those of a sequence, (query, head of the group).
struct RowTile {
  Sequence seq;
  int rows, r0;
  bool on;
};
template <typename Wave>
constexpr RowTile row_tile(const Starts &s, int group, int tile, int index, Wave wave) {
  const int which = find_sequence(s.q, s.n, s.q_total, group, tile, index, wave);
  RowTile t = {sequence_at(s, which), 0, 0, false};
  if (which == s.n) t.seq.nq = s.q_total - t.seq.q0;  // rows of no sequence: no keys
  t.rows = t.seq.nq * group;
  t.r0 = (index - first_tile(s.q, which, s.q_total, group, tile)) * tile;
  t.on = t.r0 >= 0 && t.r0 < t.rows;
  return t;
}

// Keys [kb, kb + keys) of a sequence, and the rows from `begin` on that see one
// of them, in `tiles` tiles of tile_rows.
struct KeyTile {
  Sequence seq;
  int which, kb, begin, rows, tiles;
  bool on;
};
template <typename Wave>
constexpr KeyTile key_tile(const Starts &s, int group, bool causal, int keys, int tile_rows,
                           int index, Wave wave) {
  const int which = find_sequence(s.k, s.n, s.k_total, 1, keys, index, wave);
  KeyTile t = {sequence_at(s, which), which, 0, 0, 0, 0, false};
  if (which == s.n) t.seq.nk = s.k_total - t.seq.k0;  // keys of no sequence: no queries
  t.kb = (index - first_tile(s.k, which, s.k_total, 1, keys)) * keys;
  t.rows = t.seq.nq * group;
  if (causal) {  // key j is seen by the queries from j - (nk - nq) on
    const int seen_from = t.kb - (t.seq.nk - t.seq.nq);
    t.begin = (seen_from < 0 ? 0 : seen_from < t.seq.nq ? seen_from : t.seq.nq) * group;
  }
  t.tiles = (t.rows - t.begin + tile_rows - 1) / tile_rows;
  t.on = t.kb >= 0 && t.kb < t.seq.nk;
  return t;
}

}  // namespace sequences

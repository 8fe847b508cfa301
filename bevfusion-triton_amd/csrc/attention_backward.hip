// attention_backward.hip -- gradients of attention over packed sequences
// (gfx950).
//
// With P_ij = exp(s_ij - L_i) from the saved L and D_i = dout_i out_i:
//   dS_ij = P_ij (dout_i v_j - D_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
//   dv_j = sum_i P_ij dout_i
// Two kernels, one that owns rows of queries and one that owns keys, each
// sums in registers in one order: no atomics, so the result does not depend
// on the launch.  That costs seven matrix products instead of the five of a
// single pass that would add dq atomically.  The keys' kernel walks the rows
// of all heads of the group, so shared heads' gradients are summed there.
// P and dS are rounded to the operands' type before their products, as the
// matrix instructions ask; all else is fp32.
#include "attention_tiles.h"
#include "host_calls.h"

namespace {

using namespace attention;
using bevpool_host::check_grid;
using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

struct BackwardArgs : PackedArgs {
  const float2 *stats;  // (tokens, heads): L in units of log 2, and D
};

// D and L / log 2 of every (token, head): a row's 16-byte chunks on kLanes
// lanes.
template <typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void stats_kernel(PackedArgs A, float2 *stats) {
  constexpr int kPer = 16 / sizeof(T);
  const int64_t row = int64_t(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  const int chunk = threadIdx.x % kLanes;
  if (row >= int64_t(A.q_total) * A.q_heads) return;
  const int64_t token = row / A.q_heads, head = row - token * A.q_heads;
  float sum = 0.f;
  if (chunk < A.chunks) {
    typedef T Chunk __attribute__((ext_vector_type(16 / sizeof(T))));
    const Chunk o = *reinterpret_cast<const Chunk *>(A.out.at + token * A.out.row +
                                                     head * A.out.head + chunk * 16);
    const Chunk g = *reinterpret_cast<const Chunk *>(A.dout.at + token * A.dout.row +
                                                     head * A.dout.head + chunk * 16);
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += float(o[i]) * float(g[i]);
  }
#pragma unroll
  for (int m = 1; m < kLanes; m <<= 1) sum += __shfl_xor(sum, m, 64);
  if (chunk == 0) stats[row] = make_float2(A.lse[row] * kLog2e, sum);
}

// dq: rows and tiles as in the forward.
template <typename T, int DP, int kKeys>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && DP > 64 ? 1 : 2) void query_grad_kernel(
    BackwardArgs A) {
  using S = Shape<T, DP>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kTile = S::tile_bytes(kKeys);  // buffers: K0 V0 K1 V1
  constexpr int kRows = kWaves * kWaveRows;
  const int head = blockIdx.x % A.k_heads;
  const int index = A.tiles - 1 - int(blockIdx.x / A.k_heads);
  int first;
  const int which = find_sequence(A.q_starts, A.sequences, A.q_total, A.group.size, kRows, index,
                                  &first);
  Sequence seq = sequence_at(A.q_starts, A.k_starts, which, A.sequences, A.q_total, A.k_total);
  if (which == A.sequences) seq.nq = A.q_total - seq.q0;  // rows of no sequence: no keys
  const int rows = seq.nq * A.group.size;
  const int r0 = (index - first) * kRows;
  if (r0 >= rows) return;

  const int lane = lane_id(), wave = wave_id(), c = lane & 31, h = lane >> 5;
  const int row = r0 + wave * kWaveRows + c;
  const bool valid = row < rows;
  const int row_in = valid ? row : rows - 1;
  const int query = A.group.div(row_in);
  const int q_head = head * A.group.size + row_in - query * A.group.size;
  const int64_t token = seq.q0 + query;
  const int ahead = seq.nk - seq.nq;
  const int limit = A.causal ? min(seq.nk, query + ahead + 1) : seq.nk;
  const int last_query = A.group.div(min(r0 + kRows, rows) - 1);
  const int keys = A.causal ? max(0, min(seq.nk, last_query + ahead + 1)) : seq.nk;
  const int tiles = (keys + kKeys - 1) / kKeys;
  const int w0 = r0 + wave * kWaveRows;
  const int low = A.causal ? min(seq.nk, A.group.div(min(w0, rows - 1)) + ahead + 1) : seq.nk;
  const int high = A.causal
                       ? min(seq.nk, A.group.div(min(w0 + kWaveRows, rows) - 1) + ahead + 1)
                       : seq.nk;
  const bool wave_on = w0 < rows;

  Frags<T, DP> q, g;
  row_frags<T, DP>(q, A.q.at + token * A.q.row + q_head * A.q.head, A.chunks, true);
  row_frags<T, DP>(g, A.dout.at + token * A.dout.row + q_head * A.dout.head, A.chunks, true);
  const float2 both = A.stats[token * A.q_heads + q_head];
  float stat[2] = {both.x, both.y};
  settle(stat);
  const float lse2 = stat[0], delta = stat[1];
  const char *k_at = A.k.at + seq.k0 * A.k.row + head * A.k.head;
  const char *v_at = A.v.at + seq.k0 * A.v.row + head * A.v.head;
  const unsigned lds0 = lds_address(lds);
  Stage<T, DP, kKeys, kThreads> k_stage, v_stage;
  k_stage.set(A.chunks, [&](int r) { return r * int(A.k.row); });
  v_stage.set(A.chunks, [&](int r) { return r * int(A.v.row); });
  auto load_tile = [&](int t) {
    const unsigned to = lds0 + (t & 1) * 2 * kTile;
    load_rows(k_stage, k_at, A.k.row, t * kKeys, seq.nk, to);
    load_rows(v_stage, v_at, A.v.row, t * kKeys, seq.nk, to + kTile);
  };
  clear_rest<T, DP>(lds, 4 * kKeys, threadIdx.x, kThreads, A.chunks);

  Sums<T, DP> dq = {};
  if (tiles > 0) load_tile(0);
  for (int t = 0; t < tiles; ++t) {
    wait_loads<0>();
    __syncthreads();  // tile t is there, and tile t - 1 has been read
    if (t + 1 < tiles) load_tile(t + 1);
    const char *k_tile = lds + (t & 1) * 2 * kTile, *v_tile = k_tile + kTile;
    const int k0 = t * kKeys;
    if (!wave_on || k0 >= high) continue;
    const bool masked = k0 + kKeys > low;
#pragma unroll
    for (int b = 0; b < kKeys / 32; ++b) {
      Frags<T, DP> k, v;
      read_rows<T, DP>(k, k_tile, 32 * b);
      read_rows<T, DP>(v, v_tile, 32 * b);
      pin_reads();
      const f32x16 dots = dot_rows<T, DP>(k, q);
      const f32x16 dp = dot_rows<T, DP>(v, g);
      Columns<T, DP> kt;
      kt.read(k_tile, 32 * b);
      pin_reads();
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        p[r] = exp2_fast(fmaf(dots[r], A.scale_log2, -lse2)) * (dp[r] - delta);
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * b + c_row(r, h) >= limit) p[r] = 0.f;
      }
      Weights<T> w;
      w.set(p);
      kt.add(dq, w);
    }
  }
  store_row<T, DP>(A.dq.at + token * A.dq.row + q_head * A.dq.head, dq, A.scale, A.dim, valid);
}

// How the keys' kernel keeps a wave's 32 keys: their K and V fragments and
// both sums take 6 DP / 4 registers a lane in the 16-bit types (twice that in
// float).  Up to 6 * 128 bytes / 4 that leaves room for two waves a SIMD,
// which hide each other's waits; for heads of more than 192 bytes it does so
// with V in LDS, read again for every 32 rows.
template <typename T, int DP>
struct KeyPlan {
  static constexpr bool kTwoWaves = DP * sizeof(T) <= 256;
  static constexpr bool kValuesInLds = kTwoWaves && DP * sizeof(T) > 192;
  // Two groups of four waves with the same keys take the rows' tiles in
  // turn: a sequence's first keys are seen by all its rows, and the longest
  // walk is what the launch ends with.
  static constexpr int kGroups = kTwoWaves ? 2 : 1;
  static constexpr int kThreads = 256 * kGroups;
  static constexpr int kRows = 32;  // of a tile
  static constexpr int kTile = Shape<T, DP>::tile_bytes(kRows);
  // Three buffers of Q and dout rows: a tile's loads are given the time of
  // two tiles, as many rows come from beyond L2.  Behind them the rows' L and
  // D, in pairs.
  static constexpr int kBuffers = 3;
  static constexpr int kGroupLds = kBuffers * (2 * kTile + 8 * kRows);
  static constexpr int kValues =
      kValuesInLds ? Shape<T, DP>::tile_bytes(kWaves * kWaveRows) : 0;
  // (the second group's sums pass through LDS at the end)
  static constexpr int kSums = kGroups > 1 ? 256 * 64 * Shape<T, DP>::kBlocks : 0;
  static constexpr int kTiles = kGroups * kGroupLds + kValues;
  static constexpr int kLds = kTiles > kSums ? kTiles : kSums;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

// dk and dv: a wave owns 32 keys and walks the sequence's rows (query, head
// of the group) in tiles of 32, from the last to the first that sees one of
// its keys: blocks of one sequence start together there, and find each
// other's rows in L2.
template <typename T, int DP>
__global__ __launch_bounds__((KeyPlan<T, DP>::kThreads), 1) void key_grad_kernel(BackwardArgs A) {
  using Plan = KeyPlan<T, DP>;
  constexpr int kRows = Plan::kRows, kTile = Plan::kTile, kGroups = Plan::kGroups;
  constexpr int kSteps = Shape<T, DP>::kSteps, kBlocks = Shape<T, DP>::kBlocks;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kKeys = kWaves * kWaveRows;
  const int head = blockIdx.x % A.k_heads;
  const int index = int(blockIdx.x / A.k_heads);
  int first;
  const int which =
      find_sequence(A.k_starts, A.sequences, A.k_total, 1, kKeys, index, &first);
  Sequence seq = sequence_at(A.q_starts, A.k_starts, which, A.sequences, A.q_total, A.k_total);
  if (which == A.sequences) seq.nk = A.k_total - seq.k0;  // keys of no sequence: no queries
  const int kb = (index - first) * kKeys;
  if (kb >= seq.nk) return;

  const int lane = lane_id(), c = lane & 31, h = lane >> 5;
  const int group_of = kGroups == 1 ? 0 : wave_id() / kWaves, wave = wave_id() % kWaves;
  char *tiles_at = lds + group_of * Plan::kGroupLds;
  constexpr int kBuffers = Plan::kBuffers;
  const float *stats = reinterpret_cast<const float *>(tiles_at + kBuffers * 2 * kTile);
  char *values = lds + kGroups * Plan::kGroupLds;
  const int key0 = kb + wave * kWaveRows, key = key0 + c;
  const bool valid = key < seq.nk;
  const int64_t k_row = seq.k0 + (valid ? key : seq.nk - 1);
  const int heads = A.group.size, rows = seq.nq * heads;
  const int ahead = seq.nk - seq.nq;
  // key j is seen by the queries from j - ahead on: packed rows from
  // (j - ahead) * heads; first for the block, for this key, for the wave's
  // last key and its first
  const int begin = A.causal ? max(0, min(kb - ahead, seq.nq)) * heads : 0;
  const int from = A.causal ? (key - ahead) * heads : 0;
  const int from_last = A.causal ? (key0 + kWaveRows - 1 - ahead) * heads : 0;
  const int from_first = A.causal ? (key0 - ahead) * heads : 0;
  const int tiles = (rows - begin + kRows - 1) / kRows;

  Frags<T, DP> k, v;
  row_frags<T, DP>(k, A.k.at + k_row * A.k.row + head * A.k.head, A.chunks, true);
  if constexpr (Plan::kValuesInLds) {
    Stage<T, DP, kKeys, Plan::kThreads> v_stage;
    v_stage.set(A.chunks, [&](int r) { return r * int(A.v.row); });
    load_rows(v_stage, A.v.at + seq.k0 * A.v.row + head * A.v.head, A.v.row, kb, seq.nk,
              lds_address(values));
    clear_rest<T, DP>(values, kKeys, threadIdx.x, Plan::kThreads, A.chunks);
  } else {
    row_frags<T, DP>(v, A.v.at + k_row * A.v.row + head * A.v.head, A.chunks, true);
  }
  const char *q_at = A.q.at + seq.q0 * A.q.row + int64_t(head) * heads * A.q.head;
  const char *g_at = A.dout.at + seq.q0 * A.dout.row + int64_t(head) * heads * A.dout.head;
  const int64_t stat0 = int64_t(seq.q0) * A.q_heads + head * heads;
  const unsigned tiles0 = lds_address(lds) + group_of * Plan::kGroupLds;
  // Where kRows is a multiple of the group's heads, a tile's rows lie alike
  // in every tile (the first one starts with a query), but for the last's.
  const bool alike = kRows % heads == 0;
  Stage<T, DP, kRows, 256> q_stage, g_stage;
  auto place = [&](int row, const Operand &o) {
    const int i = A.group.div(row);
    return i * int(o.row) + (row - i * heads) * int(o.head);
  };
  q_stage.set(A.chunks, [&](int r) { return alike ? place(r, A.q) : 0; });
  g_stage.set(A.chunks, [&](int r) { return alike ? place(r, A.dout) : 0; });
  auto load_tile = [&](int t, int buffer) {
    const unsigned to = tiles0 + buffer * 2 * kTile;
    const int r0 = begin + (tiles - 1 - t) * kRows, i0 = A.group.div(r0);
    // rows from r0 on, as rows from the query that r0 belongs to on
    const int skip = r0 - i0 * heads, last = rows - 1 - i0 * heads;
    const char *q_base = q_at + i0 * A.q.row, *g_base = g_at + i0 * A.dout.row;
    if (alike && r0 + kRows <= rows) {
      q_stage.load(q_base, to);
      g_stage.load(g_base, to + kTile);
    } else {
      q_stage.load(q_base, to, [&](int r) { return place(min(skip + r, last), A.q); });
      g_stage.load(g_base, to + kTile, [&](int r) { return place(min(skip + r, last), A.dout); });
    }
    // L and D of 32 rows, a lane each (by every wave: all count the same loads)
    const int row = min(skip + (lane >> 1), last), i = A.group.div(row);
    load_to_lds4(reinterpret_cast<const char *>(A.stats + stat0 + int64_t(i0) * A.q_heads),
                 unsigned((i * A.q_heads + row - i * heads) * 2 + (lane & 1)) * 4,
                 tiles0 + kBuffers * 2 * kTile + buffer * kRows * 8);
  };
  constexpr int kTileLoads = 2 * Stage<T, DP, kRows, 256>::kLoads + 1;
  clear_rest<T, DP>(tiles_at, kBuffers * 2 * kRows, threadIdx.x % 256, 256, A.chunks);

  Sums<T, DP> dk = {}, dv = {};
  if (group_of < tiles) load_tile(group_of, 0);
  if (group_of + kGroups < tiles) load_tile(group_of + kGroups, 1);
  int buffer = 0;
  // (both groups go round as often: they share the barrier)
  for (int t0 = 0; t0 < tiles; t0 += kGroups, buffer = buffer == kBuffers - 1 ? 0 : buffer + 1) {
    const int t = t0 + group_of;
    if (t + kGroups < tiles)
      wait_loads<kTileLoads>();  // all but the next tile's
    else
      wait_loads<0>();
    tile_barrier();  // tile t is there, and the last one has been read
    if (t + 2 * kGroups < tiles)
      load_tile(t + 2 * kGroups, buffer == 0 ? kBuffers - 1 : buffer - 1);
    const char *q_tile = tiles_at + buffer * 2 * kTile, *g_tile = q_tile + kTile;
    const float *stat_row = stats + buffer * 2 * kRows;
    const int r0 = begin + (tiles - 1 - t) * kRows;
    if (t >= tiles || key0 >= seq.nk || r0 + kRows <= from_first) continue;
    const bool masked = r0 < from_last || r0 + kRows > rows;
    // (hides that the addresses of the reads are the same in every round: to
    // keep them all takes more registers than there are)
    int at_lane = lane;
    if constexpr (DP * sizeof(T) > 192) asm volatile("" : "+v"(at_lane));
    // Four fragments are read while four are in use.
    f32x16 dots = {}, dp = {};
    Piece<T> x[2];
    read_piece<T, DP, 4>(x[0], q_tile, 0, 0, at_lane);
    constexpr int kDotPieces = (kSteps + 3) / 4;
#pragma unroll
    for (int n = 0; n < kDotPieces; ++n) {
      if (n + 1 < kDotPieces) {
        read_piece<T, DP, 4>(x[(n + 1) & 1], q_tile, 0, 4 * n + 4, at_lane);
      } else if constexpr (Plan::kValuesInLds) {
        read_piece<T, DP, 2>(x[(n + 1) & 1], g_tile, 0, 0, at_lane);
        read_piece<T, DP, 2, 2>(x[(n + 1) & 1], values, wave * kWaveRows, 0, at_lane);
      } else {
        read_piece<T, DP, 4>(x[(n + 1) & 1], g_tile, 0, 0, at_lane);
      }
      pin_reads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * n + i < kSteps) dots = Mat<T>::mma(x[n & 1][i], k[4 * n + i], dots);
      pin_reads();
    }
    constexpr int kPer = Plan::kValuesInLds ? 2 : 4;
    constexpr int kGradPieces = (kSteps + kPer - 1) / kPer;
#pragma unroll
    for (int n = 0; n < kGradPieces; ++n) {
      Piece<T> &now = x[(kDotPieces + n) & 1], &next = x[(kDotPieces + n + 1) & 1];
      if (n + 1 < kGradPieces) {
        if constexpr (Plan::kValuesInLds) {
          read_piece<T, DP, 2>(next, g_tile, 0, 2 * n + 2, at_lane);
          read_piece<T, DP, 2, 2>(next, values, wave * kWaveRows, 2 * n + 2, at_lane);
        } else {
          read_piece<T, DP, 4>(next, g_tile, 0, 4 * n + 4, at_lane);
        }
      }
      pin_reads();
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (kPer * n + i < kSteps) {
          if constexpr (Plan::kValuesInLds)
            dp = Mat<T>::mma(now[i], now[2 + i], dp);
          else
            dp = Mat<T>::mma(now[i], v[kPer * n + i], dp);
        }
      pin_reads();
    }
    float p[16], ds[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // L and D of four rows
      const f32x4 s01 = *reinterpret_cast<const f32x4 *>(stat_row + 16 * i + 8 * h);
      const f32x4 s23 = *reinterpret_cast<const f32x4 *>(stat_row + 16 * i + 8 * h + 4);
      const float l[4] = {s01[0], s01[2], s23[0], s23[2]};
      const float d[4] = {s01[1], s01[3], s23[1], s23[3]};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * i + j;
        p[r] = exp2_fast(fmaf(dots[r], A.scale_log2, -l[j]));
        ds[r] = p[r] * (dp[r] - d[j]);
        if (masked) {
          const int at = r0 + c_row(r, h);
          if (at < from || at >= rows) p[r] = ds[r] = 0.f;
        }
      }
    }
    Weights<T> w, u;
    w.set(p);
    u.set(ds);
    if constexpr (sizeof(T) == 4) {
      Columns<T, DP> g, q;
      g.read(g_tile, 0);
      q.read(q_tile, 0);
      g.add(dv, w, at_lane);
      q.add(dk, u, at_lane);
    } else {
      constexpr int kAt = kDotPieces + kGradPieces, kPieces = (kBlocks + 1) / 2;
      pin_reads();
      read_column_piece<T, DP>(x[kAt & 1], g_tile, 0, 0, at_lane);
#pragma unroll
      for (int n = 0; n < 2 * kPieces; ++n) {
        Piece<T> &now = x[(kAt + n) & 1], &next = x[(kAt + n + 1) & 1];
        if (n + 1 < 2 * kPieces)
          read_column_piece<T, DP>(next, n + 1 < kPieces ? g_tile : q_tile, 0,
                                   2 * ((n + 1) % kPieces), at_lane);
        pin_reads();
        if (n < kPieces)
          add_column_piece<T, DP>(dv, now, w, 2 * n);
        else
          add_column_piece<T, DP>(dk, now, u, 2 * (n - kPieces));
        pin_reads();
      }
    }
  }

  if constexpr (kGroups > 1) {
    // the second group hands its sums over, dk and then dv
    float *sums = reinterpret_cast<float *>(lds) + wave * (kBlocks * 16 * 64) + lane;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      Sums<T, DP> &mine = n == 0 ? dk : dv;
      __syncthreads();
      if (group_of == 1) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) sums[(b * 16 + r) * 64] = mine[b][r];
      }
      __syncthreads();
      if (group_of == 0) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) mine[b][r] += sums[(b * 16 + r) * 64];
      }
    }
    if (group_of == 1) return;
  }
  store_row<T, DP>(A.dk.at + k_row * A.dk.row + head * A.dk.head, dk, A.scale, A.dim, valid);
  store_row<T, DP>(A.dv.at + k_row * A.dv.row + head * A.dv.head, dv, 1.f, A.dim, valid);
}

template <typename T, int DP>
int launch_backward(BackwardArgs &A, float2 *stats, hipStream_t s) {
  constexpr int kLanes = sizeof(T) == 4 ? 32 : 16;
  constexpr int kKeys = sizeof(T) == 4 ? 32 : 64;
  constexpr int kLds = 4 * Shape<T, DP>::tile_bytes(kKeys);
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  int st = BEVPOOL_OK;
  if (A.q_total > 0) {
    const int64_t rows = int64_t(A.q_total) * A.q_heads, per = kThreads / kLanes;
    st = check_grid((rows + per - 1) / per, kThreads, "attention row sums");
    if (st) return st;
    {
      LaunchScope scope("attention_stats", s);
      hipLaunchKernelGGL((stats_kernel<T, kLanes>), dim3(unsigned((rows + per - 1) / per)),
                         dim3(kThreads), 0, s, static_cast<const PackedArgs &>(A), stats);
    }
    st = check_launch("attention row sums");
    if (st) return st;
    A.tiles = int(int64_t(A.q_total) * A.group.size / (kWaves * kWaveRows)) + A.sequences + 1;
    const int64_t blocks = int64_t(A.tiles) * A.k_heads;
    st = check_grid(blocks, kThreads, "attention query gradient");
    if (st) return st;
    {
      LaunchScope scope("attention_query_grad", s);
      hipLaunchKernelGGL((query_grad_kernel<T, DP, kKeys>), dim3(unsigned(blocks)),
                         dim3(kThreads), kLds, s, A);
    }
    st = check_launch("attention query gradient");
    if (st) return st;
  }
  if (A.k_total > 0) {
    A.tiles = A.k_total / (kWaves * kWaveRows) + A.sequences + 1;
    using Plan = KeyPlan<T, DP>;
    const int64_t blocks = int64_t(A.tiles) * A.k_heads;
    st = check_grid(blocks, Plan::kThreads, "attention key gradient");
    if (st) return st;
    LaunchScope scope("attention_key_grad", s);
    hipLaunchKernelGGL((key_grad_kernel<T, DP>), dim3(unsigned(blocks)), dim3(Plan::kThreads),
                       Plan::kLds, s, A);
    st = check_launch("attention key gradient");
  }
  return st;
}

}  // namespace

extern "C" {

size_t bevpool_attention_backward_scratch_bytes(int64_t q_total, int32_t q_heads) {
  if (q_total < 1 || q_heads < 1) return 0;
  return size_t(q_total) * size_t(q_heads) * 2 * sizeof(float);
}

int bevpool_attention_backward(const void *q, int64_t q_row, int64_t q_head, const void *k,
                               int64_t k_row, int64_t k_head, const void *v, int64_t v_row,
                               int64_t v_head, const void *out, const void *dout,
                               int64_t dout_row, int64_t dout_head, const float *lse,
                               int32_t dtype, int64_t q_total, int64_t k_total, int32_t q_heads,
                               int32_t k_heads, int32_t dim, const int32_t *q_starts,
                               const int32_t *k_starts, int32_t sequences, int32_t causal,
                               float scale, void *dq, void *dk, void *dv, void *scratch,
                               size_t scratch_bytes, void *stream) {
  bevpool_host::clear_error();
  BackwardArgs A = {};
  const int elem = dtype == BEVPOOL_F32 ? 4 : 2;
  const int64_t q_dense = int64_t(q_heads) * dim, k_dense = int64_t(k_heads) * dim;
  int st = check_packed(A, dtype, q_total, k_total, sequences, q_heads, k_heads, dim, q_starts,
                        k_starts, causal, scale);
  if (!st) st = set_operand(A.q, "q", q, q_row, q_head, elem, q_total);
  if (!st) st = set_operand(A.k, "k", k, k_row, k_head, elem, k_total);
  if (!st) st = set_operand(A.v, "v", v, v_row, v_head, elem, k_total);
  if (!st) st = set_operand(A.out, "out", out, q_dense, dim, elem, q_total);
  if (!st) st = set_operand(A.dout, "dout", dout, dout_row, dout_head, elem, q_total);
  if (!st) st = set_operand(A.dq, "dq", dq, q_dense, dim, elem, q_total);
  if (!st) st = set_operand(A.dk, "dk", dk, k_dense, dim, elem, k_total);
  if (!st) st = set_operand(A.dv, "dv", dv, k_dense, dim, elem, k_total);
  if (st) return st;
  if (q_total > 0 && !lse) return fail(BEVPOOL_EINVAL, "lse: null");
  // (as are those of a tile's rows, heads of a group among them)
  const int64_t heads = A.group.size < 64 ? A.group.size : 64;
  if (A.q.head * heads >= (1 << 30) || A.dout.head * heads >= (1 << 30))
    return fail(BEVPOOL_EINVAL, "q, dout: the heads of a group must lie within 2^30 bytes");
  const size_t need = bevpool_attention_backward_scratch_bytes(q_total, q_heads);
  if (scratch_bytes < need || (need > 0 && !scratch))
    return fail(BEVPOOL_ESPACE, "attention backward scratch: %zu bytes, %zu needed",
                scratch_bytes, need);
  A.lse = const_cast<float *>(lse);
  float2 *stats = static_cast<float2 *>(scratch);
  A.stats = stats;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == BEVPOOL_BF16  ? (ATTENTION_DIM(__bf16, launch_backward, A, stats, s))
         : dtype == BEVPOOL_F16 ? (ATTENTION_DIM(_Float16, launch_backward, A, stats, s))
                                : (ATTENTION_DIM(float, launch_backward, A, stats, s));
}

}  // extern "C"

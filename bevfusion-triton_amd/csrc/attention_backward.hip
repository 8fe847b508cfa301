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
//
// dS grows with dout, and fp16 holds only 2^-14 to 2^16 in full: small
// gradients would be lost in its last bits, large ones past its range.  So in
// fp16 dS is formed times a power of two that brings dout's largest magnitude
// to between 4 and 8 (where a dout of order 1 has it already), and the sums,
// in fp32, are brought back: in dq's kernel by row, in the keys' kernels by the
// rows that a block walks.
#include "attention_tiles.h"
#include "host_calls.h"

namespace {

using namespace attention;
using bevpool_host::check_grid;
using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

struct BackwardArgs : PackedArgs {
  // (tokens, heads): -L / scale, where the sums of q k begin, and -D.  In fp32
  // -L in units of log 2: sums begun so far from zero lose a bit there.
  float2 *stats;
  // fp16: the largest magnitude of dout in 32 rows, [key head][row tile * tile
  // rows / 32 + 32 rows], tops_stride for a head
  float *tops;
  int tops_stride;
  int row_tile;  // rows of a tile of the query kernel
};

// log2 of what dS is formed times, where dout's largest finite magnitude is
// `top` (0: anything will do).
__device__ __forceinline__ int raise_of(float top) {
  return 3 - __builtin_amdgcn_frexp_expf(top);  // top = m 2^e, m in [0.5, 1)
}

// A lane's part of the dot product of two rows.
template <typename T, int DP>
__device__ __forceinline__ float row_dot(const Frags<T, DP> &a, const Frags<T, DP> &b) {
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < Shape<T, DP>::kSteps; ++s)
#pragma unroll
    for (int i = 0; i < int(16 / sizeof(T)); ++i) sum = fmaf(float(a[s][i]), float(b[s][i]), sum);
  return sum;
}

// dq: rows and tiles as in the forward.  Also writes -L / scale and -D of its
// rows (in fp32 -L), for the keys' kernels.  D is a small difference of what dS subtracts
// it from where a row sees few keys, so it is formed from the output before
// its rounding (out and its rest): with out alone the error of dq and dk grew
// by a fifth.
//
// Three products of 2 dim operations a pair.  The matrix instructions are busy
// in half of the cycles: two waves a SIMD, and of each block of 32 keys the
// exponentials stand between the second product and the third.  By events, in
// bf16: 11 causal prompts of up to 4,096 over heads of 128 331 us, 940 TFLOP/s;
// six cameras of 2,816 tokens, heads of 80, 406 us, 900 TFLOP/s (of 80 of the
// 96 columns that it computes).  fp32, 9 windows of 900, heads of 32: 81 us.
template <typename T, int DP, int kKeys, bool kHalves>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && DP > 64 ? 1 : 2) void query_grad_kernel(
    BackwardArgs A) {
  using S = Shape<T, DP>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kTile = S::tile_bytes(kKeys);  // buffers: K0 V0 K1 V1
  constexpr int kRows = (kHalves ? 2 : 4) * kWaveRows;
  constexpr int kMine = kHalves ? 1 : kKeys / 32;  // blocks of 32 keys a wave takes of a tile
  // dP's sums begin at -D (16 registers of it) but for the longest heads, which
  // have none left: whole backward in 16 bits 474 us begun at zero and 461 at
  // -D for heads of 32, 1,064 and 1,053 for 96, but 945 and 957 for 128.
  constexpr bool kBegin = DP * sizeof(T) <= 192;
  const int head = blockIdx.x % A.k_heads;
  const int index = A.tiles - 1 - int(blockIdx.x / A.k_heads);
  const sequences::RowTile at_rows =
      sequences::row_tile(starts_of(A), A.group.size, kRows, index, Wave{});
  if (!at_rows.on) return;
  const Sequence seq = at_rows.seq;
  const int rows = at_rows.rows, r0 = at_rows.r0;

  const int lane = lane_id(), c = lane & 31, h = lane >> 5;
  const int wave = wave_id() / (kHalves ? 2 : 1), half = kHalves ? wave_id() % 2 : 0;
  const int mine = 32 * half;
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
  const int64_t stat_at = token * A.q_heads + q_head;
  float stat[2] = {A.lse[stat_at] * kLog2e, 0.f};
  {
    const int64_t at = token * A.out.row + q_head * A.out.head;
    Frags<T, DP> o;
    row_frags<T, DP>(o, A.out.at + at, A.chunks, true);
    stat[1] = row_dot<T, DP>(o, g);
    if (sizeof(T) == 2 && A.rest) {
      row_frags<T, DP>(o, A.rest + at, A.chunks, true);
      stat[1] += row_dot<T, DP>(o, g);
    }
    stat[1] = sum_halves(stat[1]);
  }
  settle(stat);
  const float lse2 = stat[0], delta = stat[1];
  constexpr bool kRaise = __is_same(T, _Float16);
  float from = -lse2;  // of the exponents
  int raise = 0;
  if constexpr (kRaise) {
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float size = fabsf(float(g[s][i]));
        top = fmaxf(top, size < kInf ? size : 0.f);  // (no number: fmaxf's other)
      }
    top = max_halves(top);
    raise = raise_of(top);
    from += float(raise);
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    if (wave_on && half == 0 && lane == 0)
      A.tops[int64_t(head) * A.tops_stride + index * (kRows / 32) + wave] = top;
  }
  if (valid && h == 0 && half == 0) A.stats[stat_at] = make_float2(sizeof(T) == 4 ? -lse2 : -lse2 / A.scale_log2, -delta);
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
    if (!wave_on || k0 + mine >= high) continue;
    const bool masked = k0 + mine + 32 * kMine > low;
    // (hides that the addresses of the reads are the same in every round: kept,
    // they take more registers than there are)
    int at_lane = lane;
    if constexpr (DP * sizeof(T) > 192) asm volatile("" : "+v"(at_lane));
#pragma unroll
    for (int b = 0; b < kMine; ++b) {
      // Four fragments are read while four are in use.
      constexpr int kSteps = S::kSteps, kPieces = (kSteps + 3) / 4;
      constexpr int kColumns = (S::kBlocks + 1) / 2;  // pieces of 64
      f32x16 dots = {}, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = kBegin ? -delta : 0.f;
      Piece<T> x[2];
      read_piece<T, DP, 4>(x[0], k_tile, mine + 32 * b, 0, at_lane);
#pragma unroll
      for (int n = 0; n < 2 * kPieces; ++n) {
        Piece<T> &now = x[n & 1], &next = x[(n + 1) & 1];
        const int s0 = n % kPieces * 4, s1 = (n + 1) % kPieces * 4;
        if (n + 1 < 2 * kPieces)
          read_piece<T, DP, 4>(next, n + 1 < kPieces ? k_tile : v_tile, mine + 32 * b, s1, at_lane);
        else if constexpr (sizeof(T) == 2)
          read_column_piece<T, DP>(next, k_tile, mine + 32 * b, 0, at_lane);
        pin_reads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (s0 + i < kSteps) {
            if (n < kPieces)
              dots = Mat<T>::mma(now[i], q[s0 + i], dots);
            else
              dp = Mat<T>::mma(now[i], g[s0 + i], dp);
          }
        pin_reads();
      }
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        p[r] = exp2_fast(fmaf(dots[r], A.scale_log2, from)) * (kBegin ? dp[r] : dp[r] - delta);
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + mine + 32 * b + c_row(r, h) >= limit) p[r] = 0.f;
      }
      Weights<T> w;
      w.set(p);
      if constexpr (sizeof(T) == 4) {
        Columns<T, DP> kt;
        kt.read(k_tile, mine + 32 * b);
        kt.add(dq, w, at_lane);
      } else {
#pragma unroll
        for (int n = 0; n < kColumns; ++n) {
          Piece<T> &now = x[n & 1], &next = x[(n + 1) & 1];
          if (n + 1 < kColumns) read_column_piece<T, DP>(next, k_tile, mine + 32 * b, 2 * n + 2, at_lane);
          pin_reads();
          add_column_piece<T, DP>(dq, now, w, 2 * n);
          pin_reads();
        }
      }
    }
  }
  if constexpr (kHalves) {
    float *sums = reinterpret_cast<float *>(lds) + wave * (64 * 16 * S::kBlocks);
    __syncthreads();  // the tiles have been read
    if (half == 1) put_sums<T, DP>(sums, dq);
    __syncthreads();
    if (half == 1) return;
    add_sums<T, DP>(dq, sums);
  }
  const float by = kRaise ? __builtin_amdgcn_ldexpf(A.scale, -raise) : A.scale;
  store_row<T, DP>(A.dq.at + token * A.dq.row + q_head * A.dq.head, dq, by, A.dim, valid);
}

// How the keys' kernel keeps a wave's 32 keys: their K and V fragments and
// both sums take 6 DP / 4 registers a lane in the 16-bit types (twice that in
// float).  For heads of up to 192 bytes that leaves room for two blocks a CU,
// which hide each other's waits; for longer heads dk and dv are two launches
// of half the sums each: five products in place of four, at two blocks in
// place of one.  In bf16, together and apart, before the exponentials ran
// beside products: heads of 128, 1,150 us and 431 + 341; heads of 80, 700 us
// and 568 + 458.
template <typename T, int DP, bool kHalves>
struct KeyPlan {
  static constexpr int kKeys = (kHalves ? 2 : 4) * kWaveRows;
  static constexpr bool kApart = DP * sizeof(T) > 192;
  static constexpr int kBlocksPerCu = DP * sizeof(T) > 320 ? 1 : 2;
  // Buffers of Q and dout rows, and behind them the first statistic of 32 rows
  // and their second.
  static constexpr int kRows = sizeof(T) == 4 && !kHalves ? 32 : 64;  // of a tile
  static constexpr int kTile = Shape<T, DP>::tile_bytes(kRows);
  static constexpr int kBuffers = kRows == 32 ? 3 : 2;
  static constexpr int kTiles = kBuffers * (2 * kTile + 8 * kRows);
  static constexpr int kHanded = kHalves ? 2 * 64 * 16 * Shape<T, DP>::kBlocks * 4 : 0;
  static constexpr int kLds = kTiles > kHanded ? kTiles : kHanded;
  static_assert(kLds <= 160 * 1024 / kBlocksPerCu, "LDS of a CU");
  static constexpr int kSums = 16 * Shape<T, DP>::kBlocks;  // registers of dk, and of dv
};

// Walks over the rows are cut where there are few of them: `splits` blocks a
// key tile at most, each with about `steps` tiles of rows or more.  Backward in
// bf16, uncut and cut: 11 causal prompts of up to 4,096, 16 heads over 4 of
// 128 (forward too) 1,657 and 1,409 us; one of 8,192, 8 heads over 1 of 128,
// 2,813 and 843 us; one of 4,096 without a mask, 8 over 2 of 64, 359 and 165.
struct Splits {
  int most, steps;
  float *sums;  // [key tile, head][split][dk, dv][32 keys][register][lane]
  __device__ __forceinline__ int of(int tiles) const {
    return max(1, min(most, (tiles + steps - 1) / steps));
  }
};

// dk and dv: a wave owns 32 keys and walks the sequence's rows (query, head
// of the group) in tiles of 32, from the last to the first that sees one of
// its keys: blocks of one sequence start together there, and find each
// other's rows in L2.
//
// Two waves a SIMD, each a chain from product to exponential to product, with Q
// and dout read from LDS twice (as rows for one product, as columns for the
// next) and a barrier a tile.  The exponentials run beside the products of dP:
// with the sums of q k begun at -L / scale they wait for no read, and the mask
// is apart from them, with one branch for all (profiled, 719 us became 605).  By
// events, in bf16: six cameras of 2,816 tokens, heads of 80, dk and dv together
// 537 us, 910 TFLOP/s; 11 causal prompts of up to 4,096, 16 heads over 4 of
// 128, dk 369 us, 850 TFLOP/s, dv 281 us, 740 TFLOP/s, sums of the cuts 29 us.
// fp32, 9 windows of 900, heads of 32: 115 us.
template <typename T, int DP, bool kHalves, bool kDk, bool kDv>
__global__ __launch_bounds__(kThreads, (KeyPlan<T, DP, kHalves>::kBlocksPerCu)) void
key_grad_kernel(BackwardArgs A, Splits splits) {
  using Plan = KeyPlan<T, DP, kHalves>;
  constexpr int kMine = kHalves ? 1 : Plan::kRows / 32;  // blocks of 32 rows a wave takes
  constexpr int kRows = Plan::kRows, kTile = Plan::kTile, kBuffers = Plan::kBuffers;
  constexpr int kSteps = Shape<T, DP>::kSteps, kBlocks = Shape<T, DP>::kBlocks;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int head = blockIdx.x % A.k_heads;
  // the cuts of the long walks first
  const int index = int(blockIdx.x / A.k_heads) % A.tiles;
  const int split = splits.most - 1 - int(blockIdx.x / A.k_heads) / A.tiles;
  const sequences::KeyTile tile = sequences::key_tile(starts_of(A), A.group.size, A.causal,
                                                      Plan::kKeys, kRows, index, Wave{});
  if (!tile.on) return;
  const int n_splits = splits.of(tile.tiles);
  if (split >= n_splits) return;
  const Sequence seq = tile.seq;
  const int kb = tile.kb, begin = tile.begin, rows = tile.rows;
  // this block's tiles of rows, counted from the last
  const int per_split = (tile.tiles + n_splits - 1) / n_splits;
  const int t_begin = split * per_split, t_end = min(tile.tiles, t_begin + per_split);

  const int lane = lane_id(), c = lane & 31, h = lane >> 5;
  const int wave = wave_id() / (kHalves ? 2 : 1), half = kHalves ? wave_id() % 2 : 0;
  const int mine = 32 * half;
  const float *stats = reinterpret_cast<const float *>(lds + kBuffers * 2 * kTile);
  const int key0 = kb + wave * kWaveRows, key = key0 + c;
  const bool valid = key < seq.nk;
  const int64_t k_row = seq.k0 + (valid ? key : seq.nk - 1);
  const int heads = A.group.size;
  const int ahead = seq.nk - seq.nq;
  // the first packed row that sees this key, the wave's last key, its first
  const int from = A.causal ? (key - ahead) * heads : 0;
  const int from_last = A.causal ? (key0 + kWaveRows - 1 - ahead) * heads : 0;
  const int from_first = A.causal ? (key0 - ahead) * heads : 0;

  Frags<T, DP> k, v;
  row_frags<T, DP>(k, A.k.at + k_row * A.k.row + head * A.k.head, A.chunks, true);
  if constexpr (kDk)
    row_frags<T, DP>(v, A.v.at + k_row * A.v.row + head * A.v.head, A.chunks, true);
  // fp16: dS times 2^raise.  As much of it as P may have for dv as well (2^15 P
  // fits, and less than P would lose its last bits) is in the exponents; what
  // is left, of a dout far from 1, is apart with the mask (a product for all
  // cost 7% of heads of 32).
  constexpr bool kRaise = __is_same(T, _Float16) && kDk;
  int raise = 0, raise_p = 0;
  if constexpr (kRaise) {
    const int first = sequences::first_tile(A.q_starts, tile.which, A.q_total, heads, A.row_tile);
    const float *tops = A.tops + int64_t(head) * A.tops_stride + first * (A.row_tile / 32);
    const int low = begin + (tile.tiles - t_end) * kRows;
    const int high = min(rows, begin + (tile.tiles - t_begin) * kRows);
    float top = 0.f;
    for (int i = low / 32 + lane; i * 32 < high; i += 64) top = fmaxf(top, tops[i]);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    raise = __builtin_amdgcn_readfirstlane(raise_of(top));
  }
  if constexpr (kRaise) raise_p = kDv ? max(0, min(raise, 15)) : raise;
  const float raise_e = float(raise_p), raise_rest = __builtin_amdgcn_ldexpf(1.f, raise - raise_p);
  const char *q_at = A.q.at + seq.q0 * A.q.row + int64_t(head) * heads * A.q.head;
  const char *g_at = A.dout.at + seq.q0 * A.dout.row + int64_t(head) * heads * A.dout.head;
  const int64_t stat0 = int64_t(seq.q0) * A.q_heads + head * heads;
  const unsigned tiles0 = lds_address(lds);
  // Where kRows is a multiple of the group's heads, a tile's rows lie alike
  // in every tile (the first one starts with a query), but for the last's.
  const bool alike = kRows % heads == 0;
  Stage<T, DP, kRows, kThreads> q_stage, g_stage;
  auto place = [&](int row, const Operand &o) {
    const int i = A.group.div(row);
    return i * int(o.row) + (row - i * heads) * int(o.head);
  };
  q_stage.set(A.chunks, [&](int r) { return alike ? place(r, A.q) : 0; });
  g_stage.set(A.chunks, [&](int r) { return alike ? place(r, A.dout) : 0; });
  auto load_tile = [&](int t, int buffer) {
    const unsigned to = tiles0 + buffer * 2 * kTile;
    const int r0 = begin + (tile.tiles - 1 - t) * kRows, i0 = A.group.div(r0);
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
    // both statistics of 32 rows, a lane each (by every wave: all count the
    // same loads)
#pragma unroll
    for (int j = 0; j < kRows / 32; ++j) {
      const int row = min(skip + 32 * j + c, last), i = A.group.div(row);
      load_to_lds4(reinterpret_cast<const char *>(A.stats + stat0 + int64_t(i0) * A.q_heads),
                   unsigned((i * A.q_heads + row - i * heads) * 2 + h) * 4,
                   tiles0 + kBuffers * 2 * kTile + (buffer * kRows + 32 * j) * 8);
    }
  };
  constexpr int kTileLoads = 2 * Stage<T, DP, kRows, kThreads>::kLoads + kRows / 32;
  clear_rest<T, DP>(lds, kBuffers * 2 * kRows, threadIdx.x, kThreads, A.chunks);

  Sums<T, DP> dk = {}, dv = {};
#pragma unroll
  for (int i = 0; i < kBuffers - 1; ++i)
    if (t_begin + i < t_end) load_tile(t_begin + i, i);
  int buffer = 0;
  for (int t = t_begin; t < t_end; ++t, buffer = buffer == kBuffers - 1 ? 0 : buffer + 1) {
    if (kBuffers == 3 && t + 1 < t_end)
      wait_loads<kTileLoads>();  // all but the next tile's
    else
      wait_loads<0>();
    tile_barrier();  // tile t is there, and the last one has been read
    if (t + kBuffers - 1 < t_end)
      load_tile(t + kBuffers - 1, buffer == 0 ? kBuffers - 1 : buffer - 1);
    const char *q_tile = lds + buffer * 2 * kTile, *g_tile = q_tile + kTile;
    const float *stat_row = stats + buffer * 2 * kRows;
    const int r0 = begin + (tile.tiles - 1 - t) * kRows;
    const int r_mine = r0 + mine, r_end = r_mine + 32 * kMine;
    if (key0 >= seq.nk || r_end <= from_first || r_mine >= rows) continue;
    const bool masked = r_mine < from_last || r_end > rows || raise != raise_p;
    // (hides that the addresses of the reads are the same in every round: kept,
    // they take more registers than there are)
    int at_lane = lane;
    if constexpr ((kDk && kDv && DP >= (kRaise ? 80 : 96)) || (sizeof(T) == 4 && DP > 64))
      asm volatile("" : "+v"(at_lane));
#pragma unroll
    for (int b = 0; b < kMine; ++b) {
      // Four fragments are read while four are in use.
      f32x16 dots, dp;
      const float *stat = stat_row + 2 * mine + 64 * b + 4 * h;  // of rows 8 i + 4 h on: 8 i more
      // q k - L / scale and dP - D: the sums begin at what is taken off
      auto begin_at = [&](f32x16 &sums, const float *from) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 s = *reinterpret_cast<const f32x4 *>(from + 8 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) sums[4 * i + j] = s[j];
        }
      };
      Piece<T> x[2];
      constexpr int kPieces = (kSteps + 3) / 4;  // of a row's fragments
      // the first columns are read before the exponentials (dk alone, of long
      // heads, has no registers for them)
      constexpr bool kEarly = sizeof(T) == 2 && kDv;
      constexpr int kProducts = (kDk ? 2 : 1) * kPieces;
      float l[16];
      if constexpr (sizeof(T) == 4) {
        dots = {};
#pragma unroll
        for (int i = 0; i < 16; ++i) l[i] = stat[i / 4 * 8 + i % 4];
      } else {
        begin_at(dots, stat);
      }
      read_piece<T, DP, 4>(x[0], q_tile, mine + 32 * b, 0, at_lane);
#pragma unroll
      for (int n = 0; n < kProducts; ++n) {
        Piece<T> &now = x[n & 1], &next = x[(n + 1) & 1];
        const int s0 = n % kPieces * 4, s1 = (n + 1) % kPieces * 4;
        if (n + 1 < kPieces)
          read_piece<T, DP, 4>(next, q_tile, mine + 32 * b, s1, at_lane);
        else if (kDk && n + 1 < 2 * kPieces)
          read_piece<T, DP, 4>(next, g_tile, mine + 32 * b, s1, at_lane);
        else if constexpr (kEarly)
          read_column_piece<T, DP>(next, g_tile, mine + 32 * b, 0, at_lane);
        if (kDk && n == kPieces - 1) begin_at(dp, stat + 32);
        pin_reads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (s0 + i < kSteps) {
            if (n < kPieces)
              dots = Mat<T>::mma(now[i], k[s0 + i], dots);
            else
              dp = Mat<T>::mma(now[i], v[s0 + i], dp);
          }
        pin_reads();
      }
      float p[16], ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = exp2_fast(sizeof(T) == 4 ? fmaf(dots[r], A.scale_log2, l[r])
                         : kRaise       ? fmaf(dots[r], A.scale_log2, raise_e)
                                        : dots[r] * A.scale_log2);
        ds[r] = kDk ? p[r] * dp[r] : 0.f;
      }
      if (masked) {  // (apart from the exponentials, which so run beside the products of dP)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int at = r_mine + 32 * b + c_row(r, h);
          if (kRaise && kDv) ds[r] *= raise_rest;
          if (at < from || at >= rows) p[r] = ds[r] = 0.f;
        }
      }
      Weights<T> w, u;
      if constexpr (kDv) w.set(p);
      if constexpr (kDk) u.set(ds);
      if constexpr (sizeof(T) == 4) {
        Columns<T, DP> g, q;
        g.read(g_tile, mine + 32 * b);
        q.read(q_tile, mine + 32 * b);
        if constexpr (kDv) g.add(dv, w, at_lane);
        if constexpr (kDk) q.add(dk, u, at_lane);
      } else {
        constexpr int kColumns = (kBlocks + 1) / 2;  // pieces of 64 columns
        constexpr int kFirst = kDv ? 0 : kColumns, kLast = kDk ? 2 * kColumns : kColumns;
        if constexpr (!kEarly) {
          pin_reads();
          read_column_piece<T, DP>(x[kProducts & 1], q_tile, mine + 32 * b, 0, at_lane);
        }
#pragma unroll
        for (int n = kFirst; n < kLast; ++n) {
          Piece<T> &now = x[(kProducts + n - kFirst) & 1], &next = x[(kProducts + n - kFirst + 1) & 1];
          if (n + 1 < kLast)
            read_column_piece<T, DP>(next, n + 1 < kColumns ? g_tile : q_tile, mine + 32 * b,
                                     2 * ((n + 1) % kColumns), at_lane);
          pin_reads();
          if (n < kColumns)
            add_column_piece<T, DP>(dv, now, w, 2 * n);
          else
            add_column_piece<T, DP>(dk, now, u, 2 * (n - kColumns));
          pin_reads();
        }
      }
    }
  }

  if constexpr (kHalves) {
    float *sums = reinterpret_cast<float *>(lds) + wave * (64 * 16 * kBlocks);
#pragma unroll
    for (int n = kDk ? 0 : 1; n < (kDv ? 2 : 1); ++n) {
      __syncthreads();  // the tiles, or dk's sums, have been read
      if (half == 1) put_sums<T, DP>(sums, n == 0 ? dk : dv);
      __syncthreads();
      if (half == 0) add_sums<T, DP>(n == 0 ? dk : dv, sums);
    }
    if (half == 1) return;
  }
  if constexpr (kRaise) {
    const float by = __builtin_amdgcn_ldexpf(1.f, -raise);
    const float by_p = __builtin_amdgcn_ldexpf(1.f, -raise_p);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dk[b][r] *= by;
        if constexpr (kDv) dv[b][r] *= by_p;
      }
  }
  if (n_splits > 1) {
    float *put = splits.sums +
                 ((int64_t(index) * A.k_heads + head) * splits.most + split) *
                     (2 * (Plan::kKeys / 32) * Plan::kSums * 64) +
                 wave * Plan::kSums * 64 + lane;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if constexpr (kDk) put[(b * 16 + r) * 64] = dk[b][r];
        if constexpr (kDv) put[(Plan::kKeys / 32 * Plan::kSums + b * 16 + r) * 64] = dv[b][r];
      }
    return;
  }
  if constexpr (kDk)
    store_row<T, DP>(A.dk.at + k_row * A.dk.row + head * A.dk.head, dk, A.scale, A.dim, valid);
  if constexpr (kDv)
    store_row<T, DP>(A.dv.at + k_row * A.dv.row + head * A.dv.head, dv, 1.f, A.dim, valid);
}

// Adds the sums of a key tile whose walk was cut, in the order of the cuts: a
// wave for 32 keys' dk, and one for their dv.
template <typename T, int DP, bool kHalves>
__global__ __launch_bounds__(64) void key_sum_kernel(BackwardArgs A, Splits splits) {
  using Plan = KeyPlan<T, DP, kHalves>;
  constexpr int kParts = Plan::kKeys / 32;
  const int n = blockIdx.x & 1, wave = (blockIdx.x >> 1) % kParts;
  const int head = blockIdx.x / (2 * kParts) % A.k_heads;
  const int index = blockIdx.x / (2 * kParts) / A.k_heads;
  const sequences::KeyTile tile = sequences::key_tile(starts_of(A), A.group.size, A.causal,
                                                      Plan::kKeys, Plan::kRows, index, Wave{});
  if (!tile.on) return;
  const int n_splits = splits.of(tile.tiles);
  if (n_splits == 1) return;
  const int lane = lane_id();
  const int key = tile.kb + wave * kWaveRows + (lane & 31);
  const bool valid = key < tile.seq.nk;
  const int64_t k_row = tile.seq.k0 + (valid ? key : tile.seq.nk - 1);
  Sums<T, DP> sum = {};
  const float *from =
      splits.sums +
      (int64_t(index) * A.k_heads + head) * splits.most * (2 * kParts * Plan::kSums * 64) +
      (n * kParts + wave) * Plan::kSums * 64 + lane;
  for (int i = 0; i < n_splits; ++i, from += 2 * kParts * Plan::kSums * 64)
#pragma unroll
    for (int b = 0; b < Shape<T, DP>::kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[b][r] += from[(b * 16 + r) * 64];
  const Operand &to = n == 0 ? A.dk : A.dv;
  store_row<T, DP>(to.at + k_row * to.row + head * to.head, sum, n == 0 ? A.scale : 1.f, A.dim,
                   valid);
}

// Cuts of the keys' kernel, from what the host knows.  Blocks of one wave
// each of about 512 (two a CU) last as long as their longest walk, so there
// are to be about 2048; a cut below 1024 rows would not pay for its sums.  The
// steps are a block's share if the sequences are alike.
Splits plan_splits(int64_t q_total, int64_t k_total, int group, int k_heads, int sequences,
                   int causal, int tile_keys, int tile_rows) {
  Splits s = {1, 1 << 30, nullptr};
  const int64_t tiles = k_total / tile_keys + sequences + 1;
  const int64_t walk = q_total * group / tile_rows + 1;  // of one sequence of all
  const int64_t most = (2048 + tiles * k_heads - 1) / (tiles * k_heads);
  // (`most` decides the scratch, and so goes by the rows alone)
  const int64_t limit = q_total * group / 1024;
  s.most = int(most < limit ? most : limit);
  if (s.most < 2) {
    s.most = 1;
    return s;
  }
  if (s.most > 16) s.most = 16;
  const int64_t share =
      walk * tiles * k_heads / (sequences > 0 ? sequences : 1) / 512 / (causal ? 2 : 1);
  s.steps = int(share < 1024 / tile_rows ? 1024 / tile_rows : share > (1 << 20) ? (1 << 20) : share);
  return s;
}

// Whether the keys' kernel takes 64 keys a block: where key tiles of 128, with
// the cuts that sequences of the mean length have, do not fill the card.
bool halve_keys(int64_t q_total, int64_t k_total, int group, int k_heads, int sequences, int dim,
                int elem) {
  if (elem == 4 && dim > 64) return false;
  const Splits s = plan_splits(q_total, k_total, group, k_heads, sequences, 1, 128, 64);
  const int64_t mean = q_total * group / 1024 / (sequences > 0 ? sequences : 1);
  const int64_t cuts = mean < 1 ? 1 : mean < s.most ? mean : s.most;
  return (k_total / 128 + sequences + 1) * k_heads * cuts < kFullBlocks;
}

Splits plan_for(int64_t q_total, int64_t k_total, int group, int k_heads, int dim, int elem,
                int sequences, int causal) {
  const bool halves = halve_keys(q_total, k_total, group, k_heads, sequences, dim, elem);
  return plan_splits(q_total, k_total, group, k_heads, sequences, causal, halves ? 64 : 128,
                     elem == 4 && !halves ? 32 : 64);
}

size_t split_bytes(const Splits &s, int64_t q_total, int64_t k_total, int group, int k_heads,
                   int dim, int elem, int sequences) {
  if (s.most == 1) return 0;
  const int keys =
      halve_keys(q_total, k_total, group, k_heads, sequences, dim, elem) ? 64 : 128;
  const int64_t tiles = k_total / keys + sequences + 1;
  const int width = dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128;
  return size_t(tiles) * k_heads * s.most * 2 * keys * width * sizeof(float);
}

template <typename T, int DP, bool kHalves>
int launch_query(BackwardArgs &A, hipStream_t s) {
  constexpr int kKeys = sizeof(T) == 4 && !kHalves ? 32 : 64;
  constexpr int kTiles = 4 * Shape<T, DP>::tile_bytes(kKeys);
  constexpr int kSums = kHalves ? 2 * 64 * 16 * Shape<T, DP>::kBlocks * 4 : 0;
  constexpr int kLds = kTiles > kSums ? kTiles : kSums;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  A.tiles = int(int64_t(A.q_total) * A.group.size / (kHalves ? 64 : 128)) + A.sequences + 1;
  const int64_t blocks = int64_t(A.tiles) * A.k_heads;
  int st = check_grid(blocks, kThreads, "attention query gradient");
  if (st) return st;
  A.row_tile = kHalves ? 64 : 128;
  LaunchScope scope("attention_query_grad", s);
  hipLaunchKernelGGL((query_grad_kernel<T, DP, kKeys, kHalves>), dim3(unsigned(blocks)),
                     dim3(kThreads), kLds, s, A);
  return check_launch("attention query gradient");
}

template <typename T, int DP, bool kHalves>
int launch_keys(BackwardArgs &A, const Splits &splits, hipStream_t s) {
  using Plan = KeyPlan<T, DP, kHalves>;
  A.tiles = A.k_total / Plan::kKeys + A.sequences + 1;
  const int64_t blocks = int64_t(A.tiles) * A.k_heads;
  int st = check_grid(blocks * splits.most, kThreads, "attention key gradient");
  if (st) return st;
  const dim3 grid(unsigned(blocks * splits.most));
  if constexpr (Plan::kApart) {
    {
      LaunchScope scope("attention_key_grad", s);
      hipLaunchKernelGGL((key_grad_kernel<T, DP, kHalves, true, false>), grid, dim3(kThreads),
                         Plan::kLds, s, A, splits);
    }
    LaunchScope scope("attention_value_grad", s);
    hipLaunchKernelGGL((key_grad_kernel<T, DP, kHalves, false, true>), grid, dim3(kThreads),
                       Plan::kLds, s, A, splits);
  } else {
    LaunchScope scope("attention_key_grad", s);
    hipLaunchKernelGGL((key_grad_kernel<T, DP, kHalves, true, true>), grid, dim3(kThreads),
                       Plan::kLds, s, A, splits);
  }
  st = check_launch("attention key gradient");
  if (st || splits.most == 1) return st;
  const int64_t sums = blocks * 2 * (Plan::kKeys / 32);
  st = check_grid(sums, 64, "attention key sums");
  if (st) return st;
  LaunchScope scope("attention_key_sum", s);
  hipLaunchKernelGGL((key_sum_kernel<T, DP, kHalves>), dim3(unsigned(sums)), dim3(64), 0, s, A,
                     splits);
  return check_launch("attention key sums");
}

template <typename T, int DP>
int launch_backward(BackwardArgs &A, const Splits &splits, hipStream_t s) {
  int st = BEVPOOL_OK;
  if (A.q_total > 0) {
    bool halves = false;
    if constexpr (kMayHalve<T, DP>) {
      halves = row_blocks(A) < kFullBlocks;
      if (halves) st = launch_query<T, DP, true>(A, s);
    }
    if (!halves) st = launch_query<T, DP, false>(A, s);
    if (st) return st;
  }
  if (A.k_total == 0) return st;
  if constexpr (kMayHalve<T, DP>)
    if (halve_keys(A.q_total, A.k_total, A.group.size, A.k_heads, A.sequences, A.dim, sizeof(T)))
      return launch_keys<T, DP, true>(A, splits, s);
  return launch_keys<T, DP, false>(A, splits, s);
}

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

size_t stats_bytes(int64_t q_total, int q_heads) {
  return aligned(size_t(q_total) * size_t(q_heads) * sizeof(float2));
}

// Places for the tops of a key head: 2 of every tile of 64 rows, or 4 of 128.
int64_t tops_of_head(int64_t q_total, int group, int sequences) {
  return q_total * group / 32 + 4 * (int64_t(sequences) + 1);
}

size_t tops_bytes(int64_t q_total, int group, int k_heads, int dtype, int sequences) {
  return dtype == BEVPOOL_F16
             ? aligned(size_t(tops_of_head(q_total, group, sequences)) * k_heads * sizeof(float))
             : 0;
}

}  // namespace

extern "C" {

size_t bevpool_attention_backward_scratch_bytes(int64_t q_total, int64_t k_total, int32_t q_heads,
                                                int32_t k_heads, int32_t dim, int32_t dtype,
                                                int32_t sequences) {
  if (q_total < 1 || q_heads < 1 || k_heads < 1 || k_total < 0 || sequences < 0) return 0;
  const int elem = dtype == BEVPOOL_F32 ? 4 : 2;
  const int group = q_heads / k_heads;
  const Splits s = plan_for(q_total, k_total, group, k_heads, dim, elem, sequences, 1);
  return stats_bytes(q_total, q_heads) + tops_bytes(q_total, group, k_heads, dtype, sequences) +
         split_bytes(s, q_total, k_total, group, k_heads, dim, elem, sequences);
}

int bevpool_attention_backward(const void *q, int64_t q_row, int64_t q_head, const void *k,
                               int64_t k_row, int64_t k_head, const void *v, int64_t v_row,
                               int64_t v_head, const void *out, const void *out_rest, const void *dout,
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
  // (a tile's rows may begin with any head of the group, and their offsets from
  // the group's first are 32-bit)
  const int64_t reach = (int64_t(1) << 30) / A.group.size;
  if (q_total > 0 && (A.q.head >= reach || A.dout.head >= reach))
    return fail(BEVPOOL_EINVAL, "q, dout: the heads of a group must lie within 2^30 bytes");
  const size_t need = bevpool_attention_backward_scratch_bytes(q_total, k_total, q_heads, k_heads,
                                                               dim, dtype, sequences);
  if (scratch_bytes < need || (need > 0 && !scratch))
    return fail(BEVPOOL_ESPACE, "attention backward scratch: %zu bytes, %zu needed",
                scratch_bytes, need);
  if (reinterpret_cast<uintptr_t>(out_rest) % 16)
    return fail(BEVPOOL_EINVAL, "out_rest must start at a multiple of 16 bytes");
  A.rest = static_cast<char *>(const_cast<void *>(out_rest));
  A.lse = const_cast<float *>(lse);
  A.stats = static_cast<float2 *>(scratch);
  Splits splits =
      plan_for(q_total, k_total, A.group.size, k_heads, dim, elem, sequences, A.causal);
  A.row_tile = 128;  // (no queries, no query kernel to set it)
  char *at = static_cast<char *>(scratch) + stats_bytes(q_total, q_heads);
  A.tops = reinterpret_cast<float *>(at);
  A.tops_stride = int(tops_of_head(q_total, A.group.size, sequences));
  at += tops_bytes(q_total, A.group.size, k_heads, dtype, sequences);
  splits.sums = reinterpret_cast<float *>(at);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == BEVPOOL_BF16  ? (ATTENTION_DIM(__bf16, launch_backward, A, splits, s))
         : dtype == BEVPOOL_F16 ? (ATTENTION_DIM(_Float16, launch_backward, A, splits, s))
                                : (ATTENTION_DIM(float, launch_backward, A, splits, s));
}

}  // extern "C"

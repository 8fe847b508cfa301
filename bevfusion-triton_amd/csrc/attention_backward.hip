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
  const float *lse2;  // (tokens, heads): L in units of log 2
};

// D and L / log 2 of every (token, head): a row's 16-byte chunks on kLanes
// lanes.
template <typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void delta_kernel(PackedArgs A, float *lse2, float *delta) {
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
  if (chunk == 0) {
    delta[row] = sum;
    lse2[row] = A.lse[row] * kLog2e;
  }
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
  const float lse2 = A.lse2[token * A.q_heads + q_head];
  const float delta = A.delta[token * A.q_heads + q_head];
  const char *k_at = A.k.at + seq.k0 * A.k.row + head * A.k.head;
  const char *v_at = A.v.at + seq.k0 * A.v.row + head * A.v.head;
  auto load_tile = [&](int t) {
    char *to = lds + (t & 1) * 2 * kTile;
    const int k0 = t * kKeys, most = seq.nk - 1;
    stage<T, DP, kKeys, kThreads>(to, threadIdx.x, A.chunks, [&](int r) {
      return k_at + int64_t(min(k0 + r, most)) * A.k.row;
    });
    stage<T, DP, kKeys, kThreads>(to + kTile, threadIdx.x, A.chunks, [&](int r) {
      return v_at + int64_t(min(k0 + r, most)) * A.v.row;
    });
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
      const f32x16 dots = dot_rows<T, DP>(k_tile, 32 * b, q);
      const f32x16 dp = dot_rows<T, DP>(v_tile, 32 * b, g);
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
      add_transposed<T, DP>(dq, k_tile, 32 * b, w);
    }
  }
  store_row<T, DP>(A.dq.at + token * A.dq.row + q_head * A.dq.head, dq, A.scale, A.dim, valid);
}

// dk and dv: a wave owns 32 keys and walks the sequence's rows (query, head
// of the group), kRows at a time, in two buffers.
template <typename T, int DP, int kRows>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) > 128 ? 1 : 2) void key_grad_kernel(
    BackwardArgs A) {
  using S = Shape<T, DP>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // buffers: Q0 G0 Q1 G1, then L0 D0 L1 D1 of kRows floats
  constexpr int kTile = S::tile_bytes(kRows);
  float *stats = reinterpret_cast<float *>(lds + 4 * kTile);
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

  const int lane = lane_id(), wave = wave_id(), c = lane & 31, h = lane >> 5;
  const int key0 = kb + wave * kWaveRows, key = key0 + c;
  const bool valid = key < seq.nk;
  const int64_t k_row = seq.k0 + (valid ? key : seq.nk - 1);
  const int group = A.group.size, rows = seq.nq * group;
  const int ahead = seq.nk - seq.nq;
  // key j is seen by the queries from j - ahead on: packed rows from
  // (j - ahead) * group; first for the block, for this key, for the wave's
  // last key and its first
  const int begin = A.causal ? max(0, min(kb - ahead, seq.nq)) * group : 0;
  const int from = A.causal ? (key - ahead) * group : 0;
  const int from_last = A.causal ? (key0 + kWaveRows - 1 - ahead) * group : 0;
  const int from_first = A.causal ? (key0 - ahead) * group : 0;
  const int tiles = (rows - begin + kRows - 1) / kRows;

  Frags<T, DP> k, v;
  row_frags<T, DP>(k, A.k.at + k_row * A.k.row + head * A.k.head, A.chunks, true);
  row_frags<T, DP>(v, A.v.at + k_row * A.v.row + head * A.v.head, A.chunks, true);
  const char *q_at = A.q.at + seq.q0 * A.q.row + int64_t(head) * group * A.q.head;
  const char *g_at = A.dout.at + seq.q0 * A.dout.row + int64_t(head) * group * A.dout.head;
  const int64_t stat0 = int64_t(seq.q0) * A.q_heads + head * group;
  auto load_tile = [&](int t) {
    char *to = lds + (t & 1) * 2 * kTile;
    const int r0 = begin + t * kRows;
    stage<T, DP, kRows, kThreads>(to, threadIdx.x, A.chunks, [&](int r) {
      const int row = min(r0 + r, rows - 1), i = A.group.div(row);
      return q_at + i * A.q.row + (row - i * group) * A.q.head;
    });
    stage<T, DP, kRows, kThreads>(to + kTile, threadIdx.x, A.chunks, [&](int r) {
      const int row = min(r0 + r, rows - 1), i = A.group.div(row);
      return g_at + i * A.dout.row + (row - i * group) * A.dout.head;
    });
    // wave 0: L of the rows, wave 1: D
    if (wave < 2 && lane < kRows) {
      const int row = min(r0 + lane, rows - 1), i = A.group.div(row);
      const float *at = (wave ? A.delta : A.lse2) + stat0 + int64_t(i) * A.q_heads + row - i * group;
      float *put = stats + ((t & 1) * 2 + wave) * kRows;
      load_to_lds4(reinterpret_cast<const char *>(at), reinterpret_cast<const char *>(put));
    }
  };
  clear_rest<T, DP>(lds, 4 * kRows, threadIdx.x, kThreads, A.chunks);

  Sums<T, DP> dk = {}, dv = {};
  if (tiles > 0) load_tile(0);
  for (int t = 0; t < tiles; ++t) {
    wait_loads<0>();
    __syncthreads();  // tile t is there, and tile t - 1 has been read
    if (t + 1 < tiles) load_tile(t + 1);
    const char *q_tile = lds + (t & 1) * 2 * kTile, *g_tile = q_tile + kTile;
    const float *l_row = stats + (t & 1) * 2 * kRows, *d_row = l_row + kRows;
    const int r0 = begin + t * kRows;
    if (key0 >= seq.nk || r0 + kRows <= from_first) continue;
    const bool masked = r0 < from_last || r0 + kRows > rows;
#pragma unroll
    for (int b = 0; b < kRows / 32; ++b) {
      const f32x16 dots = dot_rows<T, DP>(q_tile, 32 * b, k);
      const f32x16 dp = dot_rows<T, DP>(g_tile, 32 * b, v);
      float p[16], ds[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 l = *reinterpret_cast<const f32x4 *>(l_row + 32 * b + 8 * i + 4 * h);
        const f32x4 d = *reinterpret_cast<const f32x4 *>(d_row + 32 * b + 8 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * i + j;
          p[r] = exp2_fast(fmaf(dots[r], A.scale_log2, -l[j]));
          ds[r] = p[r] * (dp[r] - d[j]);
          if (masked) {
            const int at = r0 + 32 * b + c_row(r, h);
            if (at < from || at >= rows) p[r] = ds[r] = 0.f;
          }
        }
      }
      Weights<T> w;
      w.set(p);
      add_transposed<T, DP>(dv, g_tile, 32 * b, w);
      w.set(ds);
      add_transposed<T, DP>(dk, q_tile, 32 * b, w);
    }
  }
  store_row<T, DP>(A.dk.at + k_row * A.dk.row + head * A.dk.head, dk, A.scale, A.dim, valid);
  store_row<T, DP>(A.dv.at + k_row * A.dv.row + head * A.dv.head, dv, 1.f, A.dim, valid);
}

template <typename T, int DP>
int launch_backward(BackwardArgs &A, float *lse2, float *delta, hipStream_t s) {
  constexpr int kLanes = sizeof(T) == 4 ? 32 : 16;
  constexpr int kKeys = sizeof(T) == 4 ? 32 : 64;  // rows of a tile, too
  constexpr int kLds = 4 * Shape<T, DP>::tile_bytes(kKeys);
  static_assert(kLds + 16 * kKeys <= 160 * 1024, "LDS of a CU");
  int st = BEVPOOL_OK;
  if (A.q_total > 0) {
    const int64_t rows = int64_t(A.q_total) * A.q_heads, per = kThreads / kLanes;
    st = check_grid((rows + per - 1) / per, kThreads, "attention delta");
    if (st) return st;
    {
      LaunchScope scope("attention_delta", s);
      hipLaunchKernelGGL((delta_kernel<T, kLanes>), dim3(unsigned((rows + per - 1) / per)),
                         dim3(kThreads), 0, s, static_cast<const PackedArgs &>(A), lse2, delta);
    }
    st = check_launch("attention delta");
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
    const int64_t blocks = int64_t(A.tiles) * A.k_heads;
    st = check_grid(blocks, kThreads, "attention key gradient");
    if (st) return st;
    LaunchScope scope("attention_key_grad", s);
    hipLaunchKernelGGL((key_grad_kernel<T, DP, kKeys>), dim3(unsigned(blocks)), dim3(kThreads),
                       kLds + 16 * kKeys, s, A);
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
  const size_t need = bevpool_attention_backward_scratch_bytes(q_total, q_heads);
  if (scratch_bytes < need || (need > 0 && !scratch))
    return fail(BEVPOOL_ESPACE, "attention backward scratch: %zu bytes, %zu needed",
                scratch_bytes, need);
  A.lse = const_cast<float *>(lse);
  float *lse2 = static_cast<float *>(scratch);
  float *delta = lse2 + q_total * q_heads;
  A.lse2 = lse2;
  A.delta = delta;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == BEVPOOL_BF16  ? (ATTENTION_DIM(__bf16, launch_backward, A, lse2, delta, s))
         : dtype == BEVPOOL_F16 ? (ATTENTION_DIM(_Float16, launch_backward, A, lse2, delta, s))
                                : (ATTENTION_DIM(float, launch_backward, A, lse2, delta, s));
}

}  // extern "C"

// attention.hip -- attention over packed sequences, forward (gfx950).
//
//   s_ij = scale q_i k_j over the keys j that query i sees,
//   L_i = log sum_j exp(s_ij),  o_i = sum_j exp(s_ij - L_i) v_j
// for sequences of nq queries and nk keys; causal: j <= i + nk - nq.  A
// query that sees no key has o = 0 and L = -inf.
#include "attention_tiles.h"
#include "host_calls.h"

namespace {

using namespace attention;
using bevpool_host::check_grid;
using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

// Rows of a tile are pairs (query, head of the group), the group's heads next
// to each other: the heads that share keys share their tiles, and short
// sequences still fill rows.  A wave has 32 rows and all of the tile's keys
// (kHalves: half of them); K and V tiles are staged in two buffers, the next
// one's loads in flight while one is used.
//
// 4 dim operations a visible pair against 2 dim elements a key and block, so
// the matrix instructions bound it (busy in 61% of the cycles at the rate that
// a large library product reaches, heads of 128).  128 rows a block, so that a wave's query
// and output rows stay in registers and two blocks a CU hide each other's
// softmax.  Times by events, steps one after another.  One causal sequence of 32,768 over 8 heads of 128 in bf16: 2.01 ms
// or 1,090 TFLOP/s, where a library product of 8,192^3 reaches 1,110; 11
// prompts of up to 4,096, 16 heads over 4: 237 us, 880 TFLOP/s; six cameras of
// 2,816 tokens, heads of 80 (a sixth of the product is padding to 96): 308 us,
// 790 TFLOP/s; 9 windows of 900 in fp32, heads of 32: 61 us, 61 TFLOP/s,
// one wave a SIMD and its walk.
template <typename T, int DP, int kKeys, bool kHalves>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && DP > 64 ? 1 : 2) void packed_forward_kernel(
    PackedArgs A) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int kRows = (kHalves ? 2 : 4) * kWaveRows;
  const int head = blockIdx.x % A.k_heads;
  // late tiles, the long ones of a causal sequence, start first
  const int index = A.tiles - 1 - int(blockIdx.x / A.k_heads);
  const sequences::RowTile at_rows =
      sequences::row_tile(starts_of(A), A.group.size, kRows, index, Wave{});
  if (!at_rows.on) return;
  const Sequence seq = at_rows.seq;
  const int rows = at_rows.rows, r0 = at_rows.r0;

  const int wave = wave_id() / (kHalves ? 2 : 1), c = lane_id() & 31, h = lane_id() >> 5;
  const int row = r0 + wave * kWaveRows + c;
  const bool valid = row < rows;
  const int row_in = valid ? row : rows - 1;
  const int query = A.group.div(row_in);
  const int q_head = head * A.group.size + row_in - query * A.group.size;
  const int64_t token = seq.q0 + query;
  const int ahead = seq.nk - seq.nq;  // causal: query i sees keys up to i + ahead
  // keys [0, limit) are this row's; keys of the block's last row
  const int limit = A.causal ? min(seq.nk, query + ahead + 1) : seq.nk;
  const int last_query = A.group.div(min(r0 + kRows, rows) - 1);
  const int keys = A.causal ? max(0, min(seq.nk, last_query + ahead + 1)) : seq.nk;
  // the wave's least limit (no mask below it) and its greatest (nothing above)
  const int w0 = r0 + wave * kWaveRows;
  const int low = A.causal ? min(seq.nk, A.group.div(min(w0, rows - 1)) + ahead + 1) : seq.nk;
  const int high = A.causal
                       ? min(seq.nk, A.group.div(min(w0 + kWaveRows, rows) - 1) + ahead + 1)
                       : seq.nk;
  const bool wave_on = w0 < rows;

  Frags<T, DP> q;
  row_frags<T, DP>(q, A.q.at + token * A.q.row + q_head * A.q.head, A.chunks, true);
  Sums<T, DP> out = {};
  Softmax x;
  const int half = kHalves ? wave_id() % 2 : 0;
  attend_tiles<T, DP, kKeys, kHalves>(lds, q, A.k.at + seq.k0 * A.k.row + head * A.k.head, A.k.row,
                             A.v.at + seq.k0 * A.v.row + head * A.v.head, A.v.row, A.chunks, 0,
                             keys, seq.nk, limit, low, wave_on ? high : 0, A.scale_log2, x, out, half);

  float sum = sum_halves(x.sum);
  if constexpr (kHalves) {
    constexpr int kSums = 64 * 16 * Shape<T, DP>::kBlocks;
    float *sums = reinterpret_cast<float *>(lds) + wave * (kSums + 128);
    float2 *tops = reinterpret_cast<float2 *>(sums + kSums);
    __syncthreads();  // the tiles have been read
    if (half == 1) {
      put_sums<T, DP>(sums, out);
      tops[lane_id()] = make_float2(x.top, sum);
    }
    __syncthreads();
    if (half == 1) return;
    const float2 other = tops[lane_id()];
    const float top = fmaxf(x.top, other.x);
    // (a half that saw nothing has -inf, and -inf less -inf is no number)
    const float mine = x.top == -kInf ? 1.f : exp2_fast((x.top - top) * A.scale_log2);
    const float by = other.x == -kInf ? 1.f : exp2_fast((other.x - top) * A.scale_log2);
    x.top = top;
    sum = mine * sum + by * other.y;
#pragma unroll
    for (int b = 0; b < Shape<T, DP>::kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[b][r] *= mine;
    add_sums<T, DP>(out, sums, by);
  }
  const bool any = x.top > -kInf || sum != 0.f;
  const float by = any ? 1.f / sum : 0.f;
  const int64_t at = token * A.out.row + q_head * A.out.head;
  if (sizeof(T) == 2 && A.rest)
    store_row<T, DP, true>(A.out.at + at, out, by, A.dim, valid, A.rest + at);
  else
    store_row<T, DP>(A.out.at + at, out, by, A.dim, valid);
  if (valid && h == 0 && A.lse)
    A.lse[token * A.q_heads + q_head] =
        any ? (x.top * A.scale_log2 + __builtin_amdgcn_logf(sum)) / kLog2e : -kInf;
}

template <typename T, int DP, bool kHalves>
int launch_rows(PackedArgs &A, hipStream_t s) {
  constexpr int kKeys = sizeof(T) == 4 && !kHalves ? 32 : 64;
  constexpr int kTiles = 4 * Shape<T, DP>::tile_bytes(kKeys);
  constexpr int kSums = kHalves ? 2 * (64 * 16 * Shape<T, DP>::kBlocks + 128) * 4 : 0;
  constexpr int kLds = kTiles > kSums ? kTiles : kSums;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  A.tiles = int(int64_t(A.q_total) * A.group.size / (kHalves ? 64 : 128)) + A.sequences + 1;
  const int64_t blocks = int64_t(A.tiles) * A.k_heads;
  int st = check_grid(blocks, kThreads, "attention forward");
  if (st) return st;
  LaunchScope scope("attention_forward", s);
  hipLaunchKernelGGL((packed_forward_kernel<T, DP, kKeys, kHalves>), dim3(unsigned(blocks)),
                     dim3(kThreads), kLds, s, A);
  return check_launch("attention forward");
}

template <typename T, int DP>
int launch_forward(PackedArgs &A, hipStream_t s) {
  if constexpr (kMayHalve<T, DP>)
    if (row_blocks(A) < kFullBlocks) return launch_rows<T, DP, true>(A, s);
  return launch_rows<T, DP, false>(A, s);
}

}  // namespace

namespace attention {

// Shared by forward and backward: sizes and operands of a packed call.
int check_packed(PackedArgs &A, int dtype, int64_t q_total, int64_t k_total, int sequences,
                 int q_heads, int k_heads, int dim, const void *q_starts, const void *k_starts,
                 int causal, float scale) {
  if (dtype < BEVPOOL_F32 || dtype > BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d", dtype);
  if (q_total < 0 || k_total < 0 || sequences < 0)
    return fail(BEVPOOL_EINVAL, "negative number of tokens or sequences");
  if (q_heads < 1 || k_heads < 1 || q_heads % k_heads)
    return fail(BEVPOOL_EINVAL, "%d query heads are no multiple of %d key heads", q_heads,
                k_heads);
  if (dim < 8 || dim > 128 || dim % 8)
    return fail(BEVPOOL_EINVAL, "head size %d: must be a multiple of 8 up to 128", dim);
  // (the gradients divide L by the scale)
  if (!(scale >= 1e-30f) || !(scale < 3e38f))
    return fail(BEVPOOL_EINVAL, "scale must be positive (1e-30 or more) and finite");
  const int64_t group = q_heads / k_heads;
  // (packed row numbers, and their quotients by the group, in 32 bits)
  if (q_total * group * group >= (int64_t(1) << 31) ||
      (k_total + 256) * group >= (int64_t(1) << 31))
    return fail(BEVPOOL_EINVAL, "too many tokens (%lld queries in groups of %lld, %lld keys)",
                (long long)q_total, (long long)group, (long long)k_total);
  if ((q_total > 0 || k_total > 0) && (!q_starts || !k_starts))
    return fail(BEVPOOL_EINVAL, "null starts");
  A.q_starts = static_cast<const int32_t *>(q_starts);
  A.k_starts = static_cast<const int32_t *>(k_starts);
  A.sequences = sequences;
  A.q_total = int(q_total);
  A.k_total = int(k_total);
  A.q_heads = q_heads;
  A.k_heads = k_heads;
  A.group = make_group(int(group));
  A.dim = dim;
  A.chunks = dim * (dtype == BEVPOOL_F32 ? 4 : 2) / 16;
  A.causal = causal != 0;
  A.scale = scale;
  A.scale_log2 = scale * kLog2e;
  return BEVPOOL_OK;
}

int set_operand(Operand &o, const char *what, const void *at, int64_t row, int64_t head, int elem,
                int64_t total) {
  o.at = static_cast<char *>(const_cast<void *>(at));
  o.row = row * elem;
  o.head = head * elem;
  if (total > 0 && !at) return fail(BEVPOOL_EINVAL, "%s: null", what);
  // (the offsets of 64 rows are 32-bit)
  if (total > 0 && (o.row < 0 || o.head < 0 || o.row >= (1 << 24)))
    return fail(BEVPOOL_EINVAL, "%s: strides must be positive, a row's below 2^24 bytes", what);
  if (total > 0 && (reinterpret_cast<uintptr_t>(at) % 16 || o.row % 16 || o.head % 16))
    return fail(BEVPOOL_EINVAL, "%s: rows and heads must start at multiples of 16 bytes", what);
  return BEVPOOL_OK;
}

}  // namespace attention

extern "C" {

int bevpool_attention_forward(const void *q, int64_t q_row, int64_t q_head, const void *k,
                              int64_t k_row, int64_t k_head, const void *v, int64_t v_row,
                              int64_t v_head, int32_t dtype, int64_t q_total, int64_t k_total,
                              int32_t q_heads, int32_t k_heads, int32_t dim,
                              const int32_t *q_starts, const int32_t *k_starts, int32_t sequences,
                              int32_t causal, float scale, void *out, void *out_rest, float *lse,
                              void *stream) {
  bevpool_host::clear_error();
  PackedArgs A = {};
  const int elem = dtype == BEVPOOL_F32 ? 4 : 2;
  int st = check_packed(A, dtype, q_total, k_total, sequences, q_heads, k_heads, dim, q_starts,
                        k_starts, causal, scale);
  if (!st) st = set_operand(A.q, "q", q, q_row, q_head, elem, q_total);
  if (!st) st = set_operand(A.k, "k", k, k_row, k_head, elem, k_total);
  if (!st) st = set_operand(A.v, "v", v, v_row, v_head, elem, k_total);
  if (!st) st = set_operand(A.out, "out", out, int64_t(q_heads) * dim, dim, elem, q_total);
  if (st) return st;
  if (reinterpret_cast<uintptr_t>(out_rest) % 16)
    return fail(BEVPOOL_EINVAL, "out_rest must start at a multiple of 16 bytes");
  if (q_total == 0) return BEVPOOL_OK;
  A.lse = lse;
  A.rest = static_cast<char *>(out_rest);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == BEVPOOL_BF16  ? (ATTENTION_DIM(__bf16, launch_forward, A, s))
         : dtype == BEVPOOL_F16 ? (ATTENTION_DIM(_Float16, launch_forward, A, s))
                                : (ATTENTION_DIM(float, launch_forward, A, s));
}

}  // extern "C"

// attention_cached.hip -- attention of new tokens over caches that may share
// a prefix (gfx950).
//
// Request b has `length` keys in a cache of its own, its newest `tokens` of
// them those of its new tokens, and `prefix` keys that all requests share.
// New token i sees the whole prefix and its own cache's first
// length - (tokens - 1 - i) keys.
//
// Few rows meet many keys, so the work is bound by reading the keys and is
// split along them: a part is a range of keys, with its own maximum, sum and
// unnormed output in fp32; a last kernel joins a row's parts.  The prefix is
// read once for the rows of all requests.
#include "attention_tiles.h"
#include "host_calls.h"

namespace {

using namespace attention;
using bevpool_host::check_grid;
using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

struct Cache {  // (requests, rows, heads, dim); strides in bytes
  const char *at;
  int64_t request, row, head;
};

struct CachedArgs {
  Operand q, out;  // (requests * tokens, heads, dim)
  Cache k, v;      // own caches, or the prefix as the one cache of all
  const int32_t *lengths;  // of the requests, or null: `capacity`, no mask
  int requests, tokens, capacity;
  int q_heads, k_heads;
  Group group;
  int dim, chunks;
  float scale_log2;
  int range;        // keys of a part
  int parts;        // parts of a request
  int row_tiles;
  // a row's parts: part p of row r at (part0 + p) * rows + r
  int part0;
  int64_t rows;
  float *part_out;  // [parts][rows][dim]
  float2 *part_top; // [parts][rows]: maximum (times scale_log2), sum
};

__device__ __forceinline__ int length_of(const CachedArgs &A, int request) {
  if (!A.lengths) return A.capacity;
  const int n = A.lengths[request];
  return n < 0 ? 0 : n > A.capacity ? A.capacity : n;
}

// Rows of one request and key head (token, head of the group), 32 of them a
// block, against one range of its keys.  The waves take 32 keys each in
// turn, every wave with buffers of its own and no barrier in the loop; their
// sums are joined at the end.  kFinal: the only part, written as the result.
//
// LDS for two blocks a CU: where a wave's two buffers of 32 keys fit half of
// it (rows of up to 128 bytes), the next keys' loads are in flight while 32
// are used; longer rows have one buffer, whose keys are loaded again as soon
// as the scores are formed, and its values once they are added.
template <typename T, int DP>
struct PartPlan {
  static constexpr int kTile = Shape<T, DP>::tile_bytes(32);
  static constexpr int kBuffers = kTile > 4096 ? 1 : 2;
  static constexpr int kOut = DP + 4;  // floats of a row of sums (4: other banks for the next)
  // a wave's: K0 V0 K1 V1, and its sums at the end
  static constexpr int kMine =
      kBuffers * 2 * kTile > 128 * kOut ? kBuffers * 2 * kTile : 128 * kOut;
  static constexpr int kLds = kWaves * kMine + kWaves * 32 * 8;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};
template <typename T, int DP, bool kFinal>
__device__ __forceinline__ void cached_part(const CachedArgs &A, char *lds, int at) {
  using S = Shape<T, DP>;
  constexpr int kTile = PartPlan<T, DP>::kTile, kBuffers = PartPlan<T, DP>::kBuffers;
  constexpr int kMine = PartPlan<T, DP>::kMine;
  const int part = at % A.parts;
  at /= A.parts;
  const int head = at % A.k_heads;
  at /= A.k_heads;
  const int tile = at % A.row_tiles, request = at / A.row_tiles;
  const int length = length_of(A, request);
  const int begin = part * A.range, end = min(length, begin + A.range);
  if (begin >= length && !kFinal) return;

  const int lane = lane_id(), wave = wave_id(), c = lane & 31, h = lane >> 5;
  const int group = A.group.size, rows = A.tokens * group;
  const int row = tile * 32 + c;
  const bool valid = row < rows;
  const int row_in = valid ? row : rows - 1;
  const int token = A.group.div(row_in);
  const int q_head = head * group + row_in - token * group;
  const int64_t q_row = int64_t(request) * A.tokens + token;
  const int limit = A.lengths ? min(end, length - A.tokens + 1 + token) : end;

  Frags<T, DP> q;
  row_frags<T, DP>(q, A.q.at + q_row * A.q.row + q_head * A.q.head, A.chunks, true);
  const char *k_at = A.k.at + request * A.k.request + head * A.k.head;
  const char *v_at = A.v.at + request * A.v.request + head * A.v.head;
  char *mine = lds + wave * kMine;
  const unsigned mine0 = lds_address(lds) + wave * kMine;
  Stage<T, DP, 32, 64> k_stage, v_stage;
  k_stage.set(A.chunks, [&](int r) { return r * int(A.k.row); });
  v_stage.set(A.chunks, [&](int r) { return r * int(A.v.row); });
  auto load_keys = [&](int k0, int buffer) {
    load_rows(k_stage, k_at, A.k.row, k0, length, mine0 + buffer * 2 * kTile);
  };
  auto load_values = [&](int k0, int buffer) {
    load_rows(v_stage, v_at, A.v.row, k0, length, mine0 + buffer * 2 * kTile + kTile);
  };
  clear_rest<T, DP>(mine, kBuffers * 64, lane, 64, A.chunks);

  Sums<T, DP> out = {};
  Softmax x;
  constexpr int kStep = kWaves * 32, kLoads = Stage<T, DP, 32, 64>::kLoads;
  const int first = begin + wave * 32;
  if (first < end) {
    load_keys(first, 0);
    load_values(first, 0);
  }
  int buffer = 0;
  for (int k0 = first; k0 < end; k0 += kStep) {
    const bool more = k0 + kStep < end;
    if (kBuffers == 2 && more) {
      wait_reads();  // of the last round, from the buffer that is filled now
      load_keys(k0 + kStep, buffer ^ 1);
      load_values(k0 + kStep, buffer ^ 1);
      wait_loads<2 * kLoads>();  // all but the loads just issued
    } else {
      wait_loads<kBuffers == 2 ? 0 : kLoads>();  // (one buffer: the keys, not yet the values)
    }
    const char *k_tile = mine + buffer * 2 * kTile;
    float s[16];
    Frags<T, DP> k;
    read_rows<T, DP>(k, k_tile, 0);
    pin_reads();
    const f32x16 dots = dot_rows<T, DP>(k, q);
    if (kBuffers == 1 && more) {
      wait_reads();
      load_keys(k0 + kStep, 0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = k0 + c_row(r, h) < limit ? dots[r] : -kInf;
    softmax_step(s, x, out, A.scale_log2);
    Weights<T> w;
    w.set(s);
    if (kBuffers == 1) {
      if (more)
        wait_loads<kLoads>();  // the values: all but the next keys
      else
        wait_loads<0>();
    }
    Columns<T, DP> v;
    v.read(k_tile + kTile, 0);
    pin_reads();
    v.add(out, w);
    if (kBuffers == 2) {
      buffer ^= 1;
    } else if (more) {
      wait_reads();
      load_values(k0 + kStep, 0);
    }
  }

  // Join the waves: outputs as rows of floats over each wave's buffers.
  constexpr int kOut = PartPlan<T, DP>::kOut;
  float2 *tops = reinterpret_cast<float2 *>(lds + kWaves * kMine);
  const float sum = sum_halves(x.sum);
  if (h == 0) tops[wave * 32 + c] = make_float2(x.top * A.scale_log2, sum);
  float *put = reinterpret_cast<float *>(mine) + c * kOut;
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * b + 8 * g + 4 * h;
      if (d < DP)
        *reinterpret_cast<f32x4 *>(put + d) = f32x4{out[b][4 * g], out[b][4 * g + 1],
                                                    out[b][4 * g + 2], out[b][4 * g + 3]};
    }
  __syncthreads();
  // eight threads a row, four elements each at a time
  const int r = threadIdx.x >> 3;
  const int r_global = tile * 32 + r;
  if (r_global >= rows) return;
  float top = -kInf;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w * 32 + r].x);
  float by[kWaves], total = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    // (a wave that saw nothing has -inf, and -inf less -inf is no number)
    by[w] = tops[w * 32 + r].x == -kInf ? 0.f : exp2_fast(tops[w * 32 + r].x - top);
    total += by[w] * tops[w * 32 + r].y;
  }
  const int t = A.group.div(r_global);
  const int64_t q_at = int64_t(request) * A.tokens + t;
  const int o_head = head * group + r_global - t * group;
  const int64_t slot = int64_t(A.part0 + part) * A.rows + q_at * A.q_heads + o_head;
  const float norm = total > 0.f || total != total ? 1.f / total : 0.f;
  for (int d = (threadIdx.x & 7) * 4; d < A.dim; d += 32) {
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      v += by[w] * *reinterpret_cast<const f32x4 *>(lds + w * kMine + (r * kOut + d) * 4);
    if constexpr (kFinal) {
      typedef T Four __attribute__((ext_vector_type(4)));
      *reinterpret_cast<Four *>(A.out.at + q_at * A.out.row + o_head * A.out.head +
                                d * sizeof(T)) =
          Four{T(v[0] * norm), T(v[1] * norm), T(v[2] * norm), T(v[3] * norm)};
    } else {
      *reinterpret_cast<f32x4 *>(A.part_out + slot * A.dim + d) = v;
    }
  }
  if (!kFinal && (threadIdx.x & 7) == 0) A.part_top[slot] = make_float2(top, total);
}

// Rows of all requests (128 a block, 32 a wave) against one range of the
// prefix, as in attention over a packed sequence.
template <typename T, int DP>
__device__ __forceinline__ void prefix_part(const CachedArgs &A, char *lds, int at) {
  const int head = at % A.k_heads;
  at /= A.k_heads;
  const int tile = at % A.row_tiles, part = at / A.row_tiles;
  const int wave = wave_id(), c = lane_id() & 31, h = lane_id() >> 5;
  const int group = A.group.size, rows = A.tokens * group;
  const int w0 = (tile * kWaves + wave) * kWaveRows;
  const int row = w0 + c;
  const bool valid = row < rows;
  const int row_in = valid ? row : rows - 1;
  const int token = A.group.div(row_in);
  const int q_head = head * group + row_in - token * group;
  Frags<T, DP> q;
  row_frags<T, DP>(q, A.q.at + int64_t(token) * A.q.row + q_head * A.q.head, A.chunks, true);
  const int begin = part * A.range, end = min(A.capacity, begin + A.range);
  Sums<T, DP> out = {};
  Softmax x;
  attend_tiles<T, DP, 64>(lds, q, A.k.at + head * A.k.head, A.k.row, A.v.at + head * A.v.head,
                             A.v.row, A.chunks, begin, end, A.capacity, end, end,
                             w0 < rows ? end : begin, A.scale_log2, x, out);
  const float sum = sum_halves(x.sum);
  if (!valid) return;
  const int64_t slot = int64_t(A.part0 + part) * A.rows + int64_t(token) * A.q_heads + q_head;
  if (h == 0) A.part_top[slot] = make_float2(x.top * A.scale_log2, sum);
  float *put = A.part_out + slot * A.dim;
#pragma unroll
  for (int b = 0; b < Shape<T, DP>::kBlocks; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * b + 8 * g + 4 * h;
      if (d < A.dim)
        *reinterpret_cast<f32x4 *>(put + d) = f32x4{out[b][4 * g], out[b][4 * g + 1],
                                                    out[b][4 * g + 2], out[b][4 * g + 3]};
    }
}

// All parts of a call in one launch: the prefix' are bound by the matrix
// instructions where many rows share it, the own caches' by memory, and side
// by side on a CU they hide each other.  The blocks of the one are spread
// evenly among those of the other.
//
// 24 requests of 4 tokens with up to 16,384 keys, 8 heads of 64 in f16: 83 us,
// 4.9 TB/s of the caches, as a large copy; 64 requests of one token, up to
// 1,024 keys each and 16,896 of all, 8 heads of 128 in bf16: 56 us, 3.7 TB/s
// (the caches alone 33, the prefix alone 45); one request of 4,099 keys: 7.5
// us, the launch and one round of loads.
template <typename T, int DP, bool kByRows, bool kFinal>
__global__ __launch_bounds__(kThreads, DP * sizeof(T) > 256 ? 1 : 2) void parts_kernel(
    CachedArgs own, CachedArgs shared, int shared_blocks) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int64_t i = blockIdx.x, n = gridDim.x;
  const int before = int(i * shared_blocks / n);
  if (int((i + 1) * shared_blocks / n) == before) {
    cached_part<T, DP, kFinal>(own, lds, int(i) - before);
  } else if constexpr (kByRows) {
    prefix_part<T, DP>(shared, lds, before);
  } else if constexpr (!kFinal) {
    cached_part<T, DP, false>(shared, lds, before);
  }
}

// Joins the parts of a row, a block a row: a wave takes every fourth part, two
// neighbouring elements a lane.  `shared` parts are every row's, the rest as
// many as the request's length has ranges.  Bound by the latency of its two
// reads: 3.5 us for 32 rows, 7 us for 2,048, 8 us for 24 requests of
// 4 tokens and 32 heads with up to 19 parts (the loads of eight parts are in flight at a time).
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(CachedArgs A, int shared) {
  __shared__ float2 sums[kWaves][64];
  __shared__ float totals[kWaves];
  const int64_t row = blockIdx.x;
  const int lane = lane_id(), wave = wave_id();
  const int token = int(row / A.q_heads);
  const int parts = shared + (length_of(A, token / A.tokens) + A.range - 1) / A.range;
  float top = -kInf;
  for (int p = lane; p < parts; p += 64) top = fmaxf(top, A.part_top[p * A.rows + row].x);
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  const int d = 2 * lane < A.dim ? 2 * lane : A.dim - 2;  // (the lanes past dim read along)
  float total = 0.f, a = 0.f, b = 0.f;
#pragma unroll 8
  for (int p = wave; p < parts; p += kWaves) {
    const float2 t = A.part_top[p * A.rows + row];
    const float2 v =
        *reinterpret_cast<const float2 *>(A.part_out + (p * A.rows + row) * A.dim + d);
    const float by = t.x == -kInf ? 0.f : exp2_fast(t.x - top);
    total += by * t.y;
    a += by * v.x;
    b += by * v.y;
  }
  sums[wave][lane] = make_float2(a, b);
  if (lane == 0) totals[wave] = total;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    total += totals[w];
    a += sums[w][lane].x;
    b += sums[w][lane].y;
  }
  const float norm = total > 0.f || total != total ? 1.f / total : 0.f;
  if (2 * lane < A.dim) {
    typedef T Pair __attribute__((ext_vector_type(2)));
    *reinterpret_cast<Pair *>(A.out.at + token * A.out.row +
                              (row - int64_t(token) * A.q_heads) * A.out.head + d * sizeof(T)) =
        Pair{T(a * norm), T(b * norm)};
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Keys of a part: the least multiple of `step` such that `blocks` row tiles
// and heads times the parts are no more than `target` blocks.
int range_for(int64_t blocks, int keys, int64_t target, int step) {
  const int64_t parts = target / blocks > 1 ? target / blocks : 1;
  const int64_t range = ((keys + parts - 1) / parts + step - 1) / step * step;
  return int(range < step ? step : range);
}

struct CachedPlan {
  int own_range, own_parts, own_tiles;
  int shared_range, shared_parts, shared_tiles;
  bool by_rows;  // the prefix by prefix_part
  bool final;    // one part: no join
};

CachedPlan plan_cached(bool f32, int requests, int tokens, int capacity, int prefix, int q_heads,
                       int k_heads) {
  CachedPlan p = {};
  const int64_t group = q_heads / k_heads;
  p.own_tiles = int((tokens * group + 31) / 32);
  // About 4096 blocks even out caches of different lengths (24 requests of up
  // to 16,384 keys: 93 us, at 1024 blocks 101), but a part below 512 keys
  // costs more than it evens out (64 requests of up to 1,024 keys: 62 us at
  // 512, 73 at 256), unless the card would not be full.
  const int64_t own_blocks = int64_t(requests) * k_heads * p.own_tiles;
  p.own_range = own_blocks > 0 ? range_for(own_blocks, capacity, 4096, 128) : 128;
  if (p.own_range < 512) {
    const int full = own_blocks > 0 ? range_for(own_blocks, capacity, 512, 128) : 128;
    if (p.own_range < full) p.own_range = full < 512 ? full : 512;
  }
  p.own_parts = (capacity + p.own_range - 1) / p.own_range;
  if (prefix > 0) {
    const int64_t rows = requests * tokens * group;
    // The prefix by rows reads it once for 128 of them, by keys for 32, but by
    // rows most waves have none where there are few.  16,896 keys, own caches
    // of 100, us by rows and by keys: 8 heads of 128 in bf16 32 and 31 at 64
    // rows, 35 and 39 at 96, 54 and 97 at 256; 8 heads of 64 in f16 26 and 24,
    // 27 and 28, 41 and 52.  Float is bound by its matrix instructions, and
    // its tiles by rows hold half the keys: 4 heads of 64, 56 and 31 at 64
    // rows, 94 and 76 at 256, 312 and 264 at 1024.
    // Parts: by rows one block a CU, by keys two, for a part costs its sums and
    // the join.  us at half the blocks, as it is, twice and four times: 256
    // rows by rows, heads of 128, 16,896 keys 74, 55, 57 and 64, 4,096 keys 34,
    // 33, 40 and 50, heads of 64, 32,768 keys 44, 37, 37 and 46; 1,024 rows
    // (each tile for 32 parts and more) 241, 156, 142 and 139; by keys in fp32,
    // 64 rows 40, 31, 37 and 37, 1,024 rows 313, 261, 330 and 226.
    p.by_rows = !f32 && rows > 64;
    p.shared_tiles = int(p.by_rows ? (rows + 127) / 128 : (rows + 31) / 32);
    p.shared_range = range_for(int64_t(k_heads) * p.shared_tiles, prefix, p.by_rows ? 256 : 512,
                               p.by_rows ? 64 : 128);
    p.shared_parts = (prefix + p.shared_range - 1) / p.shared_range;
  }
  p.final = p.shared_parts == 0 && p.own_parts <= 1;
  return p;
}

template <typename T, int DP>
int launch_cached(const CachedArgs &own, const CachedArgs &shared, const CachedPlan &p,
                  hipStream_t s) {
  const int64_t shared_blocks =
      p.shared_parts > 0 ? int64_t(shared.row_tiles) * shared.k_heads * shared.parts : 0;
  const int64_t blocks =
      shared_blocks + int64_t(own.requests) * own.row_tiles * own.k_heads * own.parts;
  int st = check_grid(blocks, kThreads, "attention parts");
  if (st) return st;
  constexpr int kPrefixLds = 4 * Shape<T, DP>::tile_bytes(64);
  constexpr int kOwnLds = PartPlan<T, DP>::kLds;
  constexpr int kBothLds = kPrefixLds > kOwnLds ? kPrefixLds : kOwnLds;
  if (blocks > 0) {
    LaunchScope scope("attention_parts", s);
    const dim3 grid{unsigned(blocks)}, block{kThreads};
    if (p.final)
      hipLaunchKernelGGL((parts_kernel<T, DP, false, true>), grid, block, kOwnLds, s, own, shared,
                         0);
    else if (sizeof(T) == 2 && p.by_rows)
      hipLaunchKernelGGL((parts_kernel<T, DP, sizeof(T) == 2, false>), grid, block, kBothLds, s, own, shared,
                         int(shared_blocks));
    else
      hipLaunchKernelGGL((parts_kernel<T, DP, false, false>), grid, block, kOwnLds, s, own,
                         shared, int(shared_blocks));
  }
  st = check_launch("attention parts");
  if (st || p.final) return st;
  st = check_grid(own.rows, kThreads, "attention join");
  if (st) return st;
  LaunchScope scope("attention_join", s);
  hipLaunchKernelGGL((join_kernel<T>), dim3(unsigned(own.rows)), dim3(kThreads), 0, s, own,
                     p.shared_parts);
  return check_launch("attention join");
}

size_t scratch_for(const CachedPlan &p, int64_t rows, int dim) {
  if (p.final) return 0;
  return size_t(p.own_parts + p.shared_parts) * size_t(rows) * (size_t(dim) + 2) * sizeof(float);
}

bool cached_sizes_ok(int requests, int tokens, int capacity, int prefix, int q_heads,
                     int k_heads) {
  return requests >= 0 && tokens >= 1 && capacity >= 0 && prefix >= 0 && k_heads >= 1 &&
         q_heads >= k_heads && q_heads % k_heads == 0 &&
         int64_t(requests) * tokens * q_heads * (q_heads / k_heads) < (int64_t(1) << 31) &&
         capacity < (1 << 30) && prefix < (1 << 30);
}

}  // namespace

extern "C" {

size_t bevpool_attention_cached_scratch_bytes(int32_t requests, int32_t tokens, int32_t capacity,
                                              int32_t prefix, int32_t q_heads, int32_t k_heads,
                                              int32_t dim) {
  if (!cached_sizes_ok(requests, tokens, capacity, prefix, q_heads, k_heads) || dim < 1) return 0;
  size_t most = 0;  // of the types' plans
  for (const bool f32 : {false, true}) {
    const size_t need =
        scratch_for(plan_cached(f32, requests, tokens, capacity, prefix, q_heads, k_heads),
                    int64_t(requests) * tokens * q_heads, dim);
    if (need > most) most = need;
  }
  return most;
}

int bevpool_attention_cached(const void *q, int64_t q_row, int64_t q_head, const void *k,
                             int64_t k_request, int64_t k_row, int64_t k_head, const void *v,
                             int64_t v_request, int64_t v_row, int64_t v_head,
                             const void *prefix_k, int64_t prefix_k_row, int64_t prefix_k_head,
                             const void *prefix_v, int64_t prefix_v_row, int64_t prefix_v_head,
                             const int32_t *lengths, int32_t dtype, int32_t requests,
                             int32_t tokens, int32_t capacity, int32_t prefix, int32_t q_heads,
                             int32_t k_heads, int32_t dim, float scale, void *out, void *scratch,
                             size_t scratch_bytes, void *stream) {
  bevpool_host::clear_error();
  if (dtype < BEVPOOL_F32 || dtype > BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d", dtype);
  if (!cached_sizes_ok(requests, tokens, capacity, prefix, q_heads, k_heads))
    return fail(BEVPOOL_EINVAL,
                "bad sizes (%d requests of %d tokens, caches of %d, prefix of %d, %d heads over "
                "%d)",
                requests, tokens, capacity, prefix, q_heads, k_heads);
  if (dim < 8 || dim > 128 || dim % 8)
    return fail(BEVPOOL_EINVAL, "head size %d: must be a multiple of 8 up to 128", dim);
  if (!(scale >= 1e-30f) || !(scale < 3e38f))
    return fail(BEVPOOL_EINVAL, "scale must be positive (1e-30 or more) and finite");
  if (requests == 0) return BEVPOOL_OK;
  if (!lengths) return fail(BEVPOOL_EINVAL, "lengths: null");
  const int elem = dtype == BEVPOOL_F32 ? 4 : 2;
  const int64_t rows = int64_t(requests) * tokens;
  Operand oq, oo, okey, oval, opk, opv;
  int st = set_operand(oq, "q", q, q_row, q_head, elem, rows);
  if (!st) st = set_operand(oo, "out", out, int64_t(q_heads) * dim, dim, elem, rows);
  if (!st) st = set_operand(okey, "k", k, k_row, k_head, elem, capacity);
  if (!st) st = set_operand(oval, "v", v, v_row, v_head, elem, capacity);
  if (!st) st = set_operand(opk, "prefix_k", prefix_k, prefix_k_row, prefix_k_head, elem, prefix);
  if (!st) st = set_operand(opv, "prefix_v", prefix_v, prefix_v_row, prefix_v_head, elem, prefix);
  if (st) return st;
  if (capacity > 0 && (k_request * elem % 16 || v_request * elem % 16))
    return fail(BEVPOOL_EINVAL, "caches of requests must start at multiples of 16 bytes");
  const CachedPlan p = plan_cached(dtype == BEVPOOL_F32, requests, tokens, capacity, prefix, q_heads, k_heads);
  const size_t need = scratch_for(p, rows * q_heads, dim);
  if (scratch_bytes < need || (need > 0 && !scratch))
    return fail(BEVPOOL_ESPACE, "attention scratch: %zu bytes, %zu needed", scratch_bytes, need);

  CachedArgs own = {};
  own.q = oq;
  own.out = oo;
  own.k = {okey.at, k_request * elem, okey.row, okey.head};
  own.v = {oval.at, v_request * elem, oval.row, oval.head};
  own.lengths = lengths;
  own.requests = requests;
  own.tokens = tokens;
  own.capacity = capacity;
  own.q_heads = q_heads;
  own.k_heads = k_heads;
  own.group = make_group(q_heads / k_heads);
  own.dim = dim;
  own.chunks = dim * elem / 16;
  own.scale_log2 = scale * kLog2e;
  own.range = p.own_range;
  own.parts = p.final ? 1 : p.own_parts;
  own.row_tiles = p.own_tiles;
  own.part0 = p.shared_parts;
  own.rows = rows * q_heads;
  own.part_out = static_cast<float *>(scratch);
  own.part_top = reinterpret_cast<float2 *>(
      own.part_out + int64_t(p.own_parts + p.shared_parts) * own.rows * dim);
  // the prefix: one request of all the rows, with a cache that all of them see
  CachedArgs shared = own;
  shared.k = {opk.at, 0, opk.row, opk.head};
  shared.v = {opv.at, 0, opv.row, opv.head};
  shared.lengths = nullptr;
  shared.requests = 1;
  shared.tokens = int(rows);
  shared.capacity = prefix;
  shared.range = p.shared_range;
  shared.parts = p.shared_parts;
  shared.row_tiles = p.shared_tiles;
  shared.part0 = 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == BEVPOOL_BF16  ? (ATTENTION_DIM(__bf16, launch_cached, own, shared, p, s))
         : dtype == BEVPOOL_F16 ? (ATTENTION_DIM(_Float16, launch_cached, own, shared, p, s))
                                : (ATTENTION_DIM(float, launch_cached, own, shared, p, s));
}

}  // extern "C"

// rotate.hip -- norm of queries and keys for each head and rotation by
// positions with several axes, in one pass, forward and backward (gfx950).
//
//   r      = 1 / sqrt(mean_d x_d^2 + eps)             (with weights; else 1)
//   n_d    = x_d r w_d
//   angle  = pos[t, axis(p)] * frequency[p]           for pair p = (a, b)
//   y_a    = n_a cos - n_b sin,  y_b = n_b cos + n_a sin
// Pair p is (p, P + p) of the first 2P elements, or (2p, 2p + 1) where the
// pairs are interleaved; elements from 2P on are only normed.
//
// Backward, with g the gradient turned back by the same angles:
//   dw_d = sum over tokens and heads of g_d x_d r
//   dx_d = r (g_d w_d - x_d r^2 mean_j(g_j w_j x_j))
//
// Both are bound by memory: x (and dy) read once, y (dx) written once.  16,896
// tokens of 16 + 16 heads of 80 in bf16: forward 39 us (4.5 TB/s of what has
// to move; a large copy reaches 5.1), backward 64 us (4.1 TB/s) and 4 us for
// the weights' sums.  32,400 tokens of 8 + 8 heads of 64 in fp32: 45 us (5.9
// TB/s, part of it from the caches), 80 us (5.0 TB/s) and 4.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bevpool.h"
#include "host_calls.h"

namespace {

using bevpool_host::check_grid;
using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;    // elements of a head
constexpr int kMaxAxes = 4;

struct Heads {  // one operand: (tokens, heads, dim), unit stride along dim
  const void *x;
  const void *dy;      // backward
  void *y;             // dx in the backward
  const void *weight;  // (dim) or null
  float *partial;      // backward: [blocks][dim] of the weight's gradient
  int64_t x_token, x_head, dy_token, dy_head, y_token, y_head;
  int heads;
};

struct RotateArgs {
  Heads q, k;  // k.heads may be 0
  const void *positions;
  const float *frequencies;
  int64_t tokens, pos_stride;
  int dim, pairs, interleaved, pos_kind;  // pos_kind: 0 int32, 1 int64, 2 float32
  int axis_end[kMaxAxes];                 // pairs [axis_end[i - 1], axis_end[i]) turn by axis i
  int units;                              // units of 2 V elements in a row
  float eps, inv_dim;
};

template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load(float (&to)[V], const T *from) {
  const Pack<T, V> p = *reinterpret_cast<const Pack<T, V> *>(from);
#pragma unroll
  for (int i = 0; i < V; ++i) to[i] = float(p.v[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store(T *to, const float (&from)[V]) {
  Pack<T, V> p;
#pragma unroll
  for (int i = 0; i < V; ++i) p.v[i] = T(from[i]);
  *reinterpret_cast<Pack<T, V> *>(to) = p;
}

// Where a thread stands: rows are worked on by groups of `lanes` consecutive
// lanes of a wave, as many as fit it; the lanes left over have a group past
// all rows and a lane past all units.
struct Place {
  int lane, group, groups;
};
__device__ __forceinline__ Place place_of(int lanes) {
  const int in_wave = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per_wave = 64 / lanes, g = in_wave / lanes;
  if (g >= per_wave) return {1 << 20, 1 << 30, 1 << 30};
  return {in_wave - g * lanes, wave * per_wave + g, per_wave * (kThreads / 64)};
}

// Sum over a group's lanes, in all of them.
__device__ __forceinline__ float group_sum(float v, int lanes) {
  if ((lanes & (lanes - 1)) == 0) {
    for (int m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m, 64);
    return v;
  }
  // lane i collects the lanes i .. i + 2 m - 1 that there are; the first has
  // all in the end
  const int in_wave = threadIdx.x & 63, first = in_wave / lanes * lanes, lane = in_wave - first;
  for (int m = 1; m < lanes; m <<= 1) {
    const float other = __shfl(v, in_wave + m, 64);
    if (lane + m < lanes) v += other;
  }
  return __shfl(v, first, 64);
}

// cos and sin of pos * frequency.  The product in double (an angle of 10^5
// in 32 bits is off by 4e-3) and reduced there to one turn, so the functions
// see at most half a turn whatever the position.
__device__ __forceinline__ float2 turn(const RotateArgs &A, int64_t token, int pair) {
  int axis = 0;
#pragma unroll
  for (int i = 0; i < kMaxAxes - 1; ++i) axis += pair >= A.axis_end[i];
  const int64_t at = token * A.pos_stride + axis;
  const double pos = A.pos_kind == 0   ? double(static_cast<const int32_t *>(A.positions)[at])
                     : A.pos_kind == 1 ? double(static_cast<const int64_t *>(A.positions)[at])
                                       : double(static_cast<const float *>(A.positions)[at]);
  const double half_turns = pos * double(A.frequencies[pair]) * 0.31830988618379067154;
  const double whole = 2.0 * rint(0.5 * half_turns);
  float2 cs;
  sincospif(float(half_turns - whole), &cs.y, &cs.x);
  return cs;
}

// Where unit u of a row lies: elements [a, a + V) and [b, b + V), and the
// first of its V pairs (pairs or more: not turned).  In the halves' layout a
// unit is V pairs, or 2 V neighbours past the pairs; interleaved, 2 V
// neighbours.
struct Unit {
  int a, b, pair;
};

template <int V>
__device__ __forceinline__ Unit unit_at(const RotateArgs &A, int u) {
  if (A.interleaved) return {2 * V * u, 2 * V * u + V, V * u};
  const int turned = A.pairs / V;
  if (u < turned) return {V * u, A.pairs + V * u, V * u};
  const int d = 2 * A.pairs + 2 * V * (u - turned);
  return {d, d + V, A.pairs};
}

// Turns the unit's elements by its pairs' angles, or back.
template <int V>
__device__ __forceinline__ void turn_unit(float (&a)[V], float (&b)[V], const float2 *cs,
                                          const RotateArgs &A, const Unit &u, bool back) {
  if (A.interleaved) {
    // element 2 i of the unit pairs with 2 i + 1; i runs through a, then b
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (u.pair + i >= A.pairs) break;
      const float2 c = cs[u.pair + i];
      const float s = back ? -c.y : c.y;
      // (V == 1: the pair is (a[0], b[0]))
      float &lo = V == 1 ? a[0] : 2 * i < V ? a[(2 * i) % V] : b[(2 * i) % V];
      float &hi = V == 1 ? b[0] : 2 * i < V ? a[(2 * i + 1) % V] : b[(2 * i + 1) % V];
      const float l = lo, h = hi;
      lo = l * c.x - h * s;
      hi = h * c.x + l * s;
    }
  } else if (u.pair < A.pairs) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 c = cs[u.pair + i];
      const float s = back ? -c.y : c.y;
      const float l = a[i], h = b[i];
      a[i] = l * c.x - h * s;
      b[i] = h * c.x + l * s;
    }
  }
}

// A block takes `tile` tokens: the tile's angles once into LDS, then the
// rows (token, head), each by a group of `lanes` lanes with one unit a lane.
// The lanes of a row hold all of it, so norm, rotation and store need no
// second read.  kUnits > 1: rows of more units than the group has lanes.
template <typename T, int V, int kUnits>
__global__ __launch_bounds__(kThreads) void norm_rotate_kernel(RotateArgs A, int tile, int lanes) {
  extern __shared__ float2 cs[];
  const int64_t t0 = int64_t(blockIdx.x) * tile;
  const int n_tokens = int(A.tokens - t0 < tile ? A.tokens - t0 : tile);
  for (int i = threadIdx.x; i < n_tokens * A.pairs; i += kThreads) {
    const int t = i / A.pairs;
    cs[i] = turn(A, t0 + t, i - t * A.pairs);
  }
  __syncthreads();
  const Place place = place_of(lanes);
  const int lane = place.lane, group = place.group, groups = place.groups;
  const int heads = A.q.heads + A.k.heads;
  // group-uniform: the lanes of one sum leave the loop together
  for (int row = group; row < n_tokens * heads; row += groups) {
    const int t = row / heads, h = row - t * heads;
    const bool is_q = h < A.q.heads;
    const Heads &X = is_q ? A.q : A.k;
    const int head = is_q ? h : h - A.q.heads;
    const T *x = static_cast<const T *>(X.x) + (t0 + t) * X.x_token + head * X.x_head;
    T *y = static_cast<T *>(X.y) + (t0 + t) * X.y_token + head * X.y_head;
    const T *w = static_cast<const T *>(X.weight);
    float a[kUnits][V], b[kUnits][V];
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int u = lane + j * lanes;
      if (u >= A.units) continue;
      const Unit at = unit_at<V>(A, u);
      load<T, V>(a[j], x + at.a);
      load<T, V>(b[j], x + at.b);
#pragma unroll
      for (int i = 0; i < V; ++i) sum += a[j][i] * a[j][i] + b[j][i] * b[j][i];
    }
    const float r = w ? 1.0f / sqrtf(group_sum(sum, lanes) * A.inv_dim + A.eps) : 1.0f;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int u = lane + j * lanes;
      if (u >= A.units) continue;
      const Unit at = unit_at<V>(A, u);
      if (w) {
        float wa[V], wb[V];
        load<T, V>(wa, w + at.a);
        load<T, V>(wb, w + at.b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a[j][i] = a[j][i] * r * wa[i];
          b[j][i] = b[j][i] * r * wb[i];
        }
      }
      turn_unit<V>(a[j], b[j], cs + t * A.pairs, A, at, false);
      store<T, V>(y + at.a, a[j]);
      store<T, V>(y + at.b, b[j]);
    }
  }
}

// One row's elements of this lane, as they lie in memory.
template <typename T, int V, int kUnits>
struct RowData {
  Pack<T, V> xa[kUnits], xb[kUnits], ga[kUnits], gb[kUnits];
};

// Backward of one operand's rows of a tile; dwa, dwb collect this lane's part
// of the weight's gradient (a lane keeps its units over all its rows, and
// their weights wa, wb).  The next row's loads are in flight while one is
// worked on.
template <typename T, int V, int kUnits>
__device__ __forceinline__ void backward_rows(const RotateArgs &A, const Heads &X, int64_t t0,
                                              int n_tokens, int lanes, const float2 *cs,
                                              const Pack<T, V> (&wa)[kUnits],
                                              const Pack<T, V> (&wb)[kUnits],
                                              float (&dwa)[kUnits][V], float (&dwb)[kUnits][V]) {
  const Place place = place_of(lanes);
  const int lane = place.lane, group = place.group, groups = place.groups;
  const bool w = X.weight != nullptr;
  const int rows = n_tokens * X.heads;
  auto fetch = [&](int row, RowData<T, V, kUnits> &d) {
    const int t = row / X.heads, head = row - t * X.heads;
    const T *x = static_cast<const T *>(X.x) + (t0 + t) * X.x_token + head * X.x_head;
    const T *dy = static_cast<const T *>(X.dy) + (t0 + t) * X.dy_token + head * X.dy_head;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int u = lane + j * lanes;
      if (u >= A.units) continue;
      const Unit at = unit_at<V>(A, u);
      d.ga[j] = *reinterpret_cast<const Pack<T, V> *>(dy + at.a);
      d.gb[j] = *reinterpret_cast<const Pack<T, V> *>(dy + at.b);
      if (w) {
        d.xa[j] = *reinterpret_cast<const Pack<T, V> *>(x + at.a);
        d.xb[j] = *reinterpret_cast<const Pack<T, V> *>(x + at.b);
      }
    }
  };
  RowData<T, V, kUnits> next;
  if (group < rows) fetch(group, next);
  for (int row = group; row < rows; row += groups) {
    const RowData<T, V, kUnits> d = next;
    if (row + groups < rows) fetch(row + groups, next);
    const int t = row / X.heads, head = row - t * X.heads;
    T *dx = static_cast<T *>(X.y) + (t0 + t) * X.y_token + head * X.y_head;
    float ga[kUnits][V], gb[kUnits][V];
    float sum = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int u = lane + j * lanes;
      if (u >= A.units) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ga[j][i] = float(d.ga[j].v[i]);
        gb[j][i] = float(d.gb[j].v[i]);
      }
      turn_unit<V>(ga[j], gb[j], cs + t * A.pairs, A, unit_at<V>(A, u), true);
      if (w) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float a = float(d.xa[j].v[i]), b = float(d.xb[j].v[i]);
          sum += a * a + b * b;
          dot += ga[j][i] * float(wa[j].v[i]) * a + gb[j][i] * float(wb[j].v[i]) * b;
        }
      }
    }
    float r = 1.f, back = 0.f;
    if (w) {
      r = 1.0f / sqrtf(group_sum(sum, lanes) * A.inv_dim + A.eps);
      back = group_sum(dot, lanes) * A.inv_dim * r * r;
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const int u = lane + j * lanes;
      if (u >= A.units) continue;
      const Unit at = unit_at<V>(A, u);
      if (w) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float a = float(d.xa[j].v[i]), b = float(d.xb[j].v[i]);
          dwa[j][i] += ga[j][i] * (a * r);
          dwb[j][i] += gb[j][i] * (b * r);
          ga[j][i] = r * (ga[j][i] * float(wa[j].v[i]) - a * back);
          gb[j][i] = r * (gb[j][i] * float(wb[j].v[i]) - b * back);
        }
      }
      store<T, V>(dx + at.a, ga[j]);
      store<T, V>(dx + at.b, gb[j]);
    }
  }
}

// This lane's weights.
template <typename T, int V, int kUnits>
__device__ __forceinline__ void load_weights(const RotateArgs &A, const Heads &X, int lanes,
                                             Pack<T, V> (&wa)[kUnits], Pack<T, V> (&wb)[kUnits]) {
  const T *w = static_cast<const T *>(X.weight);
  const int lane = place_of(lanes).lane;
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int u = lane + j * lanes;
    if (!w || u >= A.units) continue;
    const Unit at = unit_at<V>(A, u);
    wa[j] = *reinterpret_cast<const Pack<T, V> *>(w + at.a);
    wb[j] = *reinterpret_cast<const Pack<T, V> *>(w + at.b);
  }
}

// The groups' parts of a weight's gradient, added in the groups' order.
template <int V, int kUnits>
__device__ __forceinline__ void flush_weight(const RotateArgs &A, const Heads &X, int block,
                                             int lanes, float *sums, const float (&dwa)[kUnits][V],
                                             const float (&dwb)[kUnits][V]) {
  if (!X.weight) return;
  const Place place = place_of(lanes);
  const int lane = place.lane, group = place.group;
  const int all = 64 / lanes * (kThreads / 64);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const int u = lane + j * lanes;
    if (u >= A.units) continue;
    const Unit at = unit_at<V>(A, u);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sums[group * A.dim + at.a + i] = dwa[j][i];
      sums[group * A.dim + at.b + i] = dwb[j][i];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < A.dim; d += kThreads) {
    float s = 0.f;
    for (int g = 0; g < all; ++g) s += sums[g * A.dim + d];
    X.partial[int64_t(block) * A.dim + d] = s;
  }
}

// As the forward, but a block walks an equal share of one operand's tokens, so
// that its weight's gradient leaves it once, and holds one weight and one
// gradient of it: in 128 registers, four blocks a CU.
template <typename T, int V, int kUnits>
__global__ __launch_bounds__(kThreads, (kUnits == 1 ? 4 : 2)) void norm_rotate_backward_kernel(
    RotateArgs A, int tile, int lanes, int q_blocks) {
  extern __shared__ float2 cs[];
  const bool is_q = int(blockIdx.x) < q_blocks;
  const Heads &X = is_q ? A.q : A.k;
  const int block = is_q ? blockIdx.x : blockIdx.x - q_blocks;
  const int blocks = is_q ? q_blocks : gridDim.x - q_blocks;
  float dwa[kUnits][V] = {}, dwb[kUnits][V] = {};
  Pack<T, V> wa[kUnits], wb[kUnits];
  load_weights<T, V, kUnits>(A, X, lanes, wa, wb);
  const int64_t share = (A.tokens + blocks - 1) / blocks;
  const int64_t end = A.tokens < (block + 1) * share ? A.tokens : (block + 1) * share;
  for (int64_t t0 = block * share; t0 < end; t0 += tile) {
    const int n_tokens = int(end - t0 < tile ? end - t0 : tile);
    __syncthreads();  // the last tile's angles have been read
    for (int i = threadIdx.x; i < n_tokens * A.pairs; i += kThreads) {
      const int t = i / A.pairs;
      cs[i] = turn(A, t0 + t, i - t * A.pairs);
    }
    __syncthreads();
    backward_rows<T, V, kUnits>(A, X, t0, n_tokens, lanes, cs, wa, wb, dwa, dwb);
  }
  flush_weight<V, kUnits>(A, X, block, lanes, reinterpret_cast<float *>(cs), dwa, dwb);
}

// Column sums of the blocks' parts: a wave an element, lanes along the
// blocks, always in the same order.
template <typename T>
__global__ __launch_bounds__(64) void weight_sum_kernel(const float *q_partial, T *dq_weight,
                                                        const float *k_partial, T *dk_weight,
                                                        int q_blocks, int k_blocks, int dim) {
  const bool is_q = int(blockIdx.x) < dim;
  const int d = is_q ? blockIdx.x : blockIdx.x - dim;
  const float *from = is_q ? q_partial : k_partial;
  T *to = is_q ? dq_weight : dk_weight;
  const int blocks = is_q ? q_blocks : k_blocks;
  if (!to) return;
  float s = 0.f;
  for (int b = threadIdx.x; b < blocks; b += 64) s += from[int64_t(b) * dim + d];
  s = group_sum(s, 64);
  if (threadIdx.x == 0) to[d] = T(s);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

struct Plan {
  int vec;    // elements of one access
  int units;  // a row's units of 2 vec elements
  int lanes;  // lanes of a row
  int tile;   // tokens whose angles a block holds
};

// The widest access, up to 16 bytes, whose units tile both the pairs and the
// rest of a row.
Plan plan_for(int elem, int dim, int pairs, int interleaved, int heads,
              int64_t tokens) {
  Plan p;
  for (p.vec = 16 / elem; p.vec > 1; p.vec /= 2) {
    if (interleaved ? dim % (2 * p.vec) == 0
                    : pairs % p.vec == 0 && (dim - 2 * pairs) % (2 * p.vec) == 0)
      break;
  }
  p.units = dim / (2 * p.vec);
  // A power of two, whose sums take fewer steps, unless that leaves a fifth of
  // the lanes without a unit (5 units of a head of 80 on 8 lanes: backward of
  // 16,896 x 32 rows 76 us, on 5 lanes 64).
  p.lanes = 1;
  while (p.lanes < p.units && p.lanes < 64) p.lanes *= 2;
  if (p.units * 5 < p.lanes * 4) p.lanes = p.units;
  // Enough rows for four rounds of the block's groups, at most 16 tokens, and
  // no fewer blocks than CUs.  Forward, us at 1 token, by this rule, at 16:
  // 30,011 tokens of 8 heads 43, 22, 22; 16,896 of 32 48, 40, 43; 5,000 of 32
  // 21, 21, 27; 16 of 40 28, 26, 33.
  p.tile = 1;
  while (p.tile < 16 && p.tile * heads < 4 * (kThreads / p.lanes) && tokens >= p.tile * 512)
    p.tile *= 2;
  return p;
}

int check_operand(const char *what, const void *x, const void *y, const void *weight, int heads,
                  int64_t tokens) {
  if (heads < 0) return fail(BEVPOOL_EINVAL, "%s: negative number of heads", what);
  if (tokens > 0 && heads > 0 && (!x || !y)) return fail(BEVPOOL_EINVAL, "%s: null rows", what);
  if (heads == 0 && weight) return fail(BEVPOOL_EINVAL, "%s: a weight, but no heads", what);
  return BEVPOOL_OK;
}

int fill_args(RotateArgs &A, int dtype, int64_t tokens, int dim, const void *positions,
              int pos_kind, int64_t pos_stride, const float *frequencies, const int32_t *axis_pairs,
              int n_axes, int interleaved, float eps) {
  if (dtype < BEVPOOL_F32 || dtype > BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d", dtype);
  if (tokens < 0) return fail(BEVPOOL_EINVAL, "negative number of tokens");
  if (dim < 2 || dim > kMaxDim || dim % 2)
    return fail(BEVPOOL_EINVAL, "head size %d: must be even and in [2, %d]", dim, kMaxDim);
  if (n_axes < 0 || n_axes > kMaxAxes || (n_axes > 0 && !axis_pairs))
    return fail(BEVPOOL_EINVAL, "between 0 and %d axes", kMaxAxes);
  int pairs = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    if (i < n_axes) {
      if (axis_pairs[i] < 0 || axis_pairs[i] > dim / 2)
        return fail(BEVPOOL_EINVAL, "axis %d: %d pairs do not fit a head of %d", i, axis_pairs[i],
                    dim);
      pairs += axis_pairs[i];
    }
    A.axis_end[i] = pairs;
  }
  if (2 * pairs > dim)
    return fail(BEVPOOL_EINVAL, "%d pairs do not fit a head of %d elements", pairs, dim);
  if (pairs > 0 && tokens > 0 && (!positions || !frequencies))
    return fail(BEVPOOL_EINVAL, "null positions or frequencies");
  if (pos_kind < 0 || pos_kind > 2)
    return fail(BEVPOOL_EINVAL, "position type %d: 0 int32, 1 int64, 2 float32", pos_kind);
  if (!(eps >= 0.f)) return fail(BEVPOOL_EINVAL, "eps must not be negative");
  A.positions = positions;
  A.frequencies = frequencies;
  A.tokens = tokens;
  A.pos_stride = pos_stride;
  A.dim = dim;
  A.pairs = pairs;
  A.interleaved = interleaved != 0;
  A.pos_kind = pos_kind;
  A.eps = eps;
  A.inv_dim = 1.0f / float(dim);
  return BEVPOOL_OK;
}

// Blocks of the backward, of both operands by their heads: as many as the card
// holds at once (256 CUs, 4 each), or as there are tiles.
constexpr int kBackwardBlocks = 1024;
void backward_blocks(int64_t tokens, const Plan &p, int q_heads, int k_heads, int *q_blocks,
                     int *k_blocks) {
  const int64_t tiles = (tokens + p.tile - 1) / p.tile, heads = q_heads + k_heads;
  auto share = [&](int64_t n) {
    const int64_t part = heads > 0 ? (kBackwardBlocks * n + heads - 1) / heads : 0;
    return int(tiles < part ? tiles : part);
  };
  *q_blocks = share(q_heads);
  *k_blocks = share(k_heads);
}

template <typename T, int V>
void launch_forward(const RotateArgs &A, const Plan &p, unsigned grid, hipStream_t s) {
  const size_t lds = sizeof(float2) * size_t(p.tile) * A.pairs;
  const int per_lane = (A.units + p.lanes - 1) / p.lanes;
  if (per_lane == 1)
    hipLaunchKernelGGL((norm_rotate_kernel<T, V, 1>), dim3(grid), dim3(kThreads), lds, s, A,
                       p.tile, p.lanes);
  else
    hipLaunchKernelGGL((norm_rotate_kernel<T, V, 2>), dim3(grid), dim3(kThreads), lds, s, A,
                       p.tile, p.lanes);
}

template <typename T, int V>
void launch_backward(const RotateArgs &A, const Plan &p, int q_blocks, int k_blocks,
                     hipStream_t s) {
  const unsigned grid = q_blocks + k_blocks;
  const size_t angles = sizeof(float2) * size_t(p.tile) * A.pairs;
  const size_t sums = sizeof(float) * size_t(kThreads / p.lanes) * A.dim;
  const size_t lds = angles > sums ? angles : sums;
  const int per_lane = (A.units + p.lanes - 1) / p.lanes;
  if (per_lane == 1)
    hipLaunchKernelGGL((norm_rotate_backward_kernel<T, V, 1>), dim3(grid), dim3(kThreads), lds, s,
                       A, p.tile, p.lanes, q_blocks);
  else
    hipLaunchKernelGGL((norm_rotate_backward_kernel<T, V, 2>), dim3(grid), dim3(kThreads), lds, s,
                       A, p.tile, p.lanes, q_blocks);
}

#define ROTATE_VEC(T, FN, ...)                       \
  switch (p.vec) {                                   \
    case 8: FN<T, 8>(__VA_ARGS__); break;            \
    case 4: FN<T, 4>(__VA_ARGS__); break;            \
    case 2: FN<T, 2>(__VA_ARGS__); break;            \
    default: FN<T, 1>(__VA_ARGS__); break;           \
  }
#define ROTATE_TYPE(FN, ...)                                                        \
  if (dtype == BEVPOOL_F32) {                                                       \
    switch (p.vec) {                                                                \
      case 4: FN<float, 4>(__VA_ARGS__); break;                                     \
      case 2: FN<float, 2>(__VA_ARGS__); break;                                     \
      default: FN<float, 1>(__VA_ARGS__); break;                                    \
    }                                                                               \
  } else if (dtype == BEVPOOL_F16) {                                                \
    ROTATE_VEC(_Float16, FN, __VA_ARGS__)                                           \
  } else {                                                                          \
    ROTATE_VEC(__bf16, FN, __VA_ARGS__)                                             \
  }

}  // namespace

extern "C" {

int bevpool_norm_rotate_forward(const void *q, int64_t q_token, int64_t q_head, int32_t q_heads,
                                const void *k, int64_t k_token, int64_t k_head, int32_t k_heads,
                                int32_t dtype, int64_t tokens, int32_t dim, const void *positions,
                                int32_t pos_kind, int64_t pos_stride, const float *frequencies,
                                const int32_t *axis_pairs, int32_t n_axes, int32_t interleaved,
                                const void *q_weight, const void *k_weight, float eps, void *q_out,
                                void *k_out, void *stream) {
  bevpool_host::clear_error();
  RotateArgs A = {};
  int st = fill_args(A, dtype, tokens, dim, positions, pos_kind, pos_stride, frequencies,
                     axis_pairs, n_axes, interleaved, eps);
  if (!st) st = check_operand("q", q, q_out, q_weight, q_heads, tokens);
  if (!st) st = check_operand("k", k, k_out, k_weight, k_heads, tokens);
  if (st) return st;
  const int heads = q_heads + k_heads;
  if (tokens == 0 || heads == 0) return BEVPOOL_OK;
  const int64_t d = dim;
  A.q = {q, nullptr, q_out, q_weight, nullptr, q_token, q_head, 0, 0, q_heads * d, d, q_heads};
  A.k = {k, nullptr, k_out, k_weight, nullptr, k_token, k_head, 0, 0, k_heads * d, d, k_heads};
  const Plan p = plan_for(dtype == BEVPOOL_F32 ? 4 : 2, dim, A.pairs, A.interleaved, heads,
                          tokens);
  A.units = p.units;
  const int64_t grid = (tokens + p.tile - 1) / p.tile;
  st = check_grid(grid, kThreads, "norm_rotate");
  if (st) return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  LaunchScope scope("norm_rotate", s);
  ROTATE_TYPE(launch_forward, A, p, unsigned(grid), s)
  return check_launch("norm_rotate");
}

size_t bevpool_norm_rotate_backward_scratch_bytes(int32_t dim) {
  return dim < 1 ? 0 : size_t(2) * kBackwardBlocks * size_t(dim) * sizeof(float);
}

int bevpool_norm_rotate_backward(
    const void *q, int64_t q_token, int64_t q_head, int32_t q_heads, const void *k,
    int64_t k_token, int64_t k_head, int32_t k_heads, const void *dq_out, int64_t dq_token,
    int64_t dq_head, const void *dk_out, int64_t dk_token, int64_t dk_head, int32_t dtype,
    int64_t tokens, int32_t dim, const void *positions, int32_t pos_kind, int64_t pos_stride,
    const float *frequencies, const int32_t *axis_pairs, int32_t n_axes, int32_t interleaved,
    const void *q_weight, const void *k_weight, float eps, void *dq, void *dk, void *dq_weight,
    void *dk_weight, void *scratch, size_t scratch_bytes, void *stream) {
  bevpool_host::clear_error();
  RotateArgs A = {};
  int st = fill_args(A, dtype, tokens, dim, positions, pos_kind, pos_stride, frequencies,
                     axis_pairs, n_axes, interleaved, eps);
  if (!st) st = check_operand("dq_out", dq_out, dq, q_weight, q_heads, tokens);
  if (!st) st = check_operand("dk_out", dk_out, dk, k_weight, k_heads, tokens);
  if (!st && q_weight) st = check_operand("q", q, dq, q_weight, q_heads, tokens);
  if (!st && k_weight) st = check_operand("k", k, dk, k_weight, k_heads, tokens);
  if (st) return st;
  if ((q_weight && !dq_weight) || (k_weight && !dk_weight))
    return fail(BEVPOOL_EINVAL, "a weight without the place of its gradient");
  if ((q_weight || k_weight) &&
      (!scratch || scratch_bytes < bevpool_norm_rotate_backward_scratch_bytes(dim)))
    return fail(BEVPOOL_ESPACE, "norm_rotate backward scratch too small");
  const int heads = q_heads + k_heads;
  const int64_t d = dim;
  float *parts = static_cast<float *>(scratch);
  A.q = {q, dq_out, dq, q_weight, parts, q_token, q_head, dq_token, dq_head, q_heads * d, d,
         q_heads};
  A.k = {k, dk_out, dk, k_weight, parts + (q_weight || k_weight ? kBackwardBlocks * d : 0), k_token, k_head,
         dk_token, dk_head, k_heads * d, d, k_heads};
  Plan p = plan_for(dtype == BEVPOOL_F32 ? 4 : 2, dim, A.pairs, A.interleaved,
                    heads > 0 ? heads : 1, tokens);
  // (a block walks tiles here, and each begins with two barriers: up to 16
  // tokens while that leaves the blocks a tile each; 16,896 tokens of 32 heads
  // of 80 67 us, by the forward's rule 83, 32,400 of 16 of 64 in fp32 91 and
  // 89, longer ones alike)
  while (p.tile < 16 && tokens >= int64_t(p.tile) * kBackwardBlocks) p.tile *= 2;
  A.units = p.units;
  int q_blocks, k_blocks;
  backward_blocks(tokens, p, q_heads, k_heads, &q_blocks, &k_blocks);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (q_blocks + k_blocks > 0) {
    LaunchScope scope("norm_rotate_backward", s);
    ROTATE_TYPE(launch_backward, A, p, q_blocks, k_blocks, s)
    st = check_launch("norm_rotate_backward");
    if (st) return st;
  }
  if (!q_weight && !k_weight) return BEVPOOL_OK;
  // (no tokens: the sums of nothing, zeros)
  void *wq = q_weight ? dq_weight : nullptr, *wk = k_weight ? dk_weight : nullptr;
  LaunchScope scope("norm_rotate_weight_sum", s);
  const float *pk = A.k.partial;
  if (dtype == BEVPOOL_F32)
    hipLaunchKernelGGL((weight_sum_kernel<float>), dim3(2 * dim), dim3(64), 0, s, parts,
                       static_cast<float *>(wq), pk, static_cast<float *>(wk), q_blocks, k_blocks,
                       dim);
  else if (dtype == BEVPOOL_F16)
    hipLaunchKernelGGL((weight_sum_kernel<_Float16>), dim3(2 * dim), dim3(64), 0, s, parts,
                       static_cast<_Float16 *>(wq), pk, static_cast<_Float16 *>(wk), q_blocks,
                       k_blocks, dim);
  else
    hipLaunchKernelGGL((weight_sum_kernel<__bf16>), dim3(2 * dim), dim3(64), 0, s, parts,
                       static_cast<__bf16 *>(wq), pk, static_cast<__bf16 *>(wk), q_blocks,
                       k_blocks, dim);
  return check_launch("norm_rotate_weight_sum");
}

}  // extern "C"

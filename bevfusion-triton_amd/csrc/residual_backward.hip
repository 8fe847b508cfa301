// residual_backward.hip -- gradients of residual.hip's norms, gate and scale
// (gfx950).  With D the gradient of x', H that of h, r = 1 / sqrt(mean(x'^2) +
// eps), r_u alike of u (1 without update_weight), c = scale gate
// update_weight:
//
//   G  = D + r (H weight - x' r^2 mean(H weight x'))
//   dx = G,  dweight = sum over rows of H x' r
//   du = r_u (G c - n mean(G c n))         (without update_weight: G c)
//   dgate = G scale update_weight n        (summed over the rows that share it)
//   Q  = sum over rows of G gate n:  dupdate_weight = scale Q,
//                                    dscale = update_weight Q
// So one sum over rows serves three gradients, and with a gate that rows
// share, its parts (without the gate) serve dgate too.
//
// Bound by memory: x, u, D and H (and a gate of each value) read once, dx and
// du (and dgate) written once.  x' and n are formed again from x and u.  16,896
// rows of 1,280 in bf16 56 us (4.6 TB/s) and 9 for the sums of six rows of gate;
// from checkpoints, with an fp32 stream, 71 us (4.3 TB/s) and 5.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "bevpool.h"
#include "host_calls.h"
#include "residual.h"

namespace residual {

using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

int check(Args &A, int dtype, int x_dtype, int64_t rows, int width, int64_t gate_rows, float eps);

// The groups' sums of a block, added in the groups' order, to `to`.
template <int kLanes, int kChunks, bool kWhole>
__device__ __forceinline__ void flush(float (&v)[kChunks][8], float *to,
                                      const Place<kLanes, kChunks, kWhole> &at, float *lds) {
  constexpr int kGroups = threads_of(kLanes) / kLanes;
  const int width = at.width;
  if constexpr (kGroups == 1) {
    store_row<float>(to, 0, v, at);
  } else {
    __syncthreads();  // what was there has been read
    store_row<float>(lds, at.group * width, v, at);
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += threads_of(kLanes)) {
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) s += lds[g * width + c];
      to[c] = s;
    }
  }
}

// What a row's lanes read of it; x and update as they were or as checkpoints.
template <typename T, typename X, int kChunks>
struct Operands {
  Raw<X, kChunks> x;
  Raw<T, kChunks> update;
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void load(const Args &A, int64_t row,
                                       const Place<kLanes, kChunks, kWhole> &at) {
    x.load(A.x, row * A.x_row, at);
    update.load(A.update, row * A.update_row, at);
  }
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void get(float (&u)[kChunks][8], float (&v)[kChunks][8],
                                      const Place<kLanes, kChunks, kWhole> &) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        u[j][i] = update.get(j, i);
        v[j][i] = x.get(j, i);
      }
  }
};
template <typename T, typename X, int kChunks>
struct KeptOperands {
  Packed<X, kChunks> x;
  Packed<T, kChunks> update;
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void load(const Args &A, int64_t row,
                                       const Place<kLanes, kChunks, kWhole> &at) {
    const int64_t offset = row * rows::checkpoint_pitch(at.width);
    x.load(A.x_kept + offset, at);
    update.load(A.update_kept + offset, at);
  }
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void get(float (&u)[kChunks][8], float (&v)[kChunks][8],
                                      const Place<kLanes, kChunks, kWhole> &at) const {
    update.get(u, at);
    x.get(v, at);
  }
};
template <typename Of, typename T, typename X, int kChunks>
struct Inputs {
  Of of;
  Raw<X, kChunks> dsum;
  Raw<T, kChunks> dnormed, gate;
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void load(const Args &A, int64_t row, bool own_gate,
                                       const Place<kLanes, kChunks, kWhole> &at) {
    of.load(A, row, at);
    dsum.load(A.dsum, row * A.dsum_row, at);
    dnormed.load(A.dnormed, row * A.dnormed_row, at);
    if (own_gate) gate.load(A.gate, row * A.gate_row, at);
  }
};

// A block walks items, each an equal part of the rows that share a row of
// gate (without such a gate: of all), and leaves each item's sums.  Its groups
// of lanes take rows, the next one's loads on their way while one is worked on.
template <typename T, typename X, int kLanes, int kChunks, bool kWhole, bool kKept>
__global__ __launch_bounds__(threads_of(kLanes),
                             backward_waves(kLanes, kChunks, kKept, sizeof(X) == 4))
void residual_backward_kernel(Args A) {
  constexpr int kGroups = threads_of(kLanes) / kLanes;
  typedef std::conditional_t<kKept, KeptOperands<T, X, kChunks>, Operands<T, X, kChunks>> Of;
  extern __shared__ float lds[];
  __shared__ float shared[6][2 * (threads_of(kLanes) / 64)];
  const Place<kLanes, kChunks, kWhole> at(A.width);
  const int64_t width = A.width;
  const bool own_gate = A.has_gate && A.gate_each == 1;
  const int64_t part_rows = (A.has_gate && !own_gate ? A.gate_each : A.rows);
  const int64_t share = (part_rows + A.parts_each - 1) / A.parts_each;
  // scale times the update's weight, and the norm's weight
  float c[kChunks][8], dweight[kChunks][8] = {};
  Raw<T, kChunks> weight;
  {
    Raw<T, kChunks> w;
    if (A.update_weight) w.load(A.update_weight, 0, at);
    if (A.scale) weight.load(A.scale, 0, at);
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        c[j][i] = (A.update_weight ? w.get(j, i) : 1.f) * (A.scale ? weight.get(j, i) : 1.f);
  }
  if (A.weight) weight.load(A.weight, 0, at);
  int turn = 0;
  for (int64_t item = blockIdx.x; item < A.items; item += gridDim.x) {
    const int64_t owner = item / A.parts_each, part = item % A.parts_each;
    const int64_t first = owner * part_rows;
    const int64_t begin = first + part * share;
    const int64_t end = min(begin + share, first + part_rows);
    float q[kChunks][8] = {};
    Inputs<Of, T, X, kChunks> in, next;
    int64_t row = begin + at.group;
    if (A.has_gate && !own_gate) next.gate.load(A.gate, owner * A.gate_row, at);
    if (row < end) next.load(A, row, own_gate, at);
    for (; row < end; row += kGroups, turn = 3 - turn) {
      in = next;
      next.load(A, row + kGroups < end ? row + kGroups : row, own_gate, at);
      float n[kChunks][8], x[kChunks][8];
      in.of.get(n, x, at);
      float r_u = 1.f;
      if (A.update_weight) {
        float s[1] = {own_sum(at, [&](int j, int i) { return n[j][i] * n[j][i]; })};
        row_sums<kLanes>(s, shared[turn]);
        r_u = 1.0f / sqrtf(s[0] * A.inv_width + A.eps);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) n[j][i] *= r_u;
      }
      float g[kChunks][8];
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) g[j][i] = A.has_dsum ? in.dsum.get(j, i) : 0.f;
      if (A.weight) {
        if (A.has_update) {
#pragma unroll
          for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float v = n[j][i] * c[j][i];
              x[j][i] += A.has_gate ? v * in.gate.get(j, i) : v;
            }
        }
        float s[2] = {own_sum(at, [&](int j, int i) { return x[j][i] * x[j][i]; }),
                      own_sum(at, [&](int j, int i) {
                        return in.dnormed.get(j, i) * weight.get(j, i) * x[j][i];
                      })};
        row_sums<kLanes>(s, shared[turn + 1]);
        const float r = 1.0f / sqrtf(s[0] * A.inv_width + A.eps);
        const float back = s[1] * A.inv_width * r * r;
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float h = in.dnormed.get(j, i);
            dweight[j][i] += h * (x[j][i] * r);
            g[j][i] += r * (h * weight.get(j, i) - x[j][i] * back);
          }
      }
      if (!A.has_update) {
        store_row<X>(A.dx, row * width, g, at);
        continue;
      }
      // dn: the gradient of n, with gate and weights
      float dn[kChunks][8];
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float t = g[j][i] * n[j][i], gate = A.has_gate ? in.gate.get(j, i) : 1.f;
          q[j][i] += own_gate ? t * gate : t;
          dn[j][i] = g[j][i] * (c[j][i] * gate);
        }
      float back = 0.f;
      if (A.update_weight) {
        float s[1] = {own_sum(at, [&](int j, int i) { return dn[j][i] * n[j][i]; })};
        row_sums<kLanes>(s, shared[turn + 2]);
        back = s[0] * A.inv_width;
      }
      store_row<X>(A.dx, row * width, g, at);
      if (own_gate) {
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) g[j][i] *= n[j][i] * c[j][i];
        store_row<T>(A.dgate, row * width, g, at);
      }
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) dn[j][i] = r_u * (dn[j][i] - n[j][i] * back);
      store_row<T>(A.dupdate, row * width, dn, at);
    }
    if (A.parts) flush(q, A.parts + item * width, at, lds);
  }
  if (A.weight_parts)
    flush(dweight, A.weight_parts + int64_t(blockIdx.x) * width, at, lds);
}

constexpr int kSumThreads = 1024, kSumColumns = 32, kSlices = kSumThreads / kSumColumns;

// The slices' sums, added in the slices' order; the first slice has them.
__device__ __forceinline__ float slices_sum(float v, float *lds) {
  __syncthreads();  // what was there has been read
  lds[threadIdx.x] = v;
  __syncthreads();
  v = 0.f;
  if (threadIdx.x < kSumColumns)
#pragma unroll
    for (int i = 0; i < kSlices; ++i) v += lds[i * kSumColumns + threadIdx.x];
  return v;
}

// Sum of rows first, first + step, .. below n of a column.
__device__ __forceinline__ float strided_sum(const float *from, int64_t first, int64_t n, int step,
                                             int width) {
  float s = 0.f;
#pragma unroll 8
  for (int64_t i = first; i < n; i += step) s += from[i * width];
  return s;
}

// The gradients that are sums over rows, from the items' and the blocks' sums:
// grid.y 0 those of the update's weight and of the scale, 1 that of the norm's
// weight, from 2 on that of a gate that rows share, by its rows, or, where these
// have so few parts that a slice sums them, by kSlices of them (us of all sums of
// 16,896 rows of 1,280, by events: 40 rows of gate 10, by a block each 22; 1,000 11
// and 119).
constexpr int kFewParts = kSlices;
template <typename T>
__global__ __launch_bounds__(kSumThreads) void sums_kernel(Args A, int64_t weight_blocks, T *dgate,
                                                           T *dupdate_weight, T *dscale,
                                                           T *dweight) {
  __shared__ float lds[kSumThreads];
  const int slice = int(threadIdx.x) / kSumColumns;
  const int c = blockIdx.x * kSumColumns + int(threadIdx.x) % kSumColumns;
  const bool on = c < A.width, writes = slice == 0 && on;
  if (blockIdx.y == 1) {
    if (!dweight) return;
    float s = on ? strided_sum(A.weight_parts + c, slice, weight_blocks, kSlices, A.width) : 0.f;
    s = slices_sum(s, lds);
    if (writes) dweight[c] = T(s);
    return;
  }
  if (blockIdx.y == 0 && !dupdate_weight && !dscale) return;
  float w = 1.f, scale = 1.f;
  if (on && A.update_weight) w = float(static_cast<const T *>(A.update_weight)[c]);
  if (on && A.scale) scale = float(static_cast<const T *>(A.scale)[c]);
  const float *parts = A.parts + c;
  const bool shared = A.has_gate && A.gate_each > 1;  // (the items' sums are without the gate)
  const int64_t owners = A.items / A.parts_each;
  if (blockIdx.y == 0) {
    float s = 0.f;
    if (on && shared && owners > 1) {
      const T *gate = static_cast<const T *>(A.gate) + c;
      // (item, its owner and its place among the owner's parts)
      const int each = int(A.parts_each), owners_on = kSlices / each, places_on = kSlices % each;
      int64_t owner = slice / each;
      int place = slice % each;
#pragma unroll 8
      for (int64_t i = slice; i < A.items; i += kSlices) {
        s += parts[i * A.width] * float(gate[owner * A.gate_row]);
        owner += owners_on;
        place += places_on;
        if (place >= each) {
          place -= each;
          ++owner;
        }
      }
    } else if (on) {
      s = strided_sum(parts, slice, A.items, kSlices, A.width);
      if (shared) s *= float(static_cast<const T *>(A.gate)[c]);
    }
    s = slices_sum(s, lds);
    if (writes && dupdate_weight) dupdate_weight[c] = T(s * scale);
    if (writes && dscale) dscale[c] = T(s * w);
    return;
  }
  const int64_t first = blockIdx.y - 2, step = gridDim.y - 2;
  if (A.parts_each <= kFewParts) {
    if (on)
      for (int64_t owner = first * kSlices + slice; owner < owners; owner += step * kSlices) {
        const int64_t at = owner * A.parts_each;
        const float s = strided_sum(parts, at, at + A.parts_each, 1, A.width);
        dgate[owner * A.width + c] = T(s * w * scale);
      }
    return;
  }
  for (int64_t owner = first; owner < owners; owner += step) {
    const int64_t at = owner * A.parts_each;
    float s = on ? strided_sum(parts, at + slice, at + A.parts_each, kSlices, A.width) : 0.f;
    s = slices_sum(s, lds);
    if (writes) dgate[owner * A.width + c] = T(s * w * scale);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

struct Split {
  int64_t items, parts_each, blocks;
};
Split split_for(int64_t rows, int width, int64_t gate_rows, bool kept, bool wide) {
  int64_t most_blocks = 0, at_once = 0;
#define RESIDUAL_BLOCKS(kLanes, kChunks, kWhole, ...)                                   \
  {                                                                             \
    most_blocks = blocks_for(kLanes, backward_waves(kLanes, kChunks, kept, wide));    \
    at_once = threads_of(kLanes) / kLanes;                                      \
  }
  RESIDUAL_LAYOUT(RESIDUAL_BLOCKS, width)
#undef RESIDUAL_BLOCKS
  const bool shared = gate_rows > 0 && gate_rows < rows;
  const int64_t owners = shared ? gate_rows : 1, each = rows / owners;
  const int64_t most = (each + at_once - 1) / at_once;
  // As many parts of each owner's rows as give every block an item, or one more,
  // whichever leaves a block fewer rows at most: 16,896 rows of 1,280 of six owners,
  // 1,278 items on 1,280 blocks in place of 1,284, four of them with two; 16,800 of
  // 600 owners 56.7 us for 59.5.
  auto load = [&](int64_t parts) {
    const int64_t items = owners * parts, blocks = items < most_blocks ? items : most_blocks;
    return (items + blocks - 1) / blocks * ((each + parts - 1) / parts);
  };
  int64_t parts = most_blocks / owners;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  if (parts < most && load(parts + 1) < load(parts)) ++parts;
  Split s;
  s.parts_each = parts;
  s.items = owners * parts;
  s.blocks = s.items < most_blocks ? s.items : most_blocks;
  return s;
}

template <typename T, typename X, int kLanes, int kChunks, bool kWhole>
void launch(const Args &A, int64_t blocks, bool kept, hipStream_t s) {
  constexpr int kGroups = threads_of(kLanes) / kLanes;
  const size_t lds = kGroups == 1 ? 0 : sizeof(float) * kGroups * size_t(A.width);
  if (kept)
    hipLaunchKernelGGL((residual_backward_kernel<T, X, kLanes, kChunks, kWhole, true>),
                       dim3(unsigned(blocks)), dim3(threads_of(kLanes)), lds, s, A);
  else
    hipLaunchKernelGGL((residual_backward_kernel<T, X, kLanes, kChunks, kWhole, false>),
                       dim3(unsigned(blocks)), dim3(threads_of(kLanes)), lds, s, A);
}

template <typename T, typename X>
void launch_width(const Args &A, int64_t blocks, bool kept, hipStream_t s) {
#define RESIDUAL_LAUNCH(kLanes, kChunks, kWhole, ...) \
  launch<T, X, kLanes, kChunks, kWhole>(A, blocks, kept, s);
  RESIDUAL_LAYOUT(RESIDUAL_LAUNCH, A.width)
#undef RESIDUAL_LAUNCH
}

template <typename T>
void launch_sums(const Args &A, int64_t blocks, void *dgate, void *dupdate_weight, void *dscale,
                 void *dweight, hipStream_t s) {
  const int64_t owners = A.has_gate && A.gate_each > 1 ? A.items / A.parts_each : 0;
  if (!owners && !dupdate_weight && !dscale && !dweight) return;
  const int64_t sums = A.parts_each <= kFewParts ? (owners + kSlices - 1) / kSlices : owners;
  const dim3 grid((A.width + kSumColumns - 1) / kSumColumns,
                  unsigned(2 + (sums < 4096 ? sums : 4096)));
  hipLaunchKernelGGL((sums_kernel<T>), grid, dim3(kSumThreads), 0, s, A, blocks,
                     static_cast<T *>(dgate), static_cast<T *>(dupdate_weight),
                     static_cast<T *>(dscale), static_cast<T *>(dweight));
}

}  // namespace residual

extern "C" {

size_t bevpool_residual_norm_backward_scratch_bytes(int64_t rows, int32_t width,
                                                    int64_t gate_rows, int32_t x_dtype,
                                                    int32_t kept) {
  using namespace residual;
  if (rows < 1 || width < 1 || width > kMaxWidth || gate_rows < 0) return 0;
  const Split s = split_for(rows, width, gate_rows, kept != 0, x_dtype == BEVPOOL_F32);
  return size_t(s.items + s.blocks) * size_t(width) * sizeof(float);
}

int bevpool_residual_norm_backward(
    const void *x, int64_t x_row, int32_t x_dtype, const void *update, int64_t update_row,
    const void *update_weight, const void *scale, const void *gate, int64_t gate_row,
    int64_t gate_rows, const void *weight, int32_t kept, const void *dsum, int64_t dsum_row,
    const void *dnormed, int64_t dnormed_row, int32_t dtype, int64_t rows, int32_t width, float eps,
    void *dx, void *dupdate, void *dgate, void *dupdate_weight, void *dscale, void *dweight,
    void *scratch, size_t scratch_bytes, void *stream) {
  using namespace residual;
  bevpool_host::clear_error();
  Args A = {};
  const int st = check(A, dtype, x_dtype, rows, width, gate ? gate_rows : 0, eps);
  if (st) return st;
  if ((update_weight && !dupdate_weight) || (scale && !dscale) || (weight && !dweight))
    return fail(BEVPOOL_EINVAL, "a weight without the place of its gradient");
  if ((dupdate_weight && !update_weight) || (dscale && !scale) || (dweight && !weight))
    return fail(BEVPOOL_EINVAL, "a gradient of a weight that is not there");
  if (rows > 0) {
    if (!update && !weight) return fail(BEVPOOL_EINVAL, "neither an update nor a norm");
    if (gate && gate_rows < 1) return fail(BEVPOOL_EINVAL, "a gate without rows");
    if (!update && (update_weight || scale || gate))
      return fail(BEVPOOL_EINVAL, "update_weight, scale and gate are of an update");
    if (!dx || (update && !dupdate) || (gate && !dgate) || (weight && (!x || !dnormed)))
      return fail(BEVPOOL_EINVAL, "null rows");
    if (!scratch ||
        scratch_bytes < bevpool_residual_norm_backward_scratch_bytes(
                            rows, width, gate ? gate_rows : 0, x_dtype, kept))
      return fail(BEVPOOL_ESPACE, "residual_norm backward scratch too small");
  }
  A.x = x;
  A.x_row = x_row;
  A.update = update;
  A.update_row = update_row;
  if (kept) {
    A.x_kept = static_cast<uint8_t *>(const_cast<void *>(x));
    A.update_kept = static_cast<uint8_t *>(const_cast<void *>(update));
  }
  A.update_weight = update_weight;
  A.scale = scale;
  A.gate = gate;
  A.gate_row = gate_row;
  A.weight = weight;
  A.dsum = dsum;
  A.dsum_row = dsum_row;
  A.dnormed = dnormed;
  A.dnormed_row = dnormed_row;
  A.dx = dx;
  A.dupdate = dupdate;
  A.dgate = dgate;
  A.has_update = update != nullptr;
  A.has_gate = gate != nullptr;
  A.has_dsum = dsum != nullptr;
  // What is read and not used: rows that are there and no shorter.  (dx is read
  // by the lanes that write it, before they do.)
  if (!dsum) {
    A.dsum = dx;
    A.dsum_row = width;
  }
  if (!weight) {
    A.x = A.dsum;
    A.x_row = A.dsum_row;
    A.x_kept = A.update_kept;
    A.dnormed = A.dsum;
    A.dnormed_row = 0;
  }
  if (!update) {
    A.update = A.dnormed;
    A.update_row = 0;
    A.update_kept = A.x_kept;
  }
  Split split = {0, 1, 0};
  if (rows > 0) {
    split = split_for(rows, width, gate ? gate_rows : 0, kept != 0, x_dtype == BEVPOOL_F32);
    A.weight_parts = weight ? static_cast<float *>(scratch) : nullptr;
    const bool shared = gate && gate_rows < rows;
    if (update && (update_weight || scale || shared))
      A.parts = static_cast<float *>(scratch) + split.blocks * width;
  }
  A.items = split.items;
  A.parts_each = split.parts_each;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    LaunchScope scope("residual_norm_backward", s);
    if (dtype == BEVPOOL_F32)
      launch_width<float, float>(A, split.blocks, kept != 0, s);
    else if (dtype == BEVPOOL_F16)
      x_dtype == BEVPOOL_F32 ? launch_width<_Float16, float>(A, split.blocks, kept != 0, s)
                             : launch_width<_Float16, _Float16>(A, split.blocks, kept != 0, s);
    else
      x_dtype == BEVPOOL_F32 ? launch_width<__bf16, float>(A, split.blocks, kept != 0, s)
                             : launch_width<__bf16, __bf16>(A, split.blocks, kept != 0, s);
    const int e = check_launch("residual_norm_backward");
    if (e) return e;
  }
  // (no rows: the sums of nothing, zeros)
  LaunchScope scope("residual_norm_sums", s);
  if (dtype == BEVPOOL_F32)
    launch_sums<float>(A, split.blocks, dgate, dupdate_weight, dscale, dweight, s);
  else if (dtype == BEVPOOL_F16)
    launch_sums<_Float16>(A, split.blocks, dgate, dupdate_weight, dscale, dweight, s);
  else
    launch_sums<__bf16>(A, split.blocks, dgate, dupdate_weight, dscale, dweight, s);
  return check_launch("residual_norm_sums");
}

}  // extern "C"

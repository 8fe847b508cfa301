// residual.hip -- the norms on both sides of a residual, with the residual's
// gate and scale, in one pass (gfx950): the forward; residual_backward.hip has
// the gradients.
//
//   n  = u / sqrt(mean(u^2) + eps)     (update_weight given; else n = u)
//   x' = x + scale gate update_weight n
//   h  = x' / sqrt(mean(x'^2) + eps) weight
// x is the residual stream, u a block's output, h the next block's input.
//
// Bound by memory: x and u (and a gate of each value) read once, x' and h
// written once.  A row stays in the registers of its lanes from the first sum
// to the last store.  16,896 rows of 1,280 in bf16 35 us (4.9 TB/s of what has
// to move; a large copy reaches 5.1), with an fp32 stream and the checkpoints
// 62 us (4.9 TB/s); 30,011 rows of 1,283 in fp16 with a gate of each value, rows
// that begin at any address, 89 us (4.3 TB/s).
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bevpool.h"
#include "host_calls.h"
#include "residual.h"

namespace residual {

using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

// What a row's lanes read of it.
template <typename T, typename X, int kChunks>
struct Inputs {
  Raw<X, kChunks> x;
  Raw<T, kChunks> update, gate;
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void load(const Args &A, int64_t row,
                                       const Place<kLanes, kChunks, kWhole> &at) {
    x.load(A.x, row * A.x_row, at);
    update.load(A.update, row * A.update_row, at);
    const int64_t owner = A.gate_each == 1        ? row
                          : A.rows < (1LL << 32) ? unsigned(row) / unsigned(A.gate_each)
                                                 : row / A.gate_each;
    gate.load(A.gate, owner * A.gate_row, at);
  }
  __device__ __forceinline__ void settle() {
    x.settle();
    update.settle();
    gate.settle();
  }
};

// 8-bit checkpoint of a row: of chunks in their place as they are in registers,
// of the last one from memory, for it begins earlier there.
template <typename T, int kLanes, int kChunks, bool kWhole>
__device__ __forceinline__ void keep(uint8_t *kept, const Raw<T, kChunks> &raw, const void *base,
                                     int64_t offset, const Place<kLanes, kChunks, kWhole> &at) {
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = raw.get(j, i);
    if (at.skip(j) > 0)
      rows::load(v, static_cast<const T *>(base) + offset + at.chunk(j) * 8, at.left(j));
    rows::store_packed(kept, at.chunk(j), rows::blocks_of(at.width), v);
  }
}

// A group of lanes takes rows, the next one's loads on their way while one is
// worked on; weights stay in registers.
template <typename T, typename X, int kLanes, int kChunks, bool kWhole>
__global__ __launch_bounds__(threads_of(kLanes), forward_waves(kChunks)) void residual_kernel(
    Args A) {
  constexpr int kGroups = threads_of(kLanes) / kLanes;
  __shared__ float shared[4][threads_of(kLanes) / 64];
  const Place<kLanes, kChunks, kWhole> at(A.width);
  const int64_t width = A.width, pitch = rows::checkpoint_pitch(width);
  // scale times the update's weight, and the norm's weight
  float c[kChunks][8];
  Raw<T, kChunks> w, weight;
  if (A.update_weight) w.load(A.update_weight, 0, at);
  if (A.scale) weight.load(A.scale, 0, at);
#pragma unroll
  for (int j = 0; j < kChunks; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[j][i] = (A.update_weight ? w.get(j, i) : 1.f) * (A.scale ? weight.get(j, i) : 1.f);
  if (A.weight) weight.load(A.weight, 0, at);
  const int64_t step = int64_t(gridDim.x) * kGroups;
  int64_t row = int64_t(blockIdx.x) * kGroups + at.group;
  if (row >= A.rows) return;  // (all of a block whose rows pass barriers)
  Inputs<T, X, kChunks> in, next;
  in.load(A, row, at);
  for (int turn = 0; row < A.rows; row += step, turn ^= 2) {
    next.load(A, row + step < A.rows ? row + step : row, at);
    float x[kChunks][8];
    if (A.has_update) {
      float r = 1.f;
      if (A.update_weight) {
        float s[1] = {own_sum(at, [&](int j, int i) {
          const float u = in.update.get(j, i);
          return u * u;
        })};
        row_sums<kLanes>(s, shared[turn]);
        r = 1.0f / sqrtf(s[0] * A.inv_width + A.eps);
      }
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v = in.update.get(j, i) * r * c[j][i];
          if (A.has_gate) v *= in.gate.get(j, i);
          x[j][i] = in.x.get(j, i) + v;
        }
    } else {
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = in.x.get(j, i);
    }
    float r = 0.f;
    if (A.weight) {
      float s[1] = {own_sum(at, [&](int j, int i) { return x[j][i] * x[j][i]; })};
      row_sums<kLanes>(s, shared[turn + 1]);
      r = 1.0f / sqrtf(s[0] * A.inv_width + A.eps);
    }
    next.settle();  // (before the stores, for which it would wait behind them)
    if (A.keeps) {
      if (A.x_kept) keep<X>(A.x_kept + row * pitch, in.x, A.x, row * A.x_row, at);
      if (A.update_kept)
        keep<T>(A.update_kept + row * pitch, in.update, A.update, row * A.update_row, at);
    }
    if (A.has_update) store_row<X>(A.sum, row * width, x, at);
    if (A.weight) {
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] *= r * weight.get(j, i);
      store_row<T>(A.normed, row * width, x, at);
    }
    in = next;
  }
}

template <typename T, typename X, int kLanes, int kChunks, bool kWhole>
void launch(const Args &A, hipStream_t s) {
  constexpr int kGroups = threads_of(kLanes) / kLanes;
  constexpr int kBlocks = blocks_for(kLanes, forward_waves(kChunks));
  const int64_t blocks = (A.rows + kGroups - 1) / kGroups;
  hipLaunchKernelGGL((residual_kernel<T, X, kLanes, kChunks, kWhole>),
                     dim3(unsigned(blocks < kBlocks ? blocks : kBlocks)),
                     dim3(threads_of(kLanes)), 0, s, A);
}

template <typename T, typename X>
void launch_width(const Args &A, hipStream_t s) {
#define RESIDUAL_LAUNCH(kLanes, kChunks, kWhole, ...) launch<T, X, kLanes, kChunks, kWhole>(A, s);
  RESIDUAL_LAYOUT(RESIDUAL_LAUNCH, A.width)
#undef RESIDUAL_LAUNCH
}

// Sizes and operands that both directions check.
int check(Args &A, int dtype, int x_dtype, int64_t rows, int width, int64_t gate_rows, float eps) {
  if (dtype < BEVPOOL_F32 || dtype > BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d", dtype);
  if (x_dtype != dtype && x_dtype != BEVPOOL_F32)
    return fail(BEVPOOL_EINVAL, "x of dtype code %d: the other operands' or fp32", x_dtype);
  if (width < 1 || width > kMaxWidth)
    return fail(BEVPOOL_EINVAL, "width %d: must be in [1, %d]", width, kMaxWidth);
  if (rows < 0 || rows > (int64_t(1) << 40)) return fail(BEVPOOL_EINVAL, "bad number of rows");
  if (!(eps >= 0.f)) return fail(BEVPOOL_EINVAL, "eps must not be negative");
  if (gate_rows < 0 || (gate_rows > 0 && rows % gate_rows))
    return fail(BEVPOOL_EINVAL, "%lld rows of gate do not divide %lld rows",
                static_cast<long long>(gate_rows), static_cast<long long>(rows));
  A.rows = rows;
  A.width = width;
  A.eps = eps;
  A.inv_width = 1.0f / float(width);
  A.gate_each = gate_rows > 0 && rows > 0 ? rows / gate_rows : 1;
  return BEVPOOL_OK;
}

}  // namespace residual

extern "C" {

int64_t bevpool_checkpoint_pitch(int32_t width) {
  return width < 1 ? 0 : rows::checkpoint_pitch(width);
}

int bevpool_residual_norm_forward(const void *x, int64_t x_row, int32_t x_dtype,
                                  const void *update, int64_t update_row,
                                  const void *update_weight, const void *scale, const void *gate,
                                  int64_t gate_row, int64_t gate_rows, const void *weight,
                                  int32_t dtype, int64_t rows, int32_t width, float eps, void *sum,
                                  void *normed, void *x_kept, void *update_kept, void *stream) {
  using namespace residual;
  bevpool_host::clear_error();
  Args A = {};
  const int st = check(A, dtype, x_dtype, rows, width, gate ? gate_rows : 0, eps);
  if (st) return st;
  if (rows == 0) return BEVPOOL_OK;
  if (gate && gate_rows < 1) return fail(BEVPOOL_EINVAL, "a gate without rows");
  if (!update && (update_weight || scale || gate || update_kept))
    return fail(BEVPOOL_EINVAL, "update_weight, scale and gate are of an update");
  if (!update && !weight) return fail(BEVPOOL_EINVAL, "neither an update nor a norm");
  if (!x || (update && !sum) || (weight && !normed)) return fail(BEVPOOL_EINVAL, "null rows");
  A.x = x;
  A.x_row = x_row;
  A.update = update;
  A.update_row = update_row;
  A.update_weight = update_weight;
  A.scale = scale;
  A.gate = gate;
  A.gate_row = gate_row;
  A.weight = weight;
  A.sum = sum;
  A.normed = normed;
  A.x_kept = static_cast<uint8_t *>(x_kept);
  A.update_kept = static_cast<uint8_t *>(update_kept);
  A.keeps = x_kept || update_kept;
  A.has_update = update != nullptr;
  A.has_gate = gate != nullptr;
  // (read and not used: x's first row, which is no shorter than one of theirs)
  if (!update) {
    A.update = x;
    A.update_row = 0;
  }
  if (!gate) {
    A.gate = x;
    A.gate_row = 0;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  LaunchScope scope("residual_norm", s);
  if (dtype == BEVPOOL_F32)
    launch_width<float, float>(A, s);
  else if (dtype == BEVPOOL_F16)
    x_dtype == BEVPOOL_F32 ? launch_width<_Float16, float>(A, s)
                           : launch_width<_Float16, _Float16>(A, s);
  else
    x_dtype == BEVPOOL_F32 ? launch_width<__bf16, float>(A, s)
                           : launch_width<__bf16, __bf16>(A, s);
  return check_launch("residual_norm");
}

}  // extern "C"

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
// to the last store.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bevpool.h"
#include "host_calls.h"
#include "residual.h"

namespace residual {

using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

template <typename T, typename X, int kLanes, int kChunks>
__global__ __launch_bounds__(threads_of(kLanes)) void residual_kernel(Args A) {
  constexpr int kGroups = threads_of(kLanes) / kLanes;
  __shared__ float shared[4][threads_of(kLanes) / 64];
  const Place<kLanes, kChunks> at;
  const int width = A.width;
  const int64_t blocks = rows::blocks_of(width);
  int turn = 0;
  for (int64_t row = int64_t(blockIdx.x) * kGroups + at.group; row < A.rows;
       row += int64_t(gridDim.x) * kGroups, turn ^= 2) {
    float x[kChunks][8], u[kChunks][8], w[kChunks][8];
    load_row<X>(x, A.x, row * A.x_row, width, at);
    if (A.update) {
      load_row<T>(u, A.update, row * A.update_row, width, at);
      if (A.update_kept) {
        uint8_t *kept = A.update_kept + row * rows::checkpoint_pitch(width);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) rows::store_packed(kept, at.chunk(j), blocks, u[j]);
      }
    }
    if (A.x_kept) {
      uint8_t *kept = A.x_kept + row * rows::checkpoint_pitch(width);
#pragma unroll
      for (int j = 0; j < kChunks; ++j) rows::store_packed(kept, at.chunk(j), blocks, x[j]);
    }
    if (A.update) {
      if (A.update_weight) {
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) s[0] += u[j][i] * u[j][i];
        row_sums<kLanes>(s, shared[turn]);
        const float r = 1.0f / sqrtf(s[0] * A.inv_width + A.eps);
        load_row<T>(w, A.update_weight, 0, width, at);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) u[j][i] *= r * w[j][i];
      }
      if (A.scale) {
        load_row<T>(w, A.scale, 0, width, at);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) u[j][i] *= w[j][i];
      }
      if (A.gate) {
        const int64_t owner = A.gate_each == 1        ? row
                              : A.rows < (1LL << 32) ? unsigned(row) / unsigned(A.gate_each)
                                                     : row / A.gate_each;
        load_row<T>(w, A.gate, owner * A.gate_row, width, at);
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) u[j][i] *= w[j][i];
      }
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] += u[j][i];
      store_row<X>(A.sum, row * width, width, x, at);
    }
    if (A.weight) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[0] += x[j][i] * x[j][i];
      row_sums<kLanes>(s, shared[turn + 1]);
      const float r = 1.0f / sqrtf(s[0] * A.inv_width + A.eps);
      load_row<T>(w, A.weight, 0, width, at);
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] *= r * w[j][i];
      store_row<T>(A.normed, row * width, width, x, at);
    }
  }
}

// Blocks: as many as the card holds at once, or as there are rows.
constexpr int kForwardBlocks = 2048;

template <typename T, typename X, int kLanes, int kChunks>
void launch(const Args &A, hipStream_t s) {
  constexpr int kGroups = threads_of(kLanes) / kLanes;
  const int64_t blocks = (A.rows + kGroups - 1) / kGroups;
  hipLaunchKernelGGL((residual_kernel<T, X, kLanes, kChunks>),
                     dim3(unsigned(blocks < kForwardBlocks ? blocks : kForwardBlocks)),
                     dim3(threads_of(kLanes)), 0, s, A);
}

template <typename T, typename X>
void launch_width(const Args &A, hipStream_t s) {
#define RESIDUAL_LAUNCH(kLanes, kChunks, ...) launch<T, X, kLanes, kChunks>(A, s);
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

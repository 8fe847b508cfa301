// What the forward and the backward kernels of residual.hip share.
#pragma once

#include "rows.h"

namespace residual {

constexpr int kMaxWidth = 8192;

struct Args {
  // inputs (null: not there)
  const void *x, *update, *gate, *update_weight, *scale, *weight;
  int64_t x_row, update_row, gate_row;  // strides in values
  uint8_t *x_kept, *update_kept;        // 8-bit checkpoints
  int64_t rows;
  int64_t gate_each;                    // rows that share a row of gate
  int width;
  float eps, inv_width;
  // forward
  void *sum, *normed;
  // backward
  const void *dsum, *dnormed;
  int64_t dsum_row, dnormed_row;
  void *dx, *dupdate, *dgate;           // dgate: only of a gate with a row for each
  float *weight_parts;                  // [blocks][width]: sums of dnormed n(x')
  float *parts;                         // [items][width]: sums of dx' n (gate)
  int64_t items, parts_each;            // parts_each: items of one row of gate
};

// Lanes that share a row and chunks that each holds: the fewest lanes for
// short rows, so that a wave takes several, and no more than three chunks,
// which leave room for the gradients' values of a row in registers.
#define RESIDUAL_LAYOUT(FN, width, ...)                                         \
  if ((width) <= 128) FN(16, 1, __VA_ARGS__)                                    \
  else if ((width) <= 256) FN(32, 1, __VA_ARGS__)                               \
  else if ((width) <= 512) FN(64, 1, __VA_ARGS__)                               \
  else if ((width) <= 1024) FN(64, 2, __VA_ARGS__)                              \
  else if ((width) <= 1536) FN(64, 3, __VA_ARGS__)                              \
  else if ((width) <= 2048) FN(256, 1, __VA_ARGS__)                             \
  else if ((width) <= 4096) FN(256, 2, __VA_ARGS__)                             \
  else FN(512, 2, __VA_ARGS__)

constexpr int threads_of(int lanes) { return lanes > 256 ? lanes : 256; }
inline int lanes_for(int width) {
  return width <= 128 ? 16 : width <= 256 ? 32 : width <= 1536 ? 64 : width <= 4096 ? 256 : 512;
}
inline int rows_at_once(int width) {
  const int lanes = lanes_for(width);
  return threads_of(lanes) / lanes;
}

// A lane's place: its row of a block's, and what of it is its own.
template <int kLanes, int kChunks>
struct Place {
  int lane, group;
  __device__ __forceinline__ Place() {
    lane = int(threadIdx.x) % kLanes;
    group = int(threadIdx.x) / kLanes;
  }
  __device__ __forceinline__ int chunk(int j) const { return lane + j * kLanes; }
  __device__ __forceinline__ int left(int j, int width) const {
    return width - chunk(j) * rows::kChunk;
  }
};

template <typename T, int kLanes, int kChunks>
__device__ __forceinline__ void load_row(float (&v)[kChunks][rows::kChunk], const void *base,
                                         int64_t offset, int width,
                                         const Place<kLanes, kChunks> &at) {
  const T *row = static_cast<const T *>(base) + offset;
#pragma unroll
  for (int j = 0; j < kChunks; ++j)
    rows::load(v[j], row + at.chunk(j) * rows::kChunk, at.left(j, width));
}
template <typename T, int kLanes, int kChunks>
__device__ __forceinline__ void store_row(void *base, int64_t offset, int width,
                                          const float (&v)[kChunks][rows::kChunk],
                                          const Place<kLanes, kChunks> &at) {
  T *row = static_cast<T *>(base) + offset;
#pragma unroll
  for (int j = 0; j < kChunks; ++j)
    rows::store(row + at.chunk(j) * rows::kChunk, v[j], at.left(j, width));
}

// Sums over a row's lanes, kN at once, in all of them.  Rows of more than a
// wave pass through `shared`, whose slots a caller alternates: a slot is
// written again only behind the barrier of another.
template <int kLanes, int kN>
__device__ __forceinline__ void row_sums(float (&v)[kN], float *shared) {
  if constexpr (kLanes <= 64) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = rows::lanes_sum<kLanes>(v[i]);
  } else {
    constexpr int kWaves = kLanes / 64;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      v[i] = rows::lanes_sum<64>(v[i]);
      if (threadIdx.x % 64 == 0) shared[i * kWaves + threadIdx.x / 64] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v[i] += shared[i * kWaves + w];
    }
  }
}

}  // namespace residual

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

// Lanes that share a row and chunks that each holds: one, so that few registers
// hold a row's values and several rows' loads are on their way at once (chunks
// past 4096 values: two), by whole waves, or parts of one for short rows.
#define RESIDUAL_LAYOUT(FN, width, ...)                                         \
  if ((width) <= 128) FN(16, 1, __VA_ARGS__)                                    \
  else if ((width) <= 256) FN(32, 1, __VA_ARGS__)                               \
  else if ((width) <= 512) FN(64, 1, __VA_ARGS__)                               \
  else if ((width) <= 1024) FN(128, 1, __VA_ARGS__)                             \
  else if ((width) <= 1536) FN(192, 1, __VA_ARGS__)                             \
  else if ((width) <= 2048) FN(256, 1, __VA_ARGS__)                             \
  else if ((width) <= 4096) FN(512, 1, __VA_ARGS__)                             \
  else FN(512, 2, __VA_ARGS__)

// (rows of more than a wave pass barriers: a block of them has one)
constexpr int threads_of(int lanes) { return lanes > 64 ? lanes : 256; }
// Waves of a SIMD that the registers of a kernel leave room for (they are
// compiled to), and the blocks of the whole card: the kernels walk rows by as
// many as are there at once.  More only begin later: backward of 200,000 rows of
// 80 by three blocks a CU, as many as there is room for, 57 us, by four 71; one
// block a row instead, forward of 16,896 rows of 1,280 63 us for 43.
constexpr int forward_waves(int chunks) { return chunks > 1 ? 3 : 4; }
constexpr int backward_waves(int lanes, int chunks, bool kept, bool wide) {
  return chunks > 1 ? 2 : kept || lanes < 64 || wide ? 3 : 4;  // (wide: a stream in fp32)
}
constexpr int blocks_for(int lanes, int waves) {
  const int each = 4 * waves * 64 / threads_of(lanes);
  return 256 * (each > 1 ? each : 1);
}

// A lane's place: its row of a block's, and its chunks.  With kWhole, where the
// width is no whole number of chunks the last one begins earlier, and shares
// its first `skip` values with the one before: both form the same of them, and
// only sums leave them out, so that every access is a whole one (of rows of a
// chunk at least).  Without, its values past the row's end are zeros.
template <int kLanes, int kChunks, bool kWhole = true>
struct Place {
  int lane, group, width;
  __device__ __forceinline__ explicit Place(int width) : width(width) {
    lane = int(threadIdx.x) % kLanes;
    group = int(threadIdx.x) / kLanes;
    if constexpr (kLanes >= 64) group = __builtin_amdgcn_readfirstlane(group);
  }
  __device__ __forceinline__ int chunk(int j) const { return lane + j * kLanes; }
  __device__ __forceinline__ bool on(int j) const { return chunk(j) * rows::kChunk < width; }
  __device__ __forceinline__ int begin(int j) const {
    const int at = chunk(j) * rows::kChunk;
    return kWhole ? max(0, min(at, width - rows::kChunk)) : at;
  }
  __device__ __forceinline__ int skip(int j) const {
    return kWhole && on(j) && width >= rows::kChunk ? chunk(j) * rows::kChunk - begin(j) : 0;
  }
  __device__ __forceinline__ int left(int j) const { return width - begin(j); }
};

// A row's values of a lane, and those of its 8-bit checkpoint, as they lie in
// memory.
template <typename T, int kChunks>
struct Raw {
  rows::Words<T> c[kChunks];
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void load(const void *base, int64_t offset,
                                       const Place<kLanes, kChunks, kWhole> &at) {
    const T *row = static_cast<const T *>(base) + offset;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
      c[j].load(row + at.begin(j), at.on(j) ? at.left(j) : 0);
  }
  __device__ __forceinline__ float get(int j, int i) const { return c[j].get(i); }
};
template <int kChunks>
struct Packed {
  rows::PackedChunk c[kChunks];
  template <int kLanes>
  __device__ __forceinline__ void load(const uint8_t *row,
                                       const Place<kLanes, kChunks, false> &at) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
      if (at.on(j)) c[j].load(row, at.chunk(j), rows::blocks_of(at.width));
  }
  __device__ __forceinline__ void get(float (&v)[kChunks][rows::kChunk]) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) c[j].get(v[j]);
  }
};

template <typename T, int kLanes, int kChunks, bool kWhole>
__device__ __forceinline__ void store_row(void *base, int64_t offset,
                                          const float (&v)[kChunks][rows::kChunk],
                                          const Place<kLanes, kChunks, kWhole> &at) {
  T *row = static_cast<T *>(base) + offset;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    if (!at.on(j)) continue;
    rows::store(row + at.begin(j), v[j], at.left(j));
  }
}

// Sum of f(j, i) over a lane's values, none twice.
template <int kLanes, int kChunks, bool kWhole, typename F>
__device__ __forceinline__ float own_sum(const Place<kLanes, kChunks, kWhole> &at, F f) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int skip = at.skip(j);
    if (skip == 0) {
#pragma unroll
      for (int i = 0; i < rows::kChunk; ++i) s += f(j, i);
    } else {
#pragma unroll
      for (int i = 0; i < rows::kChunk; ++i) s += i >= skip ? f(j, i) : 0.f;
    }
  }
  return s;
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

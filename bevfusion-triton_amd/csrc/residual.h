// What the forward and the backward kernels of residual.hip share.
#pragma once

#include "rows.h"

namespace residual {

constexpr int kMaxWidth = 8192;

struct Args {
  // inputs.  Weights that are not there are null; rows that are not there are
  // other rows, read all the same and not used (see the flags), so that no load
  // of a row in turn is behind a condition (but a gate's of its own).
  const void *x, *update, *gate, *update_weight, *scale, *weight;
  bool has_update, has_gate, has_dsum, keeps;
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
// past 4096 values: two), by whole waves, or parts of one for short rows.  More
// lanes hold the last chunk again: us of forward and backward, 43 MB of rows in
// bf16, by these lanes and by the next layout,
//   128 values 28 and 51, 38 and 72      512 values 27 and 51, 38 and 72
//   768 29 and 57, 43 and 78             1024 27 and 56, 32 and 63
//   1280 30 and 57, 33 and 62            1536 28 and 54, 29 and 55
//   2048 28 and 55, 42 and 72
// So rows just past a step lose: 2,304 values 43 and 72, 4,096 35 and 64, 5,120 43
// and 75 (other data than the above, none of it in the cache).  In fp32 two chunks
// do not fit the registers beside two rows (14 to 19 are spilled): 43 MB of rows of
// 4,096 38 and 62 us, of 8,192 63 and 86.
#define RESIDUAL_LAYOUT(FN, width, ...)                                         \
  if ((width) < 8) FN(16, 1, false, __VA_ARGS__)                                \
  else if ((width) <= 128) FN(16, 1, true, __VA_ARGS__)                         \
  else if ((width) <= 256) FN(32, 1, true, __VA_ARGS__)                         \
  else if ((width) <= 512) FN(64, 1, true, __VA_ARGS__)                         \
  else if ((width) <= 1024) FN(128, 1, true, __VA_ARGS__)                       \
  else if ((width) <= 1536) FN(192, 1, true, __VA_ARGS__)                       \
  else if ((width) <= 2048) FN(256, 1, true, __VA_ARGS__)                       \
  else if ((width) <= 4096) FN(512, 1, true, __VA_ARGS__)                       \
  else FN(512, 2, true, __VA_ARGS__)

// (rows of more than a wave pass barriers: a block of them has one)
constexpr int threads_of(int lanes) { return lanes > 64 ? lanes : 256; }
// Waves of a SIMD that the registers of a kernel leave room for (they are
// compiled to), and the blocks of the whole card: the kernels walk rows by as
// many as are there at once.  More only begin later: backward of 200,000 rows of
// 80 by three blocks a CU, as many as there is room for, 48 us, by four 50, 80,000
// of 256 49 and 54; one block a row instead, forward of 16,896 rows of 1,280 45 us
// for 35.
constexpr int forward_waves(int chunks) { return chunks > 1 ? 3 : 4; }
constexpr int backward_waves(int lanes, int chunks, bool kept, bool wide) {
  return chunks > 1 ? 2 : kept || lanes < 64 || wide ? 3 : 4;  // (wide: a stream in fp32)
}
constexpr int blocks_for(int lanes, int waves) {
  const int each = 4 * waves * 64 / threads_of(lanes);
  return 256 * (each > 1 ? each : 1);
}

// A lane's place: its row of a block's, and its chunks.  With kWhole (rows of a
// chunk at least) every lane reads and writes whole chunks, whatever the width:
// where it is no whole number of chunks the last one begins earlier, and lanes
// past it have the last one too.  So the first `skip` values of a chunk are
// another lane's as well; all form the same of them, and only sums leave them
// out.  No access is behind a condition, so the compiler can count them, and a
// row's loads wait for no store of the row before (16,896 rows of 1,280: forward
// 35 us for 39, backward 56 for 65).
template <int kLanes, int kChunks, bool kWhole>
struct Place {
  int lane, group, width;
  __device__ __forceinline__ explicit Place(int width) : width(width) {
    lane = int(threadIdx.x) % kLanes;
    group = int(threadIdx.x) / kLanes;
    if constexpr (kLanes >= 64) group = __builtin_amdgcn_readfirstlane(group);
  }
  __device__ __forceinline__ int chunk(int j) const { return lane + j * kLanes; }
  __device__ __forceinline__ int begin(int j) const {
    const int at = chunk(j) * rows::kChunk;
    return kWhole ? min(at, width - rows::kChunk) : at;
  }
  __device__ __forceinline__ int skip(int j) const {
    return kWhole ? min(rows::kChunk, chunk(j) * rows::kChunk - begin(j)) : 0;
  }
  // values from the chunk's place (not its begin) to the row's end
  __device__ __forceinline__ int left(int j) const { return width - chunk(j) * rows::kChunk; }
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
    for (int j = 0; j < kChunks; ++j) {
      if constexpr (kWhole)
        c[j] = *reinterpret_cast<const rows::Words<T> *>(row + at.begin(j));
      else
        c[j].load(row + at.begin(j), at.left(j));
    }
  }
  __device__ __forceinline__ float get(int j, int i) const { return c[j].get(i); }
  // has arrived here
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
      for (int i = 0; i < rows::Words<T>::kWords; ++i) asm volatile("" : "+v"(c[j].w[i]));
  }
};
template <typename T, int kChunks>
struct Packed {
  rows::Bytes c[kChunks];
  unsigned first[kChunks], last[kChunks];  // scales of a chunk's ends
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void load(const uint8_t *row,
                                       const Place<kLanes, kChunks, kWhole> &at) {
    struct __attribute__((packed, aligned(1))) Eight {
      rows::Bytes b;
    };
    const uint8_t *scales = row + rows::blocks_of(at.width) * rows::kBlock;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      // (without kWhole rows are one block, whose bytes are all there)
      const int begin = kWhole ? at.begin(j) : min(at.begin(j), rows::kBlock - rows::kChunk);
      c[j] = reinterpret_cast<const Eight *>(row + begin)->b;
      first[j] = scales[begin / rows::kBlock];
      last[j] = scales[(begin + rows::kChunk - 1) / rows::kBlock];
    }
  }
  template <int kLanes, bool kWhole>
  __device__ __forceinline__ void get(float (&v)[kChunks][rows::kChunk],
                                      const Place<kLanes, kChunks, kWhole> &at) const {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      rows::unpack<T>(v[j], c[j], first[j]);
      if (at.width % rows::kChunk != 0) {  // (two blocks' values may lie in it)
        float w[rows::kChunk];
        rows::unpack<T>(w, c[j], last[j]);
        const int begin = at.begin(j);
#pragma unroll
        for (int i = 0; i < rows::kChunk; ++i) {
          if ((begin + i) / rows::kBlock != begin / rows::kBlock) v[j][i] = w[i];
          if (!kWhole && i >= at.left(j)) v[j][i] = 0.f;
        }
      }
    }
  }
};

template <typename T, int kLanes, int kChunks, bool kWhole>
__device__ __forceinline__ void store_row(void *base, int64_t offset,
                                          const float (&v)[kChunks][rows::kChunk],
                                          const Place<kLanes, kChunks, kWhole> &at) {
  T *row = static_cast<T *>(base) + offset;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    rows::Words<T> words;
    words.set(v[j]);
    if constexpr (kWhole)
      *reinterpret_cast<rows::Words<T> *>(row + at.begin(j)) = words;
    else
      words.store(row + at.begin(j), at.left(j));
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

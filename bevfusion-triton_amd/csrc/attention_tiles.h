// Tiles, fragments and work lists shared by the attention kernels (gfx950).
//
// Everything is built on the 32 x 32 matrix instructions, one tile a wave.
// With lane = 32 h + c:
//   A (32 x K): lane holds row c, B (K x 32): lane holds column c, both 16
//     bytes of consecutive contraction indices, the half h the later ones;
//   C (32 x 32): lane holds column c; register r holds row
//     8 (r / 4) + 4 h + r % 4.
// A product's contraction index may be permuted as long as both operands
// are.  So the scores are formed with the softmax's rows as columns of C
// (keys x rows, or rows x keys in the key gradients): a lane holds 16 or 32
// scores of ONE row, its maximum and sum need one exchange with lane ^ 32,
// and the weights go back into the next product as B straight from the
// registers they are in, with the rows of C as the contraction index in the
// order above.  The A of that product is the transpose of a row-major tile
// and comes from LDS by the transposing read (16-bit types) or one element a
// lane (float).
//
// Tiles lie in LDS as rows of kPitch 16-byte chunks, swizzled so that reads
// spread over the banks (see swizzle()).  They are filled by
// loads from global memory straight to LDS; since such a load writes its
// lanes' 16 bytes in lane order, the swizzle is on the side of the global
// address.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bevpool.h"
#include "sequences.h"

namespace attention {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;  // four waves
constexpr int kWaves = 4;
constexpr int kWaveRows = 32;  // rows (or keys) that a wave owns
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

#define ATTENTION_LDS __attribute__((address_space(3)))

template <typename T>
struct Mat;
template <>
struct Mat<__bf16> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mat<_Float16> {
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mat<float> {
  typedef f32x4 Frag;
  // four products of two contraction indices, element i of each half
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// A head of up to DP elements of T.
template <typename T, int DP>
struct Shape {
  static constexpr int kSteps = DP * int(sizeof(T)) / 32;        // fragments of a row (2 chunks)
  static constexpr int kChunks = 2 * kSteps;
  // chunks of a row in LDS: whole groups of four (float: eight), see swizzle()
  static constexpr int kPitch =
      sizeof(T) == 2 ? (kChunks + 3) / 4 * 4 : (kChunks + 7) / 8 * 8;
  static constexpr int kBlocks = (DP + 31) / 32;                 // blocks of 32 elements
  static constexpr int tile_bytes(int rows) { return rows * kPitch * 16; }
};

template <typename T, int DP>
using Frags = typename Mat<T>::Frag[Shape<T, DP>::kSteps];  // of one row
template <typename T, int DP>
using Sums = f32x16[Shape<T, DP>::kBlocks];  // 32 columns of elements

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }
__device__ __forceinline__ int wave_id() {
  return __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
}

// The row of C that register r of this lane holds.
__device__ __forceinline__ int c_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// The low half's value and the high half's, each in both halves.  (Elements
// are copied out before the cast: hipcc 7.2 takes __builtin_bit_cast of any
// element of a vector for that of its first.)
struct Halves {
  float low, high;
};
__device__ __forceinline__ Halves halves_of(float v) {
  const unsigned a = __builtin_bit_cast(unsigned, v);
  const auto x = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const unsigned low = x[0], high = x[1];
  return {__builtin_bit_cast(float, low), __builtin_bit_cast(float, high)};
}
__device__ __forceinline__ float max_halves(float v) {
  const Halves x = halves_of(v);
  return fmaxf(x.low, x.high);
}
__device__ __forceinline__ float sum_halves(float v) {
  const Halves x = halves_of(v);
  return x.low + x.high;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Waits until this wave's reads of LDS are done (before a load overwrites
// what they read).
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Waits until this wave's loads to LDS, all but the newest `left` of them,
// have arrived.
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
  static_assert(kLeft >= 0 && kLeft < 64, "vmcnt has 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}

// A barrier behind this wave's reads of LDS.  Unlike __syncthreads() it does
// not wait for loads to LDS that are still on their way to other buffers.
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// One load of 16 bytes a lane from `base` + `offset` to LDS, lane i's at `to`
// (the same for the wave) + 16 i; lanes that are off load nothing.  As asm,
// for the compiler would make the next read of LDS, of whatever buffer, wait
// for it: wait_loads() and a barrier stand before the reads that need it.  It
// writes no register.  The compiler does not see a memory access here, so the
// block itself keeps the five wait states that one needs behind a vector
// instruction that wrote its scalar base (a reload of a spilled one, say),
// and the one behind a write of m0.  It cannot be told that m0 is written
// either (the compiler takes it as reserved); nothing else in these kernels
// uses it, and no vector register is spilled, whose reloads the hand-counted
// waits would count too: tests/test_built_kernels.py looks at the built code.
__device__ __forceinline__ void load_to_lds(const char *base, unsigned offset, unsigned to) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 3\n\t"
      "global_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(int(to))),
      "v"(offset), "s"(base)
      : "memory");
}
// The same of 4 bytes a lane.
__device__ __forceinline__ void load_to_lds4(const char *base, unsigned offset, unsigned to) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 3\n\t"
      "global_load_lds_dword %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(int(to))),
      "v"(offset), "s"(base)
      : "memory");
}

__device__ __forceinline__ unsigned lds_address(const char *p) {
  return unsigned(uintptr_t((const ATTENTION_LDS char *)p));
}

// Where chunk c of row r lies in its row: at c ^ swizzle(r).  LDS gives 256
// bytes a cycle, 16 chunks.  A fragment read takes one chunk of 16 rows at
// once, a transposing read four chunks, a group, of four rows.  With rows of
// a multiple of 256 bytes all four low bits of r have to tell the places
// apart, those of r % 4 by whole groups; rows of an odd number of 128 or 64
// bytes already start in different halves or quarters, and the bits left do
// the rest.  For float the second kind of read is 8 chunks of the rows r and
// r + 4.
template <typename T, int DP>
__device__ __forceinline__ int swizzle(int r) {
  constexpr int kPitch = Shape<T, DP>::kPitch;
  if constexpr (kPitch % 8 != 0) return (r >> 2) & 3;
  if constexpr (kPitch % 16 != 0) return (r & 2) << 1 | ((r >> 2) & 3);
  if constexpr (sizeof(T) == 4) return (r & 4) << 1 | (r & 3) << 1 | ((r >> 3) & 1);
  return (r & 3) << 2 | ((r >> 2) & 3);
}

// Fills tiles of kRows rows with kLanes lanes: this lane's 16-byte pieces of
// a tile, as offsets that stay the same from tile to tile.  Chunks past the
// head's `chunks` are left as they are.  Every wave issues kLoads loads for a
// tile (each of its rounds has a chunk 0).
template <typename T, int DP, int kRows, int kLanes>
struct Stage {
  static constexpr int kPitch = Shape<T, DP>::kPitch;
  static constexpr int kLoads = kRows * kPitch / kLanes;
  static_assert(kRows * kPitch % kLanes == 0, "whole rounds");
  unsigned at[kLoads];
  bool on[kLoads];
  __device__ __forceinline__ static int row(int i) {
    return (i * kLanes + int(threadIdx.x) % kLanes) / kPitch;
  }
  __device__ __forceinline__ static int chunk(int i) {
    return (i * kLanes + int(threadIdx.x) % kLanes) % kPitch ^ swizzle<T, DP>(row(i));
  }
  // place(r): bytes from a tile's base to its row r
  template <typename Place>
  __device__ __forceinline__ void set(int chunks, Place place) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      at[i] = unsigned(place(row(i))) + chunk(i) * 16;
      on[i] = chunk(i) < chunks;
    }
  }
  __device__ __forceinline__ void load(const char *base, unsigned tile) const {
    const unsigned wave = wave_id() % (kLanes / 64) * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (on[i]) load_to_lds(base, at[i], tile + i * kLanes * 16 + wave);
  }
  // the same with rows placed for this tile alone
  template <typename Place>
  __device__ __forceinline__ void load(const char *base, unsigned tile, Place place) const {
    const unsigned wave = wave_id() % (kLanes / 64) * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (on[i])
        load_to_lds(base, unsigned(place(row(i))) + chunk(i) * 16,
                    tile + i * kLanes * 16 + wave);
  }
};

// Rows [k0, k0 + kRows) of an operand into a tile, rows from `stored` on as
// the last one there is.  (Offsets within a tile fit 32 bits: strides are
// checked.)
template <typename T, int DP, int kRows, int kLanes>
__device__ __forceinline__ void load_rows(const Stage<T, DP, kRows, kLanes> &stage, const char *at,
                                          int64_t stride, int k0, int stored, unsigned tile) {
  const char *base = at + k0 * stride;
  if (k0 + kRows <= stored)
    stage.load(base, tile);
  else
    stage.load(base, tile, [&](int r) { return min(r, stored - 1 - k0) * int(stride); });
}

// Chunks [chunks, kChunks) of a tile's rows, which no load fills but a
// product reads: zeros.
template <typename T, int DP>
__device__ __forceinline__ void clear_rest(char *tile, int rows, int thread, int lanes,
                                           int chunks) {
  constexpr int kPitch = Shape<T, DP>::kPitch, kChunks = Shape<T, DP>::kChunks;
  if (chunks >= kChunks) return;
  for (int i = thread; i < rows * kPitch; i += lanes) {
    const int r = i / kPitch, c = (i % kPitch) ^ swizzle<T, DP>(r);
    if (c >= chunks) *reinterpret_cast<u32x4 *>(tile + i * 16) = u32x4{0, 0, 0, 0};
  }
}

// Keeps reads of LDS and matrix products above it above and those below it
// below; all else may cross.  hipcc 7.2 otherwise puts each read right before
// the product that needs it, and every product waits for LDS.
__device__ __forceinline__ void pin_reads() { __builtin_amdgcn_sched_barrier(0x476); }

// The fragments of rows r0 .. r0 + 31 of a tile (r0 a multiple of 32).
template <typename T, int DP>
__device__ __forceinline__ void read_rows(Frags<T, DP> &f, const char *tile, int r0) {
  const int lane = lane_id(), c = lane & 31, h = lane >> 5;
#pragma unroll
  for (int s = 0; s < Shape<T, DP>::kSteps; ++s) {
    const int chunk = (2 * s + h) ^ swizzle<T, DP>(c);
    f[s] = *reinterpret_cast<const typename Mat<T>::Frag *>(
        tile + (r0 + c) * (Shape<T, DP>::kPitch * 16) + chunk * 16);
  }
}

// Has the compiler's own loads into these registers arrive here: in a loop
// behind loads to LDS that it does not count, it would wait for all of them.
template <typename F, int kN>
__device__ __forceinline__ void settle(F (&f)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) asm volatile("" : "+v"(f[i]));
}

// Fragments of one row in global memory (chunks past the head's: zeros).
template <typename T, int DP>
__device__ __forceinline__ void row_frags(Frags<T, DP> &f, const char *row, int chunks, bool valid) {
  const int h = lane_id() >> 5;
#pragma unroll
  for (int s = 0; s < Shape<T, DP>::kSteps; ++s) {
    typename Mat<T>::Frag z = {};
    if (valid && 2 * s + h < chunks)
      z = *reinterpret_cast<const typename Mat<T>::Frag *>(row + (2 * s + h) * 16);
    f[s] = z;
  }
  settle(f);
}

// C = (rows of a) x (rows of b): scores.
template <typename T, int DP>
__device__ __forceinline__ f32x16 dot_rows(const Frags<T, DP> &a, const Frags<T, DP> &b) {
  f32x16 c = {};
#pragma unroll
  for (int s = 0; s < Shape<T, DP>::kSteps; ++s) c = Mat<T>::mma(a[s], b[s], c);
  return c;
}

// The weights of a 32 x 32 block of scores as B of the next product.
template <typename T>
struct Weights {
  typename Mat<T>::Frag f[2];
  __device__ __forceinline__ void set(const float (&p)[16]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) f[r >> 3][r & 7] = T(p[r]);
  }
};
template <>
struct Weights<float> {
  float f[16];
  __device__ __forceinline__ void set(const float (&p)[16]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) f[r] = p[r];
  }
};

// Rows r0 .. r0 + 31 of a tile, transposed: A of a product over the rows, in
// the order in which Weights holds them.
template <typename T, int DP>
struct Columns {
  static constexpr int kBlocks = Shape<T, DP>::kBlocks;
  typename Mat<T>::Frag f[kBlocks][2];
  __device__ __forceinline__ void read(const char *tile, int r0) {
    // the transposing read gives lane i (of 16) element i of four rows; it
    // reads row i / 4, elements 4 (i % 4) .. + 3
    constexpr int kRow = Shape<T, DP>::kPitch * 16;
    const int lane = lane_id(), h = lane >> 5;
    const int row = 4 * h + ((lane & 15) >> 2);
    const int chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const char *at = tile + (r0 + row) * kRow + (lane & 1) * 8;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const char *low = at + ((4 * b + chunk) ^ swizzle<T, DP>(row)) * 16;
      const char *high = at + 8 * kRow + ((4 * b + chunk) ^ swizzle<T, DP>(row + 8)) * 16;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (ATTENTION_LDS i16x4 *)(low + 16 * j * kRow));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (ATTENTION_LDS i16x4 *)(high + 16 * j * kRow));
        const i16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        f[b][j] = __builtin_bit_cast(typename Mat<T>::Frag, a);
      }
    }
  }
  // acc[b] += (columns 32 b .. 32 b + 31)^T x weights
  __device__ __forceinline__ void add(Sums<T, DP> &acc, const Weights<T> &w) const {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        acc[b] = Mat<T>::mma(f[b][j], w.f[j], acc[b]);
  }
};
// float: one element a lane of register r's row, read as they are used.
template <int DP>
struct Columns<float, DP> {
  static constexpr int kBlocks = Shape<float, DP>::kBlocks;
  const char *at;
  __device__ __forceinline__ void read(const char *tile, int r0) {
    at = tile + r0 * (Shape<float, DP>::kPitch * 16);
  }
  __device__ __forceinline__ void add(Sums<float, DP> &acc, const Weights<float> &w,
                                      int lane = lane_id()) const {
    constexpr int kRow = Shape<float, DP>::kPitch * 16;
    const int h = lane >> 5, c = lane & 31;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = c_row(r, h);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const float a = *reinterpret_cast<const float *>(
            at + row * kRow + ((8 * b + (c >> 2)) ^ swizzle<float, DP>(row)) * 16 + (c & 3) * 4);
        acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w.f[r], acc[b], 0, 0, 0);
      }
    }
  }
};

// Pieces of the above, four fragments at a time, for kernels that are short of
// registers: rows' fragments s0 .. s0 + kN - 1, and column blocks b0, b0 + 1.
template <typename T>
using Piece = typename Mat<T>::Frag[4];

template <typename T, int DP, int kN>
__device__ __forceinline__ void read_piece(Piece<T> &f, const char *tile, int r0, int s0,
                                           int lane) {
  const int c = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i = 0; i < kN; ++i)
    if (s0 + i < Shape<T, DP>::kSteps)
      f[i] = *reinterpret_cast<const typename Mat<T>::Frag *>(
          tile + (r0 + c) * (Shape<T, DP>::kPitch * 16) +
          ((2 * (s0 + i) + h) ^ swizzle<T, DP>(c)) * 16);
}
template <typename T, int DP>
__device__ __forceinline__ void read_column_piece(Piece<T> &f, const char *tile, int r0, int b0,
                                                  int lane) {
  constexpr int kRow = Shape<T, DP>::kPitch * 16;
  const int h = lane >> 5;
  const int row = 4 * h + ((lane & 15) >> 2);
  const int chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const char *at = tile + (r0 + row) * kRow + (lane & 1) * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (b0 + i >= Shape<T, DP>::kBlocks) continue;
    const char *low = at + ((4 * (b0 + i) + chunk) ^ swizzle<T, DP>(row)) * 16;
    const char *high = at + 8 * kRow + ((4 * (b0 + i) + chunk) ^ swizzle<T, DP>(row + 8)) * 16;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const i16x4 lo =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((ATTENTION_LDS i16x4 *)(low + 16 * j * kRow));
      const i16x4 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((ATTENTION_LDS i16x4 *)(high + 16 * j * kRow));
      const i16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      f[2 * i + j] = __builtin_bit_cast(typename Mat<T>::Frag, a);
    }
  }
}
template <typename T, int DP>
__device__ __forceinline__ void add_column_piece(Sums<T, DP> &acc, const Piece<T> &f,
                                                 const Weights<T> &w, int b0) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (b0 + i < Shape<T, DP>::kBlocks)
        acc[b0 + i] = Mat<T>::mma(f[2 * i + j], w.f[j], acc[b0 + i]);
}

// Running softmax of one row: a lane and lane ^ 32 share it, with half of a
// block's keys each.
struct Softmax {
  float top = -kInf;  // the maximum that the weights are relative to
  float sum = 0.f;    // of this lane's half of the keys
};

// Takes kN scores of this lane's row (raw products, -inf where masked):
// they become weights exp2(scale_log2 (s - top)).  top follows the maximum
// only where the row's new maximum is more than kSlack above it (in log2),
// so most blocks leave the sums as they are: weights stay below 2^kSlack,
// far from the types' largest values, and relative to each other as exact.
constexpr float kSlack = 8.f;
template <int kN, int kB>
__device__ __forceinline__ void softmax_step(float (&s)[kN], Softmax &x, f32x16 (&out)[kB],
                                             float scale_log2) {
  float most = s[0];
#pragma unroll
  for (int i = 1; i < kN; ++i) most = fmaxf(most, s[i]);
  most = max_halves(most);
  // (no comparison is true for a row that has seen nothing but -inf)
  if (__ballot((most - x.top) * scale_log2 > kSlack)) {
    const float top = fmaxf(most, x.top);
    const float by = top == -kInf ? 1.f : exp2_fast((x.top - top) * scale_log2);
    x.top = top;
    x.sum *= by;
#pragma unroll
    for (int b = 0; b < kB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[b][r] *= by;
  }
  const float shift = x.top == -kInf ? 0.f : x.top * scale_log2;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    s[i] = exp2_fast(fmaf(s[i], scale_log2, -shift));
    sum += s[i];
  }
  x.sum += sum;
}

// A wave's 32 rows (fragments q) against the keys [begin, end) of one head,
// in tiles of kKeys keys staged by the whole block in two buffers (K0 V0 K1
// V1), the next tile's loads in flight while one is used.  This lane's row
// sees the keys below `limit`; every row of the wave those below `low` (no
// mask there), none those from `high` on.  Keys from `stored` on are not
// read.  The block calls it together, with the same begin and end.  With
// kHalves the wave takes 32 keys of each tile of 64, those from 32 * half on.
template <typename T, int DP, int kKeys, bool kHalves = false>
__device__ __forceinline__ void attend_tiles(char *lds, const Frags<T, DP> &q, const char *k_at,
                                             int64_t k_row, const char *v_at, int64_t v_row,
                                             int chunks, int begin, int end, int stored, int limit,
                                             int low, int high, float scale_log2, Softmax &x,
                                             Sums<T, DP> &out, int half = 0) {
  constexpr int kTile = Shape<T, DP>::tile_bytes(kKeys);
  constexpr int kMine = kHalves ? 1 : kKeys / 32;  // blocks of 32 keys
  static_assert(!kHalves || kKeys == 64, "two halves of 32");
  const int mine = kHalves ? 32 * half : 0;
  const int h = lane_id() >> 5;
  const unsigned lds0 = lds_address(lds);
  Stage<T, DP, kKeys, kThreads> k_stage, v_stage;
  k_stage.set(chunks, [&](int r) { return r * int(k_row); });
  v_stage.set(chunks, [&](int r) { return r * int(v_row); });
  auto load_tile = [&](int k0, int buffer) {
    const unsigned to = lds0 + buffer * 2 * kTile;
    load_rows(k_stage, k_at, k_row, k0, stored, to);
    load_rows(v_stage, v_at, v_row, k0, stored, to + kTile);
  };
  clear_rest<T, DP>(lds, 4 * kKeys, threadIdx.x, kThreads, chunks);
  if (begin < end) load_tile(begin, 0);
  int buffer = 0;
  for (int k0 = begin; k0 < end; k0 += kKeys, buffer ^= 1) {
    wait_loads<0>();
    __syncthreads();  // this tile is there, and the last one has been read
    if (k0 + kKeys < end) load_tile(k0 + kKeys, buffer ^ 1);
    const char *k_tile = lds + buffer * 2 * kTile, *v_tile = k_tile + kTile;
    if (k0 + mine >= high) continue;
    float s[16 * kMine];
#pragma unroll
    for (int b = 0; b < kMine; ++b) {
      Frags<T, DP> k;
      read_rows<T, DP>(k, k_tile, mine + 32 * b);
      pin_reads();
      const f32x16 dots = dot_rows<T, DP>(k, q);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[16 * b + r] = dots[r];
    }
    if (k0 + mine + 32 * kMine > low) {
#pragma unroll
      for (int b = 0; b < kMine; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + mine + 32 * b + c_row(r, h) >= limit) s[16 * b + r] = -kInf;
    }
    softmax_step(s, x, out, scale_log2);
#pragma unroll
    for (int b = 0; b < kMine; ++b) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = s[16 * b + r];
      Weights<T> w;
      w.set(p);
      Columns<T, DP> v;
      v.read(v_tile, mine + 32 * b);
      pin_reads();
      v.add(out, w);
    }
  }
}

// Writes a lane's column of acc times `by`, rounded to T once, as a row; with
// kRest what the rounding took off, rounded to T itself, to another.
template <typename T, int DP, bool kRest = false>
__device__ __forceinline__ void store_row(char *row, const Sums<T, DP> &acc, float by, int dim,
                                          bool valid, char *rest = nullptr) {
  const int h = lane_id() >> 5;
#pragma unroll
  for (int b = 0; b < Shape<T, DP>::kBlocks; ++b) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * b + 8 * g + 4 * h;
        if (valid && d < dim)
          *reinterpret_cast<f32x4 *>(row + d * 4) =
              f32x4{acc[b][4 * g] * by, acc[b][4 * g + 1] * by, acc[b][4 * g + 2] * by,
                    acc[b][4 * g + 3] * by};
      }
    } else {
      // four neighbours a lane; the halves trade so that each has eight
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        typedef T Pair __attribute__((ext_vector_type(2)));
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = acc[b][8 * p + i] * by;
        const int d = 32 * b + 16 * p + 8 * h;
#pragma unroll
        for (int n = 0; n < (kRest ? 2 : 1); ++n) {
          unsigned x[4];  // v[0..1], v[2..3], v[4..5], v[6..7]
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const Pair pair{T(v[2 * i]), T(v[2 * i + 1])};
            x[i] = __builtin_bit_cast(unsigned, pair);
            if (kRest) {
              v[2 * i] -= float(pair[0]);
              v[2 * i + 1] -= float(pair[1]);
            }
          }
          const auto a = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
          const auto c = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
          if (valid && d < dim)
            *reinterpret_cast<u32x4 *>((n == 0 ? row : rest) + d * 2) =
                u32x4{a[0], c[0], a[1], c[1]};
        }
      }
    }
  }
}

// A lane's sums pass from the waves of one half to those of the other through
// LDS, at `at` (the pair's, 64 * 16 * kBlocks floats).
template <typename T, int DP>
__device__ __forceinline__ void put_sums(float *at, const Sums<T, DP> &acc) {
#pragma unroll
  for (int b = 0; b < Shape<T, DP>::kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) at[(b * 16 + r) * 64 + lane_id()] = acc[b][r];
}
template <typename T, int DP>
__device__ __forceinline__ void add_sums(Sums<T, DP> &acc, const float *at, float by = 1.f) {
#pragma unroll
  for (int b = 0; b < Shape<T, DP>::kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] += by * at[(b * 16 + r) * 64 + lane_id()];
}

// ---------------------------------------------------------------------------
// packed sequences
// ---------------------------------------------------------------------------

// Blocks of four waves take 128 rows (or keys), 32 a wave, where that fills
// the card: two blocks a CU.  Below that they take 64, and two waves halve
// the walk over the other side, whose length is then the time of the launch.
// Forward in bf16, us of whole and of halved walks: one causal sequence of
// 4,096 (256 blocks) and of 6,000 (376) over 8 heads of 128, 80 and 63, 117
// and 93; one of 3,500 over 16 heads of 64 without a mask (448) 71 and 76, so
// the bound is not higher up.
constexpr int kFullBlocks = 512;
template <typename T, int DP>
constexpr bool kMayHalve = DP * int(sizeof(T)) <= 256;  // (a tile of 64 in LDS, twice)

// The wave's side of the search over the starts (sequences.h).
struct Wave {
  template <typename Ok>
  __device__ __forceinline__ int count(Ok ok) const {
    return __popcll(__ballot(ok(lane_id())));
  }
  __device__ __forceinline__ int uniform(int v) const { return __builtin_amdgcn_readfirstlane(v); }
};

using sequences::Group;
using sequences::make_group;
using sequences::Sequence;

// ---------------------------------------------------------------------------
// arguments
// ---------------------------------------------------------------------------

struct Operand {  // (rows, heads, dim), unit stride along dim; strides in bytes
  char *at;
  int64_t row, head;
};

struct PackedArgs {
  Operand q, k, v, out, dout, dq, dk, dv;
  char *rest;          // as out: what out's rounding took off, or null
  float *lse;          // (tokens, heads): log of the sum of exponentials
  const int32_t *q_starts, *k_starts;  // sequences + 1
  int sequences, q_total, k_total;
  int q_heads, k_heads;
  Group group;
  int dim, chunks;     // elements and 16-byte chunks of a head
  int causal;
  float scale, scale_log2;
  int tiles;
};

__device__ __forceinline__ sequences::Starts starts_of(const PackedArgs &A) {
  return {A.q_starts, A.k_starts, A.sequences, A.q_total, A.k_total};
}

// Blocks of 128 rows that a call has.
inline int64_t row_blocks(const PackedArgs &A) {
  return (int64_t(A.q_total) * A.group.size / 128 + A.sequences + 1) * A.k_heads;
}

// Host side (attention.hip): sizes and operands of a packed call.
__attribute__((visibility("hidden"))) int check_packed(
    PackedArgs &A, int dtype, int64_t q_total, int64_t k_total, int sequences, int q_heads,
    int k_heads, int dim, const void *q_starts, const void *k_starts, int causal, float scale);
__attribute__((visibility("hidden"))) int set_operand(Operand &o, const char *what, const void *at,
                                                      int64_t row, int64_t head, int elem,
                                                      int64_t total);

}  // namespace attention

// FN of the smallest instance that holds a head of `dim` elements.
#define ATTENTION_DIM(T, FN, ...)                                                   \
  dim <= 32   ? FN<T, 32>(__VA_ARGS__)                                              \
  : dim <= 64 ? FN<T, 64>(__VA_ARGS__)                                              \
  : dim <= 80 ? FN<T, 80>(__VA_ARGS__)                                              \
  : dim <= 96 ? FN<T, 96>(__VA_ARGS__)                                              \
              : FN<T, 128>(__VA_ARGS__)

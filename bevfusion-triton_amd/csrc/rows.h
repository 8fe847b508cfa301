// Rows of values in registers, and their 8-bit checkpoints (gfx950): shared by
// the kernels of the block around the attention.
//
// A lane holds eight neighbouring values of a row (a chunk), four lanes a
// block of 32.  A checkpoint holds a block as 32 bytes and one for its scale:
//   scale  2^e, e the least with 127 2^e >= the largest magnitude (e >= -126,
//          and at most 121, so that nothing comes back infinite)
//   value  rint(x / 2^e), ties to even, as an unsigned byte 128 higher; 0
//          stands for a value that is not finite and comes back as NaN
// The scale is a power of two, so that neither the quotient nor the product
// is rounded: the byte depends on nothing but x, and what it stands for has 7
// bits, exact in bf16.  A value is off by half a scale at most, which is less than
// 1/127 of its block's largest magnitude, on average over normal values by 0.7% of
// their deviation (3 bits of mantissa in 8, the other way to spend them, are 2.6%).
// A row is the bytes of its blocks, then their scales, padded to 16 bytes: 33
// bytes for 32 values of wide rows, 48 at least (8 values in 16 bits are 16).
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace rows {

constexpr int kChunk = 8;   // values of a lane's access
constexpr int kBlock = 32;  // values that share a scale

__host__ __device__ inline int64_t blocks_of(int64_t width) { return (width + kBlock - 1) / kBlock; }
__host__ __device__ inline int64_t checkpoint_pitch(int64_t width) {
  return (blocks_of(width) * (kBlock + 1) + 15) / 16 * 16;
}

// A chunk as it lies in memory, in whole registers: what reads it is apart from
// what converts it, so that the loads of several are on their way together.
// (Accesses of 16 bytes need no more than the type's own alignment.)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Words {
  static constexpr int kWords = kChunk * int(sizeof(T)) / 4;
  unsigned w[kWords];
  // `left` values are there (the others: zeros)
  __device__ __forceinline__ void load(const T *at, int left) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    if (left >= kChunk) {
      *this = *reinterpret_cast<const Words *>(at);
    } else if (left > 0) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        if (i >= left) continue;
        const T v = at[i];
        if constexpr (sizeof(T) == 4)
          w[i] = __builtin_bit_cast(unsigned, v);
        else
          w[i / 2] |= unsigned(__builtin_bit_cast(uint16_t, v)) << (i % 2 * 16);
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __builtin_bit_cast(float, w[i]);
    } else if constexpr (__is_same(T, __bf16)) {  // (the upper half of the same number in fp32)
      return __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    } else {
      return float(__builtin_bit_cast(T, uint16_t(i % 2 ? w[i / 2] >> 16 : w[i / 2])));
    }
  }
  __device__ __forceinline__ void set(const float (&v)[kChunk]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __builtin_bit_cast(unsigned, v[i]);
      } else {
        typedef T Pair __attribute__((ext_vector_type(2)));
        const Pair pair{T(v[2 * i]), T(v[2 * i + 1])};
        w[i] = __builtin_bit_cast(unsigned, pair);
      }
    }
  }
  __device__ __forceinline__ void store(T *at, int left) const {
    if (left >= kChunk) {
      *reinterpret_cast<Words *>(at) = *this;
    } else if (left > 0) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        if (i >= left) continue;
        if constexpr (sizeof(T) == 4)
          at[i] = __builtin_bit_cast(T, w[i]);
        else
          at[i] = __builtin_bit_cast(T, uint16_t(w[i / 2] >> (i % 2 * 16)));
      }
    }
  }
};

// The same at once.
template <typename T>
__device__ __forceinline__ void load(float (&to)[kChunk], const T *at, int left) {
  Words<T> words;
  words.load(at, left);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) to[i] = words.get(i);
}
template <typename T>
__device__ __forceinline__ void store(T *at, const float (&from)[kChunk], int left) {
  Words<T> words;
  words.set(from);
  words.store(at, left);
}

template <int kControl>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return unsigned(__builtin_amdgcn_mov_dpp(int(v), kControl, 0xf, 0xf, true));
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E;             // lane ^ 1, lane ^ 2
constexpr int kMirror8 = 0x141, kMirror16 = 0x140;      // within 8 and 16 lanes

// Sum over kLanes (16, 32 or 64) neighbouring lanes, in all of them.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
  auto add = [&](unsigned other) { v += __builtin_bit_cast(float, other); };
  auto bits = [&] { return __builtin_bit_cast(unsigned, v); };
  add(dpp<kSwap1>(bits()));
  add(dpp<kSwap2>(bits()));
  add(dpp<kMirror8>(bits()));  // (the quads hold their sums: any lane of the other does)
  add(dpp<kMirror16>(bits()));
  if constexpr (kLanes >= 32) {
    const auto x = __builtin_amdgcn_permlane16_swap(bits(), bits(), false, false);
    const unsigned a = x[0], b = x[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  if constexpr (kLanes >= 64) {
    const auto x = __builtin_amdgcn_permlane32_swap(bits(), bits(), false, false);
    const unsigned a = x[0], b = x[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  return v;
}

__device__ __forceinline__ float power(unsigned biased) {
  return __builtin_bit_cast(float, biased << 23);
}

struct Bytes {
  unsigned low, high;
};
// The low bytes of eight words.
__device__ __forceinline__ Bytes low_bytes(const unsigned (&q)[kChunk]) {
  auto four = [](unsigned a, unsigned b, unsigned c, unsigned d) {
    const unsigned ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);
    const unsigned cd = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return ab | cd << 16;
  };
  return {four(q[0], q[1], q[2], q[3]), four(q[4], q[5], q[6], q[7])};
}

// A chunk as bytes, and its block's scale (a biased exponent).  The block's
// four lanes call it together; values past a row's end are zeros.
__device__ __forceinline__ Bytes pack(const float (&v)[kChunk], unsigned &scale) {
  constexpr unsigned kInfinite = 0x7f800000u;
  unsigned top = 0, worst = 0;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const unsigned m = __builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu;
    worst = worst > m ? worst : m;
  }
  top = worst;
  if (worst >= kInfinite) {  // (rare: the largest of those that are finite)
    top = 0;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const unsigned m = __builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu;
      top = m < kInfinite && m > top ? m : top;
    }
  }
  unsigned other = dpp<kSwap1>(top);
  top = top > other ? top : other;
  other = dpp<kSwap2>(top);
  top = top > other ? top : other;
  // 127 = 1.984375 2^6: a mantissa above 0x7E0000 takes the next exponent
  const int e = int((top + 0x1ffffu) >> 23) - 6;
  scale = unsigned(e < 1 ? 1 : e > 248 ? 248 : e);
  const float inverse = power(254 - scale);
  // Added to 1.5 2^23 a quotient is rounded to a whole number, ties to even,
  // whose low byte is that of the sum's bits.  (Beyond 127 it gets only where
  // the scale is at its upper end.)
  unsigned q[kChunk];
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const float x = __builtin_amdgcn_fmed3f(v[i] * inverse, -127.f, 127.f);
    q[i] = __builtin_bit_cast(unsigned, x + (12582912.f + 128.f));
  }
  if (worst >= kInfinite) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if ((__builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu) >= kInfinite) q[i] = 0;
  }
  return low_bytes(q);
}

// A chunk of values of T from its bytes.
template <typename T>
__device__ __forceinline__ void unpack(float (&v)[kChunk], Bytes b, unsigned scale) {
  const float by = power(scale);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    v[i] = (float(((i < 4 ? b.low : b.high) >> (i % 4 * 8)) & 0xffu) - 128.f) * by;
    // (64 2^10, which stands for fp16 values from 65,024 on, is none itself: their
    // largest.  A step of 16,896 rows of 1,283 149 us, by the branch below 155.)
    if constexpr (__is_same(T, _Float16)) v[i] = __builtin_amdgcn_fmed3f(v[i], -65504.f, 65504.f);
  }
  // a byte of zero borrows: one test for four
  auto zero = [](unsigned x) { return (x - 0x01010101u) & ~x & 0x80808080u; };
  if ((zero(b.low) | zero(b.high)) != 0) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if ((((i < 4 ? b.low : b.high) >> (i % 4 * 8)) & 0xffu) == 0) v[i] = __builtin_nanf("");
  }
}

// Chunk c of a row of a checkpoint as it lies there.  (Chunks of the last block
// behind the row's end are there: zeros.)
struct PackedChunk {
  Bytes bytes = {0x80808080u, 0x80808080u};  // zeros
  unsigned scale = 1;
  __device__ __forceinline__ void load(const uint8_t *row, int c, int64_t blocks) {
    bytes = *reinterpret_cast<const Bytes *>(row + c * int64_t(kChunk));
    scale = row[blocks * kBlock + c / 4];
  }
  template <typename T>
  __device__ __forceinline__ void get(float (&v)[kChunk]) const {
    unpack<T>(v, bytes, scale);
  }
};
// The block's four lanes call it together.
__device__ __forceinline__ void store_packed(uint8_t *row, int c, int64_t blocks,
                                             const float (&v)[kChunk]) {
  unsigned scale;
  const Bytes b = pack(v, scale);
  if (c / 4 >= blocks) return;
  *reinterpret_cast<Bytes *>(row + c * int64_t(kChunk)) = b;
  if (c % 4 == 0) row[blocks * kBlock + c / 4] = uint8_t(scale);
}

}  // namespace rows

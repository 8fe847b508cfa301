// linear8.hip -- products in 8-bit integers with a scale for each token and
// each channel (gfx950).
//
//   s_t    = the least bf16 number with 127 s_t >= max_k |x_tk|
//   q_tk   = rint(x_tk / s_t), ties to even
//   y_tn   = (sum_k q_tk w_nk) s_t c_n + bias_n
// The sums are whole numbers and exact.  A scale of 8 bits makes the codes
// exact too: 127 s_t and the borders between codes, odd multiples of s_t / 2,
// need no rounding in fp32, so a code is checked against them, whatever the
// quotient's rounding.
//
// Tokens' codes lie in rows of a multiple of 128 bytes, zeros behind the last
// value.  So whatever is read of a row of weights past its end counts nothing.
//
// Large products are bound by the matrix instructions at the clock that the
// card's power leaves (busy in 47% of the cycles): 8192 x 8192 x 8192 487 us,
// 2,260 TOPS (a library's product to 32-bit sums 2,050), 16,896 x 1,280 x 10,240
// 255 us, 1,740 TOPS, and 15 for the codes; a few tokens by the weights' bytes:
// one of 4,096 x 6,144 8.1 us, codes and all, 67 of 5,000 x 4,099 10.5 and 4.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "attention_tiles.h"
#include "bevpool.h"
#include "host_calls.h"
#include "rows.h"

namespace {

using bevpool_host::check_grid;
using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kPitch = 128;          // rows of codes are a multiple of it
constexpr int kMaxWidth = 1 << 17;   // 2^17 128 127 < 2^31

// ---------------------------------------------------------------------------
// tokens to codes
// ---------------------------------------------------------------------------

// The scale of a row whose largest magnitude is `top` (not finite: NaN).
__device__ __forceinline__ float scale_of(float top) {
  // (the quotient is correctly rounded, so its upper 16 bits are the number
  // or the one below it)
  const unsigned t = __builtin_bit_cast(unsigned, __fdiv_rn(top, 127.f)) & 0xffff0000u;
  float s = __builtin_bit_cast(float, t);
  if (127.f * s < top) s = __builtin_bit_cast(float, t + 0x10000u);
  s = fmaxf(s, 0x1p-126f);
  return top < __builtin_inff() ? s : __builtin_nanf("");
}

// rint(x / s), ties to even, for |x| <= 127 s, as the low byte of a word.  The
// quotient comes from 1 / s with one correction, which makes it exact where it
// has few enough bits, as halves of whole numbers have.  Quotients of a number
// of at most 11 bits (fp16, bf16) by one of 8 are such a half or 2^-12 away from
// it, far more than the 2^-16 that they may be off.  In fp32 they can be nearer:
// there x is compared with the border itself; x - k s is exact.
template <typename T>
__device__ __forceinline__ unsigned code_of(float x, float s, float inverse) {
  float q = x * inverse;
  q = fmaf(fmaf(-q, s, x), inverse, q);
  if constexpr (sizeof(T) == 4) {
    const float k = rintf(q), d = 2.f * fmaf(-k, s, x);
    q = fabsf(d) > s ? k + copysignf(1.f, d) : k;
    // (an exact tie went to the even one: its quotient is exact)
  }
  // added to 1.5 2^23 a number is rounded to a whole one, ties to even
  return __builtin_bit_cast(unsigned, q + 12582912.f);
}

// The largest magnitude of a chunk, as the bits of an fp32 number (those of
// infinities and NaN are the largest).
template <typename T>
__device__ __forceinline__ unsigned top_of(const rows::Words<T> &c) {
  unsigned top = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, c.w[i] & 0x7fffffffu);
    return top;
  } else {
    typedef unsigned short Pair __attribute__((ext_vector_type(2)));
    Pair most = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(Pair, c.w[i] & 0x7fff7fffu));
    top = max(unsigned(most[0]), unsigned(most[1]));
    return __builtin_bit_cast(unsigned, float(__builtin_bit_cast(T, uint16_t(top)))) & 0x7fffffffu;
  }
}

// A row of codes by kLanes lanes that hold it (kChunks chunks each), or, with
// kChunks 0, read it twice.
template <typename T, int kLanes, int kChunks>
__global__ __launch_bounds__(256) void codes_kernel(const T *x, int64_t x_row, int64_t n, int width,
                                                    int pitch, int8_t *codes, float *scales) {
  __shared__ unsigned shared[4];
  constexpr int kHold = kChunks > 0 ? kChunks : 1;
  const int lane = int(threadIdx.x) % kLanes;
  const int64_t row = int64_t(blockIdx.x) * (256 / kLanes) + int(threadIdx.x) / kLanes;
  const bool on = row < n;  // (the same for a row's lanes)
  const T *at = x + (on ? row : 0) * x_row;
  rows::Words<T> c[kHold];
  unsigned top = 0;
  if constexpr (kChunks > 0) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int d = (lane + j * kLanes) * 8;
      c[j].load(at + d, width - d);
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) top = max(top, top_of(c[j]));
  } else {
    for (int d = lane * 8; d < width; d += kLanes * 8) {
      c[0].load(at + d, width - d);
      top = max(top, top_of(c[0]));
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = max(top, unsigned(__shfl_xor(int(top), m, 64)));
  if constexpr (kLanes > 64) {
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = top;
    __syncthreads();
    top = max(max(shared[0], shared[1]), max(shared[2], shared[3]));
  }
  if (!on) return;
  const float s = scale_of(__builtin_bit_cast(float, top)), inverse = 1.f / s;
  if (lane == 0) scales[row] = s;
  auto put = [&](const rows::Words<T> &words, int d) {
    unsigned q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = code_of<T>(words.get(i), s, inverse);
    *reinterpret_cast<rows::Bytes *>(codes + row * pitch + d) = rows::low_bytes(q);
  };
  if constexpr (kChunks > 0) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int d = (lane + j * kLanes) * 8;
      if (d < pitch) put(c[j], d);
    }
  } else {
    for (int d = lane * 8; d < pitch; d += kLanes * 8) {
      c[0].load(at + d, width - d);
      put(c[0], d);
    }
  }
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------

struct ProductArgs {
  const int8_t *x;       // [tokens][x_pitch]
  const int8_t *w;       // [channels], w_row bytes apart
  const float *x_scale, *w_scale;
  const void *bias;      // [channels] or null
  void *y;               // [tokens][channels]
  int64_t w_row;
  int x_pitch, w_chunks;  // 16-byte chunks of a row of w that are there
  int tokens, channels;
  int steps;              // of 64 bytes
  int x_tiles, w_tiles;
};

// Four neighbouring channels' results: whole numbers to T, with both scales.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
  T v[4];
};

// A token's scale around the channel's: ahead of it where it makes a sum smaller,
// behind it where larger.  So nothing on the way passes fp32's range where the
// result does not, whatever the channel's scale.  (One multiplication more:
// 16,896 x 1,280 x 10,240 takes 0.5% longer, with a choice for each value 1.3%.)
struct TokenScale {
  float ahead, behind;
  __device__ __forceinline__ explicit TokenScale(float s)
      : ahead(s >= 1.f ? 1.f : s), behind(s >= 1.f ? s : 1.f) {}
  __device__ __forceinline__ float of(int sum, float channel) const {
    return float(sum) * ahead * channel * behind;
  }
};

// Rows of 64 or 128 bytes in LDS, kChunks of 16: chunk c of row r lies at c ^
// (r / 4) % 4, or c ^ (r / 2) % 8, so the 16 rows of which a fragment read takes
// one chunk each use all of the 256 bytes that LDS gives a cycle.
template <int kChunks>
__device__ __forceinline__ int place(int r, int c) {
  return kChunks == 4 ? c ^ ((r >> 2) & 3) : c ^ ((r >> 1) & 7);
}

// Blocks of one XCD (every eighth) take tiles that lie together: eight tiles of
// channels by as many of tokens as run at once share what their L2 holds.
__device__ __forceinline__ bool tile_of(const ProductArgs &A, int &x_tile, int &w_tile) {
  const int total = A.x_tiles * A.w_tiles, each = (total + 7) / 8;
  const int i = int(blockIdx.x % 8) * each + int(blockIdx.x / 8);
  if (int(blockIdx.x / 8) >= each || i >= total) return false;
  const int group = i / (8 * A.x_tiles), first = group * 8;
  const int wide = min(8, A.w_tiles - first), in = i - first * A.x_tiles;
  x_tile = in / wide;
  w_tile = first + in - x_tile * wide;
  return true;
}

// Waits for all but the newest min(kMost, left) steps' loads, kLoads each.
template <int kLoads, int kMost>
__device__ __forceinline__ void wait_steps(int left) {
  if (kMost == 0 || left >= kMost)
    attention::wait_loads<kLoads * kMost>();
  else
    wait_steps<kLoads, (kMost > 0 ? kMost - 1 : 0)>(left);
}

// One block: kX tokens by kW channels, kWavesX x kWavesW waves of 32 kTx x 32 kTw.  Channels
// are the rows of the matrix instruction's result, tokens its columns: a lane
// holds one token's channels, four neighbours a register group.  kGroups such
// groups of waves take equal parts of the rows' length, each with tiles of its
// own, and the first adds their sums.
template <typename T, int kTx, int kTw, int kWavesX, int kWavesW, int kStep, int kBuffers,
          int kGroups>
__global__ __launch_bounds__(64 * kWavesX * kWavesW * kGroups, kGroups > 2 ? kGroups : 2)
void product_kernel(ProductArgs A) {
  constexpr int kThreads = 64 * kWavesX * kWavesW;  // of a group
  constexpr int kX = 32 * kTx * kWavesX, kW = 32 * kTw * kWavesW;
  constexpr int kChunks = kStep / 16;
  constexpr int kLoadsX = kX * kChunks / kThreads, kLoadsW = kW * kChunks / kThreads;
  constexpr int kTileX = kX * kStep, kTile = (kX + kW) * kStep;
  static_assert(kX * kChunks % kThreads == 0 && kW * kChunks % kThreads == 0, "whole rounds");
  extern __shared__ __align__(16) char lds[];
  float *scales = reinterpret_cast<float *>(lds + kGroups * kBuffers * kTile);
  float *biases = scales + kW;
  int x_tile, w_tile;
  if (!tile_of(A, x_tile, w_tile)) return;
  const int lane = attention::lane_id(), group = attention::wave_id() / (kThreads / 64);
  const int wave = attention::wave_id() % (kThreads / 64), thread = int(threadIdx.x) % kThreads;
  const int x0 = x_tile * kX, w0 = w_tile * kW;
  for (int i = threadIdx.x; i < kW; i += kThreads * kGroups) {
    const bool on = w0 + i < A.channels;
    scales[i] = on ? A.w_scale[w0 + i] : 0.f;
    biases[i] = on && A.bias ? float(static_cast<const T *>(A.bias)[w0 + i]) : 0.f;
  }
  const unsigned lds0 = attention::lds_address(lds) + group * kBuffers * kTile;
  char *const tiles = lds + group * kBuffers * kTile;
  // this group's steps
  const int all = A.x_pitch / kStep, most = (all + kGroups - 1) / kGroups, first = group * most;
  const int steps = min(most, all - first);
  // this lane's pieces of the tiles: offsets from a step's first byte
  const char *x_at =
      reinterpret_cast<const char *>(A.x) + int64_t(x0) * A.x_pitch + int64_t(first) * kStep;
  const char *w_at = reinterpret_cast<const char *>(A.w) + w0 * A.w_row;
  unsigned x_off[kLoadsX], w_off[kLoadsW];
  int w_chunk[kLoadsW];
#pragma unroll
  for (int i = 0; i < kLoadsX; ++i) {
    const int slot = i * kThreads + thread, r = slot / kChunks, c = place<kChunks>(r, slot % kChunks);
    x_off[i] = unsigned(min(r, A.tokens - 1 - x0) * A.x_pitch + c * 16);
  }
#pragma unroll
  for (int i = 0; i < kLoadsW; ++i) {
    const int slot = i * kThreads + thread, r = slot / kChunks;
    w_chunk[i] = first * kChunks + place<kChunks>(r, slot % kChunks);
    w_off[i] = unsigned(min(r, A.channels - 1 - w0) * int(A.w_row));
  }
  auto load = [&](int step, int buffer) {
    const unsigned to = lds0 + buffer * kTile + wave * 1024;
    const char *x = x_at + int64_t(step) * kStep;
#pragma unroll
    for (int i = 0; i < kLoadsX; ++i)
      attention::load_to_lds(x, x_off[i], to + i * kThreads * 16);
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i) {
      // (past a row's end: its last chunk once more, which meets zeros)
      const int c = min(step * kChunks + w_chunk[i], A.w_chunks - 1);
      attention::load_to_lds(w_at, w_off[i] + c * 16, to + kTileX + i * kThreads * 16);
    }
  };
  i32x16 acc[kTw][kTx] = {};
  const int wx = wave % kWavesX * 32 * kTx, ww = wave / kWavesX * 32 * kTw;
  const int c = lane & 31, h = lane >> 5;
  // (the compiler's own loads, of scales, are done: what is counted is the tiles')
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int i = 0; i < kBuffers - 1; ++i)
    if (i < steps) load(i, i);
  int buffer = 0;
  for (int step = 0; step < most; ++step) {  // (as many barriers for every group)
    wait_steps<kLoadsX + kLoadsW, kBuffers - 2>(steps - 1 - step);
    attention::tile_barrier();  // this step's tiles are there, and the last one's have been read
    if (kGroups > 1 && step >= steps) continue;
    if (step + kBuffers - 1 < steps)
      load(step + kBuffers - 1, buffer == 0 ? kBuffers - 1 : buffer - 1);
    const char *x_tile = tiles + buffer * kTile, *w_tile = x_tile + kTileX;
    buffer = buffer == kBuffers - 1 ? 0 : buffer + 1;
#pragma unroll
    for (int s = 0; s < kStep / 32; ++s) {
      i32x4 x[kTx], w[kTw];
#pragma unroll
      for (int i = 0; i < kTx; ++i)
        x[i] = *reinterpret_cast<const i32x4 *>(x_tile + (wx + 32 * i + c) * kStep +
                                                place<kChunks>(c, 2 * s + h) * 16);
#pragma unroll
      for (int i = 0; i < kTw; ++i)
        w[i] = *reinterpret_cast<const i32x4 *>(w_tile + (ww + 32 * i + c) * kStep +
                                                place<kChunks>(c, 2 * s + h) * 16);
#pragma unroll
      for (int i = 0; i < kTw; ++i)
#pragma unroll
        for (int j = 0; j < kTx; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[i], x[j], acc[i][j], 0, 0, 0);
    }
  }
  if constexpr (kGroups > 1) {
    // the groups' sums, each in the place of tiles of its own (all read by now)
    static_assert(kBuffers * kTile >= kX * kW * 4, "a group's sums fit its tiles");
    __syncthreads();
    if (group > 0) {
      int *to = reinterpret_cast<int *>(tiles) + wave * (kTw * kTx * 1024) + lane;
#pragma unroll
      for (int i = 0; i < kTw * kTx * 16; ++i) to[i * 64] = acc[i / 16 / kTx][i / 16 % kTx][i % 16];
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) {
      const int *from = reinterpret_cast<const int *>(lds + g * kBuffers * kTile) +
                        wave * (kTw * kTx * 1024) + lane;
#pragma unroll
      for (int i = 0; i < kTw * kTx * 16; ++i) acc[i / 16 / kTx][i / 16 % kTx][i % 16] += from[i * 64];
    }
  }
#pragma unroll
  for (int j = 0; j < kTx; ++j) {
    const int token = x0 + wx + 32 * j + c;
    const bool valid = token < A.tokens;
    const TokenScale by(valid ? A.x_scale[token] : 0.f);
    T *y = static_cast<T *>(A.y) + int64_t(token) * A.channels;
#pragma unroll
    for (int i = 0; i < kTw; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        // channels 16 p + 4 h .. + 3 and those 8 further
        const int n = ww + 32 * i + 16 * p + 4 * h;
        float v[8];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const attention::f32x4 scale = *reinterpret_cast<attention::f32x4 *>(scales + n + 8 * g);
          const attention::f32x4 bias = *reinterpret_cast<attention::f32x4 *>(biases + n + 8 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            v[4 * g + r] = by.of(acc[i][j][8 * p + 4 * g + r], scale[r]) + bias[r];
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int at = w0 + n + 8 * g;
            if (valid && at + 4 <= A.channels) {
              *reinterpret_cast<Four<T> *>(y + at) = {v[4 * g], v[4 * g + 1], v[4 * g + 2],
                                                      v[4 * g + 3]};
            } else if (valid) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (at + r < A.channels) y[at + r] = v[4 * g + r];
            }
          }
        } else {
          // the halves trade four channels so that each has eight neighbours
          typedef T Pair __attribute__((ext_vector_type(2)));
          unsigned q[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const Pair pair{T(v[2 * r]), T(v[2 * r + 1])};
            q[r] = __builtin_bit_cast(unsigned, pair);
          }
          const auto a = __builtin_amdgcn_permlane32_swap(q[0], q[2], false, false);
          const auto b = __builtin_amdgcn_permlane32_swap(q[1], q[3], false, false);
          const rows::Words<T> out{{a[0], b[0], a[1], b[1]}};
          const int at = w0 + ww + 32 * i + 16 * p + 8 * h;
          out.store(y + at, valid ? A.channels - at : 0);
        }
      }
  }
}

// Few tokens and channels: 16 kTx tokens by 16 channels a block, whose eight waves
// take every eighth 64 bytes of the rows straight to registers, so that the
// weights are on their way all at once, and add their sums in LDS.
constexpr int kFewWaves = 8, kFewThreads = 64 * kFewWaves;

// The waves' sums of a block to its results.
template <typename T, int kTx>
__device__ __forceinline__ void finish_few(const ProductArgs &A, i32x4 (&sums)[kFewWaves][kTx][64],
                                           const i32x4 (&acc)[kTx], const float *x_scale, int w0,
                                           int lane, int wave) {
  const int c = lane & 15, q = lane >> 4;
#pragma unroll
  for (int j = 0; j < kTx; ++j) sums[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave >= kTx) return;
  i32x4 sum = sums[0][wave][lane];
#pragma unroll
  for (int i = 1; i < kFewWaves; ++i) sum += sums[i][wave][lane];
  // lane 16 q + c: channels 4 q .. + 3 of token c
  const T *bias = static_cast<const T *>(A.bias);
  const int token = wave * 16 + c, n = w0 + 4 * q;
  if (token >= A.tokens) return;
  const TokenScale by(x_scale[token]);
  T *y = static_cast<T *>(A.y) + int64_t(token) * A.channels + n;
  Four<T> four;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int at = min(n + r, A.channels - 1);
    four.v[r] = T(by.of(sum[r], A.w_scale[at]) + (bias ? float(bias[at]) : 0.f));
  }
  if (n + 4 <= A.channels) {
    *reinterpret_cast<Four<T> *>(y) = four;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < A.channels) y[r] = four.v[r];
  }
}

template <typename T, int kTx>
__global__ __launch_bounds__(kFewThreads, 4) void few_kernel(ProductArgs A) {
  __shared__ i32x4 sums[kFewWaves][kTx][64];
  constexpr int kDeep = 4;  // steps whose loads are on their way together
  const int lane = attention::lane_id(), wave = attention::wave_id();
  const int c = lane & 15, q = lane >> 4;
  const int w0 = int(blockIdx.x) * 16;
  const int8_t *w_at = A.w + int64_t(min(w0 + c, A.channels - 1)) * A.w_row, *x_at[kTx];
#pragma unroll
  for (int i = 0; i < kTx; ++i)
    x_at[i] = A.x + int64_t(min(16 * i + c, A.tokens - 1)) * A.x_pitch;
  i32x4 acc[kTx] = {};
  for (int first = wave; first < A.steps; first += kFewWaves * kDeep) {
    i32x4 w[kDeep], x[kDeep][kTx];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int step = first + d * kFewWaves, chunk = step * 4 + q;
      w[d] = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kTx; ++i) x[d][i] = i32x4{0, 0, 0, 0};
      if (step >= A.steps) continue;
      // (past a row's end: as above)
      w[d] = *reinterpret_cast<const i32x4 *>(w_at + min(chunk, A.w_chunks - 1) * 16);
#pragma unroll
      for (int i = 0; i < kTx; ++i)
        x[d][i] = *reinterpret_cast<const i32x4 *>(x_at[i] + chunk * 16);
    }
    __builtin_amdgcn_sched_barrier(0);  // (else the compiler takes loads to their products)
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
#pragma unroll
      for (int j = 0; j < kTx; ++j)
        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d], x[d][j], acc[j], 0, 0, 0);
  }
  finish_few<T, kTx>(A, sums, acc, A.x_scale, w0, lane, wave);
}

// Up to eight short tokens: every block forms their codes itself, beside its
// weights' way, instead of a launch before.  Tokens' values go to registers
// first, so that what waits for them does not wait for the weights; a token has
// 512, 256, 128 or 64 of the block's lanes, codes lie in LDS.  us by events, in
// one launch and in two: 1 x 4096 x 6144 10.3, 6.2 + 9.8; 1 x 8192 x 8192 16.6,
// 6.5 + 22.3; 4 x 1280 x 10240 8.9, 6.2 + 7.9; 8 x 2048 x 8192 9.9, 6.6 + 8.0.
// Weights of eight steps are on their way together, of short rows four (1 x 1280
// x 10240 8.6, by eight 11.2; 1 x 4096 x 4096 8.2, by four 11.1).
constexpr int kOwnTokens = 8;
constexpr int kOwnBytes = 16384;  // of codes, tokens rounded up to a power of two
template <typename T, int kDeep>
__global__ __launch_bounds__(kFewThreads, 4) void token_kernel(ProductArgs A, const T *x, int64_t x_row,
                                                               int width, int row_lanes) {
  constexpr int kHold = kOwnBytes / kFewThreads / rows::kChunk;
  __shared__ i32x4 sums[kFewWaves][1][64];
  __shared__ __align__(16) int8_t codes[kOwnBytes + kOwnTokens * 16];  // (16 bytes between rows: banks)
  __shared__ float scales[kOwnTokens];
  __shared__ unsigned tops[kFewWaves];
  const int lane = attention::lane_id(), wave = attention::wave_id();
  const int c = lane & 15, q = lane >> 4;
  const int w0 = int(blockIdx.x) * 16, code_row = A.x_pitch + 16;
  const int token = int(threadIdx.x) / row_lanes, own = int(threadIdx.x) % row_lanes;
  const T *at = x + min(token, A.tokens - 1) * x_row;
  rows::Words<T> words[kHold];
#pragma unroll
  for (int j = 0; j < kHold; ++j) {
    const int d = (own + j * row_lanes) * rows::kChunk;
    words[j].load(at + d, width - d);
  }
  __builtin_amdgcn_sched_barrier(0);
  const int8_t *w_at = A.w + int64_t(min(w0 + c, A.channels - 1)) * A.w_row;
  i32x4 w[kDeep];
  auto fetch = [&](int first) {
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      // (past a row's end, and behind the last step: as above)
      const int chunk = min((first + d * kFewWaves) * 4 + q, A.w_chunks - 1);
      w[d] = *reinterpret_cast<const i32x4 *>(w_at + chunk * 16);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  fetch(wave);
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < kHold; ++j) top = max(top, top_of(words[j]));
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = max(top, unsigned(__shfl_xor(int(top), m, 64)));
  if (lane == 0) tops[wave] = top;
  attention::tile_barrier();
  const int first_wave = token * row_lanes / 64;
  for (int i = 0; i < row_lanes / 64; ++i) top = max(top, tops[first_wave + i]);
  const float s = scale_of(__builtin_bit_cast(float, top)), inverse = 1.f / s;
  if (token < A.tokens) {
    if (own == 0) scales[token] = s;
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      const int d = (own + j * row_lanes) * rows::kChunk;
      if (d >= A.x_pitch) continue;
      unsigned code[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) code[i] = code_of<T>(words[j].get(i), s, inverse);
      *reinterpret_cast<rows::Bytes *>(codes + token * code_row + d) = rows::low_bytes(code);
    }
  }
  attention::tile_barrier();
  const int8_t *x_at = codes + min(c, A.tokens - 1) * code_row;
  i32x4 acc[1] = {};
  for (int first = wave; first < A.steps; first += kFewWaves * kDeep) {
    if (first != wave) fetch(first);
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int step = first + d * kFewWaves;
      i32x4 x = {0, 0, 0, 0};
      if (step < A.steps) x = *reinterpret_cast<const i32x4 *>(x_at + (step * 4 + q) * 16);
      acc[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d], x, acc[0], 0, 0, 0);
    }
  }
  finish_few<T, 1>(A, sums, acc, scales, w0, lane, wave);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int64_t code_pitch(int64_t width) { return (width + kPitch - 1) / kPitch * kPitch; }

template <typename T>
void launch_codes(const void *x, int64_t x_row, int64_t n, int width, int pitch, int8_t *codes,
                  float *scales, hipStream_t s) {
#define LINEAR8_CODES(kLanes, kChunks)                                                           \
  hipLaunchKernelGGL((codes_kernel<T, kLanes, kChunks>),                                         \
                     dim3(unsigned((n + 256 / kLanes - 1) / (256 / kLanes))), dim3(256), 0, s,   \
                     static_cast<const T *>(x), x_row, n, width, pitch, codes, scales)
  if (pitch <= 512)
    LINEAR8_CODES(64, 1);
  else if (pitch <= 1024)
    LINEAR8_CODES(64, 2);
  else if (pitch <= 2048)
    LINEAR8_CODES(64, 4);
  else if (pitch <= 8192)
    LINEAR8_CODES(256, 4);
  else
    LINEAR8_CODES(256, 0);
#undef LINEAR8_CODES
}

int codes_for(const void *x, int64_t x_row, int dtype, int64_t n, int width, int pitch, void *codes,
              void *scales, hipStream_t s) {
  // (a block takes four rows at most, and one at least)
  const int st = check_grid(pitch > 2048 ? n : (n + 3) / 4, 256, "linear8 codes");
  if (st) return st;
  LaunchScope scope("linear8_codes", s);
  int8_t *to = static_cast<int8_t *>(codes);
  float *scale = static_cast<float *>(scales);
  if (dtype == BEVPOOL_F32)
    launch_codes<float>(x, x_row, n, width, pitch, to, scale, s);
  else if (dtype == BEVPOOL_F16)
    launch_codes<_Float16>(x, x_row, n, width, pitch, to, scale, s);
  else
    launch_codes<__bf16>(x, x_row, n, width, pitch, to, scale, s);
  return check_launch("linear8_codes");
}

template <typename T, int kTx, int kTw, int kWavesX, int kWavesW, int kStep, int kBuffers,
          int kGroups = 1>
int launch_tiles(ProductArgs &A, hipStream_t s) {
  constexpr int kThreads = 64 * kWavesX * kWavesW * kGroups, kX = 32 * kTx * kWavesX, kW = 32 * kTw * kWavesW;
  A.x_tiles = (A.tokens + kX - 1) / kX;
  A.w_tiles = (A.channels + kW - 1) / kW;
  const int64_t blocks = (int64_t(A.x_tiles) * A.w_tiles + 7) / 8 * 8;
  const int st = check_grid(blocks, kThreads, "linear8");
  if (st) return st;
  hipLaunchKernelGGL((product_kernel<T, kTx, kTw, kWavesX, kWavesW, kStep, kBuffers, kGroups>),
                     dim3(unsigned(blocks)), dim3(kThreads),
                     kGroups * kBuffers * (kX + kW) * kStep + 2 * kW * sizeof(float), s, A);
  return check_launch("linear8");
}

// Lanes of a token where every block forms the codes itself; else 0.
int own_lanes(int64_t tokens, int pitch) {
  if (tokens > kOwnTokens) return 0;
  const int places = tokens > 4 ? 8 : tokens > 2 ? 4 : int(tokens);
  return places * pitch <= kOwnBytes ? kFewThreads / places : 0;
}

template <typename T, int kDeep>
int launch_token(const ProductArgs &A, const void *x, int64_t x_row, int width, int row_lanes,
                 hipStream_t s) {
  hipLaunchKernelGGL((token_kernel<T, kDeep>), dim3((A.channels + 15) / 16), dim3(kFewThreads), 0, s,
                     A, static_cast<const T *>(x), x_row, width, row_lanes);
  return check_launch("linear8");
}
template <typename T>
int launch_own(const ProductArgs &A, const void *x, int64_t x_row, int width, int row_lanes,
               hipStream_t s) {
  return A.steps > 4 * kFewWaves ? launch_token<T, 8>(A, x, x_row, width, row_lanes, s)
                                 : launch_token<T, 4>(A, x, x_row, width, row_lanes, s);
}

template <typename T, int kTx>
int launch_few(const ProductArgs &A, hipStream_t s) {
  hipLaunchKernelGGL((few_kernel<T, kTx>), dim3((A.channels + 15) / 16), dim3(kFewThreads), 0, s, A);
  return check_launch("linear8");
}

template <typename T>
int launch_product(ProductArgs &A, hipStream_t s) {
  auto tiles = [&](int x, int w) {
    return int64_t((A.tokens + x - 1) / x) * ((A.channels + w - 1) / w);
  };
  // Small tiles where few of larger ones would leave CUs idle, and the rows' length
  // in parts.  us of products by events:
  //   few tokens and channels: blocks of 16 channels; 1 x 32768 x 4096 34.5, by 32 x
  //   32 in four parts 37.2, 5 x 5000 x 300 7.6 and 8.7, but 24 x 4096 x 4096 (128
  //   tiles) 10.2 and 8.8, 32 x 8192 x 8192 25.2 and 17.0
  const int64_t least = tiles(32, 32);
  if (A.tokens <= 32 && least < 128)
    return A.tokens <= 16 ? launch_few<T, 1>(A, s) : launch_few<T, 2>(A, s);
  //   no more than CUs: 32 x 32 in four parts, then 64 x 32; 64 x 4096 x 4096 9.2 and
  //   9.9; 33 x 8192 x 8192 (512 and 256) 24.5 and 18.3, by 64 x 64 in two 22.9
  if (least <= 256) return launch_tiles<T, 1, 1, 1, 1, 128, 4, 4>(A, s);
  if (tiles(64, 32) <= 256) return launch_tiles<T, 1, 1, 2, 1, 128, 3, 4>(A, s);
  //   twice as many: 32 x 32 in three parts, two blocks a CU; 67 x 5000 x 4099 12.6, by
  //   64 x 64 in two 14.8, 33 x 8192 x 8192 20.3; always for up to 32 tokens, 32 x 4096
  //   x 20000 24.3 and by blocks of 32 channels as above 30.2; 48 x 1280 x 10240 10.4,
  //   by 64 x 64 in two 8.0
  if (A.tokens <= 32 || least <= 512) return launch_tiles<T, 1, 1, 1, 1, 128, 3, 3>(A, s);
  //   64 x 64 in two parts, 64 x 64 and 64 x 128: 200 x 4096 x 4096 12.8, 15.0 and 18.5;
  //   512 x 4096 x 4096 21.6, 18.7 and 20.3, 1024 x 1280 x 1280 12.1, 9.2 and 10.8; 800
  //   x 4096 x 4096 37.4, 30.3 and 24.0
  const int64_t small = tiles(64, 64);
  if (small <= 256) return launch_tiles<T, 1, 1, 2, 2, 128, 4, 2>(A, s);
  if (small <= 512) return launch_tiles<T, 1, 1, 2, 2, 128, 4>(A, s);
  // Larger tiles read operands less often, smaller ones leave less of a last round
  // and of a tile's edge empty: by what a round takes, 100 being 512 tiles of 128 x
  // 256, two a CU, and a last one of up to 256, one a CU, less.  us by 256 x 256, 128
  // x 256 and 64 x 128: 8192 x 8192 x 8192 487, 590; 1500 x 1280 x 10240 29, 33, 38;
  // 4000 x 4096 x 2500 59, 66, 66; 1024 x 4096 x 8192 56, 48, 53; 10325 x 1787 x 624
  // 33, 27, 29; 17223 x 5288 x 288 78, 83, 66; 7000 x 2560 x 1100 40, 43, 36.
  auto rounds = [&](int x, int w, int64_t each, int64_t full, int64_t last) {
    const int64_t n = tiles(x, w), rest = n % each;
    return n / each * full + (rest > 256 ? full : rest > 0 ? last : 0);
  };
  const int64_t large = rounds(256, 256, 256, 83, 83), middle = rounds(128, 256, 512, 100, 63);
  const int64_t little = rounds(64, 128, 512, 33, 29);
  if (large <= middle && large <= little) return launch_tiles<T, 4, 2, 2, 4, 128, 2>(A, s);
  if (middle <= little) return launch_tiles<T, 2, 4, 2, 2, 64, 3>(A, s);
  return launch_tiles<T, 1, 2, 2, 2, 128, 3>(A, s);
}

int check_sizes(int dtype, int64_t tokens, int64_t width, int64_t channels) {
  if (dtype < BEVPOOL_F32 || dtype > BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d", dtype);
  if (width < 1 || width > kMaxWidth)
    return fail(BEVPOOL_EINVAL, "width %lld: must be in [1, %d]", static_cast<long long>(width),
                kMaxWidth);
  if (tokens < 0 || tokens > (1 << 30) || channels < 0 || channels > (1 << 30))
    return fail(BEVPOOL_EINVAL, "bad number of tokens or channels");
  return BEVPOOL_OK;
}

}  // namespace

extern "C" {

int64_t bevpool_linear8_pitch(int32_t width) { return width < 1 ? 0 : code_pitch(width); }

int bevpool_linear8_codes(const void *x, int64_t x_row, int32_t dtype, int64_t rows, int32_t width,
                          void *codes, void *scales, void *stream) {
  bevpool_host::clear_error();
  int st = check_sizes(dtype, rows, width, 0);
  if (st) return st;
  if (rows == 0) return BEVPOOL_OK;
  if (!x || !codes || !scales) return fail(BEVPOOL_EINVAL, "null rows");
  return codes_for(x, x_row, dtype, rows, width, int(code_pitch(width)), codes, scales,
                   static_cast<hipStream_t>(stream));
}

size_t bevpool_linear8_scratch_bytes(int64_t tokens, int32_t width) {
  if (tokens < 1 || width < 1) return 0;
  return size_t(tokens) * size_t(code_pitch(width) + 4);
}

int bevpool_linear8(const void *x, int64_t x_row, int32_t dtype, const void *weight,
                    int64_t weight_row, const void *weight_scales, const void *bias, int64_t tokens,
                    int32_t width, int64_t channels, void *y, void *scratch, size_t scratch_bytes,
                    void *stream) {
  bevpool_host::clear_error();
  int st = check_sizes(dtype, tokens, width, channels);
  if (st) return st;
  if (tokens == 0 || channels == 0) return BEVPOOL_OK;
  if (!x || !weight || !weight_scales || !y) return fail(BEVPOOL_EINVAL, "null rows");
  if (reinterpret_cast<uintptr_t>(weight) % 16 || weight_row % 16 ||
      (channels > 1 && weight_row < (width + 15) / 16 * 16) || weight_row >= (int64_t(1) << 22))
    return fail(BEVPOOL_EINVAL,
                "weights: rows must start at multiples of 16 bytes, less than 4 MiB apart");
  if (!scratch || scratch_bytes < bevpool_linear8_scratch_bytes(tokens, width) ||
      reinterpret_cast<uintptr_t>(scratch) % 16)
    return fail(BEVPOOL_ESPACE, "linear8 scratch too small, or not at a multiple of 16 bytes");
  // (before anything is launched: the blocks of any plan of launch_product)
  st = tokens <= 32 ? check_grid((channels + 15) / 16, 64 * kFewWaves, "linear8")
                    : check_grid(((tokens + 63) / 64) * ((channels + 127) / 128), 256, "linear8");
  if (st) return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int pitch = int(code_pitch(width));
  int8_t *codes = static_cast<int8_t *>(scratch);
  float *scales = reinterpret_cast<float *>(codes + tokens * pitch);
  const int row_lanes = own_lanes(tokens, pitch);
  if (!row_lanes) {
    st = codes_for(x, x_row, dtype, tokens, width, pitch, codes, scales, s);
    if (st) return st;
  }
  ProductArgs A = {};
  A.x = codes;
  A.w = static_cast<const int8_t *>(weight);
  A.x_scale = scales;
  A.w_scale = static_cast<const float *>(weight_scales);
  A.bias = bias;
  A.y = y;
  A.w_row = weight_row;
  A.x_pitch = pitch;
  A.w_chunks = (width + 15) / 16;
  A.tokens = int(tokens);
  A.channels = int(channels);
  A.steps = pitch / 64;
  LaunchScope scope("linear8", s);
  if (row_lanes && dtype == BEVPOOL_F32) return launch_own<float>(A, x, x_row, width, row_lanes, s);
  if (row_lanes && dtype == BEVPOOL_F16)
    return launch_own<_Float16>(A, x, x_row, width, row_lanes, s);
  if (row_lanes) return launch_own<__bf16>(A, x, x_row, width, row_lanes, s);
  if (dtype == BEVPOOL_F32) return launch_product<float>(A, s);
  if (dtype == BEVPOOL_F16) return launch_product<_Float16>(A, s);
  return launch_product<__bf16>(A, s);
}

}  // extern "C"

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

constexpr int kStep = 128;           // bytes of a row that a tile holds
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

// rint(x / s), ties to even, for |x| <= 127 s: the product with the rounded
// 1 / s is off by less than 2^-15, so k is right or one off where x is next to
// a border; x - k s is exact.
__device__ __forceinline__ int code_of(float x, float s, float inverse) {
  const float k = rintf(x * inverse);
  const float d = 2.f * fmaf(-k, s, x);
  const int q = int(k);
  if (fabsf(d) > s || (fabsf(d) == s && (q & 1))) return d > 0.f ? q + 1 : q - 1;
  return q;
}

// A row of codes by kLanes lanes that hold it (kChunks chunks each), or, with
// kChunks 0, read it twice.
template <typename T, int kLanes, int kChunks>
__global__ __launch_bounds__(256) void codes_kernel(const T *x, int64_t x_row, int64_t n, int width,
                                                    int pitch, int8_t *codes, float *scales) {
  __shared__ float shared[4];
  constexpr int kHold = kChunks > 0 ? kChunks : 1;
  const int lane = int(threadIdx.x) % kLanes;
  const int64_t row = int64_t(blockIdx.x) * (256 / kLanes) + int(threadIdx.x) / kLanes;
  const bool on = row < n;  // (the same for a row's lanes)
  const T *at = x + (on ? row : 0) * x_row;
  const int chunks = kChunks > 0 ? kChunks : (pitch / 8 + kLanes - 1) / kLanes;
  float v[kHold][8], top = 0.f;
  bool finite = true;
  auto look = [&](const float (&c)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top = fmaxf(top, fabsf(c[i]));  // (passes over NaN)
      finite = finite && c[i] == c[i];
    }
  };
  for (int j = 0; j < chunks; ++j) {
    float(&c)[8] = v[kChunks > 0 ? j : 0];
    const int d = (lane + j * kLanes) * 8;
    rows::load(c, at + d, width - d);
    look(c);
  }
  if (!finite) top = __builtin_inff();
#pragma unroll
  for (int m = 1; m < (kLanes < 64 ? kLanes : 64); m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  if (kLanes > 64) {
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = top;
    __syncthreads();
    top = fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
  }
  if (!on) return;
  const float s = scale_of(top), inverse = 1.f / s;
  if (lane == 0) scales[row] = s;
  for (int j = 0; j < chunks; ++j) {
    float(&c)[8] = v[kChunks > 0 ? j : 0];
    const int d = (lane + j * kLanes) * 8;
    if (d >= pitch) continue;
    if (kChunks == 0) rows::load(c, at + d, width - d);
    unsigned q[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i / 4] |= (unsigned(code_of(c[i], s, inverse)) & 0xffu) << (i % 4 * 8);
    *reinterpret_cast<rows::Bytes *>(codes + row * pitch + d) = {q[0], q[1]};
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
  int steps;              // of kStep bytes
  int x_tiles, w_tiles;
};

// Rows of kStep bytes in LDS, 8 chunks of 16: chunk c of row r lies at c ^
// (r / 2) % 8, so the 16 rows of which a fragment read takes one chunk each
// use all of the 256 bytes that LDS gives a cycle.
__device__ __forceinline__ int place(int r, int c) { return c ^ ((r >> 1) & 7); }

// One block: kX tokens by kW channels, by waves of 32 kTx x 32 kTw.  Channels
// are the rows of the matrix instruction's result, tokens its columns: a lane
// holds one token's channels, four neighbours a register group.
template <typename T, int kX, int kW, int kTx, int kTw>
__global__ __launch_bounds__(64 * (kX / (32 * kTx)) * (kW / (32 * kTw))) void product_kernel(
    ProductArgs A) {
  constexpr int kThreads = 64 * (kX / (32 * kTx)) * (kW / (32 * kTw));
  constexpr int kWavesX = kX / (32 * kTx);
  constexpr int kLoadsX = kX * 8 / kThreads, kLoadsW = kW * 8 / kThreads;
  constexpr int kTileX = kX * kStep, kTile = (kX + kW) * kStep;
  extern __shared__ __align__(16) char lds[];
  const int lane = attention::lane_id(), wave = attention::wave_id();
  const int x0 = int(blockIdx.x % A.x_tiles) * kX, w0 = int(blockIdx.x / A.x_tiles) * kW;
  const unsigned lds0 = attention::lds_address(lds);
  // this lane's pieces of the tiles: offsets from the step's first byte
  const char *x_at = reinterpret_cast<const char *>(A.x) + int64_t(x0) * A.x_pitch;
  const char *w_at = reinterpret_cast<const char *>(A.w) + w0 * A.w_row;
  unsigned x_off[kLoadsX], w_off[kLoadsW];
  int w_chunk[kLoadsW];
#pragma unroll
  for (int i = 0; i < kLoadsX; ++i) {
    const int slot = i * kThreads + int(threadIdx.x), r = slot / 8, c = place(r, slot % 8);
    x_off[i] = unsigned(min(r, A.tokens - 1 - x0) * A.x_pitch + c * 16);
  }
#pragma unroll
  for (int i = 0; i < kLoadsW; ++i) {
    const int slot = i * kThreads + int(threadIdx.x), r = slot / 8;
    w_chunk[i] = place(r, slot % 8);
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
      const int c = min(step * 8 + w_chunk[i], A.w_chunks - 1);
      attention::load_to_lds(w_at, w_off[i] + c * 16, to + kTileX + i * kThreads * 16);
    }
  };
  i32x16 acc[kTw][kTx] = {};
  const int wx = wave % kWavesX * 32 * kTx, ww = wave / kWavesX * 32 * kTw;
  const int c = lane & 31, h = lane >> 5;
  load(0, 0);
  int buffer = 0;
  for (int step = 0; step < A.steps; ++step, buffer ^= 1) {
    attention::wait_loads<0>();
    __syncthreads();  // this step's tiles are there, and the last one's have been read
    if (step + 1 < A.steps) load(step + 1, buffer ^ 1);
    const char *x_tile = lds + buffer * kTile, *w_tile = x_tile + kTileX;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      i32x4 x[kTx], w[kTw];
#pragma unroll
      for (int i = 0; i < kTx; ++i)
        x[i] = *reinterpret_cast<const i32x4 *>(x_tile + (wx + 32 * i + c) * kStep +
                                                place(c, 2 * s + h) * 16);
#pragma unroll
      for (int i = 0; i < kTw; ++i)
        w[i] = *reinterpret_cast<const i32x4 *>(w_tile + (ww + 32 * i + c) * kStep +
                                                place(c, 2 * s + h) * 16);
#pragma unroll
      for (int i = 0; i < kTw; ++i)
#pragma unroll
        for (int j = 0; j < kTx; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[i], x[j], acc[i][j], 0, 0, 0);
    }
  }
  const T *bias = static_cast<const T *>(A.bias);
#pragma unroll
  for (int j = 0; j < kTx; ++j) {
    const int token = x0 + wx + 32 * j + c;
    if (token >= A.tokens) continue;
    const float by = A.x_scale[token];
    T *y = static_cast<T *>(A.y) + int64_t(token) * A.channels;
#pragma unroll
    for (int i = 0; i < kTw; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = w0 + ww + 32 * i + attention::c_row(r, h);
        if (n < A.channels)
          y[n] = T(float(acc[i][j][r]) * by * A.w_scale[n] + (bias ? float(bias[n]) : 0.f));
      }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int64_t code_pitch(int64_t width) { return (width + kStep - 1) / kStep * kStep; }

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

template <typename T>
int launch_product(ProductArgs &A, hipStream_t s) {
  constexpr int kX = 128, kW = 128;
  A.x_tiles = (A.tokens + kX - 1) / kX;
  A.w_tiles = (A.channels + kW - 1) / kW;
  const int64_t blocks = int64_t(A.x_tiles) * A.w_tiles;
  const int st = check_grid(blocks, 256, "linear8");
  if (st) return st;
  hipLaunchKernelGGL((product_kernel<T, kX, kW, 2, 2>), dim3(unsigned(blocks)), dim3(256),
                     2 * (kX + kW) * kStep, s, A);
  return check_launch("linear8");
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int pitch = int(code_pitch(width));
  int8_t *codes = static_cast<int8_t *>(scratch);
  float *scales = reinterpret_cast<float *>(codes + tokens * pitch);
  st = codes_for(x, x_row, dtype, tokens, width, pitch, codes, scales, s);
  if (st) return st;
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
  A.steps = pitch / kStep;
  LaunchScope scope("linear8", s);
  if (dtype == BEVPOOL_F32) return launch_product<float>(A, s);
  if (dtype == BEVPOOL_F16) return launch_product<_Float16>(A, s);
  return launch_product<__bf16>(A, s);
}

}  // extern "C"

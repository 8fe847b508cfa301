// gated.hip -- the gated activation of a block's hidden values, forward and
// backward, and 8-bit checkpoints of rows (gfx950).
//
//   y = act(a) b,   a the first half of a row, b the second
//   da = dy b act'(a),  db = dy act(a)
// act: silu a s(a), gelu a Phi(a), sigmoid s(a), with s(a) = 1 / (1 + exp(-a))
// and Phi the normal distribution's integral.  The backward pass takes a and b
// as they were, or their 8-bit checkpoints, which the forward writes beside y.
//
// Bound by memory: everything read and written once.  16,896 rows of 2 x 5,120
// in bf16: forward with the checkpoints 121 us, backward from them 125 us (5.8 and
// 5.6 TB/s of what has to move; a large copy reaches 5.1), without 94 and 146 us;
// 4,097 rows of 2 x 1,031 in fp32 13 and 18 us.  A checkpoint of 16,896 x 1,280
// in bf16 12 us, and back 13.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bevpool.h"
#include "host_calls.h"
#include "rows.h"

namespace {

using bevpool_host::check_grid;
using bevpool_host::check_launch;
using bevpool_host::fail;
using bevpool_host::LaunchScope;

constexpr int kThreads = 256;
constexpr int kMaxWidth = 1 << 18;

enum Act { kSilu, kGelu, kSigmoid };

// (16-bit results: the hardware's exponential and reciprocal, good to 2 units
// of fp32; fp32 results: the correctly rounded quotient and the exact one)
template <typename T>
__device__ __forceinline__ float exp_of(float x) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f);
  return expf(x);
}
template <typename T>
__device__ __forceinline__ float inverse_of(float x) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(x);
  return 1.0f / x;
}

// The normal distribution's integral up to -z, without its factor exp(-z^2 /
// 2), z >= 0: a polynomial in t = 1 / (1 + 0.3 z), fitted to 0.5 erfcx(z /
// sqrt(2)) / t on z in [0, 15] with the least largest relative error (2e-7; 5e-7
// as it is evaluated in fp32), past which the factor is zero.  For 16-bit
// results; forward and backward of 16,896 x 5,120 hidden values with it and with
// the library's erfc: 143 and 134 us,
// and 178 and 222.
__device__ __forceinline__ float normal_tail(float z) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, z, 1.f));
  float p = 0.03517865762114525f;
  p = fmaf(p, t, -0.15514202415943146f);
  p = fmaf(p, t, 0.2028157114982605f);
  p = fmaf(p, t, -0.05044356361031532f);
  p = fmaf(p, t, 0.12685833871364594f);
  p = fmaf(p, t, 0.10042549669742584f);
  p = fmaf(p, t, 0.12067274749279022f);
  p = fmaf(p, t, 0.11963453143835068f);
  return p * t;
}

// The function at a and its slope there.
template <typename T, int kAct>
__device__ __forceinline__ void activate(float a, float &y, float &slope) {
  if constexpr (kAct == kGelu) {
    const float e = exp_of<T>(-0.5f * a * a);
    float p;
    if constexpr (sizeof(T) == 2) {
      p = normal_tail(fabsf(a)) * e;
      if (a > 0.f) p = 1.f - p;
    } else {
      p = 0.5f * erfcf(a * -0.70710678118654752440f);
    }
    y = a * p;
    slope = p + a * (0.39894228040143267794f * e);
  } else {
    // from exp(-|a|), which neither overflows nor cancels
    const float e = exp_of<T>(-fabsf(a)), s = inverse_of<T>(1.f + e), t = e * s;
    const float p = a < 0.f ? t : s, q = a < 0.f ? s : t;  // s(a), s(-a)
    y = kAct == kSilu ? a * p : p;
    slope = kAct == kSilu ? p + a * (p * q) : p * q;
  }
}

// A launch's chunks, row after row, four of every block of 32 values: `each`
// a row, one a thread.  (More of them a thread, their loads together, are
// slower: backward of 16,896 x 5,120 hidden values 131 us by one, 171 by two, 219
// by four.)  A block's first is divided in 64 bits, the others' offsets from it
// by a multiplication (each <= 2^15, so offset * each < 2^32).
struct Chunks {
  int64_t rows;
  unsigned each, inverse;  // inverse: ceil(2^32 / each)
  int width;
};
struct At {
  int64_t row;
  int chunk, left;  // left: values from the chunk's first to the row's end
  bool on;
};
__device__ __forceinline__ At chunk_of(const Chunks &C) {
  const int64_t first = int64_t(blockIdx.x) * kThreads;
  const int64_t row = first / C.each;
  const unsigned i = unsigned(first - row * C.each) + threadIdx.x;
  const unsigned down = __umulhi(i, C.inverse);
  At at;
  at.row = row + down;
  at.chunk = int(i - down * C.each);
  at.on = at.row < C.rows;
  at.left = at.on ? C.width - at.chunk * rows::kChunk : 0;
  return at;
}

struct GatedArgs {
  Chunks c;
  const void *x, *dout;
  int64_t x_row, dout_row;
  uint8_t *kept;
  void *out, *dx;
};

template <typename T, int kAct, bool kKeep>
__global__ __launch_bounds__(kThreads) void gated_kernel(GatedArgs A) {
  const At at = chunk_of(A.c);
  const int width = A.c.width, begin = at.chunk * rows::kChunk;
  const T *x = static_cast<const T *>(A.x) + at.row * A.x_row + begin;
  rows::Words<T> aw, bw;
  aw.load(x, at.left);
  bw.load(x + width, at.left);
  float a[8], b[8], y[8], slope;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = aw.get(i);
    b[i] = bw.get(i);
    activate<T, kAct>(a[i], y[i], slope);
    y[i] *= b[i];
  }
  rows::store(static_cast<T *>(A.out) + at.row * width + begin, y, at.left);
  if (kKeep && at.on) {  // (whole blocks of 32 values)
    const int64_t pitch = rows::checkpoint_pitch(width), blocks = rows::blocks_of(width);
    uint8_t *kept = A.kept + at.row * 2 * pitch;
    rows::store_packed(kept, at.chunk, blocks, a);
    rows::store_packed(kept + pitch, at.chunk, blocks, b);
  }
}

template <typename T, int kAct, bool kKept>
__global__ __launch_bounds__(kThreads) void gated_backward_kernel(GatedArgs A) {
  const At at = chunk_of(A.c);
  const int width = A.c.width, begin = at.chunk * rows::kChunk;
  float a[8], b[8];
  rows::Words<T> g;
  g.load(static_cast<const T *>(A.dout) + at.row * A.dout_row + begin, at.left);
  if constexpr (kKept) {
    rows::PackedChunk ap, bp;
    if (at.left > 0) {
      const int64_t pitch = rows::checkpoint_pitch(width), blocks = rows::blocks_of(width);
      const uint8_t *kept = A.kept + at.row * 2 * pitch;
      ap.load(kept, at.chunk, blocks);
      bp.load(kept + pitch, at.chunk, blocks);
    }
    ap.template get<T>(a);
    bp.template get<T>(b);
  } else {
    const T *x = static_cast<const T *>(A.x) + at.row * A.x_row + begin;
    rows::Words<T> aw, bw;
    aw.load(x, at.left);
    bw.load(x + width, at.left);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = aw.get(i);
      b[i] = bw.get(i);
    }
  }
  float da[8], db[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float y, slope;
    activate<T, kAct>(a[i], y, slope);
    da[i] = g.get(i) * b[i] * slope;
    db[i] = g.get(i) * y;
  }
  T *dx = static_cast<T *>(A.dx) + at.row * 2 * width + begin;
  rows::store(dx, da, at.left);
  rows::store(dx + width, db, at.left);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pack_kernel(Chunks C, const T *x, int64_t x_row,
                                                        uint8_t *kept) {
  const At at = chunk_of(C);
  if (!at.on) return;  // (whole blocks of 32 values)
  float v[8];
  rows::load(v, x + at.row * x_row + at.chunk * rows::kChunk, at.left);
  rows::store_packed(kept + at.row * rows::checkpoint_pitch(C.width), at.chunk,
                     rows::blocks_of(C.width), v);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack_kernel(Chunks C, const uint8_t *kept, T *out) {
  const At at = chunk_of(C);
  if (at.left <= 0) return;
  rows::PackedChunk chunk;
  chunk.load(kept + at.row * rows::checkpoint_pitch(C.width), at.chunk, rows::blocks_of(C.width));
  float v[8];
  chunk.template get<T>(v);
  rows::store(out + at.row * C.width + at.chunk * rows::kChunk, v, at.left);
}

int check_chunks(Chunks &C, unsigned &grid, int dtype, int64_t rows, int width, const char *what) {
  if (dtype < BEVPOOL_F32 || dtype > BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d", dtype);
  if (rows < 0 || rows > (int64_t(1) << 40)) return fail(BEVPOOL_EINVAL, "bad number of rows");
  if (width < 1 || width > kMaxWidth)
    return fail(BEVPOOL_EINVAL, "width %d: must be in [1, %d]", width, kMaxWidth);
  C.rows = rows;
  C.width = width;
  C.each = unsigned(rows::blocks_of(width) * (rows::kBlock / rows::kChunk));
  C.inverse = unsigned(((uint64_t(1) << 32) + C.each - 1) / C.each);
  const int64_t blocks = (rows * C.each + kThreads - 1) / kThreads;
  grid = unsigned(blocks);
  return check_grid(blocks, kThreads, what);
}

template <typename T, int kAct>
void launch_gated(const GatedArgs &A, unsigned grid, bool backward, hipStream_t s) {
  const dim3 g(grid), t(kThreads);
  if (backward && A.kept)
    hipLaunchKernelGGL((gated_backward_kernel<T, kAct, true>), g, t, 0, s, A);
  else if (backward)
    hipLaunchKernelGGL((gated_backward_kernel<T, kAct, false>), g, t, 0, s, A);
  else if (A.kept)
    hipLaunchKernelGGL((gated_kernel<T, kAct, true>), g, t, 0, s, A);
  else
    hipLaunchKernelGGL((gated_kernel<T, kAct, false>), g, t, 0, s, A);
}

template <typename T>
void launch_act(const GatedArgs &A, int act, unsigned grid, bool backward, hipStream_t s) {
  if (act == kSilu)
    launch_gated<T, kSilu>(A, grid, backward, s);
  else if (act == kGelu)
    launch_gated<T, kGelu>(A, grid, backward, s);
  else
    launch_gated<T, kSigmoid>(A, grid, backward, s);
}

int launch_type(const GatedArgs &A, int dtype, int act, unsigned grid, bool backward,
                hipStream_t s) {
  const char *what = backward ? "gated_backward" : "gated";
  LaunchScope scope(what, s);
  if (dtype == BEVPOOL_F32)
    launch_act<float>(A, act, grid, backward, s);
  else if (dtype == BEVPOOL_F16)
    launch_act<_Float16>(A, act, grid, backward, s);
  else
    launch_act<__bf16>(A, act, grid, backward, s);
  return check_launch(what);
}

}  // namespace

extern "C" {

int bevpool_gated_forward(const void *x, int64_t x_row, int32_t dtype, int64_t rows, int32_t width,
                          int32_t act, void *out, void *kept, void *stream) {
  bevpool_host::clear_error();
  GatedArgs A = {};
  unsigned grid;
  const int st = check_chunks(A.c, grid, dtype, rows, width, "gated");
  if (st) return st;
  if (act < kSilu || act > kSigmoid) return fail(BEVPOOL_EINVAL, "unknown activation %d", act);
  if (rows == 0) return BEVPOOL_OK;
  if (!x || !out) return fail(BEVPOOL_EINVAL, "null rows");
  A.x = x;
  A.x_row = x_row;
  A.out = out;
  A.kept = static_cast<uint8_t *>(kept);
  return launch_type(A, dtype, act, grid, false, static_cast<hipStream_t>(stream));
}

int bevpool_gated_backward(const void *x, int64_t x_row, int32_t kept, const void *dout,
                           int64_t dout_row, int32_t dtype, int64_t rows, int32_t width,
                           int32_t act, void *dx, void *stream) {
  bevpool_host::clear_error();
  GatedArgs A = {};
  unsigned grid;
  const int st = check_chunks(A.c, grid, dtype, rows, width, "gated backward");
  if (st) return st;
  if (act < kSilu || act > kSigmoid) return fail(BEVPOOL_EINVAL, "unknown activation %d", act);
  if (rows == 0) return BEVPOOL_OK;
  if (!x || !dout || !dx) return fail(BEVPOOL_EINVAL, "null rows");
  A.x = x;
  A.x_row = x_row;
  A.kept = kept ? static_cast<uint8_t *>(const_cast<void *>(x)) : nullptr;
  A.dout = dout;
  A.dout_row = dout_row;
  A.dx = dx;
  return launch_type(A, dtype, act, grid, true, static_cast<hipStream_t>(stream));
}

int bevpool_checkpoint_pack(const void *x, int64_t x_row, int32_t dtype, int64_t rows,
                            int32_t width, void *kept, void *stream) {
  bevpool_host::clear_error();
  Chunks C = {};
  unsigned grid;
  const int st = check_chunks(C, grid, dtype, rows, width, "checkpoint pack");
  if (st) return st;
  if (rows == 0) return BEVPOOL_OK;
  if (!x || !kept) return fail(BEVPOOL_EINVAL, "null rows");
  hipStream_t s = static_cast<hipStream_t>(stream);
  LaunchScope scope("checkpoint_pack", s);
  uint8_t *to = static_cast<uint8_t *>(kept);
  if (dtype == BEVPOOL_F32)
    hipLaunchKernelGGL((pack_kernel<float>), dim3(grid), dim3(kThreads), 0, s, C,
                       static_cast<const float *>(x), x_row, to);
  else if (dtype == BEVPOOL_F16)
    hipLaunchKernelGGL((pack_kernel<_Float16>), dim3(grid), dim3(kThreads), 0, s, C,
                       static_cast<const _Float16 *>(x), x_row, to);
  else
    hipLaunchKernelGGL((pack_kernel<__bf16>), dim3(grid), dim3(kThreads), 0, s, C,
                       static_cast<const __bf16 *>(x), x_row, to);
  return check_launch("checkpoint_pack");
}

int bevpool_checkpoint_unpack(const void *kept, int32_t dtype, int64_t rows, int32_t width,
                              void *out, void *stream) {
  bevpool_host::clear_error();
  Chunks C = {};
  unsigned grid;
  const int st = check_chunks(C, grid, dtype, rows, width, "checkpoint unpack");
  if (st) return st;
  if (rows == 0) return BEVPOOL_OK;
  if (!kept || !out) return fail(BEVPOOL_EINVAL, "null rows");
  hipStream_t s = static_cast<hipStream_t>(stream);
  LaunchScope scope("checkpoint_unpack", s);
  const uint8_t *from = static_cast<const uint8_t *>(kept);
  if (dtype == BEVPOOL_F32)
    hipLaunchKernelGGL((unpack_kernel<float>), dim3(grid), dim3(kThreads), 0, s, C, from,
                       static_cast<float *>(out));
  else if (dtype == BEVPOOL_F16)
    hipLaunchKernelGGL((unpack_kernel<_Float16>), dim3(grid), dim3(kThreads), 0, s, C, from,
                       static_cast<_Float16 *>(out));
  else
    hipLaunchKernelGGL((unpack_kernel<__bf16>), dim3(grid), dim3(kThreads), 0, s, C, from,
                       static_cast<__bf16 *>(out));
  return check_launch("checkpoint_unpack");
}

}  // extern "C"

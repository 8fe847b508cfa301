// weight_grad.hip -- the gradient of a linear layer's weight from the 8-bit
// checkpoint of its input, and of its bias (gfx950).
//
//   dW[n][k] = sum over tokens t of dy[t][n] x[t][k],   db[n] = sum of dy[t][n]
// x is what the checkpoint stands for: numbers of 7 bits times a power of two,
// exact in the operands' type, so the products are those of the type's matrix
// instructions and only their sums are rounded, in fp32.
//
// A block takes 256 x 256 of dW and a part of the tokens, 32 at a time: rows of
// dy go to LDS as they are, bytes of x through LDS and registers, where they
// become numbers of the type, to a tile of their own.  Both tiles have tokens as
// rows and are read transposed.  The parts' sums are joined in their order.
//
// Bound by the products beside what they wait for (the matrix instructions are
// busy in 38% of the cycles, LDS in 25%): 16,896 tokens of 1,280 x 1,280 in bf16
// 75 us (740 TFLOP/s) and 11 for the parts, 4,096 of 4,096 x 4,096 810 TFLOP/s.
// The bytes' way to numbers beside the products took 8 us of the first; blocks
// of 256 x 128, two a CU, 82 us.
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

constexpr int kThreads = 256;            // (join and sums)
constexpr int kGradThreads = 512;        // eight waves of 128 x 64
constexpr int kSide = 256;               // a block's part of dW, both ways
constexpr int kTokens = 32;              // of a step
constexpr int kHalf = kTokens * 256;     // bytes of 128 columns
constexpr int kTile = 2 * kHalf;         // of 256
constexpr int kScales = kTokens * kSide; // where the scales of x's bytes begin
constexpr int kRaw = kScales + kTokens * 8;
constexpr int kLds = 4 * kTile + 2 * kTile + 3 * kRaw;

struct GradArgs {
  const char *dy;
  int64_t dy_row;       // bytes
  const uint8_t *kept;
  int64_t pitch;
  float *parts;         // [parts][n][k]
  int64_t tokens, share;  // share: tokens of a part, whole steps
  int n, k, blocks;     // blocks: of 32 values in a row of the checkpoint
  int n_tiles, k_tiles, n_parts;
};

template <typename T>
__global__ __launch_bounds__(kGradThreads, 2) void weight_grad_kernel(GradArgs A) {
  extern __shared__ __align__(16) char lds[];
  char *const x_lds = lds + 4 * kTile, *const raw_lds = x_lds + 2 * kTile;
  // blocks of one XCD (every eighth) take parts of the tokens that lie together,
  // all tiles of one part before the next: they read the same rows at the same time
  const int tiles = A.n_tiles * A.k_tiles, total = tiles * A.n_parts, each = (total + 7) / 8;
  const int id = int(blockIdx.x % 8) * each + int(blockIdx.x / 8);
  if (int(blockIdx.x / 8) >= each || id >= total) return;
  const int part = id / tiles, tile = id - part * tiles;
  const int n0 = tile / A.k_tiles * kSide, k0 = tile % A.k_tiles * kSide;
  const int64_t begin = part * A.share, end = min(begin + A.share, A.tokens);
  const int steps = int((end - begin + kTokens - 1) / kTokens);
  const int lane = attention::lane_id(), wave = attention::wave_id();
  const unsigned lds0 = attention::lds_address(lds), raw0 = attention::lds_address(raw_lds);

  // this lane's pieces of a step: two chunks of dy, one of x's bytes and, for
  // eight lanes of a wave, the scales of the four rows that the wave converts
  int dy_r[2];
  unsigned dy_off[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int in = int(threadIdx.x);  // (the tile's half i)
    dy_r[i] = in / 16;
    const int chunk = in % 16 ^ attention::swizzle<T, 128>(dy_r[i]);
    const int col = min(n0 + i * 128 + chunk * 8, A.n - 8);  // (past n: not stored)
    dy_off[i] = unsigned(dy_r[i] * int(A.dy_row) + col * 2);
  }
  const int raw_r = int(threadIdx.x) / 16, raw_c = int(threadIdx.x) % 16;
  const unsigned raw_off = unsigned(raw_r * int(A.pitch) + min(k0 + raw_c * 16, A.blocks * 32 - 16));
  const int scale_r = wave * 4 + (lane & 7) / 2;
  const unsigned scale_off =
      unsigned(scale_r * int(A.pitch) + A.blocks * 32 + k0 / 32 + lane % 2 * 4);

  auto load = [&](int step) {
    const int64_t t0 = begin + int64_t(step) * kTokens;
    const int rows = int(min(int64_t(kTokens), end - t0));
    const char *dy = A.dy + t0 * A.dy_row;
    const char *kept = reinterpret_cast<const char *>(A.kept) + t0 * A.pitch;
    const unsigned to = lds0 + step % 4 * kTile + wave * 1024, raw = raw0 + step % 3 * kRaw;
    if (rows == kTokens) {
      attention::load_to_lds(dy, dy_off[0], to);
      attention::load_to_lds(dy, dy_off[1], to + kHalf);
      attention::load_to_lds(kept, raw_off, raw + wave * 1024);
      if (lane < 8) attention::load_to_lds4(kept, scale_off, raw + kScales + wave * 32);
    } else {  // (rows past the part: zeros)
      const attention::u32x4 zero = {0, 0, 0, 0};
      const unsigned none = 0x80808080u;
      char *at = lds + step % 4 * kTile + int(threadIdx.x) * 16, *raw_at = raw_lds + step % 3 * kRaw;
      if (raw_r < rows) {  // (dy's row of a lane is that of its bytes)
        attention::load_to_lds(dy, dy_off[0], to);
        attention::load_to_lds(dy, dy_off[1], to + kHalf);
        attention::load_to_lds(kept, raw_off, raw + wave * 1024);
      } else {
        *reinterpret_cast<attention::u32x4 *>(at) = zero;
        *reinterpret_cast<attention::u32x4 *>(at + kHalf) = zero;
        *reinterpret_cast<attention::u32x4 *>(raw_at + int(threadIdx.x) * 16) =
            attention::u32x4{none, none, none, none};
      }
      if (lane < 8) {
        if (scale_r < rows)
          attention::load_to_lds4(kept, scale_off, raw + kScales + wave * 32);
        else
          *reinterpret_cast<unsigned *>(raw_at + kScales + wave * 32 + lane * 4) = 0x01010101u;
      }
    }
  };
  // bytes of x (of this lane's own load) as numbers.  Without a branch, so that
  // it runs beside the products: what is not finite, and the largest scale, whose
  // 128 times is infinite, are left to mend().
  struct Numbers {
    attention::u32x4 bytes;
    unsigned scale;
    rows::Words<T> words[2];
  };
  auto fetch = [&](int step, Numbers &x) {
    const char *raw = raw_lds + step % 3 * kRaw;
    x.bytes = *reinterpret_cast<const attention::u32x4 *>(raw + int(threadIdx.x) * 16);
    const unsigned scales =
        *reinterpret_cast<const unsigned *>(raw + kScales + (raw_r * 2 + raw_c / 8) * 4);
    x.scale = scales >> (raw_c % 8 / 2 * 8) & 0xffu;
  };
  auto convert = [&](Numbers &x) {
    const float by = rows::power(x.scale), less = -128.f * by;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = fmaf(float(x.bytes[2 * i + j / 4] >> (j % 4 * 8) & 0xffu), by, less);
      // (64 2^10 stands for the largest numbers of fp16, and is none)
      if constexpr (__is_same(T, _Float16))
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __builtin_amdgcn_fmed3f(v[j], -65504.f, 65504.f);
      x.words[i].set(v);
    }
  };
  auto mend = [&](Numbers &x) {
    auto zero = [](unsigned b) { return (b - 0x01010101u) & ~b & 0x80808080u; };
    if ((zero(x.bytes[0]) | zero(x.bytes[1]) | zero(x.bytes[2]) | zero(x.bytes[3])) == 0 &&
        x.scale < 248)
      return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float v[8];
      rows::unpack<T>(v, rows::Bytes{x.bytes[2 * i], x.bytes[2 * i + 1]}, x.scale);
      x.words[i].set(v);
    }
  };
  auto put = [&](int step, const Numbers &x) {
    char *to = x_lds + step % 2 * kTile + raw_c / 8 * kHalf + raw_r * 256;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<rows::Words<T> *>(
          to + ((2 * (raw_c % 8) + i) ^ attention::swizzle<T, 128>(raw_r)) * 16) = x.words[i];
  };

  const int wn = wave / 4, wk = wave % 4;
  attention::f32x16 acc[4][2] = {};
  Numbers x;
  load(0);
  if (steps > 1) load(1);
  if (steps > 2) load(2);
  attention::wait_loads<0>();
  fetch(0, x);
  convert(x);
  mend(x);
  put(0, x);
  attention::tile_barrier();
  for (int step = 0; step < steps; ++step) {
    // there: both tiles of this step, this wave's bytes of the next
    if (step + 3 < steps) load(step + 3);
    attention::Piece<T> b, a0, a1;
    attention::read_column_piece<T, 128>(b, x_lds + step % 2 * kTile + wk / 2 * kHalf, 0,
                                         2 * (wk % 2), lane);
    const char *dy_tile = lds + step % 4 * kTile + wn * kHalf;
    attention::read_column_piece<T, 128>(a0, dy_tile, 0, 0, lane);
    attention::read_column_piece<T, 128>(a1, dy_tile, 0, 2, lane);
    fetch(step + 1, x);  // (behind the last step: what is there, which nothing reads)
    __builtin_amdgcn_sched_barrier(0);
    convert(x);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          acc[p][q] = attention::Mat<T>::mma(p < 2 ? a0[2 * p + j] : a1[2 * p - 4 + j],
                                             b[2 * q + j], acc[p][q]);
    // a few of the conversion's instructions behind each product
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (step + 1 < steps) {
      mend(x);
      put(step + 1, x);
      // the loads of the step behind it have arrived: all but those of the third
      // (the last step's may be fewer)
      if (step + 3 < steps - 1)
        attention::wait_loads<4>();
      else
        attention::wait_loads<0>();
    }
    attention::tile_barrier();  // tiles of the next step are there, this one's have been read
  }
  float *out = A.parts + int64_t(part) * A.n * A.k;
  const int c = lane & 31, h = lane >> 5;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int k = k0 + wk * 64 + q * 32 + c;
    if (k >= A.k) continue;
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = n0 + wn * 128 + p * 32 + attention::c_row(r, h);
        if (n < A.n) out[int64_t(n) * A.k + k] = acc[p][q][r];
      }
  }
}

// Sums of the parts, in their order.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(const float *parts, int n_parts,
                                                        int64_t values, T *out) {
  const int64_t i = (int64_t(blockIdx.x) * kThreads + threadIdx.x) * rows::kChunk;
  if (i >= values) return;  // (whole chunks: n is a multiple of 8)
  float sum[8] = {};
#pragma unroll 4
  for (int p = 0; p < n_parts; ++p) {
    const float *at = parts + p * values + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] += at[j];
  }
  rows::store(out + i, sum, 8);
}

// ---------------------------------------------------------------------------
// sums of columns
// ---------------------------------------------------------------------------

constexpr int kColumns = 64, kRowsAtOnce = kThreads / kColumns, kColumnParts = 256;

template <typename From, typename To>
__global__ __launch_bounds__(kThreads) void column_sum_kernel(const From *x, int64_t x_row,
                                                              int64_t n_rows, int width, To *out) {
  __shared__ float lds[kThreads];
  const int c = int(blockIdx.x) * kColumns + int(threadIdx.x) % kColumns;
  const int64_t share = (n_rows + gridDim.y - 1) / gridDim.y, begin = blockIdx.y * share;
  const int64_t end = min(begin + share, n_rows);
  float s = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int64_t r = begin + threadIdx.x / kColumns; r < end; r += kRowsAtOnce)
      s += float(x[r * x_row + c]);
  }
  lds[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x >= kColumns || c >= width) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < kRowsAtOnce; ++i) s += lds[i * kColumns + threadIdx.x];
  out[int64_t(blockIdx.y) * width + c] = To(s);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

struct Split {
  int64_t share;
  int parts, n_tiles, k_tiles;
};

// Parts of the tokens: one block a CU together, each of eight steps at least.
Split split_for(int64_t tokens, int n, int k) {
  Split s;
  s.n_tiles = (n + kSide - 1) / kSide;
  s.k_tiles = (k + kSide - 1) / kSide;
  const int64_t tiles = int64_t(s.n_tiles) * s.k_tiles;
  const int64_t steps = (tokens + kTokens - 1) / kTokens;
  int64_t parts = 256 / tiles;
  if (parts > steps / 8) parts = steps / 8;
  if (parts < 1) parts = 1;
  const int64_t each = (steps + parts - 1) / parts;
  s.share = each * kTokens;
  s.parts = int((steps + each - 1) / each);
  return s;
}

template <typename T>
int launch(const GradArgs &A, T *dweight, hipStream_t s) {
  const int64_t total = int64_t(A.n_tiles) * A.k_tiles * A.n_parts;
  const int64_t grid = (total + 7) / 8 * 8, values = int64_t(A.n) * A.k;
  const int64_t join = (values / rows::kChunk + kThreads - 1) / kThreads;
  int st = check_grid(grid, kGradThreads, "weight_grad");
  if (!st) st = check_grid(join, kThreads, "weight_grad");
  if (st) return st;
  {
    LaunchScope scope("weight_grad", s);
    hipLaunchKernelGGL((weight_grad_kernel<T>), dim3(unsigned(grid)), dim3(kGradThreads), kLds, s, A);
    st = check_launch("weight_grad");
    if (st) return st;
  }
  LaunchScope scope("weight_grad_join", s);
  hipLaunchKernelGGL((join_kernel<T>), dim3(unsigned(join)), dim3(kThreads), 0, s, A.parts,
                     A.n_parts, values, dweight);
  return check_launch("weight_grad_join");
}

template <typename T>
int launch_columns(const void *x, int64_t x_row, int64_t n_rows, int width, void *out,
                   float *scratch, hipStream_t s) {
  // Parts of 32 rows at least: us of both by events, 300 x 1280 9.3, by 256 parts
  // 11 to 16, 86 x 3577 9.0 and 15.
  const int64_t some = (n_rows + 31) / 32;
  const int64_t parts = some < 1 ? 1 : some < kColumnParts ? some : kColumnParts;
  const dim3 grid((width + kColumns - 1) / kColumns, unsigned(parts));
  const int st = check_grid(int64_t(grid.x) * kColumnParts, kThreads, "column_sums");
  if (st) return st;
  LaunchScope scope("column_sums", s);
  hipLaunchKernelGGL((column_sum_kernel<T, float>), grid, dim3(kThreads), 0, s,
                     static_cast<const T *>(x), x_row, n_rows, width, scratch);
  hipLaunchKernelGGL((column_sum_kernel<float, T>), dim3(grid.x, 1), dim3(kThreads), 0, s, scratch,
                     int64_t(width), parts, width, static_cast<T *>(out));
  return check_launch("column_sums");
}

}  // namespace

extern "C" {

size_t bevpool_checkpoint_weight_grad_scratch_bytes(int64_t tokens, int32_t n, int32_t k) {
  if (tokens < 1 || n < 1 || k < 1) return 0;
  return size_t(split_for(tokens, n, k).parts) * size_t(n) * size_t(k) * sizeof(float);
}

int bevpool_checkpoint_weight_grad(const void *dy, int64_t dy_row, const void *kept, int32_t dtype,
                                   int64_t tokens, int32_t n, int32_t k, void *dweight,
                                   void *scratch, size_t scratch_bytes, void *stream) {
  bevpool_host::clear_error();
  if (dtype != BEVPOOL_F16 && dtype != BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d: 16-bit types", dtype);
  if (tokens < 1 || tokens > (int64_t(1) << 40)) return fail(BEVPOOL_EINVAL, "bad number of tokens");
  if (n < 8 || n % 8 || n > (1 << 20) || k < 1 || k > (1 << 18))
    return fail(BEVPOOL_EINVAL, "weights of %d x %d: the first a multiple of 8, at most 2^20, the "
                "other at most 2^18", n, k);
  if (!dy || !kept || !dweight) return fail(BEVPOOL_EINVAL, "null rows");
  if (reinterpret_cast<uintptr_t>(dy) % 16 || dy_row % 8 || dy_row < 0 || dy_row >= (1 << 24) ||
      reinterpret_cast<uintptr_t>(kept) % 16)
    return fail(BEVPOOL_EINVAL, "rows must start at multiples of 16 bytes, less than 32 MiB apart");
  if (!scratch || scratch_bytes < bevpool_checkpoint_weight_grad_scratch_bytes(tokens, n, k))
    return fail(BEVPOOL_ESPACE, "weight gradient scratch too small");
  const Split split = split_for(tokens, n, k);
  GradArgs A = {};
  A.dy = static_cast<const char *>(dy);
  A.dy_row = dy_row * 2;
  A.kept = static_cast<const uint8_t *>(kept);
  A.pitch = rows::checkpoint_pitch(k);
  A.parts = static_cast<float *>(scratch);
  A.tokens = tokens;
  A.share = split.share;
  A.n = n;
  A.k = k;
  A.blocks = int(rows::blocks_of(k));
  A.n_tiles = split.n_tiles;
  A.k_tiles = split.k_tiles;
  A.n_parts = split.parts;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == BEVPOOL_F16) return launch(A, static_cast<_Float16 *>(dweight), s);
  return launch(A, static_cast<__bf16 *>(dweight), s);
}

size_t bevpool_column_sums_scratch_bytes(int32_t width) {
  return width < 1 ? 0 : size_t(kColumnParts) * size_t(width) * sizeof(float);
}

int bevpool_column_sums(const void *x, int64_t x_row, int32_t dtype, int64_t rows, int32_t width,
                        void *out, void *scratch, size_t scratch_bytes, void *stream) {
  bevpool_host::clear_error();
  if (dtype < BEVPOOL_F32 || dtype > BEVPOOL_BF16)
    return fail(BEVPOOL_EINVAL, "unsupported dtype code %d", dtype);
  if (rows < 0 || rows > (int64_t(1) << 40)) return fail(BEVPOOL_EINVAL, "bad number of rows");
  if (width < 1 || width > (1 << 28)) return fail(BEVPOOL_EINVAL, "bad width %d", width);
  if ((rows > 0 && !x) || !out) return fail(BEVPOOL_EINVAL, "null rows");
  if (!scratch || scratch_bytes < bevpool_column_sums_scratch_bytes(width))
    return fail(BEVPOOL_ESPACE, "column sums scratch too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  float *parts = static_cast<float *>(scratch);
  if (dtype == BEVPOOL_F32) return launch_columns<float>(x, x_row, rows, width, out, parts, s);
  if (dtype == BEVPOOL_F16) return launch_columns<_Float16>(x, x_row, rows, width, out, parts, s);
  return launch_columns<__bf16>(x, x_row, rows, width, out, parts, s);
}

}  // extern "C"

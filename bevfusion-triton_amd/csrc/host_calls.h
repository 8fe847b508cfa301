// Host side shared by the library's source files: the calling thread's error
// text, launch checks and the optional per-kernel timing (defined in
// bevpool.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "bevpool.h"

namespace bevpool_host __attribute__((visibility("hidden"))) {

void clear_error();
int set_error(int code, const char *text);  // returns code

__attribute__((format(printf, 2, 3))) inline int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}

inline int check_launch(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(BEVPOOL_EHIP, "%s: %s", what, hipGetErrorString(e));
  return BEVPOOL_OK;
}

// A launch carries its size in work-items as 32 bits; one past that is
// refused here instead of being truncated.
inline int check_grid(int64_t blocks, int threads, const char *what) {
  if (blocks < 0 || blocks * int64_t(threads) > int64_t(UINT32_MAX))
    return fail(BEVPOOL_EINVAL, "%s: %lld blocks of %d threads exceed the 2^32 work-item grid",
                what, static_cast<long long>(blocks), threads);
  return BEVPOOL_OK;
}

// Brackets one kernel launch with events while timing is enabled.
class LaunchScope {
 public:
  LaunchScope(const char *name, hipStream_t stream);
  ~LaunchScope();
  LaunchScope(const LaunchScope &) = delete;
  LaunchScope &operator=(const LaunchScope &) = delete;

 private:
  void *timer_;
};

}  // namespace bevpool_host

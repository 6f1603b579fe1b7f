// Library-wide ABI entry points: version and thread-local error reporting.
#include <stdio.h>
#include <string.h>

#include <atomic>

#include <hip/hip_runtime_api.h>

#include "bi_internal.h"

namespace {
thread_local char g_last_error[512] = "";
}

namespace bi {

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

int launch_error(int hip_error, const char* what) {
  return fail(BI_ELAUNCH, "%s: HIP error %d (%s)", what, hip_error,
              hipGetErrorString(static_cast<hipError_t>(hip_error)));
}

int device_cus() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n <= 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        n <= 0)
      n = 256;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace bi

extern "C" int bi_abi_version(void) { return BI_ABI_VERSION; }

extern "C" const char* bi_last_error(void) { return g_last_error; }

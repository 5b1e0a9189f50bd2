// Host helpers shared by the translation units of libgoenv.so: the thread's last error, the device of a call, streams.
#pragma once

#include <hip/hip_runtime.h>

#include <string>

namespace goenv {

// goenv_last_error's text.  One per thread, the same for every translation unit of the library.
inline thread_local std::string g_err;

inline int fail(const char* what, hipError_t e = hipSuccess) {
  g_err = what;
  if (e != hipSuccess) {
    g_err += ": ";
    g_err += hipGetErrorString(e);
  }
  return -1;
}

#define HIPCHK(x)                                  \
  do {                                             \
    hipError_t e_ = (x);                           \
    if (e_ != hipSuccess) return fail(#x, e_);     \
  } while (0)

inline hipStream_t S(void* s) { return (hipStream_t)s; }

// Entry points that launch or copy run with the context's device current and put the caller's
// device back on return (one host thread may drive several GPUs; a kernel launched on the null
// stream of another device would be handed pointers that device cannot reach).
struct DeviceScope {
  int prev = -1;
  bool switched = false;
  hipError_t err;
  explicit DeviceScope(int dev) {
    err = hipGetDevice(&prev);
    if (err == hipSuccess && prev != dev) {
      err = hipSetDevice(dev);
      switched = err == hipSuccess;
    }
  }
  ~DeviceScope() {
    if (switched) (void)hipSetDevice(prev);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

}  // namespace goenv

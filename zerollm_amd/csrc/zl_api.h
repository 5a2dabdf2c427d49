// What the C entry points share: the calling thread's error message, the device, and the frame that turns exceptions into
// status codes.
#pragma once
#include "zl_common.h"

namespace zl {

std::string &last_error();   // of the calling thread
void ensure_init();          // selects GPU 0 where zl_init has not run
int device();                // the library's GPU (after ensure_init)
void zero_now(void *p, size_t n);

// Makes `dev` the calling thread's current device for a scope: the default stream is the current device's, and a thread
// other than the one that called zl_init starts with device 0.
struct OnDevice {
  int prev = -1, dev;
  explicit OnDevice(int d) : dev(d) {
    ZL_HIP(hipGetDevice(&prev));
    if (prev != dev) ZL_HIP(hipSetDevice(dev));
  }
  ~OnDevice() {
    if (prev >= 0 && prev != dev) hipSetDevice(prev);
  }
};

}  // namespace zl

#define ZL_API_BEGIN try {
#define ZL_API_END                              \
  zl::last_error().clear();                     \
  return ZL_OK;                                 \
  }                                             \
  catch (const zl::Error &e) {                  \
    zl::last_error() = e.what();                \
    return e.code;                              \
  }                                             \
  catch (const std::exception &e) {             \
    zl::last_error() = e.what();                \
    return ZL_ERR_HIP;                          \
  }

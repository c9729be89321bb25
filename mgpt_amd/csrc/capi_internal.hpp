// capi_internal.hpp -- host-side helpers shared by the C ABI's source files.
#pragma once

namespace mgpt {

// Records a printf-style description for mgpt_moe_last_error() on this host
// thread and returns `code`.
int fail(int code, const char* fmt, ...);

}  // namespace mgpt

// Returns MGPT_ERR_HIP, with the call that failed as the description, from a
// function that uses a status (mgpt_moe.h and the HIP runtime are included there).
#define HIP_TRY(expr)                                                             \
  do {                                                                            \
    hipError_t _e = (expr);                                                       \
    if (_e != hipSuccess)                                                         \
      return mgpt::fail(MGPT_ERR_HIP, "%s failed: %s (%s:%d)", #expr,             \
                        hipGetErrorString(_e), __FILE__, __LINE__);               \
  } while (0)

// Errors of the C entry points: thrown as Error inside, turned into a status and
// the calling thread's message at the boundary.
#pragma once

#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

#include "chonk.h"

namespace chonk {

extern thread_local std::string g_last_error;  // chonk_last_error (engine.hip)

struct Error : std::runtime_error {
  int code;
  Error(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

#define HIP_OK(expr)                                                                                      \
  do {                                                                                                    \
    hipError_t e_ = (expr);                                                                               \
    if (e_ != hipSuccess)                                                                                 \
      throw chonk::Error(CHONK_EHIP, std::string("HIP error ") + hipGetErrorString(e_) + " at " #expr);   \
  } while (0)

// Entry points without an engine.
template <typename F>
int api_free(F&& f) {
  try {
    f();
    return CHONK_OK;
  } catch (const Error& x) {
    g_last_error = x.what();
    return x.code;
  } catch (const std::exception& x) {
    g_last_error = x.what();
    return CHONK_EIO;
  }
}

}  // namespace chonk

// The library's error state, shared by its translation units (grlhip_last_error reads it), and the guard of the C entry
// points: nothing leaves them as an exception.
#pragma once
#include <cstddef>
#include <exception>
#include <string>

#include "../../include/grlhip.h"

namespace grlhip {
int set_error(int code, const std::string& message) noexcept;

template <class F>
int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (const std::exception& e) {
    return set_error(GRLHIP_ERR_INVALID, e.what());
  } catch (...) {
    return set_error(GRLHIP_ERR_INVALID, "unknown exception");
  }
}
template <class F>
size_t guarded_size(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    set_error(GRLHIP_ERR_INVALID, "exception while sizing a workspace");
    return 0;
  }
}
}  // namespace grlhip

#define LAUNCH_TRY(expr)                                                                                                      \
  do {                                                                                                                        \
    const hipError_t e_ = (expr);                                                                                             \
    if (e_ != hipSuccess) return grlhip::set_error(GRLHIP_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(e_)); \
  } while (0)

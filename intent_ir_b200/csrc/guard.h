// No exception (an allocation that failed, for a message or a map) leaves a C entry.
#pragma once
#include <exception>
#include <string>

namespace ib200 {

// f()'s answer, or `failed` with a message that says what was thrown
template <typename F> int guarded(std::string& message, int failed, F f) noexcept {
  const char* what = "unknown exception";
  try {
    return f();
  } catch (const std::exception& e) {
    try {
      message = std::string("exception: ") + e.what();
      return failed;
    } catch (...) {
      what = "out of memory";
    }
  } catch (...) {
  }
  try {
    message = what;
  } catch (...) {
    message.clear();  // an older message does not stand for this failure
  }
  return failed;
}

}  // namespace ib200

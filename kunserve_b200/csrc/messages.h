// Error messages of the Python bindings.  Numbers are formatted with
// to_string: streaming them needs the locale tables of one C++ runtime, and
// the extension may be linked with another than the libraries it is loaded
// into.
#pragma once
#include <torch/extension.h>
#include <string>

namespace kus {

inline std::string text(const char* s) { return s; }
inline std::string text(int64_t v) { return std::to_string(v); }
inline std::string text(torch::ScalarType t) { return c10::toString(t); }
inline std::string text(const torch::Device& d) { return d.str(); }
inline std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <typename... A>
std::string say(const A&... a) {
  std::string s;
  ((s += text(a)), ...);
  return s;
}

}  // namespace kus

#define KUS_CHECK(cond, ...) TORCH_CHECK(cond, ::kus::say(__VA_ARGS__))

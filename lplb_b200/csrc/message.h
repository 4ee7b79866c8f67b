// Messages of the bindings' refusals, put together from strings: a number written to an ostringstream ends the
// process where the compiler's C++ library is newer than the one that is loaded.
#pragma once

#include <string>
#include <type_traits>

namespace lplb {

class Message {
 public:
  Message& operator<<(const std::string& s) {
    text_ += s;
    return *this;
  }
  Message& operator<<(const char* s) {
    text_ += s;
    return *this;
  }
  template <typename T, std::enable_if_t<std::is_arithmetic_v<T>, int> = 0>
  Message& operator<<(T n) {
    text_ += std::to_string(n);
    return *this;
  }
  const std::string& str() const { return text_; }

 private:
  std::string text_;
};

}  // namespace lplb

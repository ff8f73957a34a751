// Launchers with dozens of arguments, called with one: a block of memory that holds the arguments one behind the other, each
// at its type's alignment, as the C struct of them would.  (Converting every argument on its own costs the caller 0.2 us each,
// more than the smallest kernels run.)
#pragma once
#include <stddef.h>
#include <string.h>

#include <utility>

namespace distie {

template <typename T>
T packed_at(const unsigned char* block, size_t& at) {
  at = (at + alignof(T) - 1) / alignof(T) * alignof(T);
  T value;
  memcpy(&value, block + at, sizeof(T));
  at += sizeof(T);
  return value;
}

template <typename... Args>
struct Packed {
  int (*launcher)(Args...);
  int operator()(const void* block) const {
    size_t at = 0;
    struct Call {  // (braces evaluate from left to right, the arguments of a call in any order)
      int result;
      Call(int (*launcher)(Args...), Args... args) : result(launcher(args...)) {}
    };
    return Call{launcher, packed_at<Args>(reinterpret_cast<const unsigned char*>(block), at)...}.result;
  }
};

template <typename... Args>
Packed<Args...> packed(int (*launcher)(Args...)) { return {launcher}; }

}  // namespace distie

#define DISTIE_PACKED(name) \
  extern "C" int name##_packed(const void* block) { return distie::packed(&name)(block); }

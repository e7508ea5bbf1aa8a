// What the C entry points share: workspace carving, argument checks and the
// macros that hand an error on.
#pragma once

#include <initializer_list>
#include <string>

#include "common.h"

namespace rpx {

// Bump allocator over a caller-provided workspace.
struct Arena {
  uint8_t* base;
  size_t cap;
  size_t used = 0;
  bool overflow = false;
  Arena(void* p, size_t c) : base(static_cast<uint8_t*>(p)), cap(c) {}
  template <typename T>
  T* take(int64_t count) {
    const size_t bytes = (static_cast<size_t>(count) * sizeof(T) + 255) & ~static_cast<size_t>(255);
    if (used + bytes > cap) {
      overflow = true;
      return nullptr;
    }
    T* p = reinterpret_cast<T*>(base + used);
    used += bytes;
    return p;
  }
};

// Size-only twin of Arena.
struct Sizer {
  size_t used = 0;
  template <typename T>
  void take(int64_t count) {
    used += (static_cast<size_t>(count) * sizeof(T) + 255) & ~static_cast<size_t>(255);
  }
};

inline size_t elem_size(int dtype) { return dtype == kBF16 ? 2 : 4; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Every non-null pointer 16-byte aligned.
inline bool aligned16_all(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (p != nullptr && !aligned16(p)) return false;
  return true;
}
inline bool pow2(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }

inline int check_dtype(int dtype) {
  if (dtype != kF32 && dtype != kBF16) return fail_invalid("dtype must be RPX_DTYPE_F32 or RPX_DTYPE_BF16");
  return kOk;
}

}  // namespace rpx

#define RPX_TRY(expr)            \
  do {                           \
    const int _rc = (expr);      \
    if (_rc != kOk) return _rc;  \
  } while (0)

#define RPX_HIP(expr, what) RPX_TRY(check_hip((expr), (what)))

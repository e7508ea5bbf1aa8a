// Eight consecutive values of a row as float32, from and to bf16 or float32
// memory of any alignment: the loads and stores are the widest there are (global
// memory takes them at any address), and the last vector of a row whose length is
// no multiple of eight goes value by value.
#pragma once

#include "common.h"

namespace rpx {

struct Bf16 {
  uint16_t bits;
};

__device__ __forceinline__ void load8(const Bf16* p, float* v) {
  u32x4_t w;
  __builtin_memcpy(&w, p, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16lo_to_f32(w[i]);
    v[2 * i + 1] = bf16hi_to_f32(w[i]);
  }
}
__device__ __forceinline__ void load8(const float* p, float* v) {
  f32x4_t a, b;
  __builtin_memcpy(&a, p, 16);
  __builtin_memcpy(&b, p + 4, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}
__device__ __forceinline__ void store8(Bf16* p, const float* v) {
  const u32x4_t w{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                  pack_bf16x2(v[6], v[7])};
  __builtin_memcpy(p, &w, 16);
}
__device__ __forceinline__ void store8(float* p, const float* v) {
  const f32x4_t a{v[0], v[1], v[2], v[3]}, b{v[4], v[5], v[6], v[7]};
  __builtin_memcpy(p, &a, 16);
  __builtin_memcpy(p + 4, &b, 16);
}
__device__ __forceinline__ float load1(const Bf16* p) { return bf16_to_f32(p->bits); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(Bf16* p, float v) { p->bits = f32_to_bf16(v); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
// To the type's nearest value.
__device__ __forceinline__ float rounded(const Bf16*, float v) { return round_bf16(v); }
__device__ __forceinline__ float rounded(const float*, float v) { return v; }

// Eight values as they lie in memory, for loads that run ahead of their use.
template <typename T>
struct Raw8;
template <>
struct Raw8<Bf16> {
  u32x4_t w;
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16lo_to_f32(w[i]);
      v[2 * i + 1] = bf16hi_to_f32(w[i]);
    }
  }
  __device__ __forceinline__ void set(int i, const Bf16* p) {
    w[i >> 1] |= static_cast<uint32_t>(p->bits) << (16 * (i & 1));
  }
  __device__ __forceinline__ void load(const Bf16* p) { __builtin_memcpy(&w, p, 16); }
  __device__ __forceinline__ void zero() { w = u32x4_t{0u, 0u, 0u, 0u}; }
};
template <>
struct Raw8<float> {
  f32x4_t a, b;
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  }
  __device__ __forceinline__ void set(int i, const float* p) {
    if (i < 4) a[i] = *p;
    else b[i - 4] = *p;
  }
  __device__ __forceinline__ void load(const float* p) {
    __builtin_memcpy(&a, p, 16);
    __builtin_memcpy(&b, p + 4, 16);
  }
  __device__ __forceinline__ void zero() { a = b = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}; }
};
// The first `count` of eight (the rest zero); WHOLE: all of them.
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_raw8(const T* p, int count, Raw8<T>& r) {
  if (WHOLE || count >= 8) {
    r.load(p);
    return;
  }
  r.zero();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) r.set(i, p + i);
}

// The first `count` of eight (the rest zero); WHOLE: all of them.
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_row8(const T* p, int count, float* v) {
  if (WHOLE || count >= 8) {
    load8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < count ? load1(p + i) : 0.0f;
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store_row8(T* p, int count, const float* v) {
  if (WHOLE || count >= 8) {
    store8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) store1(p + i, v[i]);
}

}  // namespace rpx

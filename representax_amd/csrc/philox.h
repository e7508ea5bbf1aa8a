// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011): ten rounds of two 32 x 32 -> 64 bit products over a
// 128-bit counter, and the dropout that is made from it.
//
// Element i of a tensor, in its dense order, takes the 16 bits number i % 8 of
// the counter (i / 8, its high word, site, step) under the key `seed`, and is
// kept where they are below a threshold of 65536ths. 16 bits an element let one
// counter serve a vector of eight: 20 products for 16 bytes of bf16, which stay
// below the time that the memory takes for them (a float32 threshold, 32 bits an
// element, doubles them). The rate is rounded to a 65536th, and the scale is that
// of the rounded rate, so the expectation is exact.
#pragma once

#include "common.h"

namespace rpx {

struct Dropout {
  const int64_t* key;  // device: seed, step
  uint32_t site;
  uint32_t threshold;  // kept below it, 1 .. 65536; 65536: no dropout
  float scale;         // 65536 / threshold
};

// The counter's words that are the same for a whole call.
struct PhiloxCall {
  uint32_t k0, k1, site, step;
};

__device__ __forceinline__ PhiloxCall philox_call(const Dropout& d) {
  const uint64_t seed = static_cast<uint64_t>(d.key[0]);
  return PhiloxCall{static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), d.site,
                    static_cast<uint32_t>(d.key[1])};
}

__device__ __forceinline__ u32x4_t philox(const PhiloxCall& call, uint64_t counter) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32);
  uint32_t c2 = call.site, c3 = call.step, k0 = call.k0, k1 = call.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0;
    const uint64_t b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4_t{c0, c1, c2, c3};
}

// The bits of the eight elements from `first` on, element j's in half j % 2 of
// word j / 2. ALIGNED: first is a multiple of 8.
template <bool ALIGNED>
__device__ __forceinline__ u32x4_t dropout_bits(const PhiloxCall& call, int64_t first) {
  const uint64_t at = static_cast<uint64_t>(first) >> 3;
  u32x4_t a = philox(call, at);
  if constexpr (!ALIGNED) {
    // eight halves out of two counters' sixteen, from half first % 8 on
    const u32x4_t b = philox(call, at + 1);
    uint32_t w[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    if (first & 4) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (first & 2) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (first & 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (w[i] >> 16) | (w[i + 1] << 16);
    }
    a = u32x4_t{w[0], w[1], w[2], w[3]};
  }
  return a;
}

// Whether element j of the eight is kept.
__device__ __forceinline__ bool dropout_kept(const u32x4_t& bits, int j, uint32_t threshold) {
  return ((j & 1) ? bits[j >> 1] >> 16 : bits[j >> 1] & 0xFFFFu) < threshold;
}

// v through the dropout, in place: a dropped element is zero whatever it was.
template <bool ALIGNED>
__device__ __forceinline__ void dropout8(const PhiloxCall& call, const Dropout& d, int64_t first,
                                         float* v) {
  const u32x4_t bits = dropout_bits<ALIGNED>(call, first);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = dropout_kept(bits, j, d.threshold) ? v[j] * d.scale : 0.0f;
}

// v, or zero where bit `bit` of the mask is clear: as bits, so that a NaN goes too.
__device__ __forceinline__ float dropout_masked(float v, uint32_t mask, int bit) {
  const int32_t all = static_cast<int32_t>(mask << (31 - bit)) >> 31;
  return __builtin_bit_cast(float, __builtin_bit_cast(int32_t, v) & all);
}

// Which of a lane's 16 values of a 32 x 32 matrix-core block are kept: its row begins
// (at the block's first column) at element `first`, a multiple of 8, and register v
// holds column 8 (v / 4) + 4 (lane / 32) + v % 4: bit v. The two lanes of a row take two
// of its four counters each and exchange what the other needs.
__device__ __forceinline__ uint32_t dropout_block(const PhiloxCall& call, uint32_t threshold,
                                                  int64_t first, int half) {
  const uint64_t at = (static_cast<uint64_t>(first) >> 3) + 2 * half;
  uint32_t mask = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4_t w = philox(call, at + i);
    // columns 8 i + and 8 (i + 2) +: this lane's two words of each
    const u32x2_t a =
        __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false));
    const u32x2_t b =
        __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int v = 4 * (i + 2 * k);
      mask |= static_cast<uint32_t>((a[k] & 0xFFFFu) < threshold) << v;
      mask |= static_cast<uint32_t>((a[k] >> 16) < threshold) << (v + 1);
      mask |= static_cast<uint32_t>((b[k] & 0xFFFFu) < threshold) << (v + 2);
      mask |= static_cast<uint32_t>((b[k] >> 16) < threshold) << (v + 3);
    }
  }
  return mask;
}

}  // namespace rpx

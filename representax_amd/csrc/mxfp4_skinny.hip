// Products of a few rows with a weight kept in MXFP4 (a query's token, a short
// query): y = x W^T, or silu(x G^T) * (x U^T), x in bf16 or float32 and encoded on
// the way, in one launch.
//
// Such a call is the read of the weight, 0.53 bytes a value, and the launch. A
// workgroup owns 16 rows of the weight over all columns; its waves split the
// columns by slices and meet in LDS, in wave order. On the 16x16x128 MFMA lane l
// holds 32 values of row l % 16, and with q = l / 16 it takes the slice's blocks 2 q
// and 2 q + 1 in its two steps: 32 contiguous bytes of codes and two scale bytes.
// The same lane of the other operand holds the same two blocks of token l % 16, so
// a block of x is encoded by the lane that needs it, with no exchange: 64 values
// a slice, while the weight's loads are in flight. Every workgroup encodes x anew;
// for a few tokens that is cheaper than a launch that would do it once.
//
// One row, weights from HBM, graph replays: 2048 -> 6144 4.8 us (6.7 MB, 1.4 TB/s: the
// launch and two dependent trips to memory), two weights of it 5.9 (13.4 MB, 2.3 TB/s),
// 6144 -> 2048 6.2. Sixteen rows 7.7, 8.3 and 9.7.
#include <hip/hip_runtime.h>

#include "act.h"
#include "kernels.h"
#include "mxfp4.h"

namespace rpx {

namespace {

constexpr int kTokens = 16;  // of an MFMA
constexpr int kMaxWaves = 16;

// A block of a row of x: columns c .. c + 31, zeros past the end.
template <int DTYPE>
struct Block {
  static constexpr int WORDS = DTYPE == kBF16 ? 16 : 32;
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const uint8_t* row, int64_t c, int64_t columns) {
    if (c + kMxBlock <= columns) {  // any alignment
      __builtin_memcpy(w, row + c * (WORDS / 8), sizeof(w));
      return;
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < kMxBlock; ++i) {
      const int64_t at = c + i < columns ? c + i : columns - 1;
      const uint32_t in = c + i < columns ? ~0u : 0u;
      if constexpr (DTYPE == kBF16)
        w[i / 2] |= (reinterpret_cast<const uint16_t*>(row)[at] & in) << (16 * (i & 1));
      else
        w[i] = reinterpret_cast<const uint32_t*>(row)[at] & in;
    }
  }

  // Its codes (any under a NaN scale) and scale byte.
  __device__ __forceinline__ u32x4_t encode(uint32_t* byte) const {
    uint32_t top;
    if constexpr (DTYPE == kBF16) {
      typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
      u16x2_t m = {0, 0};
#pragma unroll
      for (int i = 0; i < WORDS; ++i)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w[i] & 0x7FFF7FFFu));
      top = static_cast<uint32_t>(m.x > m.y ? m.x : m.y) << 16;
    } else {
      top = 0;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) top = (w[i] & 0x7FFFFFFFu) > top ? w[i] & 0x7FFFFFFFu : top;
    }
    *byte = mx_scale_byte(top);
    const float scale = mx_scale_operand(*byte);
    u32x4_t code;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if constexpr (DTYPE == kBF16) {
        code[g] = mx_encode8(u32x4_t{w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]}, scale);
      } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(float, w[8 * g + e]);
        code[g] = mx_encode8(v, scale);
      }
    }
    return code;
  }
};

__device__ __forceinline__ f32x4_t mfma16(u32x4_t a, uint32_t sa, u32x4_t b, uint32_t sb,
                                          f32x4_t c) {
  const i32x8_t av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, kMxFp4, kMxFp4, 0, (int)sa, 0,
                                                          (int)sb);
}

// One token's outputs at the weight's rows n ... n + 3 from their sums.
template <int DTYPE, bool GATED>
__device__ __forceinline__ void store_rows(const MxSkinny& p, int64_t token, int64_t n,
                                           const f32x4_t* sum) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = sum[0][e];
    if constexpr (GATED) {
      const float zg = DTYPE == kBF16 ? round_bf16(sum[0][e]) : sum[0][e];
      const float zu = DTYPE == kBF16 ? round_bf16(sum[1][e]) : sum[1][e];
      y[e] = act_apply<kActSiluMulFwd>(zu, zg, 0.0f, nullptr);
    }
  }
  if constexpr (DTYPE == kBF16) {
    uint16_t* d = static_cast<uint16_t*>(p.y) + token * p.n + n;
    if ((p.n & 3) == 0 && n < p.n) {
      *reinterpret_cast<u32x2_t*>(d) = u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    } else {
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) d[e] = f32_to_bf16(y[e]);
    }
  } else {
    float* d = static_cast<float*>(p.y) + token * p.n + n;
    for (int e = 0; e < 4; ++e)
      if (n + e < p.n) d[e] = y[e];
  }
}

// A wave takes AHEAD slices at a time: x's loads first, then the weight's (loads
// return in order, so x, which is small and soon in the L2, is encoded while the
// weight is on its way), then the encoding, then the MFMAs.
template <int DTYPE, int AHEAD, bool GATED>
__global__ void __launch_bounds__(64 * kMaxWaves) k_mx_skinny(MxSkinny p) {
  constexpr int G = GATED ? 2 : 1;
  extern __shared__ __align__(16) float partial[];  // [wave][G][lane][4]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int waves = blockDim.x >> 6;
  const int q = lane >> 4;
  const int token = lane & 15;
  const int64_t n0 = block_of_grid() * kTokens;
  if (n0 >= p.n) return;  // the whole workgroup
  const int64_t r = n0 + token < p.n ? n0 + token : p.n - 1;  // the lane's row of the weight
  const int64_t pad = mx_pad_rows(p.n);
  const uint8_t* row = static_cast<const uint8_t*>(p.x) +
                       (token < p.m ? token : p.m - 1) * p.row_stride * (DTYPE == kBF16 ? 2 : 4);
  f32x4_t acc[G];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = f32x4_t{0, 0, 0, 0};

  for (int64_t s0 = wave; s0 < p.slices; s0 += AHEAD * waves) {
    Block<DTYPE> x[AHEAD][2];
    u32x4_t w[AHEAD][G][2];
    uint32_t ws[AHEAD][G];
    // a slice past the end is read as the one before, and not multiplied
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int64_t s = s0 + a * waves < p.slices ? s0 + a * waves : s0;
#pragma unroll
      for (int step = 0; step < 2; ++step)
        x[a][step].load(row, s * kMxSlice + 64 * q + kMxBlock * step, p.k);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int64_t s = s0 + a * waves < p.slices ? s0 + a * waves : s0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint8_t* codes =
            (g == 0 ? p.codes : p.codes2) + (r * p.slices + s) * kMxSliceBytes + 32 * q;
        const uint8_t* scales =
            (g == 0 ? p.scales : p.scales2) + (s * pad + r) * kMxSliceBlocks + 2 * q;
        w[a][g][0] = *reinterpret_cast<const u32x4_t*>(codes);
        w[a][g][1] = *reinterpret_cast<const u32x4_t*>(codes + 16);
        ws[a][g] = *reinterpret_cast<const uint16_t*>(scales);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t code[AHEAD][2];
    uint32_t byte[AHEAD][2];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
#pragma unroll
      for (int step = 0; step < 2; ++step) code[a][step] = x[a][step].encode(&byte[a][step]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (s0 + a * waves >= p.slices) break;
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int g = 0; g < G; ++g)
          acc[g] = mfma16(w[a][g][step], ws[a][g] >> (8 * step), code[a][step], byte[a][step],
                          acc[g]);
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
    *reinterpret_cast<f32x4_t*>(partial + ((wave * G + g) * 64 + lane) * 4) = acc[g];
  __syncthreads();
  if (wave != 0 || token >= p.m) return;
  // the lane holds token l % 16 and rows n0 + 4 (l / 16) ... + 3 of the weight
  f32x4_t sum[G];
#pragma unroll
  for (int g = 0; g < G; ++g) sum[g] = f32x4_t{0, 0, 0, 0};
  for (int v = 0; v < waves; ++v)
#pragma unroll
    for (int g = 0; g < G; ++g)
      sum[g] += *reinterpret_cast<const f32x4_t*>(partial + ((v * G + g) * 64 + lane) * 4);
  store_rows<DTYPE, GATED>(p, token, n0 + 4 * q, sum);
}

// The same for up to TILES x 16 rows of x that are encoded already: a lane reads its
// blocks' codes and scales as it reads the weight's. 32 rows of 2048 -> 6144 with their
// encoding 8.8 us.
template <int DTYPE, int TILES, bool GATED>
__global__ void __launch_bounds__(64 * kMaxWaves) k_mx_thin(MxSkinny p) {
  constexpr int G = GATED ? 2 : 1;
  extern __shared__ __align__(16) float partial[];  // [wave][tile][G][lane][4]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int waves = blockDim.x >> 6;
  const int q = lane >> 4;
  const int64_t n0 = block_of_grid() * kTokens;
  if (n0 >= p.n) return;  // the whole workgroup
  const int64_t r = n0 + (lane & 15) < p.n ? n0 + (lane & 15) : p.n - 1;
  const int64_t pad = mx_pad_rows(p.n);
  const int64_t x_pad = mx_pad_rows(p.m);
  int64_t token[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    token[t] = t * kTokens + (lane & 15);
    token[t] = token[t] < p.m ? token[t] : p.m - 1;
  }
  f32x4_t acc[TILES][G];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int g = 0; g < G; ++g) acc[t][g] = f32x4_t{0, 0, 0, 0};
  for (int64_t s = wave; s < p.slices; s += waves) {
    u32x4_t w[G][2], x[TILES][2];
    uint32_t ws[G], xs[TILES];
    auto at = [&](const uint8_t* codes, int64_t row) {
      return reinterpret_cast<const u32x4_t*>(codes + (row * p.slices + s) * kMxSliceBytes + 32 * q);
    };
    auto scales_at = [&](const uint8_t* scales, int64_t rows, int64_t row) {
      return *reinterpret_cast<const uint16_t*>(scales + (s * rows + row) * kMxSliceBlocks + 2 * q);
    };
#pragma unroll
    for (int g = 0; g < G; ++g) {
      w[g][0] = at(g == 0 ? p.codes : p.codes2, r)[0];
      w[g][1] = at(g == 0 ? p.codes : p.codes2, r)[1];
      ws[g] = scales_at(g == 0 ? p.scales : p.scales2, pad, r);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      x[t][0] = at(static_cast<const uint8_t*>(p.x), token[t])[0];
      x[t][1] = at(static_cast<const uint8_t*>(p.x), token[t])[1];
      xs[t] = scales_at(p.x_scales, x_pad, token[t]);
    }
#pragma unroll
    for (int step = 0; step < 2; ++step)
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g)
          acc[t][g] = mfma16(w[g][step], ws[g] >> (8 * step), x[t][step], xs[t] >> (8 * step),
                             acc[t][g]);
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int g = 0; g < G; ++g)
      *reinterpret_cast<f32x4_t*>(partial + (((wave * TILES + t) * G + g) * 64 + lane) * 4) =
          acc[t][g];
  __syncthreads();
  for (int t = wave; t < TILES; t += waves) {
    f32x4_t sum[G];
#pragma unroll
    for (int g = 0; g < G; ++g) sum[g] = f32x4_t{0, 0, 0, 0};
    for (int v = 0; v < waves; ++v)
#pragma unroll
      for (int g = 0; g < G; ++g)
        sum[g] += *reinterpret_cast<const f32x4_t*>(
            partial + (((v * TILES + t) * G + g) * 64 + lane) * 4);
    if (t * kTokens + (lane & 15) < p.m)
      store_rows<DTYPE, GATED>(p, t * kTokens + (lane & 15), n0 + 4 * q, sum);
  }
}

template <int DTYPE, int AHEAD, bool GATED>
hipError_t launch_one(const MxSkinny& p, hipStream_t stream) {
  const int64_t want = ceil_div(p.slices, AHEAD);
  const int waves = static_cast<int>(want < kMaxWaves ? want : kMaxWaves);
  const size_t lds = static_cast<size_t>(waves) * (GATED ? 2 : 1) * 64 * 4 * sizeof(float);
  hipLaunchKernelGGL((k_mx_skinny<DTYPE, AHEAD, GATED>), grid_of(ceil_div(p.n, kTokens)),
                     dim3(64 * waves), lds, stream, p);
  return hipGetLastError();
}

template <int DTYPE, int TILES, bool GATED>
hipError_t launch_thin(const MxSkinny& p, hipStream_t stream) {
  constexpr int G = GATED ? 2 : 1;
  // partial sums of at most 64 KB
  constexpr int kWaves = 64 / (TILES * G) < kMaxWaves ? 64 / (TILES * G) : kMaxWaves;
  const int waves = static_cast<int>(p.slices < kWaves ? p.slices : kWaves);
  const size_t lds = static_cast<size_t>(waves) * TILES * G * 64 * 4 * sizeof(float);
  hipLaunchKernelGGL((k_mx_thin<DTYPE, TILES, GATED>), grid_of(ceil_div(p.n, kTokens)),
                     dim3(64 * waves), lds, stream, p);
  return hipGetLastError();
}

template <int DTYPE, bool GATED>
hipError_t launch_thin_tiles(const MxSkinny& p, hipStream_t stream) {
  switch (ceil_div(p.m, kTokens)) {
    case 1: return launch_thin<DTYPE, 1, GATED>(p, stream);
    case 2: return launch_thin<DTYPE, 2, GATED>(p, stream);
    case 3: return launch_thin<DTYPE, 3, GATED>(p, stream);
    case 4: return launch_thin<DTYPE, 4, GATED>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

// A wave takes one slice while there are waves for it. Beyond, two of bf16's fit
// its registers where there is one weight.
hipError_t launch_mx_skinny(const MxSkinny& p, int dtype, hipStream_t stream) {
  if (p.m > (p.x_scales != nullptr ? kMxThinRows : kMxSkinnyRows)) return hipErrorInvalidValue;
  const bool gated = p.codes2 != nullptr;
  if (p.x_scales != nullptr) {
    if (dtype == kBF16)
      return gated ? launch_thin_tiles<kBF16, true>(p, stream)
                   : launch_thin_tiles<kBF16, false>(p, stream);
    return gated ? launch_thin_tiles<kF32, true>(p, stream)
                 : launch_thin_tiles<kF32, false>(p, stream);
  }
  if (dtype != kBF16)
    return gated ? launch_one<kF32, 1, true>(p, stream) : launch_one<kF32, 1, false>(p, stream);
  if (gated) return launch_one<kBF16, 1, true>(p, stream);
  return p.slices <= kMaxWaves ? launch_one<kBF16, 1, false>(p, stream)
                               : launch_one<kBF16, 2, false>(p, stream);
}

}  // namespace rpx

// Encoding to MXFP4 and back (mxfp4.h states the format).
#include <type_traits>

#include <hip/hip_runtime.h>

#include "act.h"
#include "kernels.h"
#include "mxfp4.h"

namespace rpx {

namespace {

constexpr int kThreads = 256;
// Waves of the fused form (32 KB read each) from which both encodings come from one
// read; below, each from its own. The two meet earlier where the matrix lies in the caches,
// later where it comes from memory; the limit is where their mean does. Fused against
// apart, us, from the caches and from memory:
//   bf16     8192 x 768 (384 waves)   11.6 / 8.0, 15.4 / 9.9
//            5632 x 2048 (704)        13.7 / 13.8, 18.2 / 16.1
//            6144 x 2048 (768)        14.0 / 14.7, 18.6 / 17.5
//            7168 x 2048 (896)        15.2 / 16.6, 19.9 / 19.6
//            8192 x 2048 (1024)       15.9 / 18.6, 20.8 / 22.2
//   float32  3072 x 1024 (384)        11.1 / 6.4, 13.4 / 9.2
//            6144 x 768 (576)         11.1 / 10.8, 14.2 / 12.6
//            5120 x 1024 (640)        11.2 / 11.6, 14.5 / 13.5
//            5003 x 1000 (640)        10.9 / 12.4, 14.3 / 14.0
//            8192 x 768 (768)         11.6 / 13.5, 15.2 / 16.0
constexpr int64_t kMxFusedWavesBF16 = 800;
constexpr int64_t kMxFusedWavesF32 = 640;

// Maximum over the LANES neighbouring lanes that share a block.
template <int LANES>
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  static_assert(LANES == 4 || LANES == 8 || LANES == 16, "lanes of a block");
  auto with = [](uint32_t x, uint32_t y) { return y > x ? y : x; };
  v = with(v, __builtin_amdgcn_update_dpp(0u, v, 0xB1, 0xF, 0xF, false));  // lane ^ 1
  v = with(v, __builtin_amdgcn_update_dpp(0u, v, 0x4E, 0xF, 0xF, false));  // lane ^ 2
  if constexpr (LANES >= 8)
    v = with(v, __builtin_amdgcn_update_dpp(0u, v, 0x141, 0xF, 0xF, false));  // 7 - lane
  if constexpr (LANES >= 16)
    v = with(v, __builtin_amdgcn_update_dpp(0u, v, 0x140, 0xF, 0xF, false));  // 15 - lane
  return v;
}

__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a),
                                                                __builtin_bit_cast(u16x2_t, b)));
}

__device__ __forceinline__ float as_f32(uint32_t v) { return __builtin_bit_cast(float, v); }

// What a thread holds of one row: W words, COLS consecutive columns.
template <int DTYPE, int W>
struct Piece {
  static constexpr int COLS = DTYPE == kBF16 ? 2 * W : W;
  static constexpr int LANES = kMxBlock / COLS;  // that share a block
  static constexpr int SIZE = DTYPE == kBF16 ? 2 : 4;
  uint32_t w[W];

  // Largest magnitude's float32 bits (an integer maximum: infinities and NaN on top).
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t a = 0;
    if constexpr (DTYPE == kBF16) {
#pragma unroll
      for (int i = 0; i < W; ++i) a = pk_max(a, w[i] & 0x7FFF7FFFu);
      return (a << 16) > (a & 0xFFFF0000u) ? a << 16 : a & 0xFFFF0000u;
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) a = (w[i] & 0x7FFFFFFFu) > a ? w[i] & 0x7FFFFFFFu : a;
      return a;
    }
  }

  // The codes of the block with scale `byte`, stored at column c of a row of codes.
  __device__ __forceinline__ void store(uint8_t* codes, int64_t c, uint32_t byte) const {
    const float scale = mx_scale_operand(byte);
    uint32_t code = 0;
    if constexpr (DTYPE == kBF16) {
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, mx_as_bf16x2(w[0]), scale, 0);
      if constexpr (W > 1)
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, mx_as_bf16x2(w[1]), scale, 1);
      if constexpr (W > 2) {
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, mx_as_bf16x2(w[2]), scale, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, mx_as_bf16x2(w[3]), scale, 3);
      }
    } else {
      static_assert(W > 1, "a byte of codes holds two columns");
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, as_f32(w[0]), as_f32(w[1]), scale, 0);
      if constexpr (W > 2)
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, as_f32(w[2]), as_f32(w[3]), scale, 1);
    }
    code = byte == 255u ? 0u : code;
    if constexpr (COLS == 8)
      *reinterpret_cast<uint32_t*>(codes + c / 2) = code;
    else if constexpr (COLS == 4)
      *reinterpret_cast<uint16_t*>(codes + c / 2) = static_cast<uint16_t>(code);
    else
      codes[c / 2] = static_cast<uint8_t>(code);
  }
};

// The loads of a thread's column: whole words wherever the row has them, also at
// addresses that are not aligned (the hardware takes any), with the columns past
// the end masked off. Reading past a row's end runs into the next row, so the
// last row, and rows narrower than a piece, are read element by element.
template <int DTYPE, int W>
struct Column {
  using P = Piece<DTYPE, W>;
  const uint8_t* base;
  int64_t stride, c, columns;
  uint32_t mask[W];

  __device__ __forceinline__ Column(const MxPart& part, int64_t col)
      : base(static_cast<const uint8_t*>(part.t)), stride(part.row_stride * P::SIZE), c(col),
        columns(part.columns) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (DTYPE == kBF16)
        mask[i] = (c + 2 * i < columns ? 0xFFFFu : 0u) | (c + 2 * i + 1 < columns ? 0xFFFF0000u : 0u);
      else
        mask[i] = c + i < columns ? ~0u : 0u;
    }
  }

  __device__ __forceinline__ P whole(int64_t row) const {
    struct Words {
      uint32_t w[W];
    };
    Words x;
    __builtin_memcpy(&x, base + row * stride + (c < columns ? c : 0) * P::SIZE, sizeof(x));
    P v;
#pragma unroll
    for (int i = 0; i < W; ++i) v.w[i] = x.w[i] & mask[i];
    return v;
  }
  // Element by element, the columns past the end re-reading the last.
  __device__ __forceinline__ P some(int64_t row) const {
    P v;
#pragma unroll
    for (int i = 0; i < W; ++i) v.w[i] = 0;
#pragma unroll
    for (int e = 0; e < P::COLS; ++e) {
      const int64_t at = c + e < columns ? c + e : columns - 1;
      if constexpr (DTYPE == kBF16)
        v.w[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(base + row * stride)[at])
                      << (16 * (e & 1));
      else
        v.w[e] = reinterpret_cast<const uint32_t*>(base + row * stride)[at];
    }
#pragma unroll
    for (int i = 0; i < W; ++i) v.w[i] &= mask[i];
    return v;
  }
};

// The work of block b of `total`: runs of `run` consecutive pieces go to one XCD (blocks
// go round the eight), whose L2 then has whole lines of what they write; the rest at the
// end as they come.
__device__ __forceinline__ int64_t of_xcd(int64_t b, int64_t total, int64_t run) {
  const int64_t round = 8 * run;
  return b < total / round * round ? b / round * round + b % 8 * run + b % round / 8 : b;
}

// A pass over a large matrix by 64 blocks an XCD against one, us: bf16 40.0 / 44.2 for 16384
// x 6144, 15.8 / 17.2 for 16384 x 2048, 7.2 / 7.1 for 6144 x 2048; float32 93 / 91, 26.4 /
// 26.5, 11.7 / 11.8.
constexpr int64_t kRowsRun = 64;

// Along the columns only: a thread takes 16 bytes of a row, neighbouring lanes a
// block. A pass over memory (serving: the input of a product): 50 us for 16384 x 6144 bf16
// from HBM (5.1 TB/s).
template <int DTYPE>
__device__ __forceinline__ void quantize_rows(const MxPart& part, int64_t i) {
  using P = Piece<DTYPE, 4>;
  const int64_t per = mx_slices(part.columns) * (kMxSlice / P::COLS);
  const int64_t row = i / per;
  const int64_t c = (i % per) * P::COLS;
  if (row >= part.along.scale_rows) return;  // whole blocks: `per` is a multiple of their lanes
  uint32_t byte = 0;
  if (row < part.rows) {
    P v;
    if (c + P::COLS <= part.columns) {
      __builtin_memcpy(&v,
                       static_cast<const uint8_t*>(part.t) + (row * part.row_stride + c) * P::SIZE,
                       sizeof(v));
    } else if (c < part.columns) {
      v = Column<DTYPE, 4>(part, c).some(row);
    } else {
      v = P{};
    }
    byte = mx_scale_byte(block_max<P::LANES>(v.amax()));
    v.store(part.along.codes + row * part.along.row_bytes, c, byte);
  }
  if (c % kMxBlock == 0) *mx_scale_at(part.along, row, c / kMxBlock) = static_cast<uint8_t>(byte);
}

__global__ void __launch_bounds__(kThreads) k_mx_quantize_rows(MxParts parts) {
  int64_t blk = block_of_grid();
  const int64_t total = parts.first[kMxParts];
  if (blk >= total) return;
  blk = of_xcd(blk, total, kRowsRun);
  int p = 0;
  while (blk >= parts.first[p + 1]) ++p;
  const int64_t i = (blk - parts.first[p]) * kThreads + threadIdx.x;
  if (parts.part[p].dtype == kBF16)
    quantize_rows<kBF16>(parts.part[p], i);
  else
    quantize_rows<kF32>(parts.part[p], i);
}

// Waves of `cols` columns that cover a part's.
__host__ __device__ __forceinline__ int64_t mx_tiles_of_row(const MxPart& part, int cols) {
  return ceil_div(part.along.codes != nullptr ? mx_slices(part.columns) * kMxSlice
                                              : part.across.scale_rows,
                  cols);
}

// Along both axes from one read. A thread owns 32 rows of its W words: whole
// blocks of the transpose, in registers, so nothing goes through LDS; a block
// along the columns is shared by neighbouring lanes as above. A wave covers 128
// rows of 16 pieces, so that its stores of the transpose are 64 contiguous bytes
// of a row of codes. 23.0 us for 16384 x 2048 bf16 (4.5 TB/s); half the columns a thread,
// twice the waves, 27.9.
template <int DTYPE, int W>
__device__ __forceinline__ void quantize_both(const MxPart& part, int64_t tile, int lane) {
  using P = Piece<DTYPE, W>;
  constexpr int COLS = 16 * P::COLS;
  const int64_t per = mx_tiles_of_row(part, COLS);
  const int64_t r0 = (tile / per) * 128 + (lane >> 4) * 32;
  const int64_t c = (tile % per) * COLS + (lane & 15) * P::COLS;
  const Column<DTYPE, W> col(part, c);
  P v[32];
  const int64_t last = part.rows - 1;
  if (last > 0 && part.columns >= P::COLS) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = col.whole(r0 + i < last ? r0 + i : last - 1);
    if (r0 + 31 >= last) {
      const P end = col.some(last);
#pragma unroll
      for (int i = 0; i < 32; ++i)
#pragma unroll
        for (int q = 0; q < W; ++q)
          v[i].w[q] = r0 + i < last ? v[i].w[q] : r0 + i == last ? end.w[q] : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      v[i] = col.some(r0 + i < last ? r0 + i : last);
#pragma unroll
      for (int q = 0; q < W; ++q) v[i].w[q] = r0 + i <= last ? v[i].w[q] : 0u;
    }
  }
  constexpr int LANES = P::LANES;
  if constexpr (LANES > 16) {  // across only
  } else if (part.along.codes != nullptr && r0 < part.along.scale_rows) {
    uint32_t kept = 0;  // the scale of this lane's share of LANES rows
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint32_t byte = mx_scale_byte(block_max<LANES>(v[i].amax()));
      if (r0 + i < part.rows)
        v[i].store(part.along.codes + (r0 + i) * part.along.row_bytes, c, byte);
      kept = (lane & (LANES - 1)) == i % LANES ? byte : kept;
      if (i % LANES == LANES - 1)
        *mx_scale_at(part.along, r0 + i - (LANES - 1) + (lane & (LANES - 1)), c / kMxBlock) =
            static_cast<uint8_t>(kept);
    }
  }
  if (part.across.codes == nullptr) return;
  auto store = [&](int64_t at, u32x4_t code, uint32_t byte) {
    if (at < part.columns)
      *reinterpret_cast<u32x4_t*>(part.across.codes + at * part.across.row_bytes + r0 / 2) = code;
    if (at < part.across.scale_rows)
      *mx_scale_at(part.across, at, r0 / kMxBlock) = static_cast<uint8_t>(byte);
  };
#pragma unroll
  for (int q = 0; q < W; ++q) {
    if constexpr (DTYPE == kBF16) {  // columns c + 2 q and c + 2 q + 1
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) top = pk_max(top, v[i].w[q] & 0x7FFF7FFFu);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const uint32_t byte = mx_scale_byte(odd ? top & 0xFFFF0000u : top << 16);
        const float scale = mx_scale_operand(byte);
        u32x4_t code;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          u32x4_t pairs;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            pairs[e] = __builtin_amdgcn_perm(v[8 * g + 2 * e + 1].w[q], v[8 * g + 2 * e].w[q],
                                             odd ? 0x07060302u : 0x05040100u);
          code[g] = byte == 255u ? 0u : mx_encode8(pairs, scale);
        }
        store(c + 2 * q + odd, code, byte);
      }
    } else {
      float x[kMxBlock];
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = as_f32(v[i].w[q]);
      uint32_t byte;
      const u32x4_t code = mx_encode_block(x, &byte);
      store(c + q, code, byte);
    }
  }
}

template <int DTYPE>
__global__ void __launch_bounds__(kThreads) k_mx_quantize_both(MxParts parts) {
  const int64_t blk = block_of_grid();
  if (blk >= parts.first[kMxParts]) return;
  int p = 0;
  while (blk >= parts.first[p + 1]) ++p;
  // In a launch of a workgroup a CU, two rows of tiles, 256 rows of the matrix, run on one
  // XCD, whose L2 then has whole lines of the transpose's codes: 12.3 / 14.0 us for 8192 x
  // 1024 float32 and, forced into this form, 13.4 / 15.4 for 6144 x 2048 bf16, 13.3 / 14.3
  // for 2048 x 6144; longer launches lose by it: 23.9 / 22.9 for 16384 x 2048 bf16, 119 /
  // 112 for 16384 x 6144 float32.
  const MxPart& part = parts.part[p];
  int64_t block = blk - parts.first[p];
  if (parts.first[kMxParts] <= 256) {
    const int64_t run = mx_tiles_of_row(part, 16 * Piece<DTYPE, 4>::COLS) * 2 / (kThreads / 64);
    block = of_xcd(block, parts.first[p + 1] - parts.first[p], run > 0 ? run : 1);
  }
  const int64_t wave = block * (kThreads / 64) + (threadIdx.x >> 6);
  if (wave >= part.tiles) return;
  quantize_both<DTYPE, 4>(part, wave, threadIdx.x & 63);
}

// The two encodings of a small matrix by different workgroups, each from its own
// read: a part is along its columns or across them. A wave of the fused form above
// is a chain of 5 us of instructions in a launch of few waves; the two halves of it
// run side by side instead.
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4)))
    k_mx_quantize_apart(MxParts parts) {
  const int64_t blk = block_of_grid();
  if (blk >= parts.first[kMxParts]) return;
  int p = 0;
  while (blk >= parts.first[p + 1]) ++p;
  const MxPart& part = parts.part[p];
  const int64_t first = blk - parts.first[p];
  if (part.across.codes == nullptr) {
    const int64_t i = first * kThreads + threadIdx.x;
    if (part.dtype == kBF16)
      quantize_rows<kBF16>(part, i);
    else
      quantize_rows<kF32>(part, i);
    return;
  }
  const int64_t wave = first * (kThreads / 64) + (threadIdx.x >> 6);
  if (wave >= part.tiles) return;
  if (part.dtype == kBF16)
    quantize_both<kBF16, 1>(part, wave, threadIdx.x & 63);
  else
    quantize_both<kF32, 1>(part, wave, threadIdx.x & 63);
}

// max(|a|, |b|, |c|), NaN if any is one.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The gradients of a gated block's projections, z_gate and z_up [m, n]:
//   dz_gate = dh z_up silu'(z_gate),  dz_up = dh silu(z_gate)
// encoded along their columns as [dz_gate | dz_up] (`along`) and along their rows
// as their transposes, stacked (`across`). A wave takes 32 rows of 128 columns, a
// thread two columns of them: whole blocks of the transposes, in registers; sixteen
// lanes share a block along the columns, row by row.
//
// What bounds it is both memory (6 bytes read and 2.1 written a pair of gradients)
// and the 55 VALU operations that a pair takes here, four of them transcendental,
// so the bookkeeping is kept small: one exponential a pair, a maximum that takes two
// new values an operation, no test for infinities and NaN but one of the whole tile
// (the tile is then encoded again, with the tests).
constexpr int kGatedWaves = 4;
constexpr int kGatedThreads = 64 * kGatedWaves;

// What a workgroup's waves have of 128 columns of both transposes: 64 bytes of a row of
// codes, padded by 16 for the banks, and four of its scales.
struct __align__(16) GatedAcross {
  uint8_t codes[2][128][kGatedWaves * 16 + 16];
  uint8_t scales[2][128][kGatedWaves];
};

template <int DTYPE, bool WHOLE, bool PAIRS>
struct GatedTile {
  static constexpr int WORDS = DTYPE == kBF16 ? 1 : 2;
  static constexpr int CHUNK = 4;  // rows loaded at a time, one chunk ahead
  const uint8_t* src[3];  // row 0 of the tile of dh, z_gate and z_up
  int64_t stride;         // bytes
  int left;               // rows of the tile
  uint32_t at[2];         // byte offsets of the thread's columns
  uint32_t in_column[WORDS];
  uint32_t raw[2][CHUNK][3][WORDS];
  float d[2][2][32];  // [gate, up][column][row]

  __device__ __forceinline__ void load(int chunk) {
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
      int row = chunk * CHUNK + i;
      if (!WHOLE) row = row < left ? row : left > 0 ? left - 1 : 0;  // past the end: the last
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        const uint8_t* p = src[t] + row * stride;
        uint32_t(&to)[WORDS] = raw[chunk & 1][i][t];
        if constexpr (DTYPE != kBF16) {
          to[0] = *reinterpret_cast<const uint32_t*>(p + at[0]);
          to[1] = *reinterpret_cast<const uint32_t*>(p + at[1]);
        } else if constexpr (PAIRS) {
          to[0] = *reinterpret_cast<const uint32_t*>(p + at[0]);
        } else {
          to[0] = *reinterpret_cast<const uint16_t*>(p + at[0]) |
                  static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + at[1])) << 16;
        }
      }
    }
  }

  __device__ __forceinline__ void gradients(int chunk) {
    auto value = [](const uint32_t(&w)[WORDS], int e) {
      if constexpr (DTYPE == kBF16)
        return e == 0 ? bf16lo_to_f32(w[0]) : bf16hi_to_f32(w[0]);
      else
        return as_f32(w[e]);
    };
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
      const int row = chunk * CHUNK + i;
      uint32_t(&w)[3][WORDS] = raw[chunk & 1][i];
      if constexpr (!WHOLE) {  // zeros where the tile ends, which have zero gradients
        const uint32_t in_row = static_cast<uint32_t>((row - left) >> 31);
#pragma unroll
        for (int t = 0; t < 3; ++t)
#pragma unroll
          for (int e = 0; e < WORDS; ++e) w[t][e] &= in_row & in_column[e];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        act_silu_mul_grads(value(w[0], e), value(w[1], e), value(w[2], e), &d[0][e][row],
                           &d[1][e][row]);
    }
  }

  // Rows `from` ... `from` + ROWS - 1 along the columns. TEST: with the scale NaN for
  // blocks that are not finite. Returns the largest magnitude's bits of the blocks.
  template <int ROWS, bool TEST>
  __device__ __forceinline__ uint32_t encode_along(const MxOut& o, int64_t r0, int64_t c, int lane,
                                                   int from, uint32_t (&kept)[2]) const {
    uint32_t seen = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int row = from + i;
        const float x = d[z][0][row], y = d[z][1][row];
        const uint32_t top = block_max<16>(__builtin_bit_cast(uint32_t, max_abs(x, y, y)));
        seen = top > seen ? top : seen;
        // the scale's exponent field, in place
        uint32_t field = top & 0x7F800000u;
        field = (field > 0x01000000u ? field : 0x01000000u) - 0x01000000u;
        uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x, y, as_f32(field), 0);
        uint32_t byte = field >> 23;
        if (TEST && top >= 0x7F800000u) {
          code = 0;
          byte = 255;
        }
        const int64_t half = o.row_bytes / 2;  // bytes of one projection's columns
        if (WHOLE || row < left)
          (o.codes + (r0 + row) * o.row_bytes + z * half)[static_cast<uint32_t>(c) / 2] =
              static_cast<uint8_t>(code);
        kept[z] = (lane & 15) == row % 16 ? byte : kept[z];
        if (row % 16 == 15)
          *mx_scale_at(o, r0 + row - 15 + (lane & 15), (z * 2 * half + c) / kMxBlock) =
              static_cast<uint8_t>(kept[z]);
      }
    return seen;
  }

  __device__ __forceinline__ void run(const MxOut& along, bool to_across, int64_t r0, int64_t c,
                                      int lane, int wave, GatedAcross& staged) {
    uint32_t kept[2] = {0, 0};  // this lane's share of the scales of sixteen rows
    uint32_t seen = 0;
    const bool to_along = along.codes != nullptr && left > 0;
    load(0);
#pragma unroll
    for (int chunk = 0; chunk < 32 / CHUNK; ++chunk) {
      if (chunk + 1 < 32 / CHUNK) load(chunk + 1);
      __builtin_amdgcn_sched_barrier(0);
      gradients(chunk);
      if (to_along) {
        const uint32_t top =
            encode_along<CHUNK, false>(along, r0, c, lane, chunk * CHUNK, kept);
        seen = top > seen ? top : seen;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (to_along && __any(seen >= 0x7F800000u)) encode_along<32, true>(along, r0, c, lane, 0, kept);
    if (!to_across) return;
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float* v = d[z][e];
        float top = max_abs(v[0], v[1], v[1]);
#pragma unroll
        for (int i = 2; i < kMxBlock; i += 2) top = max_abs(top, v[i], v[i + 1]);
        const uint32_t byte = mx_scale_byte(__builtin_bit_cast(uint32_t, top));
        const float scale = mx_scale_operand(byte);
        u32x4_t code = {mx_encode8(v, scale), mx_encode8(v + 8, scale), mx_encode8(v + 16, scale),
                        mx_encode8(v + 24, scale)};
        if (byte == 255u) code = u32x4_t{0, 0, 0, 0};
        *reinterpret_cast<u32x4_t*>(staged.codes[z][2 * lane + e] + 16 * wave) = code;
        staged.scales[z][2 * lane + e][wave] = static_cast<uint8_t>(byte);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
};

template <int DTYPE, bool PAIRS>
__global__ void __launch_bounds__(kGatedThreads) __attribute__((amdgpu_waves_per_eu(2)))
    k_mx_gated_backward(const void* __restrict__ dh, const void* __restrict__ z_gate,
                        const void* __restrict__ z_up, int64_t m, int64_t n, int64_t per,
                        int64_t rows, MxOut along, MxOut across) {
  // The waves of a workgroup take consecutive rows of the same columns, and what they
  // have of the transposes meets in LDS, to be stored 64 bytes of a row of codes at a
  // time: 188 us for 16384 x 6144, 205 with each wave's own stores of 16 bytes (160 and
  // 175 for the transposes alone). The wave's index is made uniform so that rows are
  // addressed from scalar registers.
  __shared__ GatedAcross staged;
  // The two groups of a slice of columns run on one XCD, whose L2 then has whole lines of
  // their scales (178 us against 188).
  const int64_t group = of_xcd(block_of_grid(), per * ceil_div(rows, 32 * kGatedWaves), 2);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int64_t first_row = group / per * (kGatedWaves * 32);
  const int64_t r0 = first_row + wave * 32;
  const int64_t tile = group % per;
  if (r0 >= rows) return;  // with transposes the whole workgroup: `rows` is padded to 256
  const int lane = threadIdx.x & 63;
  const int64_t c0 = tile * 128;
  const int64_t c = c0 + 2 * lane;
  const int64_t first = r0 < m ? r0 : m - 1;
  constexpr int SIZE = DTYPE == kBF16 ? 2 : 4;
  auto run = [&](auto whole) {
    GatedTile<DTYPE, decltype(whole)::value, PAIRS> t;
    t.src[0] = static_cast<const uint8_t*>(dh) + first * n * SIZE;
    t.src[1] = static_cast<const uint8_t*>(z_gate) + first * n * SIZE;
    t.src[2] = static_cast<const uint8_t*>(z_up) + first * n * SIZE;
    t.stride = n * SIZE;
    t.left = static_cast<int>(m - first < 32 ? m - first : 32);
    if (r0 >= m) t.left = 0;
    // columns past the end read the last ones
    const int64_t a = PAIRS ? (c < n ? c : n - 2) : (c < n ? c : n - 1);
    t.at[0] = static_cast<uint32_t>(a * SIZE);
    t.at[1] = static_cast<uint32_t>((c + 1 < n ? c + 1 : n - 1) * SIZE);
    if constexpr (DTYPE == kBF16) {
      t.in_column[0] = (c < n ? 0xFFFFu : 0u) | (c + 1 < n ? 0xFFFF0000u : 0u);
    } else {
      t.in_column[0] = c < n ? ~0u : 0u;
      t.in_column[1] = c + 1 < n ? ~0u : 0u;
    }
    t.run(along, across.codes != nullptr, r0, c, lane, wave, staged);
  };
  if constexpr (PAIRS) {
    if (r0 + 32 <= m && c0 + 128 <= n)
      run(std::true_type{});
    else
      run(std::false_type{});
  } else {
    run(std::false_type{});
  }
  if (across.codes == nullptr) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2 * 128 * 4 / kGatedThreads; ++i) {
    const int row = (i * kGatedThreads + static_cast<int>(threadIdx.x)) / 4;  // of 2 x 128
    const int piece = threadIdx.x % 4;
    const int64_t column = c0 + row % 128;
    if (column < n)
      *reinterpret_cast<u32x4_t*>(across.codes + (row / 128 * n + column) * across.row_bytes +
                                  first_row / 2 + 16 * piece) =
          *reinterpret_cast<const u32x4_t*>(staged.codes[row / 128][row % 128] + 16 * piece);
  }
  {
    const int row = threadIdx.x;
    const int64_t column = c0 + row % 128;
    if (column < n)
      *reinterpret_cast<uint32_t*>(mx_scale_at(across, row / 128 * n + column,
                                               first_row / kMxBlock)) =
          *reinterpret_cast<const uint32_t*>(staged.scales[row / 128][row % 128]);
  }
  // rows of scales past the last of the stack
  if (tile == 0 && 2 * n + lane < across.scale_rows)
    *mx_scale_at(across, 2 * n + lane, r0 / kMxBlock) = 0;
}

// Eight columns of one row per thread: a pass over memory, 6.6 us for 6144 x 2048 to bf16
// (4.8 TB/s).
template <int DTYPE>
__global__ void __launch_bounds__(kThreads)
    k_mx_dequantize(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                    int64_t rows, int64_t columns, void* __restrict__ out) {
  const int64_t i = block_of_grid() * kThreads + threadIdx.x;
  const int64_t per = ceil_div(columns, 8);
  const int64_t row = i / per;
  const int64_t c = (i % per) * 8;
  if (row >= rows) return;
  const int64_t block = c / kMxBlock;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(
      codes + row * mx_slices(columns) * kMxSliceBytes + c / 2);
  const float scale = mx_scale_operand(
      scales[((block / kMxSliceBlocks) * mx_pad_rows(rows) + row) * kMxSliceBlocks +
             block % kMxSliceBlocks]);
  float v[8];
  const f32x2_t v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
  const f32x2_t v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  const f32x2_t v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
  const f32x2_t v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  v[0] = v0[0], v[1] = v0[1], v[2] = v1[0], v[3] = v1[1];
  v[4] = v2[0], v[5] = v2[1], v[6] = v3[0], v[7] = v3[1];
  if ((columns & 7) == 0) {
    if constexpr (DTYPE == kBF16) {
      *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(out) + row * columns + c) =
          u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                  pack_bf16x2(v[6], v[7])};
    } else {
      f32x4_t* d = reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + row * columns + c);
      d[0] = f32x4_t{v[0], v[1], v[2], v[3]};
      d[1] = f32x4_t{v[4], v[5], v[6], v[7]};
    }
    return;
  }
  for (int e = 0; e < 8 && c + e < columns; ++e) {
    if constexpr (DTYPE == kBF16)
      static_cast<uint16_t*>(out)[row * columns + c + e] = f32_to_bf16(v[e]);
    else
      static_cast<float*>(out)[row * columns + c + e] = v[e];
  }
}

__global__ void __launch_bounds__(kThreads) k_mx_zero(uint8_t* out, int64_t bytes) {
  const int64_t i = (block_of_grid() * kThreads + threadIdx.x) * 2;
  if (i < bytes) *reinterpret_cast<uint16_t*>(out + i) = 0;
}

}  // namespace

hipError_t launch_mx_zero(void* out, int64_t bytes, hipStream_t stream) {
  if (bytes == 0) return hipSuccess;
  hipLaunchKernelGGL(k_mx_zero, grid_of(ceil_div(bytes, 2 * kThreads)), dim3(kThreads), 0, stream,
                     static_cast<uint8_t*>(out), bytes);
  return hipGetLastError();
}

// One launch for the parts encoded along both axes of each type and size class, one
// for those along their columns only.
hipError_t launch_mx_quantize(MxParts parts, int count, hipStream_t stream) {
  // waves of 128 rows of 16 pieces of `cols` columns
  auto tiles_of = [](const MxPart& part, int cols) {
    return mx_slices(part.rows) * 2 * mx_tiles_of_row(part, 16 * cols);
  };
  int64_t bf16_waves = 0, f32_waves = 0;
  for (int p = 0; p < count; ++p) {
    const MxPart& part = parts.part[p];
    if (part.across.codes == nullptr) continue;
    if (part.dtype == kBF16)
      bf16_waves += tiles_of(part, 8);
    else
      f32_waves += tiles_of(part, 4);
  }
  const bool both_axes = bf16_waves + f32_waves > 0;
  const bool fused = bf16_waves * kMxFusedWavesF32 + f32_waves * kMxFusedWavesBF16 >=
                     kMxFusedWavesBF16 * kMxFusedWavesF32;
  enum { kRows, kFusedF32, kFusedBF16, kApart, kKinds };
  MxParts some[kKinds] = {};
  int jobs[kKinds] = {};
  auto add = [&](int kind, const MxPart& part, int64_t blocks) {
    MxParts& to = some[kind];
    int& j = jobs[kind];
    to.part[j] = part;
    to.first[j + 1] = to.first[j] + blocks;
    ++j;
  };
  auto row_blocks = [](const MxPart& part) {
    return ceil_div(part.along.scale_rows * mx_slices(part.columns) *
                        (kMxSlice / (part.dtype == kBF16 ? 8 : 4)),
                    kThreads);
  };
  for (int p = 0; p < count; ++p) {
    MxPart part = parts.part[p];
    const bool bf16 = part.dtype == kBF16;
    if (part.across.codes == nullptr) {
      // beside encodings along both axes it costs no launch of its own
      add(both_axes && !fused ? kApart : kRows, part, row_blocks(part));
    } else if (fused && part.along.codes != nullptr) {
      part.tiles = tiles_of(part, bf16 ? 8 : 4);
      add(bf16 ? kFusedBF16 : kFusedF32, part, ceil_div(part.tiles, kThreads / 64));
    } else {
      MxPart across = part;
      across.along = MxOut{};
      across.tiles = tiles_of(across, bf16 ? 2 : 1);
      add(kApart, across, ceil_div(across.tiles, kThreads / 64));
      if (part.along.codes != nullptr) {
        part.across = MxOut{};
        add(kApart, part, row_blocks(part));
      }
    }
  }
  for (int kind = 0; kind < kKinds; ++kind) {
    if (jobs[kind] == 0) continue;
    const int64_t total = some[kind].first[jobs[kind]];
    for (int j = jobs[kind]; j < kMxParts; ++j) some[kind].first[j + 1] = total;
    auto* kernel = kind == kRows        ? k_mx_quantize_rows
                   : kind == kFusedF32  ? k_mx_quantize_both<kF32>
                   : kind == kFusedBF16 ? k_mx_quantize_both<kBF16>
                                        : k_mx_quantize_apart;
    hipLaunchKernelGGL(kernel, grid_of(total), dim3(kThreads), 0, stream, some[kind]);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_mx_gated_backward(const void* dh, const void* z_gate, const void* z_up, int dtype,
                                    int64_t m, int64_t n, MxOut along, MxOut across,
                                    hipStream_t stream) {
  const int64_t per =
      along.codes != nullptr ? mx_slices(n) * (kMxSlice / 128) : ceil_div(n, 128);
  // rows that something is written for
  const int64_t rows =
      across.codes != nullptr ? mx_slices(m) * kMxSlice : mx_pad_rows(m);
  const int64_t groups = per * ceil_div(rows, 32 * kGatedWaves);
  if (groups == 0) return hipSuccess;
  auto* kernel = dtype == kBF16 ? (n % 2 == 0 ? k_mx_gated_backward<kBF16, true>
                                              : k_mx_gated_backward<kBF16, false>)
                                : (n % 2 == 0 ? k_mx_gated_backward<kF32, true>
                                              : k_mx_gated_backward<kF32, false>);
  hipLaunchKernelGGL(kernel, grid_of(groups), dim3(kGatedThreads), 0, stream, dh, z_gate, z_up, m,
                     n, per, rows, along, across);
  return hipGetLastError();
}

hipError_t launch_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                int64_t columns, void* out, int dtype, hipStream_t stream) {
  const int64_t threads = rows * ceil_div(columns, 8);
  if (threads == 0) return hipSuccess;
  const dim3 grid = grid_of(ceil_div(threads, kThreads));
  if (dtype == kBF16)
    hipLaunchKernelGGL(k_mx_dequantize<kBF16>, grid, dim3(kThreads), 0, stream, codes, scales, rows,
                       columns, out);
  else
    hipLaunchKernelGGL(k_mx_dequantize<kF32>, grid, dim3(kThreads), 0, stream, codes, scales, rows,
                       columns, out);
  return hipGetLastError();
}

}  // namespace rpx

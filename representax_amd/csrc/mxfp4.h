// MXFP4: the OCP microscaled 4-bit format (Microscaling Formats specification
// v1.0) as the kernels of this library hold it. A matrix [rows, columns] has
// blocks of 32 consecutive columns of one row; a block's values are 2^e times
// 4-bit e2m1 numbers (sign, and 0, 0.5, 1, 1.5, 2, 3, 4 or 6):
//   e     = max(floor(log2(max |v|)) - 2, -127), so the largest value lands in
//           [4, 8); an all-zero block takes e = -127
//   code  = v / 2^e rounded to nearest, ties to the even code, at most 6
// A block with an infinity or a NaN gets the scale NaN and zero codes: all of
// it stands for NaN, and so does every sum that it enters.
//
// In memory:
//   codes  uint8 [rows, C / 2], C = columns rounded up to 256; column 2 j in
//          the low half of byte j, zeros past the end. 256 columns (a slice)
//          are 128 bytes: a row of an LDS stage and one line of the L2.
//   scales uint8 [C / 256, R, 8], R = rows rounded up to 32: block b of row i
//          at [b / 8, i, b % 8], e + 127 (255: NaN). A tile's scales of one
//          slice are contiguous, and a lane's four scales of the slice (below)
//          are one aligned word. Blocks and rows past the end are zero.
//
// Every product contracts the columns of two such matrices on the scaled f8f6f4
// MFMA. Its lane l takes 32 values of one block (16 bytes) of row l % 32 (or
// l % 16), and that block's scale byte from one of the four bytes of a register.
// The order of a slice's blocks is free, as long as both operands take the same
// one: with the 32x32x64 form, step s of a slice gives half h (lanes 32 h ...)
// block 4 h + s, so that bytes 4 h ... 4 h + 3 of a row's eight scales are the
// lane's word and step s picks byte s of it. Measured on this card: the
// conversions below are exact over every exponent, and the MFMA's sums are exact
// where the scales of a block are within a factor of 16 of each other and 5e-8
// off (a float32 chain 2e-7) where they differ by up to 2^40.
#pragma once

#include "common.h"

namespace rpx {

constexpr int kMxBlock = 32;
constexpr int kMxSlice = 256;      // columns per slice
constexpr int kMxSliceBytes = 128;
constexpr int kMxSliceBlocks = 8;
constexpr int kMxRowPad = 32;
constexpr int kMxFp4 = 4;  // the f8f6f4 MFMA's code for e2m1 operands

__host__ __device__ inline int64_t mx_slices(int64_t columns) {
  return ceil_div(columns, kMxSlice);
}
__host__ __device__ inline int64_t mx_pad_rows(int64_t rows) {
  return ceil_div(rows, kMxRowPad) * kMxRowPad;
}
__host__ __device__ inline int64_t mx_code_bytes(int64_t rows, int64_t columns) {
  return rows * mx_slices(columns) * kMxSliceBytes;
}
__host__ __device__ inline int64_t mx_scale_bytes(int64_t rows, int64_t columns) {
  return mx_slices(columns) * mx_pad_rows(rows) * kMxSliceBlocks;
}

// Where an encoded matrix goes. scale_rows: the R of its scales.
struct MxOut {
  uint8_t* codes;
  uint8_t* scales;
  int64_t row_bytes;
  int64_t scale_rows;
};
__device__ __forceinline__ uint8_t* mx_scale_at(const MxOut& o, int64_t row, int64_t block) {
  return o.scales + ((block / kMxSliceBlocks) * o.scale_rows + row) * kMxSliceBlocks +
         block % kMxSliceBlocks;
}

// The scale byte of a block from the largest |v|'s float32 bits (as an
// unsigned integer maximum over the values' bits without their signs, which
// orders magnitudes and puts infinities and NaN on top).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  const uint32_t field = amax_bits >> 23;
  return field == 255u ? 255u : (field < 2u ? 2u : field) - 2u;
}
// The float32 whose exponent field is the scale byte: what the conversions take.
__device__ __forceinline__ float mx_scale_operand(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

// Eight values as one word of codes (value i in bits [4 i, 4 i + 4)).
__device__ __forceinline__ uint32_t mx_encode8(const float* v, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}
// By value: a bit cast of a vector's element would read the vector's first.
__device__ __forceinline__ bf16x2_t mx_as_bf16x2(uint32_t w) {
  return __builtin_bit_cast(bf16x2_t, w);
}
__device__ __forceinline__ uint32_t mx_encode8(u32x4_t bf16s, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_as_bf16x2(bf16s[0]), scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_as_bf16x2(bf16s[1]), scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_as_bf16x2(bf16s[2]), scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_as_bf16x2(bf16s[3]), scale, 3);
  return w;
}

// A block of 32 float32 values in registers: its codes, and its scale byte.
__device__ __forceinline__ u32x4_t mx_encode_block(const float* v, uint32_t* byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kMxBlock; ++i) {
    const uint32_t a = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
    top = a > top ? a : top;
  }
  const uint32_t b = mx_scale_byte(top);
  *byte = b;
  if (b == 255u) return u32x4_t{0, 0, 0, 0};
  const float scale = mx_scale_operand(b);
  return u32x4_t{mx_encode8(v, scale), mx_encode8(v + 8, scale), mx_encode8(v + 16, scale),
                 mx_encode8(v + 24, scale)};
}

// One step of a product: a and b are 16 bytes of codes per lane; SA and SB say
// which byte of the scale words belongs to this step.
template <int SA, int SB>
__device__ __forceinline__ f32x16_t mx_mfma32(u32x4_t a, uint32_t sa, u32x4_t b, uint32_t sb,
                                              f32x16_t c) {
  const i32x8_t av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, kMxFp4, kMxFp4, SA, (int)sa, SB,
                                                         (int)sb);
}

}  // namespace rpx

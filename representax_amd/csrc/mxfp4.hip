// Encoding to MXFP4 and back (mxfp4.h states the format).
#include <hip/hip_runtime.h>

#include "act.h"
#include "kernels.h"
#include "mxfp4.h"

namespace rpx {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load_f32(const void* p, int dtype, int64_t i) {
  return dtype == kBF16 ? bf16_to_f32(static_cast<const uint16_t*>(p)[i])
                        : static_cast<const float*>(p)[i];
}

// Codes and scale of one block; rows past the end have a scale only (zero).
__device__ __forceinline__ void store_block(const MxOut& o, int64_t row, int64_t rows,
                                            int64_t block, const float* v) {
  uint32_t byte = 0;
  if (row < rows) {
    const u32x4_t c = mx_encode_block(v, &byte);
    *reinterpret_cast<u32x4_t*>(o.codes + row * o.row_bytes + block * 16) = c;
  }
  *mx_scale_at(o, row, block) = static_cast<uint8_t>(byte);
}

// One thread per block.
__global__ void __launch_bounds__(kThreads) k_mx_quantize(MxParts parts) {
  const int64_t blk = block_of_grid();
  if (blk >= parts.first[kMxParts]) return;
  int p = 0;
  while (blk >= parts.first[p + 1]) ++p;
  const MxPart& part = parts.part[p];
  const int64_t i = (blk - parts.first[p]) * kThreads + threadIdx.x;
  const int64_t nblocks = mx_slices(part.columns) * kMxSliceBlocks;
  const int64_t row = i / nblocks;
  const int64_t block = i % nblocks;
  if (row >= part.out.scale_rows) return;
  float v[kMxBlock];
#pragma unroll
  for (int j = 0; j < kMxBlock; ++j) {
    const int64_t c = block * kMxBlock + j;
    v[j] = row < part.rows && c < part.columns
               ? load_f32(part.t, part.dtype, row * part.row_stride + c * part.column_stride)
               : 0.0f;
  }
  store_block(part.out, row, part.rows, block, v);
}

// The gradients of a gated block's projections, z_gate and z_up [m, n]:
//   dz_gate = dh z_up silu'(z_gate),  dz_up = dh silu(z_gate)
// encoded along their columns as [dz_gate | dz_up] (`along`, the second half
// at `up_block` blocks) and along their rows as their transposes, stacked.
__global__ void __launch_bounds__(kThreads)
    k_mx_gated_backward(const void* dh, const void* z_gate, const void* z_up, int dtype, int64_t m,
                        int64_t n, MxOut along, MxOut stacked) {
  const int64_t i = block_of_grid() * kThreads + threadIdx.x;
  const int64_t nblocks = mx_slices(n) * kMxSliceBlocks;
  const int64_t mblocks = mx_slices(m) * kMxSliceBlocks;
  const int64_t first = along.codes == nullptr ? 0 : along.scale_rows * 2 * nblocks;
  const bool transposed = i >= first;
  const int64_t q = transposed ? i - first : i;
  const int64_t per = transposed ? mblocks : 2 * nblocks;
  const int64_t row = q / per;
  const int64_t block = q % per;
  const MxOut& o = transposed ? stacked : along;
  const int64_t rows = transposed ? 2 * n : m;
  if (o.codes == nullptr || row >= o.scale_rows) return;
  float v[kMxBlock];
#pragma unroll
  for (int j = 0; j < kMxBlock; ++j) {
    int64_t r, c;
    bool up;
    if (transposed) {
      up = row >= n;
      r = block * kMxBlock + j;
      c = up ? row - n : row;
    } else {
      up = block >= nblocks;
      r = row;
      c = (up ? block - nblocks : block) * kMxBlock + j;
    }
    v[j] = 0.0f;
    if (row < rows && r < m && c < n) {
      const int64_t at = r * n + c;
      float second;
      const float g = load_f32(z_gate, dtype, at);
      const float d = act_apply<kActSiluMulBwd>(load_f32(dh, dtype, at), g,
                                                load_f32(z_up, dtype, at), &second);
      v[j] = up ? d : second;
    }
  }
  store_block(o, row, rows, block, v);
}

// Eight columns of one row per thread.
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

hipError_t launch_mx_quantize(MxParts parts, int count, hipStream_t stream) {
  parts.first[0] = 0;
  for (int p = 0; p < kMxParts; ++p) {
    int64_t threads = 0;
    if (p < count)
      threads = parts.part[p].out.scale_rows * mx_slices(parts.part[p].columns) * kMxSliceBlocks;
    parts.first[p + 1] = parts.first[p] + ceil_div(threads, kThreads);
  }
  if (parts.first[kMxParts] == 0) return hipSuccess;
  hipLaunchKernelGGL(k_mx_quantize, grid_of(parts.first[kMxParts]), dim3(kThreads), 0, stream,
                     parts);
  return hipGetLastError();
}

hipError_t launch_mx_gated_backward(const void* dh, const void* z_gate, const void* z_up, int dtype,
                                    int64_t m, int64_t n, MxOut along, MxOut stacked,
                                    hipStream_t stream) {
  const int64_t threads =
      (along.codes == nullptr ? 0 : along.scale_rows * 2 * mx_slices(n) * kMxSliceBlocks) +
      (stacked.codes == nullptr ? 0 : stacked.scale_rows * mx_slices(m) * kMxSliceBlocks);
  if (threads == 0) return hipSuccess;
  hipLaunchKernelGGL(k_mx_gated_backward, grid_of(ceil_div(threads, kThreads)), dim3(kThreads), 0,
                     stream, dh, z_gate, z_up, dtype, m, n, along, stacked);
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

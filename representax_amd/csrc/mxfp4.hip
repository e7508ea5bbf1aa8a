// Encoding to MXFP4 and back (mxfp4.h states the format).
#include <hip/hip_runtime.h>

#include "act.h"
#include "kernels.h"
#include "mxfp4.h"

namespace rpx {

namespace {

constexpr int kThreads = 256;

// Maximum over the four (or, EIGHT, eight) neighbouring lanes that share a block.
template <bool EIGHT>
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  auto with = [](uint32_t x, uint32_t y) { return y > x ? y : x; };
  v = with(v, __builtin_amdgcn_update_dpp(0u, v, 0xB1, 0xF, 0xF, false));  // lane ^ 1
  v = with(v, __builtin_amdgcn_update_dpp(0u, v, 0x4E, 0xF, 0xF, false));  // lane ^ 2
  if constexpr (EIGHT)
    v = with(v, __builtin_amdgcn_update_dpp(0u, v, 0x141, 0xF, 0xF, false));  // 7 - lane
  return v;
}

__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a),
                                                                __builtin_bit_cast(u16x2_t, b)));
}

// What a thread reads of one row: 16 bytes, VPT values.
template <int DTYPE>
struct Piece {
  static constexpr int VPT = DTYPE == kBF16 ? 8 : 4;
  static constexpr bool EIGHT = DTYPE != kBF16;  // lanes per block: 32 / VPT
  u32x4_t w;

  // Columns c .. c + VPT - 1; zeros outside [0, columns). ALIGNED: 16-byte loads
  // may be used.
  __device__ __forceinline__ void load(const void* row, int64_t c, int64_t columns, bool aligned) {
    const uint8_t* p = static_cast<const uint8_t*>(row) + c * (16 / VPT);
    if (aligned && c + VPT <= columns) {
      w = *reinterpret_cast<const u32x4_t*>(p);
      return;
    }
    w = u32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
      if (c + e >= columns) continue;
      if constexpr (DTYPE == kBF16)
        w[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[e]) << (16 * (e & 1));
      else
        w[e] = reinterpret_cast<const uint32_t*>(p)[e];
    }
  }

  // Largest magnitude's float32 bits (an integer maximum: infinities and NaN on top).
  __device__ __forceinline__ uint32_t amax() const {
    if constexpr (DTYPE == kBF16) {
      const uint32_t m = 0x7FFF7FFFu;
      const uint32_t a = pk_max(pk_max(w[0] & m, w[1] & m), pk_max(w[2] & m, w[3] & m));
      return (a << 16) > (a & 0xFFFF0000u) ? a << 16 : a & 0xFFFF0000u;
    } else {
      uint32_t a = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) a = (w[e] & 0x7FFFFFFFu) > a ? w[e] & 0x7FFFFFFFu : a;
      return a;
    }
  }

  // VPT codes (4 VPT bits).
  __device__ __forceinline__ uint32_t encode(uint32_t byte) const {
    const float scale = mx_scale_operand(byte);
    uint32_t c;
    if constexpr (DTYPE == kBF16) {
      c = mx_encode8(w, scale);
    } else {
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, as_f32(w[0]), as_f32(w[1]), scale, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, as_f32(w[2]), as_f32(w[3]), scale, 1);
    }
    return byte == 255u ? 0u : c;
  }

  static __device__ __forceinline__ float as_f32(uint32_t v) { return __builtin_bit_cast(float, v); }
};

template <int DTYPE>
__device__ __forceinline__ void store_piece(uint8_t* codes, int64_t c, uint32_t code) {
  if constexpr (DTYPE == kBF16)
    *reinterpret_cast<uint32_t*>(codes + c / 2) = code;
  else
    *reinterpret_cast<uint16_t*>(codes + c / 2) = static_cast<uint16_t>(code);
}

// Along the columns only: a thread takes 16 bytes of a row, neighbouring lanes a
// block. A pass over memory (serving: the input of a product).
template <int DTYPE>
__device__ __forceinline__ void quantize_rows(const MxPart& part, int64_t i) {
  using P = Piece<DTYPE>;
  const int64_t per = mx_slices(part.columns) * (kMxSlice / P::VPT);
  const int64_t row = i / per;
  const int64_t c = (i % per) * P::VPT;
  if (row >= part.along.scale_rows) return;  // whole blocks: `per` is a multiple of their lanes
  P v;
  v.w = u32x4_t{0, 0, 0, 0};
  if (row < part.rows)
    v.load(static_cast<const uint8_t*>(part.t) + row * part.row_stride * (16 / P::VPT), c,
           part.columns, part.aligned);
  const uint32_t byte = row < part.rows ? mx_scale_byte(block_max<P::EIGHT>(v.amax())) : 0u;
  if (row < part.rows)
    store_piece<DTYPE>(part.along.codes + row * part.along.row_bytes, c, v.encode(byte));
  if (c % kMxBlock == 0) *mx_scale_at(part.along, row, c / kMxBlock) = static_cast<uint8_t>(byte);
}

__global__ void __launch_bounds__(kThreads) k_mx_quantize_rows(MxParts parts) {
  const int64_t blk = block_of_grid();
  if (blk >= parts.first[kMxParts]) return;
  int p = 0;
  while (blk >= parts.first[p + 1]) ++p;
  const int64_t i = (blk - parts.first[p]) * kThreads + threadIdx.x;
  if (parts.part[p].dtype == kBF16)
    quantize_rows<kBF16>(parts.part[p], i);
  else
    quantize_rows<kF32>(parts.part[p], i);
}

// Along both axes from one read. A thread owns 32 rows of its 16 bytes: whole
// blocks of the transpose, in registers, so nothing goes through LDS; a block
// along the columns is shared by neighbouring lanes as above. A wave covers 128
// rows of 16 pieces, so that its stores of either encoding are 64 contiguous bytes
// of a row of codes.
template <int DTYPE>
__device__ __forceinline__ void quantize_both(const MxPart& part, int64_t tile, int lane) {
  using P = Piece<DTYPE>;
  constexpr int COLS = 16 * P::VPT;
  const int64_t per = ceil_div(part.along.codes != nullptr ? mx_slices(part.columns) * kMxSlice
                                                           : part.columns, COLS);
  const int64_t r0 = (tile / per) * 128 + (lane >> 4) * 32;
  const int64_t c = (tile % per) * COLS + (lane & 15) * P::VPT;
  P v[32];
  const uint8_t* base =
      static_cast<const uint8_t*>(part.t) + r0 * part.row_stride * (16 / P::VPT);
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i].w = u32x4_t{0, 0, 0, 0};
    if (r0 + i < part.rows)
      v[i].load(base + i * part.row_stride * (16 / P::VPT), c, part.columns, part.aligned);
  }
  if (part.along.codes != nullptr && r0 < part.along.scale_rows) {
    uint32_t kept = 0;  // the scale of this lane's share of four (eight) rows
    constexpr int LANES = kMxBlock / P::VPT;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const uint32_t byte = mx_scale_byte(block_max<P::EIGHT>(v[i].amax()));
      if (r0 + i < part.rows)
        store_piece<DTYPE>(part.along.codes + (r0 + i) * part.along.row_bytes, c,
                           v[i].encode(byte));
      if ((lane & (LANES - 1)) == i % LANES) kept = byte;
      if (i % LANES == LANES - 1)
        *mx_scale_at(part.along, r0 + i - (LANES - 1) + (lane & (LANES - 1)), c / kMxBlock) =
            static_cast<uint8_t>(kept);
    }
  }
  if (part.across.codes == nullptr) return;
  if constexpr (DTYPE == kBF16) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // columns c + 2 q and c + 2 q + 1
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) top = pk_max(top, v[i].w[q] & 0x7FFF7FFFu);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const int64_t col = c + 2 * q + odd;
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
        if (col < part.columns)
          *reinterpret_cast<u32x4_t*>(part.across.codes + col * part.across.row_bytes + r0 / 2) =
              code;
        if (col < part.across.scale_rows)
          *mx_scale_at(part.across, col, r0 / kMxBlock) = static_cast<uint8_t>(byte);
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t col = c + q;
      float x[kMxBlock];
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = P::as_f32(v[i].w[q]);
      uint32_t byte;
      const u32x4_t code = mx_encode_block(x, &byte);
      if (col < part.columns)
        *reinterpret_cast<u32x4_t*>(part.across.codes + col * part.across.row_bytes + r0 / 2) = code;
      if (col < part.across.scale_rows)
        *mx_scale_at(part.across, col, r0 / kMxBlock) = static_cast<uint8_t>(byte);
    }
  }
}

template <int DTYPE>
__global__ void __launch_bounds__(kThreads) k_mx_quantize_both(MxParts parts) {
  const int64_t blk = block_of_grid();
  if (blk >= parts.first[kMxParts]) return;
  int p = 0;
  while (blk >= parts.first[p + 1]) ++p;
  const int64_t wave = (blk - parts.first[p]) * (kThreads / 64) + (threadIdx.x >> 6);
  if (wave >= parts.part[p].tiles) return;
  quantize_both<DTYPE>(parts.part[p], wave, threadIdx.x & 63);
}

// The gradients of a gated block's projections, z_gate and z_up [m, n]:
//   dz_gate = dh z_up silu'(z_gate),  dz_up = dh silu(z_gate)
// encoded along their columns as [dz_gate | dz_up] (`along`) and along their rows
// as their transposes, stacked (`across`). A thread owns 32 rows of two columns of
// both, as above: sixteen lanes share a block along the columns.
template <int DTYPE>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
    k_mx_gated_backward(const void* __restrict__ dh, const void* __restrict__ z_gate,
                        const void* __restrict__ z_up, int64_t m, int64_t n, int64_t per,
                        int64_t tiles, MxOut along, MxOut across) {
  // uniform over the wave, so rows are addressed from scalar registers
  const int64_t tile = block_of_grid() * (kThreads / 64) +
                       __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  if (tile >= tiles) return;
  const int lane = threadIdx.x & 63;
  const int64_t r0 = (tile / per) * 32;
  const int64_t c = (tile % per) * 128 + 2 * lane;
  float d[2][2][32];  // [gate, up][column][row]
  constexpr int CHUNK = 4;  // rows whose loads are in flight at once
  constexpr int WORDS = DTYPE == kBF16 ? 1 : 2;
  uint32_t raw[2][CHUNK][3][WORDS];
  // columns past the end read the last ones and rows past the end the last row;
  // their gradients are set to zero below
  const bool pair = (n & 1) == 0;
  const uint32_t c0 = static_cast<uint32_t>(c < n ? c : n - 1);
  const uint32_t c1 = static_cast<uint32_t>(c + 1 < n ? c + 1 : n - 1);
  const uint32_t cp = static_cast<uint32_t>(c < n ? c : n - 2);
  const uint32_t in_column[2] = {c < n ? ~0u : 0u, c + 1 < n ? ~0u : 0u};
  const int left = static_cast<int>(m - r0 < 32 ? m - r0 : 32);
  auto load = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
      const int64_t r = r0 + chunk * CHUNK + i < m ? r0 + chunk * CHUNK + i : m - 1;
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        const void* src = t == 0 ? dh : t == 1 ? z_gate : z_up;
        uint32_t(&to)[WORDS] = raw[chunk & 1][i][t];
        if constexpr (DTYPE == kBF16) {
          const uint16_t* p = static_cast<const uint16_t*>(src) + r * n;
          if (pair)
            to[0] = *reinterpret_cast<const uint32_t*>(p + cp);
          else
            to[0] = p[c0] | static_cast<uint32_t>(p[c1]) << 16;
        } else {
          const uint32_t* p = static_cast<const uint32_t*>(src) + r * n;
          to[0] = p[c0];
          to[1] = p[c1];
        }
      }
    }
  };
  auto value = [](const uint32_t(&w)[WORDS], int e) {
    if constexpr (DTYPE == kBF16)
      return e == 0 ? bf16lo_to_f32(w[0]) : bf16hi_to_f32(w[0]);
    else
      return __builtin_bit_cast(float, w[e]);
  };
  // scale byte of a block of sixteen lanes
  auto along_byte = [](float x, float y) {
    const uint32_t a = __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu;
    const uint32_t b = __builtin_bit_cast(uint32_t, y) & 0x7FFFFFFFu;
    const uint32_t h = block_max<true>(a > b ? a : b);
    const uint32_t o = __builtin_amdgcn_update_dpp(0u, h, 0x140, 0xF, 0xF, false);  // 15 - lane
    return mx_scale_byte(o > h ? o : h);
  };
  uint32_t kept[2] = {0, 0};  // this lane's share of the scales of sixteen rows
  load(0);
#pragma unroll
  for (int chunk = 0; chunk < 32 / CHUNK; ++chunk) {
    if (chunk + 1 < 32 / CHUNK) load(chunk + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < CHUNK; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = chunk * CHUNK + i;
        float gate;
        const float up =
            act_apply<kActSiluMulBwd>(value(raw[chunk & 1][i][0], e), value(raw[chunk & 1][i][1], e),
                                      value(raw[chunk & 1][i][2], e), &gate);
        // all ones where the row is below m and the column below n
        const uint32_t in = static_cast<uint32_t>((row - left) >> 31) & in_column[e];
        d[0][e][row] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, gate) & in);
        d[1][e][row] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, up) & in);
      }
    if (along.codes != nullptr && left > 0) {
#pragma unroll
      for (int i = 0; i < CHUNK; ++i)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int row = chunk * CHUNK + i;
          const uint32_t byte = along_byte(d[z][0][row], d[z][1][row]);
          const uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(
              0u, d[z][0][row], d[z][1][row], mx_scale_operand(byte), 0);
          if (row < left)
            along.codes[(r0 + row) * along.row_bytes + z * (along.row_bytes / 2) + c / 2] =
                static_cast<uint8_t>(byte == 255u ? 0u : code);
          kept[z] = (lane & 15) == row % 16 ? byte : kept[z];
          if (row % 16 == 15)
            *mx_scale_at(along, r0 + row - 15 + (lane & 15), (z * along.row_bytes + c) / kMxBlock) =
                static_cast<uint8_t>(kept[z]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (across.codes == nullptr) return;
#pragma unroll
  for (int z = 0; z < 2; ++z)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t byte;
      const u32x4_t code = mx_encode_block(d[z][e], &byte);
      if (c + e < n) {
        const int64_t row = z * n + c + e;
        *reinterpret_cast<u32x4_t*>(across.codes + row * across.row_bytes + r0 / 2) = code;
        *mx_scale_at(across, row, r0 / kMxBlock) = static_cast<uint8_t>(byte);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  // rows of scales past the last of the stack
  if (tile % per == 0 && 2 * n + lane < across.scale_rows)
    *mx_scale_at(across, 2 * n + lane, r0 / kMxBlock) = 0;
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

hipError_t launch_mx_quantize(MxParts parts, int count, hipStream_t stream) {
  // Parts along both axes (or across only) go to one launch per type, the others
  // to one more.
  for (int kind = 0; kind < 3; ++kind) {
    MxParts some{};
    int jobs = 0;
    for (int p = 0; p < count; ++p) {
      MxPart part = parts.part[p];
      const bool both = part.across.codes != nullptr;
      if (kind != (both ? (part.dtype == kBF16 ? 0 : 1) : 2)) continue;
      const int vpt = part.dtype == kBF16 ? 8 : 4;
      const int size = part.dtype == kBF16 ? 2 : 4;
      part.aligned = (reinterpret_cast<uintptr_t>(part.t) & 15) == 0 &&
                     (part.row_stride * size) % 16 == 0;
      int64_t blocks;
      if (both) {
        const int64_t columns =
            part.along.codes != nullptr ? mx_slices(part.columns) * kMxSlice : part.columns;
        part.tiles = mx_slices(part.rows) * 2 * ceil_div(columns, 16 * vpt);
        blocks = ceil_div(part.tiles, kThreads / 64);
      } else {
        blocks = ceil_div(part.along.scale_rows * mx_slices(part.columns) * (kMxSlice / vpt),
                          kThreads);
      }
      some.part[jobs] = part;
      some.first[jobs + 1] = some.first[jobs] + blocks;
      ++jobs;
    }
    if (jobs == 0) continue;
    const int64_t total = some.first[jobs];
    for (int j = jobs; j < kMxParts; ++j) some.first[j + 1] = total;
    if (kind == 0)
      hipLaunchKernelGGL(k_mx_quantize_both<kBF16>, grid_of(total), dim3(kThreads), 0, stream, some);
    else if (kind == 1)
      hipLaunchKernelGGL(k_mx_quantize_both<kF32>, grid_of(total), dim3(kThreads), 0, stream, some);
    else
      hipLaunchKernelGGL(k_mx_quantize_rows, grid_of(total), dim3(kThreads), 0, stream, some);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_mx_gated_backward(const void* dh, const void* z_gate, const void* z_up, int dtype,
                                    int64_t m, int64_t n, MxOut along, MxOut across,
                                    hipStream_t stream) {
  const int64_t per =
      along.codes != nullptr ? mx_slices(n) * (kMxSlice / 128) : ceil_div(n, 128);
  const int64_t tiles =
      per * (across.codes != nullptr ? mx_slices(m) * kMxSliceBlocks : ceil_div(m, kMxBlock));
  if (tiles == 0) return hipSuccess;
  const dim3 grid = grid_of(ceil_div(tiles, kThreads / 64));
  if (dtype == kBF16)
    hipLaunchKernelGGL(k_mx_gated_backward<kBF16>, grid, dim3(kThreads), 0, stream, dh, z_gate,
                       z_up, m, n, per, tiles, along, across);
  else
    hipLaunchKernelGGL(k_mx_gated_backward<kF32>, grid, dim3(kThreads), 0, stream, dh, z_gate, z_up,
                       m, n, per, tiles, along, across);
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

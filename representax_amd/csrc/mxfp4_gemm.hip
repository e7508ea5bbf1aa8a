// Products of MXFP4 matrices: out[i, j] = sum_c A[i, c] B[j, c], and the first
// half of a gated feed-forward block, silu(A G^T) * (A U^T), from one pass over
// A. mxfp4.h states the format and the order in which a slice's blocks meet.
#include <hip/hip_runtime.h>

#include "act.h"
#include "kernels.h"
#include "mxfp4.h"

namespace rpx {

namespace {

__device__ __forceinline__ void store_as(void* out, int dtype, int64_t i, float v) {
  if (dtype == kBF16)
    static_cast<uint16_t*>(out)[i] = f32_to_bf16(v);
  else
    static_cast<float*>(out)[i] = v;
}

// One wave per 32 x 32 tile, fragments straight from memory. GATED: B is the
// gate's weight and B2 the up projection's.
template <bool GATED>
__global__ void __launch_bounds__(64) k_mx_gemm_simple(MxGemm p) {
  const int64_t tile = block_of_grid();
  const int64_t tiles_n = ceil_div(p.n, 32);
  if (tile >= ceil_div(p.m, 32) * tiles_n) return;
  const int64_t m0 = tile / tiles_n * 32;
  const int64_t n0 = tile % tiles_n * 32;
  const int lane = threadIdx.x;
  const int half = lane >> 5;
  int64_t ra = m0 + (lane & 31), rb = n0 + (lane & 31);
  ra = ra < p.m ? ra : p.m - 1;
  rb = rb < p.n ? rb : p.n - 1;
  const int64_t row_bytes = p.slices * kMxSliceBytes;
  const int64_t ra_pad = mx_pad_rows(p.m), rb_pad = mx_pad_rows(p.n);
  f32x16_t acc, acc2;
#pragma unroll
  for (int v = 0; v < 16; ++v) acc[v] = acc2[v] = 0.0f;
  for (int64_t s = 0; s < p.slices; ++s) {
    const int64_t ca = ra * row_bytes + s * kMxSliceBytes + 64 * half;
    const int64_t cb = rb * row_bytes + s * kMxSliceBytes + 64 * half;
    const int64_t sb_at = (s * rb_pad + rb) * kMxSliceBlocks + 4 * half;
    const uint32_t sa = *reinterpret_cast<const uint32_t*>(
        p.a_scales + (s * ra_pad + ra) * kMxSliceBlocks + 4 * half);
    auto a = [&](int j) { return *reinterpret_cast<const u32x4_t*>(p.a_codes + ca + 16 * j); };
    auto run = [&](const uint8_t* codes, const uint8_t* scales, f32x16_t c) {
      const uint32_t sb = *reinterpret_cast<const uint32_t*>(scales + sb_at);
      auto b = [&](int j) { return *reinterpret_cast<const u32x4_t*>(codes + cb + 16 * j); };
      c = mx_mfma32<0, 0>(b(0), sb, a(0), sa, c);
      c = mx_mfma32<1, 1>(b(1), sb, a(1), sa, c);
      c = mx_mfma32<2, 2>(b(2), sb, a(2), sa, c);
      return mx_mfma32<3, 3>(b(3), sb, a(3), sa, c);
    };
    acc = run(p.b_codes, p.b_scales, acc);
    if constexpr (GATED) acc2 = run(p.b2_codes, p.b2_scales, acc2);
  }
  // lane l holds row m0 + l % 32 and columns n0 + 8 g + 4 (l / 32) + e in acc[4 g + e]
  const int64_t m = m0 + (lane & 31);
  if (m >= p.m) return;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int64_t n = n0 + 8 * (v / 4) + 4 * half + v % 4;
    if (n >= p.n) continue;
    const int64_t at = m * p.n + n;
    if constexpr (GATED) {
      const float g = p.dtype == kBF16 ? round_bf16(acc[v]) : acc[v];
      const float u = p.dtype == kBF16 ? round_bf16(acc2[v]) : acc2[v];
      store_as(p.out, p.dtype, at, act_apply<kActSiluMulFwd>(u, g, 0.0f, nullptr));
      if (p.z_gate != nullptr) {
        store_as(p.z_gate, p.dtype, at, g);
        store_as(p.z_up, p.dtype, at, u);
      }
    } else {
      store_as(p.out, p.dtype, at, acc[v]);
    }
  }
}

}  // namespace

int64_t mx_gemm_workspace_floats(int64_t m, int64_t n, int64_t slices) { return 0; }

hipError_t launch_mx_gemm(const MxGemm& p, float* partials, hipStream_t stream) {
  const int64_t tiles = ceil_div(p.m, 32) * ceil_div(p.n, 32);
  if (tiles == 0) return hipSuccess;
  if (p.b2_codes != nullptr)
    hipLaunchKernelGGL(k_mx_gemm_simple<true>, grid_of(tiles), dim3(64), 0, stream, p);
  else
    hipLaunchKernelGGL(k_mx_gemm_simple<false>, grid_of(tiles), dim3(64), 0, stream, p);
  return hipGetLastError();
}

}  // namespace rpx

// C entry points of the MXFP4 operators: validation, workspace carving and
// launch order. None allocates device memory or synchronizes.
#include <string>

#include "../../include/representax_amd.h"
#include "capi.h"
#include "common.h"
#include "kernels.h"
#include "mxfp4.h"

namespace rpx {

namespace {

// Extents whose products (elements, workgroups) stay far from 2^63.
constexpr int64_t kMaxExtent = int64_t{1} << 30;

int check_extents(const char* who, std::initializer_list<int64_t> extents) {
  for (int64_t e : extents)
    if (e < 0 || e > kMaxExtent) return fail_invalid(std::string(who) + ": invalid extents");
  return kOk;
}

int check_pointers(const char* who, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (p == nullptr) return fail_invalid(std::string(who) + ": null pointer");
  for (const void* p : pointers)
    if (!aligned16(p))
      return fail_invalid(std::string(who) + ": pointers must be 16-byte aligned");
  return kOk;
}

// The encoded forms of x that a call makes in its workspace.
struct Encoded {
  uint8_t* codes;
  uint8_t* scales;
};

Encoded take_encoded(Arena* arena, int64_t rows, int64_t columns) {
  Encoded e;
  e.codes = arena->take<uint8_t>(mx_code_bytes(rows, columns));
  e.scales = arena->take<uint8_t>(mx_scale_bytes(rows, columns));
  return e;
}

size_t encoded_bytes(int64_t rows, int64_t columns) {
  Sizer s;
  s.take<uint8_t>(mx_code_bytes(rows, columns));
  s.take<uint8_t>(mx_scale_bytes(rows, columns));
  return s.used;
}

size_t linear_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  Sizer s;
  s.used = encoded_bytes(m, k);
  s.take<float>(mx_gemm_workspace_floats(m, n, mx_slices(k)));
  return s.used;
}

int zero_fill(void* out, int64_t m, int64_t n, int dtype, hipStream_t st, const char* who) {
  RPX_HIP(launch_mx_zero(out, m * n * static_cast<int64_t>(elem_size(dtype)), st), who);
  return kOk;
}

// x W^T, or the gated block where `up` is given, from x in the caller's dtype.
int serve(const char* who, const void* x, int dtype, int64_t m, int64_t k, int64_t row_stride,
          const uint8_t* codes, const uint8_t* scales, const uint8_t* up_codes,
          const uint8_t* up_scales, bool gated, int64_t n, void* y, void* workspace,
          size_t workspace_bytes, hipStream_t st) {
  RPX_TRY(check_dtype(dtype));
  RPX_TRY(check_extents(who, {m, n, k}));
  if (m == 0 || n == 0) return kOk;
  if (k == 0) {
    RPX_TRY(check_pointers(who, {y}));
    return zero_fill(y, m, n, dtype, st, who);
  }
  if (row_stride < k && m > 1) return fail_invalid(std::string(who) + ": rows of x overlap");
  if (x == nullptr) return fail_invalid(std::string(who) + ": null pointer");
  RPX_TRY(check_pointers(who, {codes, scales, y}));
  if (gated) RPX_TRY(check_pointers(who, {up_codes, up_scales}));
  Arena arena(workspace, workspace == nullptr ? 0 : workspace_bytes);
  const Encoded e = take_encoded(&arena, m, k);
  float* partials = gated ? nullptr : arena.take<float>(mx_gemm_workspace_floats(m, n, mx_slices(k)));
  if (arena.overflow) return fail_invalid(std::string(who) + ": workspace too small");
  RPX_TRY(check_pointers(who, {workspace}));
  MxParts parts{};
  parts.part[0] = MxPart{x, dtype, m, k, row_stride,
                         MxOut{e.codes, e.scales, mx_slices(k) * kMxSliceBytes, mx_pad_rows(m)},
                         MxOut{}, 0};
  RPX_HIP(launch_mx_quantize(parts, 1, st), who);
  const MxGemm g{e.codes, e.scales, codes, scales, up_codes, up_scales, m, n, mx_slices(k),
                 y, nullptr, nullptr, dtype};
  RPX_HIP(launch_mx_gemm(g, partials, st), who);
  return kOk;
}

}  // namespace
}  // namespace rpx

using namespace rpx;

extern "C" {

size_t rpx_mxfp4_code_bytes(int64_t rows, int64_t columns) {
  if (rows <= 0 || columns <= 0) return 0;
  return static_cast<size_t>(mx_code_bytes(rows, columns));
}

size_t rpx_mxfp4_scale_bytes(int64_t rows, int64_t columns) {
  if (rows <= 0 || columns <= 0) return 0;
  return static_cast<size_t>(mx_scale_bytes(rows, columns));
}

int rpx_mxfp4_quantize(const rpx_mxfp4_part* parts, int64_t count, void* stream) {
  const char* who = "rpx_mxfp4_quantize";
  if (count < 0 || count > kMxParts / 2)
    return fail_invalid("rpx_mxfp4_quantize: need 0 <= count <= 4");
  if (count > 0 && parts == nullptr) return fail_invalid("rpx_mxfp4_quantize: null pointer");
  MxParts args{};
  int jobs = 0;
  for (int64_t i = 0; i < count; ++i) {
    const rpx_mxfp4_part& in = parts[i];
    RPX_TRY(check_dtype(in.dtype));
    RPX_TRY(check_extents(who, {in.rows, in.columns}));
    if ((in.codes == nullptr) != (in.scales == nullptr) ||
        (in.codes_t == nullptr) != (in.scales_t == nullptr))
      return fail_invalid("rpx_mxfp4_quantize: codes and scales come together");
    if (in.rows == 0 || in.columns == 0) continue;
    if (in.codes == nullptr && in.codes_t == nullptr)
      return fail_invalid("rpx_mxfp4_quantize: no output requested");
    if (in.t == nullptr) return fail_invalid("rpx_mxfp4_quantize: null pointer");
    if (in.row_stride < in.columns && in.rows > 1)
      return fail_invalid("rpx_mxfp4_quantize: rows overlap");
    const int64_t dense = mx_slices(in.columns) * kMxSliceBytes;
    const int64_t dense_t = mx_slices(in.rows) * kMxSliceBytes;
    const int64_t stride = in.code_stride == 0 ? dense : in.code_stride;
    const int64_t stride_t = in.code_stride_t == 0 ? dense_t : in.code_stride_t;
    if (stride < dense || stride_t < dense_t || stride % 16 != 0 || stride_t % 16 != 0)
      return fail_invalid("rpx_mxfp4_quantize: invalid code stride");
    if (in.codes != nullptr) RPX_TRY(check_pointers(who, {in.codes, in.scales}));
    if (in.codes_t != nullptr) RPX_TRY(check_pointers(who, {in.codes_t, in.scales_t}));
    args.part[jobs++] =
        MxPart{in.t, in.dtype, in.rows, in.columns, in.row_stride,
               MxOut{in.codes, in.scales, stride, mx_pad_rows(in.rows)},
               MxOut{in.codes_t, in.scales_t, stride_t, mx_pad_rows(in.columns)}, 0};
  }
  RPX_HIP(launch_mx_quantize(args, jobs, static_cast<hipStream_t>(stream)), who);
  return kOk;
}

int rpx_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                         int64_t columns, void* out, int dtype, void* stream) {
  const char* who = "rpx_mxfp4_dequantize";
  RPX_TRY(check_dtype(dtype));
  RPX_TRY(check_extents(who, {rows, columns}));
  if (rows == 0 || columns == 0) return kOk;
  RPX_TRY(check_pointers(who, {codes, scales, out}));
  RPX_HIP(launch_mx_dequantize(codes, scales, rows, columns, out, dtype,
                               static_cast<hipStream_t>(stream)),
          who);
  return kOk;
}

size_t rpx_mxfp4_gemm_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  return static_cast<size_t>(mx_gemm_workspace_floats(m, n, mx_slices(k))) * sizeof(float);
}

int rpx_mxfp4_gemm(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                   const uint8_t* b_scales, int64_t m, int64_t n, int64_t k, void* out,
                   int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "rpx_mxfp4_gemm";
  RPX_TRY(check_dtype(out_dtype));
  RPX_TRY(check_extents(who, {m, n, k}));
  if (m == 0 || n == 0) return kOk;
  RPX_TRY(check_pointers(who, {out}));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (k == 0) return zero_fill(out, m, n, out_dtype, st, who);
  RPX_TRY(check_pointers(who, {a_codes, a_scales, b_codes, b_scales}));
  const size_t need = rpx_mxfp4_gemm_workspace(m, n, k);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need)
      return fail_invalid("rpx_mxfp4_gemm: workspace too small");
    RPX_TRY(check_pointers(who, {workspace}));
  }
  const MxGemm g{a_codes, a_scales, b_codes, b_scales, nullptr, nullptr, m, n, mx_slices(k),
                 out, nullptr, nullptr, out_dtype};
  RPX_HIP(launch_mx_gemm(g, static_cast<float*>(workspace), st), who);
  return kOk;
}

int rpx_mxfp4_gated_gemm(const uint8_t* a_codes, const uint8_t* a_scales,
                         const uint8_t* gate_codes, const uint8_t* gate_scales,
                         const uint8_t* up_codes, const uint8_t* up_scales, int64_t m, int64_t n,
                         int64_t k, void* h, void* z_gate, void* z_up, int dtype, void* stream) {
  const char* who = "rpx_mxfp4_gated_gemm";
  RPX_TRY(check_dtype(dtype));
  RPX_TRY(check_extents(who, {m, n, k}));
  if ((z_gate == nullptr) != (z_up == nullptr))
    return fail_invalid("rpx_mxfp4_gated_gemm: z_gate and z_up come together");
  if (m == 0 || n == 0) return kOk;
  RPX_TRY(check_pointers(who, {h}));
  if (z_gate != nullptr) RPX_TRY(check_pointers(who, {z_gate, z_up}));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (k == 0) {
    for (void* p : {h, z_gate, z_up})
      if (p != nullptr) RPX_TRY(zero_fill(p, m, n, dtype, st, who));
    return kOk;
  }
  RPX_TRY(check_pointers(who, {a_codes, a_scales, gate_codes, gate_scales, up_codes, up_scales}));
  const MxGemm g{a_codes, a_scales, gate_codes, gate_scales, up_codes, up_scales, m, n,
                 mx_slices(k), h, z_gate, z_up, dtype};
  RPX_HIP(launch_mx_gemm(g, nullptr, st), who);
  return kOk;
}

int rpx_mxfp4_gated_backward(const void* dh, const void* z_gate, const void* z_up, int dtype,
                             int64_t m, int64_t n, uint8_t* codes, uint8_t* scales,
                             uint8_t* codes_t, uint8_t* scales_t, void* stream) {
  const char* who = "rpx_mxfp4_gated_backward";
  RPX_TRY(check_dtype(dtype));
  RPX_TRY(check_extents(who, {m, n}));
  if ((codes == nullptr) != (scales == nullptr) || (codes_t == nullptr) != (scales_t == nullptr))
    return fail_invalid("rpx_mxfp4_gated_backward: codes and scales come together");
  if (m == 0 || n == 0) return kOk;
  if (codes == nullptr && codes_t == nullptr)
    return fail_invalid("rpx_mxfp4_gated_backward: no output requested");
  RPX_TRY(check_pointers(who, {dh, z_gate, z_up}));
  if (codes != nullptr) RPX_TRY(check_pointers(who, {codes, scales}));
  if (codes_t != nullptr) RPX_TRY(check_pointers(who, {codes_t, scales_t}));
  MxOut along{codes, scales, 2 * mx_slices(n) * kMxSliceBytes, mx_pad_rows(m)};
  MxOut across{codes_t, scales_t, mx_slices(m) * kMxSliceBytes, mx_pad_rows(2 * n)};
  RPX_HIP(launch_mx_gated_backward(dh, z_gate, z_up, dtype, m, n, along, across,
                                   static_cast<hipStream_t>(stream)),
          who);
  return kOk;
}

size_t rpx_mxfp4_linear_workspace(int64_t m, int64_t n, int64_t k) {
  return linear_workspace(m, n, k);
}

int rpx_mxfp4_linear(const void* x, int dtype, int64_t m, int64_t k, int64_t row_stride,
                     const uint8_t* codes, const uint8_t* scales, int64_t n, void* y,
                     void* workspace, size_t workspace_bytes, void* stream) {
  return serve("rpx_mxfp4_linear", x, dtype, m, k, row_stride, codes, scales, nullptr, nullptr,
               false, n, y, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

size_t rpx_mxfp4_gated_workspace(int64_t m, int64_t n, int64_t k) {
  return m <= 0 || n <= 0 || k <= 0 ? 0 : encoded_bytes(m, k);
}

int rpx_mxfp4_gated(const void* x, int dtype, int64_t m, int64_t k, int64_t row_stride,
                    const uint8_t* gate_codes, const uint8_t* gate_scales,
                    const uint8_t* up_codes, const uint8_t* up_scales, int64_t n, void* h,
                    void* workspace, size_t workspace_bytes, void* stream) {
  return serve("rpx_mxfp4_gated", x, dtype, m, k, row_stride, gate_codes, gate_scales, up_codes,
               up_scales, true, n, h, workspace, workspace_bytes,
               static_cast<hipStream_t>(stream));
}

}  // extern "C"

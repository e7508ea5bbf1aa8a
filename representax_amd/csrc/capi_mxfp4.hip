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

// An encoded matrix in a buffer.
struct Encoded {
  uint8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  int64_t rows = 0, columns = 0;
  MxOut out() const {
    return codes == nullptr ? MxOut{}
                            : MxOut{codes, scales, mx_slices(columns) * kMxSliceBytes,
                                    mx_pad_rows(rows)};
  }
};

// Carves an encoded matrix (or, not wanted, nothing) from an Arena, or counts its
// bytes in a Sizer.
Encoded take(Arena* a, bool wanted, int64_t rows, int64_t columns) {
  Encoded e;
  e.rows = rows;
  e.columns = columns;
  if (!wanted || rows == 0 || columns == 0) return e;
  e.codes = a->take<uint8_t>(mx_code_bytes(rows, columns));
  e.scales = a->take<uint8_t>(mx_scale_bytes(rows, columns));
  return e;
}
void take(Sizer* s, bool wanted, int64_t rows, int64_t columns) {
  if (!wanted || rows == 0 || columns == 0) return;
  s->take<uint8_t>(mx_code_bytes(rows, columns));
  s->take<uint8_t>(mx_scale_bytes(rows, columns));
}

// A B^T into out, zeros where nothing is summed; nothing for an empty output.
int product(const char* who, const Encoded& a, const Encoded& b, void* out, int dtype,
            float* partials, hipStream_t st) {
  if (a.rows == 0 || b.rows == 0) return kOk;
  if (a.columns == 0) {
    RPX_HIP(launch_mx_zero(out, a.rows * b.rows * static_cast<int64_t>(elem_size(dtype)), st), who);
    return kOk;
  }
  const MxGemm g{a.codes, a.scales, b.codes, b.scales, nullptr, nullptr, a.rows, b.rows,
                 mx_slices(a.columns), out, nullptr, nullptr, dtype};
  RPX_HIP(launch_mx_gemm(g, partials, st), who);
  return kOk;
}

// Two such products.
int products(const char* who, const Encoded& a0, const Encoded& b0, void* out0, int dtype0,
             const Encoded& a1, const Encoded& b1, void* out1, int dtype1, float* partials,
             hipStream_t st) {
  if (out0 == nullptr || out1 == nullptr || a0.columns == 0 || a1.columns == 0) {
    if (out0 != nullptr) RPX_TRY(product(who, a0, b0, out0, dtype0, partials, st));
    if (out1 != nullptr) RPX_TRY(product(who, a1, b1, out1, dtype1, partials, st));
    return kOk;
  }
  const MxGemm g0{a0.codes, a0.scales, b0.codes, b0.scales, nullptr, nullptr, a0.rows, b0.rows,
                  mx_slices(a0.columns), out0, nullptr, nullptr, dtype0};
  const MxGemm g1{a1.codes, a1.scales, b1.codes, b1.scales, nullptr, nullptr, a1.rows, b1.rows,
                  mx_slices(a1.columns), out1, nullptr, nullptr, dtype1};
  RPX_HIP(launch_mx_gemm_pair(g0, g1, partials, st), who);
  return kOk;
}

int64_t product_floats(int64_t m, int64_t n, int64_t k) {
  return m <= 0 || n <= 0 || k <= 0 ? 0 : mx_gemm_workspace_floats(m, n, mx_slices(k));
}

// A weight as its product's right operand [k, n]: row-major, or (a transposed
// view of a row-major weight [n, k]) column-major. Fills the part that encodes it
// along k into w [n, k] and, where wanted, along n into wt [k, n].
int weight_part(const char* who, const void* right, int dtype, int64_t k, int64_t n,
                int64_t row_stride, int64_t col_stride, const Encoded& w, MxOut wt, MxPart* part) {
  if (right == nullptr) return fail_invalid(std::string(who) + ": null pointer");
  if (row_stride == 1 && (col_stride >= k || n <= 1)) {
    *part = MxPart{right, dtype, n, k, n <= 1 ? k : col_stride, w.out(), wt, 0};
  } else if (col_stride == 1 && (row_stride >= n || k <= 1)) {
    *part = MxPart{right, dtype, k, n, k <= 1 ? n : row_stride, wt, w.out(), 0};
  } else {
    return fail_invalid(std::string(who) + ": one stride of the right operand must be 1, the "
                                           "other span it");
  }
  return kOk;
}

// Whether a serving call encodes x within its product's launch: up to 16 rows,
// which every workgroup (16 rows of the weight) reads, 24 MB of such reads in all.
// One launch against two, us (cold weights, graph replays; then eager calls, of which
// a launch is 4): bf16, 13 rows of 2048 to 2048, 6 MB, 4.7 / 6.3, 9.2 / 12.6; 13 of
// 2048 to 6144, 20 MB, 7.0 / 7.3, 9.1 / 12.9; 13 of 6144 to 2048, 20 MB, 8.8 / 8.2, 9.0 /
// 12.9; 16 of 6144 to 2048, 24 MB, 9.7 / 8.4, 9.4 / 14.3; float32, 8 rows of 2048 to
// 6144, 24 MB, 8.1 / 7.1, 9.1 / 14.0; 16 of 1024 to 8192, 32 MB, 6.9 / 6.6, 9.1 / 14.0; 13
// of 2048 to 6144, 39 MB, 9.3 / 7.3, 9.8 / 14.7; 16 of 6144 to 2048, 48 MB, 14.5 / 8.4, 14.5
// / 14.3.
constexpr int64_t kMxSkinnyReads = int64_t{24} << 20;
bool encodes_on_the_way(int64_t m, int64_t n, int64_t k, int dtype) {
  return m <= kMxSkinnyRows &&
         m * k * static_cast<int64_t>(elem_size(dtype)) <= kMxSkinnyReads / ceil_div(n, 16);
}

size_t serve_workspace(int64_t m, int64_t n, int64_t k, bool gated) {
  if (m <= 0 || n <= 0 || k <= 0 || encodes_on_the_way(m, n, k, kF32)) return 0;
  Sizer s;
  take(&s, true, m, k);
  if (!gated && m > kMxThinRows) s.take<float>(product_floats(m, n, k));
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
  MxSkinny few{x, nullptr, m, k, row_stride, codes, scales, up_codes, up_scales, n, mx_slices(k), y};
  if (encodes_on_the_way(m, n, k, dtype)) {
    RPX_HIP(launch_mx_skinny(few, dtype, st), who);
    return kOk;
  }
  Arena arena(workspace, workspace == nullptr ? 0 : workspace_bytes);
  const Encoded e = take(&arena, true, m, k);
  float* partials =
      gated || m <= kMxThinRows ? nullptr : arena.take<float>(product_floats(m, n, k));
  if (arena.overflow) return fail_invalid(std::string(who) + ": workspace too small");
  RPX_TRY(check_pointers(who, {workspace}));
  MxParts parts{};
  parts.part[0] = MxPart{x, dtype, m, k, row_stride, e.out(), MxOut{}, 0};
  RPX_HIP(launch_mx_quantize(parts, 1, st), who);
  if (m <= kMxThinRows) {
    few.x = e.codes;
    few.x_scales = e.scales;
    RPX_HIP(launch_mx_skinny(few, dtype, st), who);
    return kOk;
  }
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
  return serve_workspace(m, n, k, false);
}

int rpx_mxfp4_linear(const void* x, int dtype, int64_t m, int64_t k, int64_t row_stride,
                     const uint8_t* codes, const uint8_t* scales, int64_t n, void* y,
                     void* workspace, size_t workspace_bytes, void* stream) {
  return serve("rpx_mxfp4_linear", x, dtype, m, k, row_stride, codes, scales, nullptr, nullptr,
               false, n, y, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

size_t rpx_mxfp4_gated_workspace(int64_t m, int64_t n, int64_t k) {
  return serve_workspace(m, n, k, true);
}

int rpx_mxfp4_gated(const void* x, int dtype, int64_t m, int64_t k, int64_t row_stride,
                    const uint8_t* gate_codes, const uint8_t* gate_scales,
                    const uint8_t* up_codes, const uint8_t* up_scales, int64_t n, void* h,
                    void* workspace, size_t workspace_bytes, void* stream) {
  return serve("rpx_mxfp4_gated", x, dtype, m, k, row_stride, gate_codes, gate_scales, up_codes,
               up_scales, true, n, h, workspace, workspace_bytes,
               static_cast<hipStream_t>(stream));
}

// --- a linear's training step -------------------------------------------------
namespace {

int check_operand(const char* who, const void* t, int64_t rows, int64_t columns, int64_t stride) {
  if (rows > 0 && columns > 0 && t == nullptr)
    return fail_invalid(std::string(who) + ": null pointer");
  if (stride < columns && rows > 1) return fail_invalid(std::string(who) + ": rows overlap");
  return kOk;
}

}  // namespace

size_t rpx_mxfp4_linear_saved_bytes(int64_t m, int64_t n, int64_t k, int need_left,
                                    int need_right) {
  if (m < 0 || n < 0 || k < 0) return 0;
  Sizer s;
  take(&s, need_right != 0, k, m);
  take(&s, need_left != 0, k, n);
  return s.used;
}

size_t rpx_mxfp4_linear_forward_workspace(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return 0;
  Sizer s;
  take(&s, true, m, k);
  take(&s, true, n, k);
  s.take<float>(product_floats(m, n, k));
  return s.used;
}

int rpx_mxfp4_linear_forward(const void* left, int left_dtype, int64_t m, int64_t k,
                             int64_t left_stride, const void* right, int right_dtype, int64_t n,
                             int64_t right_row_stride, int64_t right_col_stride, void* y,
                             int out_dtype, void* saved, size_t saved_bytes, int need_left,
                             int need_right, void* workspace, size_t workspace_bytes,
                             void* stream) {
  const char* who = "rpx_mxfp4_linear_forward";
  RPX_TRY(check_dtype(left_dtype));
  RPX_TRY(check_dtype(right_dtype));
  RPX_TRY(check_dtype(out_dtype));
  RPX_TRY(check_extents(who, {m, n, k}));
  RPX_TRY(check_operand(who, left, m, k, left_stride));
  if (m > 0 && n > 0) RPX_TRY(check_pointers(who, {y}));
  if ((saved != nullptr && !aligned16(saved)) || (workspace != nullptr && !aligned16(workspace)))
    return fail_invalid("rpx_mxfp4_linear_forward: pointers must be 16-byte aligned");
  Arena keep(saved, saved == nullptr ? 0 : saved_bytes);
  const Encoded xt = take(&keep, need_right != 0, k, m);
  const Encoded wt = take(&keep, need_left != 0, k, n);
  if (keep.overflow) return fail_invalid("rpx_mxfp4_linear_forward: saved buffer too small");
  Arena arena(workspace, workspace == nullptr ? 0 : workspace_bytes);
  const Encoded xq = take(&arena, true, m, k);
  const Encoded wq = take(&arena, true, n, k);
  float* partials = arena.take<float>(product_floats(m, n, k));
  if (arena.overflow) return fail_invalid("rpx_mxfp4_linear_forward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  MxParts parts{};
  int jobs = 0;
  if (m > 0 && k > 0)
    parts.part[jobs++] = MxPart{left, left_dtype, m, k, m > 1 ? left_stride : k, xq.out(), xt.out(), 0};
  if (n > 0 && k > 0)
    RPX_TRY(weight_part(who, right, right_dtype, k, n, right_row_stride, right_col_stride, wq,
                        wt.out(), &parts.part[jobs++]));
  RPX_HIP(launch_mx_quantize(parts, jobs, st), who);
  return product(who, xq, wq, y, out_dtype, partials, st);
}

size_t rpx_mxfp4_linear_backward_workspace(int64_t m, int64_t n, int64_t k, int need_left,
                                           int need_right) {
  if (m < 0 || n < 0 || k < 0) return 0;
  Sizer s;
  take(&s, need_left != 0, m, n);
  take(&s, need_right != 0, n, m);
  const int64_t left = need_left != 0 ? product_floats(m, k, n) : 0;
  const int64_t right = need_right != 0 ? product_floats(n, k, m) : 0;
  s.take<float>(left > right ? left : right);
  return s.used;
}

int rpx_mxfp4_linear_backward(const void* grad, int grad_dtype, int64_t m, int64_t n,
                              int64_t grad_stride, const void* saved, size_t saved_bytes,
                              int64_t k, int need_left, int need_right, void* d_left,
                              int left_dtype, void* d_right, int right_dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* who = "rpx_mxfp4_linear_backward";
  RPX_TRY(check_dtype(grad_dtype));
  RPX_TRY(check_dtype(left_dtype));
  RPX_TRY(check_dtype(right_dtype));
  RPX_TRY(check_extents(who, {m, n, k}));
  RPX_TRY(check_operand(who, grad, m, n, grad_stride));
  if (d_left == nullptr && d_right == nullptr) return kOk;
  if ((d_left != nullptr && need_left == 0) || (d_right != nullptr && need_right == 0))
    return fail_invalid("rpx_mxfp4_linear_backward: the forward saved nothing for this gradient");
  for (const void* p : {static_cast<const void*>(d_left), static_cast<const void*>(d_right), saved,
                        static_cast<const void*>(workspace)})
    if (!aligned16(p))
      return fail_invalid("rpx_mxfp4_linear_backward: pointers must be 16-byte aligned");
  Arena keep(const_cast<void*>(saved), saved == nullptr ? 0 : saved_bytes);
  const Encoded xt = take(&keep, need_right != 0, k, m);
  const Encoded wt = take(&keep, need_left != 0, k, n);
  if (keep.overflow) return fail_invalid("rpx_mxfp4_linear_backward: saved buffer too small");
  Arena arena(workspace, workspace == nullptr ? 0 : workspace_bytes);
  const Encoded gq = take(&arena, d_left != nullptr, m, n);
  const Encoded gt = take(&arena, d_right != nullptr, n, m);
  const int64_t left = d_left != nullptr ? product_floats(m, k, n) : 0;
  const int64_t right = d_right != nullptr ? product_floats(n, k, m) : 0;
  float* partials = arena.take<float>(left > right ? left : right);
  if (arena.overflow) return fail_invalid("rpx_mxfp4_linear_backward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (m > 0 && n > 0) {
    MxParts parts{};
    parts.part[0] = MxPart{grad, grad_dtype, m, n, m > 1 ? grad_stride : n, gq.out(), gt.out(), 0};
    RPX_HIP(launch_mx_quantize(parts, 1, st), who);
  }
  return products(who, gt, xt, d_right, right_dtype, gq, wt, d_left, left_dtype, partials, st);
}

// --- the gated block's training step --------------------------------------------
size_t rpx_mxfp4_gated_saved_bytes(int64_t m, int64_t n, int64_t k, int need_left,
                                   int need_weights) {
  if (m < 0 || n < 0 || k < 0) return 0;
  Sizer s;
  take(&s, need_weights != 0, k, m);
  take(&s, need_left != 0, k, 2 * mx_slices(n) * kMxSlice);
  return s.used;
}

size_t rpx_mxfp4_gated_forward_workspace(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return 0;
  Sizer s;
  take(&s, true, m, k);
  take(&s, true, n, k);
  take(&s, true, n, k);
  return s.used;
}

int rpx_mxfp4_gated_forward(const void* left, int left_dtype, int64_t m, int64_t k,
                            int64_t left_stride, const void* gate, int gate_dtype,
                            int64_t gate_row_stride, int64_t gate_col_stride, const void* up,
                            int up_dtype, int64_t up_row_stride, int64_t up_col_stride, int64_t n,
                            void* h, void* z_gate, void* z_up, int out_dtype, void* saved,
                            size_t saved_bytes, int need_left, int need_weights, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* who = "rpx_mxfp4_gated_forward";
  for (int d : {left_dtype, gate_dtype, up_dtype, out_dtype}) RPX_TRY(check_dtype(d));
  RPX_TRY(check_extents(who, {m, n, k}));
  RPX_TRY(check_operand(who, left, m, k, left_stride));
  if ((z_gate == nullptr) != (z_up == nullptr))
    return fail_invalid("rpx_mxfp4_gated_forward: z_gate and z_up come together");
  for (const void* p : {static_cast<const void*>(h), static_cast<const void*>(z_gate),
                        static_cast<const void*>(z_up), static_cast<const void*>(saved),
                        static_cast<const void*>(workspace)})
    if (!aligned16(p))
      return fail_invalid("rpx_mxfp4_gated_forward: pointers must be 16-byte aligned");
  if (m > 0 && n > 0) RPX_TRY(check_pointers(who, {h}));
  Arena keep(saved, saved == nullptr ? 0 : saved_bytes);
  const int64_t wide = mx_slices(n) * kMxSlice;  // a projection's columns in the joint transpose
  const Encoded xt = take(&keep, need_weights != 0, k, m);
  const Encoded both = take(&keep, need_left != 0, k, 2 * wide);
  if (keep.overflow) return fail_invalid("rpx_mxfp4_gated_forward: saved buffer too small");
  Arena arena(workspace, workspace == nullptr ? 0 : workspace_bytes);
  const Encoded xq = take(&arena, true, m, k);
  const Encoded gq = take(&arena, true, n, k);
  const Encoded uq = take(&arena, true, n, k);
  if (arena.overflow) return fail_invalid("rpx_mxfp4_gated_forward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  MxParts parts{};
  int jobs = 0;
  if (m > 0 && k > 0)
    parts.part[jobs++] = MxPart{left, left_dtype, m, k, m > 1 ? left_stride : k, xq.out(), xt.out(), 0};
  if (n > 0 && k > 0) {
    MxOut halves[2] = {both.out(), both.out()};
    if (both.codes != nullptr) {
      halves[1].codes += wide / 2;
      halves[1].scales += mx_slices(n) * mx_pad_rows(k) * kMxSliceBlocks;
    }
    RPX_TRY(weight_part(who, gate, gate_dtype, k, n, gate_row_stride, gate_col_stride, gq,
                        halves[0], &parts.part[jobs++]));
    RPX_TRY(weight_part(who, up, up_dtype, k, n, up_row_stride, up_col_stride, uq, halves[1],
                        &parts.part[jobs++]));
  }
  RPX_HIP(launch_mx_quantize(parts, jobs, st), who);
  return rpx_mxfp4_gated_gemm(xq.codes, xq.scales, gq.codes, gq.scales, uq.codes, uq.scales, m, n,
                              k, h, z_gate, z_up, out_dtype, stream);
}

size_t rpx_mxfp4_gated_backward_workspace(int64_t m, int64_t n, int64_t k, int need_left,
                                          int need_weights) {
  if (m < 0 || n < 0 || k < 0) return 0;
  const int64_t wide = 2 * mx_slices(n) * kMxSlice;
  Sizer s;
  take(&s, need_left != 0, m, wide);
  take(&s, need_weights != 0, 2 * n, m);
  const int64_t left = need_left != 0 ? product_floats(m, k, wide) : 0;
  const int64_t weights = need_weights != 0 ? product_floats(2 * n, k, m) : 0;
  s.take<float>(left > weights ? left : weights);
  return s.used;
}

int rpx_mxfp4_gated_backward_products(const void* dh, const void* z_gate, const void* z_up,
                                      int dtype, int64_t m, int64_t n, const void* saved,
                                      size_t saved_bytes, int64_t k, int need_left,
                                      int need_weights, void* d_left, int left_dtype,
                                      void* d_weights, int weights_dtype, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const char* who = "rpx_mxfp4_gated_backward_products";
  RPX_TRY(check_dtype(left_dtype));
  RPX_TRY(check_dtype(weights_dtype));
  RPX_TRY(check_extents(who, {m, n, k}));
  if (d_left == nullptr && d_weights == nullptr) return kOk;
  if ((d_left != nullptr && need_left == 0) || (d_weights != nullptr && need_weights == 0))
    return fail_invalid(
        "rpx_mxfp4_gated_backward_products: the forward saved nothing for this gradient");
  for (const void* p : {static_cast<const void*>(d_left), static_cast<const void*>(d_weights),
                        saved, static_cast<const void*>(workspace)})
    if (!aligned16(p))
      return fail_invalid("rpx_mxfp4_gated_backward_products: pointers must be 16-byte aligned");
  const int64_t wide = 2 * mx_slices(n) * kMxSlice;
  Arena keep(const_cast<void*>(saved), saved == nullptr ? 0 : saved_bytes);
  const Encoded xt = take(&keep, need_weights != 0, k, m);
  const Encoded both = take(&keep, need_left != 0, k, wide);
  if (keep.overflow)
    return fail_invalid("rpx_mxfp4_gated_backward_products: saved buffer too small");
  Arena arena(workspace, workspace == nullptr ? 0 : workspace_bytes);
  const Encoded dz = take(&arena, d_left != nullptr, m, wide);
  const Encoded dzt = take(&arena, d_weights != nullptr, 2 * n, m);
  const int64_t left = d_left != nullptr ? product_floats(m, k, wide) : 0;
  const int64_t weights = d_weights != nullptr ? product_floats(2 * n, k, m) : 0;
  float* partials = arena.take<float>(left > weights ? left : weights);
  if (arena.overflow)
    return fail_invalid("rpx_mxfp4_gated_backward_products: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  RPX_TRY(rpx_mxfp4_gated_backward(dh, z_gate, z_up, dtype, m, n, dz.codes, dz.scales, dzt.codes,
                                   dzt.scales, stream));
  return products(who, dzt, xt, d_weights, weights_dtype, dz, both, d_left, left_dtype, partials,
                  st);
}

}  // extern "C"

// C entry points of dropout and of the boundary between two blocks.
#include <string>

#include "../../include/representax_amd.h"
#include "capi.h"
#include "kernels.h"

namespace rpx {

namespace {

int check_dropout(const int64_t* key, int64_t site, int64_t threshold, const std::string& who,
                  Dropout* out) {
  if (threshold < 1 || threshold > 65536)
    return fail_invalid(who + ": threshold must be 1 to 65536");
  if (site < 0 || site > 0xFFFFFFFFll) return fail_invalid(who + ": site must be 0 to 2^32 - 1");
  if (threshold < 65536) {
    if (key == nullptr) return fail_invalid(who + ": null dropout key");
    if (reinterpret_cast<uintptr_t>(key) & 7)
      return fail_invalid(who + ": the dropout key must be 8-byte aligned");
  }
  *out = Dropout{key, static_cast<uint32_t>(site), static_cast<uint32_t>(threshold),
                 65536.0f / static_cast<float>(threshold)};
  return kOk;
}

int check_block_norm(const rpx_block_norm& n, const std::string& who, BlockNorm* out) {
  *out = BlockNorm{n.weight, nullptr, n.dtype, n.kind, n.eps};
  if (n.weight == nullptr) return kOk;
  RPX_TRY(check_dtype(n.dtype));
  if (n.kind != RPX_NORM_LAYER && n.kind != RPX_NORM_RMS)
    return fail_invalid(who + ": unknown kind of norm");
  if (n.kind == RPX_NORM_LAYER) {
    if (n.bias == nullptr) return fail_invalid(who + ": a LayerNorm needs its bias");
    out->bias = n.bias;
  }
  return kOk;
}

bool unaligned(std::initializer_list<const void*> ps, size_t bytes) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0) return true;
  return false;
}

int check_block(const rpx_block* b, const std::string& who, BlockArgs* out) {
  if (b == nullptr) return fail_invalid(who + ": null block");
  RPX_TRY(check_dtype(b->dtype));
  if (b->rows < 0 || b->size < 1 || b->size > kBlockMaxSize)
    return fail_invalid(who + ": need rows >= 0 and 1 <= size <= 8192");
  if (b->gate != nullptr) {
    RPX_TRY(check_dtype(b->gate_dtype));
    if (b->rows_per_gate < 1 || b->rows % b->rows_per_gate != 0)
      return fail_invalid(who + ": rows_per_gate must divide rows");
  }
  BlockArgs a{};
  a.x = b->x;
  a.u = b->u;
  a.gate = b->gate;
  a.gate_dtype = b->gate_dtype;
  a.rows_per_gate = b->gate != nullptr ? b->rows_per_gate : (b->rows > 0 ? b->rows : 1);
  RPX_TRY(check_block_norm(b->post, who, &a.post));
  RPX_TRY(check_block_norm(b->norm, who, &a.norm));
  RPX_TRY(check_dropout(b->key, b->site, b->threshold, who, &a.drop));
  a.scale = b->scale;
  a.dtype = b->dtype;
  a.rows = b->rows;
  a.size = static_cast<int>(b->size);
  a.t = b->t;
  a.h = b->h;
  const size_t bytes = elem_size(b->dtype);
  if (unaligned({b->x, b->u, b->t, b->h}, bytes) ||
      (b->gate != nullptr && unaligned({b->gate}, elem_size(b->gate_dtype))) ||
      (b->post.weight != nullptr &&
       unaligned({b->post.weight, a.post.bias}, elem_size(b->post.dtype))) ||
      (b->norm.weight != nullptr &&
       unaligned({b->norm.weight, a.norm.bias}, elem_size(b->norm.dtype))))
    return fail_invalid(who + ": pointers must be aligned to their type");
  *out = a;
  return kOk;
}

bool any_column(const rpx_block_gradients& g) {
  return g.d_weight != nullptr || g.d_bias != nullptr || g.d_post_weight != nullptr ||
         g.d_post_bias != nullptr;
}

size_t block_backward_bytes(const BlockArgs& a, const rpx_block_gradients& g) {
  return sizeof(float) *
         static_cast<size_t>(block_gradients_floats(a, any_column(g), g.d_gate != nullptr));
}

}  // namespace

}  // namespace rpx

using namespace rpx;

extern "C" {

int rpx_dropout(const void* x, int dtype, int64_t count, const int64_t* key, int64_t site,
                int64_t threshold, void* out, void* stream) {
  const std::string who = "rpx_dropout";
  RPX_TRY(check_dtype(dtype));
  if (count < 0) return fail_invalid(who + ": count must be non-negative");
  Dropout d;
  RPX_TRY(check_dropout(key, site, threshold, who, &d));
  if (count == 0) return kOk;
  if (x == nullptr || out == nullptr) return fail_invalid(who + ": null pointer");
  if (!aligned16_all({x, out})) return fail_invalid(who + ": pointers must be 16-byte aligned");
  RPX_HIP(launch_dropout(x, dtype, count, d, out, static_cast<hipStream_t>(stream)), "rpx_dropout");
  return kOk;
}

int rpx_block_forward(const rpx_block* block, void* stream) {
  const std::string who = "rpx_block_forward";
  BlockArgs a;
  RPX_TRY(check_block(block, who, &a));
  if (a.rows == 0) return kOk;
  if (a.x == nullptr || a.u == nullptr || a.t == nullptr ||
      (a.norm.weight != nullptr && a.h == nullptr))
    return fail_invalid(who + ": null pointer");
  RPX_HIP(launch_block_forward(a, static_cast<hipStream_t>(stream)), "rpx_block_forward");
  return kOk;
}

size_t rpx_block_backward_workspace(const rpx_block* block, const rpx_block_gradients* gradients) {
  BlockArgs a;
  if (gradients == nullptr || check_block(block, "rpx_block_backward_workspace", &a) != kOk) return 0;
  return block_backward_bytes(a, *gradients);
}

int rpx_block_backward(const rpx_block* block, const rpx_block_gradients* gradients,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const std::string who = "rpx_block_backward";
  BlockArgs a;
  RPX_TRY(check_block(block, who, &a));
  if (gradients == nullptr) return fail_invalid(who + ": null gradients");
  const rpx_block_gradients& g = *gradients;
  if ((g.d_gate != nullptr && a.gate == nullptr) ||
      (g.d_weight != nullptr && a.norm.weight == nullptr) ||
      (g.d_bias != nullptr && a.norm.bias == nullptr) ||
      (g.d_post_weight != nullptr && a.post.weight == nullptr) ||
      (g.d_post_bias != nullptr && a.post.bias == nullptr))
    return fail_invalid(who + ": a gradient of what the block does not have");
  if (a.rows == 0 && (any_column(g) || g.d_gate != nullptr))
    return fail_invalid(who + ": no rows to take gradients of weights from");
  if (a.rows == 0) return kOk;
  if (g.dh != nullptr && a.norm.weight == nullptr)
    return fail_invalid(who + ": a gradient of h without its norm");
  const bool reads_u = a.post.weight != nullptr || a.gate != nullptr;
  if ((g.dh != nullptr && a.t == nullptr) || (reads_u && a.u == nullptr))
    return fail_invalid(who + ": null pointer");
  const size_t bytes = elem_size(a.dtype);
  if (unaligned({g.dt, g.dh, g.dx, g.du}, bytes) ||
      (a.gate != nullptr && unaligned({g.d_gate}, elem_size(a.gate_dtype))) ||
      unaligned({g.d_weight, g.d_bias}, elem_size(a.norm.dtype)) ||
      unaligned({g.d_post_weight, g.d_post_bias}, elem_size(a.post.dtype)))
    return fail_invalid(who + ": pointers must be aligned to their type");
  const size_t need = block_backward_bytes(a, g);
  if (need > workspace_bytes || (need > 0 && workspace == nullptr))
    return fail_invalid(who + ": workspace too small");
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail_invalid(who + ": workspace must be 16-byte aligned");
  BlockGradients b{};
  b.forward = a;
  b.dt = g.dt;
  b.dh = g.dh;
  b.dx = g.dx;
  b.du = g.du;
  b.dgate = g.d_gate;
  void* columns[4] = {g.d_weight, g.d_bias, g.d_post_weight, g.d_post_bias};
  for (int i = 0; i < 4; ++i) b.columns[i] = columns[i];
  RPX_HIP(launch_block_backward(b, static_cast<float*>(workspace), static_cast<hipStream_t>(stream)),
          "rpx_block_backward");
  return kOk;
}

}  // extern "C"

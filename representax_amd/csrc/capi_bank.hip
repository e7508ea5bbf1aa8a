// C entry points of low-rank adapters of many requests beside one INT4 projection.
#include <string>
#include <type_traits>

#include "../../include/representax_amd.h"
#include "act.h"
#include "bank.h"
#include "capi.h"
#include "tuning.h"

namespace rpx {

namespace {

constexpr int64_t kMaxRows = int64_t{1} << 25;

struct Bank {
  const uint16_t* x;
  int64_t m, k, n;
  Int4Operand w;
  const uint16_t *bias, *a, *b;
  const float* scalings;
  int64_t adapters, rank;
  BankPlan plan;
  Dropout drop;
};

int check_plan_shape(int64_t m, int64_t adapters, const std::string& who) {
  if (m < 0 || m > kMaxRows) return fail_invalid(who + ": rows must be 0 to 2^25");
  if (adapters < 1 || adapters > kBankMaxAdapters)
    return fail_invalid(who + ": a bank has 1 to 1024 adapters");
  return kOk;
}

int check_bank(const rpx_bank* p, const std::string& who, Bank* out) {
  if (p == nullptr) return fail_invalid(who + ": null bank");
  RPX_TRY(check_plan_shape(p->m, p->adapters, who));
  if (p->n < 1 || p->k < 1) return fail_invalid(who + ": need n >= 1 and k >= 1");
  if (p->n >= (int64_t{1} << 23) || p->k >= (int64_t{1} << 23))
    return fail_invalid(who + ": n and k must be below 2^23");
  if (p->rank < 1 || p->rank > kBankMaxRank) return fail_invalid(who + ": rank must be 1 to 64");
  Bank b{};
  b.w.n_groups = 1;
  b.w.group = p->k;
  if (p->group_size > 0 && p->group_size != p->k) {
    if (p->k % p->group_size != 0 || p->group_size % 2 != 0)
      return fail_invalid(who + ": group_size must be even and divide the input size");
    b.w.n_groups = p->k / p->group_size;
    b.w.group = p->group_size;
  }
  if (p->threshold < 1 || p->threshold > 65536)
    return fail_invalid(who + ": threshold must be 1 to 65536");
  if (p->site < 0 || p->site > 0xFFFFFFFFll) return fail_invalid(who + ": site must be 0 to 2^32 - 1");
  if (p->threshold < 65536 && (p->key == nullptr || (reinterpret_cast<uintptr_t>(p->key) & 7)))
    return fail_invalid(who + ": the dropout needs an 8-byte aligned key");
  if (p->packed == nullptr || p->scale_bits == nullptr || p->lora_a == nullptr ||
      p->lora_b == nullptr || p->scalings == nullptr || p->plan == nullptr ||
      (p->m > 0 && p->x == nullptr))
    return fail_invalid(who + ": null pointer");
  if (!aligned16_all({p->x, p->packed, p->scale_bits, p->lora_a, p->lora_b, p->plan}))
    return fail_invalid(who + ": x, packed, scale_bits, lora_a, lora_b and plan must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(p->scalings) & 3) || (reinterpret_cast<uintptr_t>(p->bias_bits) & 1))
    return fail_invalid(who + ": scalings and bias must be aligned to their type");
  b.x = static_cast<const uint16_t*>(p->x);
  b.m = p->m;
  b.k = p->k;
  b.n = p->n;
  b.w.packed = p->packed;
  b.w.packed_cols = (p->k + 1) / 2;
  b.w.scales = p->scale_bits;
  b.bias = p->bias_bits;
  b.a = static_cast<const uint16_t*>(p->lora_a);
  b.b = static_cast<const uint16_t*>(p->lora_b);
  b.scalings = p->scalings;
  b.adapters = p->adapters;
  b.rank = p->rank;
  b.plan = bank_plan(const_cast<void*>(p->plan), p->m, p->adapters);
  if (p->plan_bytes < static_cast<size_t>(b.plan.words) * 4)
    return fail_invalid(who + ": the plan is smaller than one of these rows and adapters");
  b.drop = Dropout{p->key, static_cast<uint32_t>(p->site), static_cast<uint32_t>(p->threshold),
                   65536.0f / static_cast<float>(p->threshold)};
  *out = b;
  return kOk;
}

// The MFMA kernels' weights: whole 64-column slices, groups that a 32-column piece
// does not straddle.
bool fast(const Bank& b) {
  return b.k % 64 == 0 && (b.w.n_groups == 1 || (b.w.group % 32 == 0 && pow2(b.w.group)));
}

BankSkinny skinny_of(const Bank& b, uint16_t* y, uint16_t* h) {
  return BankSkinny{b.x, b.m, b.k, b.w, b.n, b.bias, b.a, b.b, b.rank, b.scalings, b.plan, y, h};
}

bool skinny(const Bank& b) { return bank_skinny_ok(b.m, b.n, b.k, b.w.n_groups, b.w.group); }

// The adapters' term of a product over `columns` columns, added in its epilogue.
LowRankEpilogue bank_epilogue(const Bank& b, const uint16_t* h, const uint16_t* rows,
                              int64_t columns) {
  LowRankEpilogue epi;
  epi.rows = rows;
  epi.rows_sn = b.rank;
  epi.rows_sj = 1;
  epi.cols = h;
  epi.cols_sm = bank_rank_stride(b.rank);
  epi.cols_sj = 1;
  epi.rank = b.rank;
  epi.act = kActBank;
  epi.row_order = b.plan.order;
  epi.row_adapters = b.plan.sorted;
  epi.adapter_scales = b.scalings;
  epi.adapter_stride = columns * b.rank;
  return epi;
}

int wide_tile(const Bank& b) {
  return wide_plan(b.m, b.n, b.k, tune(kTuneInt4Tile), kActBank, true);
}

// Products that dequantize the weight first and run over the copy: the wide tiles; more
// groups than the 64 KB of a tile's scales in LDS hold; and long sums in one round of 64-row
// tiles, whose 64-column slices take 0.37 us over bf16 and 0.58 over packed weights, while
// the copy costs 2 us and 0.67 more for every million of weights (and the host 4). Total us
// with rank 16 and groups of 64, packed / copied: 6144 -> 2048 at 1000 rows 71 / 64, 8192 ->
// 1024 90 / 72, 4096 -> 1024 50 / 44, 14336 -> 4096 at 333 rows 145 / 135.
bool copied(const Bank& b) {
  if (wide_tile(b) != 0 || b.w.n_groups > 256) return true;
  const double k = static_cast<double>(b.k), weights = k * static_cast<double>(b.n);
  return ceil_div(b.m, 64) * ceil_div(b.n, 128) <= 256 &&
         (0.58 - 0.37) * k / 64 > 6.0 + 0.67e-6 * weights;
}

// The wide tiles read whole pieces of eight ranks: B of another rank is copied to rows of
// them, with zeros behind (h has those zeros too).
bool padded(const Bank& b) { return wide_tile(b) != 0 && b.rank % 8 != 0; }

struct ForwardScratch {
  float* sums = nullptr;    // partial sums of h, or the base product of the generic path
  uint16_t* h = nullptr;
  uint16_t* weight = nullptr;
  uint16_t* b = nullptr;
};

template <typename A>
void forward_scratch(A& arena, const Bank& b, bool h_given, ForwardScratch* s) {
  ForwardScratch none;
  if (s == nullptr) s = &none;
  auto floats = [&](int64_t n) -> float* {
    if constexpr (std::is_same<A, Arena>::value) return arena.template take<float>(n);
    arena.template take<float>(n);
    return nullptr;
  };
  auto halves = [&](int64_t n) -> uint16_t* {
    if constexpr (std::is_same<A, Arena>::value) return arena.template take<uint16_t>(n);
    arena.template take<uint16_t>(n);
    return nullptr;
  };
  const int64_t stride = bank_rank_stride(b.rank);
  if (skinny(b)) {
    const int64_t n = bank_skinny_floats(skinny_of(b, nullptr, nullptr), b.drop);
    if (n > 0) s->sums = floats(n);
    return;
  }
  if (!h_given) s->h = halves(b.m * stride);
  if (!fast(b))
    s->sums = floats(b.m * b.n);
  else if (copied(b))
    s->weight = halves(b.n * b.k);
  if (fast(b) && padded(b)) s->b = halves(b.adapters * b.n * stride);
}

struct BackwardScratch {
  uint16_t *at = nullptr, *bt = nullptr, *dh = nullptr, *wt = nullptr, *g = nullptr;
  float *base = nullptr, *partials = nullptr;
};

template <typename A>
void backward_scratch(A& arena, const Bank& b, bool dx, bool da, bool db, BackwardScratch* s) {
  BackwardScratch none;
  if (s == nullptr) s = &none;
  auto floats = [&](int64_t n) -> float* {
    if constexpr (std::is_same<A, Arena>::value) return arena.template take<float>(n);
    arena.template take<float>(n);
    return nullptr;
  };
  auto halves = [&](int64_t n) -> uint16_t* {
    if constexpr (std::is_same<A, Arena>::value) return arena.template take<uint16_t>(n);
    arena.template take<uint16_t>(n);
    return nullptr;
  };
  if (dx || da) {
    s->bt = halves(b.adapters * b.rank * b.n);
    s->dh = halves(b.m * bank_rank_stride(b.rank));
  }
  if (dx) {
    s->at = halves(b.adapters * b.rank * b.k);
    if (fast(b)) {
      const int64_t n64 = ceil_div(b.n, 64) * 64;
      s->wt = halves(b.k * n64);
      if (n64 != b.n) s->g = halves(b.m * n64);
    } else {
      s->base = floats(b.m * b.k);
    }
  }
  if (da || db) s->partials = floats(bank_gradients_floats(b.plan, b.n, b.k, b.rank, da, db));
}

constexpr Dropout kNoDropout{nullptr, 0, 65536u, 1.0f};

}  // namespace

}  // namespace rpx

using namespace rpx;

extern "C" {

size_t rpx_adapter_plan_bytes(int64_t m, int64_t adapters) {
  if (check_plan_shape(m, adapters, "rpx_adapter_plan_bytes") != kOk) return 0;
  return static_cast<size_t>(bank_plan(nullptr, m, adapters).words) * 4;
}

int rpx_adapter_plan(const void* index, int index_bytes, int64_t m, int64_t adapters, void* plan,
                     size_t plan_bytes, void* stream) {
  const std::string who = "rpx_adapter_plan";
  RPX_TRY(check_plan_shape(m, adapters, who));
  if (index_bytes != 4 && index_bytes != 8)
    return fail_invalid(who + ": the index is int32 or int64");
  if ((m > 0 && index == nullptr) || plan == nullptr) return fail_invalid(who + ": null pointer");
  if (!aligned16(plan) || (reinterpret_cast<uintptr_t>(index) % index_bytes) != 0)
    return fail_invalid(who + ": plan must be 16-byte aligned, index aligned to its type");
  const BankPlan p = bank_plan(plan, m, adapters);
  if (plan_bytes < static_cast<size_t>(p.words) * 4) return fail_invalid(who + ": plan too small");
  RPX_HIP(launch_bank_plan(index, index_bytes, p, static_cast<hipStream_t>(stream)), who.c_str());
  return kOk;
}

size_t rpx_bank_forward_workspace(const rpx_bank* bank, int h_given) {
  Bank b;
  if (check_bank(bank, "rpx_bank_forward_workspace", &b) != kOk) return 0;
  Sizer s;
  forward_scratch(s, b, h_given != 0, nullptr);
  return s.used;
}

int rpx_bank_forward(const rpx_bank* bank, void* y_out, void* h_out, void* workspace,
                     size_t workspace_bytes, void* stream) {
  const std::string who = "rpx_bank_forward";
  Bank b;
  RPX_TRY(check_bank(bank, who, &b));
  if (b.m == 0) return kOk;
  if (y_out == nullptr) return fail_invalid(who + ": null pointer");
  if (!aligned16_all({y_out, h_out, workspace}))
    return fail_invalid(who + ": y, h and workspace must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint16_t* y = static_cast<uint16_t*>(y_out);
  uint16_t* h = static_cast<uint16_t*>(h_out);
  Arena arena(workspace, workspace_bytes);
  ForwardScratch s;
  forward_scratch(arena, b, h != nullptr, &s);
  if (arena.overflow) return fail_invalid(who + ": workspace too small");
  if (skinny(b)) {
    RPX_HIP(launch_bank_skinny(skinny_of(b, y, h), b.drop, s.sums, st), "rpx_bank_forward: few rows");
    return kOk;
  }
  if (h == nullptr) h = s.h;
  RPX_HIP(launch_bank_shrink(b.x, b.k, b.a, b.rank, b.plan, b.drop, h, st),
          "rpx_bank_forward: down-projections");
  if (fast(b)) {
    LowRankEpilogue epi = bank_epilogue(b, h, b.b, b.n);
    epi.bias = b.bias;
    if (padded(b)) {
      const int64_t stride = bank_rank_stride(b.rank);
      RPX_HIP(launch_bank_pad(b.b, b.adapters * b.n, b.rank, s.b, stride, st),
              "rpx_bank_forward: adapters");
      epi.rows = s.b;
      epi.rows_sn = epi.rank = stride;
      epi.adapter_stride = b.n * stride;
    }
    const int tile = wide_tile(b);
    const bool wide =
        tile != 0 && wide_gemm_ok(b.x, b.k, s.weight, b.k, b.m, b.n, b.k, y, b.n, epi);
    const bool copy = copied(b);
    if (copy)
      RPX_HIP(launch_int4_dequant(b.w.packed, b.w.scales, s.weight, b.n, b.k, b.w.packed_cols,
                                  b.w.n_groups, b.w.group, st),
              "rpx_bank_forward: weight");
    if (wide)
      RPX_HIP(launch_gemm_wide(tile, b.x, b.k, s.weight, b.k, b.m, b.n, b.k, y, b.n, epi, st),
              "rpx_bank_forward: product");
    else if (copy)
      RPX_HIP(launch_gemm_bf16(b.x, b.k, s.weight, b.k, b.m, b.n, b.k, y, b.n, epi, st),
              "rpx_bank_forward: product");
    else
      RPX_HIP(launch_gemm_int4(b.x, b.k, b.w, b.m, b.n, b.k, y, b.n, epi, st),
              "rpx_bank_forward: product");
  } else {
    // the terms meet the float32 sums, and their total is rounded
    RPX_HIP(launch_generic_gemm(b.x, kBF16, b.k, 1, nullptr, kBF16, 0, 0, &b.w, false, b.m, b.n, b.k,
                                s.sums, st),
            "rpx_bank_forward: base product");
    RPX_HIP(launch_bank_expand(h, b.b, b.rank, b.n, b.scalings, b.plan, kNoDropout, s.sums, st),
            "rpx_bank_forward: up-projections");
    RPX_HIP(launch_bank_store(s.sums, b.bias, b.m, b.n, y, st), "rpx_bank_forward: y");
  }
  return kOk;
}

size_t rpx_bank_backward_workspace(const rpx_bank* bank, int need_x, int need_a, int need_b) {
  Bank b;
  if (check_bank(bank, "rpx_bank_backward_workspace", &b) != kOk) return 0;
  Sizer s;
  backward_scratch(s, b, need_x != 0, need_a != 0, need_b != 0, nullptr);
  return s.used;
}

int rpx_bank_backward(const rpx_bank* bank, const void* grad, const void* h, void* dx_out,
                      void* d_a, int a_dtype, void* d_b, int b_dtype, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const std::string who = "rpx_bank_backward";
  Bank b;
  RPX_TRY(check_bank(bank, who, &b));
  RPX_TRY(check_dtype(a_dtype));
  RPX_TRY(check_dtype(b_dtype));
  const bool dx_wanted = dx_out != nullptr, da = d_a != nullptr, db = d_b != nullptr;
  if (!dx_wanted && !da && !db) return kOk;
  if (b.m > 0 && (grad == nullptr || (db && h == nullptr)))
    return fail_invalid(who + ": null pointer");
  if (!aligned16_all({grad, h, dx_out, d_a, d_b, workspace}))
    return fail_invalid(who + ": pointers must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint16_t* g = static_cast<const uint16_t*>(grad);
  uint16_t* dx = static_cast<uint16_t*>(dx_out);
  Arena arena(workspace, workspace_bytes);
  BackwardScratch s;
  backward_scratch(arena, b, dx_wanted, da, db, &s);
  if (arena.overflow) return fail_invalid(who + ": workspace too small");
  if (b.m > 0 && (dx_wanted || da)) {
    const BankTranspose ta{dx_wanted ? b.a : nullptr, s.at, b.rank, b.k};
    const BankTranspose tb{b.b, s.bt, b.n, b.rank};
    RPX_HIP(launch_bank_transpose(tb, ta, b.adapters, st), "rpx_bank_backward: transposes");
    RPX_HIP(launch_bank_shrink(g, b.n, s.bt, b.rank, b.plan, kNoDropout, s.dh, st),
            "rpx_bank_backward: dh");
  }
  if (b.m > 0 && dx_wanted) {
    if (fast(b)) {
      const int64_t n64 = ceil_div(b.n, 64) * 64;
      const uint16_t* ga = g;
      if (n64 != b.n) {
        // whole slices of the sum over n: zeros past its end
        RPX_HIP(launch_fill_f32(reinterpret_cast<float*>(s.wt), b.k * n64 / 2, 0.0f, st),
                "rpx_bank_backward: weight");
        RPX_HIP(launch_bank_pad(g, b.m, b.n, s.g, n64, st), "rpx_bank_backward: gradient");
        ga = s.g;
      }
      RPX_HIP(launch_int4_dequant_t(b.w.packed, b.w.scales, s.wt, b.n, b.k, b.w.packed_cols,
                                    b.w.n_groups, b.w.group, n64, st),
              "rpx_bank_backward: weight");
      // a dropout's mask lies on the adapters' part alone; the epilogue applies it there
      LowRankEpilogue epi = bank_epilogue(b, s.dh, s.at, b.k);
      if (b.drop.threshold < 65536u) {
        epi.act = kActBankDrop;
        epi.drop = b.drop;
      }
      RPX_HIP(launch_gemm_bf16(ga, n64, s.wt, n64, b.m, b.k, n64, dx, b.k, epi, st),
              "rpx_bank_backward: dx");
    } else {
      RPX_HIP(launch_generic_gemm(g, kBF16, b.n, 1, nullptr, kBF16, 0, 0, &b.w, true, b.m, b.k, b.n,
                                  s.base, st),
              "rpx_bank_backward: dx");
      RPX_HIP(launch_bank_expand(s.dh, s.at, b.rank, b.k, b.scalings, b.plan, b.drop, s.base, st),
              "rpx_bank_backward: dx of the adapters");
      RPX_HIP(launch_bank_store(s.base, nullptr, b.m, b.k, dx, st), "rpx_bank_backward: dx");
    }
  }
  if (da || db) {
    const BankAdapterGradients p{b.x, g, static_cast<const uint16_t*>(h), s.dh, b.k, b.n, b.rank,
                                 b.scalings, b.drop, d_a, d_b, a_dtype, b_dtype};
    RPX_HIP(launch_bank_gradients(p, b.plan, s.partials, st), "rpx_bank_backward: dA and dB");
  }
  return kOk;
}

}  // extern "C"

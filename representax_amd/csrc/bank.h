// Low-rank adapters of many requests beside one projection (bank.hip,
// bank_skinny.hip): the batch's plan and the launches.
#pragma once

#include "common.h"
#include "kernels.h"
#include "philox.h"

namespace rpx {

constexpr int64_t kBankMaxAdapters = 1024;
constexpr int64_t kBankMaxRank = 64;
constexpr int64_t kBankSkinnyRows = 1024;

// Rows of one adapter: positions [pos, end) of the plan's order.
struct BankTile {
  int32_t adapter;  // -1: unused record
  int32_t pos, end;
  int32_t pad;
};

// What a batch's plan holds, in one int32 buffer.
struct BankPlan {
  const int32_t* rows;         // [m] a row's adapter, -1: none
  const int32_t* order;        // [m] the rows by adapter, in their own order within one, and
                               // those without one last
  const int32_t* sorted;       // [m] the adapter of each position of that order
  const int32_t* first;        // [adapters + 1] an adapter's first position
  const int32_t* chunk_first;  // [adapters + 1] its first chunk
  const BankTile* tiles;       // of `tile` rows each, `tile_count` records
  const BankTile* chunks;      // of `chunk` rows each, `chunk_count` records
  int64_t m, adapters;
  int tile, chunk;
  int64_t tile_count, chunk_count;  // records, more than are used
  int64_t words;
};
BankPlan bank_plan(void* buffer, int64_t m, int64_t adapters);
hipError_t launch_bank_plan(const void* index, int index_bytes, const BankPlan& plan,
                            hipStream_t stream);

// Columns of h and dh in memory.
constexpr int64_t bank_rank_stride(int64_t rank) { return (rank + 7) / 8 * 8; }

// h[m, j] = sum_k drop(x[m, k]) w[adapter(m), j, k] for the rows that have an
// adapter, bf16 [m, stride]; w [adapters, rank, k].
hipError_t launch_bank_shrink(const uint16_t* x, int64_t k, const uint16_t* w, int64_t rank,
                              const BankPlan& plan, const Dropout& drop, uint16_t* h,
                              hipStream_t stream);
// out[m, n] += s[adapter(m)] drop(sum_j h[m, j] w[adapter(m), n, j]); w [adapters, n, rank],
// out f32.
hipError_t launch_bank_expand(const uint16_t* h, const uint16_t* w, int64_t rank, int64_t n,
                              const float* scalings, const BankPlan& plan, const Dropout& drop,
                              float* out, hipStream_t stream);
// Both gradients of the adapters:
//   d_a[e, j, k] = s_e sum_{m of e} dh[m, j] drop(x[m, k]),
//   d_b[e, n, j] = s_e sum_{m of e} g[m, n] h[m, j].
struct BankAdapterGradients {
  const uint16_t *x, *g, *h, *dh;
  int64_t k, n, rank;
  const float* scalings;
  Dropout drop;
  void *d_a, *d_b;  // nullptr: not wanted
  int a_dtype, b_dtype;
};
int64_t bank_gradients_floats(const BankPlan& plan, int64_t n, int64_t k, int64_t rank, bool a,
                              bool b);
hipError_t launch_bank_gradients(const BankAdapterGradients& p, const BankPlan& plan,
                                 float* partials, hipStream_t stream);
// out[e, c, r] = in[e, r, c] for up to two stacks of matrices.
struct BankTranspose {
  const uint16_t* in;
  uint16_t* out;
  int64_t rows, cols;
};
hipError_t launch_bank_transpose(const BankTranspose& a, const BankTranspose& b, int64_t adapters,
                                 hipStream_t stream);
// out [m, ld] bf16 = in [m, n] and zeros.
hipError_t launch_bank_pad(const uint16_t* in, int64_t m, int64_t n, uint16_t* out, int64_t ld,
                           hipStream_t stream);
// out = bf16(in + bias), [m, n] f32.
hipError_t launch_bank_store(const float* in, const uint16_t* bias, int64_t m, int64_t n,
                             uint16_t* out, hipStream_t stream);

// A whole forward over few rows.
struct BankSkinny {
  const uint16_t* x;
  int64_t m, k;
  Int4Operand w;
  int64_t n;
  const uint16_t* bias;
  const uint16_t *a, *b;
  int64_t rank;
  const float* scalings;
  BankPlan plan;
  uint16_t* y;
  uint16_t* h;  // [m, stride] or nullptr
};
bool bank_skinny_ok(int64_t m, int64_t n, int64_t k, int64_t n_groups, int64_t group);
// f32 partial sums of a call.
int64_t bank_skinny_floats(const BankSkinny& p, const Dropout& drop);
hipError_t launch_bank_skinny(const BankSkinny& p, const Dropout& drop, float* partials,
                              hipStream_t stream);

}  // namespace rpx

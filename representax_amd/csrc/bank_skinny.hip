// A projection of few rows, each with its own adapter of a bank, over the packed INT4
// weight:
//   y[m, n] = sum_k x[m, k] W[n, k] + bias[n] + s_e sum_j h[m, j] B_e[n, j].
// Bound by launches and latency, then by the packed weight's bytes. Two launches, with
// everything that is long in the first:
//
//   k_bank_few: workgroups for h = drop(x) A_e^T (16 rows of one adapter and a slice of
//     K each) beside workgroups for x W^T (16 columns, up to 64 rows and a slice of K
//     each). The latter read their packed rows once, dequantize them, bf16(q s), into
//     matrix-core operands and multiply them with all their rows of x; eight waves take
//     128-column chunks in turn and meet in LDS. Both leave f32 partial sums.
//   k_bank_few_finish: adds the partial sums in slice order, bias and adapter term, and
//     rounds once.
//
// One or two rows with a small A (up to 64 KB) take one launch, in which every workgroup
// computes h itself (A comes from L2): 768 -> 768, one row 5.5 us against 8.3.
#include "bank.h"

namespace rpx {

namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;

__device__ __forceinline__ u32x4_t ld16(const void* p) {
  return *reinterpret_cast<const u32x4_t*>(p);
}
__device__ __forceinline__ u32x4_t keep(u32x4_t v, bool ok) {
  return ok ? v : u32x4_t{0u, 0u, 0u, 0u};
}
__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// The values of register i of lanes 16 p .. 16 p + 15 change places with those of
// register p of lanes 16 i .. 16 i + 15.
__device__ __forceinline__ u32x4_t transposed(u32x4_t v) {
  auto swap32 = [](uint32_t& a, uint32_t& b) {
    const u32x2_t t =
        __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(a, b, false, false));
    a = t[0];
    b = t[1];
  };
  auto swap16 = [](uint32_t& a, uint32_t& b) {
    const u32x2_t t =
        __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(a, b, false, false));
    a = t[0];
    b = t[1];
  };
  uint32_t w0 = v[0], w1 = v[1], w2 = v[2], w3 = v[3];
  swap32(w0, w2);
  swap32(w1, w3);
  swap16(w0, w1);
  swap16(w2, w3);
  return u32x4_t{w0, w1, w2, w3};
}

// Eight nibbles as bf16(q s): with u = nibble ^ 8, q s = fma(u, s, -8 s) is exact.
__device__ __forceinline__ u32x4_t dequant8(uint32_t word, float s) {
  const float m8s = -8.0f * s;
  const uint32_t x = word ^ 0x88888888u;
  const uint32_t lo = x & 0x0F0F0F0Fu, hi = (x >> 4) & 0x0F0F0F0Fu;
  u32x4_t o;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    o[b] = pack_bf16x2(__builtin_fmaf(static_cast<float>((lo >> (8 * b)) & 0xFFu), s, m8s),
                       __builtin_fmaf(static_cast<float>((hi >> (8 * b)) & 0xFFu), s, m8s));
  return o;
}

struct FewArgs {
  BankSkinny p;
  Dropout drop;
  int group_shift;
  int stride;
  // h: blocks [0, h_blocks), tile-major, h_slices slices of h_slice columns
  int h_blocks, h_slices, h_slice;
  float* h_sums;  // [h_slices][m][stride]
  // products: column blocks fastest, then slices of `chunks` chunks, then rows
  int columns, slices, chunks;
  float* sums;  // [slices][m][n]
};

// This lane's chunks' loads and products: step s of chunk c multiplies k = 128 c + 32 s +
// 8 part + [0, 8) (NATURAL), or 128 c + 32 part + 8 s + [0, 8), which spares the codes and
// the scale their change of places between the lanes of a row; x then comes as 16 bytes
// of every 64. With up to 16 rows the latter is faster (13 rows, 6144 -> 2048: by 0.3 us),
// with more the former (32 rows, 2048 -> 6144: by 2.6 us).
template <int MT, int U>
struct FewProduct {
  static constexpr bool NATURAL = MT > 1;
  const uint8_t* packed;
  const uint16_t* scales;
  const uint16_t* xrow[MT];
  int k_end, group_shift, part;
  bool grouped;
  u32x4_t wq[U], xf[U][4][MT];
  uint32_t ws[U];
  f32x4_t acc[MT];

  __device__ __forceinline__ FewProduct(const FewArgs& a, int64_t n0, int row0, int lane) {
    const BankSkinny& p = a.p;
    const int r = lane & 15;
    part = lane >> 4;
    const int64_t wrow = n0 + r < p.n ? n0 + r : p.n - 1;
    packed = p.w.packed + wrow * p.w.packed_cols;
    scales = p.w.scales + wrow * p.w.n_groups;
    grouped = p.w.n_groups > 1;
    group_shift = a.group_shift;
    k_end = static_cast<int>(p.k);
    const int m = static_cast<int>(p.m);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int row = row0 + 16 * mt + r;
      xrow[mt] = p.x + static_cast<int64_t>(row < m ? row : m - 1) * p.k + (NATURAL ? 8 * part : 0);
      acc[mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  // unconditional: what lies past K's end is read from its beginning and not used
  __device__ __forceinline__ void load(int c0, int step) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int mine = (c0 + step * u) * 128 + 32 * part;
      const int piece = mine < k_end ? mine : 0;
      wq[u] = ld16(packed + piece / 2);
      ws[u] = scales[grouped ? piece >> group_shift : 0];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = (c0 + step * u) * 128 + 32 * s;
        const int at = NATURAL ? (k < k_end ? k : 0) : piece + 8 * s;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) xf[u][s][mt] = ld16(xrow[mt] + at);
      }
    }
  }
  __device__ __forceinline__ bool in(int c0, int step, int u, int s) const {
    return (c0 + step * u) * 128 + (NATURAL ? 32 * s : 32 * part) < k_end;
  }
  __device__ __forceinline__ void multiply(int c0, int step) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      u32x4_t codes = wq[u];
      u32x4_t scale{ws[u], ws[u], ws[u], ws[u]};
      if constexpr (NATURAL) {
        codes = transposed(codes);
        scale = transposed(scale);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const bool ok = in(c0, step, u, s);
        u32x4_t w = dequant8(codes[s], bf16_to_f32(static_cast<uint16_t>(scale[s])));
        w = keep(w, ok);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt] = mfma(w, keep(xf[u][s][mt], ok), acc[mt]);
      }
    }
  }
};

// h of 16 rows of one adapter over one slice of K: wave w takes every eighth pair of
// 32-deep steps.
template <int RB, bool DROP>
__device__ __forceinline__ void few_shrink(const FewArgs& a, int block, float* lds) {
  const BankSkinny& p = a.p;
  const BankTile tile = p.plan.tiles[block / a.h_slices];
  if (tile.adapter < 0) return;
  const int slice = block % a.h_slices;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15;
  const int part = lane >> 4;
  const int rank = static_cast<int>(p.rank);
  const int pos = tile.pos + j;
  const int64_t row = p.plan.order[pos < tile.end ? pos : tile.pos];
  const uint16_t* x = p.x + row * p.k;
  const uint16_t* w = p.a + static_cast<int64_t>(tile.adapter) * rank * p.k;
  const int k_end = static_cast<int>(p.k);
  const int k0 = slice * a.h_slice;
  const int k1 = k0 + a.h_slice < k_end ? k0 + a.h_slice : k_end;
  PhiloxCall call{};
  if constexpr (DROP) call = philox_call(a.drop);
  f32x4_t acc[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) acc[rb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kb = k0 + 64 * wave; kb < k1; kb += 64 * kWaves) {
    u32x4_t xv[2], wv[2][RB];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = kb + 32 * u;
      const int at = (k < k1 ? k : k0) + 8 * part;
      xv[u] = ld16(x + at);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int jj = 16 * rb + j;
        wv[u][rb] = ld16(w + static_cast<int64_t>(jj < rank ? jj : 0) * p.k + at);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = kb + 32 * u;
      u32x4_t v = keep(xv[u], k < k1);
      if constexpr (DROP) {
        const u32x4_t bits = dropout_bits<true>(call, row * p.k + k + 8 * part);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] &= ((bits[i] & 0xFFFFu) < a.drop.threshold ? 0x0000FFFFu : 0u) |
                  ((bits[i] >> 16) < a.drop.threshold ? 0xFFFF0000u : 0u);
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        acc[rb] = mfma(v, keep(wv[u][rb], k < k1 && 16 * rb + j < rank), acc[rb]);
    }
  }
  // lane: rows 4 part + v, column 16 rb + j
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int v = 0; v < 4; ++v) lds[((wave * RB + rb) * 4 + v) * 64 + lane] = acc[rb][v];
  __syncthreads();
  const float scale = DROP ? a.drop.scale : 1.0f;
  for (int at = threadIdx.x; at < RB * 256; at += kThreads) {
    const int rb = at / 256, v = (at / 64) % 4, l = at % 64;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += lds[((i * RB + rb) * 4 + v) * 64 + l];
    const int q = tile.pos + 4 * (l >> 4) + v;
    const int jj = 16 * rb + (l & 15);
    if (q >= tile.end || jj >= a.stride) continue;
    const int64_t to = slice * p.m + p.plan.order[q];
    a.h_sums[to * a.stride + jj] = jj < rank ? scale * s : 0.0f;
  }
}

// MT: tiles of 16 rows a product's workgroup takes. U: chunks a wave has in flight.
template <int MT, int U, int RB, bool DROP>
__global__ void __launch_bounds__(kThreads) k_bank_few(FewArgs a) {
  constexpr int kLds = kWaves * 256 * (MT > RB ? MT : RB);
  __shared__ float lds[kLds];
  int block = blockIdx.x;
  if (block < a.h_blocks) {
    few_shrink<RB, DROP>(a, block, lds);
    return;
  }
  block -= a.h_blocks;
  const BankSkinny& p = a.p;
  const int64_t n0 = static_cast<int64_t>(block % a.columns) * 16;
  const int rest = block / a.columns;
  const int slice = rest % a.slices;
  const int row0 = rest / a.slices * 16 * MT;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = static_cast<int>(p.m);
  const int all = static_cast<int>((p.k + 127) / 128);
  const int c0 = slice * a.chunks;
  int c1 = c0 + a.chunks;
  c1 = c1 < all ? c1 : all;
  FewProduct<MT, U> f(a, n0, row0, lane);
  f.k_end = c1 * 128 < f.k_end ? c1 * 128 : f.k_end;
  for (int c = c0 + wave; c < c1; c += kWaves * U) {
    f.load(c, kWaves);
    f.multiply(c, kWaves);
  }
  // lane: columns n0 + 4 part + v of row 16 mt + (lane & 15)
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int v = 0; v < 4; ++v)
      lds[(wave * MT + mt) * 256 + (lane & 15) * 16 + 4 * (lane >> 4) + v] = f.acc[mt][v];
  __syncthreads();
#pragma unroll
  for (int at = tid; at < MT * 256; at += kThreads) {
    const int row = row0 + at / 16;
    const int64_t col = n0 + at % 16;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += lds[w * MT * 256 + at];
    if (row < m && col < p.n) a.sums[(static_cast<int64_t>(slice) * m + row) * p.n + col] = s;
  }
}

// t = sum_j h[j] b[j] in f32, rank values of bf16 at any alignment.
__device__ __forceinline__ float adapter_term(const float* h, const uint16_t* b, int rank) {
  float t = 0.0f;
  int j = 0;
  for (; j + 8 <= rank; j += 8) {
    u32x4_t w;
    __builtin_memcpy(&w, b + j, 16);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      t = __builtin_fmaf(h[j + 2 * q], bf16lo_to_f32(w[q]), t);
      t = __builtin_fmaf(h[j + 2 * q + 1], bf16hi_to_f32(w[q]), t);
    }
  }
  for (; j < rank; ++j) t = __builtin_fmaf(h[j], bf16_to_f32(b[j]), t);
  return t;
}

constexpr int kFinishRows = 4;
constexpr int kMaxSlices = 8;

// 64 columns of four rows a workgroup.
__global__ void __launch_bounds__(256) k_bank_few_finish(FewArgs a) {
  __shared__ float hs[kFinishRows][kBankMaxRank];
  const BankSkinny& p = a.p;
  const int m = static_cast<int>(p.m);
  const int rank = static_cast<int>(p.rank);
  const int row0 = static_cast<int>(blockIdx.y) * kFinishRows;
  const int row = row0 + static_cast<int>(threadIdx.x >> 6);
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63);
  const bool in = row < m && col < p.n;
  const int adapter = row < m ? p.plan.rows[row] : -1;
  const float* from = a.sums + static_cast<int64_t>(row < m ? row : 0) * p.n + (col < p.n ? col : 0);
  float part[kMaxSlices];
#pragma unroll
  for (int i = 0; i < kMaxSlices; ++i)
    part[i] = i < a.slices ? from[static_cast<int64_t>(i) * m * p.n] : 0.0f;
  for (int at = threadIdx.x; at < kFinishRows * a.stride; at += 256) {
    const int r = row0 + at / a.stride;
    const float* q = a.h_sums + static_cast<int64_t>(r < m ? r : 0) * a.stride + at % a.stride;
    float v[kMaxSlices], s = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxSlices; ++i)
      v[i] = i < a.h_slices ? q[static_cast<int64_t>(i) * m * a.stride] : 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxSlices; ++i) s += v[i];
    hs[at / a.stride][at % a.stride] = s;
    if (p.h != nullptr && blockIdx.x == 0 && r < m && p.plan.rows[r] >= 0)
      p.h[r * a.stride + at % a.stride] = f32_to_bf16(s);
  }
  __syncthreads();
  if (!in) return;
  float y = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxSlices; ++i) y += part[i];
  if (p.bias != nullptr) y += bf16_to_f32(p.bias[col]);
  if (adapter >= 0)
    y = __builtin_fmaf(p.scalings[adapter],
                       adapter_term(hs[threadIdx.x >> 6],
                                    p.b + (static_cast<int64_t>(adapter) * p.n + col) * rank, rank),
                       y);
  p.y[static_cast<int64_t>(row) * p.n + col] = f32_to_bf16(y);
}

// One or two rows: everything in one launch, a workgroup 16 columns.
constexpr int kOneRows = 2;

template <int RB>
__global__ void __launch_bounds__(kThreads) k_bank_one(FewArgs a) {
  constexpr int U = 2;
  __shared__ float red[kWaves][256];
  __shared__ float hred[kWaves][kOneRows][16 * RB];
  __shared__ float hs[kOneRows][16 * RB];
  const BankSkinny& p = a.p;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15;
  const int part = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int m = static_cast<int>(p.m);
  const int rank = static_cast<int>(p.rank);
  const int chunks = static_cast<int>((p.k + 127) / 128);
  int32_t own[kOneRows];
#pragma unroll
  for (int i = 0; i < kOneRows; ++i) own[i] = i < m ? p.plan.rows[i] : -1;
  f32x4_t hacc[kOneRows][RB];
#pragma unroll
  for (int i = 0; i < kOneRows; ++i)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) hacc[i][rb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  FewProduct<1, U> f(a, n0, 0, lane);
  for (int c = wave; c < chunks; c += kWaves * U) {
    f.load(c, kWaves);
#pragma unroll
    for (int i = 0; i < kOneRows; ++i) {
      if (own[i] < 0) continue;  // the same in every lane
      u32x4_t af[U][RB][4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const int mine = (c + kWaves * u) * 128 + 32 * part;
          const int j = 16 * rb + r;
          const uint16_t* ap = p.a +
                               (static_cast<int64_t>(own[i]) * rank + (j < rank ? j : 0)) * p.k +
                               (mine < f.k_end ? mine : 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) af[u][rb][s] = ld16(ap + 8 * s);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const bool ok = f.in(c, kWaves, u, s);
            hacc[i][rb] = mfma(keep(af[u][rb][s], ok && 16 * rb + r < rank),
                               keep(f.xf[u][s][0], ok), hacc[i][rb]);
          }
    }
    f.multiply(c, kWaves);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) red[wave][r * 16 + 4 * part + v] = f.acc[0][v];
#pragma unroll
  for (int i = 0; i < kOneRows; ++i)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (r == i) hred[wave][i][16 * rb + 4 * part + v] = hacc[i][rb][v];
  // this thread's output: column n0 + tid % 16 of row tid / 16
  const int row = tid >> 4;
  const int64_t col = n0 + (tid & 15);
  const bool out = row < m && row < kOneRows && col < p.n;
  const int adapter = out ? p.plan.rows[row] : -1;
  __syncthreads();
  if (tid < kOneRows * 16 * RB) {
    const int i = tid / (16 * RB), j = tid % (16 * RB);
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += hred[w][i][j];
    hs[i][j] = s;
    if (p.h != nullptr && blockIdx.x == 0 && i < m && j < a.stride && own[i] >= 0)
      p.h[i * a.stride + j] = j < rank ? f32_to_bf16(s) : 0;
  }
  __syncthreads();
  if (!out) return;
  float y = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) y += red[w][row * 16 + (tid & 15)];
  if (p.bias != nullptr) y += bf16_to_f32(p.bias[col]);
  if (adapter >= 0)
    y = __builtin_fmaf(
        p.scalings[adapter],
        adapter_term(hs[row], p.b + (static_cast<int64_t>(adapter) * p.n + col) * rank, rank), y);
  p.y[static_cast<int64_t>(row) * p.n + col] = f32_to_bf16(y);
}

constexpr int64_t kOneBytes = 64 << 10;

bool one_launch(const BankSkinny& p, const Dropout& drop) {
  return p.m <= kOneRows && p.rank <= 32 && drop.threshold >= 65536u &&
         p.m * p.rank * p.k * 2 <= kOneBytes;
}

// The split of a call over workgroups. Slices of K of at least 16 chunks (two a wave)
// bring the products to about two workgroups a CU.
FewArgs plan_few(const BankSkinny& p, const Dropout& drop) {
  FewArgs a{};
  a.p = p;
  a.drop = drop;
  a.stride = static_cast<int>(bank_rank_stride(p.rank));
  if (p.w.n_groups > 1) a.group_shift = __builtin_ctzll(static_cast<uint64_t>(p.w.group));
  a.h_slices = static_cast<int>(p.k / 512);
  a.h_slices = a.h_slices < 1 ? 1 : (a.h_slices > kMaxSlices ? kMaxSlices : a.h_slices);
  a.h_slice = static_cast<int>(ceil_div(ceil_div(p.k, a.h_slices), 64) * 64);
  a.h_slices = static_cast<int>(ceil_div(p.k, a.h_slice));
  a.h_blocks = static_cast<int>(p.plan.tile_count * a.h_slices);
  a.columns = static_cast<int>(ceil_div(p.n, 16));
  const int64_t all = ceil_div(p.k, 128);
  const int64_t rows = ceil_div(p.m, p.m <= 16 ? 16 : (p.m <= 32 ? 32 : 64));
  int64_t s = 512 / (a.columns * rows);
  const int64_t most = all / 16 < kMaxSlices ? all / 16 : kMaxSlices;
  s = s > most ? most : s;
  s = s < 1 ? 1 : s;
  a.chunks = static_cast<int>(ceil_div(all, s));
  a.slices = static_cast<int>(ceil_div(all, a.chunks));
  return a;
}

template <int MT, int U>
void few(const FewArgs& a, unsigned blocks, hipStream_t stream) {
  const bool drop = a.drop.threshold < 65536u;
#define RPX_FEW(RB)                                                                            \
  if (drop)                                                                                    \
    hipLaunchKernelGGL((k_bank_few<MT, U, RB, true>), dim3(blocks), dim3(kThreads), 0, stream, \
                       a);                                                                     \
  else                                                                                         \
    hipLaunchKernelGGL((k_bank_few<MT, U, RB, false>), dim3(blocks), dim3(kThreads), 0, stream, a)
  if (a.p.rank <= 16) {
    RPX_FEW(1);
  } else if (a.p.rank <= 32) {
    RPX_FEW(2);
  } else {
    RPX_FEW(4);
  }
#undef RPX_FEW
}

}  // namespace

// Up to 64 rows, and up to 256 of few columns: each block of 64 rows costs the whole
// weight's dequantization again, while the tiles of the larger products cost 0.7 us a
// 64-column slice of K however few there are (256 rows, 6144 -> 2048: 58 us here, 79
// there; 2048 -> 6144: 63 and 45).
bool bank_skinny_ok(int64_t m, int64_t n, int64_t k, int64_t n_groups, int64_t group) {
  return m >= 1 && (m <= 64 || (m <= kBankSkinnyRows && n * ceil_div(m, 64) <= 10240)) &&
         k % 32 == 0 &&
         (n_groups == 1 || (group % 32 == 0 && (group & (group - 1)) == 0));
}

int64_t bank_skinny_floats(const BankSkinny& p, const Dropout& drop) {
  if (one_launch(p, drop)) return 0;
  const FewArgs a = plan_few(p, drop);
  return a.h_slices * p.m * a.stride + a.slices * p.m * p.n;
}

hipError_t launch_bank_skinny(const BankSkinny& p, const Dropout& drop, float* partials,
                              hipStream_t stream) {
  if (p.m <= 0 || p.n <= 0) return hipSuccess;
  FewArgs a = plan_few(p, drop);
  if (one_launch(p, drop)) {
    const dim3 grid(static_cast<unsigned>(a.columns));
    if (p.rank <= 16)
      hipLaunchKernelGGL(k_bank_one<1>, grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(k_bank_one<2>, grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
  a.sums = partials;
  a.h_sums = partials + a.slices * p.m * p.n;
  const int64_t tile = p.m <= 16 ? 16 : (p.m <= 32 ? 32 : 64);
  const unsigned blocks = static_cast<unsigned>(a.h_blocks + a.columns * a.slices *
                                                                 ceil_div(p.m, tile));
  if (tile == 16) few<1, 2>(a, blocks, stream);
  else if (tile == 32) few<2, 2>(a, blocks, stream);
  else few<4, 2>(a, blocks, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_bank_few_finish,
                     dim3(static_cast<unsigned>(ceil_div(p.n, 64)),
                          static_cast<unsigned>(ceil_div(p.m, kFinishRows))),
                     dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace rpx

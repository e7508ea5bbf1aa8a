// A projection of few rows, each with its own adapter of a bank, over the packed INT4
// weight:
//   y[m, n] = sum_k x[m, k] W[n, k] + bias[n] + s_e sum_j h[m, j] B_e[n, j].
// Bound by launches and latency, then by the packed weight's bytes, and from some 100
// rows on by the reads of x in LDS. Two launches, with everything that is long in the first:
//
//   k_bank_few (to 16 rows), k_bank_mid: workgroups for h = drop(x) A_e^T (16 rows of one
//     adapter and a slice of K each) beside workgroups for x W^T, which read their packed
//     rows once for 16 or 64 rows of x, dequantize them, bf16(q s), into matrix-core
//     operands and multiply them. Both leave f32 partial sums.
//   k_bank_few_finish: adds the partial sums in slice order, bias and adapter term, and
//     rounds once.
//
// One or two rows with a small A (up to 64 KB) take one launch, in which every workgroup
// computes h itself (A comes from L2): 768 -> 768, one row 5.5 us against 8.3.
//
// us, both launches, rank 16, groups of 64, at 1 (2048 -> 6144: one launch) / 13 / 17 / 64 /
// 100 / 200 / 333 rows: 2048 -> 6144 6 / 12 / 12 / 14.6 / 20, 6144 -> 2048 10 / 11 / 14 / 16 / 18 /
// 26 / 34, 2048 -> 2048 7 / 9.4 / 9.7 / 11 / 12.5 / 16 / 21, 768 -> 768 5.6 / 8.6 / 9.0 / 9.4 / 9.5 /
// 9.8 / 10.4.
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
  // products: column blocks fastest, then slices of `chunks` chunks of 128, then rows
  int columns, slices, chunks;
  float* sums;  // [slices][m][n]
};

// This lane's chunks' loads and products: step s of chunk c multiplies k = 128 c + 32 part +
// 8 s + [0, 8), so that a lane's 16 bytes of codes and one scale serve four steps; x
// comes as 16 bytes of every 64.
template <int U>
struct FewProduct {
  const uint8_t* packed;
  const uint16_t* scales;
  const uint16_t* xrow;
  int k_end, group_shift, part;
  bool grouped;
  u32x4_t wq[U], xf[U][4];
  uint32_t ws[U];
  f32x4_t acc{0.f, 0.f, 0.f, 0.f};

  __device__ __forceinline__ FewProduct(const FewArgs& a, int64_t n0, int lane) {
    const BankSkinny& p = a.p;
    const int r = lane & 15;
    part = lane >> 4;
    const int64_t wrow = n0 + r < p.n ? n0 + r : p.n - 1;
    packed = p.w.packed + wrow * p.w.packed_cols;
    scales = p.w.scales + wrow * p.w.n_groups;
    grouped = p.w.n_groups > 1;
    group_shift = a.group_shift;
    k_end = static_cast<int>(p.k);
    xrow = p.x + static_cast<int64_t>(r < p.m ? r : p.m - 1) * p.k;
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
      for (int s = 0; s < 4; ++s) xf[u][s] = ld16(xrow + piece + 8 * s);
    }
  }
  __device__ __forceinline__ bool in(int c0, int step, int u) const {
    return (c0 + step * u) * 128 + 32 * part < k_end;
  }
  __device__ __forceinline__ void multiply(int c0, int step) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = in(c0, step, u);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        acc = mfma(keep(dequant8(wq[u][s], bf16_to_f32(static_cast<uint16_t>(ws[u]))), ok),
                   keep(xf[u][s], ok), acc);
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

// Up to 16 rows: 16 columns and a slice of K a workgroup, whose waves take chunks of 128
// in turn, U in flight, and meet in LDS.
template <int U, int RB, bool DROP>
__global__ void __launch_bounds__(kThreads) k_bank_few(FewArgs a) {
  __shared__ float lds[kWaves * 256 * RB];
  int block = blockIdx.x;
  if (block < a.h_blocks) {
    few_shrink<RB, DROP>(a, block, lds);
    return;
  }
  block -= a.h_blocks;
  const BankSkinny& p = a.p;
  const int64_t n0 = static_cast<int64_t>(block % a.columns) * 16;
  const int slice = block / a.columns;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = static_cast<int>(p.m);
  const int all = static_cast<int>((p.k + 127) / 128);
  const int c0 = slice * a.chunks;
  int c1 = c0 + a.chunks;
  c1 = c1 < all ? c1 : all;
  FewProduct<U> f(a, n0, lane);
  f.k_end = c1 * 128 < f.k_end ? c1 * 128 : f.k_end;
  for (int c = c0 + wave; c < c1; c += kWaves * U) {
    f.load(c, kWaves);
    f.multiply(c, kWaves);
  }
  // lane: columns n0 + 4 part + v of row (lane & 15)
#pragma unroll
  for (int v = 0; v < 4; ++v) lds[wave * 256 + (lane & 15) * 16 + 4 * (lane >> 4) + v] = f.acc[v];
  __syncthreads();
  if (tid >= 256) return;
  const int row = tid / 16;
  const int64_t col = n0 + tid % 16;
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += lds[w * 256 + tid];
  if (row < m && col < p.n) a.sums[(static_cast<int64_t>(slice) * m + row) * p.n + col] = s;
}

// More rows: 64 of them, 128 columns and a slice of K a workgroup. A wave has 16 columns
// and all rows, whose columns of x the workgroup keeps in LDS, 256 at a time in two
// buffers; the next ones' loads, and the codes', run under the products. (32 columns a
// wave halve the reads of LDS, but with their registers spilled to keep two workgroups a
// CU 100 rows of 2048 -> 6144 took 25 us against 19.)
constexpr int kMidRows = 64;
constexpr int kMidStage = 256;
constexpr int kMidPitch = kMidStage + 8;  // rows 4 banks apart

template <int RB, bool DROP>
__global__ void __launch_bounds__(kThreads) k_bank_mid(FewArgs a) {
  constexpr int MT = kMidRows / 16;
  constexpr int XV = kMidRows * kMidStage / 8 / kThreads;  // 16-byte pieces a thread
  __shared__ __align__(16) uint16_t xs[2][kMidRows * kMidPitch];
  static_assert(sizeof(xs) >= sizeof(float) * kWaves * 256 * RB, "h's partial sums meet there too");
  int block = blockIdx.x;
  if (block < a.h_blocks) {
    few_shrink<RB, DROP>(a, block, reinterpret_cast<float*>(&xs[0][0]));
    return;
  }
  block -= a.h_blocks;
  const BankSkinny& p = a.p;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15;
  const int part = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(block % a.columns) * (16 * kWaves) + wave * 16;
  const int rest = block / a.columns;
  const int slice = rest % a.slices;
  const int row0 = rest / a.slices * kMidRows;
  const int m = static_cast<int>(p.m);
  const int k_begin = slice * a.chunks * 128;
  int k_end = k_begin + a.chunks * 128;
  k_end = k_end < p.k ? k_end : static_cast<int>(p.k);
  const int64_t wrow = n0 + r < p.n ? n0 + r : p.n - 1;
  const uint8_t* packed = p.w.packed + wrow * p.w.packed_cols;
  const uint16_t* scales = p.w.scales + wrow * p.w.n_groups;
  const uint16_t* xrow[XV];
#pragma unroll
  for (int i = 0; i < XV; ++i) {
    const int row = row0 + (tid + kThreads * i) / (kMidStage / 8);
    xrow[i] = p.x + static_cast<int64_t>(row < m ? row : m - 1) * p.k;
  }
  const bool grouped = p.w.n_groups > 1;
  const int kx = tid % (kMidStage / 8) * 8;
  u32x4_t xr[XV], wq[2], wc[2];
  uint32_t ws[2], wsc[2];
  // what lies past the slice's end is read from its beginning and not used
  auto load = [&](int kb) {
    const int k = kb + kx;
#pragma unroll
    for (int i = 0; i < XV; ++i) xr[i] = ld16(xrow[i] + (k < k_end ? k : k_begin));
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int mine = kb + 128 * c + 32 * part;
      const int piece = mine < k_end ? mine : k_begin;
      wq[c] = ld16(packed + piece / 2);
      ws[c] = scales[grouped ? piece >> a.group_shift : 0];
    }
  };
  f32x4_t acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  load(k_begin);
  int buffer = 0;
  for (int kb = k_begin; kb < k_end; kb += kMidStage) {
    uint16_t* x = xs[buffer];
#pragma unroll
    for (int i = 0; i < XV; ++i)
      *reinterpret_cast<u32x4_t*>(x + (tid + kThreads * i) / (kMidStage / 8) * kMidPitch + kx) =
          keep(xr[i], kb + kx < k_end);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      wc[c] = wq[c];
      wsc[c] = ws[c];
    }
    __syncthreads();
    if (kb + kMidStage < k_end) load(kb + kMidStage);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const bool ok = kb + 128 * c + 32 * part < k_end;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const u32x4_t w =
            keep(dequant8(wc[c][s], bf16_to_f32(static_cast<uint16_t>(wsc[c]))), ok);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          acc[mt] = mfma(w,
                         *reinterpret_cast<const u32x4_t*>(x + (16 * mt + r) * kMidPitch + 128 * c +
                                                           32 * part + 8 * s),
                         acc[mt]);
      }
    }
    buffer ^= 1;
  }
  // lane: columns n0 + 4 part + v of row 16 mt + r
  const int64_t col = n0 + 4 * part;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + r;
    if (row >= m) continue;
    float* out = a.sums + (static_cast<int64_t>(slice) * m + row) * p.n + col;
    if (col + 4 <= p.n) {
      __builtin_memcpy(out, &acc[mt], 16);
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (col + v < p.n) out[v] = acc[mt][v];
    }
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
  FewProduct<U> f(a, n0, lane);
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
            const bool ok = f.in(c, kWaves, u);
            hacc[i][rb] = mfma(keep(af[u][rb][s], ok && 16 * rb + r < rank),
                               keep(f.xf[u][s], ok), hacc[i][rb]);
          }
    }
    f.multiply(c, kWaves);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) red[wave][r * 16 + 4 * part + v] = f.acc[v];
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

// The rows that k_bank_few takes (13 rows of 6144 -> 2048 11.0 us, 13.6 in k_bank_mid).
constexpr int64_t kFewRows = 16;

// The split of a call over workgroups.
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
  const int64_t all = ceil_div(p.k, 128);
  int64_t s, most;
  if (p.m > kFewRows) {
    // two workgroups a CU of slices of eight chunks and more, one of shorter ones, whose
    // partial sums weigh more (100 rows of 2048 -> 6144 in two slices 19.2 us, in four 21.0;
    // 333 of 6144 -> 2048 in two 37.7, in five 32.7), down to one stage where there are few
    // (64 rows of 768 -> 768 in one slice 13.1, in three 9.4)
    a.columns = static_cast<int>(ceil_div(p.n, 16 * kWaves));
    const int64_t tiles = a.columns * ceil_div(p.m, kMidRows);
    const int64_t two = 512 / tiles < all / 8 ? 512 / tiles : all / 8;
    s = 256 / tiles > two ? 256 / tiles : two;
    most = all / 2;
  } else {
    // about two workgroups a CU, slices of at least 16 chunks (two a wave)
    a.columns = static_cast<int>(ceil_div(p.n, 16));
    s = 512 / a.columns;
    most = all / 16;
  }
  most = most < kMaxSlices ? most : kMaxSlices;
  s = s > most ? most : s;
  s = s < 1 ? 1 : s;
  a.chunks = static_cast<int>(ceil_div(all, s));
  if (p.m > kFewRows) a.chunks += a.chunks & 1;  // whole stages
  a.slices = static_cast<int>(ceil_div(all, a.chunks));
  return a;
}

void partial_sums(const FewArgs& a, unsigned blocks, hipStream_t stream) {
  const bool drop = a.drop.threshold < 65536u, few = a.p.m <= kFewRows;
#define RPX_SUMS(RB)                                                                             \
  if (few && drop)                                                                               \
    hipLaunchKernelGGL((k_bank_few<2, RB, true>), dim3(blocks), dim3(kThreads), 0, stream, a);   \
  else if (few)                                                                                  \
    hipLaunchKernelGGL((k_bank_few<2, RB, false>), dim3(blocks), dim3(kThreads), 0, stream, a);  \
  else if (drop)                                                                                 \
    hipLaunchKernelGGL((k_bank_mid<RB, true>), dim3(blocks), dim3(kThreads), 0, stream, a);      \
  else                                                                                           \
    hipLaunchKernelGGL((k_bank_mid<RB, false>), dim3(blocks), dim3(kThreads), 0, stream, a)
  if (a.p.rank <= 16) {
    RPX_SUMS(1);
  } else if (a.p.rank <= 32) {
    RPX_SUMS(2);
  } else {
    RPX_SUMS(4);
  }
#undef RPX_SUMS
}

}  // namespace

// Up to 64 rows, and up to 1024 of few columns: each 64 rows cost the whole weight's
// dequantization and their reads of x from LDS again, 0.37 to 0.49 us for every million of
// weights, while the tiles of the larger products cost 0.58 us and more a 64-column slice of
// K however few there are. us here / there: 2048 -> 6144 at 128 rows 21 / 28, at 200 31 / 29;
// 2048 -> 2048 at 500 rows 23 / 28, at 1000 35 / 30; 6144 -> 2048 at 333 rows 33 / 60, at 1000
// 80 / 64; 768 -> 768 at 1000 rows 15 / 16.
bool bank_skinny_ok(int64_t m, int64_t n, int64_t k, int64_t n_groups, int64_t group) {
  return m >= 1 && (m <= 64 || (m <= kBankSkinnyRows && n * ceil_div(m, kMidRows) <= 18432)) &&
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
  const int64_t rows = p.m <= kFewRows ? 1 : ceil_div(p.m, kMidRows);
  partial_sums(a, static_cast<unsigned>(a.h_blocks + a.columns * a.slices * rows), stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_bank_few_finish,
                     dim3(static_cast<unsigned>(ceil_div(p.n, 64)),
                          static_cast<unsigned>(ceil_div(p.m, kFinishRows))),
                     dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace rpx

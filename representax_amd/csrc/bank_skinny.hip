// A projection of few rows (up to 64), each with its own adapter of a bank, over
// the packed INT4 weight: one workgroup of eight waves per 16 output columns reads
// their packed rows once, dequantizes them, bf16(q s), into matrix-core operands
// against all rows of x, and adds bias and adapter term before the one rounding:
//   y[m, n] = sum_k x[m, k] W[n, k] + bias[n] + s_e sum_j h[m, j] B_e[n, j].
//
// The waves take 128-column chunks of K in turn and meet in LDS. h = x A_e^T is
// f32 here: either the partial sums of a launch before this one, or, where a row's
// A is small, computed by every workgroup itself (FUSED): A then comes from L2,
// which costs less than the launch.
#include "bank.h"

namespace rpx {

namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kFusedRows = 4;

struct SkinnyArgs {
  BankSkinny p;
  int group_shift;
  const float* partials;  // [splits][m][stride]
  int splits;
  int stride;
};

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

// MT: tiles of 16 rows. RB: 16-rank blocks of A (FUSED).
template <int MT, int U, bool FUSED, int RB>
__global__ void __launch_bounds__(kThreads) k_bank_skinny(SkinnyArgs a) {
  constexpr int kHRows = FUSED ? kFusedRows : 16 * MT;
  __shared__ float red[kWaves][MT][256];
  __shared__ float hs[kHRows][kBankMaxRank];
  __shared__ float hred[FUSED ? kWaves : 1][FUSED ? kFusedRows : 1][16 * RB];
  const BankSkinny& p = a.p;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15;
  const int part = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int m = static_cast<int>(p.m);
  const int rank = static_cast<int>(p.rank);
  const int64_t wrow = n0 + r < p.n ? n0 + r : p.n - 1;
  const uint8_t* packed = p.w.packed + wrow * p.w.packed_cols;
  const uint16_t* scales = p.w.scales + wrow * p.w.n_groups;
  const int chunks = static_cast<int>((p.k + 127) / 128);

  // This thread's outputs: column n0 + tid % 16 of rows (tid / 16) + 32 i.
  constexpr int kOut = (16 * MT + 31) / 32;
  const int64_t col = n0 + (tid & 15);
  const int64_t col_in = col < p.n ? col : p.n - 1;
  int32_t adapter[kOut];
  u32x4_t touched[kOut];
#pragma unroll
  for (int i = 0; i < kOut; ++i) {
    const int row = (tid >> 4) + 32 * i;
    adapter[i] = p.plan.rows[row < m ? row : m - 1];
    // the adapter's row of B starts on its way from memory
    const int64_t e = adapter[i] < 0 ? 0 : adapter[i];
    const uint16_t* b = p.b + (e * p.n + col_in) * rank;
    touched[i][0] = *b;
  }

  u32x4_t wq[U], xf[U][4][MT];
  float ws[U];
  bool in[U];
  const uint16_t* xrow[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = 16 * mt + r;
    xrow[mt] = p.x + static_cast<int64_t>(row < m ? row : m - 1) * p.k;
  }
  auto load = [&](int c0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = static_cast<int64_t>(c0 + kWaves * u) * 128 + 32 * part;
      in[u] = k < p.k;
      const int64_t at = in[u] ? k : 0;
      wq[u] = ld16(packed + at / 2);
      ws[u] = bf16_to_f32(scales[p.w.n_groups == 1 ? 0 : at >> a.group_shift]);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) xf[u][s][mt] = ld16(xrow[mt] + at + 8 * s);
    }
  };
  f32x4_t acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int kHAcc = FUSED ? kFusedRows : 1;
  f32x4_t hacc[kHAcc][RB];
#pragma unroll
  for (int i = 0; i < kHAcc; ++i)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) hacc[i][rb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  int32_t own[kHAcc];
  if constexpr (FUSED) {
#pragma unroll
    for (int i = 0; i < kFusedRows; ++i) own[i] = i < m ? p.plan.rows[i] : -1;
  }

  for (int c0 = wave; c0 < chunks; c0 += kWaves * U) {
    load(c0);
    u32x4_t af[FUSED ? U : 1][RB][4];
#pragma unroll
    for (int i = 0; i < kHAcc; ++i) {
      if constexpr (FUSED) {
        if (own[i] < 0) continue;  // the same in every lane
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const int64_t k = static_cast<int64_t>(c0 + kWaves * u) * 128 + 32 * part;
            const int j = 16 * rb + r;
            const uint16_t* ap = p.a + (static_cast<int64_t>(own[i]) * rank + (j < rank ? j : 0)) * p.k;
#pragma unroll
            for (int s = 0; s < 4; ++s) af[u][rb][s] = ld16(ap + (in[u] ? k : 0) + 8 * s);
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int s = 0; s < 4; ++s)
              hacc[i][rb] = mfma(keep(af[u][rb][s], in[u] && 16 * rb + r < rank),
                                 keep(xf[u][s][0], in[u]), hacc[i][rb]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const u32x4_t w = keep(dequant8(wq[u][s], ws[u]), in[u]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt] = mfma(w, keep(xf[u][s][mt], in[u]), acc[mt]);
      }
  }
  // lane: columns n0 + 4 part + v of row 16 mt + r
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int v = 0; v < 4; ++v) red[wave][mt][r * 16 + 4 * part + v] = acc[mt][v];
  if constexpr (FUSED) {
#pragma unroll
    for (int i = 0; i < kFusedRows; ++i)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (r == i) hred[wave][i][16 * rb + 4 * part + v] = hacc[i][rb][v];
    __syncthreads();
    if (tid < kFusedRows * 16 * RB) {
      const int i = tid / (16 * RB), j = tid % (16 * RB);
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += hred[w][i][j];
      hs[i][j] = s;
    }
  } else {
    for (int at = tid; at < m * a.stride; at += kThreads) {
      float s = 0.0f;
      for (int i = 0; i < a.splits; ++i) s += a.partials[i * m * a.stride + at];
      hs[at / a.stride][at % a.stride] = s;
    }
  }
  __syncthreads();
  if (p.h != nullptr && blockIdx.x == 0) {
    for (int at = tid; at < m * a.stride; at += kThreads) {
      const int j = at % a.stride;
      p.h[at] = j < rank ? f32_to_bf16(hs[at / a.stride][j]) : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < kOut; ++i) {
    asm volatile("" ::"v"(touched[i][0]));
    const int row = (tid >> 4) + 32 * i;
    if (row >= m || col >= p.n) continue;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) y += red[w][row / 16][(row & 15) * 16 + (tid & 15)];
    if (p.bias != nullptr) y += bf16_to_f32(p.bias[col]);
    if (adapter[i] >= 0) {
      const uint16_t* b = p.b + (static_cast<int64_t>(adapter[i]) * p.n + col) * rank;
      float t = 0.0f;
      int j = 0;
      for (; j + 8 <= rank; j += 8) {
        u32x4_t w;
        __builtin_memcpy(&w, b + j, 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          t = __builtin_fmaf(hs[row][j + 2 * q], bf16lo_to_f32(w[q]), t);
          t = __builtin_fmaf(hs[row][j + 2 * q + 1], bf16hi_to_f32(w[q]), t);
        }
      }
      for (; j < rank; ++j) t = __builtin_fmaf(hs[row][j], bf16_to_f32(b[j]), t);
      y = __builtin_fmaf(p.scalings[adapter[i]], t, y);
    }
    p.y[static_cast<int64_t>(row) * p.n + col] = f32_to_bf16(y);
  }
}

// Every workgroup reads the rows' A: up to this many bytes it does so itself.
constexpr int64_t kFusedBytes = 128 << 10;

bool fused(const BankSkinny& p, const Dropout& drop) {
  return p.m <= kFusedRows && p.rank <= 32 && drop.threshold >= 65536u &&
         p.m * p.rank * p.k * 2 <= kFusedBytes;
}

}  // namespace

bool bank_skinny_ok(int64_t m, int64_t k, int64_t n_groups, int64_t group) {
  return m >= 1 && m <= kBankSkinnyRows && k % 32 == 0 &&
         (n_groups == 1 || (group % 32 == 0 && (group & (group - 1)) == 0));
}

bool bank_skinny_fused(const BankSkinny& p, const Dropout& drop) { return fused(p, drop); }

hipError_t launch_bank_skinny(const BankSkinny& p, const Dropout& drop, float* partials,
                              hipStream_t stream) {
  if (p.m <= 0 || p.n <= 0) return hipSuccess;
  SkinnyArgs a{p, 0, partials, 0, static_cast<int>(bank_rank_stride(p.rank))};
  if (p.w.n_groups > 1) a.group_shift = __builtin_ctzll(static_cast<uint64_t>(p.w.group));
  const dim3 grid(static_cast<unsigned>(ceil_div(p.n, 16)));
  if (fused(p, drop)) {
    if (p.rank <= 16)
      hipLaunchKernelGGL((k_bank_skinny<1, 2, true, 1>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((k_bank_skinny<1, 2, true, 2>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
  const int splits = bank_shrink_splits(p.m, p.k);
  // the slices that there are of multiples of 128 columns
  a.splits = static_cast<int>(ceil_div(p.k, ceil_div(ceil_div(p.k, splits), 128) * 128));
  const hipError_t e =
      launch_bank_shrink(p.x, p.k, p.a, p.rank, p.plan, drop, nullptr, partials, splits, stream);
  if (e != hipSuccess) return e;
  if (p.m <= 16)
    hipLaunchKernelGGL((k_bank_skinny<1, 2, false, 1>), grid, dim3(kThreads), 0, stream, a);
  else if (p.m <= 32)
    hipLaunchKernelGGL((k_bank_skinny<2, 1, false, 1>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_bank_skinny<4, 1, false, 1>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace rpx

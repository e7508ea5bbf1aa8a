// Low-rank adapters of many requests beside one projection: row i takes the
// adapter e = rows[i] of a bank (or none),
//   h[i] = drop(x[i]) A_e^T,  y[i] = x[i] W^T + bias + s_e h[i] B_e^T,
// and its gradients: dh = g B_e, dx = g W + s_e drop(dh A_e), d A_e = s_e dh^T
// drop(x), d B_e = s_e g^T h over the rows of e.
//
// A batch's plan sorts the rows by adapter, so that a workgroup's rows have one:
// rows are gathered where they are read (a row is one or more whole lines of
// memory either way) and nothing is moved. The plan depends on the batch alone
// and serves every projection of a model.
//
// h and dh are rounded to bf16, the type that the matrix cores multiply, as the
// linear with one adapter rounds them; the scale multiplies the f32 sums. Against
// h and dh in f32 that takes the error of y and dx from 0.166% to 0.173% of their
// norm, and that of dA and dB, which are rounded to bf16 themselves, from 0.166% to
// 0.235%.
#include "bank.h"
#include "vector8.h"

namespace rpx {

namespace {

__device__ __forceinline__ bf16x8_t as_bf16x8(u32x4_t v) {
  return __builtin_bit_cast(bf16x8_t, v);
}

// Eight bf16 bits from p, of which `valid` are in range (the rest zero), at any
// alignment. WHOLE: valid is 0 or 8, and p can be read either way: the load is
// unconditional (one under a branch would be waited for inside it).
template <bool WHOLE = false>
__device__ __forceinline__ u32x4_t bits8(const uint16_t* p, int valid) {
  u32x4_t w{0u, 0u, 0u, 0u};
  if constexpr (WHOLE) {
    __builtin_memcpy(&w, p, 16);
    return valid > 0 ? w : u32x4_t{0u, 0u, 0u, 0u};
  }
  if (valid >= 8) {
    __builtin_memcpy(&w, p, 16);
    return w;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = 2 * i < valid ? p[2 * i] : 0u;
    const uint32_t hi = 2 * i + 1 < valid ? p[2 * i + 1] : 0u;
    w[i] = lo | (hi << 16);
  }
  return w;
}

__device__ __forceinline__ int clamp8(int64_t left) {
  return left < 0 ? 0 : (left > 8 ? 8 : static_cast<int>(left));
}

// The eight elements from `first` on with the dropped ones zero (unscaled: the
// scale is a factor of the sums).
template <bool ALIGNED>
__device__ __forceinline__ u32x4_t masked8(u32x4_t v, const PhiloxCall& call, uint32_t threshold,
                                           int64_t first) {
  const u32x4_t bits = dropout_bits<ALIGNED>(call, first);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = (bits[i] & 0xFFFFu) < threshold ? 0x0000FFFFu : 0u;
    const uint32_t hi = (bits[i] >> 16) < threshold ? 0xFFFF0000u : 0u;
    v[i] &= lo | hi;
  }
  return v;
}

// ---------------------------------------------------------------------------
// The plan: a stable counting sort in one workgroup. Wave w takes the w-th share of
// the rows; counts of (wave, adapter) give each its places, and within 64 rows one
// ballot for each bit of an adapter's number gives every lane the lanes of its own, so
// the order is the rows' own. Once a batch: 16384 rows of 8, 48 and 1024 adapters 18, 19
// and 28 us (60, 191 and 319 with the lanes of each adapter in turn), 2^20 rows of 64 1.6
// ms; a plan of several workgroups would need three launches.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

struct PlanOut {
  int32_t *rows, *order, *sorted, *first, *chunk_first;
  BankTile *tiles, *chunks;
};

template <typename I>
__global__ void __launch_bounds__(kPlanThreads)
    k_bank_plan(const I* __restrict__ index, BankPlan plan, PlanOut out, unsigned int* err) {
  constexpr int kMax = static_cast<int>(kBankMaxAdapters);
  __shared__ int32_t count[kPlanWaves][kMax];
  __shared__ int32_t none[kPlanWaves];  // rows without an adapter
  __shared__ int32_t scan[3][kMax + 1];  // positions, tiles and chunks before an adapter
  __shared__ int32_t wave_sum[kPlanWaves][3];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int adapters = static_cast<int>(plan.adapters);
  const int m = static_cast<int>(plan.m);
  for (int i = tid; i < kPlanWaves * kMax; i += kPlanThreads) count[i / kMax][i % kMax] = 0;
  if (tid < kPlanWaves) none[tid] = 0;
  __syncthreads();
  const int64_t share = ceil_div(ceil_div(m, kPlanWaves), 64) * 64;
  const int64_t begin = share * wave < m ? share * wave : m;
  const int64_t end = begin + share < m ? begin + share : m;
  bool bad = false;
  constexpr int kAhead = 4;  // loads in flight
  for (int64_t r0 = begin; r0 < end; r0 += 64 * kAhead) {
    int64_t e[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t r = r0 + 64 * i + lane;
      e[i] = static_cast<int64_t>(index[r < end ? r : end - 1]);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t r = r0 + 64 * i + lane;
      if (r >= end) continue;
      bad |= e[i] < -1 || e[i] >= adapters;
      const int32_t v = e[i] < 0 || e[i] >= adapters ? -1 : static_cast<int32_t>(e[i]);
      out.rows[r] = v;
      atomicAdd(v >= 0 ? &count[wave][v] : &none[wave], 1);
    }
  }
  if (bad && err != nullptr) atomicOr(err, kDevErrBankIndex);
  __syncthreads();
  // exclusive sums over the adapters of their rows, tiles and chunks: an adapter a
  // thread, over the lanes, then over the waves
  static_assert(kPlanThreads >= kMax, "an adapter a thread");
  int32_t run[3] = {0, 0, 0};
  if (tid < adapters) {
    int32_t n = 0;
    for (int w = 0; w < kPlanWaves; ++w) n += count[w][tid];
    run[0] = n;
    run[1] = (n + plan.tile - 1) / plan.tile;
    run[2] = (n + plan.chunk - 1) / plan.chunk;
  }
  int32_t before[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    int32_t s = run[q];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t t = __shfl_up(s, off, 64);
      if (lane >= off) s += t;
    }
    before[q] = s - run[q];
    if (lane == 63) wave_sum[wave][q] = s;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    int32_t s = before[q];
    for (int w = 0; w < wave; ++w) s += wave_sum[w][q];
    if (tid < adapters) {
      scan[q][tid] = s;
      if (tid == adapters - 1) scan[q][adapters] = s + run[q];
    }
  }
  __syncthreads();
  for (int e = tid; e <= adapters; e += kPlanThreads) {
    out.first[e] = scan[0][e];
    out.chunk_first[e] = scan[2][e];
  }
  // each wave's places within an adapter, and among the rows without one
  for (int e = tid; e < adapters; e += kPlanThreads) {
    int32_t s = scan[0][e];
    for (int w = 0; w < kPlanWaves; ++w) {
      const int32_t n = count[w][e];
      count[w][e] = s;
      s += n;
    }
  }
  if (tid == 0) {
    int32_t s = scan[0][adapters];
    for (int w = 0; w < kPlanWaves; ++w) {
      const int32_t n = none[w];
      none[w] = s;
      s += n;
    }
  }
  __syncthreads();
  // bits of an adapter's number plus one; -1 (no adapter) has none set
  const int bits = 32 - __builtin_clz(static_cast<unsigned>(adapters));
  int32_t next = begin + lane < end ? out.rows[begin + lane] : -1;
  for (int64_t r0 = begin; r0 < end; r0 += 64) {
    const int64_t r = r0 + lane;
    const int32_t e = next;
    next = r + 64 < end ? out.rows[r + 64] : -1;
    uint64_t same = __ballot(r < end);  // the lanes of this lane's adapter
    for (int i = 0; i < bits; ++i) {
      const bool set = ((e + 1) >> i) & 1;
      const uint64_t with = __ballot(set);
      same &= set ? with : ~with;
    }
    if (r < end) {
      const int leader = __builtin_ctzll(same);
      int32_t base = 0;
      if (lane == leader)
        base = atomicAdd(e >= 0 ? &count[wave][e] : &none[wave],
                         static_cast<int32_t>(__popcll(same)));
      base = __shfl(base, leader, 64);
      const int32_t at = base + __popcll(same & ((1ull << lane) - 1));
      out.order[at] = static_cast<int32_t>(r);
      out.sorted[at] = e;
    }
  }
  // the records, with the adapter found by halving
  auto records = [&](const int32_t* before_of, int64_t cap, int size, BankTile* to) {
    for (int64_t t = tid; t < cap; t += kPlanThreads) {
      BankTile rec{-1, 0, 0, 0};
      if (t < before_of[adapters]) {
        int lo = 0, hi = adapters;  // the last adapter whose first record is at most t
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (before_of[mid] <= t) lo = mid;
          else hi = mid;
        }
        rec.adapter = lo;
        rec.pos = scan[0][lo] + static_cast<int32_t>(t - before_of[lo]) * size;
        const int32_t stop = scan[0][lo + 1];
        rec.end = rec.pos + size < stop ? rec.pos + size : stop;
      }
      to[t] = rec;
    }
  };
  records(scan[1], plan.tile_count, plan.tile, out.tiles);
  records(scan[2], plan.chunk_count, plan.chunk, out.chunks);
}

// ---------------------------------------------------------------------------
// h = drop(x) A_e^T, and dh = g B_e with B_e^T in A_e's place: one workgroup per
// 16 G rows of an adapter, whose four waves take a quarter of K each and meet in LDS.
// Bound by the rows' bytes: 16384 rows of 6144, 201 MB, in 57 us between a call's other
// kernels, 3.5 TB/s where a copy reaches 5.1 (again and again, mostly out of the memory-side
// cache, 43 at rank 32 and 38 at rank 16); of 2048 with dropout 24 (25 and 17).
// ---------------------------------------------------------------------------
struct ShrinkArgs {
  const uint16_t* x;
  int64_t k;
  const uint16_t* w;
  int rank;
  int stride;  // columns of the output
  const BankTile* tiles;
  const int32_t* order;
  Dropout drop;
  uint16_t* h;
  int parts;      // workgroups a tile
};

// DROP: 0 none, 1 dropout. WHOLE: K is a multiple of eight.
template <int RB, int G, int U, bool DROP, bool WHOLE>
__global__ void __launch_bounds__(256) k_bank_shrink(ShrinkArgs a) {
  __shared__ float red[3][G][RB][4][64];
  BankTile tile = a.tiles[blockIdx.x / a.parts];
  tile.pos += 16 * G * (blockIdx.x % a.parts);
  if (tile.pos >= tile.end) return;  // an unused record has no rows
  tile.end = tile.pos + 16 * G < tile.end ? tile.pos + 16 * G : tile.end;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int koff = (lane >> 4) * 8;
  const int j = lane & 15;
  int64_t row[G];
#pragma unroll
  for (int gi = 0; gi < G; ++gi) {
    const int p = tile.pos + 16 * gi + j;
    row[gi] = a.order[p < tile.end ? p : tile.pos];
  }
  const uint16_t* w = a.w + static_cast<int64_t>(tile.adapter) * a.rank * a.k;
  PhiloxCall call{};
  if constexpr (DROP) call = philox_call(a.drop);
  f32x4_t acc[G][RB];
#pragma unroll
  for (int gi = 0; gi < G; ++gi)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) acc[gi][rb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // a wave takes a quarter of K, whole lines at a time: interleaved steps of the waves
  // put all workgroups on the same columns of rows a multiple of 4 KB apart, and so on
  // few memory channels (16384 rows of 6144: 63 us interleaved, 57 so)
  const int64_t span = ceil_div(a.k, 4 * 64) * 64;
  const int64_t w0 = wave * span;
  const int64_t w1 = w0 + span < a.k ? w0 + span : a.k;
  for (int64_t kb = w0; kb < w1; kb += 32 * U) {
    u32x4_t xv[U][G], wv[U][RB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t kc = kb + 32 * u + koff;
      const int kv = clamp8(w1 - kc);
      const int64_t at = kv > 0 ? kc : 0;  // nothing is read past a row's end
#pragma unroll
      for (int gi = 0; gi < G; ++gi) xv[u][gi] = bits8<WHOLE>(a.x + row[gi] * a.k + at, kv);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int jj = 16 * rb + j;
        wv[u][rb] = bits8<WHOLE>(w + (jj < a.rank ? jj : 0) * a.k + at, jj < a.rank ? kv : 0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        u32x4_t v = xv[u][gi];
        if constexpr (DROP)
          v = masked8<WHOLE>(v, call, a.drop.threshold,
                             row[gi] * a.k + kb + 32 * u + koff);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          acc[gi][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(v), as_bf16x8(wv[u][rb]),
                                                                acc[gi][rb], 0, 0, 0);
      }
  }
  if (wave > 0) {
#pragma unroll
    for (int gi = 0; gi < G; ++gi)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int v = 0; v < 4; ++v) red[wave - 1][gi][rb][v][lane] = acc[gi][rb][v];
  }
  __syncthreads();
  if (wave != 0) return;
  const float scale = DROP ? a.drop.scale : 1.0f;
  // lane: rows 4 (lane >> 4) + v of a group, column 16 rb + (lane & 15)
#pragma unroll
  for (int gi = 0; gi < G; ++gi)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int p = tile.pos + 16 * gi + 4 * (lane >> 4) + v;
      if (p >= tile.end) continue;
      const int64_t out_row = a.order[p];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int jj = 16 * rb + j;
        if (jj >= a.stride) continue;
        // the columns past the rank are zero, whatever x holds
        const float s = jj < a.rank ? scale * (acc[gi][rb][v] + red[0][gi][rb][v][lane] +
                                               red[1][gi][rb][v][lane] + red[2][gi][rb][v][lane])
                                    : 0.0f;
        a.h[out_row * a.stride + jj] = f32_to_bf16(s);
      }
    }
}

// ---------------------------------------------------------------------------
// out += s_e drop(h B_e^T), also dx += s_e drop(dh A_e) with A_e^T in B_e's place:
// a wave has 16 rows of one adapter and 64 columns. Row r of MFMA i is column
// 16 (r / 4) + 4 i + r % 4, so that the four give a lane 16 consecutive columns of
// its row. Only for the shapes off the matrix-core products, whose base product it finds
// as f32 sums; elsewhere the product's epilogue adds the term.
// ---------------------------------------------------------------------------
struct ExpandArgs {
  const uint16_t* h;
  int stride;
  const uint16_t* w;  // [adapters, n, rank]
  int rank;
  int64_t n;
  const float* scalings;
  const BankTile* tiles;
  const int32_t* order;
  Dropout drop;
  float* out;
};

// KB: 32-rank blocks. WHOLE: n is a multiple of eight.
template <int KB, bool DROP, bool WHOLE>
__global__ void __launch_bounds__(256) k_bank_expand(ExpandArgs a) {
  const BankTile tile = a.tiles[blockIdx.x];
  if (tile.adapter < 0) return;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.y) * 4 + wave) * 64;
  if (n0 >= a.n) return;
  const int r = lane & 15;
  const int part = lane >> 4;
  bf16x8_t wf[4][KB];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = n0 + 16 * (r >> 2) + 4 * i + (r & 3);
    const uint16_t* p =
        a.w + (static_cast<int64_t>(tile.adapter) * a.n + (c < a.n ? c : 0)) * a.rank;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int j = 32 * kb + 8 * part;
      const int valid = c < a.n ? clamp8(a.rank - j) : 0;
      wf[i][kb] = as_bf16x8(bits8(valid > 0 ? p + j : p, valid));
    }
  }
  PhiloxCall call{};
  if constexpr (DROP) call = philox_call(a.drop);
  const float s = a.scalings[tile.adapter] * (DROP ? a.drop.scale : 1.0f);
  const int64_t c0 = n0 + 16 * part;
  for (int p0 = tile.pos; p0 < tile.end; p0 += 16) {
    const int p = p0 + r;
    const bool inside = p < tile.end;
    const int64_t row = a.order[inside ? p : p0];
    f32x4_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int j = 32 * kb + 8 * part;
      const bf16x8_t hf =
          as_bf16x8(bits8<true>(a.h + row * a.stride + (j < a.stride ? j : 0), a.stride - j));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[i][kb], hf, t[i], 0, 0, 0);
    }
    if (!inside) continue;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t c = c0 + 8 * q;
      if (c >= a.n) continue;
      const int count = clamp8(a.n - c);
      float* at = a.out + row * a.n + c;
      float v[8];
      load_row8<WHOLE>(at, count, v);
      u32x4_t bits{};
      if constexpr (DROP) bits = dropout_bits<WHOLE>(call, row * a.n + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = s * t[2 * q + e / 4][e % 4];
        if (!DROP || dropout_kept(bits, e, a.drop.threshold)) v[e] += d;
      }
      store_row8<WHOLE>(at, count, v);
    }
  }
}

// ---------------------------------------------------------------------------
// The adapters' gradients: a workgroup takes a chunk of one adapter's rows and
// 128 columns of x (or g), [64 rows x 128 columns] at a time into LDS, from where
// transposing reads feed the matrix cores; the chunks' f32 sums are joined in
// order by a second launch, which also scales and rounds them. Bound by HBM: 16384 rows,
// 2048 -> 6144, rank 16: 62 us for 269 MB (x, g, h and dh, 53 us at a copy's rate), the
// joining 9.
// ---------------------------------------------------------------------------
constexpr int kGradRows = 64;
constexpr int kGradColumns = 128;
constexpr int kMaxChunk = 256;

struct GradArgs {
  const uint16_t* x;  // [m, p]
  const uint16_t* h;  // [m, stride]
  int64_t p;
  int blocks;         // of columns
  float* partials;    // [chunk][p][16 RB], or [chunk][16 RB][p] (across)
  bool across;
  bool drop;
};
struct GradPair {
  GradArgs part[2];
  int stride, rank;
  const BankTile* chunks;
  const int32_t* order;
  int64_t chunk_count;
  Dropout drop;
};

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

// Fragment of an operand whose sum runs over the rows of an LDS tile: lane l gets
// tile[m0 + 8 (l >> 4) + t][c0 + (l & 15)], t = 0 .. 7. ds_read_b64_tr_b16 hands
// lane i of 16 element i & 3 of the 8-byte chunks that lanes 4 e + (i >> 2) address.
__device__ __forceinline__ bf16x8_t rows_fragment(const uint16_t* tile, int pitch, int m0, int c0,
                                                  int lane) {
  const int j = lane & 15;
  const uint16_t* p = tile + (m0 + 8 * (lane >> 4) + (j >> 2)) * pitch + c0 + 4 * (j & 3);
  const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)p);
  const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(p + 4 * pitch));
  const i16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8_t, v);
}

// WHOLE: the columns of both products are multiples of eight.
template <int RB, bool DROP, bool WHOLE>
__global__ void __launch_bounds__(256) k_bank_gradients(GradPair a) {
  constexpr int PX = kGradColumns + 8;
  constexpr int PH = 16 * RB + 8;
  __shared__ __align__(16) uint16_t sx[kGradRows * PX];
  __shared__ __align__(16) uint16_t sh[kGradRows * PH];
  __shared__ int32_t rows[kMaxChunk];
  const int64_t blocks = a.part[0].blocks + a.part[1].blocks;
  const int64_t number = block_of_grid() / blocks;
  const int block = static_cast<int>(block_of_grid() % blocks);
  if (number >= a.chunk_count) return;
  const BankTile chunk = a.chunks[number];
  if (chunk.adapter < 0) return;
  const int which = block < a.part[0].blocks ? 0 : 1;
  const GradArgs& g = a.part[which];
  const int64_t p0 = static_cast<int64_t>(block - (which ? a.part[0].blocks : 0)) * kGradColumns;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  constexpr int XV = kGradRows * (kGradColumns / 8) / 256;      // 8
  constexpr int HV = (kGradRows * (2 * RB) + 255) / 256;
  PhiloxCall call{};
  if constexpr (DROP) call = philox_call(a.drop);
  // the chunk's rows, once: what is loaded per step does not wait for its addresses
  const int count = chunk.end - chunk.pos;
  for (int i = tid; i < count; i += 256) rows[i] = a.order[chunk.pos + i];
  __syncthreads();
  u32x4_t xr[XV], hr[HV];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < XV; ++u) {
      const int v = tid + 256 * u;
      const int pos = base + v / 16;
      const int64_t c = p0 + (v % 16) * 8;
      const bool in = pos < count;
      const int64_t row = rows[in ? pos : 0];
      const int valid = in ? clamp8(g.p - c) : 0;
      xr[u] = bits8<WHOLE>(g.x + row * g.p + (valid > 0 ? c : 0), valid);
      if constexpr (DROP) {
        if (g.drop) xr[u] = masked8<WHOLE>(xr[u], call, a.drop.threshold, row * g.p + c);
      }
    }
#pragma unroll
    for (int u = 0; u < HV; ++u) {
      const int v = tid + 256 * u;
      const int pos = base + v / (2 * RB);
      const int c = (v % (2 * RB)) * 8;
      const bool in = v < kGradRows * 2 * RB && pos < count;
      const int64_t row = rows[in ? pos : 0];
      const int valid = in ? clamp8(a.stride - c) : 0;
      hr[u] = bits8<true>(g.h + row * a.stride + (valid > 0 ? c : 0), valid);
    }
  };
  f32x4_t acc[2][RB];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) acc[i][rb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  load(0);
  for (int base = 0; base < count; base += kGradRows) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < XV; ++u) {
      const int v = tid + 256 * u;
      *reinterpret_cast<u32x4_t*>(&sx[(v / 16) * PX + (v % 16) * 8]) = xr[u];
    }
#pragma unroll
    for (int u = 0; u < HV; ++u) {
      const int v = tid + 256 * u;
      if (v < kGradRows * 2 * RB)
        *reinterpret_cast<u32x4_t*>(&sh[(v / (2 * RB)) * PH + (v % (2 * RB)) * 8]) = hr[u];
    }
    __syncthreads();
    if (base + kGradRows < count) load(base + kGradRows);
    const int left = count - base;
    const int steps = left >= kGradRows ? kGradRows / 32 : (left + 31) / 32;
    for (int st = 0; st < steps; ++st) {
      bf16x8_t hf[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) hf[rb] = rows_fragment(sh, PH, 32 * st, 16 * rb, lane);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bf16x8_t xf = rows_fragment(sx, PX, 32 * st, 32 * wave + 16 * i, lane);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          acc[i][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hf[rb], xf, acc[i][rb], 0, 0, 0);
      }
    }
  }
  constexpr int R = 16 * RB;
  float* out = g.partials + number * g.p * R;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      // lane: ranks 16 rb + 4 (lane >> 4) + v of column c
      const int64_t c = p0 + 32 * wave + 16 * i + (lane & 15);
      const int j = 16 * rb + 4 * (lane >> 4);
      if (c >= g.p) continue;
      if (g.across) {
#pragma unroll
        for (int v = 0; v < 4; ++v) out[(j + v) * g.p + c] = acc[i][rb][v];
      } else {
        *reinterpret_cast<f32x4_t*>(out + c * R + j) = acc[i][rb];
      }
    }
}

// out[e] = s_e sum over its chunks, in order: rows of `inner` values of which
// `keep` are stored.
struct JoinArgs {
  const float* partials;
  int64_t per_chunk;  // floats of a chunk
  int64_t outer, inner, keep, rows;  // partial [outer, inner]; stored [rows, keep]
  float scale;        // 1 / keep rate of the dropout
  void* out;
  int dtype;
};
struct JoinPair {
  JoinArgs part[2];
  int64_t adapters;
  int64_t blocks[2];  // workgroups an adapter
  const int32_t* chunk_first;
  const float* scalings;
};

__global__ void __launch_bounds__(256) k_bank_join(JoinPair a) {
  const int64_t per = a.blocks[0] + a.blocks[1];
  const int64_t e = block_of_grid() / per;
  if (e >= a.adapters) return;  // a grid of several rows has more workgroups than adapters
  int64_t b = block_of_grid() % per;
  const int which = b < a.blocks[0] ? 0 : 1;
  if (which) b -= a.blocks[0];
  const JoinArgs& g = a.part[which];
  const int64_t at = b * 256 + threadIdx.x;
  if (at >= g.rows * g.keep) return;
  const int64_t r = at / g.keep, c = at % g.keep;
  const float* p = g.partials + r * g.inner + c;
  const int64_t c0 = a.chunk_first[e], c1 = a.chunk_first[e + 1];
  float s = 0.0f;
  int64_t i = c0;
  for (; i + 4 <= c1; i += 4) {
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = p[(i + q) * g.per_chunk];
#pragma unroll
    for (int q = 0; q < 4; ++q) s += v[q];
  }
  for (; i < c1; ++i) s += p[i * g.per_chunk];
  // an adapter without rows has a gradient of zero, whatever its scaling is
  s = c1 > c0 ? s * (a.scalings[e] * g.scale) : 0.0f;
  const int64_t o = e * g.rows * g.keep + at;
  if (g.dtype == kBF16)
    static_cast<uint16_t*>(g.out)[o] = f32_to_bf16(s);
  else
    static_cast<float*>(g.out)[o] = s;
}

// ---------------------------------------------------------------------------
// Small passes
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_bank_transpose(BankTranspose a, BankTranspose b,
                                                        int64_t a_blocks) {
  __shared__ uint16_t tile[32][33];
  int64_t block = blockIdx.x;
  const bool second = block >= a_blocks;
  const BankTranspose& t = second ? b : a;
  if (second) block -= a_blocks;
  const int64_t e = blockIdx.y;
  const int64_t across = ceil_div(t.cols, 32);
  const int64_t r0 = (block / across) * 32, c0 = (block % across) * 32;
  const uint16_t* in = t.in + e * t.rows * t.cols;
  uint16_t* out = t.out + e * t.rows * t.cols;
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  for (int i = ty; i < 32; i += 8)
    if (r0 + i < t.rows && c0 + tx < t.cols) tile[i][tx] = in[(r0 + i) * t.cols + c0 + tx];
  __syncthreads();
  for (int i = ty; i < 32; i += 8)
    if (c0 + i < t.cols && r0 + tx < t.rows) out[(c0 + i) * t.rows + r0 + tx] = tile[tx][i];
}

__global__ void __launch_bounds__(256) k_bank_pad(const uint16_t* __restrict__ in, int64_t m,
                                                  int64_t n, uint16_t* __restrict__ out,
                                                  int64_t ld) {
  const int64_t at = (block_of_grid() * 256 + threadIdx.x) * 8;  // ld % 8 == 0
  if (at >= m * ld) return;
  const int64_t r = at / ld, c = at % ld;
  *reinterpret_cast<u32x4_t*>(out + at) =
      bits8(in + r * n + (c < n ? c : 0), c < n ? clamp8(n - c) : 0);
}

__global__ void __launch_bounds__(256) k_bank_store(const float* __restrict__ in,
                                                    const uint16_t* __restrict__ bias, int64_t m,
                                                    int64_t n, uint16_t* __restrict__ out) {
  const int64_t at = block_of_grid() * 256 + threadIdx.x;
  if (at >= m * n) return;
  const float b = bias != nullptr ? bf16_to_f32(bias[at % n]) : 0.0f;
  out[at] = f32_to_bf16(in[at] + b);
}

// The variants of a kernel by dropout and whole vectors.
#define RPX_BANK_LAUNCH(KERNEL, ...)                                                          \
  do {                                                                                        \
    if (drop && whole)                                                                        \
      hipLaunchKernelGGL((KERNEL<__VA_ARGS__, true, true>), grid, dim3(256), 0, stream, a);   \
    else if (drop)                                                                            \
      hipLaunchKernelGGL((KERNEL<__VA_ARGS__, true, false>), grid, dim3(256), 0, stream, a);  \
    else if (whole)                                                                           \
      hipLaunchKernelGGL((KERNEL<__VA_ARGS__, false, true>), grid, dim3(256), 0, stream, a);  \
    else                                                                                      \
      hipLaunchKernelGGL((KERNEL<__VA_ARGS__, false, false>), grid, dim3(256), 0, stream, a); \
  } while (0)

bool drops(const Dropout& d) { return d.threshold < 65536u; }

int rank_blocks(int64_t rank) {
  const int b = static_cast<int>(ceil_div(rank, 16));
  return b == 3 ? 4 : b;
}

}  // namespace

BankPlan bank_plan(void* buffer, int64_t m, int64_t adapters) {
  BankPlan p{};
  p.m = m;
  p.adapters = adapters;
  // Rows of a tile: 64 share the fragments of an adapter's weights between four
  // groups of 16 rows; few rows take tiles of 16, for more workgroups. A chunk of
  // the gradients' sums is a sixteenth of the rows, 64 to 256 of them (16384 rows of
  // 2048 and 6144, with the joining launch: 72 us with chunks of 256, 79 with 512, 95
  // with 1024).
  p.tile = m >= 4096 ? 64 : 16;
  int64_t chunk = ceil_div(ceil_div(m, 16), kGradRows) * kGradRows;
  p.chunk = static_cast<int>(chunk < kGradRows ? kGradRows : (chunk > kMaxChunk ? kMaxChunk : chunk));
  const int64_t used = adapters < m ? adapters : m;
  p.tile_count = m / p.tile + used;
  p.chunk_count = m / p.chunk + used;
  int32_t* w = static_cast<int32_t*>(buffer);
  int64_t at = 0;
  auto take = [&](int64_t count) {
    const int64_t here = at;
    at += (count + 3) / 4 * 4;  // 16-byte pieces
    return here;
  };
  const int64_t rows = take(m), order = take(m), sorted = take(m), first = take(adapters + 1),
                chunk_first = take(adapters + 1), tiles = take(4 * p.tile_count),
                chunks = take(4 * p.chunk_count);
  p.words = at;
  if (w == nullptr) return p;
  p.rows = w + rows;
  p.order = w + order;
  p.sorted = w + sorted;
  p.first = w + first;
  p.chunk_first = w + chunk_first;
  p.tiles = reinterpret_cast<const BankTile*>(w + tiles);
  p.chunks = reinterpret_cast<const BankTile*>(w + chunks);
  return p;
}

hipError_t launch_bank_plan(const void* index, int index_bytes, const BankPlan& plan,
                            hipStream_t stream) {
  const PlanOut out{const_cast<int32_t*>(plan.rows),  const_cast<int32_t*>(plan.order),
                    const_cast<int32_t*>(plan.sorted), const_cast<int32_t*>(plan.first),
                    const_cast<int32_t*>(plan.chunk_first), const_cast<BankTile*>(plan.tiles),
                    const_cast<BankTile*>(plan.chunks)};
  if (index_bytes == 8)
    hipLaunchKernelGGL(k_bank_plan<int64_t>, dim3(1), dim3(kPlanThreads), 0, stream,
                       static_cast<const int64_t*>(index), plan, out, device_error_word());
  else
    hipLaunchKernelGGL(k_bank_plan<int32_t>, dim3(1), dim3(kPlanThreads), 0, stream,
                       static_cast<const int32_t*>(index), plan, out, device_error_word());
  return hipGetLastError();
}

hipError_t launch_bank_shrink(const uint16_t* x, int64_t k, const uint16_t* w, int64_t rank,
                              const BankPlan& plan, const Dropout& dropout, uint16_t* h,
                              hipStream_t stream) {
  if (plan.m <= 0) return hipSuccess;
  ShrinkArgs a{x, k, w, static_cast<int>(rank), static_cast<int>(bank_rank_stride(rank)),
               plan.tiles, plan.order, dropout, h, 1};
  const bool drop = drops(dropout), whole = k % 8 == 0;
  const int rb = rank_blocks(rank);
  // tiles of 64 rows: ranks to 16 in halves, twice the workgroups (16384 rows of 2048 with
  // dropout take a fifth less time, of 6144 the same); rank 32 whole, for half the reads of
  // A (in halves 16384 rows of 6144 take a seventh more)
  if (plan.tile == 64 && rb == 1) a.parts = 2;
  const dim3 grid(static_cast<unsigned>(plan.tile_count * a.parts));
  if (plan.tile == 64) {
    if (rb == 1) RPX_BANK_LAUNCH(k_bank_shrink, 1, 2, 4);
    else if (rb == 2) RPX_BANK_LAUNCH(k_bank_shrink, 2, 4, 2);
    else RPX_BANK_LAUNCH(k_bank_shrink, 4, 4, 2);
  } else {
    if (rb == 1) RPX_BANK_LAUNCH(k_bank_shrink, 1, 1, 8);
    else if (rb == 2) RPX_BANK_LAUNCH(k_bank_shrink, 2, 1, 4);
    else RPX_BANK_LAUNCH(k_bank_shrink, 4, 1, 4);
  }
  return hipGetLastError();
}

hipError_t launch_bank_expand(const uint16_t* h, const uint16_t* w, int64_t rank, int64_t n,
                              const float* scalings, const BankPlan& plan, const Dropout& dropout,
                              float* out, hipStream_t stream) {
  if (plan.m <= 0 || n <= 0) return hipSuccess;
  const ExpandArgs a{h, static_cast<int>(bank_rank_stride(rank)), w, static_cast<int>(rank), n,
                     scalings, plan.tiles, plan.order, dropout, out};
  const dim3 grid(static_cast<unsigned>(plan.tile_count), static_cast<unsigned>(ceil_div(n, 256)));
  const bool drop = drops(dropout), whole = n % 8 == 0;
  if (rank <= 32) RPX_BANK_LAUNCH(k_bank_expand, 1);
  else RPX_BANK_LAUNCH(k_bank_expand, 2);
  return hipGetLastError();
}

int64_t bank_gradients_floats(const BankPlan& plan, int64_t n, int64_t k, int64_t rank, bool a,
                              bool b) {
  return plan.chunk_count * 16 * rank_blocks(rank) * ((a ? k : 0) + (b ? n : 0));
}

hipError_t launch_bank_gradients(const BankAdapterGradients& p, const BankPlan& plan,
                                 float* partials, hipStream_t stream) {
  const int rb = rank_blocks(p.rank);
  const int r = 16 * rb;
  GradPair a{};
  JoinPair j{};
  a.stride = static_cast<int>(bank_rank_stride(p.rank));
  a.rank = static_cast<int>(p.rank);
  a.chunks = plan.chunks;
  a.order = plan.order;
  a.chunk_count = plan.chunk_count;
  a.drop = p.drop;
  j.adapters = plan.adapters;
  j.chunk_first = plan.chunk_first;
  j.scalings = p.scalings;
  float* at = partials;
  if (p.d_a != nullptr) {
    a.part[0] = GradArgs{p.x, p.dh, p.k, static_cast<int>(ceil_div(p.k, kGradColumns)), at, true,
                         drops(p.drop)};
    j.part[0] = JoinArgs{at, p.k * r, r, p.k, p.k, p.rank,
                         drops(p.drop) ? p.drop.scale : 1.0f, p.d_a, p.a_dtype};
    j.blocks[0] = ceil_div(p.k * p.rank, 256);
    at += plan.chunk_count * p.k * r;
  }
  if (p.d_b != nullptr) {
    a.part[1] = GradArgs{p.g, p.h, p.n, static_cast<int>(ceil_div(p.n, kGradColumns)), at, false,
                         false};
    j.part[1] = JoinArgs{at, p.n * r, p.n, r, p.rank, p.n, 1.0f, p.d_b, p.b_dtype};
    j.blocks[1] = ceil_div(p.n * p.rank, 256);
  }
  const int64_t blocks = a.part[0].blocks + a.part[1].blocks;
  if (blocks == 0) return hipSuccess;
  if (plan.chunk_count > 0) {
    const dim3 grid = grid_of(blocks * plan.chunk_count);
    const bool drop = p.d_a != nullptr && drops(p.drop), whole = p.k % 8 == 0 && p.n % 8 == 0;
    if (rb == 1) RPX_BANK_LAUNCH(k_bank_gradients, 1);
    else if (rb == 2) RPX_BANK_LAUNCH(k_bank_gradients, 2);
    else RPX_BANK_LAUNCH(k_bank_gradients, 4);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k_bank_join, grid_of(plan.adapters * (j.blocks[0] + j.blocks[1])), dim3(256),
                     0, stream, j);
  return hipGetLastError();
}

hipError_t launch_bank_transpose(const BankTranspose& a, const BankTranspose& b, int64_t adapters,
                                 hipStream_t stream) {
  const int64_t na = a.in == nullptr ? 0 : ceil_div(a.rows, 32) * ceil_div(a.cols, 32);
  const int64_t nb = b.in == nullptr ? 0 : ceil_div(b.rows, 32) * ceil_div(b.cols, 32);
  if (na + nb == 0 || adapters == 0) return hipSuccess;
  hipLaunchKernelGGL(k_bank_transpose,
                     dim3(static_cast<unsigned>(na + nb), static_cast<unsigned>(adapters)),
                     dim3(256), 0, stream, a, b, na);
  return hipGetLastError();
}

hipError_t launch_bank_pad(const uint16_t* in, int64_t m, int64_t n, uint16_t* out, int64_t ld,
                           hipStream_t stream) {
  if (m <= 0) return hipSuccess;
  hipLaunchKernelGGL(k_bank_pad, grid_of(ceil_div(m * ld, 8 * 256)), dim3(256), 0, stream, in, m, n,
                     out, ld);
  return hipGetLastError();
}

hipError_t launch_bank_store(const float* in, const uint16_t* bias, int64_t m, int64_t n,
                             uint16_t* out, hipStream_t stream) {
  if (m <= 0 || n <= 0) return hipSuccess;
  hipLaunchKernelGGL(k_bank_store, grid_of(ceil_div(m * n, 256)), dim3(256), 0, stream, in, bias, m,
                     n, out);
  return hipGetLastError();
}

}  // namespace rpx

// Products of MXFP4 matrices: out[i, j] = sum_c A[i, c] B[j, c], and the first
// half of a gated feed-forward block, silu(A G^T) * (A U^T), from one pass over
// A. mxfp4.h states the format and the order in which a slice's blocks meet.
//
// What bounds them: the fp4 MFMAs issue 7.3 PFLOP/s, which zeros nearly reach (8192 x 8192
// <- 8192 6.6, 166 us); on random codes the card's power holds that product at 4.7 (235
// us; the same instructions and the same 65% of cycles with an MFMA under way, at 1.69 GHz
// against 2.26), 16384 x 2048 <- 6144 at 4.4 (94 us), so an operation saved in the loop
// counts also where it is hidden. A tile of few slices adds what runs with no MFMA beside it, the
// activation and the staging of its outputs: 3.85 for the gated block of 16384 x 2048 -> 2 x
// 6144 (214 us), 3.4 with its projections kept (244 us, 604 MB of outputs).
#include <atomic>
#include <type_traits>

#include <hip/hip_runtime.h>

#include "act.h"
#include "kernels.h"
#include "lds_pipeline.h"
#include "mxfp4.h"
#include "tuning.h"

namespace rpx {

namespace {

// Writes a wave's sub-tile of ROWS x COLS bf16 values, staged in LDS with a row
// pitch of 2 COLS + 16 bytes, as 16-byte pieces of whole row segments. m0, n0:
// its first row and column in the output. PAST: past the L2, for what is not read
// soon (the projections that a training step keeps: 267 -> 244 us for the gated block
// of 16384 x 2048 -> 2 x 6144, 917 -> 872 for its step. Outputs that the next kernel
// reads gain as much and lose it there: 16384 x 6144 <- 2048 and its encoding, 176 us
// either way when the product took 138).
template <int ROWS, int COLS, bool PAST>
__device__ __forceinline__ void store_staged(const uint8_t* reg, uint16_t* out, int64_t m0,
                                             int64_t n0, int64_t M, int64_t N, int lane) {
  constexpr int P = COLS * 2 + 16;
  constexpr int CPR = COLS / 8;     // pieces of a row
  constexpr int STEP = 64 / CPR;    // rows of an instruction
  constexpr int ITS = ROWS / STEP;
  constexpr int UN = ITS % 4 == 0 ? 4 : 1;
  const int r = lane / CPR;
  const int64_t n = n0 + 8 * (lane % CPR);
  const uint8_t* from = reg + r * P + (lane % CPR) * 16;
  // other lanes' staged values: every write of this wave before its reads
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if ((N & 7) == 0 && m0 + ROWS <= M && n0 + COLS <= N) {
    uint16_t* to = out + (m0 + r) * N + n;
#pragma unroll
    for (int i0 = 0; i0 < ITS; i0 += UN) {
      u32x4_t v[UN];
#pragma unroll
      for (int i = 0; i < UN; ++i)
        v[i] = *reinterpret_cast<const u32x4_t*>(from + (i0 + i) * STEP * P);
#pragma unroll
      for (int i = 0; i < UN; ++i, to += STEP * N) {
        if constexpr (PAST)
          __builtin_nontemporal_store(v[i], reinterpret_cast<u32x4_t*>(to));
        else
          *reinterpret_cast<u32x4_t*>(to) = v[i];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return;
  }
#pragma unroll 1
  for (int i = 0; i < ITS; ++i) {
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(from + i * STEP * P);
    const int64_t m = m0 + r + i * STEP;
    if (m >= M) return;
    uint16_t* d = out + m * N + n;
    if ((N & 7) == 0 && n + 7 < N) {
      *reinterpret_cast<u32x4_t*>(d) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < N) d[e] = static_cast<uint16_t>((v[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
    }
  }
}

// Four float32 values at columns n .. n + 3 of a row.
__device__ __forceinline__ void store4(float* d, int64_t n, int64_t N, const float* y) {
  if (n + 3 < N && (N & 3) == 0) {
    *reinterpret_cast<f32x4_t*>(d) = f32x4_t{y[0], y[1], y[2], y[3]};
  } else {
    for (int e = 0; e < 4; ++e)
      if (n + e < N) d[e] = y[e];
  }
}

// x, which the compiler may not know to be the x of the tile before: what is computed
// from it for a tile is not kept in registers over all of them.
__device__ __forceinline__ int again(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A tile to compute: of which product, over which slices, and where its partial sums
// go if the product is split.
struct MxJob {
  MxGemm p;
  int tile_m, tile_n;
  int64_t first_slice;
  int slices;
  float* partial;
};

// A tile's outputs, bf16 ones by way of LDS at `stage`, 32 rows of the wave at a time.
// Block (fn, fm): the lane holds row 32 fm + l % 32 and columns 32 fn + 8 g +
// 4 (l / 32) + e of the wave's sub-tile in acc[fn][fm][4 g + e].
template <int BM, int BN, int WM, int WN, bool GATED>
__device__ __forceinline__ void mx_store_tile(const MxJob& job,
                                              const f32x16_t (&acc)[BN / WN / 32][BM / WM / 32],
                                              uint8_t* stage, int wave, int lane) {
  constexpr int TM = BM / WM;
  constexpr int FM = TM / 32;
  constexpr int FN = BN / WN / 32;
  constexpr int OUT_N = GATED ? BN / 2 : BN;
  constexpr int COLS = OUT_N / WN;         // of the wave
  constexpr int FO = GATED ? FN / 2 : FN;  // output blocks along them
  constexpr int P = COLS * 2 + 16;
  const MxGemm& p = job.p;
  const int frow = lane & 31;
  const int half = lane >> 5;
  const int64_t mw = static_cast<int64_t>(job.tile_m) * BM + wave % WM * TM;
  const int64_t nw = static_cast<int64_t>(job.tile_n) * OUT_N + wave / WM * COLS;
  if (!GATED && job.partial != nullptr) {
    f32x4_t* dst = reinterpret_cast<f32x4_t*>(job.partial);
#pragma unroll
    for (int fn = 0; fn < FN; ++fn)
#pragma unroll
      for (int fm = 0; fm < FM; ++fm)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16_t& a = acc[fn][fm];
          dst[(((wave * FN + fn) * FM + fm) * 4 + g) * 64 + lane] =
              f32x4_t{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
        }
    return;
  }
  if (p.dtype != kBF16) {
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const int64_t m = mw + fm * 32 + frow;
      if (m >= p.m) continue;
#pragma unroll
      for (int fn = 0; fn < FO; ++fn)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int64_t n = nw + fn * 32 + 8 * g + 4 * half;
          const int64_t at = m * p.n + n;
          float y[4], z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = acc[fn][fm][4 * g + e];
            if constexpr (GATED) z[e] = acc[FO + fn][fm][4 * g + e];
          }
          if constexpr (GATED) {
            float h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              h[e] = act_apply<kActSiluMulFwd>(z[e], y[e], 0.0f, nullptr);
            store4(static_cast<float*>(p.out) + at, n, p.n, h);
            if (p.z_gate != nullptr) {
              store4(static_cast<float*>(p.z_gate) + at, n, p.n, y);
              store4(static_cast<float*>(p.z_up) + at, n, p.n, z);
            }
          } else {
            store4(static_cast<float*>(p.out) + at, n, p.n, y);
          }
        }
    }
    return;
  }
  // The wave's staged rows are its own, so its own order of LDS operations is all
  // that the passes need.
  uint8_t* reg = stage + wave * (32 * P);
  auto stage_block = [&](int fn, int g, uint32_t lo, uint32_t hi) {
    *reinterpret_cast<u32x2_t*>(reg + frow * P + (fn * 32 + 8 * g + 4 * half) * 2) =
        u32x2_t{lo, hi};
  };
#pragma unroll
  for (int fm = 0; fm < FM; ++fm) {
    const int64_t m = mw + fm * 32;
    if constexpr (GATED) {
      // h of the rounded projections; then, if asked for, the projections
#pragma unroll
      for (int fn = 0; fn < FO; ++fn)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16_t& a = acc[fn][fm];
          const f32x16_t& b = acc[FO + fn][fm];
          uint32_t h[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t zg = pack_bf16x2(a[4 * g + 2 * e], a[4 * g + 2 * e + 1]);
            const uint32_t zu = pack_bf16x2(b[4 * g + 2 * e], b[4 * g + 2 * e + 1]);
            h[e] = pack_bf16x2(
                act_apply<kActSiluMulFwd>(bf16lo_to_f32(zu), bf16lo_to_f32(zg), 0.0f, nullptr),
                act_apply<kActSiluMulFwd>(bf16hi_to_f32(zu), bf16hi_to_f32(zg), 0.0f, nullptr));
          }
          stage_block(fn, g, h[0], h[1]);
        }
      store_staged<32, COLS, false>(reg, static_cast<uint16_t*>(p.out), m, nw, p.m, p.n, lane);
      if (p.z_gate == nullptr) continue;
    }
#pragma unroll
    for (int z = 0; z < (GATED ? 2 : 1); ++z) {
#pragma unroll
      for (int fn = 0; fn < FO; ++fn)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16_t& a = acc[z * FO + fn][fm];
          stage_block(fn, g, pack_bf16x2(a[4 * g], a[4 * g + 1]),
                      pack_bf16x2(a[4 * g + 2], a[4 * g + 3]));
        }
      void* out = !GATED ? p.out : z == 0 ? p.z_gate : p.z_up;
      store_staged<32, COLS, GATED>(reg, static_cast<uint16_t*>(out), m, nw, p.m, p.n, lane);
    }
  }
}

// A workgroup of WM x WN waves computes BM x BN tiles (a wave: BM / WM x BN / WN of
// each, in blocks of 32 x 32), jobs first, first + stride, ... of job(). A slice
// (256 columns of every row of the tile, 128 bytes each, and eight scale bytes each)
// goes from memory to LDS by direct-to-LDS loads, into NS rotating stages. A
// slice is four MFMA steps; the fragments of a step are read from LDS while the
// step before it runs, and after the last reads of a stage its refill is issued
// under the last step's MFMAs:
//   steps 0, 1, 2   MFMAs, each followed by LDS reads of the next step's fragments
//   barrier         slice t + 1 has landed, every wave is done with stage t
//   step 3          MFMAs, with the loads of slice t + NS into stage t, and the
//                   reads of slice t + 1's first fragments and scales
// Refills past the end re-read the last slice, which keeps the count of loads in flight
// a constant. The weight's fragments are the MFMA's first operand, so a lane ends up
// with four consecutive output columns of one row.
//
// MANY, where a launch has more tiles than the card holds at once: the loads run on from
// a tile's last slice to the next tile's first, so that a tile begins with its first
// slice in LDS and its first fragments in registers, while the outputs of the one before
// are on their way; they are staged in the stage of its last slice, which is refilled
// after that. Against a tile a workgroup: 214 / 234 us for the gated block of 16384 x
// 2048 -> 2 x 6144 (twelve tiles a CU of eight slices), 244 / 258 with its projections
// kept, 73 / 79 of 5003 rows; 108 / 121 for 16384 x 6144 <- 2048, 18.9 / 20.9 for 8192 x
// 3072 <- 768, 235 / 243 for 8192 x 8192 <- 8192. Code that only these need costs the
// others 1.5 us: 333 x 6144 <- 2048 9.4 / 7.9 when it was theirs too.
//
// GATED: B's BN rows are, for each wave, half gate and half up projections of the
// same output columns, so that both meet in the wave's registers.
template <int BM, int BN, int WM, int WN, int NS, bool GATED, bool MANY, class JobAt>
__device__ __forceinline__ void mx_gemm_tiles(int first, int stride, int jobs,
                                              const JobAt& job_at) {
  constexpr int NW = WM * WN;
  constexpr int TM = BM / WM;
  constexpr int TN = BN / WN;
  constexpr int FM = TM / 32;
  constexpr int FN = TN / 32;
  static_assert(TM % 32 == 0 && TN % 32 == 0 && (!GATED || FN % 2 == 0), "wave tile");
  constexpr int SEGS = (BM + BN) / 8;
  static_assert(SEGS % NW == 0, "segments must split evenly over the waves");
  constexpr int CODE_LPW = SEGS / NW;
  constexpr int SCALE_SEGS = (BM + BN + 127) / 128;
  static_assert(SCALE_SEGS <= NW, "a wave loads one segment of scales");
  constexpr int LPW = CODE_LPW + 1;
  constexpr int EARLY = (LPW + 1) / 2;  // of a refill, issued in step 3; the others in step 0
  constexpr int LATE = LPW - EARLY;
  static_assert(NS >= 2 && LPW * (NS - 1) < 64, "vmcnt range");
  constexpr int SCALES = (BM + BN) * kMxSliceBytes;
  constexpr int STAGE = SCALES + SCALE_SEGS * 1024;
  constexpr int OUT_N = GATED ? BN / 2 : BN;  // output columns of the tile
  constexpr int P = OUT_N / WN * 2 + 16;      // row pitch of staged outputs
  static_assert(NW * 32 * P <= STAGE, "staged outputs fit a stage");
  extern __shared__ __align__(16) uint8_t smem[];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM;
  const int wn = wave / WM;

  // The loads' position: slice `load_slice` of `load_slices` of job `load_job`, and the
  // sources of the wave's segments in its first one: 8 rows of codes each (lane l
  // brings chunk l % 8 of row l / 8, swizzled: the segments' first rows are odd or even
  // multiples of 8 alike, so the swizzle is), and 128 rows of scales (two rows a lane).
  // Rows past the end re-read the last; they only feed outputs that are not stored.
  // Rows are counted in 32 bits, of which they leave one (launch_mx_gemm), and a row of
  // codes is below 2^32 bytes; addresses have 64.
  static_assert(NW % 2 == 0 && BM % 16 == 0, "one swizzle for all segments of a wave");
  int load_job = first, load_slice = 0, load_slices = 0;
  const uint8_t* src[LPW];
  int64_t scale_step = 0;
  auto load_from = [&](const MxJob& job) {
    const MxGemm& p = job.p;
    const int lane = again(tid & 63);
    const int m0 = job.tile_m * BM;
    const int n0 = job.tile_n * OUT_N;
    // row r of the tile's B operand: which matrix, and which of its rows
    auto b_row = [&](int r, bool* up) {
      if constexpr (GATED) {
        const int w = r / TN, q = r % TN;
        *up = q >= TN / 2;
        return n0 + w * (TN / 2) + q % (TN / 2);
      } else {
        *up = false;
        return n0 + r;
      }
    };
    const uint32_t row_bytes = static_cast<uint32_t>(p.slices * kMxSliceBytes);
    const int64_t in_row =
        job.first_slice * kMxSliceBytes + (((lane & 7) ^ swz(8 * wave + (lane >> 3))) << 4);
#pragma unroll
    for (int i = 0; i < CODE_LPW; ++i) {
      const int r = 8 * (wave + i * NW);
      const uint8_t* base = p.a_codes;
      int row = m0 + r, last = static_cast<int>(p.m) - 1;
      if (r >= BM) {
        bool up;
        row = b_row(r - BM, &up);
        last = static_cast<int>(p.n) - 1;
        base = GATED && up ? p.b2_codes : p.b_codes;
      }
      row += lane >> 3;
      row = row < last ? row : last;
      src[i] = base + in_row + static_cast<uint64_t>(static_cast<uint32_t>(row)) * row_bytes;
    }
    const int r = 128 * (wave % SCALE_SEGS) + 2 * lane;
    const uint8_t* base = p.a_scales;
    int row = m0 + r, lim = static_cast<int>(mx_pad_rows(p.m));
    if (r >= BM) {
      bool up;
      row = b_row(r - BM < BN ? r - BM : 0, &up);
      lim = static_cast<int>(mx_pad_rows(p.n));
      base = GATED && up ? p.b2_scales : p.b_scales;
    }
    row = row < lim ? row : lim - 2;
    scale_step = static_cast<int64_t>(lim) * kMxSliceBlocks;
    src[CODE_LPW] =
        base + job.first_slice * scale_step + static_cast<int64_t>(row) * kMxSliceBlocks;
    load_slice = 0;
    load_slices = job.slices;
  };
  auto load_one = [&](uint8_t* st, int i) {
    if (i < CODE_LPW)
      dma_seg(st, src[i], load_slice * kMxSliceBytes, wave + i * NW);
    else
      dma_seg(st + SCALES, src[CODE_LPW], load_slice * scale_step, wave % SCALE_SEGS);
  };
  auto load_next_job = [&] {  // past the last: its first slices again
    load_job = load_job + stride < jobs ? load_job + stride : load_job;
    load_from(job_at(load_job));
  };

  f32x16_t acc[FN][FM];
  const int frow = lane & 31;
  const int half = lane >> 5;
  constexpr int NMF = FM * FN;
  constexpr int NFR = FM + FN;
  constexpr int RPM = NFR * 2 <= NMF ? 2 : NFR <= NMF ? 2 : NFR;
  u32x4_t fx[NFR], fy[NFR];       // fragments of two consecutive steps: A's, then B's
  uint32_t sc[NFR], sc_next[NFR];  // scale words of a slice
  // The wave's rows of A and of B are whole blocks of 32, over which the swizzle repeats:
  // one offset of the lane a step, and the block's as the read's immediate (27 VALU
  // operations a slice for 32 MFMAs, 53 with an address a read: 235 / 240 us for 8192 x
  // 8192 <- 8192, 215 / 226 for the gated block of 16384 x 2048 -> 2 x 6144).
  uint32_t lane_at[4];
#pragma unroll
  for (int step = 0; step < 4; ++step)
    lane_at[step] = frow * 128 + (((4 * half + step) ^ swz(frow)) << 4);
  const int a_rows = wm * TM;
  const int b_rows = BM + wn * TN;
  auto frag_one = [&](const uint8_t* st, int step, int j, u32x4_t* f) {
    f[j] = *reinterpret_cast<const u32x4_t*>(st + (j < FM ? a_rows : b_rows) * 128 +
                                             lane_at[step] + (j < FM ? j : j - FM) * (32 * 128));
  };
  const uint32_t scale_at = SCALES + frow * kMxSliceBlocks + 4 * half;
  auto scale_one = [&](const uint8_t* st, int j, uint32_t* s) {
    s[j] = *reinterpret_cast<const uint32_t*>(st + (j < FM ? a_rows : b_rows) * kMxSliceBlocks +
                                              scale_at +
                                              (j < FM ? j : j - FM) * (32 * kMxSliceBlocks));
  };

  load_from(job_at(first));
#pragma unroll
  for (int s = 0; s < NS; ++s) {
#pragma unroll
    for (int i = 0; i < (s == NS - 1 ? EARLY : LPW); ++i) load_one(smem + s * STAGE, i);
    if (s < NS - 1) {
      if (load_slice + 1 < load_slices)
        ++load_slice;
      else if constexpr (MANY)
        load_next_job();
    }
  }
  wait_sync<(NS - 2) * LPW + EARLY>();
#pragma unroll
  for (int j = 0; j < NFR; ++j) frag_one(smem, 0, j, fx);
#pragma unroll
  for (int j = 0; j < NFR; ++j) scale_one(smem, j, sc);

  // the reads that follow MFMA i of a step: all of them behind the first MFMAs, RPM
  // behind each
  auto read_from = [](int i) { return i * RPM < NFR ? i * RPM : NFR; };
#define RPX_MX_STEP(STEP, F, MORE)                                                               \
  _Pragma("unroll") for (int i = 0; i < NMF; ++i) {                                              \
    acc[i / FM][i % FM] = mx_mfma32<STEP, STEP>(F[FM + i / FM], sc[FM + i / FM], F[i % FM],      \
                                                sc[i % FM], acc[i / FM][i % FM]);                \
    __builtin_amdgcn_sched_barrier(0);                                                           \
    MORE __builtin_amdgcn_sched_barrier(0);                                                      \
  }
#define RPX_MX_READS(ST, STEP, F)                                                                \
  _Pragma("unroll") for (int j = read_from(i); j < read_from(i + 1); ++j) frag_one(ST, STEP, j, F);

  int stage = 0;
  uint8_t* st = smem;
  // One slice. KIND: any, or of a workgroup with MANY tiles the one before a tile's last
  // (the loads go on to the next tile) or the last (its stage is not refilled yet).
  enum { kSlice, kLastButOne, kLast };
  auto slice = [&](auto kind) {
    constexpr int KIND = decltype(kind)::value;
    const int next = stage + 1 == NS ? 0 : stage + 1;
    st = smem + stage * STAGE;
    const uint8_t* nst = smem + next * STAGE;
    uint8_t* last = smem + (stage == 0 ? NS - 1 : stage - 1) * STAGE;
    RPX_MX_STEP(0, fx, {
      RPX_MX_READS(st, 1, fy)
      _Pragma("unroll") for (int d = EARLY + i * LATE / NMF; d < EARLY + (i + 1) * LATE / NMF; ++d)
          load_one(last, d);
    })
    if constexpr (KIND == kSlice)
      load_slice += load_slice + 1 < load_slices ? 1 : 0;
    else if constexpr (KIND == kLastButOne)
      load_next_job();
    RPX_MX_STEP(1, fy, RPX_MX_READS(st, 2, fx))
    RPX_MX_STEP(2, fx, RPX_MX_READS(st, 3, fy))
    wait_sync<(NS - 2) * LPW>();
    RPX_MX_STEP(3, fy, {
      if constexpr (KIND != kLast) {
        _Pragma("unroll") for (int d = i * EARLY / NMF; d < (i + 1) * EARLY / NMF; ++d)
            load_one(st, d);
      }
      RPX_MX_READS(nst, 0, fx)
      _Pragma("unroll") for (int j = read_from(i); j < read_from(i + 1); ++j)
          scale_one(nst, j, sc_next);
    })
#pragma unroll
    for (int j = 0; j < NFR; ++j) sc[j] = sc_next[j];
    stage = next;
  };
  for (int w = first;;) {
    const MxJob job = job_at(w);
#pragma unroll
    for (int fn = 0; fn < FN; ++fn)
#pragma unroll
      for (int fm = 0; fm < FM; ++fm)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[fn][fm][v] = 0.0f;
    if constexpr (!MANY) {
      for (int t = 0; t < job.slices; ++t) slice(std::integral_constant<int, kSlice>{});
    } else {
      for (int t = 0; t < job.slices - 2; ++t) slice(std::integral_constant<int, kSlice>{});
      if (job.slices > 1) slice(std::integral_constant<int, kLastButOne>{});
      slice(std::integral_constant<int, kLast>{});
    }
    // no load may be in flight to an LDS that the outputs, or the workgroup after this
    // one, get (with two stages the last wait was for all)
    if constexpr (!MANY) wait_sync<0>();
    // the tile's MFMAs before its outputs' branches
#pragma unroll
    for (int fn = 0; fn < FN; ++fn)
#pragma unroll
      for (int fm = 0; fm < FM; ++fm) asm volatile("" : "+v"(acc[fn][fm]));
    mx_store_tile<BM, BN, WM, WN, GATED>(job, acc, st, wave, again(lane));
    if (!MANY || w + stride >= jobs) return;
    if constexpr (MANY) {
      if (load_slice + 1 < load_slices)
        ++load_slice;
      else
        load_next_job();
      w += stride;
      // every wave is done with its staged outputs
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int d = 0; d < EARLY; ++d) load_one(st, d);
    }
  }
#undef RPX_MX_STEP
#undef RPX_MX_READS
}

template <int BM, int BN, int WM, int WN, int NS, int WPE, bool GATED, bool MANY>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
    k_mx_gemm(MxGemm p, int64_t slices_per_split, int tiles_m, int tiles_n, int splits, int band,
              float* partials) {
  // Tiles are dealt to the XCDs in contiguous ranges of a banded order, so the
  // tiles that an XCD runs at once share few rows of A and B in its L2; splits are
  // outermost.
  const int tiles = tiles_m * tiles_n;
  auto job_at = [&](int w) {
    MxJob job;
    job.p = p;
    const int b = xcd_block(w, tiles * splits);
    const int split = b / tiles;
    band_tile(b % tiles, tiles_m, tiles_n, band, job.tile_m, job.tile_n);
    job.first_slice = split * slices_per_split;
    const int64_t left = p.slices - job.first_slice;
    job.slices = static_cast<int>(left < slices_per_split ? left : slices_per_split);
    job.partial = partials == nullptr
                      ? nullptr
                      : partials + (static_cast<int64_t>(split) * tiles +
                                    job.tile_m * tiles_n + job.tile_n) * (BM * BN);
    return job;
  };
  mx_gemm_tiles<BM, BN, WM, WN, NS, GATED, MANY>(blockIdx.x, gridDim.x, tiles * splits, job_at);
}

// Two products in one launch: the first tiles are p's, the others q's. A workgroup takes
// one tile: they are of two lengths, which the order of dispatch evens out (the gated
// block's step of 5003 x 2048 -> 6144: 335 us, with MANY 359).
template <int BM, int BN, int WM, int WN, int NS, int WPE>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
    k_mx_gemm_pair(MxGemm p, MxGemm q, int p_tiles_n, int p_tiles, int q_tiles_n, int q_tiles,
                   int band) {
  auto job_at = [&](int w) {
    const bool first = w < p_tiles;
    const int tiles = first ? p_tiles : q_tiles;
    const int tiles_n = first ? p_tiles_n : q_tiles_n;
    MxJob job;
    job.p = first ? p : q;
    band_tile(xcd_block(first ? w : w - p_tiles, tiles), tiles / tiles_n, tiles_n, band, job.tile_m,
              job.tile_n);
    job.first_slice = 0;
    job.slices = static_cast<int>(job.p.slices);
    job.partial = nullptr;
    return job;
  };
  mx_gemm_tiles<BM, BN, WM, WN, NS, false, false>(blockIdx.x, gridDim.x, p_tiles + q_tiles, job_at);
}

// Sums the partial tiles of a split product in split order. One thread per
// 16-byte chunk: consecutive threads read consecutive chunks of every split.
template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(256)
    k_mx_split_reduce(const float* __restrict__ partials, int splits, int64_t M, int64_t N,
                      int tiles_n, int64_t tiles, void* __restrict__ out, int dtype) {
  constexpr int TM = BM / WM;
  constexpr int TN = BN / WN;
  constexpr int FM = TM / 32;
  constexpr int FN = TN / 32;
  constexpr int CHUNKS = BM * BN / 4;
  const int64_t q = block_of_grid() * 256 + threadIdx.x;
  if (q >= tiles * CHUNKS) return;
  const f32x4_t* p = reinterpret_cast<const f32x4_t*>(partials);
  f32x4_t s = p[q];
  for (int i = 1; i < splits; ++i) s += p[i * tiles * CHUNKS + q];
  const int64_t tile = q / CHUNKS;
  int r = static_cast<int>(q % CHUNKS);
  const int lane = r & 63;
  r >>= 6;
  const int g = r & 3;
  r >>= 2;
  const int fm = r % FM;
  r /= FM;
  const int fn = r % FN;
  const int wave = r / FN;
  const int64_t m = (tile / tiles_n) * BM + (wave % WM) * TM + fm * 32 + (lane & 31);
  const int64_t n = (tile % tiles_n) * BN + (wave / WM) * TN + fn * 32 + 8 * g + 4 * (lane >> 5);
  if (m >= M) return;
  const float y[4] = {s[0], s[1], s[2], s[3]};
  if (dtype != kBF16) {
    store4(static_cast<float*>(out) + m * N + n, n, N, y);
    return;
  }
  uint16_t* d = static_cast<uint16_t*>(out) + m * N + n;
  if (n + 3 < N && (N & 3) == 0) {
    *reinterpret_cast<u32x2_t*>(d) = u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  } else {
    for (int e = 0; e < 4; ++e)
      if (n + e < N) d[e] = f32_to_bf16(y[e]);
  }
}

// Tiles: id, rows of A, rows of B, waves along each, stages, waves per SIMD. (A 256 x
// 256 tile of four waves, which reads less of LDS but has one wave a SIMD, measured as
// the first: 257 against 253 us at 8192 x 8192 <- 8192; 256 x 128 with three stages 290;
// two workgroups a CU of 192 x 128, whose scales bypass LDS for room, 306 and 282 against
// 254 for the gated block of 16384 x 2048 -> 2 x 6144.)
#define RPX_MX_CONFIGS(X)     \
  X(1, 256, 256, 4, 2, 2, 2)  \
  X(2, 128, 128, 2, 2, 2, 2)  \
  X(3, 128, 128, 2, 2, 4, 1)  \
  X(4, 64, 128, 2, 2, 2, 2)   \
  X(5, 64, 64, 2, 1, 2, 2)

struct Plan {
  int id, bm, bn;
  int64_t tiles_m, tiles_n;
  int splits;
  int64_t per_split;
};

Plan plan_for(int id, int64_t m, int64_t n, int64_t slices, bool gated) {
  Plan p{};
  p.id = id;
  switch (id) {
#define X(ID, BM, BN, WM, WN, NS, WPE) \
  case ID:                             \
    p.bm = BM;                         \
    p.bn = BN;                         \
    break;
    RPX_MX_CONFIGS(X)
#undef X
  }
  p.tiles_m = ceil_div(m, p.bm);
  p.tiles_n = ceil_div(n, gated ? p.bn / 2 : p.bn);
  p.splits = 1;
  p.per_split = slices;
  return p;
}

// The tile: large where it fills the card, for fewer reads from LDS and the L2 a
// product; smaller where that leaves CUs idle. Measured (us, bf16 outputs,
// M x N <- K; tiles by id):
//   16384 x 2048 <- 6144   1: 94, 2: 114, 4: 158     8192 x 8192 <- 8192   1: 235, 2: 297
//   8192 x 3072 <- 768     1: 20.0, 2: 19.0      gated 16384 x 3072 <- 768   1: 59, 2: 71
//   8192 x 768 <- 3072     1: 20.6, 2: 16.1, 4: 20.1
//   333 x 6144 <- 2048     2: 7.5, 4: 8.0, 5: 7.7
//   1024 x 2048 <- 2048    2: 7.5, 4: 6.7, 5: 7.0
//   3072 x 768 <- 8192     2: 23.9, 3: 17.2, 4: 22.3 (144 tiles of 2 and 3: one a CU,
//                          where 3's four stages take the place of a second workgroup)
//   3500 x 768 <- 3072     2: 9.7, 3: 9.8
template <class TilesOf>
int tile_for(TilesOf tiles_of, int64_t slices) {
  if (tune(kTuneMxTile) != 0) return tune(kTuneMxTile);
  const int64_t large = tiles_of(1), medium = tiles_of(2);
  if (large >= 192 && (slices >= 6 || large >= 1024)) return 1;
  if (medium >= 140) return medium <= 256 && slices >= 24 ? 3 : 2;
  return tiles_of(4) >= 192 ? 4 : 5;
}

// Parts of a sum, for a product whose tiles leave CUs idle; the partial tiles and
// their sum cost 3 to 15 us by their size. Whole / split, us, operands from memory:
//   tiles 4 and 5, 48 slices and more:
//     256 x 256 <- 12288 (16 tiles) 27.6 / 13.9, 768 x 768 <- 12288 (144) 27.5 / 18.0,
//     <- 16384 35.1 / 19.5, 512 x 3072 <- 12288 (192) 40.2 / 31.2, 1024 x 2048 <- 12288
//     (256) 30.5 / 29.5
//   the same, 32 to 40 slices: 256 x 256 <- 8192 19.3 / 13.5, 768 x 768 <- 8192 19.4 /
//     15.4, but 1024 x 2048 <- 8192 22.1 / 22.0, 512 x 3072 <- 10240 26.0 / 26.9; and a
//     backward's other product is then not in the same launch (8192 x 1024 -> 1024, the
//     step 64.8 / 65.4)
//   tile 3 in three parts: 768 x 3072 <- 16384 40.0 / 46.4, <- 32768 74 / 72; in a
//     backward, 28672 x 3072 -> 768 147 / 159, 32768 168 / 172, 32768 x 768 -> 3072 201 /
//     192, 36864 x 3072 -> 768 203 / 195, 65536 x 768 -> 3072 387 / 358
//   tile 3 in two parts, and the larger tiles: 2048 x 2048 <- 16384 42.7 / 57.2, <- 65536
//     156 / 167; the backward of 16384 x 2048 -> 6144 276 / 312, of 16384 x 6144 -> 2048
//     240 / 285
int64_t splits_for(int id, int64_t tiles, int64_t slices) {
  if (tiles == 0) return 1;
  if (id == 3) return slices >= 128 && tiles <= 512 / 3 ? 512 / tiles : 1;
  if (id < 4 || slices < 48) return 1;
  const int64_t splits = 512 / tiles;
  return splits < slices / 16 ? splits : slices / 16;
}

Plan choose(int64_t m, int64_t n, int64_t slices, bool gated) {
  const int id = tile_for(
      [&](int c) {
        const Plan p = plan_for(c, m, n, slices, gated);
        return p.tiles_m * p.tiles_n;
      },
      slices);
  Plan p = plan_for(id, m, n, slices, gated);
  const int64_t tiles = p.tiles_m * p.tiles_n;
  int64_t splits = tune(kTuneMxSplits);
  if (splits == 0) splits = splits_for(id, tiles, slices);
  if (gated) splits = 1;
  if (splits > slices / 4) splits = slices / 4;
  if (splits > 1) {
    p.per_split = ceil_div(slices, splits);
    p.splits = static_cast<int>(ceil_div(slices, p.per_split));
  }
  return p;
}

constexpr int lds_bytes(int bm, int bn, int stages) {
  return stages * ((bm + bn) * static_cast<int>(kMxSliceBytes) + (bm + bn + 127) / 128 * 1024);
}

constexpr int64_t kCus = 256;
constexpr int64_t kMaxRows = (int64_t{1} << 31) - 1024;  // of an operand
constexpr int64_t kMaxJobs = int64_t{1} << 30;

// Workgroups that the card holds at once, of the tiles that launches of more are made
// of: two stages (waits that count loads cannot have stores between them), and not the
// small ones, which tile_for takes for products of few tiles.
constexpr int64_t resident(int bm, int bn, int stages) {
  return stages == 2 && bm * bn >= 128 * 128
             ? kCus * (160 * 1024 / lds_bytes(bm, bn, stages))
             : kMaxJobs;
}

// Launches a kernel of NW waves a workgroup with LDS bytes of shared memory; `done` is
// the kernel's own.
template <int NW, int LDS, class... Params, class... Args>
hipError_t start(void (*kernel)(Params...), std::atomic<unsigned>& done, int64_t groups,
                 hipStream_t stream, const Args&... args) {
  static_assert(LDS <= 160 * 1024, "LDS");
  if (hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(kernel), LDS, done);
      e != hipSuccess)
    return e;
  kernel<<<dim3(static_cast<unsigned>(groups)), dim3(64 * NW), LDS, stream>>>(
      static_cast<Params>(args)...);
  return hipGetLastError();
}

int band_of() { return tune(kTuneBand) > 0 ? tune(kTuneBand) : 4; }

template <int BM, int BN, int WM, int WN, int NS, int WPE>
hipError_t launch_pair_config(const MxGemm& p, const MxGemm& q, const Plan& pp, const Plan& qp,
                              hipStream_t stream) {
  constexpr int LDS = lds_bytes(BM, BN, NS);
  const int64_t p_tiles = pp.tiles_m * pp.tiles_n;
  const int64_t q_tiles = qp.tiles_m * qp.tiles_n;
  const int64_t jobs = p_tiles + q_tiles;
  if (jobs > kMaxJobs) return hipErrorInvalidValue;
  static std::atomic<unsigned> done{0};
  return start<WM * WN, LDS>(k_mx_gemm_pair<BM, BN, WM, WN, NS, WPE>, done, jobs, stream, p, q,
                             pp.tiles_n, p_tiles, qp.tiles_n, q_tiles, band_of());
}

template <int BM, int BN, int WM, int WN, int NS, int WPE, bool GATED>
hipError_t launch_config(const MxGemm& g, const Plan& p, float* partials, hipStream_t stream) {
  constexpr int LDS = lds_bytes(BM, BN, NS);
  constexpr int64_t kResident = resident(BM, BN, NS);
  const int64_t tiles = p.tiles_m * p.tiles_n;
  const int64_t jobs = tiles * p.splits;
  if (jobs > kMaxJobs) return hipErrorInvalidValue;
  if (p.splits == 1) partials = nullptr;
  static std::atomic<unsigned> one{0}, many{0};
  auto run = [&] {
    if constexpr (kResident < kMaxJobs)
      if (jobs > kResident)
        return start<WM * WN, LDS>(k_mx_gemm<BM, BN, WM, WN, NS, WPE, GATED, true>, many, kResident,
                                   stream, g, p.per_split, p.tiles_m, p.tiles_n, p.splits,
                                   band_of(), partials);
    return start<WM * WN, LDS>(k_mx_gemm<BM, BN, WM, WN, NS, WPE, GATED, false>, one, jobs, stream,
                               g, p.per_split, p.tiles_m, p.tiles_n, p.splits, band_of(), partials);
  };
  if (hipError_t e = run(); e != hipSuccess) return e;
  if (p.splits > 1) {
    const int64_t chunks = tiles * (BM * BN / 4);
    k_mx_split_reduce<BM, BN, WM, WN><<<grid_of(ceil_div(chunks, 256)), dim3(256), 0, stream>>>(
        partials, p.splits, g.m, g.n, static_cast<int>(p.tiles_n), tiles, g.out, g.dtype);
  }
  return hipGetLastError();
}

}  // namespace

int mx_tile_count() {
  int count = 0;
#define X(...) ++count;
  RPX_MX_CONFIGS(X)
#undef X
  return count;
}

int64_t mx_gemm_workspace_floats(int64_t m, int64_t n, int64_t slices) {
  const Plan p = choose(m, n, slices, false);
  return p.splits > 1 ? p.tiles_m * p.tiles_n * p.splits * p.bm * p.bn : 0;
}

hipError_t launch_mx_gemm(const MxGemm& g, float* partials, hipStream_t stream) {
  if (g.m == 0 || g.n == 0) return hipSuccess;
  if (g.m > kMaxRows || g.n > kMaxRows) return hipErrorInvalidValue;
  const bool gated = g.b2_codes != nullptr;
  const Plan p = choose(g.m, g.n, g.slices, gated);
  switch (p.id) {
#define X(ID, BM, BN, WM, WN, NS, WPE)                                            \
  case ID:                                                                        \
    return gated ? launch_config<BM, BN, WM, WN, NS, WPE, true>(g, p, partials, stream) \
                 : launch_config<BM, BN, WM, WN, NS, WPE, false>(g, p, partials, stream);
    RPX_MX_CONFIGS(X)
#undef X
  }
  return hipErrorInvalidValue;
}

// A backward's two products in one launch, in the tile that suits them together,
// the longer sums first: a product's last round of tiles leaves CUs idle, which the
// other's then fill, and there is one launch. A whole step in graph replays, one
// launch against two: the linear of 1001 x 500 -> 1300 29.7 / 34.8 us, of 3500 x 3072
// -> 768 59.7 / 67.6, of 5003 x 2048 -> 6144 162 / 173, its gated block 315 / 354; of
// 16384 x 2048 -> 2048 220 / 220.
// A product that is split runs on its own, so that an output has the same bits
// whether or not the other one is wanted.
// The 256 x 256 tile is for launches whose longest tile ends with the others: one of few
// tiles over a long sum runs on by itself, where a launch of its own takes a smaller tile.
// Slices of the longest sum beyond an even share of all, and a backward with its encoding
// in graph replays, one launch / two, us (m x k -> n): none, 5003 x 2048 -> 6144 91 / 101,
// 16384 x 2048 -> 6144 269 / 276; 8, 4096 x 2048 -> 2048 38.0 / 40.5; 16, 8192 x 2048 ->
// 2048 64 / 60 on one card and 68.5 / 69 on another; 24, 12288 x 2048 -> 2048 90 / 83; 46,
// 16384 x 768 -> 3072 118 / 89; 64, 32768 x 2048 -> 2048 276 / 204. The 128 x 128 tile has
// two workgroups a CU: 28, 16384 x 3072 -> 768 73 / 77; 35, 20480 x 3072 -> 768 88 / 92.
constexpr int64_t kMxPairExcess = 16;
hipError_t launch_mx_gemm_pair(const MxGemm& a, const MxGemm& b, float* partials,
                               hipStream_t stream) {
  const bool alone = a.m == 0 || a.n == 0 || b.m == 0 || b.n == 0 || tune(kTuneMxPair) == 0 ||
                     choose(a.m, a.n, a.slices, false).splits > 1 ||
                     choose(b.m, b.n, b.slices, false).splits > 1 ||
                     a.m > kMaxRows || a.n > kMaxRows || b.m > kMaxRows || b.n > kMaxRows;
  auto apart = [&] {
    const hipError_t e = launch_mx_gemm(a, partials, stream);
    return e != hipSuccess ? e : launch_mx_gemm(b, partials, stream);
  };
  if (alone) return apart();
  const MxGemm& p = a.slices >= b.slices ? a : b;
  const MxGemm& q = a.slices >= b.slices ? b : a;
  const int64_t slices = q.slices;
  auto tiles_of = [&](int id) {
    const Plan x = plan_for(id, p.m, p.n, p.slices, false);
    const Plan y = plan_for(id, q.m, q.n, q.slices, false);
    return x.tiles_m * x.tiles_n + y.tiles_m * y.tiles_n;
  };
  const int id = tile_for(tiles_of, slices);
  const Plan pp = plan_for(id, p.m, p.n, p.slices, false);
  const Plan qp = plan_for(id, q.m, q.n, q.slices, false);
  const int64_t share =
      ceil_div(pp.tiles_m * pp.tiles_n * p.slices + qp.tiles_m * qp.tiles_n * q.slices, kCus);
  if (id == 1 && tune(kTuneMxTile) == 0 && p.slices - share > kMxPairExcess) return apart();
  switch (id) {
#define X(ID, BM, BN, WM, WN, NS, WPE) \
  case ID:                             \
    return launch_pair_config<BM, BN, WM, WN, NS, WPE>(p, q, pp, qp, stream);
    RPX_MX_CONFIGS(X)
#undef X
  }
  return hipErrorInvalidValue;
}

}  // namespace rpx

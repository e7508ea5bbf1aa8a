// The boundary between two blocks of a transformer, for rows of x (the stream)
// and u (the update that the first block computed):
//   p = post(u)            a norm after the block, or u itself
//   t = x + c drop(g p)    its gate, dropout and residual scale; rounded to the
//                          stream's type, as it is stored
//   h = norm(t)            the norm before the next block, of that t
// and its gradients, with those of the norms' weights and of the gate. A norm is
// a LayerNorm or an RMSNorm; statistics, sums and everything between the loads
// and the stores are f32.
//
// A pass over memory: a row lives in the registers of L lanes, eight consecutive
// values a lane and chunk; x and u are read once, t and h written once. The
// backward reads dt, dh, t and u, recomputes the statistics, the normalised rows
// and the dropout's bits, and writes dx and du.
//
// The sums over rows (weights, biases, gate) are kept by the lanes that own the
// columns, over the rows that a worker (L lanes) takes one after another, and
// joined by a second launch in a fixed order: no atomics, so a call gives the
// same bits every time. A worker's rows lie in one group of rows that share a
// gate, or are whole groups.
//
// Bound by HBM: 16384 rows of 2048 bf16 with a gate and two RMSNorms 51 us forward (268
// MB, 5.3 TB/s), 89 backward (403 MB, 4.5 TB/s) and 8 for the join; 5003 rows of 768 with a
// LayerNorm 12, 18 and 6. A wave a row of 2048 took 65 us forward against 50.
#include "kernels.h"
#include "vector8.h"

namespace rpx {

namespace {

// Sums of K values over the L lanes of a row, the same in each lane, in a fixed
// order. Rows of more than one wave meet in LDS; two buffers in turn need one
// barrier a sum.
template <int L, int K>
struct RowSum {
  float (*lds)[K][L / 64 > 0 ? L / 64 : 1];
  int parity = 0;
  __device__ __forceinline__ void operator()(float (&v)[K]) {
    constexpr int W = L < 64 ? L : 64;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int off = W / 2; off > 0; off >>= 1) v[k] += __shfl_xor(v[k], off, 64);
    if constexpr (L > 64) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) lds[parity][k][wave] = v[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < L / 64; ++w) s += lds[parity][k][w];
        v[k] = s;
      }
      parity ^= 1;
    }
  }
};

constexpr int threads_of(int lanes) { return lanes > 64 ? lanes : 256; }

// Eight weights from column e on; `round` rounds a float32 master to the values'
// type first (a LayerNorm takes its weights in that type).
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_weight8(const void* w, int dtype, bool round, int64_t e,
                                             int count, float* v) {
  if (dtype == kBF16) {
    load_row8<WHOLE>(static_cast<const Bf16*>(w) + e, count, v);
    return;
  }
  load_row8<WHOLE>(static_cast<const float*>(w) + e, count, v);
  if (round) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = rounded(static_cast<const T*>(nullptr), v[i]);
  }
}

// A workgroup's rows are those it reaches in steps of the grid; the next ones' loads
// run under these ones' arithmetic, and with one chunk a lane the weights stay in
// registers.
template <typename T, int L, int C, bool WHOLE>
__global__ void __launch_bounds__(threads_of(L)) k_block_fwd(BlockArgs a) {
  constexpr int kRows = threads_of(L) / L;
  constexpr bool KEEP = C == 1;
  __shared__ float lds[2][2][L / 64 > 0 ? L / 64 : 1];
  RowSum<L, 2> row_sum{lds};
  const int lane = threadIdx.x & (L - 1);
  const int size = a.size;
  const float inv = 1.0f / static_cast<float>(size);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / L;
  const bool has_post = a.post.weight != nullptr, post_layer = a.post.kind == kNormLayer;
  const bool has_norm = a.norm.weight != nullptr, norm_layer = a.norm.kind == kNormLayer;
  auto weights = [&](const BlockNorm& n, bool there, bool layer, int c, float* w, float* b) {
    const int e = (c * L + lane) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = b[i] = 0.0f;
    if (!there || e >= size) return;
    load_weight8<WHOLE, T>(n.weight, n.dtype, layer, e, size - e, w);
    if (layer) load_weight8<WHOLE, T>(n.bias, n.dtype, true, e, size - e, b);
  };
  Raw8<T> rx[C], ru[C];
  auto load = [&](int64_t at) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * L + lane) * 8;
      rx[c].zero();
      ru[c].zero();
      if (e >= size) continue;
      load_raw8<WHOLE>(static_cast<const T*>(a.u) + at * size + e, size - e, ru[c]);
      load_raw8<WHOLE>(static_cast<const T*>(a.x) + at * size + e, size - e, rx[c]);
    }
  };
  if (row < a.rows) load(row);
  float pw[8], pb[8], nw[8], nb[8], gw[8];
  if constexpr (KEEP) {
    weights(a.post, has_post, post_layer, 0, pw, pb);
    weights(a.norm, has_norm, norm_layer, 0, nw, nb);
  }
  auto gate = [&](int64_t at, int c, float* g) {
    const int e = (c * L + lane) * 8;
    if (e < size)
      load_weight8<WHOLE, T>(a.gate, a.gate_dtype, false, (at / a.rows_per_gate) * size + e,
                             size - e, g);
  };
  PhiloxCall call{};
  const bool drop = a.drop.threshold < 65536u;
  if (drop) call = philox_call(a.drop);
  for (; row < a.rows; row += step) {
    const int64_t base = row * size;
    if (KEEP && a.gate != nullptr) gate(row, 0, gw);
    float v[C][8], r[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      ru[c].get(v[c]);
      rx[c].get(r[c]);
    }
    if (row + step < a.rows) load(row + step);
    // mean and 1 / deviation of the row in v, whose entries past the end are zero
    auto statistics = [&](bool layer, float eps, float& mean, float& rstd) {
      float s[2] = {0.0f, 0.0f};
      mean = 0.0f;
      if (layer) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) s[0] += v[c][i];
        row_sum(s);
        mean = s[0] * inv;
      }
      s[0] = s[1] = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int n = size - (c * L + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = v[c][i] - mean;
          if (WHOLE ? n > 0 : i < n) s[0] = __builtin_fmaf(d, d, s[0]);
        }
      }
      row_sum(s);
      rstd = rsqrtf(s[0] * inv + eps);
    };
    float mean, rstd;
    if (has_post) {
      statistics(post_layer, a.post.eps, mean, rstd);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if constexpr (!KEEP) weights(a.post, true, post_layer, c, pw, pb);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = __builtin_fmaf((v[c][i] - mean) * rstd, pw[i], pb[i]);
      }
    }
    if (a.gate != nullptr) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if constexpr (!KEEP) gate(row, c, gw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] *= gw[i];
      }
    }
    if (drop) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = (c * L + lane) * 8;
        if (e < size) dropout8<WHOLE>(call, a.drop, base + e, v[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * L + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[c][i] = rounded(static_cast<const T*>(nullptr),
                          i < size - e ? __builtin_fmaf(a.scale, v[c][i], r[c][i]) : 0.0f);
      if (e < size) store_row8<WHOLE>(static_cast<T*>(a.t) + base + e, size - e, v[c]);
    }
    if (!has_norm) continue;
    statistics(norm_layer, a.norm.eps, mean, rstd);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * L + lane) * 8;
      if constexpr (!KEEP) weights(a.norm, true, norm_layer, c, nw, nb);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = __builtin_fmaf((v[c][i] - mean) * rstd, nw[i], nb[i]);
      if (e < size) store_row8<WHOLE>(static_cast<T*>(a.h) + base + e, size - e, v[c]);
    }
  }
}

// What a lane sums over a worker's rows: the columns of its chunks.
enum Column : int { kWeight = 0, kBias = 1, kPostWeight = 2, kPostBias = 3, kGate = 4, kColumns = 5 };

// MEAN: one of the norms is a LayerNorm. The next row's loads run under this one's
// arithmetic; with one chunk a lane its weights stay in registers too.
template <typename T, int L, int C, bool WHOLE, bool MEAN>
__global__ void __launch_bounds__(threads_of(L)) k_block_bwd(BlockGradients a) {
  constexpr int kThreads = threads_of(L);
  constexpr int kWorkers = kThreads / L;
  constexpr bool KEEP = C == 1;
  __shared__ float sums[2][4][L / 64 > 0 ? L / 64 : 1];
  // the columns of this workgroup's workers, where there are several
  __shared__ float meet[kWorkers > 1 ? kWorkers * L * C * 8 : 1];
  RowSum<L, 4> row_sum{sums};
  const BlockArgs& f = a.forward;
  const int lane = threadIdx.x & (L - 1);
  const int64_t worker = block_of_grid() * kWorkers + threadIdx.x / L;
  const int size = f.size;
  const float inv = 1.0f / static_cast<float>(size);
  const bool has_norm = f.norm.weight != nullptr && a.dh != nullptr;
  const bool has_post = f.post.weight != nullptr;
  const bool has_gate = f.gate != nullptr;
  const bool norm_mean = MEAN && has_norm && f.norm.kind == kNormLayer;
  const bool post_mean = MEAN && has_post && f.post.kind == kNormLayer;
  const bool read_u = has_post || has_gate;
  float acc[kColumns][C][8];
#pragma unroll
  for (int k = 0; k < kColumns; ++k)
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[k][c][i] = 0.0f;
  // the worker's rows: slice worker % slices of a group, or whole groups
  int64_t row, end;
  if (a.slices > 0) {
    const int64_t group = worker / a.slices;
    row = group * a.group_rows + (worker % a.slices) * a.worker_rows;
    end = row + a.worker_rows;
    const int64_t last = (group + 1) * a.group_rows;
    end = end < last ? end : last;
  } else {
    row = worker * a.worker_rows;
    end = row + a.worker_rows;
  }
  end = end < f.rows ? end : f.rows;
  if (worker >= a.workers) row = end = 0;
  PhiloxCall call{};
  const bool drop = f.drop.threshold < 65536u;
  if (drop) call = philox_call(f.drop);
  int64_t group_left = a.slices > 0 ? end - row : a.group_rows;  // rows to the group's end

  auto norm_weight = [&](int c, float* w) {
    const int e = (c * L + lane) * 8;
    load_weight8<WHOLE, T>(f.norm.weight, f.norm.dtype, norm_mean, e, size - e, w);
  };
  auto post_weight = [&](int c, float* w, float* b) {
    const int e = (c * L + lane) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = 1.0f;
      b[i] = 0.0f;
    }
    if (!has_post) return;
    load_weight8<WHOLE, T>(f.post.weight, f.post.dtype, post_mean, e, size - e, w);
    if (post_mean) load_weight8<WHOLE, T>(f.post.bias, f.post.dtype, true, e, size - e, b);
  };
  auto gate_weight = [&](int c, int64_t at, float* k) {
    const int e = (c * L + lane) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = 1.0f;
    if (has_gate) load_weight8<WHOLE, T>(f.gate, f.gate_dtype, false, at + e, size - e, k);
  };
  float nw[8], pw[8], pb[8], gw[8];
  int64_t gate_row = -1;
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < 8; ++i) nw[i] = 0.0f;
    if (lane * 8 < size) {
      if (has_norm) norm_weight(0, nw);
      post_weight(0, pw, pb);
    }
  }
  Raw8<T> rt[C], ru[C], rg[C], rd[C];
  auto load = [&](int64_t at) {
    const int64_t base = at * size;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * L + lane) * 8;
      rt[c].zero();
      ru[c].zero();
      rg[c].zero();
      rd[c].zero();
      if (e >= size) continue;
      if (has_norm) {
        load_raw8<WHOLE>(static_cast<const T*>(f.t) + base + e, size - e, rt[c]);
        load_raw8<WHOLE>(static_cast<const T*>(a.dh) + base + e, size - e, rg[c]);
      }
      if (a.dt != nullptr) load_raw8<WHOLE>(static_cast<const T*>(a.dt) + base + e, size - e, rd[c]);
      if (read_u) load_raw8<WHOLE>(static_cast<const T*>(f.u) + base + e, size - e, ru[c]);
    }
  };
  if (row < end) load(row);
  for (; row < end; ++row) {
    const int64_t base = row * size;
    float t[C][8], u[C][8], g[C][8], d[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      rt[c].get(t[c]);
      ru[c].get(u[c]);
      rg[c].get(g[c]);
      rd[c].get(d[c]);
    }
    if (row + 1 < end) load(row + 1);
    const int64_t gate_at = has_gate ? (row / f.rows_per_gate) * size : 0;
    if constexpr (KEEP) {
      if (gate_at != gate_row && lane * 8 < size) gate_weight(0, gate_at, gw);
      gate_row = gate_at;
    }
    float mean = 0.0f, u_mean = 0.0f;
    if constexpr (MEAN) {
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[0] += t[c][i];
          s[1] += u[c][i];
        }
      row_sum(s);
      mean = norm_mean ? s[0] * inv : 0.0f;
      u_mean = post_mean ? s[1] * inv : 0.0f;
    }
    // the statistics, and what the norm's gradient takes out of its row:
    // sum (t - mean)^2, sum (u - mean)^2, sum w dh, sum w dh (t - mean)
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * L + lane) * 8;
      if (e >= size) continue;
      if constexpr (!KEEP) {
#pragma unroll
        for (int i = 0; i < 8; ++i) nw[i] = 0.0f;
        if (has_norm) norm_weight(c, nw);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!WHOLE && i >= size - e) continue;
        t[c][i] -= mean;
        s[0] = __builtin_fmaf(t[c][i], t[c][i], s[0]);
        u[c][i] -= u_mean;
        s[1] = __builtin_fmaf(u[c][i], u[c][i], s[1]);
        const float v = g[c][i] * nw[i];
        s[2] += v;
        s[3] = __builtin_fmaf(v, t[c][i], s[3]);
      }
    }
    row_sum(s);
    const float u_rstd = has_post ? rsqrtf(s[1] * inv + f.post.eps) : 1.0f;
    if (has_norm) {
      const float rstd = rsqrtf(s[0] * inv + f.norm.eps);
      const float mg = norm_mean ? s[2] * inv : 0.0f;
      const float mgt = s[3] * rstd * inv;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = (c * L + lane) * 8;
        if (e >= size) continue;
        if constexpr (!KEEP) norm_weight(c, nw);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = t[c][i] * rstd;
          acc[kWeight][c][i] = __builtin_fmaf(g[c][i], n, acc[kWeight][c][i]);
          if constexpr (MEAN) acc[kBias][c][i] += g[c][i];
          d[c][i] = __builtin_fmaf(rstd, g[c][i] * nw[i] - mg - n * mgt, d[c][i]);
        }
      }
    }
    // d is the gradient of t, and of x; from here on d becomes that of p, with
    // u the normalised row
    float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * L + lane) * 8;
      if (e >= size) continue;
      if (a.dx != nullptr) store_row8<WHOLE>(static_cast<T*>(a.dx) + base + e, size - e, d[c]);
      if (drop) dropout8<WHOLE>(call, f.drop, base + e, d[c]);
      if constexpr (!KEEP) {
        post_weight(c, pw, pb);
        gate_weight(c, gate_at, gw);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!WHOLE && i >= size - e) continue;
        u[c][i] *= u_rstd;
        d[c][i] *= f.scale;
        const float p = MEAN ? __builtin_fmaf(u[c][i], pw[i], pb[i]) : u[c][i] * pw[i];
        acc[kGate][c][i] = __builtin_fmaf(d[c][i], p, acc[kGate][c][i]);
        d[c][i] *= gw[i];
        acc[kPostWeight][c][i] = __builtin_fmaf(d[c][i], u[c][i], acc[kPostWeight][c][i]);
        if constexpr (MEAN) acc[kPostBias][c][i] += d[c][i];
        d[c][i] *= pw[i];
        q[0] += d[c][i];
        q[1] = __builtin_fmaf(d[c][i], u[c][i], q[1]);
      }
    }
    float md = 0.0f, mdu = 0.0f;
    if (has_post) {
      row_sum(q);
      md = post_mean ? q[0] * inv : 0.0f;
      mdu = q[1] * inv;
    }
    if (a.du != nullptr) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = (c * L + lane) * 8;
        if (e >= size) continue;
        if (has_post) {
#pragma unroll
          for (int i = 0; i < 8; ++i) d[c][i] = u_rstd * (d[c][i] - md - u[c][i] * mdu);
        }
        store_row8<WHOLE>(static_cast<T*>(a.du) + base + e, size - e, d[c]);
      }
    }
    if (a.dgate != nullptr && --group_left == 0) {
      // whole groups: the gate's gradient as it is; a slice: for the joining launch
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = (c * L + lane) * 8;
        if (e < size) {
          if (a.gate_partials != nullptr)
            store_row8<WHOLE>(a.gate_partials + worker * size + e, size - e, acc[kGate][c]);
          else if (f.gate_dtype == kBF16)
            store_row8<WHOLE>(static_cast<Bf16*>(a.dgate) + gate_at + e, size - e, acc[kGate][c]);
          else
            store_row8<WHOLE>(static_cast<float*>(a.dgate) + gate_at + e, size - e, acc[kGate][c]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[kGate][c][i] = 0.0f;
      }
      group_left = a.group_rows;
    }
  }
  if (a.partials == nullptr) return;
  // one row of partials a workgroup: [workgroup][column][size]
#pragma unroll
  for (int k = 0; k < kGate; ++k) {
    if (a.columns[k] == nullptr) continue;
    float* out = a.partials + (block_of_grid() * kGate + k) * size;
    if constexpr (kWorkers > 1) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          meet[(threadIdx.x / L) * (L * C * 8) + (c * L + lane) * 8 + i] = acc[k][c][i];
      __syncthreads();
      for (int e = threadIdx.x; e < size; e += kThreads) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWorkers; ++w) s += meet[w * (L * C * 8) + e];
        out[e] = s;
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = (c * L + lane) * 8;
        if (e < size) store_row8<WHOLE>(out + e, size - e, acc[k][c]);
      }
    }
  }
}

// Joins the partials of one column for 16 of its entries: 64 lanes an entry, each
// over every 64th partial, then over LDS, in a fixed order.
constexpr int kJoin = 16;
struct BlockJoin {
  const float* partials;
  int64_t count, stride;  // partials and floats from one to the next
  void* out;
  int dtype;
};

__device__ __forceinline__ void join(const BlockJoin& j, int size, int64_t e0) {
  __shared__ float lds[64][17], half[16][17];
  const int c = threadIdx.x & 15;
  const int part = threadIdx.x >> 4;
  const int64_t e = e0 + c;
  float s = 0.0f;
  if (e < size) {
    int64_t p = part;
    for (; p + 64 * 7 < j.count; p += 64 * 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = j.partials[(p + 64 * i) * j.stride + e];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; p < j.count; p += 64) s += j.partials[p * j.stride + e];
  }
  lds[part][c] = s;
  __syncthreads();
  if (part < 16) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += lds[4 * part + i][c];
    half[part][c] = s;
  }
  __syncthreads();
  if (part == 0 && e < size) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += half[i][c];
    if (j.dtype == kBF16)
      store1(static_cast<Bf16*>(j.out) + e, s);
    else
      store1(static_cast<float*>(j.out) + e, s);
  }
}

// The same for a group's slices, of which there are few: a thread an entry.
__device__ __forceinline__ void join_few(const BlockJoin& j, int size, int64_t e) {
  if (e >= size) return;
  float s = 0.0f;
  int64_t p = 0;
  for (; p + 7 < j.count; p += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = j.partials[(p + i) * j.stride + e];
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
  }
  for (; p < j.count; ++p) s += j.partials[p * j.stride + e];
  if (j.dtype == kBF16)
    store1(static_cast<Bf16*>(j.out) + e, s);
  else
    store1(static_cast<float*>(j.out) + e, s);
}

// Gates of more slices than this join as the columns do (one gate for all rows).
constexpr int64_t kFewSlices = 64;

__host__ __device__ inline int64_t join_blocks(int size, bool few) {
  return few ? ceil_div(size, 1024) : ceil_div(size, kJoin);
}

__global__ void __launch_bounds__(1024) k_block_join(BlockGradients a, int64_t workgroups,
                                                     int columns, int64_t gates) {
  const int size = a.forward.size;
  const int64_t blocks = join_blocks(size, false);
  int64_t block = block_of_grid();
  if (block < columns * blocks) {
    const int64_t job = block / blocks;
    int k = 0;
    for (int64_t left = job; k < kGate; ++k)
      if (a.columns[k] != nullptr && left-- == 0) break;
    const int dtype = k < kPostWeight ? a.forward.norm.dtype : a.forward.post.dtype;
    join(BlockJoin{a.partials + k * size, workgroups, static_cast<int64_t>(kGate) * size,
                   a.columns[k], dtype},
         size, (block % blocks) * kJoin);
    return;
  }
  block -= columns * blocks;
  const bool few = a.slices <= kFewSlices;
  const int64_t gate_blocks = join_blocks(size, few);
  const int64_t g = block / gate_blocks;
  if (g >= gates) return;
  const size_t bytes = a.forward.gate_dtype == kBF16 ? 2 : 4;
  const BlockJoin j{a.gate_partials + g * a.slices * size, a.slices, size,
                    static_cast<uint8_t*>(a.dgate) + g * size * bytes, a.forward.gate_dtype};
  if (few)
    join_few(j, size, (block % gate_blocks) * 1024 + threadIdx.x);
  else
    join(j, size, (block % gate_blocks) * kJoin);
}

// Lanes a row and chunks a lane: a wave while one chunk a lane holds the row, then more
// waves, so that rows, weights and the backward's five sums a column stay in registers.
#define RPX_BLOCK_SIZES(CALL) \
  if (size <= 128) {          \
    CALL(16, 1);              \
  } else if (size <= 512) {   \
    CALL(64, 1);              \
  } else if (size <= 1024) {  \
    CALL(128, 1);             \
  } else if (size <= 2048) {  \
    CALL(256, 1);             \
  } else if (size <= 4096) {  \
    CALL(512, 1);             \
  } else {                    \
    CALL(512, 2);             \
  }

// The split of the rows over workers: as many waves as run at a time (registers allow
// two a SIMD with a LayerNorm's sums, three without), one round of them.
constexpr int64_t kMeanWaves = 256 * 8, kWaves = 256 * 12;

bool has_mean(const BlockArgs& f) {
  return (f.norm.weight != nullptr && f.norm.kind == kNormLayer) ||
         (f.post.weight != nullptr && f.post.kind == kNormLayer);
}

constexpr int64_t kForwardWaves = 256 * 20;  // that run at a time

template <typename T, bool WHOLE>
void forward(const BlockArgs& a, hipStream_t stream) {
  const int size = a.size;
#define RPX_FWD(L, C)                                                                      \
  {                                                                                        \
    const int64_t all = ceil_div(a.rows, threads_of(L) / L);                               \
    const int64_t most = kForwardWaves * 64 / threads_of(L);                               \
    hipLaunchKernelGGL((k_block_fwd<T, L, C, WHOLE>),                                      \
                       dim3(static_cast<unsigned>(all < most ? all : most)),               \
                       dim3(threads_of(L)), 0, stream, a);                                 \
  }
  RPX_BLOCK_SIZES(RPX_FWD)
#undef RPX_FWD
}

template <typename T, bool WHOLE>
void backward(const BlockGradients& a, int64_t workgroups, hipStream_t stream) {
  const int size = a.forward.size;
  const bool mean = has_mean(a.forward);
#define RPX_BWD(L, C)                                                                         \
  if (mean)                                                                                   \
    hipLaunchKernelGGL((k_block_bwd<T, L, C, WHOLE, true>), grid_of(workgroups),              \
                       dim3(threads_of(L)), 0, stream, a);                                    \
  else                                                                                        \
    hipLaunchKernelGGL((k_block_bwd<T, L, C, WHOLE, false>), grid_of(workgroups),             \
                       dim3(threads_of(L)), 0, stream, a)
  RPX_BLOCK_SIZES(RPX_BWD)
#undef RPX_BWD
}

struct Split {
  int64_t slices, worker_rows, workers, workgroups, gates;
};

Split split_of(int64_t rows, int size, int64_t group_rows, bool mean) {
  const int at_once = size <= 128 ? 16 : (size <= 512 ? 4 : 1);  // rows of a workgroup
  const int waves = size <= 512 ? 4 : (size <= 1024 ? 2 : (size <= 2048 ? 4 : 8));
  const int64_t want = ceil_div(rows, (mean ? kMeanWaves : kWaves) / waves * at_once);
  Split s{};
  const int64_t groups = group_rows > 0 ? ceil_div(rows, group_rows) : 0;
  if (groups == 0) return s;
  if (group_rows > want) {
    s.slices = ceil_div(group_rows, want);
    s.worker_rows = ceil_div(group_rows, s.slices);
    s.slices = ceil_div(group_rows, s.worker_rows);
    s.workers = groups * s.slices;
  } else {
    s.worker_rows = (want / group_rows) * group_rows;
    s.workers = ceil_div(rows, s.worker_rows);
  }
  s.workgroups = ceil_div(s.workers, at_once);
  s.gates = s.slices > 1 ? groups : 0;
  return s;
}

}  // namespace

int64_t block_gradients_floats(const BlockArgs& f, bool columns, bool gate) {
  const int size = f.size;
  const Split s = split_of(f.rows, size, gate ? f.rows_per_gate : f.rows, has_mean(f));
  return (columns ? s.workgroups * kGate * size : 0) +
         (gate && s.gates > 0 ? s.workers * size : 0);
}

hipError_t launch_block_forward(const BlockArgs& a, hipStream_t stream) {
  if (a.rows <= 0) return hipSuccess;
  const bool whole = a.size % 8 == 0;
  if (a.dtype == kBF16)
    whole ? forward<Bf16, true>(a, stream) : forward<Bf16, false>(a, stream);
  else
    whole ? forward<float, true>(a, stream) : forward<float, false>(a, stream);
  return hipGetLastError();
}

hipError_t launch_block_backward(BlockGradients a, float* scratch, hipStream_t stream) {
  const BlockArgs& f = a.forward;
  if (f.rows <= 0) return hipSuccess;
  a.group_rows = a.dgate != nullptr ? f.rows_per_gate : f.rows;
  const Split s = split_of(f.rows, f.size, a.group_rows, has_mean(f));
  a.slices = s.slices;
  a.worker_rows = s.worker_rows;
  a.workers = s.workers;
  int columns = 0;
  for (int k = 0; k < kGate; ++k) columns += a.columns[k] != nullptr;
  a.partials = columns > 0 ? scratch : nullptr;
  const bool gates = a.dgate != nullptr && s.gates > 0;
  a.gate_partials = gates ? scratch + (columns > 0 ? s.workgroups * kGate * f.size : 0) : nullptr;
  const bool whole = f.size % 8 == 0;
  if (f.dtype == kBF16)
    whole ? backward<Bf16, true>(a, s.workgroups, stream)
          : backward<Bf16, false>(a, s.workgroups, stream);
  else
    whole ? backward<float, true>(a, s.workgroups, stream)
          : backward<float, false>(a, s.workgroups, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || (columns == 0 && !gates)) return e;
  const int64_t gate_count = gates ? s.gates : 0;
  const int64_t blocks = columns * join_blocks(f.size, false) +
                         gate_count * join_blocks(f.size, s.slices <= kFewSlices);
  hipLaunchKernelGGL(k_block_join, grid_of(blocks), dim3(1024), 0, stream, a, s.workgroups, columns,
                     gate_count);
  return hipGetLastError();
}

}  // namespace rpx

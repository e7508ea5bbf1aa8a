// Dropout with a mask that is made from a counter (philox.h) and never stored:
// forward and backward are the same pass, x in, x times 65536 / threshold or zero
// out. Bound by HBM: 16384 x 2048 bf16 (134 MB) 22 us, 6 TB/s with part of it in the
// cache; 1001 x 777 float32 3.1 us.
#include "kernels.h"
#include "vector8.h"

namespace rpx {

namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_dropout(const T* __restrict__ x, int64_t count, Dropout d, T* __restrict__ out) {
  const int64_t first = 8 * (block_of_grid() * kThreads + threadIdx.x);
  if (first >= count) return;
  const int n = count - first < 8 ? static_cast<int>(count - first) : 8;
  float v[8];
  load_row8<false>(x + first, n, v);
  // no dropout: there may be no key
  if (d.threshold < 65536u) dropout8<true>(philox_call(d), d, first, v);
  store_row8<false>(out + first, n, v);
}

}  // namespace

hipError_t launch_dropout(const void* x, int dtype, int64_t count, const Dropout& d, void* out,
                          hipStream_t stream) {
  if (count <= 0) return hipSuccess;
  const dim3 grid = grid_of(ceil_div(count, 8 * kThreads));
  if (dtype == kBF16)
    hipLaunchKernelGGL(k_dropout<Bf16>, grid, dim3(kThreads), 0, stream,
                       static_cast<const Bf16*>(x), count, d, static_cast<Bf16*>(out));
  else
    hipLaunchKernelGGL(k_dropout<float>, grid, dim3(kThreads), 0, stream,
                       static_cast<const float*>(x), count, d, static_cast<float*>(out));
  return hipGetLastError();
}

}  // namespace rpx

// dropout.cuh — y = x / (1 - p) where the element's Philox word says so, else 0.
#pragma once

#include "block.cuh"

namespace hc {

constexpr int kDropThreads = 256;

// One Philox block serves four consecutive elements, so a thread takes four.
template <typename T>
__global__ void __launch_bounds__(kDropThreads) dropout_elem(const T* x, T* y, int64_t N, DropArgs d) {
  const DropKey key = drop_key(d);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kDropThreads;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; 4 * b < N; b += stride) {
    const uint4 w = philox4(key, static_cast<uint64_t>(b));
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t i = 4 * b + e;
      if (i < N) y[i] = Elem<T>::from_f(drop_value(d, word[e], Elem<T>::to_f(x[i])));
    }
  }
}

template <typename T>
int dropout_launch(const void* x, void* y, int64_t N, const DropArgs& d, cudaStream_t s) {
  const int64_t want = ((N + 3) / 4 + kDropThreads - 1) / kDropThreads;
  const int grid = static_cast<int>(want < 8 * sm_count() ? want : 8 * sm_count());
  dropout_elem<T><<<grid, kDropThreads, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(y), N, d);
  return launch_status();
}

}  // namespace hc

// dropout.cuh — y = x / (1 - p) where the element's Philox word says so, else 0.
//
// A block of four words is ten rounds of two 32 x 32 -> 64 bit products and two
// three-input xors (the round keys, the same for all, stay in registers), about
// 80 instructions for the eight elements that a thread moves at a time. 33.5M
// elements in one direction: bf16 36 us (floor 20.5), float32 47 (41). In bf16
// no pipe is full (ALU 56%, the multipliers 37%, issue 59 of 100 cycles at 86% of
// the warps): a warp waits 28% of its time for its 16 bytes, half of it for a pipe
// or its turn.
#pragma once

#include "block.cuh"

namespace hc {

constexpr int kDropThreads = 256;

// Groups of eight elements: two generator blocks, one or two 16-byte words.
// VECTOR: x and y on 16-byte boundaries. The last N % 8 elements go to the
// thread behind the last whole group.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const T* x, T* y, int64_t N, const __grid_constant__ DropArgs d) {
  constexpr int Q = sizeof(T) / 2;
  const DropKey key = drop_key(d);
  RoundKeys rk(key);
#pragma unroll
  for (int r = 0; r < 10; ++r) asm volatile("" : "+r"(rk.a[r]), "+r"(rk.b[r]));  // made once, not in every round again
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kDropThreads, groups = N / 8;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; 8 * b < N; b += stride) {
    float f[8];
    const bool whole = b < groups;
    if (VECTOR && whole) {
#pragma unroll
      for (int i = 0; i < Q; ++i) unpack<T>(ld_nc_v4(x + 8 * b + i * (16 / sizeof(T))), f + i * (16 / sizeof(T)));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 8 * b + e < N ? Elem<T>::to_f(x[8 * b + e]) : 0.f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 w = philox4(rk, key.o0, key.o1, static_cast<uint64_t>(2 * b + h));
      const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[4 * h + e] = drop_value(d, word[e], f[4 * h + e]);
      }
    }
    if (VECTOR && whole) {
#pragma unroll
      for (int i = 0; i < Q; ++i) st_v4(y + 8 * b + i * (16 / sizeof(T)), pack<T>(f + i * (16 / sizeof(T))));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * b + e < N) y[8 * b + e] = Elem<T>::from_f(f[e]);
    }
  }
}

template <typename T>
int dropout_launch(const void* x, void* y, int64_t N, const DropArgs& d, cudaStream_t s) {
  const int64_t want = ((N + 7) / 8 + kDropThreads - 1) / kDropThreads, most = 24 * static_cast<int64_t>(sm_count());
  const int grid = static_cast<int>(want < most ? want : most);
  // x may be y, which the non-coherent loads of the vector kernel allow: a
  // thread reads its own elements before it writes them
  if (aligned16(x) && aligned16(y))
    dropout_kernel<T, true><<<grid, kDropThreads, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(y), N, d);
  else
    dropout_kernel<T, false><<<grid, kDropThreads, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(y), N, d);
  return launch_status();
}

}  // namespace hc

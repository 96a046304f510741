// ffn_simt.cu — the gated feed-forward's float32 products on the FMA units (the
// tensor cores have no float32 inputs): any size and order, 64 x 64 tiles of
// the result by 256 threads, 4 x 4 a thread.
#include "ffn.cuh"

namespace hc {
namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256, kPitch = kTile + 4;

// The tile [64 rows][16 k] of an operand into shared memory as [k][row],
// neighbouring threads along the operand's unit stride.
template <typename T>
__device__ __forceinline__ void load_tile(const FfnOperand& o, int64_t row0, int64_t k0, int64_t K, float (&r)[4]) {
  const T* p = static_cast<const T*>(o.p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x + i * kThreads;
    const int64_t row = row0 + (o.k_stride == 1 ? e / kDepth : e % kTile);
    const int64_t k = k0 + (o.k_stride == 1 ? e % kDepth : e / kTile);
    r[i] = row < o.rows && k < K ? Elem<T>::to_f(p[row * o.row_stride + k * o.k_stride]) : 0.f;
  }
}
__device__ __forceinline__ void put_tile(const FfnOperand& o, const float (&r)[4], float (*s)[kPitch]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x + i * kThreads;
    if (o.k_stride == 1)
      s[e % kDepth][e / kDepth] = r[i];
    else
      s[e / kTile][e % kTile] = r[i];
  }
}

template <typename T, int EPI>
__global__ void __launch_bounds__(kThreads) ffn_simt_kernel(FfnProduct p) {
  constexpr int NB = EPI == kGlu ? 2 : 1;
  __shared__ float sA[kDepth][kPitch], sB[NB][kDepth][kPitch];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
  float acc[NB][4][4] = {};
  for (int term = 0; term < p.terms; ++term) {
    float ra[4], rb[NB][4];
    load_tile<T>(p.A[term], m0, 0, p.K, ra);
#pragma unroll
    for (int b = 0; b < NB; ++b) load_tile<T>(p.B[term + b], n0, 0, p.K, rb[b]);
    for (int64_t k0 = 0; k0 < p.K; k0 += kDepth) {
      put_tile(p.A[term], ra, sA);
#pragma unroll
      for (int b = 0; b < NB; ++b) put_tile(p.B[term + b], rb[b], sB[b]);
      __syncthreads();
      if (k0 + kDepth < p.K) {  // the next tile travels while this one is used
        load_tile<T>(p.A[term], m0, k0 + kDepth, p.K, ra);
#pragma unroll
        for (int b = 0; b < NB; ++b) load_tile<T>(p.B[term + b], n0, k0 + kDepth, p.K, rb[b]);
      }
#pragma unroll
      for (int k = 0; k < kDepth; ++k) {
        const float4 av = *reinterpret_cast<const float4*>(&sA[k][4 * ty]);
        const float a[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float4 bv = *reinterpret_cast<const float4*>(&sB[b][k][4 * tx]);
          const float w[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[b][i][j] = fmaf(a[i], w[j], acc[b][i][j]);
        }
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + 4 * ty + i, n = n0 + 4 * tx + j;
      if (m >= p.M || n >= p.N) continue;
      const int64_t at = m * p.ldo + n;
      if constexpr (EPI == kStore) {
        static_cast<T*>(p.out)[at] = Elem<T>::from_f(acc[0][i][j]);
      } else if constexpr (EPI == kGlu) {
        const float a = acc[0][i][j], b = acc[NB - 1][i][j];
        float val, der;
        ffn_act(p.act, a, val, der);
        static_cast<T*>(p.out)[at] = Elem<T>::from_f(val * b);
        if (p.slope_gate) {
          static_cast<T*>(p.slope_gate)[at] = Elem<T>::from_f(der * b);
          static_cast<T*>(p.slope_up)[at] = Elem<T>::from_f(val);
        }
      } else {
        const float dh = acc[0][i][j];
        static_cast<T*>(p.out)[at] = Elem<T>::from_f(dh * Elem<T>::to_f(static_cast<const T*>(p.slope_gate)[at]));
        static_cast<T*>(p.out2)[at] = Elem<T>::from_f(dh * Elem<T>::to_f(static_cast<const T*>(p.slope_up)[at]));
      }
    }
}

template <typename T> int launch(const FfnProduct& p, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.N + kTile - 1) / kTile), static_cast<unsigned>((p.M + kTile - 1) / kTile));
  switch (p.epilogue) {
    case kStore: ffn_simt_kernel<T, kStore><<<grid, kThreads, 0, s>>>(p); break;
    case kGlu: ffn_simt_kernel<T, kGlu><<<grid, kThreads, 0, s>>>(p); break;
    default: ffn_simt_kernel<T, kGluBwd><<<grid, kThreads, 0, s>>>(p); break;
  }
  return launch_status();
}

}  // namespace

int ffn_simt_launch(const FfnProduct& p, cudaStream_t s) { return launch<float>(p, s); }

}  // namespace hc

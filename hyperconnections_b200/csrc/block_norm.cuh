// block_norm.cuh — the norm kernels for rows of whole 8-column chunks (D a
// multiple of 8, 16-byte aligned streams).
//
// A token belongs to a group of W = ceil(D / 256) warps: a CTA for W > 1, one
// of a CTA's four warps for W = 1. A thread owns eight columns of every row, so
// that a token is read once, kept in registers (16-bit rows stay packed) over
// the norm's sums, and written once. The groups walk the tokens grid-strided;
// several CTAs an SM keep enough loads in flight.
//
// Sums over a token: a warp folds its values by halving exchanges (every
// exchange sends half of the live values, so k values cost about k + 5 - log k
// shuffles), writes them to shared memory, and after the group's barrier every
// thread adds the W warps' in order. The backward has two rounds: the norm's
// two sums, which the gradients wait for, and the token's small matrices (R, or
// H and W), which nothing waits for: those are added one token later, behind
// the next token's barrier, so a token costs one barrier. Shared memory is
// double-buffered by token for that.
//
// The [m D] parameters' gradients are sums over tokens: a thread keeps its
// columns' sums in registers over all of its group's tokens and writes them
// once; block_capi.cu adds the groups' sums in order.
#pragma once

#include "block_elem.cuh"

namespace hc {

constexpr int kColumns = 8;      // a thread's columns
constexpr int kSmallGroups = 4;  // groups of a CTA when a group is one warp

// Threads of a CTA at most, which bounds the registers of one: the backward of
// 8 streams holds 16 rows, the float32 kernels twice the words a row.
constexpr int norm_max_threads(bool bwd, int N, int esize) {
  return N == 8 ? (bwd || esize == 4 ? 256 : 512) : (bwd && N == 4 && esize == 4) ? 256 : 512;
}

template <typename T> struct Raw8 {
  static constexpr int Q = sizeof(T) / 2;  // 16-byte words
  uint4 q[Q];
  __device__ __forceinline__ void load(const T* p, bool ok) {
#pragma unroll
    for (int i = 0; i < Q; ++i) q[i] = ok ? ld_nc_v4(p + i * (16 / sizeof(T))) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < Q; ++i) unpack<T>(q[i], f + i * (16 / sizeof(T)));
  }
};
template <typename T> __device__ __forceinline__ void put8(T* p, const float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < Raw8<T>::Q; ++i) st_v4(p + i * (16 / sizeof(T)), pack<T>(f + i * (16 / sizeof(T))));
}
// Eight values of a 16-byte aligned float32 parameter, or `none`.
__device__ __forceinline__ void param8(const float* p, int64_t c, bool ok, float none, float (&f)[8]) {
  float4 q[2] = {make_float4(none, none, none, none), make_float4(none, none, none, none)};
  if (p && ok) {
    q[0] = __ldg(reinterpret_cast<const float4*>(p + c));
    q[1] = __ldg(reinterpret_cast<const float4*>(p + c) + 1);
  }
  f[0] = q[0].x; f[1] = q[0].y; f[2] = q[0].z; f[3] = q[0].w;
  f[4] = q[1].x; f[5] = q[1].y; f[6] = q[1].z; f[7] = q[1].w;
}

constexpr int log2_of(int k) { return k <= 1 ? 0 : 1 + log2_of(k / 2); }

// Warp-wide sums of K values (a power of two up to 32): lane l ends with the
// sum of value l >> (5 - log2 K) in v[0].
template <int K, int O = 16> __device__ __forceinline__ void warp_fold(float* v, int lane) {
  if constexpr (O > 0) {
    if constexpr (K > 1) {
      tr_step<K>(v, lane, O);
      warp_fold<K / 2, O / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(kFull, v[0], O);
      warp_fold<1, O / 2>(v, lane);
    }
  }
}
template <int K> __device__ __forceinline__ void fold_to(float* v, int lane, float* dst) {
  warp_fold<K>(v, lane);
  constexpr int shift = 5 - log2_of(K);
  if ((lane & ((1 << shift) - 1)) == 0) dst[lane >> shift] = v[0];
}

// Where a thread stands: group, warp and thread in it, and its columns.
struct Place {
  int W, group, warp, lane, tid;
  int64_t d0;
  bool live;  // owns columns of the row
  __device__ __forceinline__ Place(int warps, int64_t D) {
    W = warps;
    lane = threadIdx.x & 31;
    const int w = threadIdx.x >> 5;
    group = W == 1 ? w : 0;
    warp = W == 1 ? 0 : w;
    tid = warp * 32 + lane;
    d0 = static_cast<int64_t>(tid) * kColumns;
    live = d0 < D;
  }
  __device__ __forceinline__ void sync() const {
    if (W == 1)
      __syncwarp();
    else
      __syncthreads();
  }
  __device__ __forceinline__ int64_t first() const {
    return W == 1 ? static_cast<int64_t>(blockIdx.x) * kSmallGroups + group : blockIdx.x;
  }
  __device__ __forceinline__ int64_t stride() const {
    return W == 1 ? static_cast<int64_t>(gridDim.x) * kSmallGroups : gridDim.x;
  }
  __device__ __forceinline__ int slot() const { return threadIdx.x >> 5; }  // this warp's row of a shared buffer
  __device__ __forceinline__ int slot0() const { return W == 1 ? group : 0; }
};

// Mean and 1 / root of the group's values u[0..K) of each live thread; `red` is
// one buffer, a float4 a warp. The variance of a LayerNorm is merged from
// (count, mean, sum of squared deviations) triples pair by pair, which loses
// nothing where the mean is large against the deviations.
template <int K, int MAXW>
__device__ __forceinline__ void group_stats(const Place& p, const float* u, int per_thread, int norm, float eps,
                                            float total, float4 (&red)[MAXW], float& mean, float& rstd) {
  mean = 0.f;
  if (norm == HC_NORM_RMS) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < K; ++i) s = fmaf(u[i], u[i], s);  // columns and blocks that do not exist hold 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    if (p.W > 1) {
      if (p.lane == 0) red[p.slot()].x = s;
      p.sync();
      s = 0.f;
      for (int w = 0; w < p.W; ++w) s += red[w].x;
    }
    rstd = 1.f / sqrtf(s / total + eps);
    return;
  }
  float c = p.live ? static_cast<float>(per_thread) : 0.f, mu = 0.f, m2 = 0.f;
  if (p.live) {
#pragma unroll
    for (int i = 0; i < K; ++i) mu += u[i];
    mu /= c;
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i < per_thread) m2 = fmaf(u[i] - mu, u[i] - mu, m2);
  }
  auto merge = [&](float c2, float mu2, float m22) {
    const float n = c + c2;
    if (n > 0.f) {
      const float d = mu2 - mu, share = c2 / n;
      mu = fmaf(d, share, mu);
      m2 += m22 + d * d * c * share;
      c = n;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float c2 = __shfl_xor_sync(kFull, c, o), mu2 = __shfl_xor_sync(kFull, mu, o),
                m22 = __shfl_xor_sync(kFull, m2, o);
    // both partners take the pair in the same order, so that every lane gets the same bits
    if (p.lane & o) {
      const float c1 = c, mu1 = mu, m21 = m2;
      c = c2; mu = mu2; m2 = m22;
      merge(c1, mu1, m21);
    } else {
      merge(c2, mu2, m22);
    }
  }
  if (p.W > 1) {
    if (p.lane == 0) red[p.slot()] = make_float4(c, mu, m2, 0.f);
    p.sync();
    c = mu = m2 = 0.f;
    for (int w = 0; w < p.W; ++w) {
      const float4 r = red[w];
      merge(r.x, r.y, r.z);
    }
  }
  mean = mu;
  rstd = 1.f / sqrtf(m2 / total + eps);
}

// u[k] = sum_j R[k][j] x[j] of this thread's columns.
template <typename T, int N, int M>
__device__ __forceinline__ void read_rows(const float* R, const Raw8<T> (&x)[N], int n, int m, float (&u)[M][8]) {
#pragma unroll
  for (int k = 0; k < M; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) u[k][e] = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= n) break;
    float xv[8];
    x[j].get(xv);
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (k >= m) break;
      const float r = __ldg(R + k * n + j);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[k][e] = fmaf(r, xv[e], u[k][e]);
    }
  }
}

// The groups' sums of the [m D] parameters' gradients; with several groups a
// CTA each adds its own row.
template <int M>
__device__ __forceinline__ void store_param_sums(const NormArgs& a, const Place& p, const float (&A)[M][8],
                                                 const float (&B)[M][8]) {
  if (!a.partial || !p.live) return;
  const int64_t E = a.D * a.m;
  const int64_t row = p.W == 1 ? static_cast<int64_t>(blockIdx.x) * kSmallGroups + p.group : blockIdx.x;
  float* dst = a.partial + row * 2 * E;
#pragma unroll
  for (int k = 0; k < M; ++k) {
    if (k >= a.m) break;
    const int64_t c = k * a.D + p.d0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dst[c + e] = A[k][e];
      dst[E + c + e] = B[k][e];
    }
  }
}

// ------------------------------------------------------------------- read
template <typename T, int N, int M>
__global__ void __launch_bounds__(norm_max_threads(false, N, sizeof(T)))
    read_norm_fwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  constexpr int MAXW = norm_max_threads(false, N, sizeof(T)) / 32;
  __shared__ float4 red[2][MAXW];
  const Place p(warps, a.D);
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  int buf = 0;
  for (int64_t t = p.first(); t < a.T; t += p.stride(), buf ^= 1) {
    const T* x = static_cast<const T*>(a.x) + t * n * D + p.d0;
    Raw8<T> xr[N];
#pragma unroll
    for (int j = 0; j < N; ++j) xr[j].load(x + j * D, p.live && j < n);
    float u[M][8];
    read_rows<T, N, M>(a.R + t * m * n, xr, n, m, u);
    float mean, rstd;
    group_stats<8 * M>(p, &u[0][0], 8 * m, a.norm, a.eps, static_cast<float>(E), red[buf], mean, rstd);
    if (a.stats && p.tid == 0) {
      a.stats[2 * t] = mean;
      a.stats[2 * t + 1] = rstd;
    }
    if (p.live) {
      T* y = static_cast<T*>(a.out) + t * E + p.d0;
#pragma unroll
      for (int k = 0; k < M; ++k) {
        if (k >= m) break;
        float w[8], b[8];
        param8(a.weight, k * D + p.d0, true, 1.f, w);
        param8(a.bias, k * D + p.d0, true, 0.f, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[k][e] = fmaf((u[k][e] - mean) * rstd, w[e], b[e]);
        put8<T>(y + k * D, u[k]);
      }
    }
    __syncwarp();
  }
}

template <typename T, int N, int M>
__global__ void __launch_bounds__(norm_max_threads(true, N, sizeof(T)))
    read_norm_bwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  constexpr int MAXW = norm_max_threads(true, N, sizeof(T)) / 32, G = N * M;
  __shared__ float red[2][MAXW][2], gram[2][MAXW][G];
  const Place p(warps, a.D);
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  float A[M][8] = {}, B[M][8] = {};
  int buf = 0;
  int64_t last = -1;
  // grad_R of token t, whose warps' sums lie in buffer b
  auto flush = [&](int64_t t, int b) {
    if (!a.grad_R || t < 0) return;
    for (int i = p.tid; i < G; i += 32 * p.W) {
      const int k = i / N, j = i % N;
      if (k >= m || j >= n) continue;
      float s = 0.f;
      for (int w = 0; w < p.W; ++w) s += gram[b][p.slot0() + w][i];
      a.grad_R[t * m * n + k * n + j] = s;
    }
  };
  for (int64_t t = p.first(); t < a.T; t += p.stride(), buf ^= 1) {
    const T* x = static_cast<const T*>(a.x) + t * n * D + p.d0;
    const T* g = static_cast<const T*>(a.g) + t * E + p.d0;
    const float* R = a.R + t * m * n;
    Raw8<T> xr[N], gr[M];
#pragma unroll
    for (int k = 0; k < M; ++k) gr[k].load(g + k * D, p.live && k < m);
#pragma unroll
    for (int j = 0; j < N; ++j) xr[j].load(x + j * D, p.live && j < n);
    const float mean = __ldg(a.stats + 2 * t), rstd = __ldg(a.stats + 2 * t + 1);
    float u[M][8];
    read_rows<T, N, M>(R, xr, n, m, u);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (k >= m) break;
      float w[8], gv[8];
      gr[k].get(gv);
      param8(a.weight, k * D + p.d0, p.live, 1.f, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[k][e] = (u[k][e] - mean) * rstd;  // xhat
        const float q = gv[e] * w[e];
        s[0] = fmaf(q, u[k][e], s[0]);
        s[1] += q;
        A[k][e] = fmaf(gv[e], u[k][e], A[k][e]);
        B[k][e] += gv[e];
      }
    }
    if (!p.live) s[0] = s[1] = 0.f;
    fold_to<2>(s, p.lane, red[buf][p.slot()]);
    p.sync();
    flush(last, buf ^ 1);
    float c1 = 0.f, c2 = 0.f;
    for (int w = 0; w < p.W; ++w) {
      c1 += red[buf][p.slot0() + w][0];
      c2 += red[buf][p.slot0() + w][1];
    }
    c1 /= static_cast<float>(E);
    c2 = a.norm == HC_NORM_LAYER ? c2 / static_cast<float>(E) : 0.f;
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (k >= m) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[k][e] = 0.f;
        continue;
      }
      float w[8], gv[8];
      gr[k].get(gv);
      param8(a.weight, k * D + p.d0, p.live, 1.f, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[k][e] = p.live ? rstd * (gv[e] * w[e] - c2 - u[k][e] * c1) : 0.f;  // du
    }
    if (a.grad_x && p.live) {
      T* gx = static_cast<T*>(a.grad_x) + t * n * D + p.d0;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j >= n) break;
        float r[8] = {};
#pragma unroll
        for (int k = 0; k < M; ++k) {
          if (k >= m) break;
          const float rk = __ldg(R + k * n + j);
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = fmaf(rk, u[k][e], r[e]);
        }
        put8<T>(gx + j * D, r);
      }
    }
    if (a.grad_R) {
      float acc[G];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float xv[8];
        xr[j].get(xv);
#pragma unroll
        for (int k = 0; k < M; ++k) {
          float r = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) r = fmaf(u[k][e], xv[e], r);
          acc[k * N + j] = r;
        }
      }
      fold_to<G>(acc, p.lane, gram[buf][p.slot()]);
    }
    last = t;
  }
  p.sync();
  flush(last, buf ^ 1);
  store_param_sums<M>(a, p, A, B);
}

// -------------------------------------------------------------- mix-write
// Keep factors (0 or 1 / (1 - p)) of this thread's eight columns of block k.
__device__ __forceinline__ void keep8(const DropArgs& d, const DropKey& key, uint64_t element, float (&f)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 w = philox4(key, (element >> 2) + h);
    f[4 * h] = w.x >= d.threshold ? d.scale : 0.f;
    f[4 * h + 1] = w.y >= d.threshold ? d.scale : 0.f;
    f[4 * h + 2] = w.z >= d.threshold ? d.scale : 0.f;
    f[4 * h + 3] = w.w >= d.threshold ? d.scale : 0.f;
  }
}

// H + (v - H v) v^T of token t into shared memory, by the group's first threads.
template <int N>
__device__ __forceinline__ void stage_mix(const NormArgs& a, const Place& p, int64_t t, float (&sH)[N * N]) {
  const int n = a.n;
  for (int i = p.tid; i < n * n; i += 32 * p.W)
    sH[(i / n) * N + i % n] = mix_entry(a.H + t * n * n, a.v ? a.v + t * n : nullptr, n, i / n, i % n);
}

template <typename T, int N, int M>
__global__ void __launch_bounds__(norm_max_threads(false, N, sizeof(T)))
    write_norm_fwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  constexpr int MAXW = norm_max_threads(false, N, sizeof(T)) / 32;
  __shared__ float4 red[2][MAXW];
  __shared__ float sH[2][kSmallGroups][N * N];
  const Place p(warps, a.D);
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  int buf = 0;
  for (int64_t t = p.first(); t < a.T; t += p.stride(), buf ^= 1) {
    const T* x = static_cast<const T*>(a.x) + t * n * D + p.d0;
    const T* f = static_cast<const T*>(a.f) + t * E + p.d0;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + t * E + p.d0 : nullptr;
    Raw8<T> fr[M], xr[N], ar[M];
#pragma unroll
    for (int k = 0; k < M; ++k) fr[k].load(f + k * D, p.live && k < m);
#pragma unroll
    for (int k = 0; k < M; ++k) ar[k].load(gate + k * D, gate && p.live && k < m);
#pragma unroll
    for (int j = 0; j < N; ++j) xr[j].load(x + j * D, p.live && j < n);
    stage_mix<N>(a, p, t, sH[buf][p.group]);
    float z[M][8];
#pragma unroll
    for (int k = 0; k < M; ++k) fr[k].get(z[k]);
    float mean = 0.f, rstd = 1.f;
    if (a.norm != HC_NORM_NONE) {
      group_stats<8 * M>(p, &z[0][0], 8 * m, a.norm, a.eps, static_cast<float>(E), red[buf], mean, rstd);
      if (a.stats && p.tid == 0) {
        a.stats[2 * t] = mean;
        a.stats[2 * t + 1] = rstd;
      }
    }
    if (a.norm == HC_NORM_NONE || p.W == 1) p.sync();  // sH; with a norm over several warps its barrier did it
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (k >= m || !p.live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[k][e] = 0.f;
        continue;
      }
      const int64_t c = k * D + p.d0;
      float w[8], b[8];
      param8(a.weight, c, true, 1.f, w);
      param8(a.bias, c, true, 0.f, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[k][e] = fmaf((z[k][e] - mean) * rstd, w[e], b[e]);
      if (gate) {
        ar[k].get(w);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[k][e] *= gate_value(a.gate_act, w[e]);
      }
      if (a.scale) {
        param8(a.scale, c, true, 1.f, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[k][e] *= w[e];
      }
      if (a.drop.on) {
        keep8(a.drop, key, static_cast<uint64_t>(t * E + c), w);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[k][e] = w[e] != 0.f ? z[k][e] * w[e] : 0.f;
      }
    }
    if (p.live) {
      float xv[N][8];
#pragma unroll
      for (int j = 0; j < N; ++j) xr[j].get(xv[j]);
      T* out = static_cast<T*>(a.out) + t * n * D + p.d0;
      const float* W = a.W + t * n * m;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i >= n) break;
        float r[8] = {};
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (j >= n) break;
          const float h = sH[buf][p.group][i * N + j];
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = fmaf(h, xv[j][e], r[e]);
        }
#pragma unroll
        for (int k = 0; k < M; ++k) {
          if (k >= m) break;
          const float w = __ldg(W + i * m + k);
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = fmaf(w, z[k][e], r[e]);
        }
        put8<T>(out + i * D, r);
      }
    }
    __syncwarp();
  }
}

template <typename T, int N, int M>
__global__ void __launch_bounds__(norm_max_threads(true, N, sizeof(T)))
    write_norm_bwd_kernel(const __grid_constant__ NormArgs a, int warps) {
  constexpr int MAXW = norm_max_threads(true, N, sizeof(T)) / 32;
  constexpr int GB = N * N < 32 ? N * N : 32, G = N * N + N * M;  // H's sums by batches of GB, then W's
  __shared__ float red[2][MAXW][2], gram[2][MAXW][G], sH[2][kSmallGroups][N * N], sG[kSmallGroups][N * N];
  const Place p(warps, a.D);
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  float A[M][8] = {}, B[M][8] = {};
  int buf = 0;
  int64_t last = -1;
  // grad_H, grad_v and grad_W of token t, whose warps' sums lie in buffer b
  auto flush = [&](int64_t t, int b) {
    if (t < 0) return;
    for (int i = p.tid; i < G; i += 32 * p.W) {
      float s = 0.f;
      for (int w = 0; w < p.W; ++w) s += gram[b][p.slot0() + w][i];
      if (i < N * N) {
        const int r = i / N, c = i % N;
        if (r >= n || c >= n) continue;
        if (a.v)
          sG[p.group][r * n + c] = s;
        else if (a.grad_H)
          a.grad_H[t * n * n + r * n + c] = s;
      } else if (a.grad_W) {
        const int r = (i - N * N) / M, k = (i - N * N) % M;
        if (r < n && k < m) a.grad_W[(t * n + r) * m + k] = s;
      }
    }
    if (a.v) {
      p.sync();
      for (int i = p.tid; i < n * n; i += 32 * p.W)
        mix_grads(sG[p.group], a.H + t * n * n, a.v + t * n, n, i, a.grad_H ? a.grad_H + t * n * n : nullptr,
                  a.grad_v ? a.grad_v + t * n : nullptr);
    }
  };
  for (int64_t t = p.first(); t < a.T; t += p.stride(), buf ^= 1) {
    const T* x = static_cast<const T*>(a.x) + t * n * D + p.d0;
    const T* g = static_cast<const T*>(a.g) + t * n * D + p.d0;
    const T* f = static_cast<const T*>(a.f) + t * E + p.d0;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + t * E + p.d0 : nullptr;
    const float* W = a.W + t * n * m;
    Raw8<T> gr[N], xr[N], fr[M], ar[M];
#pragma unroll
    for (int j = 0; j < N; ++j) gr[j].load(g + j * D, p.live && j < n);
#pragma unroll
    for (int k = 0; k < M; ++k) fr[k].load(f + k * D, p.live && k < m);
#pragma unroll
    for (int k = 0; k < M; ++k) ar[k].load(gate + k * D, gate && p.live && k < m);
#pragma unroll
    for (int j = 0; j < N; ++j) xr[j].load(x + j * D, p.live && j < n);
    const float mean = a.norm == HC_NORM_NONE ? 0.f : __ldg(a.stats + 2 * t);
    const float rstd = a.norm == HC_NORM_NONE ? 1.f : __ldg(a.stats + 2 * t + 1);
    stage_mix<N>(a, p, t, sH[buf][p.group]);
    // pg[k] = dz behind dropout, times act(gate); z; the gradients of gate
    float pg[M][8], z[M][8];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < M; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) pg[k][e] = z[k][e] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= n) break;
      float gv[8];
      gr[i].get(gv);
#pragma unroll
      for (int k = 0; k < M; ++k) {
        if (k >= m) break;
        const float w = __ldg(W + i * m + k);
#pragma unroll
        for (int e = 0; e < 8; ++e) pg[k][e] = fmaf(w, gv[e], pg[k][e]);
      }
    }
#pragma unroll
    for (int k = 0; k < M; ++k) {
      if (k >= m || !p.live) continue;
      const int64_t c = k * D + p.d0;
      float fac[8], xh[8], w[8], b[8], sc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) fac[e] = 1.f;
      if (a.drop.on) {
        keep8(a.drop, key, static_cast<uint64_t>(t * E + c), fac);
#pragma unroll
        for (int e = 0; e < 8; ++e) pg[k][e] = fac[e] != 0.f ? pg[k][e] * fac[e] : 0.f;
      }
      fr[k].get(xh);
      param8(a.weight, c, true, 1.f, w);
      param8(a.bias, c, true, 0.f, b);
      param8(a.scale, c, true, 1.f, sc);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[e] = (xh[e] - mean) * rstd;
        b[e] = fmaf(xh[e], w[e], b[e]);  // weight xhat + bias
      }
      if (gate) {
        float ga[8], gd[8];
        ar[k].get(ga);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = gate_value(a.gate_act, ga[e]);
          gd[e] = pg[k][e] * sc[e] * b[e] * (a.gate_act == HC_ACT_SIGMOID ? v * (1.f - v) : 1.f);
          pg[k][e] *= v;
          b[e] *= v;
        }
        if (a.grad_gate) put8<T>(static_cast<T*>(a.grad_gate) + t * E + c, gd);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[k][e] = fac[e] != 0.f ? sc[e] * b[e] * fac[e] : 0.f;
        A[k][e] = fmaf(pg[k][e], xh[e], A[k][e]);
        B[k][e] += pg[k][e];
        pg[k][e] *= sc[e] * w[e];  // q
        s[0] = fmaf(pg[k][e], xh[e], s[0]);
        s[1] += pg[k][e];
      }
    }
    fold_to<2>(s, p.lane, red[buf][p.slot()]);
    p.sync();
    flush(last, buf ^ 1);
    if (a.grad_f && p.live) {
      float c1 = 0.f, c2 = 0.f;
      for (int w = 0; w < p.W; ++w) {
        c1 += red[buf][p.slot0() + w][0];
        c2 += red[buf][p.slot0() + w][1];
      }
      c1 /= static_cast<float>(E);
      c2 = a.norm == HC_NORM_LAYER ? c2 / static_cast<float>(E) : 0.f;
#pragma unroll
      for (int k = 0; k < M; ++k) {
        if (k >= m) break;
        if (a.norm != HC_NORM_NONE) {  // without a norm f's value plays no part, be it a NaN
          float xh[8];
          fr[k].get(xh);
#pragma unroll
          for (int e = 0; e < 8; ++e) pg[k][e] = rstd * (pg[k][e] - c2 - (xh[e] - mean) * rstd * c1);
        }
        put8<T>(static_cast<T*>(a.grad_f) + t * E + k * D + p.d0, pg[k]);
      }
    }
    // grad_x = Heff^T g; g x^T, g z^T
    float xv[N][8], gx[N][8] = {}, acc[GB], accW[N * M];
#pragma unroll
    for (int j = 0; j < N; ++j) xr[j].get(xv[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float gv[8];
      gr[i].get(gv);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float r = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) r = fmaf(gv[e], xv[j][e], r);
        acc[(i * N + j) % GB] = r;
        if (i < n && j < n) {
          const float h = sH[buf][p.group][i * N + j];
#pragma unroll
          for (int e = 0; e < 8; ++e) gx[j][e] = fmaf(h, gv[e], gx[j][e]);
        }
      }
#pragma unroll
      for (int k = 0; k < M; ++k) {
        float r = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) r = fmaf(gv[e], z[k][e], r);
        accW[i * M + k] = r;
      }
      if ((i + 1) * N % GB == 0) fold_to<GB>(acc, p.lane, &gram[buf][p.slot()][(i + 1) * N - GB]);
    }
    fold_to<N * M>(accW, p.lane, &gram[buf][p.slot()][N * N]);
    if (a.grad_x && p.live) {
      T* dst = static_cast<T*>(a.grad_x) + t * n * D + p.d0;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) put8<T>(dst + j * D, gx[j]);
    }
    last = t;
  }
  p.sync();
  flush(last, buf ^ 1);
  store_param_sums<M>(a, p, A, B);
}

// ------------------------------------------------------------------- host
using NormKernel = void (*)(NormArgs, int);

template <typename T, bool WRITE, int N, int M> NormKernel norm_kernel(bool bwd) {
  if constexpr (WRITE)
    return bwd ? write_norm_bwd_kernel<T, N, M> : write_norm_fwd_kernel<T, N, M>;
  else
    return bwd ? read_norm_bwd_kernel<T, N, M> : read_norm_fwd_kernel<T, N, M>;
}

// The kernel for n streams and m blocks: the next larger of 1, 2, 4, 8 and of
// 1, 2, 4 (rows past n and m are neither read nor written); nullptr for more
// blocks than streams, which the element kernels take.
template <typename T, bool WRITE> NormKernel norm_kernel_for(bool bwd, int n, int m) {
  if (n == 1) return m == 1 ? norm_kernel<T, WRITE, 1, 1>(bwd) : nullptr;
  if (n == 2) return m == 1 ? norm_kernel<T, WRITE, 2, 1>(bwd) : m == 2 ? norm_kernel<T, WRITE, 2, 2>(bwd) : nullptr;
  if (n <= 4)
    return m == 1   ? norm_kernel<T, WRITE, 4, 1>(bwd)
           : m == 2 ? norm_kernel<T, WRITE, 4, 2>(bwd)
                    : norm_kernel<T, WRITE, 4, 4>(bwd);
  return m == 1   ? norm_kernel<T, WRITE, 8, 1>(bwd)
         : m == 2 ? norm_kernel<T, WRITE, 8, 2>(bwd)
                  : norm_kernel<T, WRITE, 8, 4>(bwd);
}

// CTAs that fit on the device at once.
inline int norm_resident(NormKernel k, int threads) {
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, threads, 0) != cudaSuccess || per_sm < 1) {
    cudaGetLastError();
    per_sm = 1;
  }
  return per_sm * sm_count();
}

template <typename T, bool WRITE>
int norm_launch(bool bwd, NormGeometry& geo, const NormArgs& a, cudaStream_t s) {
  const NormKernel k = geo.warps > 0 ? norm_kernel_for<T, WRITE>(bwd, a.n, a.m) : nullptr;
  if (!k) return norm_launch_elem<T>(WRITE, bwd, geo, a, s);
  const int groups = geo.warps == 1 ? kSmallGroups : 1, threads = 32 * geo.warps * groups;
  const int64_t want = (a.T + groups - 1) / groups;
  const int most = norm_resident(k, threads);
  geo.grid = static_cast<int>(want < most ? want : most);
  geo.rows = geo.grid * groups;
  k<<<geo.grid, threads, 0, s>>>(a, geo.warps);
  return launch_status();
}

}  // namespace hc

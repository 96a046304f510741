// block_elem.cuh — the norm kernels element by element: any n <= 8, m <= 4, D
// and alignment, one CTA a token (grid-strided). Every pass reads the token
// again (from L2 after the first), so these are for the shapes that the
// 8-column kernels (block_norm.cuh) do not take: tokens too wide for a CTA.
#pragma once

#include "block.cuh"

namespace hc {

constexpr int kElemThreads = 256;

// Sum over the CTA, the same in every thread. `red` holds a float a warp.
__device__ __forceinline__ float cta_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  __syncthreads();  // the last sum has been read
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) s += red[w];
  return s;
}

__device__ __forceinline__ float gate_value(int act, float a) {
  return act == HC_ACT_SIGMOID ? 1.f / (1.f + __expf(-a)) : a;
}

// H + (v - H v) v^T: the projected mix as one n x n matrix (element i, j).
__device__ __forceinline__ float mix_entry(const float* H, const float* v, int n, int i, int j) {
  const float h = H[i * n + j];
  if (!v) return h;
  float c = v[i];
  for (int k = 0; k < n; ++k) c -= H[i * n + k] * v[k];
  return h + c * v[j];
}

// grad_H and grad_v of one token from G = dL/d(H + (v - H v) v^T) in shared
// memory; run by the first n * n (grad_H) and n (grad_v) threads of a group.
__device__ __forceinline__ void mix_grads(const float* G, const float* H, const float* v, int n, int tid,
                                          float* grad_H, float* grad_v) {
  if (tid < n * n && grad_H) {
    const int i = tid / n, k = tid % n;
    float r = G[tid];
    if (v) {
      float dq = 0.f;
      for (int j = 0; j < n; ++j) dq += G[i * n + j] * v[j];
      r -= dq * v[k];
    }
    grad_H[tid] = r;
  }
  if (tid < n && grad_v) {
    float r = 0.f;
    for (int i = 0; i < n; ++i) {
      float q = v[i], dq = 0.f;
      for (int j = 0; j < n; ++j) {
        q -= H[i * n + j] * v[j];
        dq += G[i * n + j] * v[j];
      }
      r += q * G[i * n + tid] + (i == tid ? dq : 0.f) - H[i * n + tid] * dq;
    }
    grad_v[tid] = r;
  }
}

// ------------------------------------------------------------------- read
template <typename T>
__global__ void __launch_bounds__(kElemThreads) read_norm_fwd_elem(NormArgs a) {
  __shared__ float red[kElemThreads / 32], sR[kBlockMaxM * kBlockMaxN];
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + t * n * D;
    T* y = static_cast<T*>(a.out) + t * E;
    __syncthreads();
    if (threadIdx.x < m * n) sR[threadIdx.x] = a.R[t * m * n + threadIdx.x];
    __syncthreads();
    auto u = [&](int k, int64_t d) {
      float s = 0.f;
      for (int j = 0; j < n; ++j) s += sR[k * n + j] * Elem<T>::to_f(x[j * D + d]);
      return s;
    };
    float mean = 0.f, s = 0.f;
    if (a.norm == HC_NORM_LAYER) {
      for (int k = 0; k < m; ++k)
        for (int64_t d = threadIdx.x; d < D; d += blockDim.x) s += u(k, d);
      mean = cta_sum(s, red) / static_cast<float>(E);
    }
    s = 0.f;
    for (int k = 0; k < m; ++k)
      for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
        const float e = u(k, d) - mean;
        s += e * e;
      }
    const float rstd = 1.f / sqrtf(cta_sum(s, red) / static_cast<float>(E) + a.eps);
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * t] = mean;
      a.stats[2 * t + 1] = rstd;
    }
    for (int k = 0; k < m; ++k)
      for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
        const int64_t c = k * D + d;
        float r = (u(k, d) - mean) * rstd;
        if (a.weight) r *= a.weight[c];
        if (a.bias) r += a.bias[c];
        y[c] = Elem<T>::from_f(r);
      }
  }
}

template <typename T>
__global__ void __launch_bounds__(kElemThreads) read_norm_bwd_elem(NormArgs a) {
  __shared__ float red[kElemThreads / 32], sR[kBlockMaxM * kBlockMaxN];
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  bool first = true;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + t * n * D;
    const T* g = static_cast<const T*>(a.g) + t * E;
    T* gx = a.grad_x ? static_cast<T*>(a.grad_x) + t * n * D : nullptr;
    __syncthreads();
    if (threadIdx.x < m * n) sR[threadIdx.x] = a.R[t * m * n + threadIdx.x];
    __syncthreads();
    const float mean = a.stats[2 * t], rstd = a.stats[2 * t + 1];
    auto xhat = [&](int k, int64_t d) {
      float s = 0.f;
      for (int j = 0; j < n; ++j) s += sR[k * n + j] * Elem<T>::to_f(x[j * D + d]);
      return (s - mean) * rstd;
    };
    auto q = [&](int64_t c) { return Elem<T>::to_f(g[c]) * (a.weight ? a.weight[c] : 1.f); };
    float s1 = 0.f, s2 = 0.f;
    for (int k = 0; k < m; ++k)
      for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
        const float qc = q(k * D + d);
        s1 += qc * xhat(k, d);
        s2 += qc;
      }
    const float c1 = cta_sum(s1, red) / static_cast<float>(E);
    const float c2 = a.norm == HC_NORM_LAYER ? cta_sum(s2, red) / static_cast<float>(E) : 0.f;
    float acc[kBlockMaxM][kBlockMaxN] = {};
    for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
      float xv[kBlockMaxN], gv[kBlockMaxN] = {};
#pragma unroll
      for (int j = 0; j < kBlockMaxN; ++j) xv[j] = j < n ? Elem<T>::to_f(x[j * D + d]) : 0.f;
#pragma unroll
      for (int k = 0; k < kBlockMaxM; ++k) {
        if (k >= m) break;
        const int64_t c = k * D + d;
        const float xh = xhat(k, d);
        const float du = rstd * (q(c) - c2 - xh * c1);
#pragma unroll
        for (int j = 0; j < kBlockMaxN; ++j) {
          if (j >= n) break;
          acc[k][j] += du * xv[j];
          gv[j] += sR[k * n + j] * du;
        }
        if (a.partial) {  // this CTA's own row, a column a thread
          float* p = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * E + c;
          const float go = Elem<T>::to_f(g[c]);
          p[0] = (first ? 0.f : p[0]) + go * xh;
          p[E] = (first ? 0.f : p[E]) + go;
        }
      }
      if (gx)
#pragma unroll
        for (int j = 0; j < kBlockMaxN; ++j)
          if (j < n) gx[j * D + d] = Elem<T>::from_f(gv[j]);
    }
    first = false;
    if (a.grad_R)
#pragma unroll
      for (int k = 0; k < kBlockMaxM; ++k)
#pragma unroll
        for (int j = 0; j < kBlockMaxN; ++j)
          if (k < m && j < n) {
            const float r = cta_sum(acc[k][j], red);
            if (threadIdx.x == 0) a.grad_R[t * m * n + k * n + j] = r;
          }
  }
}

// -------------------------------------------------------------- mix-write
// Statistics of f's token: mean and 1 / root, as the norm kind has them.
template <typename T>
__device__ __forceinline__ void elem_stats(const T* f, int64_t E, int norm, float eps, float* red, float& mean,
                                           float& rstd) {
  mean = 0.f;
  rstd = 1.f;
  if (norm == HC_NORM_NONE) return;
  float s = 0.f;
  if (norm == HC_NORM_LAYER) {
    for (int64_t c = threadIdx.x; c < E; c += blockDim.x) s += Elem<T>::to_f(f[c]);
    mean = cta_sum(s, red) / static_cast<float>(E);
    s = 0.f;
  }
  for (int64_t c = threadIdx.x; c < E; c += blockDim.x) {
    const float e = Elem<T>::to_f(f[c]) - mean;
    s += e * e;
  }
  rstd = 1.f / sqrtf(cta_sum(s, red) / static_cast<float>(E) + eps);
}

template <typename T>
__global__ void __launch_bounds__(kElemThreads) write_norm_fwd_elem(NormArgs a) {
  __shared__ float red[kElemThreads / 32], sH[kBlockMaxN * kBlockMaxN], sW[kBlockMaxN * kBlockMaxM];
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + t * n * D;
    const T* f = static_cast<const T*>(a.f) + t * E;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + t * E : nullptr;
    T* out = static_cast<T*>(a.out) + t * n * D;
    __syncthreads();
    if (threadIdx.x < n * n)
      sH[threadIdx.x] = mix_entry(a.H + t * n * n, a.v ? a.v + t * n : nullptr, n, threadIdx.x / n, threadIdx.x % n);
    if (threadIdx.x < n * m) sW[threadIdx.x] = a.W[t * n * m + threadIdx.x];
    __syncthreads();
    float mean, rstd;
    elem_stats(f, E, a.norm, a.eps, red, mean, rstd);
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * t] = mean;
      a.stats[2 * t + 1] = rstd;
    }
    for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
      float xv[kBlockMaxN], z[kBlockMaxM];
#pragma unroll
      for (int j = 0; j < kBlockMaxN; ++j) xv[j] = j < n ? Elem<T>::to_f(x[j * D + d]) : 0.f;
#pragma unroll
      for (int k = 0; k < kBlockMaxM; ++k) {
        z[k] = 0.f;
        if (k >= m) continue;
        const int64_t c = k * D + d;
        float r = (Elem<T>::to_f(f[c]) - mean) * rstd;
        if (a.weight) r *= a.weight[c];
        if (a.bias) r += a.bias[c];
        if (gate) r *= gate_value(a.gate_act, Elem<T>::to_f(gate[c]));
        if (a.scale) r *= a.scale[c];
        if (a.drop.on) r = drop_value(a.drop, philox_word(key, static_cast<uint64_t>(t * E + c)), r);
        z[k] = r;
      }
      for (int i = 0; i < n; ++i) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < kBlockMaxN; ++j)
          if (j < n) s += sH[i * n + j] * xv[j];
#pragma unroll
        for (int k = 0; k < kBlockMaxM; ++k)
          if (k < m) s += sW[i * m + k] * z[k];
        out[i * D + d] = Elem<T>::from_f(s);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kElemThreads) write_norm_bwd_elem(NormArgs a) {
  __shared__ float red[kElemThreads / 32], sH[kBlockMaxN * kBlockMaxN], sW[kBlockMaxN * kBlockMaxM],
      sG[kBlockMaxN * kBlockMaxN];
  const int n = a.n, m = a.m;
  const int64_t D = a.D, E = D * m;
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  bool first = true;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + t * n * D;
    const T* g = static_cast<const T*>(a.g) + t * n * D;
    const T* f = static_cast<const T*>(a.f) + t * E;
    const T* gate = a.gate ? static_cast<const T*>(a.gate) + t * E : nullptr;
    const float* H = a.H + t * n * n;
    const float* v = a.v ? a.v + t * n : nullptr;
    __syncthreads();
    if (threadIdx.x < n * n) sH[threadIdx.x] = mix_entry(H, v, n, threadIdx.x / n, threadIdx.x % n);
    if (threadIdx.x < n * m) sW[threadIdx.x] = a.W[t * n * m + threadIdx.x];
    __syncthreads();
    const float mean = a.norm == HC_NORM_NONE ? 0.f : a.stats[2 * t];
    const float rstd = a.norm == HC_NORM_NONE ? 1.f : a.stats[2 * t + 1];
    // dz after dropout's backward, and dropout's factor
    auto dz = [&](int k, int64_t d, float& factor) {
      float s = 0.f;
      for (int i = 0; i < n; ++i) s += sW[i * m + k] * Elem<T>::to_f(g[i * D + d]);
      factor = 1.f;
      if (a.drop.on) {
        const uint32_t w = philox_word(key, static_cast<uint64_t>(t * E + k * D + d));
        factor = w > a.drop.below ? a.drop.scale : 0.f;
        return factor != 0.f ? s * factor : 0.f;
      }
      return s;
    };
    auto inner = [&](int64_t c) {  // d z / d xhat without dropout
      float r = a.weight ? a.weight[c] : 1.f;
      if (a.scale) r *= a.scale[c];
      if (gate) r *= gate_value(a.gate_act, Elem<T>::to_f(gate[c]));
      return r;
    };
    float c1 = 0.f, c2 = 0.f;
    if (a.norm != HC_NORM_NONE) {
      float s1 = 0.f, s2 = 0.f, fac;
      for (int k = 0; k < m; ++k)
        for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
          const int64_t c = k * D + d;
          const float q = dz(k, d, fac) * inner(c);
          s1 += q * (Elem<T>::to_f(f[c]) - mean) * rstd;
          s2 += q;
        }
      c1 = cta_sum(s1, red) / static_cast<float>(E);
      if (a.norm == HC_NORM_LAYER) c2 = cta_sum(s2, red) / static_cast<float>(E);
    }
    float accH[kBlockMaxN][kBlockMaxN] = {}, accW[kBlockMaxN][kBlockMaxM] = {};
    for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
      float gv[kBlockMaxN], xv[kBlockMaxN];
#pragma unroll
      for (int j = 0; j < kBlockMaxN; ++j) {
        gv[j] = j < n ? Elem<T>::to_f(g[j * D + d]) : 0.f;
        xv[j] = j < n ? Elem<T>::to_f(x[j * D + d]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kBlockMaxN; ++i)
#pragma unroll
        for (int j = 0; j < kBlockMaxN; ++j) accH[i][j] += gv[i] * xv[j];
#pragma unroll
      for (int k = 0; k < kBlockMaxM; ++k) {
        if (k >= m) continue;
        const int64_t c = k * D + d;
        float fac;
        const float p = dz(k, d, fac);
        const float xh = (Elem<T>::to_f(f[c]) - mean) * rstd;
        const float w = a.weight ? a.weight[c] : 1.f, sc = a.scale ? a.scale[c] : 1.f;
        const float b = xh * w + (a.bias ? a.bias[c] : 0.f);
        const float gp = gate ? Elem<T>::to_f(gate[c]) : 1.f;
        const float ga = gate ? gate_value(a.gate_act, gp) : 1.f;
        const float z = fac != 0.f ? sc * ga * b * fac : 0.f;
#pragma unroll
        for (int i = 0; i < kBlockMaxN; ++i) accW[i][k] += gv[i] * z;
        const float pg = p * ga;
        if (a.grad_f) {
          const float q = pg * sc * w;  // without a norm f's value plays no part, be it a NaN
          static_cast<T*>(a.grad_f)[t * E + c] =
              Elem<T>::from_f(a.norm == HC_NORM_NONE ? q : rstd * (q - c2 - xh * c1));
        }
        if (a.grad_gate)
          static_cast<T*>(a.grad_gate)[t * E + c] =
              Elem<T>::from_f(p * sc * b * (a.gate_act == HC_ACT_SIGMOID ? ga * (1.f - ga) : 1.f));
        if (a.partial) {
          float* r = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * E + c;
          r[0] = (first ? 0.f : r[0]) + pg * xh;
          r[E] = (first ? 0.f : r[E]) + pg;
        }
      }
      if (a.grad_x)
        for (int j = 0; j < n; ++j) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < kBlockMaxN; ++i)
            if (i < n) s += sH[i * n + j] * gv[i];
          static_cast<T*>(a.grad_x)[(t * n + j) * D + d] = Elem<T>::from_f(s);
        }
    }
    first = false;
    if (a.grad_H || a.grad_v) {
#pragma unroll
      for (int i = 0; i < kBlockMaxN; ++i)
#pragma unroll
        for (int j = 0; j < kBlockMaxN; ++j)
          if (i < n && j < n) {
            const float r = cta_sum(accH[i][j], red);
            if (threadIdx.x == 0) sG[i * n + j] = r;
          }
      __syncthreads();
      mix_grads(sG, H, v, n, threadIdx.x, a.grad_H ? a.grad_H + t * n * n : nullptr,
                a.grad_v ? a.grad_v + t * n : nullptr);
    }
    if (a.grad_W)
#pragma unroll
      for (int i = 0; i < kBlockMaxN; ++i)
#pragma unroll
        for (int k = 0; k < kBlockMaxM; ++k)
          if (i < n && k < m) {
            const float r = cta_sum(accW[i][k], red);
            if (threadIdx.x == 0) a.grad_W[(t * n + i) * m + k] = r;
          }
  }
}

template <typename T>
int norm_launch_elem(bool write, bool bwd, NormGeometry& geo, const NormArgs& a, cudaStream_t s) {
  const int64_t most = 4 * static_cast<int64_t>(sm_count());
  geo.grid = geo.rows = static_cast<int>(a.T < most ? a.T : most);
  if (write)
    (bwd ? write_norm_bwd_elem<T> : write_norm_fwd_elem<T>)<<<geo.grid, kElemThreads, 0, s>>>(a);
  else
    (bwd ? read_norm_bwd_elem<T> : read_norm_fwd_elem<T>)<<<geo.grid, kElemThreads, 0, s>>>(a);
  return launch_status();
}

}  // namespace hc

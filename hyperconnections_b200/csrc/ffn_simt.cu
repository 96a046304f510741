// ffn_simt.cu — the gated feed-forward's float32 products on the FMA units (the
// tensor cores have no float32 inputs): any size and order.
//
// 256 threads make a 64 x 64 tile of the result, 4 x 4 values a thread, over
// stages of 16 steps of the sum in two shared-memory buffers; a thread's loads
// are a pointer and constant steps from it. Three or four CTAs an SM hide each
// other's waits (0.75 instructions a cycle; 128 x 128 tiles of 8 x 8 values, one
// or two CTAs an SM, ran at 0.58 and took 12-18% more time at 4096 x 1024 x
// 2048, and pairs of float32 in one instruction changed nothing). Products with
// few tiles split their sum over CTAs, whose parts one more kernel adds in
// order.
#include "ffn.cuh"

namespace hc {
namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256, kPitch = kTile + 4;

// kTile rows of an operand, 16 steps at a time, neighbouring threads along its
// unit stride. Rows and steps past the operand's end count as 0.
template <typename T> struct Loader {
  static constexpr int kLoads = kTile * kDepth / kThreads;
  const T* p;
  int64_t step, advance;  // from one of a thread's loads to the next; from stage to stage
  uint32_t rows;          // bit i: the row of load i exists
  int k, k_step;          // of load 0, and from load to load
  int at, at_step;        // place in the [step][row] buffer
  __device__ __forceinline__ Loader(const FfnOperand& o, int64_t row0, int64_t k0) {
    const bool along = o.k_stride == 1;  // else along the rows
    const int row = along ? threadIdx.x / kDepth : threadIdx.x % kTile;
    const int row_step = along ? kThreads / kDepth : 0;
    k = along ? threadIdx.x % kDepth : threadIdx.x / kTile;
    k_step = along ? 0 : kThreads / kTile;
    p = static_cast<const T*>(o.p) + (row0 + row) * o.row_stride + (k0 + k) * o.k_stride;
    step = row_step * o.row_stride + k_step * o.k_stride;
    advance = kDepth * o.k_stride;
    at = k * kPitch + row;
    at_step = k_step * kPitch + row_step;
    rows = 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) rows |= (row0 + row + i * row_step < o.rows ? 1u : 0u) << i;
  }
  __device__ __forceinline__ void load(int64_t left, float (&r)[kLoads]) {  // `left` steps of the sum from this stage on
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      r[i] = (rows >> i & 1u) && k + i * k_step < left ? Elem<T>::to_f(__ldg(p + i * step)) : 0.f;
    p += advance;
  }
  __device__ __forceinline__ void put(const float (&r)[kLoads], float* buffer) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) buffer[at + i * at_step] = r[i];
  }
};

template <typename T, int EPI>
__global__ void __launch_bounds__(kThreads) ffn_simt_kernel(const __grid_constant__ FfnProduct p, float* parts, int splits) {
  constexpr int NB = EPI == kGlu ? 2 : 1, V = kTile / 16;
  __shared__ __align__(16) float sA[2][kDepth * kPitch], sB[2][NB][kDepth * kPitch];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
  float acc[NB][V][V] = {};
  // this CTA's stages of all terms' sums
  const int64_t per_term = (p.K + kDepth - 1) / kDepth, stages = per_term * p.terms;
  const int64_t s0 = stages * blockIdx.z / splits, s1 = stages * (blockIdx.z + 1) / splits;
  for (int term = 0; term < p.terms; ++term) {
    const int64_t first = s0 > term * per_term ? s0 - term * per_term : 0;
    const int64_t last = s1 - term * per_term < per_term ? s1 - term * per_term : per_term;
    if (first >= last) continue;
    Loader<T> la(p.A[term], m0, first * kDepth);
    Loader<T> lb(p.B[term], n0, first * kDepth), lb2(p.B[NB == 2 ? 1 : term], n0, first * kDepth);
    float ra[Loader<T>::kLoads], rb[NB][Loader<T>::kLoads];
    auto load = [&](int64_t st) {
      la.load(p.K - st * kDepth, ra);
      lb.load(p.K - st * kDepth, rb[0]);
      if constexpr (NB == 2) lb2.load(p.K - st * kDepth, rb[NB - 1]);
    };
    auto put = [&](int buf) {
      la.put(ra, sA[buf]);
      lb.put(rb[0], sB[buf][0]);
      if constexpr (NB == 2) lb2.put(rb[NB - 1], sB[buf][NB - 1]);
    };
    load(first);
    put(0);
    __syncthreads();
    int buf = 0;
    for (int64_t st = first; st < last; ++st, buf ^= 1) {
      if (st + 1 < last) load(st + 1);  // the next stage travels while this one is used
#pragma unroll
      for (int k = 0; k < kDepth; ++k) {
        const float4 av = *reinterpret_cast<const float4*>(&sA[buf][k * kPitch + V * ty]);
        const float a[V] = {av.x, av.y, av.z, av.w};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float4 bv = *reinterpret_cast<const float4*>(&sB[buf][b][k * kPitch + V * tx]);
          const float w[V] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
          for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[b][i][j] = fmaf(a[i], w[j], acc[b][i][j]);
        }
      }
      if (st + 1 < last) put(buf ^ 1);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int64_t m = m0 + V * ty + i, n = n0 + V * tx + j;
      if (m >= p.M || n >= p.N) continue;
      const int64_t at = m * p.ldo + n;
      if constexpr (EPI == kStore) {
        if (parts)
          parts[(blockIdx.z * p.M + m) * p.N + n] = acc[0][i][j];
        else
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

}  // namespace

namespace {
template <int EPI> int launch(const FfnProduct& p, float* parts, int splits, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.N + kTile - 1) / kTile), static_cast<unsigned>((p.M + kTile - 1) / kTile), splits);
  ffn_simt_kernel<float, EPI><<<grid, kThreads, 0, s>>>(p, parts, splits);
  return launch_status();
}
}  // namespace

// CTAs that share the sum of one tile: until there are four an SM, each with at
// least 8 stages (128 steps) of its own. (517 x 333 x 887, forward and
// backward: 210 us against 354 without.)
int ffn_simt_splits(int64_t M, int64_t N, int64_t K, int terms) {
  const int64_t tiles = ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile);
  const int64_t by_sms = 4 * sm_count() / tiles, by_depth = (K + kDepth - 1) / kDepth * terms / 8;
  const int64_t s = by_sms < by_depth ? by_sms : by_depth;
  return static_cast<int>(s < 1 ? 1 : s > 32 ? 32 : s);
}

int ffn_simt_launch(const FfnProduct& p, float* parts, cudaStream_t s) {
  if (p.epilogue == kGlu) return launch<kGlu>(p, nullptr, 1, s);
  if (p.epilogue == kGluBwd) return launch<kGluBwd>(p, nullptr, 1, s);
  const int splits = ffn_simt_splits(p.M, p.N, p.K, p.terms);
  if (splits > 1 && !parts) return HC_ERR_SCRATCH;
  if (int rc = launch<kStore>(p, splits > 1 ? parts : nullptr, splits, s)) return rc;
  return splits > 1 ? ffn_add_parts(parts, p.out, p.M * p.N, splits, HC_DTYPE_F32, s) : HC_OK;
}

}  // namespace hc

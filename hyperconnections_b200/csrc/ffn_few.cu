// ffn_few.cu — the gated feed-forward's forward products for a few tokens (at
// most 32), bf16 and fp16: bound by the weights, each read once from HBM.
//
// A CTA (or a cluster of up to 8, each with a slice of the sum) owns 16 rows of
// the weights; its eight warps split the sum further. A lane reads 16 bytes of
// rows l / 4 and l / 4 + 8 straight into registers, which are the A operands of
// mma.m16n8k16 as they lie: the sum's order is free, so lane l % 4 takes eight
// neighbouring elements where the instruction means two pairs, of the weights
// and of x alike. The tokens are the columns of B, eight a product. No shared
// memory, no barrier until the sums meet: the loads of 64 or 128 elements of the
// sum are in flight at once, 8 KB a warp. The tensor-core kernel (ffn_tc.cu)
// has 64 or 8 tiles for such shapes, too few CTAs to draw the bandwidth.
#include <type_traits>

#include "ffn.cuh"
#include "mix_warp.cuh"  // pdl_launch_dependents, pdl_wait_prior_grid

namespace hc {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 16;   // rows of the weights of a CTA
constexpr int kChunk = 32;  // elements of the sum that a warp's 16-byte loads cover
constexpr int kUnroll = 4;  // chunks in flight
// CTAs of an SM. (8 tokens, 2048 x 8192: 22.6 us with four of the down product's,
// 24.7 with its 80 registers and three; two chunks in flight and four CTAs for h
// were slower.)
constexpr int per_sm_of(int mats, int tiles) { return mats == 1 && tiles == 1 ? 4 : 2; }
// CTAs of a cluster at most: 8, or as many as shared memory holds the sums of.
constexpr int most_slices(int mats, int tiles) { return mats * tiles >= 8 ? 4 : 8; }

struct FewArgs {
  const void *x, *w0, *w1;  // x [T, K], row stride ldx; weights [rows, K], row stride ldw
  void *out, *slope_gate, *slope_up;
  int64_t T, rows, N, K, ldx, ldw, ldo;  // results [T, N], N >= rows (zeros behind)
  int act, slices;
};

template <typename T> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A weight's 16 bytes, asked for where it stands: the compiler may not move the
// load down to its use.
__device__ __forceinline__ uint4 weight16(const void* p, bool ok) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (ok)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

// MATS weights (2: w_gate and w_up of the same rows), TILES eights of tokens.
template <typename T, int MATS, int TILES>
__global__ void __launch_bounds__(kThreads, per_sm_of(MATS, TILES)) ffn_few_kernel(const __grid_constant__ FewArgs a) {
  constexpr int kSums = MATS * TILES * 4;  // accumulators of a lane
  __shared__ float sums[kWarps][kSums][32];
  __shared__ float total[most_slices(MATS, TILES)][kSums][32];  // the leader's: every slice's sums
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, q = lane & 3;
  const int slice = blockIdx.x % a.slices;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / a.slices) * kRows;
  float acc[MATS][TILES][4] = {};
  const bool cluster = a.slices > 1;  // whose first CTA has to run before the others write to it
  if (cluster) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // this warp's chunks of the sum: every (slices * 8)th run of kUnroll chunks
  const int64_t chunks = (a.K + kChunk - 1) / kChunk, runs = (chunks + kUnroll - 1) / kUnroll;
  const T* w[MATS];
  w[0] = static_cast<const T*>(a.w0);
  if constexpr (MATS == 2) w[1] = static_cast<const T*>(a.w1);
  const bool live0 = row0 + r < a.rows, live1 = row0 + r + 8 < a.rows;
  if (MATS == 2) pdl_launch_dependents();  // the down product may load its first weights meanwhile
  bool first = MATS == 1;
  for (int64_t run = slice * kWarps + warp; run < runs; run += a.slices * kWarps) {
    uint4 wa[kUnroll][MATS][2], xb[kUnroll][TILES];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t k = (run * kUnroll + u) * kChunk + q * 8;  // rows hold whole eights, zeros behind K
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        const T* p = w[m] + (row0 + r) * a.ldw + k;
        wa[u][m][0] = weight16(p, k < a.K && live0);
        wa[u][m][1] = weight16(p + 8 * a.ldw, k < a.K && live1);
      }
    }
    if (first) {  // h comes from the kernel before
      pdl_wait_prior_grid();
      first = false;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t k = (run * kUnroll + u) * kChunk + q * 8;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        xb[u][t] = make_uint4(0u, 0u, 0u, 0u);
        if (k < a.K && 8 * t + r < a.T)
          xb[u][t] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (8 * t + r) * a.ldx + k);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        const uint32_t lo[4] = {wa[u][m][0].x, wa[u][m][1].x, wa[u][m][0].y, wa[u][m][1].y};
        const uint32_t hi[4] = {wa[u][m][0].z, wa[u][m][1].z, wa[u][m][0].w, wa[u][m][1].w};
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          mma<T>(acc[m][t], lo, xb[u][t].x, xb[u][t].y);
          mma<T>(acc[m][t], hi, xb[u][t].z, xb[u][t].w);
        }
      }
  }

  if (first) pdl_wait_prior_grid();  // a warp without a run

  // the warps' sums, then the slices'
#pragma unroll
  for (int i = 0; i < kSums; ++i) sums[warp][i][lane] = acc[i / (TILES * 4)][i / 4 % TILES][i % 4];
  __syncthreads();
  if (cluster) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = threadIdx.x; i < kSums * 32; i += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) s += (&sums[k][0][0])[i];
    if (!cluster) {
      (&total[0][0][0])[i] = s;
    } else {  // to the cluster's first CTA
      uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(&total[slice][0][0] + i));
      asm volatile("mapa.shared::cluster.u32 %0, %0, 0;\n\tst.shared::cluster.f32 [%0], %1;" : "+r"(dst) : "f"(s) : "memory");
    }
  }
  if (!cluster) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (slice != 0) return;
  }

  // row l / 4 (+ 8 for values 2, 3) and token 2 (l % 4) (+ 1 for odd values) of each tile
  for (int i = threadIdx.x; i < TILES * 4 * 32; i += kThreads) {
    const int l = i & 31, v = i >> 5 & 3, t = i >> 7;
    const int64_t row = row0 + (l >> 2) + (v & 2 ? 8 : 0), tok = 8 * t + 2 * (l & 3) + (v & 1);
    if (row >= a.N || tok >= a.T) continue;
    float s[MATS] = {};
#pragma unroll
    for (int m = 0; m < MATS; ++m)
      for (int k = 0; k < a.slices; ++k) s[m] += total[k][(m * TILES + t) * 4 + v][l];
    const int64_t at = tok * a.ldo + row;
    if constexpr (MATS == 2) {
      float val, der;
      ffn_act(a.act, s[0], val, der);
      if (row >= a.rows) val = der = s[MATS - 1] = 0.f;  // read by the down product: 0 also where an infinite x made 0 x inf
      static_cast<T*>(a.out)[at] = Elem<T>::from_f(val * s[MATS - 1]);
      if (a.slope_gate) {
        static_cast<T*>(a.slope_gate)[at] = Elem<T>::from_f(der * s[MATS - 1]);
        static_cast<T*>(a.slope_up)[at] = Elem<T>::from_f(val);
      }
    } else {
      static_cast<T*>(a.out)[at] = Elem<T>::from_f(s[0]);
    }
  }
}

using Kernel = void (*)(FewArgs);
template <typename T, int MATS> Kernel kernel_of(int64_t T_) {
  return T_ <= 8 ? ffn_few_kernel<T, MATS, 1> : T_ <= 16 ? ffn_few_kernel<T, MATS, 2> : ffn_few_kernel<T, MATS, 4>;
}

}  // namespace

int ffn_few_launch(const FfnProduct& p, int dtype, cudaStream_t s) {
  const bool glu = p.epilogue == kGlu, bf = dtype == HC_DTYPE_BF16;
  FewArgs a{};
  a.x = p.A[0].p; a.ldx = p.A[0].row_stride; a.T = p.M;
  a.w0 = p.B[0].p; a.w1 = p.B[1].p; a.ldw = p.B[0].row_stride; a.rows = p.B[0].rows;
  a.N = p.N; a.K = p.K; a.ldo = p.ldo;
  a.out = p.out; a.slope_gate = p.slope_gate; a.slope_up = p.slope_up; a.act = p.act;
  const int64_t tiles = (p.N + kRows - 1) / kRows, runs = (p.K + kChunk * kUnroll - 1) / (kChunk * kUnroll);
  // slices of the sum until there are three CTAs an SM, none without a run for each of its warps
  a.slices = 1;
  const int most = most_slices(glu ? 2 : 1, p.M <= 8 ? 1 : p.M <= 16 ? 2 : 4);
  while (a.slices < most && tiles * a.slices < 3 * sm_count() && runs >= 2 * a.slices * kWarps) a.slices *= 2;
  const Kernel k = glu ? (bf ? kernel_of<__nv_bfloat16, 2>(p.M) : kernel_of<__half, 2>(p.M))
                       : (bf ? kernel_of<__nv_bfloat16, 1>(p.M) : kernel_of<__half, 1>(p.M));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.slices));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.slices;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  // the down product starts while h is still being made, and waits for it behind its first weights
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = glu ? 1 : 2;
  if (cudaLaunchKernelEx(&cfg, k, a) != cudaSuccess) {
    cudaGetLastError();
    return HC_ERR_LAUNCH;
  }
  return HC_OK;
}

}  // namespace hc

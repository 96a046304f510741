// ffn.cuh — the gated feed-forward's products, described once for every
// kernel that computes them (ffn_capi.cu makes the descriptions).
//
//   forward   [a b] = x [w_gate; w_up]^T  -> h = act(a) * b      (kGlu)
//             y     = h w_down^T                                 (kStore)
//   backward  dh    = g w_down            -> da, db              (kGluBwd)
//             dx    = da w_gate + db w_up                        (kStore, two terms)
//             dw_gate = da^T x, dw_up = db^T x, dw_down = g^T h  (kStore)
#pragma once

#include "common.cuh"

namespace hc {

enum FfnEpilogue { kStore, kGlu, kGluBwd };

// A matrix [rows, K] read as p[row * row_stride + k * k_stride]; one of the two
// strides is 1.
struct FfnOperand {
  const void* p;
  int64_t row_stride, k_stride;
  int64_t rows;  // rows that exist: the others count as 0
};

struct FfnProduct {
  int epilogue;
  int terms;            // 1, or 2 products summed into one result
  FfnOperand A[2];      // by term
  FfnOperand B[2];      // by term; kGlu: w_gate and w_up of its one term
  int64_t M, N, K;      // result [M, N], summed over K (for each term)
  void* out;            // kStore: the result; kGlu: h; kGluBwd: da
  void* out2;           // kGluBwd: db
  void *slope_gate, *slope_up;  // act'(a) b and act(a); kGlu: written (nullable); kGluBwd: read
  int64_t ldo;          // row stride of the above
  int act;
};

// act(a) and its derivative. GELU's tanh form, 0.5 a (1 + tanh u) with u = c (a +
// 0.044715 a^3) and c = sqrt(2 / pi), is a / (1 + e^-2u): no sum cancels on its
// left tail, where 1 + tanh loses every digit (a tenth of the value at a = -4.5).
__device__ __forceinline__ void ffn_act(int act, float a, float& val, float& der) {
  if (act == HC_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-a));
    val = a * s;
    der = s + val * (1.f - s);
  } else {
    const float c2 = 2.f * 0.7978845608028654f, a2 = fminf(a * a, 1e4f);  // past |a| = 100 all is 0 or a: a^2 need not grow
    const float s = 1.f / (1.f + expf(-c2 * a * (1.f + 0.044715f * a2)));
    val = a * s;
    der = s + val * (1.f - s) * (c2 * (1.f + 3.f * 0.044715f * a2));
  }
}

// A launch whose CTAs come up while the last ones of the launch before it leave:
// the kernel touches no memory before pdl_wait_prior_grid(), and lets the next
// launch in with pdl_launch_dependents().
template <typename... Args>
int ffn_launch(void (*kernel)(Args...), dim3 grid, int threads, int smem, cudaStream_t s, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return HC_OK;
  cudaGetLastError();
  return HC_ERR_LAUNCH;
}

// Up to kFfnMaxJobs products in one launch, which then share K, one term, the
// order of their operands and the epilogue kStore. `parts`: the sum of splits *
// M * N floats where the sum is split, more than one (kStore only), else
// nullptr.
constexpr int kFfnMaxJobs = 3;

// out[i] = the sum of `splits` float32 parts, `count` apart, in order
// (ffn_tc.cu); for up to kFfnMaxJobs results.
struct FfnParts {
  const float* parts;
  void* out;
  int64_t count;
  bool fours;  // (set by ffn_add_parts) four at a time
};
int ffn_add_parts(const FfnParts* jobs, int count, int splits, int dtype, cudaStream_t s);

// float32 (ffn_simt.cu); few: every job has few rows.
bool ffn_simt_few(int64_t M);
int64_t ffn_simt_tiles(int64_t M, int64_t N, bool few);
int ffn_simt_splits(int64_t tiles, int64_t K, int terms, bool few);
int ffn_simt_launch(const FfnProduct* p, int jobs, float* parts, cudaStream_t s);

// bf16 and fp16 (ffn_tc.cu): operands 16-byte aligned with strides of whole 16
// bytes.
struct FfnSize {
  int64_t M, N;
};
struct FfnTcPlan {
  int tile_n, splits;
};
FfnTcPlan ffn_tc_plan(const FfnSize* sizes, int jobs, int64_t K, int terms);
int ffn_tc_launch(const FfnProduct* p, int jobs, int dtype, float* parts, cudaStream_t s);

// bf16 and fp16, the forward's products for at most kFewTokens rows of A
// (ffn_few.cu): operands aligned as above.
constexpr int64_t kFewTokens = 32;
int ffn_few_launch(const FfnProduct& p, int dtype, cudaStream_t s);

}  // namespace hc

// block_capi.cu — C entry points of the norm kernels around a layer's block
// and of dropout (see hcops.h). Host-side checks come first; then the kernels
// of the stream dtype, and for the [m D] parameters' gradients one more launch
// that adds the CTAs' sums.
#include <math.h>

#include "block_norm.cuh"

namespace hc {
namespace {

constexpr int64_t kMaxD = int64_t(1) << 24;
constexpr int64_t kMaxTokens = (int64_t(1) << 31) - 1;

int check_shape(int64_t T, int n, int m, int64_t D, int sdt) {
  if (T < 0 || T > kMaxTokens || D < 0 || D > kMaxD) return HC_ERR_BAD_SIZE;
  if (n < 1 || n > kBlockMaxN || m < 1 || m > kBlockMaxM) return HC_ERR_UNSUPPORTED_N;
  if (dtype_size(sdt) == 0) return HC_ERR_DTYPE;
  return HC_OK;
}

bool f32_ok(std::initializer_list<const float*> ps) {
  for (const float* p : ps)
    if (!aligned4(p)) return false;
  return true;
}

// Streams are read by their elements where they are not on wider boundaries.
bool streams_ok(int sdt, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % dtype_size(sdt) != 0) return false;
  return true;
}

bool state_ok(const int64_t* state) { return reinterpret_cast<uintptr_t>(state) % sizeof(int64_t) == 0; }

// Dropout's arguments; false when p is not in [0, 1].
bool drop_args(DropArgs& d, double p, const int64_t* state, int64_t seed, int64_t offset) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  d.state = state;
  d.seed = static_cast<uint64_t>(seed);
  d.offset = static_cast<uint64_t>(offset);
  const uint64_t threshold = static_cast<uint64_t>(floor(p * 4294967296.0));
  d.on = threshold > 0;  // of p < 2^-32 nothing is left
  d.below = static_cast<uint32_t>(threshold - (threshold > 0));
  d.scale = p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.f;
  return true;
}

// The 8-column kernels take rows whose group fits a CTA, those of whole chunks
// on 16-byte boundaries by 16 bytes; the others go element by element. (16,384
// tokens of n = 4, D = 768, bf16, forward and backward: 180 us against 3,222 for
// the mix-write, 90 against 668 for the read.)
NormGeometry geometry(bool write, bool bwd, int n, int m, int64_t D, int esize,
                      std::initializer_list<const void*> ps, const float* stats) {
  if ((reinterpret_cast<uintptr_t>(stats) & 7u) != 0) return NormGeometry{};
  bool aligned = true;
  for (const void* p : ps) aligned = aligned && aligned16(p);
  return norm_geometry(write, bwd, n, m, D, esize, aligned);
}

int launch(int sdt, bool write, bool bwd, NormGeometry& g, const NormArgs& a, cudaStream_t s) {
  switch (sdt) {
    case HC_DTYPE_F32: return write ? write_norm_launch_f32(bwd, g, a, s) : read_norm_launch_f32(bwd, g, a, s);
    case HC_DTYPE_F16: return write ? write_norm_launch_f16(bwd, g, a, s) : read_norm_launch_f16(bwd, g, a, s);
    case HC_DTYPE_BF16: return write ? write_norm_launch_bf16(bwd, g, a, s) : read_norm_launch_bf16(bwd, g, a, s);
  }
  return HC_ERR_DTYPE;
}

// ------------------------------------------------ the [E] parameters' grads
// A = sum over rows of partial[.][0][c], B of partial[.][1][c]: a CTA takes 8
// columns (so that narrow blocks fill the device too) and 128 rows at a time,
// eight loads of each in flight; the lanes' and warps' sums are added in a
// fixed order, so the result does not depend on timing.
constexpr int kParamCols = 8, kParamThreads = 1024, kParamLines = kParamThreads / kParamCols;

__global__ void __launch_bounds__(kParamThreads)
    norm_param_grads_kernel(const float* partial, int rows, int64_t E, const float* weight, const float* bias,
                            const float* scale, float* gw, float* gb, float* gs) {
  __shared__ float sA[kParamThreads / 32][kParamCols], sB[kParamThreads / 32][kParamCols];
  const int col = threadIdx.x % kParamCols, line = threadIdx.x / kParamCols;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kParamCols + col;
  float A = 0.f, B = 0.f;
  constexpr int kBatch = 8;
  for (int r0 = line; r0 < rows; r0 += kBatch * kParamLines) {
    float a[kBatch], b[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = r0 + i * kParamLines;
      const bool ok = c < E && r < rows;
      a[i] = ok ? __ldg(partial + static_cast<int64_t>(r) * 2 * E + c) : 0.f;
      b[i] = ok ? __ldg(partial + static_cast<int64_t>(r) * 2 * E + E + c) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      A += a[i];
      B += b[i];
    }
  }
#pragma unroll
  for (int o = 16; o >= kParamCols; o >>= 1) {
    A += __shfl_xor_sync(kFull, A, o);
    B += __shfl_xor_sync(kFull, B, o);
  }
  if ((threadIdx.x & 31) < kParamCols) {
    sA[threadIdx.x >> 5][col] = A;
    sB[threadIdx.x >> 5][col] = B;
  }
  __syncthreads();
  if (threadIdx.x >= kParamCols || c >= E) return;
  A = B = 0.f;
  for (int i = 0; i < kParamThreads / 32; ++i) {
    A += sA[i][col];
    B += sB[i][col];
  }
  const float sc = scale ? scale[c] : 1.f;
  if (gw) gw[c] = sc * A;
  if (gb) gb[c] = sc * B;
  if (gs) gs[c] = (weight ? weight[c] : 1.f) * A + (bias ? bias[c] : 0.f) * B;
}

}  // namespace

int norm_param_grads(const float* partial, int rows, int64_t E, const float* weight, const float* bias,
                     const float* scale, float* grad_weight, float* grad_bias, float* grad_scale, cudaStream_t s) {
  norm_param_grads_kernel<<<static_cast<unsigned>((E + kParamCols - 1) / kParamCols), kParamThreads, 0, s>>>(
      partial, rows, E, weight, bias, scale, grad_weight, grad_bias, grad_scale);
  return launch_status();
}

}  // namespace hc

using namespace hc;

// Rows for as many groups as an SM can hold threads of, which no kernel's grid
// exceeds.
extern "C" int64_t hc_norm_scratch_words(int64_t T, int n, int m, int64_t D, int stream_dtype) {
  if (check_shape(T, n, m, D, stream_dtype) || T == 0 || D == 0) return 0;
  const int64_t warps = (D + 32 * kColumns - 1) / (32 * kColumns), per_sm = warps < 8 ? 64 / warps : 8;
  const int64_t groups = (T + kSmallGroups - 1) / kSmallGroups * kSmallGroups, most = per_sm * sm_count();
  return (groups < most ? groups : most) * 2 * m * D;
}

extern "C" int hc_read_norm_fwd(const float* R, const void* x, const float* weight, const float* bias, void* y,
                                float* stats, int64_t T, int n, int m, int64_t D, int norm, float eps,
                                int stream_dtype, void* stream) {
  HC_ENTRY("hc_read_norm_fwd");
  if (int rc = check_shape(T, n, m, D, stream_dtype)) return rc;
  if (norm != HC_NORM_RMS && norm != HC_NORM_LAYER) return HC_ERR_BAD_SIZE;
  if (!(eps >= 0.f)) return HC_ERR_BAD_SIZE;
  if (T == 0 || D == 0) return HC_OK;
  if (!R || !x || !y) return HC_ERR_NULL_POINTER;
  if (!f32_ok({R, weight, bias, stats}) || !streams_ok(stream_dtype, {x, y})) return HC_ERR_ALIGNMENT;
  NormArgs a{};
  a.R = R; a.x = x; a.weight = weight; a.bias = bias; a.out = y; a.stats = stats;
  a.T = T; a.D = D; a.n = n; a.m = m; a.norm = norm; a.eps = eps;
  NormGeometry geo = geometry(false, false, n, m, D, dtype_size(stream_dtype),
                              {x, y, weight, bias}, stats);
  return launch(stream_dtype, false, false, geo, a, static_cast<cudaStream_t>(stream));
}

extern "C" int hc_read_norm_bwd(const void* g, const float* R, const void* x, const float* weight, const float* stats,
                                void* grad_x, float* grad_R, float* grad_weight, float* grad_bias, float* scratch,
                                int64_t scratch_words, int64_t T, int n, int m, int64_t D, int norm,
                                int stream_dtype, void* stream) {
  HC_ENTRY("hc_read_norm_bwd");
  if (int rc = check_shape(T, n, m, D, stream_dtype)) return rc;
  if (norm != HC_NORM_RMS && norm != HC_NORM_LAYER) return HC_ERR_BAD_SIZE;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t E = m * D;
  if (T == 0 || D == 0) {  // sums over nothing
    if (!f32_ok({grad_R, grad_weight, grad_bias})) return HC_ERR_ALIGNMENT;
    if (grad_R && T > 0 && cudaMemsetAsync(grad_R, 0, sizeof(float) * T * m * n, s) != cudaSuccess) return HC_ERR_LAUNCH;
    for (float* p : {grad_weight, grad_bias})
      if (p && E > 0 && cudaMemsetAsync(p, 0, sizeof(float) * E, s) != cudaSuccess) return HC_ERR_LAUNCH;
    return HC_OK;
  }
  if (!g || !R || !x || !stats) return HC_ERR_NULL_POINTER;
  if (!f32_ok({R, weight, stats, grad_R, grad_weight, grad_bias, scratch}) || !streams_ok(stream_dtype, {g, x, grad_x}))
    return HC_ERR_ALIGNMENT;
  const bool params = grad_weight || grad_bias;
  if (params && (!scratch || scratch_words < hc_norm_scratch_words(T, n, m, D, stream_dtype))) return HC_ERR_SCRATCH;
  NormArgs a{};
  a.g = g; a.R = R; a.x = x; a.weight = weight; a.stats = const_cast<float*>(stats);
  a.grad_x = grad_x; a.grad_R = grad_R; a.partial = params ? scratch : nullptr;
  a.T = T; a.D = D; a.n = n; a.m = m; a.norm = norm;
  NormGeometry geo = geometry(false, true, n, m, D, dtype_size(stream_dtype),
                              {g, x, grad_x, weight, scratch}, nullptr);
  if (int rc = launch(stream_dtype, false, true, geo, a, s)) return rc;
  return params ? norm_param_grads(scratch, geo.rows, E, weight, nullptr, nullptr, grad_weight, grad_bias, nullptr, s)
                : HC_OK;
}

namespace {
int check_write(int norm, int gate_act, double p) {
  if (norm != HC_NORM_NONE && norm != HC_NORM_RMS && norm != HC_NORM_LAYER) return HC_ERR_BAD_SIZE;
  if (gate_act != HC_ACT_LINEAR && gate_act != HC_ACT_SIGMOID) return HC_ERR_BAD_SIZE;
  return p >= 0.0 && p <= 1.0 ? HC_OK : HC_ERR_BAD_SIZE;
}
}  // namespace

extern "C" int hc_mix_write_norm_fwd(const float* H, const void* x, const float* W, const void* f, const float* v,
                                     const float* weight, const float* bias, const void* gate, const float* scale,
                                     void* out, float* stats, int64_t T, int n, int m, int64_t D, int norm,
                                     int gate_act, float eps, double p, const int64_t* state, int64_t seed,
                                     int64_t offset, int stream_dtype, void* stream) {
  HC_ENTRY("hc_mix_write_norm_fwd");
  if (int rc = check_shape(T, n, m, D, stream_dtype)) return rc;
  if (int rc = check_write(norm, gate_act, p)) return rc;
  if (!(eps >= 0.f)) return HC_ERR_BAD_SIZE;
  if (T == 0 || D == 0) return HC_OK;
  if (!H || !x || !W || !f || !out) return HC_ERR_NULL_POINTER;
  if (!f32_ok({H, W, v, weight, bias, scale, stats}) || !streams_ok(stream_dtype, {x, f, gate, out}) || !state_ok(state))
    return HC_ERR_ALIGNMENT;
  NormArgs a{};
  a.H = H; a.x = x; a.W = W; a.f = f; a.v = v; a.weight = weight; a.bias = bias; a.gate = gate; a.scale = scale;
  a.out = out; a.stats = stats; a.T = T; a.D = D; a.n = n; a.m = m; a.norm = norm; a.gate_act = gate_act; a.eps = eps;
  drop_args(a.drop, p, state, seed, offset);
  NormGeometry geo = geometry(true, false, n, m, D, dtype_size(stream_dtype),
                              {x, f, gate, out, weight, bias, scale}, stats);
  return launch(stream_dtype, true, false, geo, a, static_cast<cudaStream_t>(stream));
}

extern "C" int hc_mix_write_norm_bwd(const void* g, const float* H, const void* x, const float* W, const void* f,
                                     const float* v, const float* weight, const float* bias, const void* gate,
                                     const float* scale, const float* stats, void* grad_x, void* grad_f,
                                     void* grad_gate, float* grad_H, float* grad_W, float* grad_v, float* grad_weight,
                                     float* grad_bias, float* grad_scale, float* scratch, int64_t scratch_words,
                                     int64_t T, int n, int m, int64_t D, int norm, int gate_act, double p,
                                     const int64_t* state, int64_t seed, int64_t offset, int stream_dtype,
                                     void* stream) {
  HC_ENTRY("hc_mix_write_norm_bwd");
  if (int rc = check_shape(T, n, m, D, stream_dtype)) return rc;
  if (int rc = check_write(norm, gate_act, p)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t E = m * D;
  if (!f32_ok({H, W, v, weight, bias, scale, stats, grad_H, grad_W, grad_v, grad_weight, grad_bias, grad_scale, scratch}) ||
      !streams_ok(stream_dtype, {g, x, f, gate, grad_x, grad_f, grad_gate}) || !state_ok(state))
    return HC_ERR_ALIGNMENT;
  if (T == 0 || D == 0) {  // sums over nothing
    const struct { float* p; int64_t words; } zero[] = {{grad_H, T * n * n}, {grad_W, T * n * m}, {grad_v, T * n},
                                                        {grad_weight, E}, {grad_bias, E}, {grad_scale, E}};
    for (const auto& z : zero)
      if (z.p && z.words > 0 && cudaMemsetAsync(z.p, 0, sizeof(float) * z.words, s) != cudaSuccess) return HC_ERR_LAUNCH;
    return HC_OK;
  }
  if (!g || !H || !x || !W || !f || (norm != HC_NORM_NONE && !stats)) return HC_ERR_NULL_POINTER;
  const bool params = grad_weight || grad_bias || grad_scale;
  if (params && (!scratch || scratch_words < hc_norm_scratch_words(T, n, m, D, stream_dtype))) return HC_ERR_SCRATCH;
  NormArgs a{};
  a.g = g; a.H = H; a.x = x; a.W = W; a.f = f; a.v = v; a.weight = weight; a.bias = bias; a.gate = gate;
  a.scale = scale; a.stats = const_cast<float*>(stats); a.grad_x = grad_x; a.grad_f = grad_f;
  a.grad_gate = gate ? grad_gate : nullptr; a.grad_H = grad_H; a.grad_W = grad_W; a.grad_v = v ? grad_v : nullptr;
  a.partial = params ? scratch : nullptr;
  a.T = T; a.D = D; a.n = n; a.m = m; a.norm = norm; a.gate_act = gate_act;
  drop_args(a.drop, p, state, seed, offset);
  NormGeometry geo = geometry(true, true, n, m, D, dtype_size(stream_dtype),
                              {g, x, f, gate, grad_x, grad_f, grad_gate, weight, bias, scale, scratch}, nullptr);
  if (int rc = launch(stream_dtype, true, true, geo, a, s)) return rc;
  return params ? norm_param_grads(scratch, geo.rows, E, weight, bias, scale, grad_weight, grad_bias, grad_scale, s)
                : HC_OK;
}

extern "C" int hc_dropout(const void* x, void* y, int64_t N, double p, const int64_t* state, int64_t seed,
                          int64_t offset, int stream_dtype, void* stream) {
  HC_ENTRY("hc_dropout");
  if (N < 0 || dtype_size(stream_dtype) == 0) return N < 0 ? HC_ERR_BAD_SIZE : HC_ERR_DTYPE;
  DropArgs d{};
  if (!drop_args(d, p, state, seed, offset)) return HC_ERR_BAD_SIZE;
  if (N == 0) return HC_OK;
  if (!x || !y) return HC_ERR_NULL_POINTER;
  if (!streams_ok(stream_dtype, {x, y}) || !state_ok(state)) return HC_ERR_ALIGNMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!d.on) {  // every element is kept, times 1
    if (x == y) return HC_OK;
    return cudaMemcpyAsync(y, x, static_cast<size_t>(N) * dtype_size(stream_dtype), cudaMemcpyDeviceToDevice, s) ==
                   cudaSuccess
               ? HC_OK
               : HC_ERR_LAUNCH;
  }
  switch (stream_dtype) {
    case HC_DTYPE_F32: return dropout_launch_f32(x, y, N, d, s);
    case HC_DTYPE_F16: return dropout_launch_f16(x, y, N, d, s);
    default: return dropout_launch_bf16(x, y, N, d, s);
  }
}

// ffn_capi.cu — C entry points of the gated feed-forward (see hcops.h): host
// checks, then its products one after the other on the caller's stream.
#include "ffn.cuh"

namespace hc {
namespace {

// A CTA's 64 rows in grid.y (at most 65,535) bound the rows of every product.
constexpr int64_t kMaxRows = int64_t(65535) * 64, kMaxWidth = int64_t(1) << 20;

int check(int64_t T, int64_t D, int64_t F, int64_t O, int act, int dtype) {
  if (T < 0 || T > kMaxRows) return HC_ERR_BAD_SIZE;
  if (D < 1 || F < 1 || O < 1 || D > kMaxWidth || F > kMaxWidth || O > kMaxWidth) return HC_ERR_BAD_SIZE;
  if (act != HC_ACT_SILU && act != HC_ACT_GELU_TANH) return HC_ERR_BAD_SIZE;
  return dtype_size(dtype) == 0 ? HC_ERR_DTYPE : HC_OK;
}

int64_t padded(int64_t F) { return (F + 7) / 8 * 8; }

int run(const FfnProduct& p, int dtype, cudaStream_t s) { return ffn_simt_launch(p, dtype, s); }

FfnProduct store(int64_t M, int64_t N, int64_t K, FfnOperand A, FfnOperand B, void* out) {
  FfnProduct p{};
  p.epilogue = kStore;
  p.terms = 1;
  p.A[0] = A;
  p.B[0] = B;
  p.M = M; p.N = N; p.K = K;
  p.out = out;
  p.ldo = N;
  return p;
}

}  // namespace
}  // namespace hc

using namespace hc;

extern "C" int64_t hc_gated_ffn_scratch_bytes(int backward, int64_t T, int64_t D, int64_t F, int64_t O, int dtype) {
  (void)backward;
  if (check(T, D, F, O, HC_ACT_SILU, dtype)) return -1;
  return 0;
}

extern "C" int hc_gated_ffn_fwd(const void* x, const void* w_gate, const void* w_up, const void* w_down, void* y,
                                void* h, void* pre_gate, void* pre_up, void* scratch, int64_t scratch_bytes, int64_t T,
                                int64_t D, int64_t F, int64_t O, int act, int dtype, void* stream) {
  HC_ENTRY("hc_gated_ffn_fwd");
  if (int rc = check(T, D, F, O, act, dtype)) return rc;
  if (T == 0) return HC_OK;
  if (!x || !w_gate || !w_up || !w_down || !y || !h || !pre_gate != !pre_up) return HC_ERR_NULL_POINTER;
  const int64_t need = hc_gated_ffn_scratch_bytes(0, T, D, F, O, dtype);
  if (need > 0 && (!scratch || scratch_bytes < need)) return HC_ERR_SCRATCH;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t Fp = padded(F);
  FfnProduct p{};
  p.epilogue = kGlu;
  p.terms = 1;
  p.A[0] = {x, D, 1, T};
  p.B[0] = {w_gate, D, 1, F};
  p.B[1] = {w_up, D, 1, F};
  p.M = T; p.N = Fp; p.K = D;
  p.out = h; p.pre_gate = pre_gate; p.pre_up = pre_up; p.ldo = Fp; p.act = act;
  if (int rc = run(p, dtype, s)) return rc;
  return run(store(T, O, F, {h, Fp, 1, T}, {w_down, F, 1, O}, y), dtype, s);
}

extern "C" int hc_gated_ffn_bwd(const void* g, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                                const void* h, const void* pre_gate, const void* pre_up, void* d_gate, void* d_up,
                                void* grad_x, void* grad_w_gate, void* grad_w_up, void* grad_w_down, void* scratch,
                                int64_t scratch_bytes, int64_t T, int64_t D, int64_t F, int64_t O, int act, int dtype,
                                void* stream) {
  HC_ENTRY("hc_gated_ffn_bwd");
  if (int rc = check(T, D, F, O, act, dtype)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // sums over no token
    const size_t es = dtype_size(dtype);
    const struct { void* p; int64_t count; } zero[] = {{grad_w_gate, F * D}, {grad_w_up, F * D}, {grad_w_down, O * F}};
    for (const auto& z : zero)
      if (z.p && cudaMemsetAsync(z.p, 0, es * z.count, s) != cudaSuccess) return HC_ERR_LAUNCH;
    return HC_OK;
  }
  const bool inner = grad_x || grad_w_gate || grad_w_up;
  if (!g || (inner && (!w_down || !pre_gate || !pre_up || !d_gate || !d_up)) || (grad_x && (!w_gate || !w_up)) ||
      ((grad_w_gate || grad_w_up) && !x) || (grad_w_down && !h))
    return HC_ERR_NULL_POINTER;
  const int64_t need = hc_gated_ffn_scratch_bytes(1, T, D, F, O, dtype);
  if (need > 0 && (!scratch || scratch_bytes < need)) return HC_ERR_SCRATCH;
  const int64_t Fp = padded(F);
  if (inner) {
    FfnProduct p{};
    p.epilogue = kGluBwd;
    p.terms = 1;
    p.A[0] = {g, O, 1, T};
    p.B[0] = {w_down, 1, F, F};
    p.M = T; p.N = Fp; p.K = O;
    p.out = d_gate; p.out2 = d_up; p.pre_gate = const_cast<void*>(pre_gate); p.pre_up = const_cast<void*>(pre_up);
    p.ldo = Fp; p.act = act;
    if (int rc = run(p, dtype, s)) return rc;
  }
  if (grad_x) {
    FfnProduct p = store(T, D, F, {d_gate, Fp, 1, T}, {w_gate, 1, D, D}, grad_x);
    p.terms = 2;
    p.A[1] = {d_up, Fp, 1, T};
    p.B[1] = {w_up, 1, D, D};
    if (int rc = run(p, dtype, s)) return rc;
  }
  if (grad_w_gate)
    if (int rc = run(store(F, D, T, {d_gate, 1, Fp, F}, {x, 1, D, D}, grad_w_gate), dtype, s)) return rc;
  if (grad_w_up)
    if (int rc = run(store(F, D, T, {d_up, 1, Fp, F}, {x, 1, D, D}, grad_w_up), dtype, s)) return rc;
  if (grad_w_down)
    if (int rc = run(store(O, F, T, {g, 1, O, O}, {h, 1, Fp, F}, grad_w_down), dtype, s)) return rc;
  return HC_OK;
}

// ffn_capi.cu — C entry points of the gated feed-forward (see hcops.h): host
// checks, then its products one after the other on the caller's stream.
#include "ffn.cuh"

namespace hc {
namespace {

// Within these every product's tiles and coordinates are 32-bit numbers.
constexpr int64_t kMaxRows = int64_t(1) << 22, kMaxWidth = int64_t(1) << 20;

int check(int64_t T, int64_t D, int64_t F, int64_t O, int act, int dtype) {
  if (T < 0 || T > kMaxRows) return HC_ERR_BAD_SIZE;
  if (D < 1 || F < 1 || O < 1 || D > kMaxWidth || F > kMaxWidth || O > kMaxWidth) return HC_ERR_BAD_SIZE;
  if (act != HC_ACT_SILU && act != HC_ACT_GELU_TANH) return HC_ERR_BAD_SIZE;
  return dtype_size(dtype) == 0 ? HC_ERR_DTYPE : HC_OK;
}

int64_t padded(int64_t F) { return (F + 7) / 8 * 8; }

bool half(int dtype) { return dtype != HC_DTYPE_F32; }

// Caller scratch handed out in 256-byte pieces; with base == nullptr it only
// counts.
struct Scratch {
  uint8_t* base;
  int64_t used;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};

// Rows of `cols` 16-bit elements to rows of `ld`, a multiple of 8, zeros behind.
__global__ void __launch_bounds__(256) ffn_pad_rows(const uint16_t* src, uint16_t* dst, int64_t rows, int64_t cols,
                                                    int64_t ld) {
  const int64_t chunks = ld / 8, count = rows * chunks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / chunks, c = (i - r * chunks) * 8;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) w[e / 2] |= static_cast<uint32_t>(src[r * cols + c + e]) << (16 * (e % 2));
    st_v4(dst + r * ld + c, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// A row-major matrix with its row stride: the caller's, or where its rows do
// not start on 16-byte boundaries (half precision with cols % 8 != 0) a padded
// copy, which the tensor copies need. The copies' bytes are a small part of
// what the products over them read.
struct Matrix {
  const void* p;
  int64_t ld;
};
int fit(Matrix& out, Scratch& scratch, const void* p, int64_t rows, int64_t cols, int dtype, cudaStream_t s) {
  out = {p, cols};
  if (!half(dtype) || cols % 8 == 0) return HC_OK;
  out.ld = padded(cols);
  void* copy = scratch.take(rows * out.ld * 2);
  out.p = copy;
  if (!scratch.base || !p) return HC_OK;
  const int64_t want = (rows * out.ld / 8 + 255) / 256, most = 8 * sm_count();
  ffn_pad_rows<<<static_cast<int>(want < most ? want : most), 256, 0, s>>>(
      static_cast<const uint16_t*>(p), static_cast<uint16_t*>(copy), rows, cols, out.ld);
  return launch_status();
}

// A few tokens: the weights bound the forward, and ffn_few.cu streams them. (D =
// 2048, F = 8192, bf16, from cold caches: 8, 16 and 32 tokens 27.5, 33.8 and 44.1 us,
// on the tensor-core tiles 33 and 128 tokens 50.2 and 56.3; 384 x 1536: 32 tokens
// 15.3, 33 tokens 27.6.)
bool few(int64_t T, int dtype) { return half(dtype) && T <= kFewTokens; }

// Float32 parts of products [M, N] summed over K in one launch.
int64_t parts_bytes(std::initializer_list<FfnSize> results, int64_t K, int terms, int dtype) {
  int64_t count = 0, tiles = 0;
  bool rows_few = true;
  for (const FfnSize& r : results) {
    count += r.M * r.N;
    rows_few = rows_few && ffn_simt_few(r.M);
  }
  for (const FfnSize& r : results) tiles += ffn_simt_tiles(r.M, r.N, rows_few);
  const int64_t splits = half(dtype) ? ffn_tc_plan(results.begin(), static_cast<int>(results.size()), K, terms).splits
                                     : ffn_simt_splits(tiles, K, terms, rows_few);
  return splits > 1 ? splits * count * 4 : 0;
}

// The largest of what a call's launches need, whichever gradients it wants.
int64_t most_parts(int backward, int64_t T, int64_t D, int64_t F, int64_t O, int dtype) {
  if (!backward) return few(T, dtype) ? 0 : parts_bytes({{T, O}}, F, 1, dtype);
  int64_t most = parts_bytes({{T, D}}, F, 2, dtype);
  const FfnSize g{F, D}, d{O, F};  // w_gate's or w_up's, w_down's
  for (const int64_t b : {parts_bytes({g}, T, 1, dtype), parts_bytes({g, g}, T, 1, dtype), parts_bytes({d}, T, 1, dtype),
                          parts_bytes({g, d}, T, 1, dtype), parts_bytes({g, g, d}, T, 1, dtype)})
    if (b > most) most = b;
  return most;
}

int run(const FfnProduct* p, int jobs, int dtype, void* parts, cudaStream_t s) {
  float* f = static_cast<float*>(parts);
  return half(dtype) ? ffn_tc_launch(p, jobs, dtype, f, s) : ffn_simt_launch(p, jobs, f, s);
}
int run(const FfnProduct& p, int dtype, void* parts, cudaStream_t s) { return run(&p, 1, dtype, parts, s); }

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

bool aligned256(const void* p) { return reinterpret_cast<uintptr_t>(p) % 256 == 0; }

bool aligned_for(int dtype, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (half(dtype) ? !aligned16(p) : !aligned4(p)) return false;
  return true;
}

}  // namespace
}  // namespace hc

using namespace hc;

extern "C" int64_t hc_gated_ffn_scratch_bytes(int backward, int64_t T, int64_t D, int64_t F, int64_t O, int dtype) {
  if (check(T, D, F, O, HC_ACT_SILU, dtype)) return -1;
  if (T == 0) return 0;
  Scratch count{};
  Matrix m;
  fit(m, count, nullptr, T, D, dtype, nullptr);  // x
  for (int i = 0; i < 2; ++i) fit(m, count, nullptr, F, D, dtype, nullptr);  // w_gate, w_up
  fit(m, count, nullptr, O, F, dtype, nullptr);  // w_down
  if (backward) fit(m, count, nullptr, T, O, dtype, nullptr);  // g
  count.take(most_parts(backward, T, D, F, O, dtype));
  return count.used;
}

extern "C" int hc_gated_ffn_fwd(const void* x, const void* w_gate, const void* w_up, const void* w_down, void* y,
                                void* h, void* slope_gate, void* slope_up, void* scratch, int64_t scratch_bytes,
                                int64_t T, int64_t D, int64_t F, int64_t O, int act, int dtype, void* stream) {
  HC_ENTRY("hc_gated_ffn_fwd");
  if (int rc = check(T, D, F, O, act, dtype)) return rc;
  if (T == 0) return HC_OK;
  if (!x || !w_gate || !w_up || !w_down || !y || !h || !slope_gate != !slope_up) return HC_ERR_NULL_POINTER;
  if (!aligned_for(dtype, {x, w_gate, w_up, w_down, y, h, slope_gate, slope_up})) return HC_ERR_ALIGNMENT;
  const int64_t need = hc_gated_ffn_scratch_bytes(0, T, D, F, O, dtype);
  if (need > 0 && (!scratch || scratch_bytes < need)) return HC_ERR_SCRATCH;
  if (need > 0 && !aligned256(scratch)) return HC_ERR_ALIGNMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t Fp = padded(F);
  Scratch space{static_cast<uint8_t*>(scratch), 0};
  Matrix mx, mg, mu, md;
  if (int rc = fit(mx, space, x, T, D, dtype, s)) return rc;
  if (int rc = fit(mg, space, w_gate, F, D, dtype, s)) return rc;
  if (int rc = fit(mu, space, w_up, F, D, dtype, s)) return rc;
  if (int rc = fit(md, space, w_down, O, F, dtype, s)) return rc;
  FfnProduct p{};
  p.epilogue = kGlu;
  p.terms = 1;
  p.A[0] = {mx.p, mx.ld, 1, T};
  p.B[0] = {mg.p, mg.ld, 1, F};
  p.B[1] = {mu.p, mu.ld, 1, F};
  p.M = T; p.N = Fp; p.K = D;
  p.out = h; p.slope_gate = slope_gate; p.slope_up = slope_up; p.ldo = Fp; p.act = act;
  const FfnProduct down = store(T, O, F, {h, Fp, 1, T}, {md.p, md.ld, 1, O}, y);
  if (few(T, dtype)) {
    if (int rc = ffn_few_launch(p, dtype, s)) return rc;
    return ffn_few_launch(down, dtype, s);
  }
  if (int rc = run(p, dtype, nullptr, s)) return rc;
  return run(down, dtype, space.take(0), s);
}

extern "C" int hc_gated_ffn_bwd(const void* g, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                                const void* h, const void* slope_gate, const void* slope_up, void* d_gate, void* d_up,
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
  if (!g || (inner && (!w_down || !slope_gate || !slope_up || !d_gate || !d_up)) || (grad_x && (!w_gate || !w_up)) ||
      ((grad_w_gate || grad_w_up) && !x) || (grad_w_down && !h))
    return HC_ERR_NULL_POINTER;
  if (!aligned_for(dtype, {g, x, w_gate, w_up, w_down, h, slope_gate, slope_up, d_gate, d_up, grad_x, grad_w_gate,
                           grad_w_up, grad_w_down}))
    return HC_ERR_ALIGNMENT;
  const int64_t need = hc_gated_ffn_scratch_bytes(1, T, D, F, O, dtype);
  if (need > 0 && (!scratch || scratch_bytes < need)) return HC_ERR_SCRATCH;
  if (need > 0 && !aligned256(scratch)) return HC_ERR_ALIGNMENT;
  const int64_t Fp = padded(F);
  Scratch space{static_cast<uint8_t*>(scratch), 0};
  Matrix mg, mx, wg, wu, wd;  // what is not needed is not copied
  if (int rc = fit(mg, space, g, T, O, dtype, s)) return rc;
  if (int rc = fit(mx, space, grad_w_gate || grad_w_up ? x : nullptr, T, D, dtype, s)) return rc;
  if (int rc = fit(wg, space, grad_x ? w_gate : nullptr, F, D, dtype, s)) return rc;
  if (int rc = fit(wu, space, grad_x ? w_up : nullptr, F, D, dtype, s)) return rc;
  if (int rc = fit(wd, space, inner ? w_down : nullptr, O, F, dtype, s)) return rc;
  void* parts = space.take(0);
  if (inner) {
    FfnProduct p{};
    p.epilogue = kGluBwd;
    p.terms = 1;
    p.A[0] = {mg.p, mg.ld, 1, T};
    p.B[0] = {wd.p, 1, wd.ld, F};
    p.M = T; p.N = Fp; p.K = O;
    p.out = d_gate; p.out2 = d_up;
    p.slope_gate = const_cast<void*>(slope_gate); p.slope_up = const_cast<void*>(slope_up);
    p.ldo = Fp; p.act = act;
    if (int rc = run(p, dtype, nullptr, s)) return rc;
  }
  if (grad_x) {
    FfnProduct p = store(T, D, F, {d_gate, Fp, 1, T}, {wg.p, 1, wg.ld, D}, grad_x);
    p.terms = 2;
    p.A[1] = {d_up, Fp, 1, T};
    p.B[1] = {wu.p, 1, wu.ld, D};
    if (int rc = run(p, dtype, parts, s)) return rc;
  }
  FfnProduct weights[kFfnMaxJobs];  // the weights' gradients, all sums over the tokens
  int jobs = 0;
  if (grad_w_gate) weights[jobs++] = store(F, D, T, {d_gate, 1, Fp, F}, {mx.p, 1, mx.ld, D}, grad_w_gate);
  if (grad_w_up) weights[jobs++] = store(F, D, T, {d_up, 1, Fp, F}, {mx.p, 1, mx.ld, D}, grad_w_up);
  if (grad_w_down) weights[jobs++] = store(O, F, T, {mg.p, 1, mg.ld, O}, {h, 1, Fp, F}, grad_w_down);
  return jobs ? run(weights, jobs, dtype, parts, s) : HC_OK;
}

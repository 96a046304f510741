// torch_block.cpp — the operators around a layer's block as C++ autograd
// Functions over the C ABI of libhcops.so, for the reason that torch_ops.cpp
// gives: one decoding step's call is 2-4 us on the GPU, and a Python Function
// around a ctypes call of 25 arguments takes 20-50 us on the host.
//
// Each function below takes tensors as the kernels want them (dtypes, one
// CUDA device, shapes; any strides) and returns None for anything else, so
// that the Python operators (ops/block.py, dropout.py, ffn.py), which name
// what is wrong or convert, run their checks only where something is to be
// said.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/hcops.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using MaybeTensor = std::optional<Tensor>;

void check(int rc, const char* what) {
  TORCH_CHECK(rc == HC_OK, what, " failed: ", hc_error_string(rc), " (hcops status ", rc, ")");
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

int code_of(c10::ScalarType t) {
  switch (t) {
    case torch::kFloat32: return HC_DTYPE_F32;
    case torch::kFloat16: return HC_DTYPE_F16;
    case torch::kBFloat16: return HC_DTYPE_BF16;
    default: return -1;
  }
}

Tensor get(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
// Dense on a 16-byte boundary: a copy where it is neither.
Tensor dense16(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
const int64_t* state_ptr(const Tensor& t) { return static_cast<const int64_t*>(ptr(t)); }
Tensor like(bool wanted, const Tensor& t) { return wanted && t.defined() ? torch::empty_like(t) : Tensor(); }

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

// One gradient buffer for each input that a gradient is wanted of; autograd
// numbers the inputs that are there.
template <typename Saved> tensor_list wanted(AutogradContext* ctx, const Saved& t, int count) {
  tensor_list d;
  size_t edge = 0;
  for (int i = 0; i < count; ++i) {
    const bool there = t[i].defined();
    d.push_back(like(there && ctx->needs_input_grad(edge), t[i]));
    edge += there;
  }
  return d;
}

// Whether a call goes through its autograd Function: a gradient may be asked of
// it, or an input carries a tangent of forward-mode differentiation (with or
// without gradients enabled), which the Function refuses; without it the tangent
// would be lost.
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  const bool grads = at::GradMode::is_enabled();
  for (const Tensor* t : ts)
    if (t->defined() && ((grads && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined())) return true;
  return false;
}

// What a backward under create_graph returns: differentiating it again raises.
tensor_list once(tensor_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  tensor_list in;
  for (const auto& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
  auto err = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator that is once differentiable", static_cast<int64_t>(in.size()));
  return (*err)(std::move(in));
}

bool f32_on(const Tensor& t, const Tensor& x) {
  return t.scalar_type() == torch::kFloat32 && t.device() == x.device();
}
// A [m D] parameter in float32: (m D) or (m, D).
bool param_ok(const Tensor& t, const Tensor& x, int64_t m, int64_t D) {
  if (!t.defined()) return true;
  return f32_on(t, x) && ((t.dim() == 1 && t.size(0) == m * D) || (t.dim() == 2 && t.size(0) == m && t.size(1) == D));
}
// t's sizes are x's leading ones, then a and b (b < 0: a alone).
bool shaped(const Tensor& t, const Tensor& x, int64_t a, int64_t b) {
  const int64_t lead = x.dim() - 2;
  if (t.dim() != lead + (b < 0 ? 1 : 2)) return false;
  for (int64_t i = 0; i < lead; ++i)
    if (t.size(i) != x.size(i)) return false;
  return t.size(lead) == a && (b < 0 || t.size(lead + 1) == b);
}
bool streams_ok(const Tensor& x) {
  return x.is_cuda() && code_of(x.scalar_type()) >= 0 && x.dim() >= 2 && x.size(-2) >= 1 && x.size(-2) <= 8;
}
int64_t tokens_of(const Tensor& x) {
  int64_t T = 1;
  for (int64_t i = 0; i < x.dim() - 2; ++i) T *= x.size(i);
  return T;
}
Tensor with_rows(const Tensor& x, int64_t m) {  // [*, m, D] for x [*, n, D]
  auto sizes = x.sizes().vec();
  sizes[sizes.size() - 2] = m;
  return torch::empty(sizes, x.options());
}
Tensor scratch_floats(int64_t words, const Tensor& x) {
  return torch::empty({std::max<int64_t>(words, 1)}, x.options().dtype(torch::kFloat32));
}

// ------------------------------------------------------------- hc_read_norm
struct ReadNorm : public torch::autograd::Function<ReadNorm> {
  static Tensor run(const Tensor& R, const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t norm,
                    double eps, Tensor* stats) {
    const int64_t T = tokens_of(x), n = x.size(-2), D = x.size(-1), m = R.size(-2);
    Tensor y = with_rows(x, m);
    if (stats) *stats = torch::empty({T, 2}, R.options());
    check(hc_read_norm_fwd(fptr(R), ptr(x), fptr(weight), fptr(bias), ptr(y), stats ? fptr(*stats) : nullptr, T,
                           static_cast<int>(n), static_cast<int>(m), D, static_cast<int>(norm),
                           static_cast<float>(eps), code_of(x.scalar_type()), stream_of(x)),
          "hc_read_norm_fwd");
    return y;
  }

  static Tensor forward(AutogradContext* ctx, const Tensor& R, const Tensor& x, const MaybeTensor& weight,
                        const MaybeTensor& bias, int64_t norm, double eps) {
    Tensor stats;
    const Tensor Rc = dense(R), xc = dense(x), wc = dense(get(weight)), bc = dense(get(bias));
    Tensor y = run(Rc, xc, wc, bc, norm, eps, &stats);
    ctx->save_for_backward({Rc, xc, wc, bc, stats});
    ctx->saved_data["norm"] = norm;
    return y;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &R = saved[0], &x = saved[1], &weight = saved[2], &stats = saved[4];
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t T = stats.size(0), n = x.size(-2), D = x.size(-1), m = R.size(-2);
    const int code = code_of(x.scalar_type());
    const Tensor g = grads[0].to(x.scalar_type()).contiguous();
    const tensor_list d = wanted(ctx, saved, 4);
    const Tensor &gR = d[0], &gx = d[1], &gw = d[2], &gb = d[3];
    Tensor scratch;
    int64_t words = 0;
    if (gw.defined() || gb.defined()) {
      words = hc_norm_scratch_words(T, static_cast<int>(n), static_cast<int>(m), D, code);
      scratch = scratch_floats(words, x);
    }
    check(hc_read_norm_bwd(ptr(g), fptr(R), ptr(x), fptr(weight), fptr(stats), ptr(gx), fptr(gR), fptr(gw), fptr(gb),
                           fptr(scratch), words, T, static_cast<int>(n), static_cast<int>(m), D,
                           static_cast<int>(ctx->saved_data["norm"].toInt()), code, stream_of(x)),
          "hc_read_norm_bwd");
    return once({gR, gx, gw, gb, Tensor(), Tensor()});
  }
};

MaybeTensor read_norm(const Tensor& R, const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_,
                      int64_t norm, double eps) {
  const Tensor weight = get(weight_), bias = get(bias_);
  if (!streams_ok(x) || (norm != HC_NORM_RMS && norm != HC_NORM_LAYER) || !(eps >= 0)) return std::nullopt;
  const int64_t n = x.size(-2), D = x.size(-1), m = R.dim() >= 2 ? R.size(-2) : 0;
  if (m < 1 || m > 4 || !f32_on(R, x) || !shaped(R, x, m, n) || !param_ok(weight, x, m, D) ||
      !param_ok(bias, x, m, D))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  if (wants_grad({&R, &x, &weight, &bias})) return ReadNorm::apply(R, x, maybe(weight), maybe(bias), norm, eps);
  return ReadNorm::run(dense(R), dense(x), dense(weight), dense(bias), norm, eps, nullptr);
}

// --------------------------------------------------------- hc_mix_write_norm
struct WriteMeta {
  int64_t norm, act, seed, offset;
  double eps, p;
};

struct MixWriteNorm : public torch::autograd::Function<MixWriteNorm> {
  // t: H, x, W, f, v, weight, bias, gate, scale
  static Tensor run(const tensor_list& t, const Tensor& state, const WriteMeta& k, Tensor* stats) {
    const Tensor& x = t[1];
    const int64_t T = tokens_of(x), n = x.size(-2), D = x.size(-1), m = t[2].size(-1);
    Tensor out = torch::empty_like(x);
    if (stats && k.norm != HC_NORM_NONE) *stats = torch::empty({T, 2}, t[0].options());
    check(hc_mix_write_norm_fwd(fptr(t[0]), ptr(x), fptr(t[2]), ptr(t[3]), fptr(t[4]), fptr(t[5]), fptr(t[6]),
                                ptr(t[7]), fptr(t[8]), ptr(out), stats ? fptr(*stats) : nullptr, T,
                                static_cast<int>(n), static_cast<int>(m), D, static_cast<int>(k.norm),
                                static_cast<int>(k.act), static_cast<float>(k.eps), k.p, state_ptr(state), k.seed,
                                k.offset, code_of(x.scalar_type()), stream_of(x)),
          "hc_mix_write_norm_fwd");
    return out;
  }

  static Tensor forward(AutogradContext* ctx, const Tensor& H, const Tensor& x, const Tensor& W, const Tensor& f,
                        const MaybeTensor& v, const MaybeTensor& weight, const MaybeTensor& bias,
                        const MaybeTensor& gate, const MaybeTensor& scale, const MaybeTensor& state,
                        c10::IntArrayRef whole, double eps, double p) {
    const WriteMeta k{whole[0], whole[1], whole[2], whole[3], eps, p};
    tensor_list t = {dense(H), dense(x), dense(W), dense(f)};
    for (const MaybeTensor* a : {&v, &weight, &bias, &gate, &scale}) t.push_back(dense(get(*a)));
    Tensor stats;
    // the caller may move its seed on before the backward draws the bits again
    const Tensor own = state.has_value() ? state->clone() : Tensor();
    Tensor out = run(t, own, k, &stats);
    t.push_back(stats);
    t.push_back(own);
    ctx->save_for_backward(t);
    ctx->saved_data["whole"] = whole.vec();
    ctx->saved_data["p"] = p;
    return out;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto t = ctx->get_saved_variables();
    const Tensor& x = t[1];
    const c10::cuda::CUDAGuard guard(x.device());
    const auto whole = ctx->saved_data["whole"].toIntVector();
    const int64_t T = tokens_of(x), n = x.size(-2), D = x.size(-1), m = t[2].size(-1);
    const int code = code_of(x.scalar_type());
    const Tensor g = grads[0].to(x.scalar_type()).contiguous();
    tensor_list d = wanted(ctx, t, 9);
    Tensor scratch;
    int64_t words = 0;
    if (d[5].defined() || d[6].defined() || d[8].defined()) {
      words = hc_norm_scratch_words(T, static_cast<int>(n), static_cast<int>(m), D, code);
      scratch = scratch_floats(words, x);
    }
    check(hc_mix_write_norm_bwd(ptr(g), fptr(t[0]), ptr(x), fptr(t[2]), ptr(t[3]), fptr(t[4]), fptr(t[5]), fptr(t[6]),
                                ptr(t[7]), fptr(t[8]), fptr(t[9]), ptr(d[1]), ptr(d[3]), ptr(d[7]), fptr(d[0]),
                                fptr(d[2]), fptr(d[4]), fptr(d[5]), fptr(d[6]), fptr(d[8]), fptr(scratch), words, T,
                                static_cast<int>(n), static_cast<int>(m), D, static_cast<int>(whole[0]),
                                static_cast<int>(whole[1]), ctx->saved_data["p"].toDouble(), state_ptr(t[10]),
                                whole[2], whole[3], code, stream_of(x)),
          "hc_mix_write_norm_bwd");
    d.resize(13);  // state, whole, eps, p have none
    return once(std::move(d));
  }
};

bool state_ok(const Tensor& state, const Tensor& x) {
  return !state.defined() || (state.scalar_type() == torch::kInt64 && state.dim() == 1 && state.size(0) == 2 &&
                              state.device() == x.device() && state.is_contiguous());
}

MaybeTensor mix_write_norm(const Tensor& H, const Tensor& x, const Tensor& W, const Tensor& f, const MaybeTensor& v_,
                           const MaybeTensor& weight_, const MaybeTensor& bias_, const MaybeTensor& gate_,
                           const MaybeTensor& scale_, const MaybeTensor& state_, int64_t norm, int64_t act, double eps,
                           double p, int64_t seed, int64_t offset) {
  const Tensor v = get(v_), weight = get(weight_), bias = get(bias_), gate = get(gate_), scale = get(scale_),
               state = get(state_);
  if (!streams_ok(x) || norm < HC_NORM_NONE || norm > HC_NORM_LAYER || act < HC_ACT_LINEAR || act > HC_ACT_SIGMOID ||
      !(eps >= 0) || !(p >= 0 && p <= 1))
    return std::nullopt;
  const int64_t n = x.size(-2), D = x.size(-1), m = W.dim() >= 2 ? W.size(-1) : 0;
  const auto stream = [&](const Tensor& t) {
    return t.scalar_type() == x.scalar_type() && t.device() == x.device() && shaped(t, x, m, D);
  };
  if (m < 1 || m > 4 || !f32_on(H, x) || !shaped(H, x, n, n) || !f32_on(W, x) || !shaped(W, x, n, m) || !stream(f) ||
      (gate.defined() && !stream(gate)) || (v.defined() && !(f32_on(v, x) && shaped(v, x, n, -1))) ||
      !param_ok(weight, x, m, D) || !param_ok(bias, x, m, D) || !param_ok(scale, x, m, D) || !state_ok(state, x))
    return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  if (wants_grad({&H, &x, &W, &f, &v, &weight, &bias, &gate, &scale})) {
    const int64_t whole[4] = {norm, act, seed, offset};
    return MixWriteNorm::apply(H, x, W, f, maybe(v), maybe(weight), maybe(bias), maybe(gate), maybe(scale),
                               maybe(state), c10::IntArrayRef(whole, 4), eps, p);
  }
  tensor_list t;
  for (const Tensor* a : {&H, &x, &W, &f, &v, &weight, &bias, &gate, &scale}) t.push_back(dense(*a));
  return MixWriteNorm::run(t, state, WriteMeta{norm, act, seed, offset, eps, p}, nullptr);
}

// ---------------------------------------------------------------- hc_dropout
struct Dropout : public torch::autograd::Function<Dropout> {
  static Tensor run(const Tensor& x, const Tensor& state, double p, int64_t seed, int64_t offset) {
    Tensor y = torch::empty_like(x);
    check(hc_dropout(ptr(x), ptr(y), x.numel(), p, state_ptr(state), seed, offset, code_of(x.scalar_type()),
                     stream_of(x)),
          "hc_dropout");
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& state, double p, int64_t seed,
                        int64_t offset) {
    const Tensor own = state.has_value() ? state->clone() : Tensor();  // as in MixWriteNorm
    ctx->save_for_backward({own});
    ctx->saved_data["p"] = p;
    ctx->saved_data["whole"] = std::vector<int64_t>{seed, offset, static_cast<int64_t>(x.scalar_type())};
    return run(x.contiguous(), own, p, seed, offset);
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const c10::cuda::CUDAGuard guard(grads[0].device());
    const auto whole = ctx->saved_data["whole"].toIntVector();
    const Tensor g = grads[0].to(static_cast<c10::ScalarType>(whole[2])).contiguous();
    return once({run(g, ctx->get_saved_variables()[0], ctx->saved_data["p"].toDouble(), whole[0], whole[1]), Tensor(),
                 Tensor(), Tensor(), Tensor()});
  }
};

MaybeTensor dropout(const Tensor& x, const MaybeTensor& state_, double p, int64_t seed, int64_t offset) {
  const Tensor state = get(state_);
  if (!x.is_cuda() || code_of(x.scalar_type()) < 0 || !(p >= 0 && p <= 1) || !state_ok(state, x)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  if (wants_grad({&x})) return Dropout::apply(x, maybe(state), p, seed, offset);
  return Dropout::run(x.contiguous(), state, p, seed, offset);
}

// ----------------------------------------------------------------- gated_ffn
struct GatedFfn : public torch::autograd::Function<GatedFfn> {
  // A width of 0: every sum is empty, and y and all gradients are 0.
  static bool nothing(const tensor_list& t) { return t[0].size(-1) == 0 || t[3].numel() == 0; }
  static Tensor scratch_bytes(int backward, int64_t T, int64_t D, int64_t F, int64_t O, const Tensor& x,
                              int64_t* size) {
    *size = hc_gated_ffn_scratch_bytes(backward, T, D, F, O, code_of(x.scalar_type()));
    return *size > 0 ? torch::empty({*size}, x.options().dtype(torch::kUInt8)) : Tensor();
  }
  // t: x, w_gate, w_up, w_down, dense; h and, where kept, the slopes come back
  static Tensor run(const tensor_list& t, int64_t act, bool keep, tensor_list* inner) {
    const Tensor& x = t[0];
    const int64_t D = x.size(-1), F = t[1].size(0), O = t[3].size(0), Fp = (F + 7) / 8 * 8;
    auto sizes = x.sizes().vec();
    int64_t T = 1;
    for (size_t i = 0; i + 1 < sizes.size(); ++i) T *= sizes[i];
    sizes.back() = O;
    if (nothing(t)) return torch::zeros(sizes, x.options());
    Tensor y = torch::empty(sizes, x.options()), h = torch::empty({T, Fp}, x.options()), sg, su;
    if (keep) {
      sg = torch::empty_like(h);
      su = torch::empty_like(h);
    }
    int64_t size = 0;
    Tensor scratch = scratch_bytes(0, T, D, F, O, x, &size);
    check(hc_gated_ffn_fwd(ptr(x), ptr(t[1]), ptr(t[2]), ptr(t[3]), ptr(y), ptr(h), ptr(sg), ptr(su), ptr(scratch),
                           size, T, D, F, O, static_cast<int>(act), code_of(x.scalar_type()), stream_of(x)),
          "hc_gated_ffn_fwd");
    if (inner) *inner = {h, sg, su};
    return y;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                        const Tensor& w_down, int64_t act) {
    tensor_list t = {dense16(x), dense16(w_gate), dense16(w_up), dense16(w_down)}, inner(3);
    Tensor y = run(t, act, true, &inner);
    t.insert(t.end(), inner.begin(), inner.end());
    ctx->save_for_backward(t);
    ctx->saved_data["act"] = act;
    return y;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto t = ctx->get_saved_variables();
    const Tensor &x = t[0], &h = t[4];
    const c10::cuda::CUDAGuard guard(x.device());
    tensor_list d = wanted(ctx, t, 4);
    if (nothing(t)) {
      for (Tensor& a : d)
        if (a.defined()) a.zero_();
      d.emplace_back();
      return once(std::move(d));
    }
    const int64_t D = x.size(-1), F = t[1].size(0), O = t[3].size(0), T = h.size(0);
    const Tensor g = dense16(grads[0].to(x.scalar_type()));
    const bool inner = d[0].defined() || d[1].defined() || d[2].defined();
    const Tensor da = like(inner, h), db = like(inner, h);
    int64_t size = 0;
    Tensor scratch = scratch_bytes(1, T, D, F, O, x, &size);
    check(hc_gated_ffn_bwd(ptr(g), ptr(x), ptr(t[1]), ptr(t[2]), ptr(t[3]), ptr(h), ptr(t[5]), ptr(t[6]), ptr(da),
                           ptr(db), ptr(d[0]), ptr(d[1]), ptr(d[2]), ptr(d[3]), ptr(scratch), size, T, D, F, O,
                           static_cast<int>(ctx->saved_data["act"].toInt()), code_of(x.scalar_type()), stream_of(x)),
          "hc_gated_ffn_bwd");
    d.emplace_back();  // act
    return once(std::move(d));
  }
};

MaybeTensor gated_ffn(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, int64_t act) {
  if (!x.is_cuda() || code_of(x.scalar_type()) < 0 || x.dim() < 1 || w_gate.dim() != 2 || w_up.dim() != 2 ||
      w_down.dim() != 2 || (act != HC_ACT_SILU && act != HC_ACT_GELU_TANH))
    return std::nullopt;
  for (const Tensor* w : {&w_gate, &w_up, &w_down})
    if (w->scalar_type() != x.scalar_type() || w->device() != x.device()) return std::nullopt;
  const int64_t F = w_gate.size(0);
  if (w_gate.size(1) != x.size(-1) || w_up.sizes() != w_gate.sizes() || w_down.size(1) != F) return std::nullopt;
  const c10::cuda::CUDAGuard guard(x.device());
  if (wants_grad({&x, &w_gate, &w_up, &w_down})) return GatedFfn::apply(x, w_gate, w_up, w_down, act);
  return GatedFfn::run({dense16(x), dense16(w_gate), dense16(w_up), dense16(w_down)}, act, false, nullptr);
}

}  // namespace

// Called by the module definition of torch_ops.cpp.
void bind_block_ops(pybind11::module_& m) {
  m.def("read_norm", &read_norm, "width-read + pre-norm, differentiable; None for tensors it does not take");
  m.def("mix_write_norm", &mix_write_norm,
        "post-norm, gate, scale and dropout + mix + depth-write, differentiable; None for tensors it does not take");
  m.def("dropout", &dropout, "counter-based dropout, differentiable; None for tensors it does not take");
  m.def("gated_ffn", &gated_ffn, "gated feed-forward, differentiable; None for tensors it does not take");
}

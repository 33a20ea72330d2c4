// Host side of the operators around the block, as a Python module
// (omniwave_b200._host): argument checks, autograd and the calls of the C ABI
// for the norms, the linear layer, the feed-forward block and the distillation
// loss, and AdamW's step over its buckets.
//
// It is native because these operators are short: a few rows take the GPU 2 to
// 5 us, and the same checks, allocations and autograd nodes took 25 us in
// Python forward, 140 us forward and backward.  No tensor value is touched here.
#include <torch/extension.h>

#include <ATen/autocast_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <atomic>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>
#include <variant>
#include <vector>

#include "omniwave_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// Raises ValueError in Python.
#define OW_VALUE(cond, ...) \
  do {                      \
    if (!(cond)) throw std::invalid_argument(c10::str(__VA_ARGS__)); \
  } while (0)

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return OW_DTYPE_F32;
    case at::kDouble: return OW_DTYPE_F64;
    case at::kBFloat16: return OW_DTYPE_BF16;
    case at::kHalf: return OW_DTYPE_F16;
    default: return -1;
  }
}

bool is16(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool is_float(at::ScalarType t) { return t == at::kFloat || is16(t); }

std::string dtype_text(at::ScalarType t) { return "torch." + std::string(t == at::kFloat ? "float32" : t == at::kDouble ? "float64" : t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" : c10::toString(t)); }

std::string shape_text(at::IntArrayRef s) {
  std::string o = "(";
  for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
  return o + (s.size() == 1 ? ",)" : ")");
}

void check_status(int status, const char* what) {
  TORCH_CHECK(status == OW_OK, what, " failed: ", ow_last_error());
}

bool device_ok(const at::Device& d) {
  static std::atomic<int> known[64];
  const int i = d.index();
  if (i < 0 || i >= 64) return ow_device_supported(i) != 0;
  int v = known[i].load(std::memory_order_relaxed);
  if (v == 0) known[i].store(v = ow_device_supported(i) ? 1 : 2, std::memory_order_relaxed);
  return v == 1;
}

Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor like(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : t; }

// The reason why tensors cannot be taken, or nothing.
std::optional<std::string> unsupported(const Tensor& x, std::initializer_list<Tensor> more) {
  if (!x.is_cuda()) return "CUDA is unavailable";
  auto bad = [&](const Tensor& t) -> std::optional<std::string> {
    if (!t.defined()) return std::nullopt;
    if (!is_float(t.scalar_type())) return "unsupported dtype " + dtype_text(t.scalar_type());
    if (t.device() != x.device()) return "tensors on " + x.device().str() + " and " + t.device().str();
    return std::nullopt;
  };
  if (auto r = bad(x)) return r;
  for (const Tensor& t : more)
    if (auto r = bad(t)) return r;
  if (!device_ok(x.device())) return "device " + std::to_string(x.device().index()) + " is not sm_100 (B200-class)";
  return std::nullopt;
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// A forward-mode tangent would be dropped without a word: the nodes below have no formula for it.
void no_tangents(const char* what, std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, " not supported: forward-mode differentiation");
}

void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the backward is not differentiable (create_graph is not supported)");
}

// ------------------------------------------------------------------ norms
struct NormCall {
  Tensor x, delta, post, gate, scale, next;
  double eps;
  at::ScalarType n_dtype;

  ow_norm_t args() const {
    ow_norm_t a{};
    const int64_t c = x.size(-1), b = x.dim() > 1 ? x.size(0) : 1;
    a.samples = b;
    a.tokens = x.numel() / std::max<int64_t>(1, b * c);
    a.channels = (int32_t)c;
    a.x = ptr(x);
    a.x_dtype = code(x.scalar_type());
    if (delta.defined()) {
      a.delta = ptr(delta);
      a.delta_dtype = code(delta.scalar_type());
      a.post_w = ptr(post);
      a.post_dtype = code(post.scalar_type());
      if (gate.defined()) {
        a.gate = ptr(gate);
        a.gate_dtype = code(gate.scalar_type());
        a.gate_rows = gate.dim() == 1 ? 1 : b;
      }
      a.sample_scale = (const float*)ptr(scale);
    }
    if (next.defined()) {
      a.next_w = ptr(next);
      a.next_dtype = code(next.scalar_type());
      a.n_dtype = code(n_dtype);
    }
    a.eps = eps;
    return a;
  }
};

struct NormOut {
  Tensor h, n, stats;  // stats [2, rows]: rstd of delta and of h
};

NormOut norm_forward(const NormCall& k, bool keep) {
  NormOut o;
  if (k.delta.defined()) o.h = at::empty(k.x.sizes(), k.x.options());
  if (k.next.defined()) o.n = at::empty(k.x.sizes(), k.x.options().dtype(k.n_dtype));
  if (k.x.numel() == 0) return o;
  const c10::cuda::CUDAGuard guard(k.x.device());
  ow_norm_t a = k.args();
  a.h = ptr(o.h);
  a.n = ptr(o.n);
  if (keep) {
    const int64_t rows = a.samples * a.tokens;
    o.stats = at::empty({2, rows}, k.x.options().dtype(at::kFloat));
    a.rstd_delta = (float*)ptr(o.stats);
    a.rstd_h = a.rstd_delta + rows;
  }
  check_status(ow_norm_fwd(&a, stream_of(k.x)), "ow_norm_fwd");
  return o;
}

struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& delta, const OptTensor& post,
                               const OptTensor& gate, const OptTensor& scale, const OptTensor& next, double eps,
                               int64_t n_dtype) {
    const NormCall k{x, value(delta), value(post), value(gate), value(scale), value(next), eps, (at::ScalarType)n_dtype};
    NormOut o = norm_forward(k, true);
    ctx->save_for_backward({k.x, k.delta, k.post, k.gate, k.scale, k.next, o.stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["n_dtype"] = n_dtype;
    ctx->set_materialize_grads(false);
    variable_list out;
    if (o.h.defined()) out.push_back(o.h);
    if (o.n.defined()) out.push_back(o.n);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("norm");
    const auto s = ctx->get_saved_variables();
    NormCall k{s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["eps"].toDouble(),
               (at::ScalarType)ctx->saved_data["n_dtype"].toInt()};
    const Tensor stats = s[6];
    Tensor dh, dn;
    if (k.delta.defined()) dh = grads[0];
    if (k.next.defined()) dn = grads[k.delta.defined() ? 1 : 0];
    variable_list out(8);
    if (!dh.defined() && !dn.defined()) return out;
    const c10::cuda::CUDAGuard guard(k.x.device());
    Tensor dx = like(k.x), dd = like(k.delta), dpost = like(k.post), dgate = like(k.gate), dnext;
    if (k.next.defined()) dnext = dn.defined() ? like(k.next) : at::zeros_like(k.next);
    if (!dn.defined()) k.next = Tensor();
    if (k.x.numel() == 0) {
      for (Tensor* t : {&dpost, &dgate, &dnext})
        if (t->defined()) t->zero_();
    } else {
      dh = dense(dh);
      dn = dense(dn);
      const int64_t rows = stats.size(1);
      ow_norm_t a = k.args();
      a.rstd_delta = (float*)ptr(stats);
      a.rstd_h = a.rstd_delta + rows;
      const size_t size = ow_norm_bwd_workspace_size(&a);
      const Tensor ws = at::empty({(int64_t)size}, k.x.options().dtype(at::kByte));
      a.workspace = ptr(ws);
      a.workspace_bytes = size;
      const ow_norm_grads_t g{ptr(dh), ptr(dn), ptr(dx), ptr(dd), ptr(dpost), ptr(dgate), dn.defined() ? ptr(dnext) : nullptr};
      check_status(ow_norm_bwd(&a, &g, stream_of(k.x)), "ow_norm_bwd");
    }
    out[0] = dx;
    out[1] = dd;
    out[2] = dpost;
    out[3] = dgate;
    out[5] = dnext;
    return out;
  }
};

at::ScalarType norm_out(const Tensor& x, const std::optional<at::ScalarType>& asked) {
  const at::ScalarType t = asked ? *asked : at::autocast::is_autocast_enabled(at::kCUDA) ? at::autocast::get_autocast_dtype(at::kCUDA) : x.scalar_type();
  TORCH_CHECK(is_float(t), "norm not supported: unsupported dtype ", dtype_text(t));
  return t;
}

// The C structs hold a row's length in 32 bits.
constexpr int64_t MOST = (int64_t)1 << 30;

void check_vector(const char* name, const Tensor& w, int64_t c) {
  OW_VALUE(w.dim() == 1 && w.size(0) == c, name, " must be [", c, "], got ", shape_text(w.sizes()));
}

variable_list norm_call(const Tensor& x, const Tensor& delta, const Tensor& post, const Tensor& gate, const Tensor& scale,
                        const Tensor& next, double eps, at::ScalarType n_dtype) {
  if (wants_grad({x, delta, post, gate, next}))
    return NormFn::apply(dense(x), maybe(dense(delta)), maybe(dense(post)), maybe(dense(gate)), maybe(scale),
                         maybe(dense(next)), eps, (int64_t)n_dtype);
  NormOut o = norm_forward(NormCall{dense(x), dense(delta), dense(post), dense(gate), scale, dense(next), eps, n_dtype}, false);
  variable_list out;
  if (o.h.defined()) out.push_back(o.h);
  if (o.n.defined()) out.push_back(o.n);
  return out;
}

Tensor rms_norm(const Tensor& x, const Tensor& weight, double eps, std::optional<at::ScalarType> out_dtype) {
  OW_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must be [..., C], got ", shape_text(x.sizes()));
  OW_VALUE(x.size(-1) < MOST, "x has too many channels: ", x.size(-1));
  OW_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
  check_vector("weight", weight, x.size(-1));
  no_tangents("norm", {x, weight});
  if (auto why = unsupported(x, {weight})) TORCH_CHECK(false, "norm not supported: ", *why);
  return norm_call(x, Tensor(), Tensor(), Tensor(), Tensor(), weight, eps, norm_out(x, out_dtype))[0];
}

variable_list norm_residual(const Tensor& x, const Tensor& delta, const Tensor& weight, const OptTensor& gate_,
                            const OptTensor& scale_, const OptTensor& next_, double eps,
                            std::optional<at::ScalarType> out_dtype) {
  OW_VALUE(x.dim() >= 2 && x.size(-1) > 0, "x must be [B, ..., C], got ", shape_text(x.sizes()));
  OW_VALUE(x.size(-1) < MOST, "x has too many channels: ", x.size(-1));
  OW_VALUE(delta.sizes() == x.sizes(), "delta must be ", shape_text(x.sizes()), ", got ", shape_text(delta.sizes()));
  OW_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
  const Tensor gate = value(gate_), next = value(next_);
  Tensor scale = value(scale_);
  const int64_t b = x.size(0), c = x.size(-1);
  check_vector("weight", weight, c);
  if (next.defined()) check_vector("next_weight", next, c);
  if (gate.defined())
    OW_VALUE((gate.dim() == 1 && gate.size(0) == c) || (gate.dim() == 2 && gate.size(0) == b && gate.size(1) == c),
                      "gate must be [", c, "] or [", b, ", ", c, "], got ", shape_text(gate.sizes()));
  if (scale.defined()) {
    OW_VALUE(scale.dim() == 1 && scale.size(0) == b, "sample_scale must be [", b, "], got ", shape_text(scale.sizes()));
    OW_VALUE(!scale.requires_grad(), "sample_scale takes no gradient");
  }
  no_tangents("norm", {x, delta, weight, gate, scale, next});
  if (auto why = unsupported(x, {delta, weight, gate, next})) TORCH_CHECK(false, "norm not supported: ", *why);
  if (scale.defined()) {
    TORCH_CHECK(scale.device() == x.device(), "norm not supported: tensors on ", x.device(), " and ", scale.device());
    scale = scale.to(at::kFloat).contiguous();
  }
  return norm_call(x, delta, weight, gate, scale, next, eps, norm_out(x, out_dtype));
}

// ------------------------------------------------------------------ layer norm
ow_layernorm_t layernorm_args(const Tensor& x, const Tensor& w, const Tensor& b, double eps, at::ScalarType n_dtype,
                              const Tensor& stats) {
  ow_layernorm_t a{};
  a.channels = (int32_t)x.size(-1);
  a.rows = x.numel() / a.channels;
  a.x = ptr(x);
  a.x_dtype = code(x.scalar_type());
  a.weight = ptr(w);
  a.weight_dtype = code(w.scalar_type());
  if (b.defined()) {
    a.bias = ptr(b);
    a.bias_dtype = code(b.scalar_type());
  }
  a.eps = eps;
  a.n_dtype = code(n_dtype);
  if (stats.defined()) {
    a.mean = (float*)ptr(stats);
    a.rstd = a.mean + a.rows;
  }
  return a;
}

// n, and the rows' means and inverse deviations [2, rows] when ``keep``.
std::pair<Tensor, Tensor> layernorm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, at::ScalarType n_dtype,
                                            bool keep) {
  const Tensor n = at::empty(x.sizes(), x.options().dtype(n_dtype));
  Tensor stats;
  if (x.numel() == 0) return {n, stats};
  const c10::cuda::CUDAGuard guard(x.device());
  if (keep) stats = at::empty({2, x.numel() / x.size(-1)}, x.options().dtype(at::kFloat));
  ow_layernorm_t a = layernorm_args(x, w, b, eps, n_dtype, stats);
  a.n = ptr(n);
  check_status(ow_layernorm_fwd(&a, stream_of(x)), "ow_layernorm_fwd");
  return {n, stats};
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b, double eps, int64_t n_dtype) {
    auto [n, stats] = layernorm_forward(x, w, value(b), eps, (at::ScalarType)n_dtype, true);
    ctx->save_for_backward({x, w, value(b), stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["n_dtype"] = n_dtype;
    return n;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("layer_norm");
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &b = s[2], &stats = s[3];
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) dx = like(x);
    if (ctx->needs_input_grad(1)) dw = like(w);
    if (b.defined() && ctx->needs_input_grad(2)) db = like(b);
    if (x.numel() == 0) {
      for (Tensor* t : {&dw, &db})
        if (t->defined()) t->zero_();
    } else {
      const Tensor dn = dense(grads[0]);
      ow_layernorm_t a = layernorm_args(x, w, b, ctx->saved_data["eps"].toDouble(), (at::ScalarType)ctx->saved_data["n_dtype"].toInt(), stats);
      const size_t size = ow_layernorm_bwd_workspace_size(&a);
      const Tensor ws = at::empty({(int64_t)size}, x.options().dtype(at::kByte));
      a.workspace = ptr(ws);
      a.workspace_bytes = size;
      const ow_layernorm_grads_t g{ptr(dn), ptr(dx), ptr(dw), ptr(db)};
      check_status(ow_layernorm_bwd(&a, &g, stream_of(x)), "ow_layernorm_bwd");
    }
    out[0] = dx;
    out[1] = dw;
    out[2] = db;
    return out;
  }
};

Tensor layer_norm(const Tensor& x0, const Tensor& w0, const OptTensor& b_, double eps, std::optional<at::ScalarType> out_dtype) {
  const Tensor b0 = value(b_);
  OW_VALUE(x0.dim() >= 1 && x0.size(-1) > 0, "x must be [..., C], got ", shape_text(x0.sizes()));
  OW_VALUE(x0.size(-1) < MOST, "x has too many channels: ", x0.size(-1));
  OW_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
  check_vector("weight", w0, x0.size(-1));
  if (b0.defined()) check_vector("bias", b0, x0.size(-1));
  no_tangents("layer_norm", {x0, w0, b0});
  if (auto why = unsupported(x0, {w0, b0})) TORCH_CHECK(false, "layer_norm not supported: ", *why);
  const at::ScalarType t = norm_out(x0, out_dtype);
  const Tensor x = dense(x0), w = dense(w0), b = dense(b0);
  if (wants_grad({x, w, b})) return LayerNormFn::apply(x, w, maybe(b), eps, (int64_t)t);
  return layernorm_forward(x, w, b, eps, t, false).first;
}

// ------------------------------------------------------------------ linear
// ``t`` as a matrix whose rows lie densely, copied only if they do not.
Tensor as_rows(const Tensor& t0) {
  if (!t0.defined()) return t0;
  Tensor t = t0.dim() == 2 ? t0 : t0.reshape({-1, t0.size(-1)});
  if ((t.stride(1) != 1 && t.size(1) > 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) t = t.contiguous();
  return t;
}
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
Tensor cast(const Tensor& t, at::ScalarType to) { return t.defined() && t.scalar_type() != to ? t.to(to) : t; }

ow_linear_t linear_args(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res, int act) {
  ow_linear_t a{};
  a.rows = x.size(0);
  a.in_features = (int32_t)x.size(1);
  a.out_features = (int32_t)w.size(0);
  a.dtype = code(w.scalar_type());
  a.activation = act;
  a.x = ptr(x);
  a.ldx = ld(x);
  a.weight = ptr(w);
  a.ldw = ld(w);
  if (bias.defined()) {
    a.bias = ptr(bias);
    a.bias_dtype = code(bias.scalar_type());
  }
  if (res.defined()) {
    a.residual = ptr(res);
    a.ldr = ld(res);
  }
  return a;
}

Tensor linear_workspace(ow_linear_t* a, const ow_linear_grads_t* g, const Tensor& x) {
  const size_t size = ow_linear_workspace_size(a, g);
  TORCH_CHECK(size > 0, "ow_linear_workspace_size failed: ", ow_last_error());
  const Tensor ws = at::empty({(int64_t)size}, x.options().dtype(at::kByte));
  a->workspace = ptr(ws);
  a->workspace_bytes = size;
  return ws;
}

std::vector<int64_t> out_shape(const Tensor& x, int64_t n) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = n;
  return s;
}

// y, in ``shape``, and z when ``keep`` and the backward needs it.
std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res, int act,
                                         bool keep, at::IntArrayRef shape) {
  const int64_t m = x.size(0), n = w.size(0);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor y = at::empty(shape, x.options());
  Tensor z;
  if (keep && act != OW_ACT_NONE) z = at::empty({m, (n + 7) / 8 * 8}, x.options());
  if (m > 0) {
    ow_linear_t a = linear_args(x, w, bias, res, act);
    a.out = ptr(y);
    a.z = ptr(z);
    const Tensor ws = linear_workspace(&a, nullptr, x);
    check_status(ow_linear_fwd(&a, stream_of(x)), "ow_linear_fwd");
  }
  return {y, z};
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_, const OptTensor& res_,
                        int64_t act, int64_t compute) {
    const Tensor bias = value(bias_), res = value(res_);
    const auto t = (at::ScalarType)compute;
    const Tensor xm = as_rows(cast(x, t)), wm = as_rows(cast(w, t));
    auto [y, z] = linear_forward(xm, wm, bias, as_rows(cast(res, t)), (int)act, true, out_shape(x, w.size(0)));
    ctx->save_for_backward({xm, wm, bias, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["x_shape"] = x.sizes().vec();
    ctx->saved_data["x_type"] = (int64_t)x.scalar_type();
    ctx->saved_data["w_type"] = (int64_t)w.scalar_type();
    ctx->saved_data["r_type"] = res.defined() ? (int64_t)res.scalar_type() : (int64_t)-1;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("linear");
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &bias = s[2], &z = s[3];
    const auto x_type = (at::ScalarType)ctx->saved_data["x_type"].toInt();
    const auto w_type = (at::ScalarType)ctx->saved_data["w_type"].toInt();
    const int64_t r_type = ctx->saved_data["r_type"].toInt();
    variable_list out(6);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    const c10::cuda::CUDAGuard guard(x.device());
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = bias.defined() && ctx->needs_input_grad(2);  // edges of the tensors that were given
    if (r_type >= 0 && ctx->needs_input_grad(bias.defined() ? 3 : 2)) out[3] = cast(dy, (at::ScalarType)r_type);
    if (!need_x && !need_w && !need_b) return out;
    const Tensor g = cast(dy, x.scalar_type()).reshape({-1, w.size(0)}).contiguous();
    Tensor dx, dw, db;
    if (need_x) dx = at::empty({x.size(0), x.size(1)}, x.options());
    if (need_w) dw = at::empty({w.size(0), w.size(1)}, x.options().dtype(w_type == at::kFloat ? at::kFloat : x.scalar_type()));
    if (need_b) db = at::empty(bias.sizes(), bias.options());
    if (g.numel() == 0) {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
    } else {
      ow_linear_t a = linear_args(x, w, bias, Tensor(), (int)ctx->saved_data["act"].toInt());
      a.z = ptr(z);
      const ow_linear_grads_t k{ptr(g), ptr(dx), ptr(dw), dw.defined() ? code(dw.scalar_type()) : 0, ptr(db)};
      const Tensor ws = linear_workspace(&a, &k, x);
      check_status(ow_linear_bwd(&a, &k, stream_of(x)), "ow_linear_bwd");
    }
    if (need_x) out[0] = cast(dx, x_type).view(ctx->saved_data["x_shape"].toIntVector());
    if (need_w) out[1] = cast(dw, w_type);
    out[2] = db;
    return out;
  }
};

at::ScalarType linear_compute(const Tensor& x) {
  return at::autocast::is_autocast_enabled(at::kCUDA) ? at::autocast::get_autocast_dtype(at::kCUDA) : x.scalar_type();
}

std::optional<std::string> linear_unsupported(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res) {
  if (!x.is_cuda()) return "CUDA is unavailable";
  const at::ScalarType t = linear_compute(x);
  if (!is16(t)) return "compute dtype " + dtype_text(t) + " is not 16-bit";
  if (auto why = unsupported(x, {w, bias, res})) return why;
  if (!at::autocast::is_autocast_enabled(at::kCUDA) && (w.scalar_type() != t || (res.defined() && res.scalar_type() != t)))
    return "weight and residual must be " + dtype_text(t) + " without autocast";
  return std::nullopt;
}

Tensor linear(const Tensor& x, const Tensor& w, const OptTensor& bias_, int64_t act, const OptTensor& res_) {
  const Tensor res = value(res_);
  Tensor bias = value(bias_);
  OW_VALUE(w.dim() == 2 && w.numel() > 0, "weight must be [N, K], got ", shape_text(w.sizes()));
  const int64_t n = w.size(0), kk = w.size(1);
  OW_VALUE(n < MOST && kk < MOST, "weight is too large: ", shape_text(w.sizes()));
  OW_VALUE(x.dim() >= 1 && x.size(-1) == kk, "x must be [..., ", kk, "], got ", shape_text(x.sizes()));
  if (bias.defined())
    OW_VALUE(bias.dim() == 1 && bias.size(0) == n, "bias must be [", n, "], got ", shape_text(bias.sizes()));
  const auto shape = out_shape(x, n);
  if (res.defined())
    OW_VALUE(res.sizes() == at::IntArrayRef(shape), "residual must be ", shape_text(shape), ", got ", shape_text(res.sizes()));
  no_tangents("linear", {x, w, bias, res});
  if (auto why = linear_unsupported(x, w, bias, res)) TORCH_CHECK(false, "linear not supported: ", *why);
  const at::ScalarType t = linear_compute(x);
  bias = dense(bias);
  if (wants_grad({x, w, bias, res})) return LinearFn::apply(x, w, maybe(bias), maybe(res), act, (int64_t)t);
  return linear_forward(as_rows(cast(x, t)), as_rows(cast(w, t)), bias, as_rows(cast(res, t)), (int)act, false, shape).first;
}

// ------------------------------------------------------------------ gated feed-forward
struct FfnCall {
  Tensor x, wg, wu, wd, bg, bu, bd;  // matrices of the compute type, their rows dense
  int act;

  ow_ffn_t args() const {
    ow_ffn_t a{};
    a.rows = x.size(0);
    a.in_features = (int32_t)x.size(1);
    a.hidden = (int32_t)wg.size(0);
    a.out_features = (int32_t)wd.size(0);
    a.dtype = code(wg.scalar_type());
    a.activation = act;
    a.x = ptr(x);
    a.ldx = ld(x);
    a.gate_weight = ptr(wg);
    a.ldg = ld(wg);
    a.up_weight = ptr(wu);
    a.ldu = ld(wu);
    a.down_weight = ptr(wd);
    a.ldd = ld(wd);
    auto bias = [](const Tensor& b, const void** p, int32_t* dt) {
      if (!b.defined()) return;
      *p = ptr(b);
      *dt = code(b.scalar_type());
    };
    bias(bg, &a.gate_bias, &a.gate_bias_dtype);
    bias(bu, &a.up_bias, &a.up_bias_dtype);
    bias(bd, &a.down_bias, &a.down_bias_dtype);
    return a;
  }

  Tensor workspace(ow_ffn_t* a, const ow_ffn_grads_t* g) const {
    const size_t size = ow_ffn_workspace_size(a, g);
    TORCH_CHECK(size > 0, "ow_ffn_workspace_size failed: ", ow_last_error());
    const Tensor ws = at::empty({(int64_t)size}, x.options().dtype(at::kByte));
    a->workspace = ptr(ws);
    a->workspace_bytes = size;
    return ws;
  }
};

struct FfnOut {
  Tensor y, h, act, slope;  // the last two for the backward
};

FfnOut ffn_forward(const FfnCall& k, const Tensor& res, bool keep, at::IntArrayRef shape) {
  const c10::cuda::CUDAGuard guard(k.x.device());
  const int64_t m = k.x.size(0), f = (k.wg.size(0) + 7) / 8 * 8;
  FfnOut o;
  o.y = at::empty(shape, k.x.options());
  if (m == 0) return o;
  o.h = at::empty({m, f}, k.x.options());
  if (keep) {
    o.act = at::empty({m, f}, k.x.options());
    o.slope = at::empty({m, f}, k.x.options());
  }
  ow_ffn_t a = k.args();
  if (res.defined()) {
    a.residual = ptr(res);
    a.ldr = ld(res);
  }
  a.out = ptr(o.y);
  a.h = ptr(o.h);
  a.act = ptr(o.act);
  a.slope = ptr(o.slope);
  const Tensor ws = k.workspace(&a, nullptr);
  check_status(ow_ffn_fwd(&a, stream_of(k.x)), "ow_ffn_fwd");
  return o;
}

struct FfnFn : torch::autograd::Function<FfnFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                        const OptTensor& bg, const OptTensor& bu, const OptTensor& bd, const OptTensor& res_, int64_t act,
                        int64_t compute) {
    const auto t = (at::ScalarType)compute;
    const Tensor res = value(res_);
    const FfnCall k{as_rows(cast(x, t)), as_rows(cast(wg, t)), as_rows(cast(wu, t)), as_rows(cast(wd, t)), value(bg), value(bu), value(bd),
                    (int)act};
    auto needs = [](const Tensor& v) { return v.defined() && v.requires_grad(); };
    // the projection back's own gradients take h alone
    const bool keep = needs(x) || needs(wg) || needs(wu) || needs(k.bg) || needs(k.bu);
    FfnOut o = ffn_forward(k, as_rows(cast(res, t)), keep, out_shape(x, wd.size(0)));
    ctx->save_for_backward({k.x, k.wg, k.wu, k.wd, k.bg, k.bu, k.bd, o.h, o.act, o.slope});
    ctx->saved_data["act"] = act;
    ctx->saved_data["x_shape"] = x.sizes().vec();
    std::vector<int64_t> types;
    for (const Tensor& v : {x, wg, wu, wd}) types.push_back((int64_t)v.scalar_type());
    types.push_back(res.defined() ? (int64_t)res.scalar_type() : (int64_t)-1);
    ctx->saved_data["types"] = types;
    return o.y;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("gated_feed_forward");
    const auto s = ctx->get_saved_variables();
    const FfnCall k{s[0], s[1], s[2], s[3], s[4], s[5], s[6], (int)ctx->saved_data["act"].toInt()};
    const std::vector<int64_t> types = ctx->saved_data["types"].toIntVector();
    variable_list out(10);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    const c10::cuda::CUDAGuard guard(k.x.device());
    // edges of the tensors that were given: those that were not have none
    bool need[8];
    for (int i = 0, edge = 0; i < 8; ++i) {
      const bool given = i < 4 || (i < 7 ? s[i].defined() : types[4] >= 0);
      need[i] = given && ctx->needs_input_grad(edge);
      edge += given;
    }
    if (need[7]) out[7] = cast(dy, (at::ScalarType)types[4]);
    if (!std::any_of(need, need + 7, [](bool b) { return b; })) return out;
    const Tensor g = cast(dy, k.x.scalar_type()).reshape({-1, k.wd.size(0)}).contiguous();
    auto type_of = [&](int i) { return types[i] == (int64_t)at::kFloat ? at::kFloat : k.x.scalar_type(); };
    Tensor d[7];
    if (need[0]) d[0] = at::empty({k.x.size(0), k.x.size(1)}, k.x.options());
    if (need[1] || need[2]) {  // they come together, in f32 if either wants it
      const auto t = type_of(1) == at::kFloat ? at::kFloat : type_of(2);
      for (int i : {1, 2}) d[i] = at::empty(k.wg.sizes(), k.x.options().dtype(t));
    }
    if (need[3]) d[3] = at::empty(k.wd.sizes(), k.x.options().dtype(type_of(3)));
    for (int i = 4; i < 7; ++i)
      if (need[i]) d[i] = at::empty(s[i].sizes(), s[i].options());
    if (k.x.size(0) == 0) {
      for (Tensor& t : d)
        if (t.defined()) t.zero_();
    } else {
      ow_ffn_t a = k.args();
      a.h = ptr(s[7]);
      a.act = ptr(s[8]);
      a.slope = ptr(s[9]);
      auto dt = [](const Tensor& t) { return t.defined() ? code(t.scalar_type()) : 0; };
      const ow_ffn_grads_t gr{ptr(g), ptr(d[0]), ptr(d[1]), dt(d[1]), ptr(d[2]), dt(d[2]), ptr(d[3]), dt(d[3]), ptr(d[4]), ptr(d[5]), ptr(d[6])};
      const Tensor ws = k.workspace(&a, &gr);
      check_status(ow_ffn_bwd(&a, &gr, stream_of(k.x)), "ow_ffn_bwd");
    }
    if (need[0]) out[0] = cast(d[0], (at::ScalarType)types[0]).view(ctx->saved_data["x_shape"].toIntVector());
    for (int i = 1; i < 4; ++i)
      if (need[i]) out[i] = cast(d[i], (at::ScalarType)types[i]);
    for (int i = 4; i < 7; ++i) out[i] = d[i];
    return out;
  }
};

std::optional<std::string> ffn_unsupported(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const Tensor& bg,
                                           const Tensor& bu, const Tensor& bd, const Tensor& res) {
  if (!x.is_cuda()) return "CUDA is unavailable";
  const at::ScalarType t = linear_compute(x);
  if (!is16(t)) return "compute dtype " + dtype_text(t) + " is not 16-bit";
  if (auto why = unsupported(x, {wg, wu, wd, bg, bu, bd, res})) return why;
  if (!at::autocast::is_autocast_enabled(at::kCUDA))
    for (const Tensor& v : {wg, wu, wd, res})
      if (v.defined() && v.scalar_type() != t) return "weights and residual must be " + dtype_text(t) + " without autocast";
  return std::nullopt;
}

Tensor gated_feed_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const OptTensor& bg_,
                          const OptTensor& bu_, const OptTensor& bd_, int64_t act, const OptTensor& res_) {
  const Tensor bg = dense(value(bg_)), bu = dense(value(bu_)), bd = dense(value(bd_)), res = value(res_);
  OW_VALUE(wg.dim() == 2 && wg.numel() > 0, "gate_weight must be [F, K], got ", shape_text(wg.sizes()));
  const int64_t f = wg.size(0), kk = wg.size(1);
  OW_VALUE(wu.sizes() == wg.sizes(), "up_weight must be ", shape_text(wg.sizes()), ", got ", shape_text(wu.sizes()));
  OW_VALUE(wd.dim() == 2 && wd.size(0) > 0 && wd.size(1) == f, "down_weight must be [N, ", f, "], got ", shape_text(wd.sizes()));
  const int64_t n = wd.size(0);
  OW_VALUE(n < MOST && kk < MOST && f < MOST / 2, "weights are too large: ", shape_text(wg.sizes()), ", ", shape_text(wd.sizes()));
  OW_VALUE(x.dim() >= 1 && x.size(-1) == kk, "x must be [..., ", kk, "], got ", shape_text(x.sizes()));
  if (bg.defined()) check_vector("gate_bias", bg, f);
  if (bu.defined()) check_vector("up_bias", bu, f);
  if (bd.defined()) check_vector("down_bias", bd, n);
  const auto shape = out_shape(x, n);
  if (res.defined())
    OW_VALUE(res.sizes() == at::IntArrayRef(shape), "residual must be ", shape_text(shape), ", got ", shape_text(res.sizes()));
  no_tangents("gated_feed_forward", {x, wg, wu, wd, bg, bu, bd, res});
  if (auto why = ffn_unsupported(x, wg, wu, wd, bg, bu, bd, res)) TORCH_CHECK(false, "gated_feed_forward not supported: ", *why);
  const at::ScalarType t = linear_compute(x);
  if (wants_grad({x, wg, wu, wd, bg, bu, bd, res}))
    return FfnFn::apply(x, wg, wu, wd, maybe(bg), maybe(bu), maybe(bd), maybe(res), act, (int64_t)t);
  const FfnCall k{as_rows(cast(x, t)), as_rows(cast(wg, t)), as_rows(cast(wu, t)), as_rows(cast(wd, t)), bg, bu, bd, (int)act};
  return ffn_forward(k, as_rows(cast(res, t)), false, shape).y;
}

// ------------------------------------------------------------------ distillation
struct DistillCall {
  Tensor logits, top, classes, labels;  // [N, V] (rows may lie apart), [N, K], [N, K], [N]
  double temperature, weight;
  int reduction;

  ow_distill_t args(const Tensor& stats, const Tensor& factors) const {
    ow_distill_t a{};
    a.rows = logits.size(0);
    a.classes = (int32_t)logits.size(1);
    a.top = (int32_t)top.size(1);
    a.logits = ptr(logits);
    a.dtype = code(logits.scalar_type());
    a.ld = ld(logits);
    a.top_logits = ptr(top);
    a.top_dtype = code(top.scalar_type());
    a.top_classes = ptr(classes);
    a.class_bytes = (int32_t)classes.element_size();
    if (labels.defined()) {
      a.labels = ptr(labels);
      a.label_bytes = (int32_t)labels.element_size();
    }
    a.temperature = temperature;
    a.weight = weight;
    a.reduction = reduction;
    a.stats = (float*)ptr(stats);
    a.factors = (float*)ptr(factors);
    return a;
  }
};

// The loss, and what the backward takes: the rows' sums and the terms' factors.
std::tuple<Tensor, Tensor, Tensor> distill_forward(const DistillCall& k, at::IntArrayRef shape) {
  const auto f32 = k.logits.options().dtype(at::kFloat);
  const int64_t rows = k.logits.size(0);
  if (rows == 0) return {at::zeros(shape, f32), Tensor(), Tensor()};
  const c10::cuda::CUDAGuard guard(k.logits.device());
  const Tensor loss = at::empty(shape, f32), stats = at::empty({5, rows}, f32);
  Tensor factors;
  if (k.reduction != OW_REDUCE_NONE) factors = at::empty({2}, f32);
  ow_distill_t a = k.args(stats, factors);
  a.loss = (float*)ptr(loss);
  const size_t size = ow_distill_workspace_size(&a);
  const Tensor ws = at::empty({(int64_t)size}, f32.dtype(at::kByte));
  a.workspace = ptr(ws);
  a.workspace_bytes = size;
  check_status(ow_distill_fwd(&a, stream_of(k.logits)), "ow_distill_fwd");
  return {loss, stats, factors};
}

struct DistillFn : torch::autograd::Function<DistillFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& top, const Tensor& classes, const OptTensor& labels,
                        double temperature, double weight, int64_t reduction, std::vector<int64_t> shape) {
    const DistillCall k{as_rows(logits), top, classes, value(labels), temperature, weight, (int)reduction};
    auto [loss, stats, factors] = distill_forward(k, shape);
    ctx->save_for_backward({k.logits, top, classes, k.labels, stats, factors});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["weight"] = weight;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["shape"] = logits.sizes().vec();
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("distill_loss");
    const auto s = ctx->get_saved_variables();
    variable_list out(8);
    if (!grads[0].defined() || !ctx->needs_input_grad(0)) return out;
    const DistillCall k{s[0], s[1], s[2], s[3], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["weight"].toDouble(),
                        (int)ctx->saved_data["reduction"].toInt()};
    const c10::cuda::CUDAGuard guard(k.logits.device());
    const Tensor dz = at::empty(ctx->saved_data["shape"].toIntVector(), k.logits.options());
    if (dz.numel() > 0) {
      const Tensor g = grads[0].to(at::kFloat).contiguous();
      const ow_distill_t a = k.args(s[4], s[5]);
      const ow_distill_grads_t d{(const float*)ptr(g), ptr(dz)};
      check_status(ow_distill_bwd(&a, &d, stream_of(k.logits)), "ow_distill_bwd");
    }
    out[0] = dz;
    return out;
  }
};

Tensor distill_loss(const Tensor& logits, const Tensor& top0, const Tensor& classes0, const OptTensor& labels_, double temperature,
                    double weight, int64_t reduction) {
  const Tensor labels0 = value(labels_);
  auto whole = [](const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; };
  OW_VALUE(logits.dim() >= 1 && logits.size(-1) > 0, "logits must be [..., V], got ", shape_text(logits.sizes()));
  OW_VALUE(logits.size(-1) < MOST, "logits has too many classes: ", logits.size(-1));
  OW_VALUE(top0.dim() == logits.dim() && top0.size(-1) > 0 && top0.sizes().slice(0, logits.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
           "top_logits must be ", shape_text(logits.sizes().slice(0, logits.dim() - 1)), " + (K,), got ", shape_text(top0.sizes()));
  OW_VALUE(classes0.sizes() == top0.sizes(), "top_classes must be ", shape_text(top0.sizes()), ", got ", shape_text(classes0.sizes()));
  OW_VALUE(whole(classes0), "top_classes must be int32 or int64, got ", dtype_text(classes0.scalar_type()));
  if (labels0.defined()) {
    OW_VALUE(labels0.sizes() == logits.sizes().slice(0, logits.dim() - 1), "labels must be ",
             shape_text(logits.sizes().slice(0, logits.dim() - 1)), ", got ", shape_text(labels0.sizes()));
    OW_VALUE(whole(labels0), "labels must be int32 or int64, got ", dtype_text(labels0.scalar_type()));
  }
  OW_VALUE(temperature >= 1e-4 && temperature <= 1e4, "temperature must be 1e-4 to 1e4, got ", temperature);
  OW_VALUE(weight >= 0.0 && weight <= 1.0, "weight must be 0 to 1, got ", weight);
  OW_VALUE(!top0.requires_grad() || !at::GradMode::is_enabled(), "top_logits takes no gradient");
  no_tangents("distill_loss", {logits, top0});
  if (auto why = unsupported(logits, {top0})) TORCH_CHECK(false, "distill_loss not supported: ", *why);
  for (const Tensor& t : {classes0, labels0})
    TORCH_CHECK(!t.defined() || t.device() == logits.device(), "distill_loss not supported: tensors on ", logits.device(), " and ", t.device());
  const int64_t kk = top0.size(-1);
  TORCH_CHECK(kk <= 1024, "distill_loss not supported: at most 1024 entries a row, got ", kk);
  const Tensor top = dense(top0).view({-1, kk}), classes = dense(classes0).view({-1, kk});
  const Tensor labels = labels0.defined() ? dense(labels0).view({-1}) : labels0;
  std::vector<int64_t> shape;
  if (reduction == OW_REDUCE_NONE) shape = logits.sizes().slice(0, logits.dim() - 1).vec();
  if (wants_grad({logits}))
    return DistillFn::apply(logits, top, classes, maybe(labels), temperature, weight, reduction, shape);
  return std::get<0>(distill_forward(DistillCall{as_rows(logits), top, classes, labels, temperature, weight, (int)reduction}, shape));
}

// ------------------------------------------------------------------ AdamW
// The parameters of one bucket as they were added, and the arguments of its
// calls (an ow_adamw_t and the arrays it points to, which the optimizer owns).
struct Bucket {
  std::vector<Tensor> params;
  std::vector<std::vector<int64_t>> sizes, strides;
  at::ScalarType dtype;
  at::Device device;
  ow_adamw_t* args;
  void** p;
  void** g;
  int32_t partials;
  std::vector<Tensor> copied;  // gradients of this step in other strides than their parameters'

  Bucket(std::vector<Tensor> ps, uintptr_t args_, uintptr_t p_, uintptr_t g_)
      : params(std::move(ps)), dtype(params.at(0).scalar_type()), device(params.at(0).device()),
        args(reinterpret_cast<ow_adamw_t*>(args_)), p(reinterpret_cast<void**>(p_)), g(reinterpret_cast<void**>(g_)),
        partials(ow_grad_norm_partials(args)) {
    for (const Tensor& t : params) {
      sizes.push_back(t.sizes().vec());
      strides.push_back(t.strides().vec());
    }
  }

  // Writes down where the parameters and gradients are now; false if no parameter has a gradient.
  bool gather() {
    bool some = false;
    for (size_t i = 0; i < params.size(); ++i) {
      const Tensor& t = params[i];
      TORCH_CHECK(t.scalar_type() == dtype && t.device() == device && t.layout() == at::kStrided &&
                      t.sizes() == at::IntArrayRef(sizes[i]) && t.strides() == at::IntArrayRef(strides[i]),
                  "a parameter moved to another device, dtype or layout since it was added to AdamW");
      p[i] = t.data_ptr();
      Tensor d = t.grad();
      if (!d.defined()) {
        g[i] = nullptr;
        continue;
      }
      TORCH_CHECK(d.layout() == at::kStrided, "AdamW does not support sparse gradients");
      TORCH_CHECK(d.scalar_type() == dtype && d.device() == device && d.sizes() == at::IntArrayRef(sizes[i]),
                  "a gradient has another dtype, device or size than its parameter");
      if (d.strides() != at::IntArrayRef(strides[i]) && d.numel() > 1) {  // dense, in the parameter's own order
        d = at::empty_strided(sizes[i], strides[i], d.options()).copy_(d.detach());
        copied.push_back(d);
      }
      g[i] = d.data_ptr();
      some = true;
    }
    return some;
  }
};

// A bucket's group: lr (or a device lr), betas, eps, weight decay.
using Hyper = std::tuple<std::variant<double, Tensor>, std::pair<double, double>, double, double>;

// One step over the buckets, with the norm of all gradients first when it is
// asked for (``partials`` given).
void adamw_step(const std::vector<Bucket*>& buckets, const std::vector<Hyper>& hyper, const OptTensor& found_,
                const OptTensor& partials_, const OptTensor& norm_, double max_norm, bool skip_nonfinite) {
  const at::NoGradGuard no_grad;
  const at::Device device = buckets.at(0)->device;
  const c10::cuda::CUDAGuard guard(device);
  const Tensor found = value(found_), partials = value(partials_);
  if (found.defined())
    OW_VALUE(found.scalar_type() == at::kFloat && found.numel() == 1 && found.device() == device,
             "found_inf must be one float32 on the parameters' device");
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  std::vector<size_t> todo;
  for (size_t i = 0; i < buckets.size(); ++i) {
    buckets[i]->copied.clear();
    if (buckets[i]->gather()) todo.push_back(i);
    if (const Tensor* lr = std::get_if<Tensor>(&std::get<0>(hyper.at(i))))
      OW_VALUE(lr->scalar_type() == at::kFloat && lr->numel() == 1 && lr->device() == device,
               "a tensor lr must be one float32 on the parameters' device");
  }
  if (partials.defined()) {
    int32_t first = 0;
    for (size_t i : todo) {
      Bucket& b = *buckets[i];
      b.args->control = buckets[0]->args->control;
      ow_grad_norm_t o{};
      o.partials = (double*)ptr(partials);
      o.first = first;
      o.capacity = (int32_t)partials.numel();
      o.finish = i == todo.back();
      o.max_norm = (float)max_norm;
      o.skip_nonfinite = skip_nonfinite;
      o.norm = (float*)ptr(value(norm_));
      o.found = (float*)ptr(found);
      check_status(ow_grad_norm(b.args, &o, stream), "ow_grad_norm");
      first += b.partials;
    }
  }
  for (size_t i : todo) {
    Bucket& b = *buckets[i];
    const auto& [lr, betas, eps, decay] = hyper.at(i);
    ow_adamw_t& a = *b.args;
    a.lr = std::holds_alternative<double>(lr) ? std::get<double>(lr) : 0.0;
    a.lr_ptr = std::holds_alternative<Tensor>(lr) ? (const float*)ptr(std::get<Tensor>(lr)) : nullptr;
    a.beta1 = betas.first;
    a.beta2 = betas.second;
    a.eps = eps;
    a.weight_decay = decay;
    a.found = (const float*)ptr(found);
    a.use_norm = partials.defined();
    a.control = buckets[0]->args->control;
    check_status(ow_adamw_step(&a, stream), "ow_adamw_step");
    // The kernel wrote the parameters: autograd nodes that saved one as it was before must not take it as it is now.
    for (size_t k = 0; k < b.params.size(); ++k)
      if (b.g[k] && !b.params[k].is_inference()) b.params[k].unsafeGetTensorImpl()->bump_version();
  }
  for (Bucket* b : buckets) b->copied.clear();
}

std::pair<bool, std::optional<std::string>> told(const std::optional<std::string>& why) { return {!why.has_value(), why}; }

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.attr("abi_version") = OW_ABI_VERSION;
  auto nogil = py::call_guard<py::gil_scoped_release>();
  m.def("rms_norm", &rms_norm, nogil);
  m.def("norm_residual", &norm_residual, nogil);
  m.def("layer_norm", &layer_norm, nogil);
  m.def("linear", &linear, nogil);
  m.def("gated_feed_forward", &gated_feed_forward, nogil);
  m.def("distill_loss", &distill_loss, nogil);
  m.def("norm_supported", [](const Tensor& x, const std::vector<OptTensor>& more) {
    for (const OptTensor& t : more)
      if (auto why = unsupported(x, {value(t)})) return told(why);
    return told(unsupported(x, {}));
  });
  m.def("linear_supported", [](const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r) {
    return told(linear_unsupported(x, w, value(b), value(r)));
  });
  m.def("gated_feed_forward_supported",
        [](const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const OptTensor& bg, const OptTensor& bu,
           const OptTensor& bd, const OptTensor& r) { return told(ffn_unsupported(x, wg, wu, wd, value(bg), value(bu), value(bd), value(r))); });
  py::class_<Bucket>(m, "Bucket")
      .def(py::init<std::vector<Tensor>, uintptr_t, uintptr_t, uintptr_t>())
      .def_readonly("partials", &Bucket::partials);
  m.def("adamw_step", &adamw_step, nogil);
}

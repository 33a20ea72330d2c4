// Host side of the operators around the block, as a Python module
// (omniwave_b200._host): argument checks, autograd and the calls of the C ABI
// for the norms and the linear layer, and AdamW's step over its buckets.
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
  m.def("linear", &linear, nogil);
  m.def("norm_supported", [](const Tensor& x, const std::vector<OptTensor>& more) {
    for (const OptTensor& t : more)
      if (auto why = unsupported(x, {value(t)})) return told(why);
    return told(unsupported(x, {}));
  });
  m.def("linear_supported", [](const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r) {
    return told(linear_unsupported(x, w, value(b), value(r)));
  });
  py::class_<Bucket>(m, "Bucket")
      .def(py::init<std::vector<Tensor>, uintptr_t, uintptr_t, uintptr_t>())
      .def_readonly("partials", &Bucket::partials);
  m.def("adamw_step", &adamw_step, nogil);
}

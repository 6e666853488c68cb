// The operators of include/nfi_learn.h as TORCH_LIBRARY(nfi, ...) operators: the argument checks, the autograd
// functions and the optimiser's call in C++ (a small layer's forward and backward take 30 us of host time through
// Python functions and the interpreter lock; the kernels behind them 5).  nfi/norms.py, grouped.py and optim.py are
// their documented front.
//
//   nfi::residual_norm(h, residual?, gate?, weight?, bias?, next_weight?, next_bias?, norm, next_norm, slope, scale,
//                      eps) -> Tensor[]       x, or x and y
//   nfi::grouped_linear(x, weight, offsets, bias?) -> Tensor
//   nfi::orthogonalize(u, steps, a, b, c, eps) -> Tensor
//   nfi::muon_step(params, grads, momenta, ...) -> ()       in place
#include <cmath>
#include <vector>

#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/library.h>
#include <torch/torch.h>

#include "../../include/nfi_learn.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Maybe;

void check(int32_t rc, const char* what) { TORCH_CHECK(rc == 0, "nfi: ", what, " failed (", rc, "): ", nfi_last_error()); }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int32_t type_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case torch::kFloat: return NFI_F32;
    case torch::kBFloat16: return NFI_BF16;
    case torch::kHalf: return NFI_F16;
    default: TORCH_CHECK(false, what, ": float32, bfloat16 or float16 is wanted, not ", t.scalar_type());
  }
}

void on_device(const char* what, const Tensor& first) {
  TORCH_CHECK(first.is_cuda(), what, ": nfi ops run on HIP devices only (got a ", first.device(), " tensor)");
}
void with(const char* what, const char* name, const Tensor& t, const Tensor& first) {
  TORCH_CHECK(!t.defined() || t.device() == first.device(), what, ": ", name, " is on ", t.device(), ", the first input on ",
              first.device());
}

Tensor get(const Maybe& t) { return t ? *t : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(int64_t n, const Tensor& like) { return n > 0 ? torch::empty({n}, like.options().dtype(torch::kByte)) : Tensor(); }
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": there is no double backward (create_graph)");
}

// ---- residual norm -------------------------------------------------------------------------------------------------

struct NormConf {
  int64_t norm, next;
  double slope, scale, eps;
};

nfi_resnorm_args norm_args(const Tensor* in, const NormConf& c) {   // in: h, residual, gate, weight, bias, next_weight, next_bias
  nfi_resnorm_args a{};
  a.h = ptr(in[0]);
  a.residual = ptr(in[1]);
  a.gate = ptr(in[2]);
  a.weight = ptr(in[3]);
  a.bias = ptr(in[4]);
  a.next_weight = ptr(in[5]);
  a.next_bias = ptr(in[6]);
  a.rows = in[0].size(0);
  a.width = (int32_t)in[0].size(1);
  a.dtype = type_code(in[0], "residual_norm");
  a.gate_dtype = in[2].defined() ? type_code(in[2], "residual_norm") : a.dtype;
  const Tensor* p = nullptr;
  for (int k = 6; k >= 3; --k)
    if (in[k].defined()) p = &in[k];
  a.param_dtype = p ? type_code(*p, "residual_norm") : a.dtype;
  a.affine_groups = p && p->dim() == 2;
  a.groups = in[2].defined() ? in[2].size(0) : a.affine_groups ? p->size(0) : 0;
  a.norm = (int32_t)c.norm;
  a.next_norm = (int32_t)c.next;
  a.slope = (float)c.slope;
  a.scale = (float)c.scale;
  a.eps = (float)c.eps;
  return a;
}

struct ResidualNorm : public torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, Tensor h, Maybe residual_, Maybe gate_, Maybe weight_, Maybe bias_, Maybe next_weight_,
                               Maybe next_bias_, int64_t norm, int64_t next, double slope, double scale, double eps, bool train) {
    const c10::DeviceGuard guard(h.device());
    const Tensor in[7] = {h, get(residual_), get(gate_), get(weight_), get(bias_), get(next_weight_), get(next_bias_)};
    const NormConf c{norm, next, slope, scale, eps};
    Tensor x = torch::empty_like(h), y = next ? torch::empty_like(h) : Tensor(), stats;
    if (h.size(0) > 0) {
      nfi_resnorm_args a = norm_args(in, c);
      if (train) stats = torch::empty({h.size(0), 4}, h.options().dtype(torch::kFloat));
      a.x = ptr(x);
      a.y = ptr(y);
      a.stats = (float*)ptr(stats);
      check(nfi_resnorm_forward(&a, stream_of(h)), "nfi_resnorm_forward");
    }
    if (train) {
      ctx->set_materialize_grads(false);
      ctx->save_for_backward({in[0], in[1], in[2], in[3], in[4], in[5], in[6], stats});
      ctx->saved_data["norm"] = norm;
      ctx->saved_data["next"] = next;
      ctx->saved_data["slope"] = slope;
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["eps"] = eps;
    }
    if (next) return {x, y};
    return {x};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("residual_norm");
    variable_list out(13);
    const Tensor gx = dense(g[0]), gy = g.size() > 1 ? dense(g[1]) : Tensor();
    if (!gx.defined() && !gy.defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const NormConf c{ctx->saved_data["norm"].toInt(), ctx->saved_data["next"].toInt(), ctx->saved_data["slope"].toDouble(),
                     ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble()};
    const c10::DeviceGuard guard(s[0].device());
    const bool none = s[0].size(0) == 0;
    for (int k = 0, edge = 0; k < 7; ++k) {   // (the graph's edges are those of the arguments that are there)
      if (!s[k].defined() || !ctx->needs_input_grad(edge++)) continue;
      // (nothing reaches the next norm's parameters without a gradient of y)
      out[k] = none || (k >= 5 && !gy.defined()) ? torch::zeros_like(s[k]) : torch::empty_like(s[k]);
    }
    if (none) return out;
    nfi_resnorm_args a = norm_args(s.data(), c);
    a.stats = (float*)ptr(s[7]);
    a.gx = ptr(gx);
    a.gy = ptr(gy);
    a.dh = ptr(out[0]);
    a.dresidual = ptr(out[1]);
    a.dgate = ptr(out[2]);
    a.dweight = ptr(out[3]);
    a.dbias = ptr(out[4]);
    if (gy.defined()) {
      a.dnext_weight = ptr(out[5]);
      a.dnext_bias = ptr(out[6]);
    }
    const Tensor work = bytes(nfi_resnorm_work_bytes(a.rows, a.groups, a.affine_groups, a.width), s[0]);
    a.work = (float*)ptr(work);
    check(nfi_resnorm_backward(&a, stream_of(s[0])), "nfi_resnorm_backward");
    return out;
  }
};

std::vector<Tensor> residual_norm(const Tensor& h, const Maybe& residual_, const Maybe& gate_, const Maybe& weight_, const Maybe& bias_,
                                  const Maybe& next_weight_, const Maybe& next_bias_, int64_t norm, int64_t next, double slope, double scale,
                                  double eps) {
  const char* what = "residual_norm";
  Tensor residual = get(residual_), gate = get(gate_);
  Tensor p[4] = {get(weight_), get(bias_), get(next_weight_), get(next_bias_)};
  static const char* names[4] = {"weight", "bias", "next_weight", "next_bias"};
  on_device(what, h);
  with(what, "residual", residual, h);
  with(what, "gate", gate, h);
  for (int k = 0; k < 4; ++k) with(what, names[k], p[k], h);
  type_code(h, what);
  TORCH_CHECK_VALUE(norm >= 0 && norm <= 2 && next >= 0 && next <= 2, what, ": norms are 0, 1 or 2");
  TORCH_CHECK_VALUE(h.dim() >= 1 && h.size(-1) >= 1 && h.size(-1) <= NFI_RESNORM_MAX_WIDTH, what, ": rows of 1 to ", NFI_RESNORM_MAX_WIDTH,
                    " values are wanted, not ", h.sizes());
  TORCH_CHECK_VALUE(eps >= 0, what, ": eps ", eps);
  const int64_t d = h.size(-1), rows = h.numel() / d;
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == h.sizes() && residual.scalar_type() == h.scalar_type()), what,
                    ": residual is ", residual.sizes(), " ", residual.defined() ? residual.scalar_type() : h.scalar_type(), ", h ", h.sizes(), " ",
                    h.scalar_type());
  TORCH_CHECK_VALUE(next != 0 || (!p[2].defined() && !p[3].defined()), what, ": next_weight and next_bias need next_norm");
  const Tensor* first = nullptr;
  for (int k = 0; k < 4; ++k) {
    if (!p[k].defined()) continue;
    type_code(p[k], what);
    const bool fits = (p[k].dim() == 1 && p[k].size(0) == d) ||
                      (p[k].dim() == 2 && p[k].size(1) == d && p[k].size(0) >= 1 && rows % p[k].size(0) == 0);
    TORCH_CHECK_VALUE(fits && (!first || (first->sizes() == p[k].sizes() && first->scalar_type() == p[k].scalar_type())), what, ": ", names[k],
                      " is ", p[k].sizes(), " ", p[k].scalar_type(), "; [", d, "], or [G, ", d, "] with G a divisor of ", rows,
                      " rows is wanted, all of one shape and type");
    if (!first) first = &p[k];
  }
  if (gate.defined()) {
    type_code(gate, what);
    if (gate.dim() == 1) gate = gate.unsqueeze(0);
    TORCH_CHECK_VALUE(gate.dim() == 2 && gate.size(1) == d && gate.size(0) >= 1 && rows % gate.size(0) == 0, what, ": gate is ", gate.sizes(),
                      "; [", d, "] or [G, ", d, "] with G a divisor of ", rows, " rows is wanted");
    if (first && first->dim() == 2 && gate.size(0) != first->size(0)) {
      TORCH_CHECK_VALUE(gate.size(0) == 1, what, ": ", gate.size(0), " gates and ", first->size(0), " groups of parameters");
      gate = gate.expand({first->size(0), d});
    }
    gate = gate.contiguous();
  }
  bool train = false;
  if (at::GradMode::is_enabled()) {
    train = h.requires_grad() || (residual.defined() && residual.requires_grad()) || (gate.defined() && gate.requires_grad());
    for (int k = 0; k < 4; ++k) train = train || (p[k].defined() && p[k].requires_grad());
  }
  const bool flat = h.dim() == 2;
  variable_list out = ResidualNorm::apply(flat ? h.contiguous() : h.reshape({rows, d}).contiguous(),
                                          maybe(!residual.defined() ? residual : flat ? residual.contiguous() : residual.reshape({rows, d}).contiguous()),
                                          maybe(gate), maybe(dense(p[0])), maybe(dense(p[1])), maybe(dense(p[2])), maybe(dense(p[3])), norm, next,
                                          slope, scale, eps, train);
  if (!flat)
    for (auto& t : out) t = t.view(h.sizes());
  return out;
}

// ---- grouped product -------------------------------------------------------------------------------------------------

nfi_grouped_args grouped_args(const Tensor& x, const Tensor& w, const Tensor& offsets) {
  nfi_grouped_args a{};
  a.x = x.data_ptr();
  a.w = w.data_ptr();
  a.offsets = offsets.data_ptr();
  a.offsets64 = offsets.scalar_type() == torch::kLong;
  a.rows = x.size(0);
  a.groups = (int32_t)w.size(0);
  a.out_width = (int32_t)w.size(1);
  a.in_width = (int32_t)w.size(2);
  a.dtype = type_code(x, "grouped_linear");
  return a;
}

struct GroupedLinear : public torch::autograd::Function<GroupedLinear> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w, Tensor offsets, Maybe bias_, bool train) {
    const Tensor bias = get(bias_);
    const c10::DeviceGuard guard(x.device());
    Tensor y = torch::empty({x.size(0), w.size(1)}, x.options());
    if (x.size(0) > 0) {
      nfi_grouped_args a = grouped_args(x, w, offsets);
      a.bias = ptr(bias);
      a.y = y.data_ptr();
      a.work_bytes = nfi_grouped_forward_work_bytes(&a);
      const Tensor work = bytes(a.work_bytes, x);
      a.work = ptr(work);
      check(nfi_grouped_forward(&a, stream_of(x)), "nfi_grouped_forward");
    }
    if (train) ctx->save_for_backward({x, w, offsets});
    ctx->saved_data["bias"] = bias.defined();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("grouped_linear");
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &offsets = s[2];
    const c10::DeviceGuard guard(x.device());
    const bool none = x.size(0) == 0;
    variable_list out(5);
    auto make = [&](const Tensor& like) { return none ? torch::zeros_like(like) : torch::empty_like(like); };
    if (ctx->needs_input_grad(0)) out[0] = make(x);
    if (ctx->needs_input_grad(1)) out[1] = make(w);
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3)) out[3] = none ? torch::zeros({w.size(0), w.size(1)}, x.options()) : torch::empty({w.size(0), w.size(1)}, x.options());
    if (none) return out;
    const Tensor gy = g[0].contiguous();
    nfi_grouped_args a = grouped_args(x, w, offsets);
    a.gy = gy.data_ptr();
    a.gx = ptr(out[0]);
    a.gw = ptr(out[1]);
    a.gb = ptr(out[3]);
    a.work_bytes = nfi_grouped_backward_work_bytes(&a);
    const Tensor work = bytes(a.work_bytes, x);
    a.work = ptr(work);
    check(nfi_grouped_backward(&a, stream_of(x)), "nfi_grouped_backward");
    return out;
  }
};

Tensor grouped_linear(const Tensor& x, const Tensor& w, const Tensor& offsets, const Maybe& bias_) {
  const char* what = "grouped_linear";
  const Tensor bias = get(bias_);
  on_device(what, x);
  with(what, "weight", w, x);
  with(what, "offsets", offsets, x);
  with(what, "bias", bias, x);
  type_code(x, what);
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 3 && w.size(2) == x.size(1), what, ": x [rows, K] and weight [groups, N, K] are wanted, not ",
                    x.sizes(), " and ", w.sizes());
  const int64_t e = w.size(0), n = w.size(1), k = w.size(2);
  TORCH_CHECK_VALUE(e >= 1 && e <= NFI_GROUPED_MAX_GROUPS && n >= 1 && n <= NFI_GROUPED_MAX_WIDTH && k >= 1 && k <= NFI_GROUPED_MAX_WIDTH, what,
                    ": 1 to ", NFI_GROUPED_MAX_GROUPS, " groups and widths of 1 to ", NFI_GROUPED_MAX_WIDTH, " are wanted, not ", w.sizes());
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.size(0) == e + 1 &&
                        (offsets.scalar_type() == torch::kInt || offsets.scalar_type() == torch::kLong),
                    what, ": offsets [", e + 1, "] int32 or int64 are wanted, not ", offsets.sizes(), " ", offsets.scalar_type());
  TORCH_CHECK(w.scalar_type() == x.scalar_type() && (!bias.defined() || bias.scalar_type() == x.scalar_type()), what,
              ": x, weight and bias are of one type, not ", x.scalar_type(), ", ", w.scalar_type());
  TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 2 && bias.size(0) == e && bias.size(1) == n), what, ": bias [", e, ", ", n,
                    "] is wanted, not ", bias.sizes());
  const bool train = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (bias.defined() && bias.requires_grad()));
  return GroupedLinear::apply(x.contiguous(), w.contiguous(), offsets.contiguous(), maybe(dense(bias)), train);
}

// ---- orthogonalised updates ------------------------------------------------------------------------------------------

int64_t ortho_bytes(const std::vector<nfi_ortho_item>& items) {
  const int64_t n = nfi_ortho_work_bytes(items.data(), (int32_t)items.size());
  if (n < 0) check(-1, "nfi_ortho_work_bytes");
  return n;
}

void ortho(const std::vector<nfi_ortho_item>& items, nfi_ortho_args a, const Tensor& work, void* stream) {
  a.items = items.data();
  a.n_items = (int32_t)items.size();
  a.work = ptr(work);
  a.work_bytes = work.defined() ? work.numel() : 0;
  check(nfi_ortho(&a, stream), "nfi_ortho");
}

Tensor orthogonalize(const Tensor& u, int64_t steps, double ca, double cb, double cc, double eps) {
  const char* what = "orthogonalize";
  on_device(what, u);
  nfi_ortho_args a{};
  a.g_type = a.w_type = type_code(u, what);
  TORCH_CHECK_VALUE(u.dim() >= 2, what, ": matrices are wanted, not ", u.sizes());
  const c10::DeviceGuard guard(u.device());
  const Tensor src = u.contiguous();
  Tensor out = torch::empty_like(src);
  if (out.numel() == 0) return out;
  const int64_t rows = u.size(-2), cols = u.size(-1), count = u.numel() / (rows * cols);
  TORCH_CHECK_VALUE(rows <= NFI_ORTHO_MAX_SIDE && cols <= NFI_ORTHO_MAX_SIDE && count < (1ll << 31), what, ": sides of 1 to ", NFI_ORTHO_MAX_SIDE,
                    " are wanted, not ", u.sizes());
  a.steps = (int32_t)steps;
  a.a = (float)ca;
  a.b = (float)cb;
  a.c = (float)cc;
  a.eps = (float)eps;
  std::vector<nfi_ortho_item> items(1);
  items[0] = {src.data_ptr(), nullptr, out.data_ptr(), (int32_t)rows, (int32_t)cols, (int32_t)count, 1.f};
  ortho(items, a, bytes(ortho_bytes(items), u), stream_of(u));
  return out;
}

void muon_step(at::TensorList params, at::TensorList grads, at::TensorList momenta, bool batched, double lr, double momentum, double decay,
               bool nesterov, int64_t steps, double ca, double cb, double cc, double eps) {
  const char* what = "Muon";
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && momenta.size() == n, what, ": ", n, " parameters, ", grads.size(), " gradients, ", momenta.size(), " buffers");
  nfi_ortho_args a{};
  a.update = 1;
  a.nesterov = nesterov;
  a.steps = (int32_t)steps;
  a.momentum = (float)momentum;
  a.step = (float)lr;
  a.decay = (float)(lr * decay);
  a.a = (float)ca;
  a.b = (float)cb;
  a.c = (float)cc;
  a.eps = (float)eps;
  // everything is checked, and every buffer is had, before anything is changed: one call for each device and pair of types (a
  // polynomial that is refused is the same for all of them, and the first call says so)
  struct Lot {
    int64_t kind;
    std::vector<nfi_ortho_item> items;
    std::vector<size_t> of;
    Tensor work;
  };
  std::vector<Tensor> g(n);
  std::vector<Lot> lots;
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &m = momenta[i];
    on_device(what, p);
    with(what, "a gradient", grads[i], p);
    with(what, "a momentum", m, p);
    TORCH_CHECK(p.dim() >= 2 && p.is_contiguous() && !grads[i].is_sparse(), what, ": dense gradients and contiguous parameters are wanted");
    TORCH_CHECK(grads[i].sizes() == p.sizes() && m.sizes() == p.sizes() && m.is_contiguous() && m.scalar_type() == torch::kFloat, what,
                ": a 32-bit momentum and a gradient of the parameter's shape ", p.sizes(), " are wanted");
    const int64_t kind = (p.device().index() * 3 + type_code(p, what)) * 3 + type_code(grads[i], what);
    if (p.numel() == 0) continue;   // (nothing to update, and no sizes to divide by)
    const int64_t cols = batched ? p.size(-1) : p.numel() / p.size(0), rows = batched ? p.size(-2) : p.size(0), count = p.numel() / (rows * cols);
    TORCH_CHECK_VALUE(rows <= NFI_ORTHO_MAX_SIDE && cols <= NFI_ORTHO_MAX_SIDE && count < (1ll << 31), what, ": sides of 1 to ", NFI_ORTHO_MAX_SIDE,
                      " are wanted, not ", count, " of ", rows, " x ", cols);
    g[i] = grads[i].contiguous();
    size_t l = 0;
    while (l < lots.size() && lots[l].kind != kind) ++l;
    if (l == lots.size()) lots.push_back({kind, {}, {}, Tensor()});
    lots[l].items.push_back({g[i].data_ptr(), m.data_ptr(), p.data_ptr(), (int32_t)rows, (int32_t)cols, (int32_t)count,
                             (float)std::sqrt(std::max(1.0, (double)rows / (double)cols))});
    lots[l].of.push_back(i);
  }
  for (Lot& l : lots) {
    const Tensor& p = params[l.of[0]];
    const c10::DeviceGuard guard(p.device());
    l.work = bytes(ortho_bytes(l.items), p);
  }
  for (Lot& l : lots) {
    const Tensor& p = params[l.of[0]];
    const c10::DeviceGuard guard(p.device());
    a.w_type = type_code(p, what);
    a.g_type = type_code(g[l.of[0]], what);
    ortho(l.items, a, l.work, stream_of(p));
    for (size_t i : l.of) {   // what is cached by a tensor's version is out of date
      params[i].unsafeGetTensorImpl()->bump_version();
      momenta[i].unsafeGetTensorImpl()->bump_version();
    }
  }
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nfi, m) {
  m.def("residual_norm(Tensor h, Tensor? residual, Tensor? gate, Tensor? weight, Tensor? bias, Tensor? next_weight, Tensor? next_bias, "
        "int norm, int next_norm, float slope, float scale, float eps) -> Tensor[]");
  m.def("grouped_linear(Tensor x, Tensor weight, Tensor offsets, Tensor? bias=None) -> Tensor");
  m.def("orthogonalize(Tensor u, int steps, float a, float b, float c, float eps) -> Tensor");
  m.def("muon_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, bool batched, float lr, float momentum, float decay, "
        "bool nesterov, int steps, float a, float b, float c, float eps) -> ()");
}

TORCH_LIBRARY_IMPL(nfi, CompositeImplicitAutograd, m) {
  m.impl("residual_norm", &residual_norm);
  m.impl("grouped_linear", &grouped_linear);
  m.impl("orthogonalize", &orthogonalize);
  m.impl("muon_step", &muon_step);
}

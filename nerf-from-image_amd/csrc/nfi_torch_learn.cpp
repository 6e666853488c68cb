// The operators of include/nfi_learn.h as TORCH_LIBRARY(nfi, ...) operators: the argument checks, the autograd
// functions and the optimiser's call in C++ (a small layer's forward and backward take 30 us of host time through
// Python functions and the interpreter lock; the kernels behind them 5).  nfi/norms.py, grouped.py and optim.py are
// their documented front.
//
//   nfi::residual_norm(h, residual?, gate?, weight?, bias?, next_weight?, next_bias?, norm, next_norm, slope, scale,
//                      eps) -> Tensor[]       x, or x and y
//   nfi::grouped_linear(x, weight, offsets, bias?) -> Tensor
//   nfi::residual_norm_fwd / _bwd, nfi::grouped_linear_fwd / _bwd      their halves as plain ops (CUDA + Meta kernels)
//   nfi::orthogonalize(u, steps, a, b, c, eps) -> Tensor               (CUDA + Meta kernels)
//   nfi::muon_step(params, grads, momenta, ...) -> ()       in place   (CUDA + Meta kernels)
//
// The autograd functions call the halves' functions themselves; where a tensor has no memory, or a dispatch mode looks on (meta and
// fake tensors, tracing), they call them through the dispatcher, whose Meta kernels give shapes and touch no pointer.
#include <algorithm>
#include <array>
#include <cmath>
#include <vector>

#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
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
  TORCH_CHECK(first.is_cuda() || first.is_meta(), what, ": nfi ops run on HIP devices only (got a ", first.device(), " tensor)");
}
// is the call one that is traced?  (its tensors may have no memory)
bool traced(const Tensor& t) {
  return t.is_meta() || t.key_set().has(c10::DispatchKey::Python) || t.key_set().has(c10::DispatchKey::Functionalize) ||
         c10::impl::TorchDispatchModeTLS::any_modes_set();
}
template <class F>
c10::TypedOperatorHandle<F> halves(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
void with(const char* what, const char* name, const Tensor& t, const Tensor& first) {
  TORCH_CHECK(!t.defined() || t.device() == first.device(), what, ": ", name, " is on ", t.device(), ", the first input on ",
              first.device());
}

Tensor get(const Maybe& t) { return t ? *t : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor listed(const Tensor& t, const Tensor& like) { return t.defined() ? t : torch::empty({0}, like.options()); }
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

// x, y and the statistics (those that are wanted); in: contiguous, h [rows, width]
variable_list norm_forward(const Tensor* in, const NormConf& c, bool keep, bool shapes_only) {
  const Tensor& h = in[0];
  Tensor x = torch::empty_like(h), y = c.next ? torch::empty_like(h) : Tensor(), stats;
  if (h.size(0) > 0) {
    if (keep) stats = torch::empty({h.size(0), 4}, h.options().dtype(torch::kFloat));
    if (!shapes_only) {
      nfi_resnorm_args a = norm_args(in, c);
      a.x = ptr(x);
      a.y = ptr(y);
      a.stats = (float*)ptr(stats);
      check(nfi_resnorm_forward(&a, stream_of(h)), "nfi_resnorm_forward");
    }
  }
  return {x, y, stats};
}

// the gradients of in[k] where needs[k]; gx, gy: contiguous, one of them at least
variable_list norm_backward(const Tensor& gx, const Tensor& gy, const Tensor* in, const Tensor& stats, const NormConf& c, const std::array<bool, 7>& needs,
                            bool shapes_only) {
  variable_list out(7);
  const bool none = in[0].size(0) == 0;
  for (int k = 0; k < 7; ++k) {
    if (!needs[k]) continue;
    // (nothing reaches the next norm's parameters without a gradient of y)
    out[k] = none || (k >= 5 && !gy.defined()) ? torch::zeros_like(in[k]) : torch::empty_like(in[k]);
  }
  if (none || shapes_only) return out;
  nfi_resnorm_args a = norm_args(in, c);
  a.stats = (float*)ptr(stats);
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
  const Tensor work = bytes(nfi_resnorm_work_bytes(a.rows, a.groups, a.affine_groups, a.width), in[0]);
  a.work = (float*)ptr(work);
  check(nfi_resnorm_backward(&a, stream_of(in[0])), "nfi_resnorm_backward");
  return out;
}

typedef std::vector<Tensor> norm_fwd_t(const Tensor&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, int64_t,
                                       int64_t, double, double, double, bool);
typedef std::vector<Tensor> norm_bwd_t(const Maybe&, const Maybe&, const Tensor&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, const Maybe&,
                                       const Maybe&, const Maybe&, int64_t, int64_t, double, double, double, std::array<bool, 7>);

struct ResidualNorm : public torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, Tensor h, Maybe residual_, Maybe gate_, Maybe weight_, Maybe bias_, Maybe next_weight_,
                               Maybe next_bias_, int64_t norm, int64_t next, double slope, double scale, double eps, bool train) {
    variable_list r;
    if (traced(h)) {
      static auto op = halves<norm_fwd_t>("nfi::residual_norm_fwd");
      r = op.call(h, residual_, gate_, weight_, bias_, next_weight_, next_bias_, norm, next, slope, scale, eps, train);
      for (int k = 1; k < 3; ++k)
        if (k == 1 ? next == 0 : !train || h.size(0) == 0) r[k] = Tensor();
    } else {
      const c10::DeviceGuard guard(h.device());
      const Tensor in[7] = {h, get(residual_), get(gate_), get(weight_), get(bias_), get(next_weight_), get(next_bias_)};
      r = norm_forward(in, NormConf{norm, next, slope, scale, eps}, train, false);
    }
    if (train) {
      ctx->set_materialize_grads(false);
      ctx->save_for_backward({h, get(residual_), get(gate_), get(weight_), get(bias_), get(next_weight_), get(next_bias_), r[2]});
      ctx->saved_data["norm"] = norm;
      ctx->saved_data["next"] = next;
      ctx->saved_data["slope"] = slope;
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["eps"] = eps;
    }
    if (next) return {r[0], r[1]};
    return {r[0]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("residual_norm");
    variable_list out(13);
    const Tensor gx = dense(g[0]), gy = g.size() > 1 ? dense(g[1]) : Tensor();
    if (!gx.defined() && !gy.defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const NormConf c{ctx->saved_data["norm"].toInt(), ctx->saved_data["next"].toInt(), ctx->saved_data["slope"].toDouble(),
                     ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble()};
    std::array<bool, 7> needs;
    for (int k = 0, edge = 0; k < 7; ++k)   // (the graph's edges are those of the arguments that are there)
      needs[k] = s[k].defined() && ctx->needs_input_grad(edge++);
    variable_list r;
    if (traced(s[0]) || traced(gx.defined() ? gx : gy)) {
      static auto op = halves<norm_bwd_t>("nfi::residual_norm_bwd");
      r = op.call(maybe(gx), maybe(gy), s[0], maybe(s[1]), maybe(s[2]), maybe(s[3]), maybe(s[4]), maybe(s[5]), maybe(s[6]), maybe(s[7]), c.norm, c.next,
                  c.slope, c.scale, c.eps, needs);
    } else {
      const c10::DeviceGuard guard(s[0].device());
      r = norm_backward(gx, gy, s.data(), s[7], c, needs, false);
    }
    for (int k = 0; k < 7; ++k)
      if (needs[k]) out[k] = r[k];
    return out;
  }
};

// in: h, residual, gate, weight, bias, next_weight, next_bias.  Returns the first of the norms' parameters
const Tensor* check_norm(const char* what, const Tensor* in, int64_t norm, int64_t next, double eps) {
  static const char* names[7] = {"h", "residual", "gate", "weight", "bias", "next_weight", "next_bias"};
  const Tensor &h = in[0], &residual = in[1], &gate = in[2];
  on_device(what, h);
  for (int k = 1; k < 7; ++k) with(what, names[k], in[k], h);
  type_code(h, what);
  TORCH_CHECK_VALUE(norm >= 0 && norm <= 2 && next >= 0 && next <= 2, what, ": norms are 0, 1 or 2");
  TORCH_CHECK_VALUE(h.dim() >= 1 && h.size(-1) >= 1 && h.size(-1) <= NFI_RESNORM_MAX_WIDTH, what, ": rows of 1 to ", NFI_RESNORM_MAX_WIDTH,
                    " values are wanted, not ", h.sizes());
  TORCH_CHECK_VALUE(eps >= 0, what, ": eps ", eps);
  const int64_t d = h.size(-1), rows = h.numel() / d;
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == h.sizes() && residual.scalar_type() == h.scalar_type()), what,
                    ": residual is ", residual.sizes(), " ", residual.defined() ? residual.scalar_type() : h.scalar_type(), ", h ", h.sizes(), " ",
                    h.scalar_type());
  TORCH_CHECK_VALUE(next != 0 || (!in[5].defined() && !in[6].defined()), what, ": next_weight and next_bias need next_norm");
  const Tensor* first = nullptr;
  for (int k = 3; k < 7; ++k) {
    const Tensor& p = in[k];
    if (!p.defined()) continue;
    type_code(p, what);
    const bool fits = (p.dim() == 1 && p.size(0) == d) || (p.dim() == 2 && p.size(1) == d && p.size(0) >= 1 && rows % p.size(0) == 0);
    TORCH_CHECK_VALUE(fits && (!first || (first->sizes() == p.sizes() && first->scalar_type() == p.scalar_type())), what, ": ", names[k],
                      " is ", p.sizes(), " ", p.scalar_type(), "; [", d, "], or [G, ", d, "] with G a divisor of ", rows,
                      " rows is wanted, all of one shape and type");
    if (!first) first = &p;
  }
  if (gate.defined()) {
    type_code(gate, what);
    const int64_t gates = gate.dim() == 2 ? gate.size(0) : 1;
    TORCH_CHECK_VALUE((gate.dim() == 1 || gate.dim() == 2) && gate.size(-1) == d && gates >= 1 && rows % gates == 0, what, ": gate is ",
                      gate.sizes(), "; [", d, "] or [G, ", d, "] with G a divisor of ", rows, " rows is wanted");
    if (first && first->dim() == 2)
      TORCH_CHECK_VALUE(gates == 1 || gates == first->size(0), what, ": ", gates, " gates and ", first->size(0), " groups of parameters");
  }
  return first;
}

// the halves as operators: everything contiguous, h and the gate [.., width]
void check_halves(const char* what, const Tensor* in, int64_t norm, int64_t next, double eps) {
  const Tensor* first = check_norm(what, in, norm, next, eps);
  TORCH_CHECK_VALUE(in[0].dim() == 2, what, ": h [rows, width] is wanted, not ", in[0].sizes());
  TORCH_CHECK_VALUE(!in[2].defined() || (in[2].dim() == 2 && (!first || first->dim() == 1 || first->size(0) == in[2].size(0))), what,
                    ": a gate [G, width], and G groups of parameters where they have groups, are wanted");
  for (int k = 0; k < 7; ++k) TORCH_CHECK_VALUE(!in[k].defined() || in[k].is_contiguous(), what, ": contiguous tensors are wanted");
}

template <bool META>
std::vector<Tensor> residual_norm_fwd(const Tensor& h, const Maybe& residual, const Maybe& gate, const Maybe& weight, const Maybe& bias,
                                      const Maybe& next_weight, const Maybe& next_bias, int64_t norm, int64_t next, double slope, double scale,
                                      double eps, bool keep) {
  const Tensor in[7] = {h, get(residual), get(gate), get(weight), get(bias), get(next_weight), get(next_bias)};
  check_halves("residual_norm_fwd", in, norm, next, eps);
  c10::OptionalDeviceGuard guard;
  if (!META) guard.reset_device(h.device());
  variable_list r = norm_forward(in, NormConf{norm, next, slope, scale, eps}, keep, META);
  for (auto& t : r) t = listed(t, h);
  return r;
}

template <bool META>
std::vector<Tensor> residual_norm_bwd(const Maybe& gx_, const Maybe& gy_, const Tensor& h, const Maybe& residual, const Maybe& gate,
                                      const Maybe& weight, const Maybe& bias, const Maybe& next_weight, const Maybe& next_bias,
                                      const Maybe& stats_, int64_t norm, int64_t next, double slope, double scale, double eps,
                                      std::array<bool, 7> needs) {
  const char* what = "residual_norm_bwd";
  const Tensor in[7] = {h, get(residual), get(gate), get(weight), get(bias), get(next_weight), get(next_bias)};
  check_halves(what, in, norm, next, eps);
  const Tensor gx = get(gx_), gy = get(gy_), stats = get(stats_);
  TORCH_CHECK_VALUE(gx.defined() || gy.defined(), what, ": no gradient");
  TORCH_CHECK_VALUE(next != 0 || !gy.defined(), what, ": gy without a next norm");
  for (const Tensor& g : {gx, gy}) {
    with(what, "a gradient", g, h);
    TORCH_CHECK_VALUE(!g.defined() || (g.sizes() == h.sizes() && g.scalar_type() == h.scalar_type() && g.is_contiguous()), what,
                      ": gradients like h, contiguous, are wanted");
  }
  with(what, "stats", stats, h);
  TORCH_CHECK_VALUE(h.size(0) == 0 || (stats.defined() && stats.dim() == 2 && stats.size(0) == h.size(0) && stats.size(1) == 4 &&
                                       stats.scalar_type() == torch::kFloat && stats.is_contiguous()),
                    what, ": the forward's stats [rows, 4] are wanted");
  for (int k = 0; k < 7; ++k) TORCH_CHECK_VALUE(!needs[k] || in[k].defined(), what, ": a gradient of an absent argument");
  c10::OptionalDeviceGuard guard;
  if (!META) guard.reset_device(h.device());
  variable_list r = norm_backward(gx, gy, in, stats, NormConf{norm, next, slope, scale, eps}, needs, META);
  for (auto& t : r) t = listed(t, h);
  return r;
}

std::vector<Tensor> residual_norm(const Tensor& h, const Maybe& residual_, const Maybe& gate_, const Maybe& weight_, const Maybe& bias_,
                                  const Maybe& next_weight_, const Maybe& next_bias_, int64_t norm, int64_t next, double slope, double scale,
                                  double eps) {
  Tensor residual = get(residual_), gate = get(gate_);
  const Tensor p[4] = {get(weight_), get(bias_), get(next_weight_), get(next_bias_)};
  const Tensor in[7] = {h, residual, gate, p[0], p[1], p[2], p[3]};
  const Tensor* first = check_norm("residual_norm", in, norm, next, eps);
  const int64_t d = h.size(-1), rows = h.numel() / d;
  if (gate.defined()) {
    if (gate.dim() == 1) gate = gate.unsqueeze(0);
    // (in 32 bits: the groups' gradients of one gate are added up unrounded)
    if (first && first->dim() == 2 && gate.size(0) != first->size(0)) gate = gate.to(torch::kFloat).expand({first->size(0), d});
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

Tensor grouped_forward(const Tensor& x, const Tensor& w, const Tensor& offsets, const Tensor& bias, bool shapes_only) {
  Tensor y = torch::empty({x.size(0), w.size(1)}, x.options());
  if (x.size(0) == 0 || shapes_only) return y;
  nfi_grouped_args a = grouped_args(x, w, offsets);
  a.bias = ptr(bias);
  a.y = y.data_ptr();
  a.work_bytes = nfi_grouped_forward_work_bytes(&a);
  const Tensor work = bytes(a.work_bytes, x);
  a.work = ptr(work);
  check(nfi_grouped_forward(&a, stream_of(x)), "nfi_grouped_forward");
  return y;
}

// the gradients of x, weight and bias, those that are needed
variable_list grouped_backward(const Tensor& gy, const Tensor& x, const Tensor& w, const Tensor& offsets, const std::array<bool, 3>& needs,
                               bool shapes_only) {
  const bool none = x.size(0) == 0;
  variable_list out(3);
  auto make = [&](at::IntArrayRef sizes) { return none ? torch::zeros(sizes, x.options()) : torch::empty(sizes, x.options()); };
  if (needs[0]) out[0] = make(x.sizes());
  if (needs[1]) out[1] = make(w.sizes());
  if (needs[2]) out[2] = make({w.size(0), w.size(1)});
  if (none || shapes_only) return out;
  nfi_grouped_args a = grouped_args(x, w, offsets);
  a.gy = gy.data_ptr();
  a.gx = ptr(out[0]);
  a.gw = ptr(out[1]);
  a.gb = ptr(out[2]);
  a.work_bytes = nfi_grouped_backward_work_bytes(&a);
  const Tensor work = bytes(a.work_bytes, x);
  a.work = ptr(work);
  check(nfi_grouped_backward(&a, stream_of(x)), "nfi_grouped_backward");
  return out;
}

typedef Tensor grouped_fwd_t(const Tensor&, const Tensor&, const Tensor&, const Maybe&);
typedef std::vector<Tensor> grouped_bwd_t(const Tensor&, const Tensor&, const Tensor&, const Tensor&, std::array<bool, 3>);

struct GroupedLinear : public torch::autograd::Function<GroupedLinear> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor w, Tensor offsets, Maybe bias_, bool train) {
    if (train) ctx->save_for_backward({x, w, offsets});
    ctx->saved_data["bias"] = bias_.has_value();
    if (traced(x)) {
      static auto op = halves<grouped_fwd_t>("nfi::grouped_linear_fwd");
      return op.call(x, w, offsets, bias_);
    }
    const c10::DeviceGuard guard(x.device());
    return grouped_forward(x, w, offsets, get(bias_), false);
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("grouped_linear");
    const variable_list s = ctx->get_saved_variables();
    const std::array<bool, 3> needs = {ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                       ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3)};
    const Tensor gy = g[0].contiguous();
    variable_list r;
    if (traced(s[0]) || traced(gy)) {
      static auto op = halves<grouped_bwd_t>("nfi::grouped_linear_bwd");
      r = op.call(gy, s[0], s[1], s[2], needs);
    } else {
      const c10::DeviceGuard guard(s[0].device());
      r = grouped_backward(gy, s[0], s[1], s[2], needs, false);
    }
    variable_list out(5);
    if (needs[0]) out[0] = r[0];
    if (needs[1]) out[1] = r[1];
    if (needs[2]) out[3] = r[2];
    return out;
  }
};

void check_grouped(const char* what, const Tensor& x, const Tensor& w, const Tensor& offsets, const Tensor& bias) {
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
}

template <bool META>
Tensor grouped_linear_fwd(const Tensor& x, const Tensor& w, const Tensor& offsets, const Maybe& bias_) {
  const char* what = "grouped_linear_fwd";
  const Tensor bias = get(bias_);
  check_grouped(what, x, w, offsets, bias);
  TORCH_CHECK_VALUE(x.is_contiguous() && w.is_contiguous() && offsets.is_contiguous() && (!bias.defined() || bias.is_contiguous()), what,
                    ": contiguous tensors are wanted");
  c10::OptionalDeviceGuard guard;
  if (!META) guard.reset_device(x.device());
  return grouped_forward(x, w, offsets, bias, META);
}

template <bool META>
std::vector<Tensor> grouped_linear_bwd(const Tensor& gy, const Tensor& x, const Tensor& w, const Tensor& offsets, std::array<bool, 3> needs) {
  const char* what = "grouped_linear_bwd";
  check_grouped(what, x, w, offsets, Tensor());
  with(what, "gy", gy, x);
  TORCH_CHECK_VALUE(gy.dim() == 2 && gy.size(0) == x.size(0) && gy.size(1) == w.size(1) && gy.scalar_type() == x.scalar_type(), what, ": gy [",
                    x.size(0), ", ", w.size(1), "] of x's type is wanted, not ", gy.sizes(), " ", gy.scalar_type());
  TORCH_CHECK_VALUE(gy.is_contiguous() && x.is_contiguous() && w.is_contiguous() && offsets.is_contiguous(), what, ": contiguous tensors are wanted");
  c10::OptionalDeviceGuard guard;
  if (!META) guard.reset_device(x.device());
  variable_list r = grouped_backward(gy, x, w, offsets, needs, META);
  for (auto& t : r) t = listed(t, x);
  return r;
}

Tensor grouped_linear(const Tensor& x, const Tensor& w, const Tensor& offsets, const Maybe& bias_) {
  const Tensor bias = get(bias_);
  check_grouped("grouped_linear", x, w, offsets, bias);
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

template <bool META>
Tensor orthogonalize(const Tensor& u, int64_t steps, double ca, double cb, double cc, double eps) {
  const char* what = "orthogonalize";
  on_device(what, u);
  nfi_ortho_args a{};
  a.g_type = a.w_type = type_code(u, what);
  TORCH_CHECK_VALUE(u.dim() >= 2, what, ": matrices are wanted, not ", u.sizes());
  if (META) return torch::empty(u.sizes(), u.options());
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

template <bool META>
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
    if (META) continue;
    g[i] = grads[i].contiguous();
    size_t l = 0;
    while (l < lots.size() && lots[l].kind != kind) ++l;
    if (l == lots.size()) {
      lots.push_back({kind, {}, {}, Tensor()});
      lots[l].items.reserve(n - i);
      lots[l].of.reserve(n - i);
    }
    lots[l].items.push_back({g[i].data_ptr(), m.data_ptr(), p.data_ptr(), (int32_t)rows, (int32_t)cols, (int32_t)count,
                             (float)std::sqrt(std::max(1.0, (double)rows / (double)cols))});
    lots[l].of.push_back(i);
  }
  // what is updated lies apart: all matrices are stepped at a time
  std::vector<std::pair<const char*, const char*>> spans;
  spans.reserve(2 * n);
  for (const Lot& l : lots)
    for (size_t i : l.of)
      for (const Tensor* t : {&params[i], &momenta[i]}) spans.emplace_back((const char*)t->data_ptr(), (const char*)t->data_ptr() + t->nbytes());
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    TORCH_CHECK_VALUE(spans[i].first >= spans[i - 1].second, what, ": parameters and momenta that share memory (each is stepped on its own)");
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
  m.def("residual_norm_fwd(Tensor h, Tensor? residual, Tensor? gate, Tensor? weight, Tensor? bias, Tensor? next_weight, Tensor? next_bias, "
        "int norm, int next_norm, float slope, float scale, float eps, bool stats) -> Tensor[]");
  m.def("residual_norm_bwd(Tensor? gx, Tensor? gy, Tensor h, Tensor? residual, Tensor? gate, Tensor? weight, Tensor? bias, "
        "Tensor? next_weight, Tensor? next_bias, Tensor? stats, int norm, int next_norm, float slope, float scale, float eps, "
        "bool[7] needs) -> Tensor[]");
  m.def("grouped_linear(Tensor x, Tensor weight, Tensor offsets, Tensor? bias=None) -> Tensor");
  m.def("grouped_linear_fwd(Tensor x, Tensor weight, Tensor offsets, Tensor? bias=None) -> Tensor");
  m.def("grouped_linear_bwd(Tensor gy, Tensor x, Tensor weight, Tensor offsets, bool[3] needs) -> Tensor[]");
  m.def("orthogonalize(Tensor u, int steps, float a, float b, float c, float eps) -> Tensor");
  m.def("muon_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, bool batched, float lr, float momentum, float decay, "
        "bool nesterov, int steps, float a, float b, float c, float eps) -> ()");
}

TORCH_LIBRARY_IMPL(nfi, CompositeImplicitAutograd, m) {
  m.impl("residual_norm", &residual_norm);
  m.impl("grouped_linear", &grouped_linear);
}

TORCH_LIBRARY_IMPL(nfi, CUDA, m) {
  m.impl("residual_norm_fwd", &residual_norm_fwd<false>);
  m.impl("residual_norm_bwd", &residual_norm_bwd<false>);
  m.impl("grouped_linear_fwd", &grouped_linear_fwd<false>);
  m.impl("grouped_linear_bwd", &grouped_linear_bwd<false>);
}

TORCH_LIBRARY_IMPL(nfi, CompositeExplicitAutograd, m) {   // (other devices' tensors are refused, and no tensors are no work)
  m.impl("orthogonalize", &orthogonalize<false>);
  m.impl("muon_step", &muon_step<false>);
}

TORCH_LIBRARY_IMPL(nfi, Autograd, m) {   // (not differentiable; the default would box every argument to say so, 2 us)
  m.impl("orthogonalize", torch::CppFunction::makeFallthrough());
  m.impl("muon_step", torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(nfi, Meta, m) {
  m.impl("residual_norm_fwd", &residual_norm_fwd<true>);
  m.impl("residual_norm_bwd", &residual_norm_bwd<true>);
  m.impl("grouped_linear_fwd", &grouped_linear_fwd<true>);
  m.impl("grouped_linear_bwd", &grouped_linear_bwd<true>);
  m.impl("orthogonalize", &orthogonalize<true>);
  m.impl("muon_step", &muon_step<true>);
}

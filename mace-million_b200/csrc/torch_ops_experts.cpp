// torch.ops.mace_b200.*: layer norm, expert routing and expert products over the C ABI (include/mace_b200.h), with their
// autograd formulas.  As in torch_ops.cpp, the ops check devices, types and shapes with TORCH_CHECK, launch on torch's
// current CUDA stream and allocate outputs and workspaces with torch's caching allocator.
#include "torch_ops_util.h"

namespace {

// ------------------------------------------------------------------------------------------------ layer norm
struct LnIn {
  Tensor rows, w, b;
  int32_t dt, pt;
  int64_t n, d;
};

LnIn ln_in(const Tensor& x, const Tensor& w, const Tensor& b) {
  LnIn a;
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last dimension of at least 1 (got ", x.sizes(), ")");
  TORCH_CHECK(x.size(-1) <= INT32_MAX, "x: last dimension too large");
  a.dt = a.pt = type_code(x, "x");
  a.d = x.size(-1);
  a.n = x.numel() / a.d;
  a.rows = a.n ? rows_of(x) : x;
  for (const Tensor* t : {&w, &b}) {
    if (!t->defined()) continue;
    on_device(*t, "weight / bias", x);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == a.d, "weight / bias must be [", a.d, "] (got ", t->sizes(), ")");
    TORCH_CHECK(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat,
                "weight / bias must have the type of x or float32");
    TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight and bias differ in type");
    a.pt = type_code(*t, "weight / bias");
  }
  a.w = w.defined() ? w.contiguous() : w;
  a.b = b.defined() ? b.contiguous() : b;
  return a;
}

std::tuple<Tensor, Tensor, Tensor> ln_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool stats) {
  LnIn a = ln_in(x, w, b);
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous), mean, rstd;
  if (stats) {
    mean = at::empty({a.n}, x.options().dtype(at::kFloat));
    rstd = at::empty({a.n}, x.options().dtype(at::kFloat));
  }
  if (a.n)
    check_rc(mace_b200_layer_norm_fwd(a.rows.data_ptr(), row_stride(a.rows), ptr(a.w), ptr(a.b), y.data_ptr(),
                                      ptr_as<float>(mean), ptr_as<float>(rstd), a.n, (int32_t)a.d, eps, a.dt, a.pt,
                                      stream_of(x)),
             "layer_norm");
  return {y, mean, rstd};
}

Tensor layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  return std::get<0>(ln_forward(x, or_none(w), or_none(b), eps, false));
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  return ln_forward(x, or_none(w), or_none(b), eps, true);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor& dy, const Tensor& x, const OptTensor& w,
                                                  const Tensor& mean, const Tensor& rstd, bool need_x, bool need_w,
                                                  bool need_b, bool bias_f32) {
  LnIn a = ln_in(x, or_none(w), none);
  // the parameters share a type: the weight's, else what the caller says of the bias
  const at::ScalarType bias_type = bias_f32 ? at::kFloat : x.scalar_type();
  if (!a.w.defined() && bias_f32) a.pt = MB_F32;
  on_device(dy, "dy", x);
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(), "dy must have the shape and type of x");
  for (const Tensor* t : {&mean, &rstd}) {
    on_device(*t, "mean / rstd", x);
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == a.n,
                "mean / rstd must be float32 with one value per row");
  }
  c10::cuda::CUDAGuard guard(x.device());
  auto popt = a.w.defined() ? a.w.options() : x.options().dtype(bias_type);
  Tensor dx = need_x ? at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous) : Tensor();
  Tensor dw = need_w ? at::empty({a.d}, popt) : Tensor(), db = need_b ? at::empty({a.d}, popt) : Tensor(), ws;
  if (need_w || need_b) {
    int64_t words = 0;
    check_rc(mace_b200_layer_norm_bwd_workspace(a.n, (int32_t)a.d, &words), "layer_norm_bwd");
    ws = at::empty({words}, x.options().dtype(at::kFloat));
  }
  Tensor g = a.n ? rows_of(dy) : dy;
  if (a.n || need_w || need_b)
    check_rc(mace_b200_layer_norm_bwd(ptr(g), a.n ? row_stride(g) : a.d, ptr(a.rows), a.n ? row_stride(a.rows) : a.d,
                                      ptr(a.w), mean.data_ptr<float>(), rstd.data_ptr<float>(), ptr(dx), ptr(dw),
                                      ptr(db), ptr_as<float>(ws), a.n, (int32_t)a.d, a.dt, a.pt, stream_of(x)),
             "layer_norm_bwd");
  return {dx, dw, db};
}

struct LayerNormGrad : torch::autograd::Function<LayerNormGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto fwd = op_of<decltype(layer_norm_fwd)>("mace_b200::layer_norm_fwd");
    auto [y, mean, rstd] = fwd.call(x, w, b, eps);
    ctx->save_for_backward({x, or_none(w), mean, rstd});
    ctx->saved_data["w"] = given(w);
    ctx->saved_data["b"] = given(b);
    ctx->saved_data["b_f32"] = given(b) && b->scalar_type() == at::kFloat;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("layer_norm");
    auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    // needs_input_grad counts the tensors that were given
    const bool has_w = ctx->saved_data["w"].toBool(), has_b = ctx->saved_data["b"].toBool();
    static auto bwd = op_of<decltype(layer_norm_bwd)>("mace_b200::layer_norm_bwd");
    auto [dx, dw, db] = bwd.call(g[0], s[0], opt(s[1]), s[2], s[3], ctx->needs_input_grad(0),
                                 has_w && ctx->needs_input_grad(1), has_b && ctx->needs_input_grad(1 + has_w),
                                 ctx->saved_data["b_f32"].toBool());
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm_autograd(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  no_dual("layer_norm", {&x, &or_none(w), &or_none(b)});
  if (wants_grad({&x, &or_none(w), &or_none(b)})) {
    TORCH_CHECK(!given(w) || !given(b) || w->scalar_type() == b->scalar_type(), "weight and bias differ in type");
    return LayerNormGrad::apply(x, w, b, eps);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = op_of<decltype(layer_norm)>("mace_b200::layer_norm");
  return op.call(x, w, b, eps);
}

// ------------------------------------------------------------------------------------------------ routing
struct RouteIn {
  Tensor l;
  int32_t dt;
};

RouteIn route_in(const Tensor& logits, int64_t k, const char* what) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(1) <= MB_ROUTE_MAX_EXPERTS,
              "logits must be [tokens, experts] with at most ", MB_ROUTE_MAX_EXPERTS, " experts (got ", logits.sizes(), ")");
  TORCH_CHECK(k >= 1 && k <= MB_ROUTE_MAX_K && k <= logits.size(1), what, ": k must be in [1, min(", MB_ROUTE_MAX_K, ", ",
              logits.size(1), ")] (got ", k, ")");
  return {logits.size(0) ? rows_of(logits) : logits, type_code(logits, "logits")};
}

std::tuple<Tensor, Tensor> route(const Tensor& logits, const OptTensor& bias, int64_t k, bool softmax, int64_t groups,
                                 int64_t top_groups, bool renormalize, double scale) {
  RouteIn a = route_in(logits, k, "route");
  const int64_t n = logits.size(0), E = logits.size(1);
  TORCH_CHECK(groups >= 1 && groups <= 32 && E % groups == 0, "route: ", E, " experts do not split into ", groups,
              " groups (at most 32)");
  TORCH_CHECK(top_groups >= 1 && top_groups <= groups, "route: top_groups must be in [1, groups]");
  Tensor b;
  if (given(bias)) {
    on_device(*bias, "bias", logits);
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == E && bias->scalar_type() == at::kFloat, "bias must be float32 [", E, "]");
    b = bias->contiguous();
  }
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor w = at::empty({n, k}, logits.options().dtype(at::kFloat)), e = at::empty({n, k}, logits.options().dtype(at::kInt));
  if (n)
    check_rc(mace_b200_route_fwd(a.l.data_ptr(), row_stride(a.l), ptr_as<float>(b), w.data_ptr<float>(),
                                 e.data_ptr<int32_t>(), n, (int32_t)E, (int32_t)k, softmax, (int32_t)groups,
                                 (int32_t)top_groups, renormalize, (float)scale, a.dt, stream_of(logits)),
             "route");
  return {w, e};
}

Tensor route_bwd(const Tensor& dweights, const Tensor& logits, const Tensor& experts, bool softmax, bool renormalize,
                 double scale) {
  TORCH_CHECK(experts.dim() == 2 && experts.scalar_type() == at::kInt, "experts must be int32 [tokens, k]");
  const int64_t k = experts.size(1), n = logits.size(0);
  RouteIn a = route_in(logits, k, "route_bwd");
  on_device(experts, "experts", logits);
  on_device(dweights, "dweights", logits);
  TORCH_CHECK(experts.size(0) == n && dweights.sizes() == experts.sizes() && dweights.scalar_type() == at::kFloat,
              "dweights must be float32 [tokens, k] like experts");
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor dl = at::empty(logits.sizes(), logits.options(), at::MemoryFormat::Contiguous);
  Tensor dw = dweights.contiguous(), ex = experts.contiguous();
  if (n)
    check_rc(mace_b200_route_bwd(dw.data_ptr<float>(), a.l.data_ptr(), row_stride(a.l), ex.data_ptr<int32_t>(),
                                 dl.data_ptr(), n, (int32_t)logits.size(1), (int32_t)k, softmax, renormalize,
                                 (float)scale, a.dt, stream_of(logits)),
             "route_bwd");
  return dl;
}

struct RouteGrad : torch::autograd::Function<RouteGrad> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& bias, int64_t k, bool softmax,
                               int64_t groups, int64_t top_groups, bool renormalize, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = op_of<decltype(route)>("mace_b200::route");
    auto [w, e] = op.call(logits, bias, k, softmax, groups, top_groups, renormalize, scale);
    ctx->save_for_backward({logits, e});
    ctx->saved_data["softmax"] = softmax;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({e});
    return {w, e};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("route");
    auto s = ctx->get_saved_variables();
    variable_list out(8);
    static auto bwd = op_of<decltype(route_bwd)>("mace_b200::route_bwd");
    if (g[0].defined())
      out[0] = bwd.call(g[0], s[0], s[1], ctx->saved_data["softmax"].toBool(), ctx->saved_data["renormalize"].toBool(),
                        ctx->saved_data["scale"].toDouble());
    return out;
  }
};

std::tuple<Tensor, Tensor> route_autograd(const Tensor& logits, const OptTensor& bias, int64_t k, bool softmax,
                                          int64_t groups, int64_t top_groups, bool renormalize, double scale) {
  no_dual("route", {&logits});
  if (wants_grad({&logits})) {
    auto r = RouteGrad::apply(logits, bias, k, softmax, groups, top_groups, renormalize, scale);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = op_of<decltype(route)>("mace_b200::route");
  return op.call(logits, bias, k, softmax, groups, top_groups, renormalize, scale);
}

// ------------------------------------------------------------------------------------------------ expert products
Tensor expert_plan(const Tensor& experts, int64_t n_experts) {
  TORCH_CHECK(experts.is_cuda() && experts.scalar_type() == at::kInt && experts.dim() == 2 && experts.is_contiguous(),
              "experts must be a contiguous int32 CUDA tensor [tokens, k]");
  int64_t words = 0;
  TORCH_CHECK(n_experts >= 1 && n_experts <= MB_PLAN_MAX_EXPERTS, "n_experts must be in [1, ", MB_PLAN_MAX_EXPERTS, "]");
  check_rc(mace_b200_expert_plan_words(experts.numel(), (int32_t)n_experts, &words), "expert_plan");
  c10::cuda::CUDAGuard guard(experts.device());
  Tensor plan = at::empty({words}, experts.options());
  check_rc(mace_b200_expert_plan(experts.data_ptr<int32_t>(), experts.numel(), (int32_t)n_experts,
                                 plan.data_ptr<int32_t>(), stream_of(experts)),
           "expert_plan");
  return plan;
}

struct XIn {
  Tensor rows, w, weights;
  bool slots;
  int32_t dt, k, E, D, O;
  int64_t T;
};

XIn x_in(const Tensor& x, const Tensor& w, const Tensor& experts, const Tensor& plan, const Tensor& weights) {
  XIn a;
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK(experts.dim() == 2 && experts.scalar_type() == at::kInt && experts.is_contiguous() && experts.size(1) >= 1,
              "experts must be contiguous int32 [tokens, k]");
  TORCH_CHECK(w.dim() == 3 && w.size(0) >= 1 && w.size(1) >= 1 && w.size(2) >= 1, "w must be [experts, out, in] (got ",
              w.sizes(), ")");
  TORCH_CHECK(w.size(0) <= MB_PLAN_MAX_EXPERTS && w.size(1) <= (1 << 24) && w.size(2) <= (1 << 24), "w is too large");
  on_device(w, "w", x);
  on_device(experts, "experts", x);
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), "x and w differ in type");
  a.T = experts.size(0);
  a.k = (int32_t)experts.size(1);
  a.E = (int32_t)w.size(0);
  a.O = (int32_t)w.size(1);
  a.D = (int32_t)w.size(2);
  a.slots = x.dim() == 3;
  TORCH_CHECK((x.dim() == 2 || (x.dim() == 3 && x.size(1) == a.k)) && x.size(0) == a.T && x.size(-1) == a.D,
              "x must be [", a.T, ", ", a.D, "] or [", a.T, ", ", a.k, ", ", a.D, "] (got ", x.sizes(), ")");
  a.dt = type_code(x, "x");
  a.rows = a.T ? rows_of(x) : x;
  a.w = w.contiguous();
  if (weights.defined()) {
    on_device(weights, "weights", x);
    TORCH_CHECK(weights.sizes() == experts.sizes() && weights.scalar_type() == at::kFloat,
                "weights must be float32 [tokens, k] like experts");
    a.weights = weights.contiguous();
  }
  if (plan.defined()) {
    on_device(plan, "plan", x);
    int64_t words = 0;
    check_rc(mace_b200_expert_plan_words(experts.numel(), a.E, &words), "expert_linear");
    TORCH_CHECK(plan.scalar_type() == at::kInt && plan.is_contiguous() && plan.numel() == words,
                "plan does not belong to ", a.T, " tokens, k = ", a.k, ", ", a.E, " experts");
  }
  return a;
}

Tensor x_workspace(const XIn& a, bool backward) {
  int64_t bytes = 0;
  check_rc(mace_b200_expert_linear_workspace(a.T, a.k, a.E, a.D, a.O, a.dt, a.slots, a.weights.defined(), backward, &bytes),
           "expert_linear");
  return at::empty({bytes}, a.w.options().dtype(at::kByte));
}

// plan given: tensor cores; plan absent: the few-slots kernel
Tensor expert_linear(const Tensor& x, const Tensor& w, const Tensor& experts, const OptTensor& plan,
                     const OptTensor& weights) {
  XIn a = x_in(x, w, experts, or_none(plan), or_none(weights));
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = a.weights.defined() ? at::empty({a.T, a.O}, x.options()) : at::empty({a.T, a.k, a.O}, x.options());
  if (a.T == 0) return out;
  if (!given(plan)) {
    check_rc(mace_b200_expert_linear_few(a.rows.data_ptr(), row_stride(a.rows), a.slots, a.w.data_ptr(),
                                         experts.data_ptr<int32_t>(), ptr_as<float>(a.weights), out.data_ptr(), a.T, a.k,
                                         a.E, a.D, a.O, a.dt, stream_of(x)),
             "expert_linear");
    return out;
  }
  Tensor ws = x_workspace(a, false);
  check_rc(mace_b200_expert_linear_fwd(a.rows.data_ptr(), row_stride(a.rows), a.slots, a.w.data_ptr(),
                                       plan->data_ptr<int32_t>(), ptr_as<float>(a.weights), out.data_ptr(),
                                       ws.data_ptr(), a.T, a.k, a.E, a.D, a.O, a.dt, stream_of(x)),
           "expert_linear");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> expert_linear_bwd(const Tensor& dy, const Tensor& x, const Tensor& w,
                                                     const Tensor& experts, const Tensor& plan, const OptTensor& weights,
                                                     bool need_x, bool need_w, bool need_weights) {
  XIn a = x_in(x, w, experts, plan, or_none(weights));
  TORCH_CHECK(plan.defined(), "the backward pass needs a plan");
  on_device(dy, "dy", x);
  TORCH_CHECK(dy.scalar_type() == x.scalar_type() && dy.numel() == (a.weights.defined() ? a.T : a.T * a.k) * a.O &&
                  dy.size(-1) == a.O,
              "dy must have the shape and type of the output");
  need_weights = need_weights && a.weights.defined();
  c10::cuda::CUDAGuard guard(x.device());
  Tensor g = dy.contiguous();
  Tensor dx = need_x ? at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous) : Tensor();
  Tensor dw = need_w ? at::empty_like(a.w) : Tensor();
  Tensor dg = need_weights ? at::empty(experts.sizes(), a.weights.options()) : Tensor();
  if (!need_x && !need_w && !need_weights) return {dx, dw, dg};
  Tensor ws = x_workspace(a, true);
  check_rc(mace_b200_expert_linear_bwd(g.data_ptr(), a.T ? a.rows.data_ptr() : nullptr, a.T ? row_stride(a.rows) : a.D,
                                       a.slots, a.w.data_ptr(), plan.data_ptr<int32_t>(), ptr_as<float>(a.weights),
                                       ptr(dx), ptr(dw), ptr_as<float>(dg), ws.data_ptr(), a.T, a.k, a.E, a.D, a.O, a.dt,
                                       stream_of(x)),
           "expert_linear_bwd");
  return {dx, dw, dg};
}

struct ExpertLinearGrad : torch::autograd::Function<ExpertLinearGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& experts, const Tensor& plan,
                        const OptTensor& weights) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({x, w, experts, plan, or_none(weights)});
    static auto op = op_of<decltype(expert_linear)>("mace_b200::expert_linear");
    return op.call(x, w, experts, plan, weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("expert_linear");
    auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(5);
    static auto bwd = op_of<decltype(expert_linear_bwd)>("mace_b200::expert_linear_bwd");
    auto [dx, dw, dg] = bwd.call(g[0], s[0], s[1], s[2], s[3], opt(s[4]), ctx->needs_input_grad(0),
                                 ctx->needs_input_grad(1), s[4].defined() && ctx->needs_input_grad(4));
    return {dx, dw, Tensor(), Tensor(), dg};
  }
};

Tensor expert_linear_autograd(const Tensor& x, const Tensor& w, const Tensor& experts, const OptTensor& plan,
                              const OptTensor& weights) {
  no_dual("expert_linear", {&x, &w, &or_none(weights)});
  if (wants_grad({&x, &w, &or_none(weights)})) {
    static auto make = op_of<decltype(expert_plan)>("mace_b200::expert_plan");
    Tensor p = given(plan) ? *plan : make.call(experts, w.size(0));
    return ExpertLinearGrad::apply(x, w, experts, p, weights);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = op_of<decltype(expert_linear)>("mace_b200::expert_linear");
  return op.call(x, w, experts, plan, weights);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mace_b200, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_bwd(Tensor dy, Tensor x, Tensor? weight, Tensor mean, Tensor rstd, bool need_x, bool need_w, "
        "bool need_b, bool bias_f32) -> (Tensor, Tensor, Tensor)");
  m.def("route(Tensor logits, Tensor? bias, int k, bool softmax, int groups, int top_groups, bool renormalize, "
        "float scale) -> (Tensor, Tensor)");
  m.def("route_bwd(Tensor dweights, Tensor logits, Tensor experts, bool softmax, bool renormalize, float scale) -> Tensor");
  m.def("expert_plan(Tensor experts, int n_experts) -> Tensor");
  m.def("expert_linear(Tensor x, Tensor w, Tensor experts, Tensor? plan, Tensor? weights) -> Tensor");
  m.def("expert_linear_bwd(Tensor dy, Tensor x, Tensor w, Tensor experts, Tensor plan, Tensor? weights, bool need_x, "
        "bool need_w, bool need_weights) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mace_b200, CUDA, m) {
  m.impl("layer_norm", &layer_norm);
  m.impl("layer_norm_fwd", &layer_norm_fwd);
  m.impl("layer_norm_bwd", &layer_norm_bwd);
  m.impl("route", &route);
  m.impl("route_bwd", &route_bwd);
  m.impl("expert_plan", &expert_plan);
  m.impl("expert_linear", &expert_linear);
  m.impl("expert_linear_bwd", &expert_linear_bwd);
}

TORCH_LIBRARY_IMPL(mace_b200, AutogradCUDA, m) {
  m.impl("layer_norm", &layer_norm_autograd);
  m.impl("route", &route_autograd);
  m.impl("expert_linear", &expert_linear_autograd);
}

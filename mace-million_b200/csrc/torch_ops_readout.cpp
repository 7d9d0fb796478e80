// torch.ops.mace_b200.*: group norm with an activation (with its autograd formula), products in 8-bit integers and orthogonalised
// matrices over the C ABI (include/mace_b200.h).  As in
// torch_ops.cpp, the ops check devices, types and shapes with TORCH_CHECK, launch on torch's current CUDA stream and
// allocate outputs and workspaces with torch's caching allocator.
#include <cmath>

#include "torch_ops_util.h"

namespace {

// ------------------------------------------------------------------------------------------------ group norm
struct GnIn {
  Tensor rows, w, b, off;
  int32_t dt, pt, off64 = 0;
  int64_t n, len, r, c;
};

GnIn gn_in(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, const Tensor& offsets, int64_t act) {
  GnIn a;
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  a.dt = a.pt = type_code(x, "x");
  TORCH_CHECK(x.dim() >= 2 && x.size(-1) >= 1, "x must be [samples, .., channels] (got ", x.sizes(), ")");
  TORCH_CHECK(x.size(-1) <= INT32_MAX, "x: too many channels");
  a.c = x.size(-1);
  TORCH_CHECK(groups >= 1 && groups <= a.c && groups <= MB_GN_MAX_GROUPS && a.c % groups == 0, "group_norm: ", a.c, " channels do not split into ", groups, " groups");
  TORCH_CHECK(act >= MB_ACT_NONE && act <= MB_ACT_RELU, "group_norm: unknown activation ", act);
  a.r = x.numel() / a.c;
  if (offsets.defined()) {
    on_device(offsets, "offsets", x);
    TORCH_CHECK(x.dim() == 2, "x must be [rows, channels] with offsets (got ", x.sizes(), ")");
    TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) >= 1 &&
                    (offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong),
                "offsets must be int32 or int64 [samples + 1] (got ", offsets.sizes(), ", ", offsets.scalar_type(), ")");
    a.off = offsets.contiguous();
    a.off64 = offsets.scalar_type() == at::kLong;
    a.n = offsets.size(0) - 1;
    a.len = 0;
  } else {
    a.n = x.size(0);
    a.len = a.n ? a.r / a.n : 0;
  }
  a.rows = a.r ? rows_of(x) : x;
  for (const Tensor* t : {&w, &b}) {
    if (!t->defined()) continue;
    on_device(*t, "weight / bias", x);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == a.c, "weight / bias must be [", a.c, "] (got ", t->sizes(), ")");
    TORCH_CHECK(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat,
                "weight / bias must have the type of x or float32");
    TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight and bias differ in type");
    a.pt = type_code(*t, "weight / bias");
  }
  a.w = w.defined() ? w.contiguous() : w;
  a.b = b.defined() ? b.contiguous() : b;
  return a;
}

Tensor gn_workspace(const GnIn& a, int64_t groups, bool backward, const Tensor& like) {
  int64_t floats = 0;
  check_rc(mace_b200_group_norm_workspace(a.r, a.n, a.len, (int32_t)a.c, (int32_t)groups, a.off.defined(), a.dt, backward, &floats),
           "group_norm");
  return floats ? at::empty({floats}, like.options().dtype(at::kFloat)) : Tensor();
}

std::tuple<Tensor, Tensor, Tensor> gn_forward(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, double eps,
                                              int64_t act, const Tensor& offsets, bool stats) {
  GnIn a = gn_in(x, groups, w, b, offsets, act);
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous), mean, rstd;
  if (stats) {
    mean = at::empty({a.n, groups}, x.options().dtype(at::kFloat));
    rstd = at::empty({a.n, groups}, x.options().dtype(at::kFloat));
  }
  if (a.r) {
    Tensor ws = gn_workspace(a, groups, false, x);
    check_rc(mace_b200_group_norm_fwd(a.rows.data_ptr(), row_stride(a.rows), ptr(a.w), ptr(a.b), ptr(a.off), a.off64,
                                      y.data_ptr(), ptr_as<float>(mean), ptr_as<float>(rstd), ptr_as<float>(ws), a.r, a.n, a.len,
                                      (int32_t)a.c, (int32_t)groups, eps, (int32_t)act, a.dt, a.pt, stream_of(x)),
             "group_norm");
  } else if (stats) {                             // empty samples, as those among others: the mean 0 and the variance 0
    mean.zero_();
    rstd.fill_(1.f / std::sqrt((float)eps));
  }
  return {y, mean, rstd};
}

Tensor group_norm(const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps, int64_t act,
                  const OptTensor& offsets) {
  return std::get<0>(gn_forward(x, groups, or_none(w), or_none(b), eps, act, or_none(offsets), false));
}

std::tuple<Tensor, Tensor, Tensor> group_norm_fwd(const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b,
                                                  double eps, int64_t act, const OptTensor& offsets) {
  return gn_forward(x, groups, or_none(w), or_none(b), eps, act, or_none(offsets), true);
}

std::tuple<Tensor, Tensor, Tensor> group_norm_bwd(const Tensor& dy, const Tensor& x, int64_t groups, const OptTensor& w,
                                                  const OptTensor& b, int64_t act, const OptTensor& offsets,
                                                  const Tensor& mean, const Tensor& rstd, bool need_x, bool need_w,
                                                  bool need_b) {
  GnIn a = gn_in(x, groups, or_none(w), or_none(b), or_none(offsets), act);
  on_device(dy, "dy", x);
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(), "dy must have the shape and type of x");
  for (const Tensor* t : {&mean, &rstd}) {
    on_device(*t, "mean / rstd", x);
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == a.n * groups,
                "mean / rstd must be float32 with one value per sample and group");
  }
  c10::cuda::CUDAGuard guard(x.device());
  auto popt = x.options().dtype(a.pt == MB_F32 ? at::kFloat : x.scalar_type());
  Tensor dx = need_x ? at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous) : Tensor();
  Tensor dw = need_w ? at::empty({a.c}, popt) : Tensor(), db = need_b ? at::empty({a.c}, popt) : Tensor(), ws;
  if (need_x || need_w || need_b) ws = gn_workspace(a, groups, true, x);
  Tensor g = a.r ? rows_of(dy) : dy;
  if (a.r || need_w || need_b)
    check_rc(mace_b200_group_norm_bwd(ptr(g), a.r ? row_stride(g) : a.c, ptr(a.rows), a.r ? row_stride(a.rows) : a.c, ptr(a.w),
                                      ptr(a.b), ptr(a.off), a.off64, mean.data_ptr<float>(), rstd.data_ptr<float>(), ptr(dx),
                                      ptr(dw), ptr(db), ptr_as<float>(ws), a.r, a.n, a.len, (int32_t)a.c, (int32_t)groups,
                                      (int32_t)act, a.dt, a.pt, stream_of(x)),
             "group_norm_bwd");
  return {dx, dw, db};
}

struct GroupNormGrad : torch::autograd::Function<GroupNormGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps,
                        int64_t act, const OptTensor& offsets) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto fwd = op_of<decltype(group_norm_fwd)>("mace_b200::group_norm_fwd");
    auto [y, mean, rstd] = fwd.call(x, groups, w, b, eps, act, offsets);
    ctx->save_for_backward({x, or_none(w), or_none(b), or_none(offsets), mean, rstd});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("group_norm");
    auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(7);
    // needs_input_grad counts the tensors that were given
    const bool has_w = s[1].defined(), has_b = s[2].defined();
    static auto bwd = op_of<decltype(group_norm_bwd)>("mace_b200::group_norm_bwd");
    auto [dx, dw, db] = bwd.call(g[0], s[0], ctx->saved_data["groups"].toInt(), opt(s[1]), opt(s[2]),
                                 ctx->saved_data["act"].toInt(), opt(s[3]), s[4], s[5], ctx->needs_input_grad(0),
                                 has_w && ctx->needs_input_grad(1), has_b && ctx->needs_input_grad(1 + has_w));
    return {dx, Tensor(), dw, db, Tensor(), Tensor(), Tensor()};
  }
};

Tensor group_norm_autograd(const Tensor& x, int64_t groups, const OptTensor& w, const OptTensor& b, double eps, int64_t act,
                           const OptTensor& offsets) {
  no_dual("group_norm", {&x, &or_none(w), &or_none(b)});
  if (wants_grad({&x, &or_none(w), &or_none(b)})) return GroupNormGrad::apply(x, groups, w, b, eps, act, offsets);
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = op_of<decltype(group_norm)>("mace_b200::group_norm");
  return op.call(x, groups, w, b, eps, act, offsets);
}

// ------------------------------------------------------------------------------------------------ products in 8-bit integers
int64_t pad16(int64_t k) { return (k + 15) / 16 * 16; }

// [rows, k] of 8-bit values as rows that start on 16 bytes: the tensor itself where it has them, else a copy
Tensor rows16(const Tensor& q) {
  const bool ok = q.stride(1) == 1 && (q.size(0) <= 1 || (q.stride(0) % 16 == 0 && q.stride(0) >= q.size(1))) &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
  if (ok) return q;
  Tensor r = at::empty({q.size(0), pad16(q.size(1))}, q.options()).narrow(1, 0, q.size(1));
  r.copy_(q);
  return r;
}
int64_t stride16(const Tensor& q) { return q.size(0) > 1 ? q.stride(0) : pad16(q.size(1)); }

void no_grad_formula(const char* what, std::initializer_list<const Tensor*> ts) {
  TORCH_CHECK(!wants_grad(ts), what, " rounds to whole numbers and has no gradient: call it under torch.no_grad()");
}

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const int32_t dt = type_code(x, "x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= INT32_MAX - 16, "x must have a last dimension of at least 1 (got ",
              x.sizes(), ")");
  const int64_t k = x.size(-1), n = x.numel() / k, ld = pad16(k);
  c10::cuda::CUDAGuard guard(x.device());
  auto shape = x.sizes().vec();
  shape.back() = ld;
  Tensor q = at::empty(shape, x.options().dtype(at::kChar));
  shape.pop_back();
  Tensor scale = at::empty(shape, x.options().dtype(at::kFloat));
  if (n) {
    Tensor r = rows_of(x);
    check_rc(mace_b200_quantize_rows(r.data_ptr(), row_stride(r), q.data_ptr<int8_t>(), ld, scale.data_ptr<float>(), n, (int32_t)k,
                                     dt, stream_of(x)),
             "quantize_rows");
  }
  return {ld == k ? q : q.narrow(-1, 0, k), scale};
}

at::ScalarType type_of_code(int64_t code) {
  TORCH_CHECK(code == MB_F32 || code == MB_BF16 || code == MB_F16, "unknown type ", code);
  return code == MB_F32 ? at::kFloat : code == MB_BF16 ? at::kBFloat16 : at::kHalf;
}

// x: float32 / bfloat16 / float16 tokens (quantized on the way), or 8-bit ones with xscale; out: type of the result
Tensor int8_linear(const Tensor& x, const OptTensor& xscale, const Tensor& w, const Tensor& wscale, const OptTensor& bias,
                   int64_t out) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const bool is8 = x.scalar_type() == at::kChar;
  TORCH_CHECK(is8 == given(xscale), is8 ? "8-bit x needs xscale" : "xscale goes with 8-bit x");
  TORCH_CHECK(x.dim() >= 1, "x must be [.., in]");
  on_device(w, "wq", x);
  TORCH_CHECK(w.dim() == 2 && w.scalar_type() == at::kChar && w.size(0) >= 1 && w.size(1) >= 1, "wq must be int8 [out, in] (got ",
              w.sizes(), ", ", w.scalar_type(), ")");
  const int64_t k = w.size(1), n = w.size(0);
  TORCH_CHECK(x.size(-1) == k, "x must be [.., ", k, "] (got ", x.sizes(), ")");
  TORCH_CHECK(k <= MB_INT8_MAX_K && n <= INT32_MAX - 255, "wq: at most ", MB_INT8_MAX_K, " columns");
  on_device(wscale, "wscale", x);
  TORCH_CHECK(wscale.dim() == 1 && wscale.size(0) == n && wscale.scalar_type() == at::kFloat, "wscale must be float32 [", n, "]");
  const at::ScalarType type = type_of_code(out);
  if (!is8) TORCH_CHECK(x.scalar_type() == type, "the result has the type of x");
  const int64_t t = x.numel() / k;
  TORCH_CHECK(t <= INT32_MAX - 255, "too many tokens (", t, ")");
  int32_t bt = (int32_t)out;
  Tensor b, xs;
  if (given(bias)) {
    on_device(*bias, "bias", x);
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == n && (bias->scalar_type() == type || bias->scalar_type() == at::kFloat),
                "bias must be [", n, "] of the result's type or float32");
    b = bias->contiguous();
    bt = type_code(b, "bias");
  }
  c10::cuda::CUDAGuard guard(x.device());
  auto shape = x.sizes().vec();
  shape.back() = n;
  Tensor y = at::empty(shape, x.options().dtype(type));
  if (t == 0) return y;
  Tensor ws = wscale.contiguous(), wq = rows16(w), q, src;
  if (is8) {
    on_device(*xscale, "xscale", x);
    TORCH_CHECK(xscale->scalar_type() == at::kFloat && xscale->sizes() == x.sizes().slice(0, x.dim() - 1),
                "xscale must be float32 with a value for each token");
    xs = xscale->contiguous();
    q = rows16(rows_of(x));
  } else {
    src = rows_of(x);
    if (!mace_b200_int8_linear_few(t, (int32_t)k)) q = at::empty({t * (pad16(k) + 4)}, w.options());   // rows, then their scales
  }
  int8_t* qp = ptr_as<int8_t>(q);
  float* xp = is8 ? xs.data_ptr<float>() : qp ? reinterpret_cast<float*>(qp + t * pad16(k)) : nullptr;
  check_rc(mace_b200_int8_linear(ptr(src), src.defined() ? row_stride(src) : k, qp, is8 ? stride16(q) : pad16(k), xp,
                                 wq.data_ptr<int8_t>(),
                                 stride16(wq), ws.data_ptr<float>(), ptr(b), y.data_ptr(), t, (int32_t)k, (int32_t)n, (int32_t)out,
                                 bt, stream_of(x)),
           "int8_linear");
  return y;
}

std::tuple<Tensor, Tensor> quantize_rows_autograd(const Tensor& x) {
  no_dual("quantize_rows", {&x});
  no_grad_formula("quantize_rows", {&x});
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = op_of<decltype(quantize_rows)>("mace_b200::quantize_rows");
  return op.call(x);
}

Tensor int8_linear_autograd(const Tensor& x, const OptTensor& xscale, const Tensor& w, const Tensor& wscale, const OptTensor& bias,
                            int64_t out) {
  no_dual("int8_linear", {&x, &or_none(xscale), &wscale, &or_none(bias)});
  no_grad_formula("int8_linear", {&x, &or_none(xscale), &wscale, &or_none(bias)});
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = op_of<decltype(int8_linear)>("mace_b200::int8_linear");
  return op.call(x, xscale, w, wscale, bias, out);
}

// ------------------------------------------------------------------------------------------------ orthogonalised matrices
// coefficients: float64 [steps, 3] in host memory
Tensor orthogonalize(const Tensor& g, const Tensor& coefficients, double eps) {
  TORCH_CHECK(g.is_cuda(), "g must be a CUDA tensor");
  const int32_t dt = type_code(g, "g");
  TORCH_CHECK(g.dim() >= 2, "g must be [.., m, n] (got ", g.sizes(), ")");
  TORCH_CHECK(coefficients.device().is_cpu() && coefficients.scalar_type() == at::kDouble && coefficients.dim() == 2 &&
                  coefficients.size(1) == 3 && coefficients.is_contiguous(),
              "coefficients must be float64 [steps, 3] in host memory");
  const int64_t m = g.size(-2), n = g.size(-1);
  Tensor out = at::empty(g.sizes(), g.options().dtype(at::kBFloat16), at::MemoryFormat::Contiguous);
  if (g.numel() == 0) return out;
  const int64_t batch = g.numel() / (m * n);
  TORCH_CHECK(batch <= 65535 && m <= MB_ORTH_MAX_DIM && n <= MB_ORTH_MAX_DIM, "g: at most 65535 matrices with sides of at most ",
              MB_ORTH_MAX_DIM, " (got ", g.sizes(), ")");
  c10::cuda::CUDAGuard guard(g.device());
  Tensor x = g.dim() == 3 ? g : g.reshape({batch, m, n});
  const bool ok = (n == 1 || x.stride(2) == 1) && (m == 1 || x.stride(1) >= n) && (batch == 1 || x.stride(0) > 0);
  if (!ok) x = x.contiguous();
  int64_t bytes = 0;
  check_rc(mace_b200_orthogonalize_workspace(batch, (int32_t)m, (int32_t)n, &bytes), "orthogonalize");
  Tensor ws = at::empty({bytes}, g.options().dtype(at::kByte));
  check_rc(mace_b200_orthogonalize(x.data_ptr(), batch > 1 ? x.stride(0) : m * n, m > 1 ? x.stride(1) : n, out.data_ptr(),
                                   ws.data_ptr(), batch, (int32_t)m, (int32_t)n, coefficients.data_ptr<double>(),
                                   (int32_t)coefficients.size(0), eps, dt, stream_of(g)),
           "orthogonalize");
  return out;
}

Tensor orthogonalize_autograd(const Tensor& g, const Tensor& coefficients, double eps) {
  no_dual("orthogonalize", {&g});
  TORCH_CHECK(!wants_grad({&g}), "orthogonalize has no gradient formula: call it under torch.no_grad()");
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = op_of<decltype(orthogonalize)>("mace_b200::orthogonalize");
  return op.call(g, coefficients, eps);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mace_b200, m) {
  m.def("group_norm(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act, Tensor? offsets) -> Tensor");
  m.def("group_norm_fwd(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act, Tensor? offsets) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("group_norm_bwd(Tensor dy, Tensor x, int groups, Tensor? weight, Tensor? bias, int act, Tensor? offsets, Tensor mean, "
        "Tensor rstd, bool need_x, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)");
  m.def("orthogonalize(Tensor g, Tensor coefficients, float eps) -> Tensor");
  m.def("quantize_rows(Tensor x) -> (Tensor, Tensor)");
  m.def("int8_linear(Tensor x, Tensor? xscale, Tensor wq, Tensor wscale, Tensor? bias, int out) -> Tensor");
}

TORCH_LIBRARY_IMPL(mace_b200, CUDA, m) {
  m.impl("group_norm", &group_norm);
  m.impl("group_norm_fwd", &group_norm_fwd);
  m.impl("group_norm_bwd", &group_norm_bwd);
  m.impl("orthogonalize", &orthogonalize);
  m.impl("quantize_rows", &quantize_rows);
  m.impl("int8_linear", &int8_linear);
}

TORCH_LIBRARY_IMPL(mace_b200, AutogradCUDA, m) {
  m.impl("group_norm", &group_norm_autograd);
  m.impl("orthogonalize", &orthogonalize_autograd);
  m.impl("quantize_rows", &quantize_rows_autograd);
  m.impl("int8_linear", &int8_linear_autograd);
}

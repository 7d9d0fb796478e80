// What the custom ops of torch_ops_*.cpp share: checks of tensors, row views, dispatch and autograd helpers.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/mace_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* stream_of(const Tensor& t) { return (void*)at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "mace_b200::", what, ": ", mace_b200_last_error(), " (code ", rc, ")");
}

int32_t type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return MB_F32;
    case at::kBFloat16: return MB_BF16;
    case at::kHalf: return MB_F16;
    default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16 (got ", t.scalar_type(), ")");
  }
}

void on_device(const Tensor& t, const char* name, const Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be a CUDA tensor on ", like.device());
}

bool given(const OptTensor& t) { return t && t->defined(); }
const Tensor none;
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
const Tensor& or_none(const OptTensor& t) { return given(t) ? *t : none; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T* ptr_as(const Tensor& t) { return t.defined() ? t.data_ptr<T>() : nullptr; }

// [.., d] as rows of d dense elements a fixed stride apart: the tensor itself where its strides allow it, else a copy
Tensor rows_of(const Tensor& x) {
  Tensor r = x.dim() == 2 ? x : x.dim() == 1 ? x.unsqueeze(0) : x.reshape({-1, x.size(-1)});
  const bool ok = (r.size(1) == 1 || r.stride(1) == 1) && (r.size(0) <= 1 || r.stride(0) >= r.size(1));
  return ok ? r : r.contiguous();
}
int64_t row_stride(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }

// An op through the dispatcher (below autograd: its device kernel, or the shape function of fake tensors)
template <typename Sig>
c10::TypedOperatorHandle<Sig> op_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " can be differentiated once: its gradients have no gradient formula");
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// a tangent would be dropped below autograd
void no_dual(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}

}  // namespace

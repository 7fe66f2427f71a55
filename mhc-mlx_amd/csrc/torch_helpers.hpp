// What the torch bindings of the operators share: dtype codes, checks of
// arguments, layouts, the current stream.
#pragma once

#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "mhc_hip.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

int dtype_code(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return MHC_DTYPE_F32;
    case at::kBFloat16: return MHC_DTYPE_BF16;
    case at::kHalf: return MHC_DTYPE_F16;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t, " of ", what, "; expected float32, bfloat16 or float16");
  }
}

at::ScalarType scalar_type(int64_t code) {
  return code == MHC_DTYPE_BF16 ? at::kBFloat16 : code == MHC_DTYPE_F16 ? at::kHalf : at::kFloat;
}

void check(int rc, const char* what) {
  if (rc == MHC_OK) return;
  const char* msg = mhc_last_error();
  TORCH_CHECK_VALUE(rc > 0, what, ": ", msg ? msg : "invalid argument");
  TORCH_CHECK(false, what, " failed (hip error ", rc, "): ", msg ? msg : "");
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check_on(const at::Tensor& x, const char* name, const at::Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(x.is_cuda(), "the HIP path needs GPU tensors (got ", name, " on ", x.device(), ")");
  TORCH_CHECK_VALUE(t.device() == x.device(), what, " must be on ", name, "'s device ", x.device(), " (got ", t.device(), ")");
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
at::Tensor get(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte).requires_grad(false));
}

// t [..., width] as rows: [R, width] with contiguous elements in a row, the
// rows any distance of at least `width` apart.  Copies only what has no such view.
at::Tensor rows_of(const at::Tensor& t, int64_t width) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
  const bool ok = (width == 1 || r.stride(1) == 1) && (r.size(0) <= 1 || r.stride(0) >= width);
  return ok ? r : r.contiguous();
}

int64_t row_stride(const at::Tensor& rows) { return rows.size(0) <= 1 ? rows.size(1) : rows.stride(0); }

// The backward's results for a caller that asked for their graph: using it raises.
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (const at::Tensor& g : grads)
    if (g.defined()) some.push_back(g);
  if (some.empty()) return grads;
  for (at::Tensor& g : some) g = g.detach().requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is not twice differentiable", (int64_t)some.size());
  variable_list marked = (*node)(std::move(some));
  size_t k = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = marked[k++];
  return grads;
}

bool needs_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

at::TensorOptions f32_options(const at::Tensor& like) { return like.options().dtype(at::kFloat).requires_grad(false); }

}  // namespace

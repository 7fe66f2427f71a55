// Torch binding of the operators of a training step around the mHC layer:
// linear_act, the clipped policy loss and the AdamW step.
//
// Arguments are checked here (ValueError for a rejected one), tensors are
// brought into the layouts that the library reads, and every launch goes to
// the current HIP stream of the tensors' device.  linear_act and policy_loss
// are autograd Functions; the calls under them (linear_fwd, linear_bwd, ...)
// are bound too, for the Python Functions that run under a kernel timer and
// while torch.jit.trace records.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
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

// ---------------------------------------------------------------------------
// linear_act
// ---------------------------------------------------------------------------

struct LinearShape {
  int64_t M, N, K;
  std::vector<int64_t> out;
};

LinearShape linear_check(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& residual,
                         int64_t out_code) {
  check_on(x, "x", w, "weight");
  const int code = dtype_code(x.scalar_type(), "x");
  TORCH_CHECK_VALUE(w.dim() == 2, "weight must be [N, K], got shape ", w.sizes());
  const int64_t N = w.size(0), K = w.size(1);
  TORCH_CHECK_VALUE(N >= 1 && K >= 1, "weight must have elements, got shape ", w.sizes());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K, "x must be [..., K]=[..., ", K, "], got shape ", x.sizes());
  TORCH_CHECK_VALUE(w.scalar_type() == x.scalar_type(), "weight must have x's dtype ", x.scalar_type(), " (got ", w.scalar_type(), ")");
  TORCH_CHECK_VALUE(out_code == code || out_code == MHC_DTYPE_F32, "output_dtype must be x's dtype or float32");
  LinearShape s = {x.numel() / K, N, K, x.sizes().vec()};
  s.out.back() = N;
  if (bias.defined()) {
    check_on(x, "x", bias, "bias");
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == N, "bias must be [N]=[", N, "], got shape ", bias.sizes());
    TORCH_CHECK_VALUE(bias.scalar_type() == x.scalar_type(), "bias must have x's dtype ", x.scalar_type(), " (got ", bias.scalar_type(), ")");
  }
  if (residual.defined()) {
    check_on(x, "x", residual, "residual");
    TORCH_CHECK_VALUE(residual.sizes() == at::IntArrayRef(s.out), "residual must have the output's shape ", at::IntArrayRef(s.out),
                      ", got ", residual.sizes());
    TORCH_CHECK_VALUE(residual.scalar_type() == scalar_type(out_code), "residual must have the output's dtype ", scalar_type(out_code),
                      " (got ", residual.scalar_type(), ")");
  }
  return s;
}

// (out, act' for the backward or an undefined tensor)
std::tuple<at::Tensor, at::Tensor> linear_fwd(const at::Tensor& x, const at::Tensor& w, const OptTensor& bias_,
                                              const OptTensor& residual_, int64_t act, int64_t out_code, bool want_dact) {
  const at::Tensor bias = get(bias_), residual = get(residual_);
  const LinearShape s = linear_check(x, w, bias, residual, out_code);
  const at::DeviceGuard guard(x.device());
  const int code = dtype_code(x.scalar_type(), "x");
  const auto plain = x.options().requires_grad(false);
  at::Tensor out = at::empty(s.out, plain.dtype(scalar_type(out_code))), dact;
  if (want_dact && act != MHC_ACT_NONE) dact = at::empty({s.M, s.N}, plain.dtype(code == MHC_DTYPE_F32 ? at::kFloat : at::kShort));
  if (s.M == 0) return {out, dact};
  const at::Tensor xr = rows_of(x, s.K), wr = rows_of(w, s.K);
  const at::Tensor b = bias.defined() ? bias.contiguous() : bias, r = residual.defined() ? residual.contiguous() : residual;
  const size_t nb = mhc_linear_act_fwd_workspace_bytes(xr.data_ptr(), row_stride(xr), wr.data_ptr(), row_stride(wr), s.M, s.N, s.K, code);
  const at::Tensor ws = nb > 0 ? workspace(nb, x) : at::Tensor();
  check(mhc_linear_act_fwd(xr.data_ptr(), row_stride(xr), wr.data_ptr(), row_stride(wr), ptr(b), ptr(r), out.data_ptr(),
                           (int)out_code, ptr(dact), (int)act, s.M, s.N, s.K, code, ptr(ws), nb, stream_of(x)),
        "mhc_linear_act_fwd");
  return {out, dact};
}

// (dx, dw, db); those not wanted are undefined
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_bwd(const at::Tensor& dout, const OptTensor& dact_, const at::Tensor& x,
                                                          const at::Tensor& w, bool want_dx, bool want_dw, bool want_db) {
  const at::DeviceGuard guard(x.device());
  const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
  const int code = dtype_code(x.scalar_type(), "x");
  const auto plain = x.options().requires_grad(false);
  at::Tensor dx, dw, db;
  if (M == 0) {
    if (want_dx) dx = at::empty(x.sizes(), plain);
    if (want_dw) dw = at::zeros({N, K}, plain);
    if (want_db) db = at::zeros({N}, plain);
    return {dx, dw, db};
  }
  if (want_dx) dx = at::empty(x.sizes(), plain);
  if (want_dw) dw = at::empty({N, K}, plain);
  if (want_db) db = at::empty({N}, plain);
  if (!want_dx && !want_dw && !want_db) return {dx, dw, db};
  const at::Tensor dact = get(dact_), xr = rows_of(x, K), wr = rows_of(w, K);
  const at::Tensor g = (dout.scalar_type() == x.scalar_type() ? dout : dout.to(at::kFloat)).contiguous();
  const int gc = dtype_code(g.scalar_type(), "dout");
  const size_t nb = mhc_linear_act_bwd_workspace_bytes(g.data_ptr(), gc, ptr(dact), xr.data_ptr(), row_stride(xr), wr.data_ptr(),
                                                       row_stride(wr), want_dx, want_dw, want_db, M, N, K, code);
  const at::Tensor ws = workspace(nb, x);
  check(mhc_linear_act_bwd(g.data_ptr(), gc, ptr(dact), xr.data_ptr(), row_stride(xr), wr.data_ptr(), row_stride(wr), ptr(dx),
                           ptr(dw), ptr(db), M, N, K, code, ws.data_ptr(), nb, stream_of(x)),
        "mhc_linear_act_bwd");
  return {dx, dw, db};
}

struct LinearActFn : public torch::autograd::Function<LinearActFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const OptTensor& bias,
                            const OptTensor& residual, int64_t act, int64_t out_code, bool want_dact) {
    auto [out, dact] = linear_fwd(x, w, bias, residual, act, out_code, want_dact);
    ctx->save_for_backward({x, w, dact});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(7);
    if (!grads[0].defined()) return r;
    const auto sv = ctx->get_saved_variables();
    // (an input that was not given has no place among those that a gradient can be asked of)
    const bool bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
    auto [dx, dw, db] = linear_bwd(grads[0], sv[2].defined() ? OptTensor(sv[2]) : OptTensor(), sv[0], sv[1],
                                   ctx->needs_input_grad(0), ctx->needs_input_grad(1), bias && ctx->needs_input_grad(2));
    r[0] = dx;
    r[1] = dw;
    r[2] = db;
    if (residual && ctx->needs_input_grad(bias ? 3 : 2)) r[3] = grads[0];
    return once(std::move(r), "linear_act");
  }
};

bool needs_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

at::Tensor linear_act(const at::Tensor& x, const at::Tensor& w, const OptTensor& bias_, const OptTensor& residual_, int64_t act,
                      int64_t out_code) {
  const at::Tensor bias = get(bias_), residual = get(residual_);
  if (!needs_grad({&x, &w, &bias, &residual})) return std::get<0>(linear_fwd(x, w, bias_, residual_, act, out_code, false));
  linear_check(x, w, bias, residual, out_code);
  return LinearActFn::apply(x, w, bias_, residual_, act, out_code, needs_grad({&x, &w, &bias}));
}

// ---------------------------------------------------------------------------
// Policy loss
// ---------------------------------------------------------------------------

struct PolicyInputs {
  at::Tensor logits, actions, old_logp, advantages, ref_logp, weights;  // as the library reads them
  mhc_policy_args args;
};

PolicyInputs policy_inputs(const at::Tensor& logits, const at::Tensor& actions, const at::Tensor& old_logp,
                           const at::Tensor& advantages, const at::Tensor& ref_logp, const at::Tensor& mask, double clip_low,
                           double clip_high, double kl_coef, double denominator) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be [..., V], got shape ", logits.sizes());
  const int64_t V = logits.size(-1), T = logits.numel() / V;
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  const auto check_one = [&](const at::Tensor& t, const char* name) {
    check_on(logits, "logits", t, name);
    TORCH_CHECK_VALUE(t.sizes() == lead, name, " must have the shape of logits without its last axis, ", lead, ", got ", t.sizes());
  };
  const auto f32 = [&](const at::Tensor& t, const char* name) {
    if (!t.defined()) return t;
    check_one(t, name);
    TORCH_CHECK_VALUE(t.is_floating_point(), name, " must be floating, got ", t.scalar_type());
    return t.detach().to(at::kFloat).contiguous();
  };
  PolicyInputs p;
  p.args = {};
  p.args.dtype = dtype_code(logits.scalar_type(), "logits");
  check_one(actions, "actions");
  TORCH_CHECK_VALUE(actions.scalar_type() == at::kLong || actions.scalar_type() == at::kInt, "actions must be int64 or int32, got ",
                    actions.scalar_type());
  p.logits = rows_of(logits.detach(), V);
  p.actions = actions.to(at::kLong).contiguous();
  p.old_logp = f32(old_logp, "old_logp");
  p.advantages = f32(advantages, "advantages");
  p.ref_logp = f32(ref_logp, "ref_logp");
  if (mask.defined()) {
    check_one(mask, "mask");
    const bool bytes = mask.scalar_type() == at::kBool || mask.scalar_type() == at::kByte;
    TORCH_CHECK_VALUE(bytes || mask.is_floating_point(), "mask must be bool, uint8 or floating weights, got ", mask.scalar_type());
    p.weights = bytes ? mask.contiguous() : mask.detach().to(at::kFloat).contiguous();
    p.args.weights_dtype = bytes ? MHC_DTYPE_U8 : MHC_DTYPE_F32;
  }
  p.args.logits = p.logits.data_ptr();
  p.args.row_stride = row_stride(p.logits);
  p.args.actions = p.actions.data_ptr<int64_t>();
  p.args.old_logp = fptr(p.old_logp);
  p.args.advantages = fptr(p.advantages);
  p.args.ref_logp = fptr(p.ref_logp);
  p.args.weights = ptr(p.weights);
  p.args.T = T;
  p.args.V = V;
  p.args.clip_low = (float)clip_low;
  p.args.clip_high = (float)clip_high;
  p.args.kl_coef = (float)kl_coef;
  p.args.denominator = (float)denominator;
  return p;
}

at::TensorOptions f32_options(const at::Tensor& like) { return like.options().dtype(at::kFloat).requires_grad(false); }

// (loss [], logp [...], stats)
std::tuple<at::Tensor, at::Tensor, at::Tensor> policy_fwd(const at::Tensor& logits, const at::Tensor& actions,
                                                          const at::Tensor& old_logp, const at::Tensor& advantages,
                                                          const OptTensor& ref_logp, const OptTensor& mask, double clip_low,
                                                          double clip_high, double kl_coef, double denominator) {
  const PolicyInputs p = policy_inputs(logits, actions, old_logp, advantages, get(ref_logp), get(mask), clip_low, clip_high,
                                       kl_coef, denominator);
  const at::DeviceGuard guard(logits.device());
  const auto opt = f32_options(logits);
  at::Tensor loss = at::empty({}, opt), logp = at::empty(actions.sizes(), opt), stats = at::empty({3 * p.args.T + 1}, opt);
  const size_t nb = mhc_policy_loss_workspace_bytes(p.args.T);
  const at::Tensor ws = workspace(nb, logits);
  check(mhc_policy_loss_fwd(&p.args, fptr(loss), fptr(logp), fptr(stats), ws.data_ptr(), nb, stream_of(logits)),
        "mhc_policy_loss_fwd");
  return {loss, logp, stats};
}

at::Tensor policy_bwd(const at::Tensor& logits, const at::Tensor& actions, const at::Tensor& old_logp, const at::Tensor& advantages,
                      const OptTensor& ref_logp, const OptTensor& mask, double clip_low, double clip_high, double kl_coef,
                      double denominator, const at::Tensor& stats, const at::Tensor& dloss) {
  const PolicyInputs p = policy_inputs(logits, actions, old_logp, advantages, get(ref_logp), get(mask), clip_low, clip_high,
                                       kl_coef, denominator);
  const at::DeviceGuard guard(logits.device());
  at::Tensor dlogits = at::empty(logits.sizes(), logits.options().requires_grad(false));
  const at::Tensor d = dloss.to(at::kFloat).contiguous();
  check(mhc_policy_loss_bwd(&p.args, fptr(stats), fptr(d), dlogits.data_ptr(), stream_of(logits)), "mhc_policy_loss_bwd");
  return dlogits;
}

// (loss, logp, dlogits)
std::tuple<at::Tensor, at::Tensor, at::Tensor> policy_loss_and_grad(const at::Tensor& logits, const at::Tensor& actions,
                                                                    const at::Tensor& old_logp, const at::Tensor& advantages,
                                                                    const OptTensor& ref_logp, const OptTensor& mask,
                                                                    double clip_low, double clip_high, double kl_coef,
                                                                    double denominator, double grad_scale) {
  const PolicyInputs p = policy_inputs(logits, actions, old_logp, advantages, get(ref_logp), get(mask), clip_low, clip_high,
                                       kl_coef, denominator);
  const at::DeviceGuard guard(logits.device());
  const auto opt = f32_options(logits);
  at::Tensor loss = at::empty({}, opt), logp = at::empty(actions.sizes(), opt);
  at::Tensor dlogits = at::empty(logits.sizes(), logits.options().requires_grad(false));
  const size_t nb = mhc_policy_loss_workspace_bytes(p.args.T);
  const at::Tensor ws = workspace(nb, logits);
  check(mhc_policy_loss_fwd_bwd(&p.args, (float)grad_scale, fptr(loss), fptr(logp), dlogits.data_ptr(), ws.data_ptr(), nb,
                                stream_of(logits)),
        "mhc_policy_loss_fwd_bwd");
  return {loss, logp, dlogits};
}

struct PolicyLossFn : public torch::autograd::Function<PolicyLossFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& actions, const at::Tensor& old_logp,
                               const at::Tensor& advantages, const OptTensor& ref_logp, const OptTensor& mask, double clip_low,
                               double clip_high, double kl_coef, double denominator) {
    auto [loss, logp, stats] = policy_fwd(logits, actions, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef,
                                          denominator);
    ctx->save_for_backward({logits, actions, old_logp, advantages, get(ref_logp), get(mask), stats});
    ctx->saved_data["clip_low"] = clip_low;
    ctx->saved_data["clip_high"] = clip_high;
    ctx->saved_data["kl_coef"] = kl_coef;
    ctx->saved_data["denominator"] = denominator;
    ctx->mark_non_differentiable({logp});
    ctx->set_materialize_grads(false);
    return {loss, logp};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(10);
    if (!grads[0].defined()) return r;
    const auto sv = ctx->get_saved_variables();
    const auto opt = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const auto num = [&](const char* name) { return ctx->saved_data[name].toDouble(); };
    r[0] = policy_bwd(sv[0], sv[1], sv[2], sv[3], opt(sv[4]), opt(sv[5]), num("clip_low"), num("clip_high"), num("kl_coef"),
                      num("denominator"), sv[6], grads[0]);
    return once(std::move(r), "policy_loss");
  }
};

std::tuple<at::Tensor, at::Tensor> policy_loss(const at::Tensor& logits, const at::Tensor& actions, const at::Tensor& old_logp,
                                               const at::Tensor& advantages, const OptTensor& ref_logp, const OptTensor& mask,
                                               double clip_low, double clip_high, double kl_coef, double denominator) {
  if (!needs_grad({&logits})) {
    auto [loss, logp, stats] = policy_fwd(logits, actions, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef,
                                          denominator);
    return {loss, logp};
  }
  const auto plain = [](const OptTensor& t) { return t.has_value() ? OptTensor(t->detach()) : t; };
  variable_list r = PolicyLossFn::apply(logits, actions, old_logp.detach(), advantages.detach(), plain(ref_logp), plain(mask),
                                        clip_low, clip_high, kl_coef, denominator);
  return {r[0], r[1]};
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------

// A Python list or tuple of tensors, read in place: hundreds of them would
// take longer to convert than the step takes.
struct TensorSeq {
  PyObject* seq = nullptr;  // borrowed from the caller's argument, or the fast sequence of it
  py::object held;

  TensorSeq(const py::object& o, const char* name) {
    if (o.is_none()) return;
    held = py::reinterpret_steal<py::object>(PySequence_Fast(o.ptr(), ""));
    if (!held) {
      PyErr_Clear();
      TORCH_CHECK_VALUE(false, name, " must be a list of tensors");
    }
    seq = held.ptr();
  }
  bool given() const { return seq != nullptr; }
  size_t size() const { return (size_t)PySequence_Fast_GET_SIZE(seq); }
  // entry i, or nullptr for None
  const at::Tensor* get(size_t i, const char* name) const {
    PyObject* o = PySequence_Fast_GET_ITEM(seq, (Py_ssize_t)i);
    if (o == Py_None) return nullptr;
    TORCH_CHECK_VALUE(THPVariable_Check(o), name, "[", i, "] is no tensor");
    return &THPVariable_Unpack(o);
  }
  const at::Tensor& at(size_t i, const char* name) const {
    const at::Tensor* t = get(i, name);
    TORCH_CHECK_VALUE(t != nullptr, name, "[", i, "] is None");
    return *t;
  }
};

// elements in the same order in memory, without holes
bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  return a.sizes() == b.sizes() && (a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous()));
}


void adamw_step(const py::object& params_, const py::object& grads_, const py::object& exp_avgs_, const py::object& exp_avg_sqs_,
                const py::object& masters_, const py::object& scales_, int64_t step, double lr, double beta1, double beta2, double eps,
                double weight_decay, double grad_scale, const OptTensor& grad_scale_tensor) {
  const TensorSeq params(params_, "params"), grads(grads_, "grads"), exp_avgs(exp_avgs_, "exp_avgs"),
      exp_avg_sqs(exp_avg_sqs_, "exp_avg_sqs"), masters(masters_, "masters"), scales(scales_, "scales");
  TORCH_CHECK_VALUE(params.given() && grads.given() && exp_avgs.given() && exp_avg_sqs.given(),
                    "params, grads, exp_avgs and exp_avg_sqs must be lists of tensors");
  const size_t n = params.size();
  const auto same = [&](const TensorSeq& s, const char* name) {
    TORCH_CHECK_VALUE(!s.given() || s.size() == n, name, " must have one entry for each of the ", n, " params, got ", s.size());
  };
  same(grads, "grads");
  same(exp_avgs, "exp_avgs");
  same(exp_avg_sqs, "exp_avg_sqs");
  same(masters, "masters");
  same(scales, "scales");
  if (n == 0) return;
  const at::Device dev = params.at(0, "params").device();
  TORCH_CHECK_VALUE(dev.is_cuda(), "the HIP path needs GPU tensors (got params[0] on ", dev, ")");
  const bool q8 = scales.given();
  const at::ScalarType st = q8 ? at::kFloat8_e4m3fn : at::kFloat;
  std::vector<at::Tensor> held;  // gradients brought into their parameter's layout
  // one call of the library for each kind: dtype, and with or without a master copy
  std::vector<mhc_adamw_tensor> of[6];
  std::vector<c10::TensorImpl*> written;
  written.reserve(n * (3 + masters.given() + q8));
  const auto bytes = [&](const at::Tensor& t) {  // of a tensor that the step writes
    written.push_back(t.unsafeGetTensorImpl());
    return t.unsafeGetTensorImpl()->mutable_data();
  };
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &p = params.at(i, "params"), &m = exp_avgs.at(i, "exp_avgs"), &v = exp_avg_sqs.at(i, "exp_avg_sqs");
    const at::Tensor* g = &grads.at(i, "grads");
    const int code = dtype_code(p.scalar_type(), "params");
    TORCH_CHECK_VALUE(p.layout() == at::kStrided && g->layout() == at::kStrided, "tensor ", i, ": params and grads must be dense");
    TORCH_CHECK_VALUE(p.device() == dev && g->device() == dev && m.device() == dev && v.device() == dev, "tensor ", i,
                      ": every tensor must be on ", dev);
    TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "tensor ", i, ": params must have their elements without holes or overlaps, got shape ",
                      p.sizes(), " with strides ", p.strides());
    TORCH_CHECK_VALUE(g->sizes() == p.sizes() && g->scalar_type() == p.scalar_type(), "tensor ", i,
                      ": the gradient must have the parameter's shape ", p.sizes(), " and dtype ", p.scalar_type(), ", got ", g->sizes(), " ",
                      g->scalar_type());
    TORCH_CHECK_VALUE(m.scalar_type() == st && v.scalar_type() == st && same_layout(p, m) && same_layout(p, v), "tensor ", i,
                      ": the states must be ", st, " in the parameter's shape and layout");
    if (!same_layout(p, *g)) {
      held.push_back(at::empty_like(p).copy_(*g));
      g = &held.back();
    }
    mhc_adamw_tensor t = {bytes(p), g->const_data_ptr(), nullptr, bytes(m), bytes(v), nullptr, p.numel()};
    if (masters.given()) {
      if (const at::Tensor* w = masters.get(i, "masters")) {
        TORCH_CHECK_VALUE(code != MHC_DTYPE_F32, "tensor ", i, ": a master copy is for 16-bit parameters");
        TORCH_CHECK_VALUE(w->device() == dev && w->scalar_type() == at::kFloat && same_layout(p, *w), "tensor ", i,
                          ": the master copy must be float32 in the parameter's shape and layout");
        t.master = static_cast<float*>(bytes(*w));
      }
    }
    if (q8) {
      const int64_t want = 2 * ((p.numel() + 255) / 256);
      const at::Tensor& s = scales.at(i, "scales");
      TORCH_CHECK_VALUE(s.device() == dev && s.scalar_type() == at::kFloat && s.is_contiguous() && s.numel() == want, "tensor ", i,
                        ": scales must be contiguous float32 [ceil(numel / 256), 2] on ", dev);
      t.scales = static_cast<float*>(bytes(s));
    }
    if (of[2 * code + (t.master != nullptr)].empty()) of[2 * code + (t.master != nullptr)].reserve(n);
    of[2 * code + (t.master != nullptr)].push_back(t);
  }
  const float* gs = nullptr;
  if (grad_scale_tensor.has_value()) {
    const at::Tensor& gst = *grad_scale_tensor;
    TORCH_CHECK_VALUE(gst.device() == dev && gst.numel() == 1 && gst.scalar_type() == at::kFloat, "grad_scale must be a number or one float32 on ",
                      dev);
    gs = gst.data_ptr<float>();
  }
  const at::DeviceGuard guard(dev);
  void* const stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  for (int k = 0; k < 6; ++k)
    if (!of[k].empty())
      check(mhc_adamw_step(of[k].data(), (int64_t)of[k].size(), k / 2, q8 ? 8 : 32, lr, beta1, beta2, eps, weight_decay, step,
                           grad_scale, gs, stream),
            "mhc_adamw_step");
  for (c10::TensorImpl* t : written)  // modified, for graphs that saved it
    if (!t->is_inference()) t->bump_version();
}

}  // namespace

void bind_train(py::module_& m) {
  m.def("linear_act", &linear_act, "act(x W^T + bias) + residual with its backward in C++");
  m.def("linear_fwd", &linear_fwd, "linear_act's output and act' (None if not asked for), without autograd");
  m.def("linear_bwd", &linear_bwd, "gradients of x, weight and bias (None where not asked for)");
  m.def("policy_loss", &policy_loss, "clipped policy loss and log probabilities with the backward in C++");
  m.def("policy_fwd", &policy_fwd, "the loss, the log probabilities and what the backward reads, without autograd");
  m.def("policy_bwd", &policy_bwd, "gradient of the logits");
  m.def("policy_loss_and_grad", &policy_loss_and_grad, "loss, log probabilities and gradient in one call, without autograd");
  m.def("adamw_step", &adamw_step, "one AdamW step over lists of tensors, in place");
}

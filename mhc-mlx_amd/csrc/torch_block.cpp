// Torch binding of the operators between the residual stream and a model's
// answer: the RMS norm with the residual's addition, int8 rows and their
// product, and the cross entropy from hidden states.  Arguments are checked
// here, as in torch_train.cpp.
#include "torch_helpers.hpp"

namespace {

// ---------------------------------------------------------------------------
// RMS norm
// ---------------------------------------------------------------------------

struct NormInputs {
  at::Tensor x, r, w;  // as the library reads them
  int64_t T, C;
  int code, w_code;
};

void norm_check(const at::Tensor& x, const at::Tensor& r, const at::Tensor& w) {
  TORCH_CHECK_VALUE(x.is_cuda(), "the HIP path needs GPU tensors (got x on ", x.device(), ")");
  dtype_code(x.scalar_type(), "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., C], got shape ", x.sizes());
  if (r.defined()) {
    check_on(x, "x", r, "residual");
    TORCH_CHECK_VALUE(r.sizes() == x.sizes(), "residual must have x's shape ", x.sizes(), ", got ", r.sizes());
    TORCH_CHECK_VALUE(r.scalar_type() == x.scalar_type(), "residual must have x's dtype ", x.scalar_type(), " (got ", r.scalar_type(), ")");
  }
  if (w.defined()) {
    check_on(x, "x", w, "weight");
    TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(-1), "weight must be [C]=[", x.size(-1), "], got shape ", w.sizes());
    TORCH_CHECK_VALUE(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "weight must have x's dtype ", x.scalar_type(),
                      " or float32 (got ", w.scalar_type(), ")");
  }
}

NormInputs norm_inputs(const at::Tensor& x, const at::Tensor& r, const at::Tensor& w) {
  norm_check(x, r, w);
  NormInputs n;
  n.C = x.size(-1);
  n.T = x.numel() / n.C;
  n.code = dtype_code(x.scalar_type(), "x");
  n.x = rows_of(x, n.C);
  if (r.defined()) n.r = rows_of(r, n.C);
  if (w.defined()) n.w = w.contiguous();
  n.w_code = w.defined() ? dtype_code(w.scalar_type(), "weight") : n.code;
  return n;
}

int64_t stride_of(const at::Tensor& rows) { return rows.defined() ? row_stride(rows) : 0; }

// (y, h or undefined without a residual, the rows' factors or undefined)
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_fwd(const at::Tensor& x, const OptTensor& r, const OptTensor& w, double eps,
                                                                bool want_rstd) {
  const NormInputs n = norm_inputs(x, get(r), get(w));
  const at::DeviceGuard guard(x.device());
  const auto plain = x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor y = at::empty(x.sizes(), plain), h, rstd;
  if (n.r.defined()) h = at::empty(x.sizes(), plain);
  if (want_rstd) rstd = at::empty({n.T}, f32_options(x));
  check(mhc_add_rms_norm_fwd(ptr(n.x), stride_of(n.x), ptr(n.r), stride_of(n.r), ptr(n.w), n.w_code, ptr(h), y.data_ptr(), fptr(rstd), n.T, n.C,
                             n.code, (float)eps, stream_of(x)),
        "mhc_add_rms_norm_fwd");
  return {y, h, rstd};
}

// (dx, which is the residual's gradient too, dw); those not wanted are undefined
std::tuple<at::Tensor, at::Tensor> add_rms_norm_bwd(const OptTensor& dy_, const OptTensor& dh_, const at::Tensor& h, const at::Tensor& rstd,
                                                    const OptTensor& w_, bool want_dx, bool want_dw) {
  const at::Tensor dy = get(dy_), dh = get(dh_), w = get(w_);
  const at::DeviceGuard guard(h.device());
  const int64_t C = h.size(-1), T = h.numel() / C;
  const auto plain = h.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor dx, dw;
  if (!dy.defined() || T == 0) {
    if (want_dx) dx = dh.defined() ? dh : at::empty(h.sizes(), plain);
    if (want_dw) dw = at::zeros({C}, w.options().requires_grad(false));
    return {dx, dw};
  }
  const int code = dtype_code(h.scalar_type(), "x"), w_code = w.defined() ? dtype_code(w.scalar_type(), "weight") : code;
  if (want_dx) dx = at::empty(h.sizes(), plain);
  if (want_dw) dw = at::empty({C}, w.options().requires_grad(false));
  const at::Tensor hr = rows_of(h, C), gy = rows_of(dy.to(h.scalar_type()), C), gh = dh.defined() ? rows_of(dh.to(h.scalar_type()), C) : dh;
  const at::Tensor wc = w.defined() ? w.contiguous() : w;
  const size_t nb = want_dw ? mhc_add_rms_norm_bwd_workspace_bytes(T, C, code) : 0;
  const at::Tensor ws = nb > 0 ? workspace(nb, h) : at::Tensor();
  check(mhc_add_rms_norm_bwd(ptr(gy), stride_of(gy), ptr(gh), stride_of(gh), ptr(hr), stride_of(hr), rstd.data_ptr<float>(), ptr(wc), w_code,
                             ptr(dx), ptr(dw), T, C, code, ptr(ws), nb, stream_of(h)),
        "mhc_add_rms_norm_bwd");
  return {dx, dw};
}

struct AddRmsNormFn : public torch::autograd::Function<AddRmsNormFn> {
  // y, and h if there is a residual
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& r, const OptTensor& w, double eps) {
    auto [y, h, rstd] = add_rms_norm_fwd(x, r, w, eps, true);
    ctx->save_for_backward({h.defined() ? h : x, rstd, get(w)});
    ctx->saved_data["residual"] = r.has_value();
    ctx->saved_data["weight"] = w.has_value();
    ctx->set_materialize_grads(false);
    if (!h.defined()) return {y};
    return {y, h};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    const bool residual = ctx->saved_data["residual"].toBool(), weight = ctx->saved_data["weight"].toBool();
    const at::Tensor dy = grads[0], dh = residual ? grads[1] : at::Tensor();
    if (!dy.defined() && !dh.defined()) return out;
    const auto sv = ctx->get_saved_variables();
    const auto opt = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    // (an input that was not given has no place among those that a gradient can be asked of)
    const bool of_x = ctx->needs_input_grad(0), of_r = residual && ctx->needs_input_grad(1);
    const bool of_w = weight && ctx->needs_input_grad(residual ? 2 : 1);
    auto [dx, dw] = add_rms_norm_bwd(opt(dy), opt(dh), sv[0], sv[1], opt(sv[2]), of_x || of_r, of_w);
    if (of_x) out[0] = dx;
    if (of_r) out[1] = dx;
    out[2] = dw;
    return once(std::move(out), "add_rms_norm");
  }
};

// (y, h); h is x without a residual
std::tuple<at::Tensor, at::Tensor> add_rms_norm(const at::Tensor& x, const OptTensor& r, const OptTensor& w, double eps) {
  const at::Tensor residual = get(r), weight = get(w);
  if (!needs_grad({&x, &residual, &weight})) {
    auto [y, h, rstd] = add_rms_norm_fwd(x, r, w, eps, false);
    return {y, h.defined() ? h : x};
  }
  norm_check(x, residual, weight);
  variable_list out = AddRmsNormFn::apply(x, r, w, eps);
  return {out[0], out.size() > 1 ? out[1] : x};
}

// (codes, scales, h or undefined without a residual)
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_int8(const at::Tensor& x, const OptTensor& r, const OptTensor& w, double eps) {
  const at::AutoGradMode plain_mode(false);
  const NormInputs n = norm_inputs(x, get(r), get(w));
  const at::DeviceGuard guard(x.device());
  const auto plain = x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor codes = at::empty(x.sizes(), plain.dtype(at::kChar)), scales = at::empty(x.sizes().slice(0, x.dim() - 1), f32_options(x)), h;
  if (n.r.defined()) h = at::empty(x.sizes(), plain);
  check(mhc_add_rms_norm_int8(ptr(n.x), stride_of(n.x), ptr(n.r), stride_of(n.r), ptr(n.w), n.w_code, ptr(h), codes.data_ptr<int8_t>(),
                              scales.data_ptr<float>(), n.T, n.C, n.code, (float)eps, stream_of(x)),
        "mhc_add_rms_norm_int8");
  return {codes, scales, h};
}

// ---------------------------------------------------------------------------
// int8 rows and their product
// ---------------------------------------------------------------------------

// (codes, scales)
std::tuple<at::Tensor, at::Tensor> quantize_int8(const at::Tensor& x) {
  const at::AutoGradMode plain_mode(false);
  const NormInputs n = norm_inputs(x, at::Tensor(), at::Tensor());
  const at::DeviceGuard guard(x.device());
  at::Tensor codes = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous).dtype(at::kChar));
  at::Tensor scales = at::empty(x.sizes().slice(0, x.dim() - 1), f32_options(x));
  check(mhc_quantize_int8(ptr(n.x), stride_of(n.x), codes.data_ptr<int8_t>(), scales.data_ptr<float>(), n.T, n.C, n.code, stream_of(x)),
        "mhc_quantize_int8");
  return {codes, scales};
}

void check_rows(const at::Tensor& like, const at::Tensor& codes, const at::Tensor& scales, const char* name) {
  check_on(like, "x", codes, name);
  check_on(like, "x", scales, name);
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kChar, name, ": codes must be int8, got ", codes.scalar_type());
  TORCH_CHECK_VALUE(codes.dim() >= 1 && codes.size(-1) >= 1, name, ": codes must be [..., K], got shape ", codes.sizes());
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat, name, ": scales must be float32, got ", scales.scalar_type());
  TORCH_CHECK_VALUE(scales.sizes() == codes.sizes().slice(0, codes.dim() - 1), name, ": scales must have the shape of codes without its last axis, ",
                    codes.sizes().slice(0, codes.dim() - 1), ", got ", scales.sizes());
}

at::Tensor dequantize_int8(const at::Tensor& codes, const at::Tensor& scales, int64_t out_code) {
  check_rows(codes, codes, scales, "rows");
  const at::DeviceGuard guard(codes.device());
  const int64_t C = codes.size(-1), T = codes.numel() / C;
  const at::Tensor rows = rows_of(codes, C), s = scales.contiguous();
  at::Tensor out = at::empty(codes.sizes(), codes.options().memory_format(at::MemoryFormat::Contiguous).dtype(scalar_type(out_code)));
  check(mhc_dequantize_int8(rows.data_ptr<int8_t>(), row_stride(rows), s.data_ptr<float>(), out.data_ptr(), (int)out_code, T, C, stream_of(codes)),
        "mhc_dequantize_int8");
  return out;
}

at::Tensor linear_int8(const at::Tensor& x, const at::Tensor& x_scales, const at::Tensor& w, const at::Tensor& w_scales, const OptTensor& bias_,
                       const OptTensor& residual_, int64_t act, int64_t out_code) {
  const at::AutoGradMode plain_mode(false);
  check_rows(x, x, x_scales, "x");
  check_rows(x, w, w_scales, "weight");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 1, "weight: codes must be [N, K], got shape ", w.sizes());
  const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
  TORCH_CHECK_VALUE(x.size(-1) == K, "x: codes must be [..., K]=[..., ", K, "], got shape ", x.sizes());
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  at::Tensor bias = get(bias_), residual = get(residual_);
  if (bias.defined()) {
    check_on(x, "x", bias, "bias");
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == N, "bias must be [N]=[", N, "], got shape ", bias.sizes());
    TORCH_CHECK_VALUE(bias.is_floating_point(), "bias must be floating, got ", bias.scalar_type());
  }
  if (residual.defined()) {
    check_on(x, "x", residual, "residual");
    TORCH_CHECK_VALUE(residual.sizes() == at::IntArrayRef(shape), "residual must have the output's shape ", at::IntArrayRef(shape), ", got ",
                      residual.sizes());
    TORCH_CHECK_VALUE(residual.scalar_type() == scalar_type(out_code), "residual must have the output's dtype ", scalar_type(out_code), " (got ",
                      residual.scalar_type(), ")");
  }
  const at::DeviceGuard guard(x.device());
  at::Tensor out = at::empty(shape, x.options().dtype(scalar_type(out_code)));
  if (M == 0) return out;
  if (bias.defined()) bias = bias.to(at::kFloat).contiguous();
  if (residual.defined()) residual = residual.contiguous();
  const at::Tensor xr = rows_of(x, K), wr = rows_of(w, K), xs = x_scales.contiguous(), wsc = w_scales.contiguous();
  const int8_t *xp = xr.data_ptr<int8_t>(), *wp = wr.data_ptr<int8_t>();
  const size_t nb = mhc_linear_int8_workspace_bytes(xp, row_stride(xr), wp, row_stride(wr), M, N, K);
  const at::Tensor ws = nb > 0 ? workspace(nb, x) : at::Tensor();
  check(mhc_linear_int8(xp, row_stride(xr), xs.data_ptr<float>(), wp, row_stride(wr), wsc.data_ptr<float>(), fptr(bias), ptr(residual), out.data_ptr(),
                        (int)out_code, (int)act, M, N, K, ptr(ws), nb, stream_of(x)),
        "mhc_linear_int8");
  return out;
}

// ---------------------------------------------------------------------------
// Cross entropy
// ---------------------------------------------------------------------------

struct CeInputs {
  at::Tensor x, w, targets, weights;  // as the library reads them
  mhc_linear_ce_args args;
};

CeInputs ce_inputs(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, const at::Tensor& mask, double denominator,
                   int64_t ignore_index) {
  check_on(x, "x", w, "weight");
  check_on(x, "x", targets, "targets");
  CeInputs c;
  c.args = {};
  c.args.dtype = dtype_code(x.scalar_type(), "x");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 1 && w.size(1) >= 1, "weight must be [V, C], got shape ", w.sizes());
  const int64_t C = w.size(1);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == C, "x must be [..., C]=[..., ", C, "], got shape ", x.sizes());
  TORCH_CHECK_VALUE(w.scalar_type() == x.scalar_type(), "weight must have x's dtype ", x.scalar_type(), " (got ", w.scalar_type(), ")");
  const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
  TORCH_CHECK_VALUE(targets.sizes() == lead, "targets must have the shape of x without its last axis, ", lead, ", got ", targets.sizes());
  TORCH_CHECK_VALUE(targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt, "targets must be int64 or int32, got ",
                    targets.scalar_type());
  c.x = rows_of(x.detach(), C);
  c.w = rows_of(w.detach(), C);
  c.targets = targets.to(at::kLong).contiguous();
  if (mask.defined()) {
    check_on(x, "x", mask, "mask");
    TORCH_CHECK_VALUE(mask.sizes() == lead, "mask must have the shape of x without its last axis, ", lead, ", got ", mask.sizes());
    const bool bytes = mask.scalar_type() == at::kBool || mask.scalar_type() == at::kByte;
    TORCH_CHECK_VALUE(bytes || mask.is_floating_point(), "mask must be bool, uint8 or floating weights, got ", mask.scalar_type());
    c.weights = bytes ? mask.contiguous() : mask.detach().to(at::kFloat).contiguous();
    c.args.weights_dtype = bytes ? MHC_DTYPE_U8 : MHC_DTYPE_F32;
  }
  c.args.x = ptr(c.x);
  c.args.ldx = row_stride(c.x);
  c.args.w = ptr(c.w);
  c.args.ldw = row_stride(c.w);
  c.args.targets = c.targets.data_ptr<int64_t>();
  c.args.weights = ptr(c.weights);
  c.args.T = x.numel() / C;
  c.args.V = w.size(0);
  c.args.C = C;
  c.args.ignore_index = ignore_index;
  c.args.denominator = (float)denominator;
  return c;
}

struct CeResult {
  at::Tensor loss, logp, state;
};

// What the forward leaves: its state and, after it, the logits that are kept.
size_t ce_state_bytes(const CeInputs& c) { return (mhc_linear_ce_state_bytes(c.args.T) + 255) / 256 * 256; }

CeResult ce_forward(CeInputs& c, const at::Tensor& x, bool keep) {
  const auto opt = f32_options(x);
  const size_t kept = keep ? mhc_linear_ce_logits_bytes(&c.args) : 0;
  CeResult r = {at::empty({}, opt), at::empty(x.sizes().slice(0, x.dim() - 1), opt), workspace(ce_state_bytes(c) + kept, x)};
  if (kept > 0) c.args.logits = reinterpret_cast<float*>(static_cast<char*>(r.state.data_ptr()) + ce_state_bytes(c));
  const size_t nb = mhc_linear_ce_fwd_workspace_bytes(&c.args);
  const at::Tensor ws = workspace(nb, x);
  check(mhc_linear_ce_fwd(&c.args, fptr(r.loss), fptr(r.logp), r.state.data_ptr(), ws.data_ptr(), nb, stream_of(x)), "mhc_linear_ce_fwd");
  return r;
}

std::tuple<at::Tensor, at::Tensor> ce_backward(CeInputs& c, const at::Tensor& x, const at::Tensor& w, const at::Tensor& state,
                                               const at::Tensor& dloss, double grad_scale, bool want_dx, bool want_dw) {
  at::Tensor dx, dw;
  if (want_dx) dx = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
  if (want_dw) dw = at::empty(w.sizes(), w.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
  if (c.args.T == 0) {
    if (want_dw) dw.zero_();
    return {dx, dw};
  }
  if ((size_t)state.numel() > ce_state_bytes(c)) c.args.logits = reinterpret_cast<float*>(static_cast<char*>(state.data_ptr()) + ce_state_bytes(c));
  const size_t nb = mhc_linear_ce_bwd_workspace_bytes(&c.args, want_dx, want_dw);
  const at::Tensor ws = workspace(nb, x);
  check(mhc_linear_ce_bwd(&c.args, state.data_ptr(), fptr(dloss), (float)grad_scale, ptr(dx), ptr(dw), ws.data_ptr(), nb, stream_of(x)),
        "mhc_linear_ce_bwd");
  return {dx, dw};
}

// (loss [], logp [...], what the backward reads: of a call that will have one, with `keep`)
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_ce_fwd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets,
                                                             const OptTensor& mask, double denominator, int64_t ignore_index, bool keep) {
  CeInputs c = ce_inputs(x, w, targets, get(mask), denominator, ignore_index);
  const at::DeviceGuard guard(x.device());
  const CeResult r = ce_forward(c, x, keep);
  return {r.loss, r.logp, r.state};
}

// (dx, dw); those not wanted are undefined
std::tuple<at::Tensor, at::Tensor> linear_ce_bwd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, const OptTensor& mask,
                                                 double denominator, int64_t ignore_index, const at::Tensor& state, const at::Tensor& dloss,
                                                 bool want_dx, bool want_dw) {
  CeInputs c = ce_inputs(x, w, targets, get(mask), denominator, ignore_index);
  const at::DeviceGuard guard(x.device());
  return ce_backward(c, x, w, state, dloss.to(at::kFloat).contiguous(), 1.0, want_dx, want_dw);
}

// (loss, logp, dx, dw)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> linear_ce_and_grad(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets,
                                                                              const OptTensor& mask, double denominator, int64_t ignore_index,
                                                                              double grad_scale, bool keep) {
  const at::AutoGradMode plain_mode(false);
  CeInputs c = ce_inputs(x, w, targets, get(mask), denominator, ignore_index);
  const at::DeviceGuard guard(x.device());
  const CeResult r = ce_forward(c, x, keep);
  auto [dx, dw] = ce_backward(c, x, w, r.state, at::Tensor(), grad_scale, true, true);
  return {r.loss, r.logp, dx, dw};
}

struct LinearCeFn : public torch::autograd::Function<LinearCeFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, const OptTensor& mask,
                               double denominator, int64_t ignore_index, bool keep) {
    auto [loss, logp, state] = linear_ce_fwd(x, w, targets, mask, denominator, ignore_index, keep);
    ctx->save_for_backward({x, w, targets, get(mask), state});
    ctx->saved_data["denominator"] = denominator;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->mark_non_differentiable({logp});
    ctx->set_materialize_grads(false);
    return {loss, logp};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list r(7);
    if (!grads[0].defined()) return r;
    const auto sv = ctx->get_saved_variables();
    auto [dx, dw] = linear_ce_bwd(sv[0], sv[1], sv[2], sv[3].defined() ? OptTensor(sv[3]) : OptTensor(), ctx->saved_data["denominator"].toDouble(),
                                  ctx->saved_data["ignore_index"].toInt(), sv[4], grads[0], ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    r[0] = dx;
    r[1] = dw;
    return once(std::move(r), "linear_cross_entropy");
  }
};

std::tuple<at::Tensor, at::Tensor> linear_ce(const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets, const OptTensor& mask,
                                             double denominator, int64_t ignore_index, bool keep) {
  if (!needs_grad({&x, &w})) {
    auto [loss, logp, state] = linear_ce_fwd(x, w, targets, mask, denominator, ignore_index, false);
    return {loss, logp};
  }
  variable_list r = LinearCeFn::apply(x, w, targets, mask.has_value() ? OptTensor(mask->detach()) : mask, denominator, ignore_index, keep);
  return {r[0], r[1]};
}

}  // namespace

void bind_block(py::module_& m) {
  m.def("add_rms_norm", &add_rms_norm, "(normed x + residual, the sum) with the backward in C++");
  m.def("add_rms_norm_fwd", &add_rms_norm_fwd, "the normed rows, the sum (None without a residual) and the rows' factors, without autograd");
  m.def("add_rms_norm_bwd", &add_rms_norm_bwd, "gradients of x (and the residual) and of the weight (None where not asked for)");
  m.def("add_rms_norm_int8", &add_rms_norm_int8, "codes and scales of the normed rows, and the sum");
  m.def("quantize_int8", &quantize_int8, "codes and scales of rows");
  m.def("dequantize_int8", &dequantize_int8, "the values of int8 rows");
  m.def("linear_int8", &linear_int8, "product of int8 rows with scales, bias, activation and residual");
  m.def("linear_ce", &linear_ce, "cross entropy from hidden states with the backward in C++");
  m.def("linear_ce_fwd", &linear_ce_fwd, "the loss, the log probabilities and what the backward reads, without autograd");
  m.def("linear_ce_bwd", &linear_ce_bwd, "gradients of the hidden states and of the weight (None where not asked for)");
  m.def("linear_ce_and_grad", &linear_ce_and_grad, "loss, log probabilities and gradients in one call, without autograd");
}

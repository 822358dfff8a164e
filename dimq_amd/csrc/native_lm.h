// The torch side of the language-model operators (part of native.cpp): RMS norm, token log probabilities, distillation from
// a teacher's top logits.  Each is an operator of the `dimq` library (the loss aside, which is an autograd node as the other
// QAT losses are), reached past the dispatcher where nothing stands between.
#pragma once

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t && wants_grad(*t); }

// ---- RMS norm ----------------------------------------------------------------------

struct RmsInputs {
  Rows x, r;
  Tensor w, h;
  RmsInputs(const Tensor& in, const OptTensor& weight, const OptTensor& residual, const char* op)
      : x(in, op, "input"), r(residual ? *residual : in, op, "residual") {
    TORCH_CHECK(x.cols > 0, op, ": rows must not be empty");
    if (weight) {
      TORCH_CHECK(weight->device() == in.device(), op, ": the weight must be on ", in.device().str());
      TORCH_CHECK(mx_float(weight->scalar_type()), op, ": weight must be fp32, fp16 or bf16, not ",
                  dtype_name(weight->scalar_type()));
      TORCH_CHECK(weight->dim() == 1 && weight->numel() == x.cols, op, ": weight must have one element for each of a row's");
      w = weight->detach().contiguous();
    }
    if (residual) {
      TORCH_CHECK(residual->device() == in.device() && residual->scalar_type() == in.scalar_type() &&
                      residual->sizes() == in.sizes(),
                  op, ": the residual must have the input's shape, dtype and device");
      h = at::empty(in.sizes(), in.options());
    } else {
      r.t = Tensor();
    }
  }
  void run(double eps, const Tensor& y, const Tensor& scales, const Tensor& at_of) const {
    const On on(at_of);
    check_rc(dimq_rms_norm(ptr(x.t), dt(x.t), x.n, x.cols, x.ld, ptr(r.t), r.ld, ptr(w), w.defined() ? dt(w) : 0, eps, ptr(y),
                           scales.defined() ? static_cast<int>(DIMQ_E4M3) : dt(y), static_cast<float*>(ptr(scales)), ptr(h),
                           on.stream));
  }
};

// (y, h); h is empty without a residual.
std::tuple<Tensor, Tensor> rms_norm(const Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual,
                                    std::optional<at::ScalarType> out_dtype) {
  const RmsInputs in(x, weight, residual, "rms_norm");
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  TORCH_CHECK(mx_float(odt), "rms_norm: output dtype must be fp32, fp16 or bf16");
  const Tensor y = at::empty(x.sizes(), x.options().dtype(odt));
  in.run(eps, y, Tensor(), x);
  return {y, residual ? in.h : at::empty({0}, x.options())};
}

// (codes, scales, h)
std::tuple<Tensor, Tensor, Tensor> rms_norm_e4m3(const Tensor& x, const OptTensor& weight, double eps,
                                                 const OptTensor& residual) {
  const RmsInputs in(x, weight, residual, "rms_norm_e4m3");
  const Tensor y = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  const Tensor scales = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  in.run(eps, y, scales, x);
  return {y, scales, residual ? in.h : at::empty({0}, x.options())};
}

// 8-bit rows have no gradient: where one may be asked for, the operator's own graph says so in the backward pass.
std::tuple<Tensor, Tensor, Tensor> rms_norm_e4m3_graph(const Tensor& x, const OptTensor& weight, double eps,
                                                       const OptTensor& residual) {
  const Direct<&rms_norm_e4m3> direct{"rms_norm_e4m3"};
  return wants_grad(x) || wants_grad(weight) || wants_grad(residual) ? direct.op(x, weight, eps, residual)
                                                                     : direct(x, weight, eps, residual);
}

std::tuple<Tensor, Tensor> rms_norm_below(const Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual,
                                          std::optional<at::ScalarType> out_dtype) {
  at::AutoDispatchBelowADInplaceOrView below;
  return Direct<&rms_norm>{"rms_norm"}(x, weight, eps, residual, out_dtype);
}

// Kept for the gradients: the normalised rows' input (x, or the sum that is returned) and the weight.
struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& residual,
                               double eps, std::optional<at::ScalarType> out_dtype) {
    const auto [y, h] = rms_norm_below(x, weight, eps, residual, out_dtype);
    ctx->save_for_backward({residual ? h : x, weight.value_or(Tensor())});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["layer"] = std::vector<int64_t>{weight.has_value(), residual.has_value()};
    ctx->set_materialize_grads(false);
    return residual ? variable_list{y, h} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* op = "rms_norm's gradient";
    untraced(op);
    once("rms_norm");
    const auto saved = ctx->get_saved_variables();
    const auto layer = ctx->saved_data["layer"].toIntVector();
    const Tensor &h = saved[0], &w = saved[1], &gy = grads[0];
    const Tensor gh = layer[1] ? grads[1] : Tensor();
    // inputs are counted without the absent ones
    const bool to_x = ctx->needs_input_grad(0), to_w = layer[0] && ctx->needs_input_grad(1),
               to_r = layer[1] && ctx->needs_input_grad(1 + layer[0]);
    Tensor gx, gw;
    if (!gy.defined()) {  // h alone was used
      gx = gh;
    } else {
      const Rows rows(h, op, "input"), g(gy, op, "gradient");
      Rows u(gh.defined() ? gh : gy, op, "gradient");
      if (!gh.defined()) u.t = Tensor();
      const Tensor wc = w.defined() ? w.detach().contiguous() : Tensor();
      if (to_x || to_r) gx = at::empty(h.sizes(), h.options());
      if (to_w) gw = at::empty(w.sizes(), w.options());
      const On on(h);
      const Tensor ws = workspace(to_w ? dimq_rms_norm_backward_workspace_bytes(rows.n, rows.cols) : 0, h);
      check_rc(dimq_rms_norm_backward(ptr(rows.t), dt(rows.t), rows.n, rows.cols, rows.ld, ptr(wc), wc.defined() ? dt(wc) : 0,
                                      ctx->saved_data["eps"].toDouble(), ptr(g.t), dt(g.t), g.ld, ptr(u.t), u.ld, ptr(gx),
                                      ptr(gw), to_w ? dt(gw) : 0, ptr(ws), ws.defined() ? ws.numel() : 0, on.stream));
    }
    return {to_x ? gx : Tensor(), gw, to_r ? gx : Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> rms_norm_graph(const Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual,
                                          std::optional<at::ScalarType> out_dtype) {
  if (wants_grad(x) || wants_grad(weight) || wants_grad(residual)) {
    const variable_list v = RmsNorm::apply(x, weight, residual, eps, out_dtype);
    return {v[0], residual ? v[1] : at::empty({0}, x.options())};
  }
  return rms_norm_below(x, weight, eps, residual, out_dtype);
}

// ---- log probabilities -------------------------------------------------------------

// Logits as rows, and an index tensor of one entry (last: `k` entries) a row.
Tensor index_rows(const Tensor& ids, const Tensor& logits, int64_t k, const char* op, const char* what) {
  TORCH_CHECK(ids.device() == logits.device(), op, ": ", what, " must be on ", logits.device().str());
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, op, ": ", what, " must be int64 or int32, not ",
              dtype_name(ids.scalar_type()));
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK(k < 0 ? ids.sizes() == lead : ids.dim() == logits.dim() && ids.sizes().slice(0, ids.dim() - 1) == lead, op, ": ",
              what, " ", tuple_of(ids.sizes()), " do not fit logits ", tuple_of(logits.sizes()));
  return ids.contiguous();
}

struct LogitRows : Rows {
  LogitRows(const Tensor& x, const char* op) : Rows(x, op, "logits") {
    TORCH_CHECK(cols > 0, op, ": there must be at least one logit a row");
  }
};

// (logprobs, entropy, top_logprobs, top_ids, norm); norm (for the gradients) only where it is kept.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_into(const Tensor& logits, const Tensor& tokens, int64_t top,
                                                                       bool keep) {
  const char* op = "token_logprobs";
  const LogitRows x(logits, op);
  const Tensor ids = index_rows(tokens, logits, -1, op, "tokens");
  TORCH_CHECK(top >= 0 && top <= 128 && top <= x.cols, op, ": top must be in [0, 128] and not above the vocabulary's ", x.cols);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const auto f = logits.options().dtype(at::kFloat);
  std::vector<int64_t> wide = lead.vec();
  wide.push_back(top);
  const Tensor lp = at::empty(lead, f), h = at::empty(lead, f), tlp = at::empty(wide, f);
  const Tensor tid = at::empty(wide, f.dtype(at::kLong)), norm = keep ? at::empty({x.n, 2}, f) : Tensor();
  const On on(logits);
  const Tensor ws = workspace(dimq_logits_workspace_bytes(x.n, x.cols, static_cast<int>(top)), logits);
  check_rc(dimq_token_logprobs(ptr(x.t), dt(x.t), x.n, x.cols, x.ld, ptr(ids), ids.scalar_type() == at::kLong,
                               static_cast<int>(top), f32(lp), f32(h), static_cast<float*>(ptr(norm)),
                               static_cast<float*>(ptr(tlp)), static_cast<int64_t*>(ptr(tid)), ptr(ws),
                               ws.defined() ? ws.numel() : 0, on.stream));
  return {lp, h, tlp, tid, norm};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t top) {
  const auto [lp, h, tlp, tid, norm] = token_logprobs_into(logits, tokens, top, false);
  return {lp, h, tlp, tid};
}

// Gradients reach the logits from the log probabilities and the entropy; the alternatives have none.
struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t top) {
    untraced("token_logprobs with gradients");
    const auto [lp, h, tlp, tid, norm] = token_logprobs_into(logits, tokens, top, true);
    ctx->save_for_backward({logits, tokens, norm, h});
    ctx->mark_non_differentiable({tlp, tid});
    ctx->set_materialize_grads(false);
    return {lp, h, tlp, tid};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* op = "token_logprobs' gradient";
    untraced(op);
    once("token_logprobs");
    const auto saved = ctx->get_saved_variables();
    const Tensor& logits = saved[0];
    const LogitRows x(logits, op);
    const Tensor ids = index_rows(saved[1], logits, -1, op, "tokens");
    const Tensor gx = at::empty(logits.sizes(), logits.options());
    const auto rows = [](const Tensor& g) { return g.defined() ? g.reshape({-1}) : Tensor(); };
    const Tensor ga = rows(grads[0]), gb = rows(grads[1]);
    const On on(logits);
    check_rc(dimq_token_logprobs_backward(ptr(x.t), dt(x.t), x.n, x.cols, x.ld, ptr(ids), ids.scalar_type() == at::kLong,
                                          f32(saved[2]), f32(saved[3]), static_cast<float*>(ptr(ga)),
                                          ga.defined() ? ga.stride(0) : 0, static_cast<float*>(ptr(gb)),
                                          gb.defined() ? gb.stride(0) : 0, ptr(gx), on.stream));
    return {gx, Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs_graph(const Tensor& logits, const Tensor& tokens, int64_t top) {
  if (wants_grad(logits)) {
    const variable_list v = TokenLogprobs::apply(logits, tokens, top);
    return {v[0], v[1], v[2], v[3]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return Direct<&token_logprobs>{"token_logprobs"}(logits, tokens, top);
}

// ---- distillation ------------------------------------------------------------------

struct DistillLoss : torch::autograd::Function<DistillLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& student, const Tensor& values, const Tensor& ids, double temperature,
                        int64_t reduction, bool keep) {
    const char* op = "top_logits_distillation_loss";
    untraced(op);
    const LogitRows x(student, op);
    const Tensor id = index_rows(ids, student, 0, op, "teacher ids");
    TORCH_CHECK(values.device() == student.device(), op, ": teacher values must be on ", student.device().str());
    TORCH_CHECK(mx_float(values.scalar_type()) && values.sizes() == ids.sizes(), op,
                ": teacher values must be fp32, fp16 or bf16 of the ids' shape");
    const Tensor v = values.detach().contiguous();
    const int64_t k = id.size(-1);
    const auto f = student.options().dtype(at::kFloat);
    const bool none = reduction == 0;
    const Tensor loss = none ? at::empty(student.sizes().slice(0, student.dim() - 1), f) : at::empty({}, f);
    // what the backward pass reads in one allocation: the divisor, norm [rows, 2], p [rows, k]; the rows' losses and the
    // workspace (16-byte aligned) in another
    const Tensor kept = at::empty({4 + x.n * (2 + k)}, f);
    const On on(student);
    const int64_t bytes = dimq_logits_workspace_bytes(x.n, x.cols, 0);
    const Tensor ws = at::empty({bytes / 4 + (none ? 0 : x.n)}, f);
    check_rc(dimq_distill_loss(ptr(x.t), dt(x.t), x.n, x.cols, x.ld, ptr(v), dt(v), ptr(id), id.scalar_type() == at::kLong, k,
                               temperature, static_cast<int>(reduction), none ? f32(loss) : f32(ws) + bytes / 4, f32(loss), f32(kept),
                               f32(kept) + 4, f32(kept) + 4 + 2 * x.n, ptr(ws), bytes, on.stream));
    if (keep && student.requires_grad()) ctx->save_for_backward({student, id, kept});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["none"] = none;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const char* op = "top_logits_distillation_loss's gradient";
    untraced(op);
    once("top_logits_distillation_loss");
    const auto saved = ctx->get_saved_variables();
    const Tensor& student = saved[0];
    const bool none = ctx->saved_data["none"].toBool();
    const LogitRows x(student, op);
    const Tensor &id = saved[1], &kept = saved[2];
    const Tensor g = grads[0].detach().reshape({-1}), gx = at::empty(student.sizes(), student.options());
    const On on(student);
    check_rc(dimq_distill_loss_backward(ptr(x.t), dt(x.t), x.n, x.cols, x.ld, ptr(id), id.scalar_type() == at::kLong, id.size(-1),
                                        f32(kept) + 4 + 2 * x.n, f32(kept) + 4, ctx->saved_data["temperature"].toDouble(), f32(g),
                                        none ? g.stride(0) : 0, none ? nullptr : f32(kept), ptr(gx), on.stream));
    return {gx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ---- 4-bit weights with group scales -----------------------------------------------

Tensor linear_grouped(const Tensor& x, const Tensor& codes, const Tensor& scales, const OptTensor& zeros, int64_t group,
                      const OptTensor& bias, const OptTensor& x_scales, const OptTensor& residual, int64_t activation,
                      std::optional<at::ScalarType> out_dtype, int64_t variant) {
  const char* op = "linear_grouped";
  TORCH_CHECK_NOT_IMPLEMENTED(x.is_cuda(), op, " expects a CUDA input");
  const bool q8 = x.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(q8 || mx_float(x.scalar_type()), op, ": input must be fp32, fp16, bf16 or float8_e4m3fn, not ",
              dtype_name(x.scalar_type()));
  TORCH_CHECK(x.dim() > 0 && codes.dim() == 2 && scales.dim() == 2, op,
              " expects an input of at least one dimension, 2-D codes and 2-D scales");
  const int64_t K = x.size(-1), N = codes.size(0), nb = mx_blocks(K);
  TORCH_CHECK(K > 0 && N > 0, "linear dimensions must be positive");
  TORCH_CHECK(group > 0 && group % 32 == 0, op, ": the group size must be a positive multiple of 32");
  const int64_t G = (K + group - 1) / group;
  const auto here = [&](const Tensor& t, const char* what) {
    TORCH_CHECK(t.device() == x.device(), op, ": ", what, " must be on ", x.device().str());
  };
  here(codes, "codes");
  here(scales, "scales");
  TORCH_CHECK(codes.scalar_type() == at::kByte, op, ": codes must be uint8");
  TORCH_CHECK(mx_float(scales.scalar_type()), op, ": scales must be fp32, fp16 or bf16");
  TORCH_CHECK(codes.size(1) == nb * 16, op, ": rows of ", K, " have codes [out_features, ", nb * 16, "], not ",
              tuple_of(codes.sizes()));
  TORCH_CHECK(scales.size(0) == N && scales.size(1) == G, op, ": groups of ", group, " have scales (", N, ", ", G, "), not ",
              tuple_of(scales.sizes()));
  Tensor z;
  if (zeros) {
    here(*zeros, "zeros");
    TORCH_CHECK(zeros->scalar_type() == at::kByte && zeros->sizes() == scales.sizes(), op,
                ": zeros must be uint8 of the scales' shape");
    z = zeros->contiguous();
  }
  TORCH_CHECK(q8 == x_scales.has_value(), op, ": float8_e4m3fn inputs, and no others, take x_scales");
  Tensor xs;
  if (q8) {
    here(*x_scales, "x_scales");
    TORCH_CHECK(x_scales->scalar_type() == at::kFloat && x_scales->sizes() == x.sizes().slice(0, x.dim() - 1), op,
                ": x_scales must be fp32, one for each row");
    xs = x_scales->contiguous();
  }
  Tensor c = codes.contiguous();
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16) c = c.clone();
  const Tensor s = scales.detach().contiguous();
  const int64_t M = x.numel() / K;
  Tensor t = x.detach();
  if (x.dim() != 2) t = t.reshape({M, K});
  if ((K > 1 && t.stride(1) != 1) || (M > 1 && t.stride(0) < K)) t = t.contiguous();
  const int64_t ld = M > 1 ? t.stride(0) : K;
  const at::ScalarType odt = out_dtype.value_or(q8 ? at::kBFloat16 : x.scalar_type());
  TORCH_CHECK(mx_float(odt), op, ": output dtype must be fp32, fp16 or bf16");
  const Bias b(bias, N, "out_features");
  const std::vector<int64_t> shape = out_shape(x, N);
  const Residual r(residual, shape, at::MemoryFormat::Contiguous);
  if (bias) here(*bias, "bias");
  if (residual) here(*residual, "residual");
  const int xdt = q8 ? static_cast<int>(DIMQ_E4M3) : dt(x);
  const Tensor y = at::empty(shape, x.options().dtype(odt));
  const On on(x);
  const Tensor ws = workspace(dimq_linear_grouped_workspace_bytes(ptr(t), xdt, M, K, ld, group, N, static_cast<int>(variant)), c);
  check_rc(dimq_linear_grouped(ptr(t), xdt, M, K, ld, static_cast<float*>(ptr(xs)), u8(c), ptr(s), dt(s),
                               static_cast<uint8_t*>(ptr(z)), group, b.p, b.dtype, N, ptr(y), dt(y), r.p, r.dtype,
                               static_cast<int>(activation), static_cast<int>(variant), ptr(ws), ws.defined() ? ws.numel() : 0,
                               on.stream));
  return y;
}

// The weights are frozen and the layer is for serving: where a gradient may be asked for, the operator's own graph refuses
// it in the backward pass.
Tensor linear_grouped_graph(const Tensor& x, const Tensor& codes, const Tensor& scales, const OptTensor& zeros, int64_t group,
                            const OptTensor& bias, const OptTensor& x_scales, const OptTensor& residual, int64_t activation,
                            std::optional<at::ScalarType> out_dtype, int64_t variant) {
  const Direct<&linear_grouped> direct{"linear_grouped"};
  return wants_grad(x) || wants_grad(scales) || wants_grad(bias) || wants_grad(x_scales) || wants_grad(residual)
             ? direct.op(x, codes, scales, zeros, group, bias, x_scales, residual, activation, out_dtype, variant)
             : direct(x, codes, scales, zeros, group, bias, x_scales, residual, activation, out_dtype, variant);
}

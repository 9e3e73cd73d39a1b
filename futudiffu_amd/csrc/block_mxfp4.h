// Host side of the MXFP4 operators (futudiffu_amd/mxfp4.py): a part of block_ops.cpp, inside its
// namespace and behind its helpers.

// ---------------------------------------------------------------- operands

int64_t mx_cols(int64_t k) { return (k + 255) / 256 * 256; }

Tensor mx_scales(int64_t rows, int64_t k, const Tensor& like) {
  return at::empty({mx_cols(k) / 256, rows, 8}, like.options().dtype(at::kByte).requires_grad(false));
}
Tensor mx_codes(c10::IntArrayRef shape, const Tensor& like) {
  std::vector<int64_t> s = shape.vec();
  s.back() = mx_cols(s.back()) / 2;
  return at::empty(s, like.options().dtype(at::kByte).requires_grad(false));
}

// Codes and scales that a caller holds, checked, as the library takes them.
struct MxRows {
  Tensor codes, scales;
  int64_t rows, k;
  MxRows(const char* name, const Tensor& c, const Tensor& s, int64_t columns) : k(columns) {
    TORCH_CHECK_VALUE(columns >= 1, name, ".columns must be at least 1, got ", columns);
    TORCH_CHECK_VALUE(c.scalar_type() == at::kByte && c.dim() >= 1 && c.size(-1) == mx_cols(k) / 2, name,
                      ".codes must be a uint8 [..., ", mx_cols(k) / 2, "] tensor for ", k, " columns, got ",
                      c.scalar_type(), " ", c.sizes());
    rows = c.numel() / c.size(-1);
    TORCH_CHECK_VALUE(s.scalar_type() == at::kByte && s.dim() == 3 && s.size(0) == mx_cols(k) / 256 &&
                          s.size(1) == rows && s.size(2) == 8 && s.device() == c.device(),
                      name, ".scales must be a uint8 [", mx_cols(k) / 256, ", ", rows, ", 8] tensor on ", c.device(),
                      ", got ", s.scalar_type(), " ", s.sizes(), " on ", s.device());
    TORCH_CHECK_VALUE(c.is_cuda(), name, " must be on a GPU (device ", c.device(), ")");
    codes = aligned(c, 16);
    scales = aligned(s, 8);
  }
  static Tensor aligned(const Tensor& t, uintptr_t to) {
    const Tensor u = t.contiguous();
    return u.numel() && reinterpret_cast<uintptr_t>(u.data_ptr()) % to ? u.clone() : u;
  }
};

std::tuple<Tensor, Tensor> mx_quantize(const Tensor& x) {
  refuse_tangents({&x});
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., K] with at least one column, got ", x.sizes());
  const int dtype = dtype_of(x);
  need_gpu(x);
  const int64_t k = x.size(-1), m = x.numel() / k;
  const Tensor codes = mx_codes(x.sizes(), x), scales = mx_scales(m, k, x);
  if (m) {
    const Matrix xm(x);
    const Launch on(x);
    check_status(lib.sage_mxfp4_quantize(xm.p(), xm.rs, m, k, dtype, codes.data_ptr(), scales.data_ptr(), on.stream));
  }
  return {codes, scales};
}

Tensor mx_dequantize(const Tensor& codes, const Tensor& scales, int64_t columns, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(dtype == at::kBFloat16 || dtype == at::kHalf, "dtype must be bfloat16 or float16, got ", dtype);
  const MxRows q("q", codes, scales, columns);
  std::vector<int64_t> shape = codes.sizes().vec();
  shape.back() = columns;
  const Tensor out = at::empty(shape, codes.options().dtype(dtype));
  if (q.rows) {
    const Launch on(codes);
    check_status(lib.sage_mxfp4_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), q.rows, columns,
                                           dtype == at::kHalf ? SAGE_DTYPE_FP16 : SAGE_DTYPE_BF16, out.data_ptr(),
                                           on.stream));
  }
  return out;
}

// ---------------------------------------------------------------- linear

// The checked arguments of a product over a weight in MXFP4: x is 16-bit, or codes whose product
// comes out as `type`.
struct MxLinear {
  int act, dtype;
  bool f32 = false;
  at::ScalarType type;
  MxRows w;
  int64_t M, N;
  std::vector<int64_t> shape;
  Tensor bias;

  MxLinear(c10::IntArrayRef rows_of, int64_t k, at::ScalarType t, const Tensor& codes, const Tensor& scales,
           int64_t columns, const OptTensor& b, const std::string& activation)
      : act(activation_of(activation)), type(t), w("weight", codes, scales, columns), shape(rows_of.vec()) {
    TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf, "x and the output must be bfloat16 or float16, got ", t);
    dtype = t == at::kHalf ? SAGE_DTYPE_FP16 : SAGE_DTYPE_BF16;
    TORCH_CHECK_VALUE(codes.dim() == 2 && w.rows >= 1, "weight must have rows [N, K], got codes ", codes.sizes());
    TORCH_CHECK_VALUE(k == columns, "x has ", k, " columns, weight ", columns);
    TORCH_CHECK_VALUE(act != SAGE_ACT_SWIGLU || w.rows % 2 == 0, "a swiglu weight has an even number of rows, got ",
                      w.rows);
    N = act == SAGE_ACT_SWIGLU ? w.rows / 2 : w.rows;
    M = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) M *= shape[i];
    shape.back() = N;
    if (b) {
      TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == w.rows && b->device() == codes.device() &&
                            (b->scalar_type() == at::kFloat || b->scalar_type() == type),
                        "bias must be a [", w.rows, "] tensor of ", type, " or float32 on ", codes.device(), ", got ",
                        b->scalar_type(), " ", b->sizes(), " on ", b->device());
      f32 = b->scalar_type() == at::kFloat;
      bias = b->contiguous();
    }
  }
  void check_out(const char* name, const Tensor& t) const {
    TORCH_CHECK_VALUE(t.sizes() == c10::IntArrayRef(shape) && t.scalar_type() == type &&
                          t.device() == w.codes.device(),
                      name, " must be a ", type, " ", c10::IntArrayRef(shape), " tensor on ", w.codes.device(),
                      ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
  }
};

std::tuple<Tensor, Tensor> mx_product(const MxLinear& a, const Tensor* x, const MxRows* xq, const OptTensor& residual,
                                      bool keep_z) {
  if (residual) a.check_out("residual", *residual);
  const auto options = a.w.codes.options();
  Tensor out = at::empty(a.shape, options.dtype(a.type)), z;
  if (keep_z && a.act != SAGE_ACT_NONE) z = at::empty({a.M, a.w.rows}, options.dtype(at::kFloat));
  if (a.M == 0) return {out, z};
  std::optional<Matrix> xm, rm;
  if (x) xm.emplace(*x);
  if (residual) rm.emplace(*residual);
  const void* rp = rm ? rm->p() : nullptr;
  const int64_t rs = rm ? rm->rs : 0;
  const bool near = x && !off16(xm->p()) && a.w.k % 8 == 0 && (a.M == 1 || (xm->rs % 8 == 0 && xm->rs < 1 << 22));
  const size_t bytes = lib.sage_mxfp4_linear_workspace_bytes(a.M, a.N, a.w.k, a.act, near ? 2 : x ? 1 : 0,
                                                             off16(rp) || off16(ptr(a.bias)) || rs % 8 != 0);
  const Tensor ws = workspace(a.w.codes, bytes);
  const Launch on(a.w.codes);
  check_status(lib.sage_mxfp4_linear(x ? xm->p() : nullptr, x ? xm->rs : 0, xq ? xq->codes.data_ptr() : nullptr,
                                     xq ? xq->scales.data_ptr() : nullptr, a.w.codes.data_ptr(),
                                     a.w.scales.data_ptr(), ptr(a.bias), a.f32, rp, rs, a.M, a.N, a.w.k, a.dtype,
                                     a.act, ptr(ws), bytes, static_cast<float*>(ptr(z)), out.data_ptr(), on.stream));
  return {out, z};
}

// out, and z where it is kept (an activation, keep_z).
std::tuple<Tensor, Tensor> mx_linear_forward(const Tensor& x, const Tensor& codes, const Tensor& scales,
                                             int64_t columns, const OptTensor& bias, const OptTensor& residual,
                                             const std::string& activation, bool keep_z) {
  refuse_tangents({&x, &some(bias), &some(residual)});
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must be [..., K], got a scalar");
  const MxLinear a(x.sizes(), x.size(-1), x.scalar_type(), codes, scales, columns, bias, activation);
  TORCH_CHECK_VALUE(x.device() == codes.device(), "x must be on the weight's device ", codes.device(), ", got ",
                    x.device());
  return mx_product(a, &x, nullptr, residual, keep_z);
}

Tensor mx_linear_codes(const Tensor& x_codes, const Tensor& x_scales, int64_t x_columns, const Tensor& codes,
                       const Tensor& scales, int64_t columns, const OptTensor& bias, const OptTensor& residual,
                       const std::string& activation, at::ScalarType dtype) {
  refuse_tangents({&some(bias), &some(residual)});
  const MxRows xq("x", x_codes, x_scales, x_columns);
  const MxLinear a(x_codes.sizes(), x_columns, dtype, codes, scales, columns, bias, activation);
  TORCH_CHECK_VALUE(x_codes.device() == codes.device(), "x must be on the weight's device ", codes.device(), ", got ",
                    x_codes.device());
  return std::get<0>(mx_product(a, nullptr, &xq, residual, false));
}

std::tuple<Tensor, Tensor> mx_linear_backward(const Tensor& dout, const Tensor& codes, const Tensor& scales,
                                              int64_t columns, const OptTensor& bias, const OptTensor& z,
                                              const std::string& activation, const Wanted& wanted) {
  refuse_tangents({&dout, &some(bias)});
  TORCH_CHECK_VALUE(wanted.size() == 2, "wanted must say whether x and the bias want a gradient, got ", wanted.size(),
                    " values");
  TORCH_CHECK_VALUE(dout.dim() >= 1, "dout must be [..., N], got a scalar");
  const MxLinear a(dout.sizes(), columns, dout.scalar_type(), codes, scales, columns, bias, activation);
  a.check_out("dout", dout);
  const bool act = a.act != SAGE_ACT_NONE;
  TORCH_CHECK_VALUE(!act || !(wanted[0] || wanted[1]) ||
                        (z && z->defined() && z->dim() == 2 && z->size(0) == a.M && z->size(1) == a.w.rows &&
                         z->scalar_type() == at::kFloat && z->device() == dout.device() && z->is_contiguous()),
                    "the gradient of an activation needs the z that the forward kept (keep_z)");
  std::vector<int64_t> shape = a.shape;
  shape.back() = columns;
  Tensor dx, db = grad_of(some(bias), wanted[1]);
  if (wanted[0]) dx = at::empty(shape, dout.options().requires_grad(false));
  const int want = (dx.defined() ? 1 : 0) | (db.defined() ? 4 : 0);
  if (a.M == 0) {
    zero({db});
  } else if (want) {
    const Matrix dm(dout);
    const size_t bytes =
        lib.sage_mxfp4_linear_bwd_workspace_bytes(dm.p(), dm.rs, a.M, a.N, columns, a.act, want);
    const Tensor ws = workspace(dout, bytes);
    const Launch on(dout);
    check_status(lib.sage_mxfp4_linear_bwd(dm.p(), dm.rs, a.w.codes.data_ptr(), a.w.scales.data_ptr(),
                                           act ? z->data_ptr<float>() : nullptr, a.M, a.N, columns, a.dtype, a.act,
                                           a.f32, ptr(ws), bytes, ptr(dx), ptr(db), on.stream));
  }
  return {dx, db};
}

// ---------------------------------------------------------------- norms

std::tuple<Tensor, Tensor> mx_modulate(const Tensor& x, const OptTensor& weight, const OptTensor& scale,
                                       const OptTensor& doc_ids, double eps) {
  refuse_tangents({&x, &some(weight), &some(scale)});
  const Norm a(x, weight, "scale", scale, doc_ids, eps);
  const Tensor codes = mx_codes(x.sizes(), x), scales = mx_scales(a.B * a.N, a.C, x);
  if (!a.empty()) {
    const Tokens xt(x);
    const Launch on(x);
    check_status(lib.sage_rms_norm_modulate_mxfp4(xt.p(), xt.bs, xt.rs, ptr(a.weight), COND(a.cond), SIZES(a), (a).eps64,
                                                  codes.data_ptr(), scales.data_ptr(), on.stream));
  }
  return {codes, scales};
}

std::tuple<Tensor, Tensor, Tensor> mx_gate_modulate(const Tensor& residual, const Tensor& x, const OptTensor& weight,
                                                    const OptTensor& gate, const OptTensor& next_weight,
                                                    const OptTensor& next_scale, const OptTensor& doc_ids, double eps) {
  refuse_tangents({&residual, &x, &some(weight), &some(gate), &some(next_weight), &some(next_scale)});
  check_like("residual", residual, x);
  const Norm a(x, weight, "gate", gate, doc_ids, eps, next_weight, next_scale);
  const Tensor hidden = at::empty(x.sizes(), x.options().requires_grad(false));
  const Tensor codes = mx_codes(x.sizes(), x), scales = mx_scales(a.B * a.N, a.C, x);
  if (!a.empty()) {
    const Tokens xt(x), rt(residual);
    const Launch on(x);
    check_status(lib.sage_rms_norm_gate_residual_modulate_mxfp4(
        rt.p(), rt.bs, rt.rs, xt.p(), xt.bs, xt.rs, ptr(a.weight), COND(a.cond), ptr(a.next_weight),
        COND(a.next_scale), SIZES(a), (a).eps64, hidden.data_ptr(), codes.data_ptr(), scales.data_ptr(), on.stream));
  }
  return {hidden, codes, scales};
}

// ---------------------------------------------------------------- autograd

// What x's gradient takes: refused before the forward, not in the backward.
void check_for_dx(int64_t rows, int64_t columns) {
  TORCH_CHECK_VALUE(rows * ((columns + 7) / 8 * 8) * 2 < (int64_t)1 << 31, "x wants a gradient: a weight of ", rows, " x ",
                    columns, " has 2^31 bytes or more in 16 bits (detach x, or split the weight)");
}

struct MxLinearFn : torch::autograd::Function<MxLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scales,
                        int64_t columns, const OptTensor& bias, const OptTensor& residual,
                        const std::string& activation) {
    if (x.requires_grad() && codes.dim() == 2) check_for_dx(codes.size(0), columns);
    // a residual's gradient alone needs no z
    const auto [out, z] = mx_linear_forward(x, codes, scales, columns, bias, residual, activation,
                                            any_requires({&x, &some(bias)}));
    ctx->save_for_backward({codes, scales, held(bias), z});
    ctx->saved_data["columns"] = columns;
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["residual"] = residual.has_value();
    // x is not saved, but its gradient and the bias's depend on it
    ctx->saved_data["x_requires"] = x.requires_grad();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto s = ctx->get_saved_variables();
    once({d[0], s[2]});
    TORCH_CHECK(!at::GradMode::is_enabled() || !ctx->saved_data["x_requires"].toBool(), kTwice);
    // x, codes, scales, bias, then the residual's edge
    const Wanted all = needs(ctx, {s[0], s[0], s[1], s[2], ctx->saved_data["residual"].toBool() ? s[0] : Tensor()});
    const Wanted w = {all[0], all[3]};
    const Tensor dr = all[4] ? d[0] : Tensor();
    const std::string& activation = ctx->saved_data["activation"].toStringRef();
    const int64_t columns = ctx->saved_data["columns"].toInt();
    if (!w[0] && !w[1]) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), dr, Tensor()};
    if (through_dispatcher({&d[0], &s[0], &s[1], &s[2], &s[3]})) {
      const auto g = gradients(call_op("mxfp4_linear_backward", d[0], s[0], s[1], columns, given(s[2]), given(s[3]),
                                       activation, list_of(w)), w);
      return {g[0], Tensor(), Tensor(), Tensor(), g[1], dr, Tensor()};
    }
    const auto [dx, db] = mx_linear_backward(d[0], s[0], s[1], columns, given(s[2]), given(s[3]), activation, w);
    return {dx, Tensor(), Tensor(), Tensor(), db, dr, Tensor()};
  }
};

// Codes carry no gradient: what asks for one is refused, or it would be lost in silence.
void refuse_grad(std::initializer_list<const Tensor*> tensors) {
  TORCH_CHECK(!wants_grad(tensors),
              "MXFP4 codes carry no gradient: quantize under torch.no_grad() or detach the input (mxfp4_linear "
              "differentiates in an x that it quantizes itself)");
}

std::tuple<Tensor, Tensor> mxfp4_quantize(const Tensor& x) {
  refuse_grad({&x});
  if (through_dispatcher({&x})) {
    const auto r = call_op("mxfp4_quantize", x);
    return {r[0].toTensor(), r[1].toTensor()};
  }
  return mx_quantize(x);
}

Tensor mxfp4_dequantize(const Tensor& codes, const Tensor& scales, int64_t columns, at::ScalarType dtype) {
  if (through_dispatcher({&codes, &scales}))
    return call_op("mxfp4_dequantize", codes, scales, columns, dtype)[0].toTensor();
  return mx_dequantize(codes, scales, columns, dtype);
}

Tensor mxfp4_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t columns, const OptTensor& bias,
                    const OptTensor& residual, const std::string& activation) {
  if (through_dispatcher({&x, &codes, &scales, &some(bias), &some(residual)})) {
    // what vmap batches does not say whether what lies under it wants a gradient: z is kept
    const bool hidden = x.key_set().has(c10::DispatchKey::FuncTorchBatched) ||
                        some(bias).key_set().has(c10::DispatchKey::FuncTorchBatched);
    const bool keep_z =
        activation != "none" && at::GradMode::is_enabled() && (hidden || any_requires({&x, &some(bias)}));
    return call_op("mxfp4_linear", x, codes, scales, columns, bias, residual, activation, keep_z)[0].toTensor();
  }
  if (wants_grad({&x, &some(bias), &some(residual)}))
    return MxLinearFn::apply(x, codes, scales, columns, bias, residual, activation);
  return std::get<0>(mx_linear_forward(x, codes, scales, columns, bias, residual, activation, false));
}

Tensor mxfp4_linear_codes(const Tensor& x_codes, const Tensor& x_scales, int64_t x_columns, const Tensor& codes,
                          const Tensor& scales, int64_t columns, const OptTensor& bias, const OptTensor& residual,
                          const std::string& activation, at::ScalarType dtype) {
  refuse_grad({&some(bias), &some(residual)});
  if (through_dispatcher({&x_codes, &x_scales, &codes, &scales, &some(bias), &some(residual)}))
    return call_op("mxfp4_linear_codes", x_codes, x_scales, x_columns, codes, scales, columns, bias, residual,
                   activation, dtype)[0].toTensor();
  return mx_linear_codes(x_codes, x_scales, x_columns, codes, scales, columns, bias, residual, activation, dtype);
}

std::tuple<Tensor, Tensor> rms_norm_modulate_mxfp4(const Tensor& x, const OptTensor& weight, const OptTensor& scale,
                                                   const OptTensor& doc_ids, double eps) {
  refuse_grad({&x, &some(weight), &some(scale)});
  if (through_dispatcher({&x, &some(weight), &some(scale), &some(doc_ids)})) {
    const auto r = call_op("rms_norm_modulate_mxfp4", x, weight, scale, doc_ids, eps);
    return {r[0].toTensor(), r[1].toTensor()};
  }
  return mx_modulate(x, weight, scale, doc_ids, eps);
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_gate_residual_modulate_mxfp4(
    const Tensor& residual, const Tensor& x, const OptTensor& weight, const OptTensor& gate,
    const OptTensor& next_weight, const OptTensor& next_scale, const OptTensor& doc_ids, double eps) {
  refuse_grad({&residual, &x, &some(weight), &some(gate), &some(next_weight), &some(next_scale)});
  if (through_dispatcher({&residual, &x, &some(weight), &some(gate), &some(next_weight), &some(next_scale),
                          &some(doc_ids)})) {
    const auto r = call_op("rms_norm_gate_residual_modulate_mxfp4", residual, x, weight, gate, next_weight, next_scale,
                           doc_ids, eps);
    return {r[0].toTensor(), r[1].toTensor(), r[2].toTensor()};
  }
  return mx_gate_modulate(residual, x, weight, gate, next_weight, next_scale, doc_ids, eps);
}

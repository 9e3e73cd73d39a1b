// Host side of the operators around the attention (futudiffu_amd/block_ops.py): the checks of
// a call's arguments, its allocations, the library call, and autograd.
//
// In C++ because the host bounds a small call and nearly all of a small training step: the
// backward runs on autograd's own thread, where Python (the interpreter's data lying in the
// other core's caches) took 50 us of a step's 150 and made the forward's next pass three times
// as slow; and a call without gradients spends 10 us in Python around a 3 us kernel.
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/extension.h>

#include "../../include/sage_mi355x.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

// The library that the package loaded (bind): its entry points.
#define SAGE_ENTRIES(X)                                                                                    \
  X(sage_last_error) X(sage_rms_norm_modulate) X(sage_rms_norm_gate_residual)                               \
  X(sage_rms_norm_gate_residual_modulate) X(sage_rms_norm_bwd_workspace_bytes)                              \
  X(sage_rms_norm_modulate_bwd) X(sage_rms_norm_gate_residual_bwd)                                          \
  X(sage_rms_norm_gate_residual_modulate_bwd) X(sage_linear_workspace_bytes) X(sage_linear)                 \
  X(sage_linear_bwd_workspace_bytes) X(sage_linear_bwd)

struct Library {
#define X(name) decltype(&::name) name = nullptr;
  SAGE_ENTRIES(X)
#undef X
} lib;

void bind(uintptr_t handle) {
  Library l;
#define X(name)                                                                                             \
  l.name = reinterpret_cast<decltype(&::name)>(dlsym(reinterpret_cast<void*>(handle), #name));              \
  TORCH_CHECK(l.name, #name " is not in the library");
  SAGE_ENTRIES(X)
#undef X
  lib = l;
}

void check_status(int status) {
  if (status == SAGE_OK) return;
  TORCH_CHECK_VALUE(status != SAGE_ERR_ARG, lib.sage_last_error());
  TORCH_CHECK(false, "sage status ", status, ": ", lib.sage_last_error());
}

// The current stream of x's device, made the current device while the guard lives (the
// library launches there).
struct Launch {
  c10::DeviceGuard guard;
  hipStream_t stream;
  explicit Launch(const Tensor& x)
      : guard(x.device()), stream(c10::hip::getCurrentHIPStream(x.device().index()).stream()) {}
};

void need_gpu(const Tensor& x) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must be a GPU tensor (device ", x.device(), ")");
}

int dtype_of(const Tensor& x) {
  const auto t = x.scalar_type();
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf, "x must be bfloat16 or float16, got ", t);
  return t == at::kHalf ? SAGE_DTYPE_FP16 : SAGE_DTYPE_BF16;
}

// Forward-mode differentiation is refused: the operators have no formula for tangents, and a
// result without one would count as constant.
void refuse_tangents(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                "the block operators have no forward-mode derivative (a tangent was given)");
}

const Tensor& some(const OptTensor& t) {
  static const Tensor none;
  return t ? *t : none;
}

bool is_param(const Tensor& p, const Tensor& x) {
  return p.device() == x.device() && (p.scalar_type() == at::kFloat || p.scalar_type() == x.scalar_type());
}

const Tensor& check_like(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK_VALUE(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type() && t.device() == like.device(),
                    name, " must be a ", like.scalar_type(), " ", like.sizes(), " tensor on ", like.device(), ", got ",
                    t.scalar_type(), " ", t.sizes(), " on ", t.device());
  return t;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor grad_of(const Tensor& t, bool wanted) {
  return wanted && t.defined() ? at::empty(t.sizes(), t.options().requires_grad(false)) : Tensor();
}
Tensor workspace(const Tensor& x, size_t bytes) {
  return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
}
void zero(std::initializer_list<Tensor> grads) {
  for (const Tensor& g : grads)
    if (g.defined()) g.zero_();
}

// ---------------------------------------------------------------- norms

// A [B, N, C] (or [N, C]) tensor with its channels contiguous, and its strides.
struct Tokens {
  Tensor t;
  int64_t bs, rs;
  explicit Tokens(const Tensor& x) : t(x.size(-1) == 1 || x.stride(-1) == 1 ? x : x.contiguous()) {
    const bool three = t.dim() == 3;
    bs = three ? t.stride(0) : 0;
    rs = t.stride(three ? 1 : 0);
  }
  const void* p() const { return t.data_ptr(); }
};

struct Cond {
  Tensor t;
  int64_t bs = 0, gs = 0, rows = 0;
};

// The checked arguments of a norm call.
struct Norm {
  int64_t B, N, C, groups = 1;
  int dtype, f32 = 0;
  float eps;
  Tensor weight, next_weight, doc;
  Cond cond, next_scale;

  Norm(const Tensor& x, const OptTensor& w, const char* cond_name, const OptTensor& k, const OptTensor& ids, double e,
       const OptTensor& w2 = std::nullopt, const OptTensor& s2 = std::nullopt)
      : eps((float)e) {
    TORCH_CHECK_VALUE(x.dim() == 2 || x.dim() == 3, "x must be [B, N, C] or [N, C], got ", x.sizes());
    B = x.dim() == 3 ? x.size(0) : 1;
    N = x.size(-2);
    C = x.size(-1);
    dtype = dtype_of(x);
    TORCH_CHECK_VALUE(e >= 0, "eps must be >= 0, got ", e);
    TORCH_CHECK_VALUE(C >= 1, "x needs at least one channel, got ", x.sizes());
    if (ids) {
      TORCH_CHECK_VALUE((ids->dim() == 2 && ids->size(0) == B && ids->size(1) == N) ||
                            (x.dim() == 2 && ids->dim() == 1 && ids->size(0) == N),
                        "doc_ids must be [B, N] = [", B, ", ", N, "], got ", ids->sizes());
      TORCH_CHECK_VALUE(at::isIntegralType(ids->scalar_type(), false), "doc_ids must hold integers, got ",
                        ids->scalar_type());
    }
    const bool docs = ids && (k || s2);  // without conditioning nothing differs between documents
    weight = param("weight", w, x, SAGE_FP32_WEIGHT);
    cond = conditioning(cond_name, k, x, docs, SAGE_FP32_COND);
    next_weight = param("next_weight", w2, x, SAGE_FP32_NEXT_WEIGHT);
    next_scale = conditioning("next_scale", s2, x, docs, SAGE_FP32_NEXT_SCALE);
    TORCH_CHECK_VALUE(!cond.rows || !next_scale.rows || cond.rows == next_scale.rows, cond_name,
                      " and next_scale must have a row for the same documents, got ", cond.rows, " and ",
                      next_scale.rows);
    if (cond.rows || next_scale.rows) groups = cond.rows ? cond.rows : next_scale.rows;
    need_gpu(x);
    if (docs) {
      // ids past 32 bits stay ids of no document (of 64 bits without a sign: those past 2^63
      // read as negative ones; of 32 bits without a sign: those past 2^31)
      Tensor i = *ids;
      if (i.scalar_type() == at::kUInt64) i = i.view(at::kLong);
      if (i.scalar_type() == at::kUInt32) i = i.view(at::kInt);
      if (i.scalar_type() == at::kLong) i = i.clamp(-1, groups);
      doc = i.to(x.device(), at::kInt).contiguous();
    }
  }
  Tensor param(const char* name, const OptTensor& p, const Tensor& x, int bit) {
    if (!p) return Tensor();
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == C && is_param(*p, x), name, " must be a [", C, "] tensor of ",
                      x.scalar_type(), " or float32 on ", x.device(), ", got ", p->scalar_type(), " ", p->sizes(),
                      " on ", p->device());
    if (p->scalar_type() == at::kFloat) f32 |= bit;
    return p->contiguous();
  }
  Cond conditioning(const char* name, const OptTensor& p, const Tensor& x, bool docs, int bit) {
    Cond c;
    if (!p) return c;
    const bool shape = docs ? p->dim() == 3 && p->size(0) == B && p->size(1) >= 1 && p->size(2) == C
                            : p->dim() == 2 && p->size(0) == B && p->size(1) == C;
    TORCH_CHECK_VALUE(shape && is_param(*p, x), name, " must be a [", B, docs ? ", G, " : ", ", C,
                      docs ? "] (with doc_ids)" : "]", " tensor of ", x.scalar_type(), " or float32 on ", x.device(),
                      ", got ", p->scalar_type(), " ", p->sizes(), " on ", p->device());
    if (p->scalar_type() == at::kFloat) f32 |= bit;
    c.t = C == 1 || p->stride(-1) == 1 ? *p : p->contiguous();
    c.bs = c.t.stride(0);
    c.gs = docs ? c.t.stride(1) : 0;
    c.rows = docs ? c.t.size(1) : 1;
    return c;
  }
  bool empty() const { return B == 0 || N == 0; }
  const int32_t* ids() const { return doc.defined() ? doc.data_ptr<int32_t>() : nullptr; }
  size_t bytes(bool fused) const {
    return lib.sage_rms_norm_bwd_workspace_bytes(B, N, C, groups, doc.defined(), fused);
  }
};

#define COND(k) ptr((k).t), (k).bs, (k).gs
#define TAIL(a) (a).groups, (a).ids(), (a).B, (a).N, (a).C, (a).dtype, (a).f32, (a).eps

Tensor modulate_forward(const Tensor& x, const OptTensor& weight, const OptTensor& scale, const OptTensor& doc_ids,
                        double eps) {
  refuse_tangents({&x, &some(weight), &some(scale)});
  const Norm a(x, weight, "scale", scale, doc_ids, eps);
  Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
  if (a.empty()) return out;
  const Tokens xt(x);
  const Launch on(x);
  check_status(lib.sage_rms_norm_modulate(xt.p(), xt.bs, xt.rs, ptr(a.weight), COND(a.cond), TAIL(a), out.data_ptr(),
                                          on.stream));
  return out;
}

Tensor gate_forward(const Tensor& residual, const Tensor& x, const OptTensor& weight, const OptTensor& gate,
                    const OptTensor& doc_ids, double eps) {
  refuse_tangents({&residual, &x, &some(weight), &some(gate)});
  check_like("residual", residual, x);
  const Norm a(x, weight, "gate", gate, doc_ids, eps);
  Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
  if (a.empty()) return out;
  const Tokens xt(x), rt(residual);
  const Launch on(x);
  check_status(lib.sage_rms_norm_gate_residual(rt.p(), rt.bs, rt.rs, xt.p(), xt.bs, xt.rs, ptr(a.weight), COND(a.cond),
                                               TAIL(a), out.data_ptr(), on.stream));
  return out;
}

std::tuple<Tensor, Tensor> gate_modulate_forward(const Tensor& residual, const Tensor& x, const OptTensor& weight,
                                                 const OptTensor& gate, const OptTensor& next_weight,
                                                 const OptTensor& next_scale, const OptTensor& doc_ids, double eps) {
  refuse_tangents({&residual, &x, &some(weight), &some(gate), &some(next_weight), &some(next_scale)});
  check_like("residual", residual, x);
  const Norm a(x, weight, "gate", gate, doc_ids, eps, next_weight, next_scale);
  Tensor hidden = at::empty(x.sizes(), x.options().requires_grad(false)), out = at::empty_like(hidden);
  if (!a.empty()) {
    const Tokens xt(x), rt(residual);
    const Launch on(x);
    check_status(lib.sage_rms_norm_gate_residual_modulate(
        rt.p(), rt.bs, rt.rs, xt.p(), xt.bs, xt.rs, ptr(a.weight), COND(a.cond), ptr(a.next_weight),
        COND(a.next_scale), TAIL(a), hidden.data_ptr(), out.data_ptr(), on.stream));
  }
  return {hidden, out};
}

typedef std::vector<bool> Wanted;

// Gradients; undefined where not wanted.  gate: the gate_residual form.
std::tuple<Tensor, Tensor, Tensor> norm_backward(bool gate, const Tensor& dout, const Tensor& x,
                                                 const OptTensor& weight, const OptTensor& cond,
                                                 const OptTensor& doc_ids, double eps, const Wanted& wanted) {
  refuse_tangents({&dout, &x, &some(weight), &some(cond)});
  check_like("dout", dout, x);
  const Norm a(x, weight, gate ? "gate" : "scale", cond, doc_ids, eps);
  Tensor dx = grad_of(x, wanted[0]), dw = grad_of(some(weight), wanted[1]), dc = grad_of(some(cond), wanted[2]);
  if (a.empty()) {
    zero({dw, dc});
  } else if (dx.defined() || dw.defined() || dc.defined()) {
    const Tokens xt(x), dt(dout);
    const size_t bytes = dw.defined() || dc.defined() ? a.bytes(false) : 0;
    const Tensor ws = workspace(x, bytes);
    const Launch on(x);
    check_status((gate ? lib.sage_rms_norm_gate_residual_bwd : lib.sage_rms_norm_modulate_bwd)(
        dt.p(), dt.bs, dt.rs, xt.p(), xt.bs, xt.rs, ptr(a.weight), COND(a.cond), TAIL(a), ptr(ws), bytes, ptr(dx),
        ptr(dw), ptr(dc), on.stream));
  }
  return {dx, dw, dc};
}

typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> Six;

// The residual's gradient, which the others come from, is always formed.
Six gate_modulate_backward(const Tensor& dhidden, const Tensor& dout, const Tensor& residual, const Tensor& x,
                           const OptTensor& weight, const OptTensor& gate, const OptTensor& next_weight,
                           const OptTensor& next_scale, const OptTensor& doc_ids, double eps, const Wanted& wanted) {
  refuse_tangents({&dhidden, &dout, &residual, &x, &some(weight), &some(gate), &some(next_weight), &some(next_scale)});
  check_like("residual", residual, x);
  check_like("dout", dout, x);
  check_like("dhidden", dhidden, x);
  const Norm a(x, weight, "gate", gate, doc_ids, eps, next_weight, next_scale);
  Tensor dr = grad_of(x, true), dx = grad_of(x, wanted[1]), dw = grad_of(some(weight), wanted[2]),
         dg = grad_of(some(gate), wanted[3]), dw2 = grad_of(some(next_weight), wanted[4]),
         ds = grad_of(some(next_scale), wanted[5]);
  if (a.empty()) {
    zero({dw, dg, dw2, ds});
  } else {
    const Tokens xt(x), rt(residual), dt(dout), ht(dhidden);
    const size_t bytes = dw.defined() || dg.defined() || dw2.defined() || ds.defined() ? a.bytes(true) : 0;
    const Tensor ws = workspace(x, bytes);
    const Launch on(x);
    check_status(lib.sage_rms_norm_gate_residual_modulate_bwd(
        ht.p(), ht.bs, ht.rs, dt.p(), dt.bs, dt.rs, rt.p(), rt.bs, rt.rs, xt.p(), xt.bs, xt.rs, ptr(a.weight),
        COND(a.cond), ptr(a.next_weight), COND(a.next_scale), TAIL(a), ptr(ws), bytes, dr.data_ptr(), ptr(dx), ptr(dw),
        ptr(dg), ptr(dw2), ptr(ds), on.stream));
  }
  return {dr, dx, dw, dg, dw2, ds};
}

// ---------------------------------------------------------------- linear

// [..., C] as rows [M, C] with contiguous columns, at least their width apart.
struct Matrix {
  Tensor t;
  int64_t rows, cols, rs;
  explicit Matrix(const Tensor& x) : t(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)})) {
    rows = t.size(0);
    cols = t.size(1);
    if ((cols != 1 && t.stride(1) != 1) || (rows > 1 && (t.stride(0) < cols || t.stride(0) >= (int64_t)1 << 22)))
      t = t.contiguous();
    rs = t.stride(0);
  }
  void* p() const { return t.data_ptr(); }
};

int activation_of(const std::string& name) {
  if (name == "none") return SAGE_ACT_NONE;
  if (name == "silu") return SAGE_ACT_SILU;
  if (name == "gelu") return SAGE_ACT_GELU;
  TORCH_CHECK_VALUE(name == "swiglu", "activation must be one of gelu, none, silu, swiglu, got '", name, "'");
  return SAGE_ACT_SWIGLU;
}

// The checked arguments of a linear call.
struct Linear {
  int act, dtype;
  bool f32 = false;
  int64_t K, rows, N, M;
  std::vector<int64_t> shape;
  Tensor bias;

  Linear(const Tensor& x, const Tensor& weight, const OptTensor& b, const OptTensor& residual,
         const std::string& activation)
      : act(activation_of(activation)), dtype(dtype_of(x)) {
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must be [..., K], got a scalar");
    K = x.size(-1);
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) == K && K >= 1 && weight.size(0) >= 1 &&
                          weight.scalar_type() == x.scalar_type() && weight.device() == x.device(),
                      "weight must be a ", x.scalar_type(), " [N, ", K, "] tensor on ", x.device(), ", got ",
                      weight.scalar_type(), " ", weight.sizes(), " on ", weight.device());
    rows = weight.size(0);
    TORCH_CHECK_VALUE(act != SAGE_ACT_SWIGLU || rows % 2 == 0, "a swiglu weight has an even number of rows, got ", rows);
    N = act == SAGE_ACT_SWIGLU ? rows / 2 : rows;
    M = x.numel() / K;
    if (b) {
      TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == rows && is_param(*b, x), "bias must be a [", rows,
                        "] tensor of ", x.scalar_type(), " or float32 on ", x.device(), ", got ", b->scalar_type(), " ",
                        b->sizes(), " on ", b->device());
      f32 = b->scalar_type() == at::kFloat;
      bias = b->contiguous();
    }
    shape = x.sizes().vec();
    shape.back() = N;
    if (residual) check_out("residual", *residual, x);
    need_gpu(x);
  }
  void check_out(const char* name, const Tensor& t, const Tensor& x) const {
    TORCH_CHECK_VALUE(t.sizes() == c10::IntArrayRef(shape) && t.scalar_type() == x.scalar_type() &&
                          t.device() == x.device(),
                      name, " must be a ", x.scalar_type(), " ", c10::IntArrayRef(shape), " tensor on ", x.device(),
                      ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
  }
};

bool off16(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15u; }

// out, and z where it is kept (an activation, keep_z).
std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                          const OptTensor& residual, const std::string& activation, bool keep_z) {
  refuse_tangents({&x, &weight, &some(bias), &some(residual)});
  const Linear a(x, weight, bias, residual, activation);
  const auto options = x.options().requires_grad(false);
  Tensor out = at::empty(a.shape, options), z;
  if (keep_z && a.act != SAGE_ACT_NONE) z = at::empty({a.M, a.rows}, options.dtype(at::kFloat));
  if (a.M == 0) return {out, z};
  const Matrix xm(x), wm(weight);
  std::optional<Matrix> rm;
  if (residual) rm.emplace(*residual);
  const void* rp = rm ? rm->p() : nullptr;
  const int64_t rs = rm ? rm->rs : 0;
  const size_t bytes = lib.sage_linear_workspace_bytes(xm.p(), xm.rs, wm.p(), wm.rs, a.M, a.N, a.K, a.act,
                                                       off16(rp) || off16(ptr(a.bias)) || rs % 8 != 0);
  const Tensor ws = workspace(x, bytes);
  const Launch on(x);
  check_status(lib.sage_linear(xm.p(), xm.rs, wm.p(), wm.rs, ptr(a.bias), a.f32, rp, rs, a.M, a.N, a.K, a.dtype, a.act,
                               ptr(ws), bytes, static_cast<float*>(ptr(z)), out.data_ptr(), on.stream));
  return {out, z};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& dout, const Tensor& x, const Tensor& weight,
                                                   const OptTensor& bias, const OptTensor& z,
                                                   const std::string& activation, const Wanted& wanted) {
  refuse_tangents({&dout, &x, &weight, &some(bias)});
  const Linear a(x, weight, bias, std::nullopt, activation);
  a.check_out("dout", dout, x);
  const bool act = a.act != SAGE_ACT_NONE;
  const bool none = !act || !(wanted[0] || wanted[1] || wanted[2]);
  TORCH_CHECK_VALUE(none || (z && z->defined() && z->dim() == 2 && z->size(0) == a.M && z->size(1) == a.rows &&
                             z->scalar_type() == at::kFloat && z->device() == x.device() && z->is_contiguous()),
                    "the gradient of an activation needs the z that the forward kept (keep_z)");
  Tensor dx = grad_of(x, wanted[0]), dw = grad_of(weight, wanted[1]), db = grad_of(some(bias), wanted[2]);
  const int want = (dx.defined() ? 1 : 0) | (dw.defined() ? 2 : 0) | (db.defined() ? 4 : 0);
  if (a.M == 0) {
    zero({dw, db});
  } else if (want) {
    const Matrix dm(dout), xm(x), wm(weight);
    const size_t bytes = lib.sage_linear_bwd_workspace_bytes(dm.p(), dm.rs, xm.p(), xm.rs, wm.p(), wm.rs, a.M, a.N,
                                                             a.K, a.act, want);
    const Tensor ws = workspace(x, bytes);
    const Launch on(x);
    check_status(lib.sage_linear_bwd(dm.p(), dm.rs, xm.p(), xm.rs, wm.p(), wm.rs, act ? z->data_ptr<float>() : nullptr, a.M,
                                     a.N, a.K, a.dtype, a.act, a.f32, ptr(ws), bytes, ptr(dx), ptr(dw), ptr(db),
                                     on.stream));
  }
  return {dx, dw, db};
}

// ---------------------------------------------------------------- tracing

// Whether a call has to go through its registered op: a tracer, a dispatch mode or a functorch
// transform is active, or an argument is a wrapper or a lazy view (negated, zeros without
// storage).  The functions below see storage alone: a trace of them would record the allocation
// of the outputs and nothing that writes them.
// A tangent is refused here too: behind the dispatcher a transform has taken it off.
bool through_dispatcher(std::initializer_list<const Tensor*> tensors) {
  using c10::DispatchKey;
  static constexpr c10::DispatchKeySet hooks(
      {DispatchKey::Fake, DispatchKey::Python, DispatchKey::PythonTLSSnapshot, DispatchKey::PythonDispatcher,
       DispatchKey::Tracer, DispatchKey::Functionalize, DispatchKey::Conjugate, DispatchKey::Negative,
       DispatchKey::ZeroTensor, DispatchKey::Batched, DispatchKey::VmapMode, DispatchKey::FuncTorchBatched,
       DispatchKey::FuncTorchBatchedDecomposition, DispatchKey::FuncTorchVmapMode, DispatchKey::FuncTorchGradWrapper,
       DispatchKey::FuncTorchDynamicLayerBackMode, DispatchKey::FuncTorchDynamicLayerFrontMode});
  const auto local = c10::impl::tls_local_dispatch_key_set();
  c10::DispatchKeySet keys = local.included_;
  for (const Tensor* t : tensors)
    if (t->defined()) keys = keys | t->key_set();
  if (((keys - local.excluded_) & hooks).raw_repr() == 0) return false;
  refuse_tangents(tensors);
  return true;
}

// The registered op futudiffu_ii::<name> on these arguments.
template <typename... Args>
torch::jit::Stack call_op(const char* name, Args&&... args) {
  torch::jit::Stack stack;
  torch::jit::push(stack, std::forward<Args>(args)...);
  c10::Dispatcher::singleton().findSchemaOrThrow((std::string("futudiffu_ii::") + name).c_str(), "").callBoxed(&stack);
  return stack;
}

// ---------------------------------------------------------------- autograd

Tensor held(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// Which of a function's tensor arguments want a gradient: an absent one has no edge.
Wanted needs(AutogradContext* ctx, const variable_list& args) {
  Wanted w;
  size_t edge = 0;
  for (const Tensor& t : args) w.push_back(t.defined() ? ctx->needs_input_grad(edge++) : false);
  return w;
}

c10::List<bool> list_of(const Wanted& w) {
  c10::List<bool> l;
  for (const bool b : w) l.push_back(b);
  return l;
}

// What a gradient op returned, undefined in the place of what is not wanted.
variable_list gradients(const torch::jit::Stack& returned, const Wanted& w) {
  variable_list g;
  for (size_t i = 0; i < returned.size(); ++i) g.push_back(w[i] ? returned[i].toTensor() : Tensor());
  return g;
}

// The gradients are not themselves differentiable.
void once(const variable_list& args) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor& t : args)
    TORCH_CHECK(!t.defined() || !t.requires_grad(),
                "the gradients of the block operators cannot be differentiated (create_graph=True)");
}

bool any_requires(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  return at::GradMode::is_enabled() && any_requires(tensors);
}

struct ModulateFn : torch::autograd::Function<ModulateFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& scale,
                        const OptTensor& doc_ids, double eps) {
    ctx->save_for_backward({x, held(weight), held(scale), held(doc_ids)});
    ctx->saved_data["eps"] = eps;
    return modulate_forward(x, weight, scale, doc_ids, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto s = ctx->get_saved_variables();
    once({d[0], s[0], s[1], s[2]});
    const Wanted w = needs(ctx, {s[0], s[1], s[2]});
    const double eps = ctx->saved_data["eps"].toDouble();
    if (through_dispatcher({&d[0], &s[0], &s[1], &s[2], &s[3]})) {
      const auto g = gradients(
          call_op("rms_norm_modulate_backward", d[0], s[0], given(s[1]), given(s[2]), given(s[3]), eps, list_of(w)), w);
      return {g[0], g[1], g[2], Tensor(), Tensor()};
    }
    const auto [dx, dw, dc] = norm_backward(false, d[0], s[0], given(s[1]), given(s[2]), given(s[3]), eps, w);
    return {dx, dw, dc, Tensor(), Tensor()};
  }
};

struct GateFn : torch::autograd::Function<GateFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& residual, const Tensor& x, const OptTensor& weight,
                        const OptTensor& gate, const OptTensor& doc_ids, double eps) {
    ctx->save_for_backward({x, held(weight), held(gate), held(doc_ids)});
    ctx->saved_data["eps"] = eps;
    return gate_forward(residual, x, weight, gate, doc_ids, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto s = ctx->get_saved_variables();
    once({d[0], s[0], s[1], s[2]});
    const Wanted all = needs(ctx, {s[0], s[0], s[1], s[2]});  // the residual's edge comes first
    const Wanted w = {all[1], all[2], all[3]};
    const Tensor dr = all[0] ? d[0] : Tensor();
    const double eps = ctx->saved_data["eps"].toDouble();
    if (through_dispatcher({&d[0], &s[0], &s[1], &s[2], &s[3]})) {
      const auto g = gradients(call_op("rms_norm_gate_residual_backward", d[0], s[0], given(s[1]), given(s[2]),
                                       given(s[3]), eps, list_of(w)), w);
      return {dr, g[0], g[1], g[2], Tensor(), Tensor()};
    }
    const auto [dx, dw, dg] = norm_backward(true, d[0], s[0], given(s[1]), given(s[2]), given(s[3]), eps, w);
    return {dr, dx, dw, dg, Tensor(), Tensor()};
  }
};

struct GateModulateFn : torch::autograd::Function<GateModulateFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& residual, const Tensor& x, const OptTensor& weight,
                               const OptTensor& gate, const OptTensor& next_weight, const OptTensor& next_scale,
                               const OptTensor& doc_ids, double eps) {
    ctx->save_for_backward({residual, x, held(weight), held(gate), held(next_weight), held(next_scale), held(doc_ids)});
    ctx->saved_data["eps"] = eps;
    const auto [hidden, out] = gate_modulate_forward(residual, x, weight, gate, next_weight, next_scale, doc_ids, eps);
    return {hidden, out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto s = ctx->get_saved_variables();
    once({d[0], d[1], s[0], s[1], s[2], s[3], s[4], s[5]});
    const Wanted w = needs(ctx, {s[0], s[1], s[2], s[3], s[4], s[5]});
    const double eps = ctx->saved_data["eps"].toDouble();
    if (through_dispatcher({&d[0], &d[1], &s[0], &s[1], &s[2], &s[3], &s[4], &s[5], &s[6]})) {
      const auto g = gradients(call_op("rms_norm_gate_residual_modulate_backward", d[0], d[1], s[0], s[1], given(s[2]),
                                       given(s[3]), given(s[4]), given(s[5]), given(s[6]), eps, list_of(w)), w);
      return {g[0], g[1], g[2], g[3], g[4], g[5], Tensor(), Tensor()};
    }
    auto [dr, dx, dw, dg, dw2, ds] = gate_modulate_backward(d[0], d[1], s[0], s[1], given(s[2]), given(s[3]),
                                                            given(s[4]), given(s[5]), given(s[6]), eps, w);
    return {w[0] ? dr : Tensor(), dx, dw, dg, dw2, ds, Tensor(), Tensor()};
  }
};

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                        const OptTensor& residual, const std::string& activation) {
    // a residual's gradient alone needs no z
    const auto [out, z] =
        linear_forward(x, weight, bias, residual, activation, any_requires({&x, &weight, &some(bias)}));
    ctx->save_for_backward({x, weight, held(bias), z});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["residual"] = residual.has_value();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto s = ctx->get_saved_variables();
    once({d[0], s[0], s[1], s[2]});
    // x, weight, bias, then the residual's edge
    const Wanted all = needs(ctx, {s[0], s[1], s[2], ctx->saved_data["residual"].toBool() ? s[0] : Tensor()});
    const Wanted w = {all[0], all[1], all[2]};
    const Tensor dr = all[3] ? d[0] : Tensor();
    const std::string& activation = ctx->saved_data["activation"].toStringRef();
    if (through_dispatcher({&d[0], &s[0], &s[1], &s[2], &s[3]})) {
      const auto g = gradients(
          call_op("fused_linear_backward", d[0], s[0], s[1], given(s[2]), given(s[3]), activation, list_of(w)), w);
      return {g[0], g[1], g[2], dr, Tensor()};
    }
    const auto [dx, dw, db] = linear_backward(d[0], s[0], s[1], given(s[2]), given(s[3]), activation, w);
    return {dx, dw, db, dr, Tensor()};
  }
};

Tensor rms_norm_modulate(const Tensor& x, const OptTensor& weight, const OptTensor& scale, const OptTensor& doc_ids,
                         double eps) {
  if (through_dispatcher({&x, &some(weight), &some(scale), &some(doc_ids)}))
    return call_op("rms_norm_modulate", x, weight, scale, doc_ids, eps)[0].toTensor();
  if (wants_grad({&x, &some(weight), &some(scale)})) return ModulateFn::apply(x, weight, scale, doc_ids, eps);
  return modulate_forward(x, weight, scale, doc_ids, eps);
}

Tensor rms_norm_gate_residual(const Tensor& residual, const Tensor& x, const OptTensor& weight, const OptTensor& gate,
                              const OptTensor& doc_ids, double eps) {
  if (through_dispatcher({&residual, &x, &some(weight), &some(gate), &some(doc_ids)}))
    return call_op("rms_norm_gate_residual", residual, x, weight, gate, doc_ids, eps)[0].toTensor();
  if (wants_grad({&residual, &x, &some(weight), &some(gate)}))
    return GateFn::apply(residual, x, weight, gate, doc_ids, eps);
  return gate_forward(residual, x, weight, gate, doc_ids, eps);
}

std::tuple<Tensor, Tensor> rms_norm_gate_residual_modulate(const Tensor& residual, const Tensor& x,
                                                           const OptTensor& weight, const OptTensor& gate,
                                                           const OptTensor& next_weight, const OptTensor& next_scale,
                                                           const OptTensor& doc_ids, double eps) {
  if (through_dispatcher({&residual, &x, &some(weight), &some(gate), &some(next_weight), &some(next_scale),
                          &some(doc_ids)})) {
    const auto r =
        call_op("rms_norm_gate_residual_modulate", residual, x, weight, gate, next_weight, next_scale, doc_ids, eps);
    return {r[0].toTensor(), r[1].toTensor()};
  }
  if (wants_grad({&residual, &x, &some(weight), &some(gate), &some(next_weight), &some(next_scale)})) {
    const auto r = GateModulateFn::apply(residual, x, weight, gate, next_weight, next_scale, doc_ids, eps);
    return {r[0], r[1]};
  }
  return gate_modulate_forward(residual, x, weight, gate, next_weight, next_scale, doc_ids, eps);
}

Tensor fused_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                    const std::string& activation) {
  if (through_dispatcher({&x, &weight, &some(bias), &some(residual)})) {
    // what vmap batches does not say whether what lies under it wants a gradient: z is kept
    const bool hidden = x.key_set().has(c10::DispatchKey::FuncTorchBatched) ||
                        weight.key_set().has(c10::DispatchKey::FuncTorchBatched) ||
                        some(bias).key_set().has(c10::DispatchKey::FuncTorchBatched);
    const bool keep_z = activation != "none" && at::GradMode::is_enabled() &&
                        (hidden || any_requires({&x, &weight, &some(bias)}));
    return call_op("fused_linear", x, weight, bias, residual, activation, keep_z)[0].toTensor();
  }
  if (wants_grad({&x, &weight, &some(bias), &some(residual)}))
    return LinearFn::apply(x, weight, bias, residual, activation);
  return std::get<0>(linear_forward(x, weight, bias, residual, activation, false));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("rms_norm_modulate", &rms_norm_modulate);
  m.def("rms_norm_gate_residual", &rms_norm_gate_residual);
  m.def("rms_norm_gate_residual_modulate", &rms_norm_gate_residual_modulate);
  m.def("fused_linear", &fused_linear);
  // what the custom ops call: no autograd
  m.def("modulate_forward", &modulate_forward);
  m.def("gate_forward", &gate_forward);
  m.def("gate_modulate_forward", &gate_modulate_forward);
  m.def("norm_backward", &norm_backward);
  m.def("gate_modulate_backward", &gate_modulate_backward);
  m.def("linear_forward", &linear_forward);
  m.def("linear_backward", &linear_backward);
}

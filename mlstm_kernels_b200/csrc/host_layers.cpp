// The host side of the operators around a recurrence - layer norm, short causal convolution, selective state space scan - in the
// manner of host.cpp: checks of the arguments, allocations, autograd nodes and launches of a call without a Python frame in
// between.  Tensors whose last axis is contiguous are read where they are, whatever their other strides.
#include "host.h"

namespace {

using namespace mlstm_host;

using OptT = std::optional<Tensor>;
OptT given(const Tensor& t) { return t.defined() ? OptT(t) : std::nullopt; }
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// All on the device of the first; no forward-mode tangents, which would be dropped without a word.
void check_tensors(const char* op, std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), kNeedsCuda);
    if (t->device() != first.device()) C10_THROW_ERROR(ValueError, c10::str(op, ": tensors on different devices (", first.device(), " and ", t->device(), ")"));
    if (t->layout() != at::kStrided) C10_THROW_ERROR(ValueError, c10::str(op, ": tensors must be dense"));
    if (t->_fw_grad(0).defined()) C10_THROW_ERROR(NotImplementedError, c10::str("mlstm_kernels_b200 has no forward-mode derivative of ", op));
  }
}
void check_kernel_dtype(const Tensor& t) {
  if (t.defined() && dtype_code(t.scalar_type()) < 0) C10_THROW_ERROR(ValueError, c10::str("Unsupported kernel dtype ", t.dtype(), "."));
}
[[noreturn]] void bad_shape(const char* op, const char* name, const Tensor& t, const char* want) {
  C10_THROW_ERROR(ValueError, c10::str(op, ": ", name, " of shape ", t.sizes(), " must be ", want));
}
void check_int_sizes(const char* op, const Tensor& t) {   // the kernels count single axes in 32 bits
  for (const int64_t n : t.sizes())
    if (n > (1ll << 30)) C10_THROW_ERROR(ValueError, c10::str(op, ": an axis of more than 2^30 elements"));
}
void no_second_derivative(const char* op) {
  if (at::GradMode::is_enabled()) C10_THROW_ERROR(NotImplementedError, c10::str("mlstm_kernels_b200 has no second derivative of ", op));
}
// A buffer that a step writes (contiguous, as are those that it reads): it may be the state that it replaces, and lies apart from
// everything else.  Autograd is told of the write, so that a graph that kept the old contents does not take the new ones for them.
void check_written(const char* op, const char* name, const Tensor& out, const Tensor& state, std::initializer_list<const Tensor*> ins) {
  const uintptr_t o = reinterpret_cast<uintptr_t>(out.const_data_ptr());
  auto meets = [&](const Tensor& t) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    return p < o + out.nbytes() && o < p + t.nbytes();
  };
  bool apart = state.const_data_ptr() == out.const_data_ptr() || !meets(state);
  for (const Tensor* t : ins) apart = apart && !(t->defined() && meets(*t));
  if (!apart) C10_THROW_ERROR(ValueError, c10::str(op, ": ", name, " overlaps a tensor that the step reads (only the whole old state may be replaced in place)"));
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}
// What a backward operator is given beside the forward's inputs
void check_size(const char* op, const char* name, const Tensor& t, at::IntArrayRef size) {
  if (t.defined() && t.sizes() != size) C10_THROW_ERROR(ValueError, c10::str(op, ": ", name, " of shape ", t.sizes(), " must be of shape ", size));
}
// as a kernel reads it: the last axis contiguous
Tensor last_dense(const Tensor& t) { return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
Tensor zeros(at::IntArrayRef size, at::ScalarType dt, const at::Device& dev) { return empty(size, dt, dev).zero_(); }
Tensor to_dtype(const Tensor& t, at::ScalarType dt) { return !t.defined() || t.scalar_type() == dt ? t : t.to(dt); }

// ---- layer norm ---------------------------------------------------------------------------------------
// The axes in front of the normalised one (and of the heads) as two, cut in front of axis k; null sizes where the strides do
// not allow that.
struct Rows {
  bool ok;
  int64_t n0, n1;
  long long s[3];
};
Rows rows_of(const Tensor& t, bool heads, int64_t k) {
  Rows r{true, 1, 1, {0, 0, heads ? (long long)t.stride(-2) : 0}};
  const int64_t outer = t.dim() - 1 - (heads ? 1 : 0);
  if (t.size(-1) > 1 && t.stride(-1) != 1) r.ok = false;
  auto group = [&](int64_t from, int64_t to, int64_t& n, long long& s) {
    for (int64_t i = to - 1; i >= from; --i) {
      if (t.size(i) == 1) continue;
      if (n == 1) s = t.stride(i);
      else if (t.stride(i) != n * s) r.ok = false;
      n *= t.size(i);
    }
  };
  group(0, k, r.n0, r.s[0]);
  group(k, outer, r.n1, r.s[1]);
  return r;
}
int64_t cut_of(const Tensor& t, bool heads) {   // -1: no cut will do
  const int64_t outer = t.dim() - 1 - (heads ? 1 : 0);
  for (int64_t k = 0; k <= outer; ++k)
    if (rows_of(t, heads, k).ok) return k;
  return -1;
}

const char* const kNorm = "layer_norm__b200";
void check_norm(const Tensor& x, const Tensor& w, const Tensor& b) {
  check_tensors(kNorm, {&x, &w, &b});
  check_kernel_dtype(x); check_kernel_dtype(w); check_kernel_dtype(b);
  if (x.dim() < 1) bad_shape(kNorm, "x", x, "(..., D)");
  check_int_sizes(kNorm, x);
  if (x.size(-1) > 16384) C10_THROW_ERROR(ValueError, c10::str("layer_norm__b200: rows of more than 16384 elements (x of shape ", x.sizes(), ")"));
  for (const Tensor* p : {&w, &b}) {
    if (!p->defined()) continue;
    const bool fits = (p->dim() == 1 && p->size(0) == x.size(-1)) ||
                      (p->dim() == 2 && x.dim() >= 2 && p->size(0) == x.size(-2) && p->size(1) == x.size(-1));
    if (!fits) bad_shape(kNorm, p == &w ? "weight" : "bias", *p, "(D,) or (NH, D) for x (..., D) or (..., NH, D)");
  }
  if (w.defined() && b.defined() && (w.sizes() != b.sizes() || w.scalar_type() != b.scalar_type()))
    C10_THROW_ERROR(ValueError, "layer_norm__b200: weight and bias must share one shape and one dtype");
}
bool norm_heads(const Tensor& w, const Tensor& b) { return (w.defined() && w.dim() == 2) || (b.defined() && b.dim() == 2); }
int norm_param(const Tensor& w, const Tensor& b) { return w.defined() ? dtype_code(w.scalar_type()) : b.defined() ? dtype_code(b.scalar_type()) : MLSTM_F32; }

struct Normed { Tensor y, mean, rstd; };
Normed norm_forward(const Tensor& x_, const Tensor& w_, const Tensor& b_, double eps, bool keep) {
  const bool heads = norm_heads(w_, b_);
  const at::Device dev = x_.device();
  Normed o;
  o.y = empty(x_.sizes(), x_.scalar_type(), dev);
  const int64_t D = x_.size(-1), rows = D > 0 ? x_.numel() / D : 0;
  if (keep) { o.mean = empty({rows}, at::kFloat, dev); o.rstd = empty({rows}, at::kFloat, dev); }
  if (x_.numel() == 0) return o;
  int64_t k = cut_of(x_, heads);
  const Tensor x = k < 0 ? x_.contiguous() : x_;
  k = std::max<int64_t>(k, 0);
  const Tensor w = w_.defined() ? w_.contiguous() : w_, b = b_.defined() ? b_.contiguous() : b_;
  const Rows r = rows_of(x, heads, k);
  check(mlstm_b200_layer_norm_fw(ptr(x), r.s, ptr(w), ptr(b), o.y.mutable_data_ptr(), fout(o.mean), fout(o.rstd), r.n0, r.n1,
                                 heads ? (int)x.size(-2) : 1, (int)D, dtype_code(x.scalar_type()), norm_param(w, b), (float)eps, current_stream(dev)),
        "mlstm_b200_layer_norm_fw");
  return o;
}
struct NormGrads { Tensor dx, dw, db; };
NormGrads norm_backward(const Tensor& x_, const Tensor& w_, const Tensor& mean, const Tensor& rstd, const Tensor& dy_, bool heads, at::ScalarType pdt,
                        bool want_w, bool want_b) {
  const at::Device dev = x_.device();
  const int64_t D = x_.size(-1), NH = heads ? x_.size(-2) : 1;
  NormGrads g;
  std::array<int64_t, 2> par{NH, D};
  const at::IntArrayRef psize = heads ? at::IntArrayRef(par) : at::IntArrayRef(par).slice(1);
  if (x_.numel() == 0) {
    g.dx = empty(x_.sizes(), x_.scalar_type(), dev);
    if (want_w) g.dw = zeros(psize, pdt, dev);
    if (want_b) g.db = zeros(psize, pdt, dev);
    return g;
  }
  int64_t k = cut_of(x_, heads);
  const Tensor x = k < 0 ? x_.contiguous() : x_;
  k = std::max<int64_t>(k, 0);
  Tensor dy = to_dtype(dy_, x.scalar_type());
  if (!rows_of(dy, heads, k).ok) dy = dy.contiguous();
  // the gradient lies as x does, where x covers its memory once: it goes on to what made x without a copy
  if (x.is_non_overlapping_and_dense()) g.dx = at::empty_like(x, x.options(), at::MemoryFormat::Preserve);
  if (!g.dx.defined() || !rows_of(g.dx, heads, k).ok) g.dx = empty(x.sizes(), x.scalar_type(), dev);
  if (want_w) g.dw = empty(psize, pdt, dev);
  if (want_b) g.db = empty(psize, pdt, dev);
  const Tensor w = w_.defined() ? w_.contiguous() : w_;
  const Rows xr = rows_of(x, heads, k), yr = rows_of(dy, heads, k), dr = rows_of(g.dx, heads, k);
  const size_t need = want_w || want_b ? mlstm_b200_layer_norm_bw_workspace_bytes(xr.n0 * xr.n1, (int)NH, (int)D) : 0;
  const Tensor ws = need > 0 ? bytes(need, dev) : Tensor();
  check(mlstm_b200_layer_norm_bw(ptr(x), xr.s, ptr(w), fptr(mean), fptr(rstd), ptr(dy), yr.s, g.dx.mutable_data_ptr(), dr.s,
                                 want_w ? g.dw.mutable_data_ptr() : nullptr, want_b ? g.db.mutable_data_ptr() : nullptr, fout(ws), need, xr.n0, xr.n1,
                                 (int)NH, (int)D, dtype_code(x.scalar_type()), dtype_code(pdt), current_stream(dev)),
        "mlstm_b200_layer_norm_bw");
  return g;
}

class NormFn : public torch::autograd::Function<NormFn> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptT& w_opt, const OptT& b_opt, double eps) {
    const Tensor w = w_opt.value_or(Tensor()), b = b_opt.value_or(Tensor());
    Normed o = norm_forward(x, w, b, eps, true);
    ctx->save_for_backward({x, w, o.mean, o.rstd});
    ctx->saved_data["cfg"] = std::vector<int64_t>{norm_heads(w, b), norm_param(w, b), w.defined() && w.requires_grad(), b.defined() && b.requires_grad()};
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative(kNorm);
    const auto saved = ctx->get_saved_variables();
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    c10::cuda::OptionalCUDAGuard guard(saved[0].device());
    const NormGrads g = norm_backward(saved[0], saved[1], saved[2], saved[3], grads[0], cfg[0] != 0, code_dtype((int)cfg[1]), cfg[2] != 0, cfg[3] != 0);
    return {g.dx, g.dw, g.db, Tensor()};
  }
};

// layer_norm(x, weight, bias, eps) -> y
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 4);
  const Tensor x = need(a[0], "x"), w = arg(a[1], "weight"), b = arg(a[2], "bias");
  const double eps = double_arg(a[3]);
  check_norm(x, w, b);
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::OptionalCUDAGuard guard(x.device());
    if (wants_grad({&x, &w, &b})) {
      y = NormFn::apply(x, given(w), given(b), eps);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      y = norm_forward(x, w, b, eps, false).y;
    }
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}
// layer_norm_fw(x, weight, bias, eps) -> (y, mean, rstd);  layer_norm_bw(x, weight, mean, rstd, dy, heads, param_dtype, want_w, want_b) -> (dx, dw, db)
PyObject* py_layer_norm_fw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 4);
  const Tensor x = need(a[0], "x"), w = arg(a[1], "weight"), b = arg(a[2], "bias");
  check_norm(x, w, b);
  c10::cuda::OptionalCUDAGuard guard(x.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Normed o = norm_forward(x, w, b, double_arg(a[3]), true);
  return Py_BuildValue("(NNN)", wrap(o.y), wrap(o.mean), wrap(o.rstd));
  END_HANDLE_TH_ERRORS
}
PyObject* py_layer_norm_bw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 9);
  const Tensor x = need(a[0], "x"), w = arg(a[1], "weight"), mean = need(a[2], "mean"), rstd = need(a[3], "rstd"), dy = need(a[4], "dy");
  check_norm(x, w, Tensor());
  check_tensors(kNorm, {&x, &mean, &rstd, &dy});
  check_size(kNorm, "dy", dy, x.sizes());
  for (const Tensor* p : {&mean, &rstd}) {
    check_size(kNorm, "mean and rstd", *p, {x.size(-1) > 0 ? x.numel() / x.size(-1) : 0});
    if (p->scalar_type() != at::kFloat || !p->is_contiguous()) C10_THROW_ERROR(ValueError, "layer_norm__b200: mean and rstd must be contiguous f32 tensors");
  }
  const bool heads = bool_arg(a[5]);
  const at::ScalarType pdt = dtype_arg(a[6]);
  if (heads && x.dim() < 2) bad_shape(kNorm, "x", x, "(..., NH, D)");
  if (w.defined() && (w.dim() == 2) != heads) bad_shape(kNorm, "weight", w, heads ? "(NH, D)" : "(D,)");
  if (dtype_code(pdt) < 0 || (w.defined() && w.scalar_type() != pdt)) C10_THROW_ERROR(ValueError, "layer_norm__b200: the weight must have the parameters' dtype, a kernel dtype");
  c10::cuda::OptionalCUDAGuard guard(x.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const NormGrads g = norm_backward(x, w, mean, rstd, dy, heads, pdt, bool_arg(a[7]), bool_arg(a[8]));
  return Py_BuildValue("(NNN)", wrap(g.dx), wrap(g.dw), wrap(g.db));
  END_HANDLE_TH_ERRORS
}

// ---- short convolution --------------------------------------------------------------------------------
const char* const kConv = "short_conv__b200";
void check_conv(const char* op, const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& before, bool one_token) {
  check_tensors(op, {&x, &w, &b, &before});
  check_kernel_dtype(x); check_kernel_dtype(w); check_kernel_dtype(b);
  if (x.dim() != (one_token ? 2 : 3)) bad_shape(op, "x", x, one_token ? "(B, D)" : "(B, S, D)");
  check_int_sizes(op, x);
  const int64_t D = x.size(-1);
  if (w.dim() != 2 || w.size(0) != D || w.size(1) < 2 || w.size(1) > 4) bad_shape(op, "weight", w, "(D, W) with 2 to 4 taps");
  if (b.defined() && (b.dim() != 1 || b.size(0) != D)) bad_shape(op, "bias", b, "(D,)");
  if (b.defined() && b.scalar_type() != w.scalar_type()) C10_THROW_ERROR(ValueError, c10::str(op, ": weight and bias must share one dtype"));
  if (before.defined()) {
    if (before.sizes() != at::IntArrayRef{x.size(0), w.size(1) - 1, D})
      bad_shape(op, one_token ? "state" : "x_initial", before, "(B, W - 1, D)");
    if (before.scalar_type() != x.scalar_type()) C10_THROW_ERROR(ValueError, c10::str(op, ": the tokens before must have x's dtype"));
  }
}
struct Conved { Tensor y, last; };
Conved conv_forward(const Tensor& x_, const Tensor& w_, const Tensor& b_, const Tensor& before_, bool want_last, bool silu) {
  const at::Device dev = x_.device();
  const int64_t B = x_.size(0), S = x_.size(1), D = x_.size(2), W = w_.size(1);
  Conved o;
  o.y = empty({B, S, D}, x_.scalar_type(), dev);
  if (want_last) o.last = empty({B, W - 1, D}, x_.scalar_type(), dev);
  if (x_.numel() == 0) {   // no token: the last ones are those before
    if (want_last) { if (before_.defined()) o.last.copy_(before_); else o.last.zero_(); }
    return o;
  }
  const Tensor x = last_dense(x_), w = w_.contiguous(), b = b_.defined() ? b_.contiguous() : b_, before = before_.defined() ? before_.contiguous() : before_;
  const long long xs[2] = {x.stride(0), x.stride(1)};
  check(mlstm_b200_short_conv_fw(ptr(x), xs, ptr(before), ptr(w), ptr(b), o.y.mutable_data_ptr(), want_last ? o.last.mutable_data_ptr() : nullptr,
                                 (int)B, (int)S, (int)D, (int)W, silu, dtype_code(x.scalar_type()), dtype_code(w.scalar_type()), current_stream(dev)),
        "mlstm_b200_short_conv_fw");
  return o;
}
struct ConvGrads { Tensor dx, dw, db, dbefore; };
// dy undefined: nothing came back for y
ConvGrads conv_backward(const Tensor& x_, const Tensor& w_, const Tensor& b_, const Tensor& before_, const Tensor& dy_, const Tensor& dlast_, bool silu,
                        bool want_w, bool want_b, bool want_before) {
  const at::Device dev = x_.device();
  const int64_t B = x_.size(0), S = x_.size(1), D = x_.size(2), W = w_.size(1);
  const at::ScalarType dt = x_.scalar_type(), pdt = w_.scalar_type();
  ConvGrads g;
  g.dx = empty({B, S, D}, dt, dev);
  if (want_w) g.dw = empty({D, W}, pdt, dev);
  if (want_b) g.db = empty({D}, pdt, dev);
  if (want_before) g.dbefore = empty({B, W - 1, D}, dt, dev);
  if (x_.numel() == 0) {
    if (want_w) g.dw.zero_();
    if (want_b) g.db.zero_();
    if (want_before) { if (dlast_.defined()) g.dbefore.copy_(dlast_); else g.dbefore.zero_(); }
    return g;
  }
  const Tensor x = last_dense(x_), w = w_.contiguous(), b = b_.defined() ? b_.contiguous() : b_, before = before_.defined() ? before_.contiguous() : before_;
  const Tensor dy = dy_.defined() ? last_dense(to_dtype(dy_, dt)) : zeros({B, S, D}, dt, dev);
  const Tensor dlast = dlast_.defined() ? conform(dlast_, dt) : dlast_;
  const long long xs[2] = {x.stride(0), x.stride(1)}, ys[2] = {dy.stride(0), dy.stride(1)};
  const size_t need = want_w || want_b ? mlstm_b200_short_conv_bw_workspace_bytes((int)B, (int)S, (int)D, (int)W) : 0;
  const Tensor ws = need > 0 ? bytes(need, dev) : Tensor();
  check(mlstm_b200_short_conv_bw(ptr(x), xs, ptr(before), ptr(w), ptr(b), ptr(dy), ys, ptr(dlast), g.dx.mutable_data_ptr(),
                                 want_before ? g.dbefore.mutable_data_ptr() : nullptr, want_w ? g.dw.mutable_data_ptr() : nullptr,
                                 want_b ? g.db.mutable_data_ptr() : nullptr, fout(ws), need, (int)B, (int)S, (int)D, (int)W, silu, dtype_code(dt),
                                 dtype_code(pdt), current_stream(dev)),
        "mlstm_b200_short_conv_bw");
  return g;
}

class ConvFn : public torch::autograd::Function<ConvFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& b_opt, const OptT& before_opt, bool want_last, bool silu) {
    const Tensor b = b_opt.value_or(Tensor()), before = before_opt.value_or(Tensor());
    Conved o = conv_forward(x, w, b, before, want_last, silu);
    ctx->save_for_backward({x, w, b, before});
    ctx->set_materialize_grads(false);
    ctx->saved_data["cfg"] = std::vector<int64_t>{silu, w.requires_grad(), b.defined() && b.requires_grad(), before.defined() && before.requires_grad()};
    if (want_last) return {o.y, o.last};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative(kConv);
    const auto saved = ctx->get_saved_variables();
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    c10::cuda::OptionalCUDAGuard guard(saved[0].device());
    const ConvGrads g = conv_backward(saved[0], saved[1], saved[2], saved[3], grads[0], grads.size() > 1 ? grads[1] : Tensor(), cfg[0] != 0,
                                      cfg[1] != 0, cfg[2] != 0, cfg[3] != 0);
    return {g.dx, g.dw, g.db, g.dbefore, Tensor(), Tensor()};
  }
};

// short_conv(x, weight, bias, x_initial, return_last, silu) -> (y, x_last or None)
PyObject* py_short_conv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 6);
  const Tensor x = need(a[0], "x"), w = need(a[1], "weight"), b = arg(a[2], "bias"), before = arg(a[3], "x_initial");
  const bool want_last = bool_arg(a[4]), silu = bool_arg(a[5]);
  check_conv(kConv, x, w, b, before, false);
  Tensor y, last;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::OptionalCUDAGuard guard(x.device());
    if (wants_grad({&x, &w, &b, &before})) {
      const auto o = ConvFn::apply(x, w, given(b), given(before), want_last, silu);
      y = o[0];
      if (want_last) last = o[1];
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      const Conved o = conv_forward(x, w, b, before, want_last, silu);
      y = o.y; last = o.last;
    }
  }
  return Py_BuildValue("(NN)", wrap(y), wrap(last));
  END_HANDLE_TH_ERRORS
}
// short_conv_bw(x, weight, bias, x_initial, dy, dx_last, silu, want_w, want_b, want_initial) -> (dx, dw, db, dx_initial)
PyObject* py_short_conv_bw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 10);
  const Tensor x = need(a[0], "x"), w = need(a[1], "weight"), b = arg(a[2], "bias"), before = arg(a[3], "x_initial"), dy = arg(a[4], "dy"), dl = arg(a[5], "dx_last");
  check_conv(kConv, x, w, b, before, false);
  check_tensors(kConv, {&x, &dy, &dl});
  check_size(kConv, "dy", dy, x.sizes());
  check_size(kConv, "dx_last", dl, {x.size(0), w.size(1) - 1, x.size(2)});
  c10::cuda::OptionalCUDAGuard guard(x.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const ConvGrads g = conv_backward(x, w, b, before, dy, dl, bool_arg(a[6]), bool_arg(a[7]), bool_arg(a[8]), bool_arg(a[9]));
  return Py_BuildValue("(NNNN)", wrap(g.dx), wrap(g.dw), wrap(g.db), wrap(g.dbefore));
  END_HANDLE_TH_ERRORS
}
// short_conv_step(x, state, weight, bias, silu, state_new) -> (y, state_new)
PyObject* py_short_conv_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 6);
  const char* const op = "short_conv_step__b200";
  Tensor x = need(a[0], "x"), state = need(a[1], "state"), w = need(a[2], "weight"), b = arg(a[3], "bias"), after = arg(a[5], "state_new");
  const bool silu = bool_arg(a[4]);
  check_conv(op, x, w, b, state, true);
  check_tensors(op, {&x, &after});
  if (after.defined() && (after.sizes() != state.sizes() || after.scalar_type() != x.scalar_type() || !after.is_contiguous()))
    C10_THROW_ERROR(ValueError, "short_conv_step__b200: state_new must be a contiguous (B, W - 1, D) tensor of x's dtype");
  at::NoGradGuard no_grad;   // the step has no gradient
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::OptionalCUDAGuard guard(x.device());
    const at::Device dev = x.device();
    x = x.contiguous(); state = state.contiguous(); w = w.contiguous();
    if (b.defined()) b = b.contiguous();
    y = empty(x.sizes(), x.scalar_type(), dev);
    if (after.defined()) check_written(op, "state_new", after, state, {&x, &w, &b});
    else after = empty(state.sizes(), x.scalar_type(), dev);
    if (x.numel() > 0)
      check(mlstm_b200_short_conv_step(ptr(x), ptr(state), ptr(w), ptr(b), y.mutable_data_ptr(), after.mutable_data_ptr(), (int)x.size(0), (int)x.size(1),
                                       (int)w.size(1), silu, dtype_code(x.scalar_type()), dtype_code(w.scalar_type()), current_stream(dev)),
            "mlstm_b200_short_conv_step");
  }
  return Py_BuildValue("(NN)", wrap(y), wrap(after));
  END_HANDLE_TH_ERRORS
}

// ---- selective state space scan -----------------------------------------------------------------------
struct SsmTensors {
  Tensor x, dt, a, b, c, skip, z, dt_bias, h0;   // skip, z, dt_bias, h0 may be undefined
  bool softplus;
};
void check_ssm(const char* op, const SsmTensors& t, bool one_token) {
  check_tensors(op, {&t.x, &t.dt, &t.a, &t.b, &t.c, &t.skip, &t.z, &t.dt_bias, &t.h0});
  for (const Tensor* p : {&t.x, &t.a, &t.skip, &t.dt_bias, &t.h0}) check_kernel_dtype(*p);
  const at::ScalarType dt = t.x.scalar_type();
  for (const Tensor* p : {&t.dt, &t.b, &t.c, &t.z})
    if (p->defined() && p->scalar_type() != dt) C10_THROW_ERROR(ValueError, c10::str(op, ": x, dt, b, c, z must share one dtype"));
  const int64_t lead = one_token ? 1 : 2;
  if (t.x.dim() != lead + 1) bad_shape(op, "x", t.x, one_token ? "(B, D)" : "(B, S, D)");
  check_int_sizes(op, t.x);
  if (t.dt.sizes() != t.x.sizes()) bad_shape(op, "dt", t.dt, "of x's shape");
  if (t.z.defined() && t.z.sizes() != t.x.sizes()) bad_shape(op, "z", t.z, "of x's shape");
  const int64_t D = t.x.size(-1);
  if (t.a.dim() != 2 || t.a.size(0) != D || t.a.size(1) < 1 || t.a.size(1) > 128) bad_shape(op, "a", t.a, "(D, N) with N from 1 to 128");
  const int64_t N = t.a.size(1);
  const bool groups = t.b.dim() == lead + 2;
  if ((!groups && t.b.dim() != lead + 1) || t.b.sizes().slice(0, lead) != t.x.sizes().slice(0, lead) || t.b.size(-1) != N ||
      (groups && (t.b.size(-2) < 1 || D % t.b.size(-2) != 0)))
    bad_shape(op, "b", t.b, one_token ? "(B, N) or (B, G, N) with D a multiple of G" : "(B, S, N) or (B, S, G, N) with D a multiple of G");
  if (t.c.sizes() != t.b.sizes()) bad_shape(op, "c", t.c, "of b's shape");
  for (const Tensor* p : {&t.skip, &t.dt_bias})
    if (p->defined() && (p->dim() != 1 || p->size(0) != D)) bad_shape(op, p == &t.skip ? "skip" : "dt_bias", *p, "(D,)");
  if (t.h0.defined() && t.h0.sizes() != at::IntArrayRef{t.x.size(0), D, N}) bad_shape(op, one_token ? "h" : "h_initial", t.h0, "(B, D, N)");
}
struct SsmSizes { int B, S, D, N, G; };
SsmSizes ssm_sizes(const SsmTensors& t) {
  return {(int)t.x.size(0), (int)t.x.size(1), (int)t.x.size(2), (int)t.a.size(1), t.b.dim() == 4 ? (int)t.b.size(2) : 1};
}
// the stride of the token axis; of a single token any number will do
long long token_stride(const Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; }
Tensor tokens_near(const Tensor& t) {   // the scan takes token strides below 2^29
  const Tensor d = last_dense(t);
  return !d.defined() || token_stride(d) < (1ll << 29) ? d : d.clone(at::MemoryFormat::Contiguous);
}
SsmTensors ssm_ready(const SsmTensors& t) {   // as the kernels read them
  return {tokens_near(t.x), tokens_near(t.dt), f32c(t.a), tokens_near(t.b), tokens_near(t.c), f32c(t.skip), tokens_near(t.z), f32c(t.dt_bias), f32c(t.h0), t.softplus};
}
std::array<long long, 12> ssm_strides(const SsmTensors& t) {
  const bool groups = t.b.dim() == 4;
  return {t.x.stride(0), token_stride(t.x), t.dt.stride(0), token_stride(t.dt), t.z.defined() ? t.z.stride(0) : 0, t.z.defined() ? token_stride(t.z) : 0,
          t.b.stride(0), token_stride(t.b), groups ? t.b.stride(2) : 0, t.c.stride(0), token_stride(t.c), groups ? t.c.stride(2) : 0};
}
struct Scanned { Tensor y, h_last, ckpt; };
Scanned ssm_forward(const SsmTensors& t_, bool want_last, bool keep) {
  const at::Device dev = t_.x.device();
  const SsmSizes q = ssm_sizes(t_);
  Scanned o;
  o.y = empty(t_.x.sizes(), t_.x.scalar_type(), dev);
  if (want_last) o.h_last = empty({q.B, q.D, q.N}, at::kFloat, dev);
  if (t_.x.numel() == 0) {   // no token: the last state is the first
    if (want_last) { if (t_.h0.defined()) o.h_last.copy_(t_.h0); else o.h_last.zero_(); }
    if (keep) o.ckpt = bytes(0, dev);
    return o;
  }
  const SsmTensors t = ssm_ready(t_);
  if (keep) o.ckpt = bytes(mlstm_b200_ssm_checkpoint_bytes(q.B, q.S, q.D, q.N), dev);
  const size_t need = mlstm_b200_ssm_workspace_bytes(q.B, q.S, q.D, q.N, q.G, 0);
  const Tensor ws = need > 0 ? bytes(need, dev) : Tensor();
  const auto st = ssm_strides(t);
  check(mlstm_b200_ssm_scan_fw(ptr(t.x), ptr(t.dt), fptr(t.a), ptr(t.b), ptr(t.c), fptr(t.skip), ptr(t.z), fptr(t.dt_bias), fptr(t.h0), st.data(),
                               o.y.mutable_data_ptr(), fout(o.h_last), fout(o.ckpt), fout(ws), need, q.B, q.S, q.D, q.N, q.G, t.softplus,
                               dtype_code(t.x.scalar_type()), current_stream(dev)),
        "mlstm_b200_ssm_scan_fw");
  return o;
}
struct ScanGrads { Tensor dx, ddt, da, db, dc, dskip, dz, ddt_bias, dh0; };
ScanGrads ssm_backward(const SsmTensors& t_, const Tensor& ckpt, const Tensor& dy_, const Tensor& dh_last_, bool want_skip, bool want_bias, bool want_h0) {
  const at::Device dev = t_.x.device();
  const at::ScalarType dt = t_.x.scalar_type();
  const SsmSizes q = ssm_sizes(t_);
  ScanGrads g;
  g.dx = empty(t_.x.sizes(), dt, dev);
  g.ddt = empty(t_.x.sizes(), dt, dev);
  if (t_.z.defined()) g.dz = empty(t_.x.sizes(), dt, dev);
  g.db = empty(t_.b.sizes(), dt, dev);
  g.dc = empty(t_.b.sizes(), dt, dev);
  g.da = empty({q.D, q.N}, at::kFloat, dev);
  if (want_skip) g.dskip = empty({q.D}, at::kFloat, dev);
  if (want_bias) g.ddt_bias = empty({q.D}, at::kFloat, dev);
  if (want_h0) g.dh0 = empty({q.B, q.D, q.N}, at::kFloat, dev);
  if (t_.x.numel() == 0) {
    for (Tensor* p : {&g.db, &g.dc, &g.da, &g.dskip, &g.ddt_bias})
      if (p->defined()) p->zero_();
    if (want_h0) { if (dh_last_.defined()) g.dh0.copy_(dh_last_); else g.dh0.zero_(); }
  } else {
    const SsmTensors t = ssm_ready(t_);
    const Tensor dy = dy_.defined() ? tokens_near(to_dtype(dy_, dt)) : zeros(t_.x.sizes(), dt, dev);
    const Tensor dhl = f32c(dh_last_);
    const long long gs[2] = {dy.stride(0), token_stride(dy)};
    const size_t need = mlstm_b200_ssm_workspace_bytes(q.B, q.S, q.D, q.N, q.G, 1);
    const Tensor ws = bytes(need, dev);
    const auto st = ssm_strides(t);
    auto out = [](const Tensor& p) { return p.defined() ? p.mutable_data_ptr() : nullptr; };
    check(mlstm_b200_ssm_scan_bw(ptr(t.x), ptr(t.dt), fptr(t.a), ptr(t.b), ptr(t.c), fptr(t.skip), ptr(t.z), fptr(t.dt_bias), st.data(), fptr(ckpt),
                                 ptr(dy), gs, fptr(dhl), out(g.dx), out(g.ddt), fout(g.da), out(g.db), out(g.dc), fout(g.dskip), out(g.dz),
                                 fout(g.ddt_bias), fout(g.dh0), fout(ws), need, q.B, q.S, q.D, q.N, q.G, t.softplus, dtype_code(dt), current_stream(dev)),
          "mlstm_b200_ssm_scan_bw");
  }
  g.da = to_dtype(g.da, t_.a.scalar_type());
  if (want_skip) g.dskip = to_dtype(g.dskip, t_.skip.scalar_type());
  if (want_bias) g.ddt_bias = to_dtype(g.ddt_bias, t_.dt_bias.scalar_type());
  if (want_h0) g.dh0 = to_dtype(g.dh0, t_.h0.scalar_type());
  return g;
}

const char* const kSsm = "ssm_scan__b200";
class ScanFn : public torch::autograd::Function<ScanFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const OptT& skip,
                               const OptT& z, const OptT& dt_bias, const OptT& h0, bool softplus, bool want_last) {
    const SsmTensors t{x, dt, a, b, c, skip.value_or(Tensor()), z.value_or(Tensor()), dt_bias.value_or(Tensor()), h0.value_or(Tensor()), softplus};
    Scanned o = ssm_forward(t, want_last, true);
    ctx->save_for_backward({t.x, t.dt, t.a, t.b, t.c, t.skip, t.z, t.dt_bias, t.h0, o.ckpt});
    ctx->set_materialize_grads(false);
    ctx->saved_data["cfg"] = std::vector<int64_t>{softplus, t.skip.defined() && t.skip.requires_grad(), t.dt_bias.defined() && t.dt_bias.requires_grad(),
                                                  t.h0.defined() && t.h0.requires_grad()};
    if (want_last) return {o.y, o.h_last};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative(kSsm);
    const auto s = ctx->get_saved_variables();
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    c10::cuda::OptionalCUDAGuard guard(s[0].device());
    const SsmTensors t{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], cfg[0] != 0};
    const ScanGrads g = ssm_backward(t, s[9], grads[0], grads.size() > 1 ? grads[1] : Tensor(), cfg[1] != 0, cfg[2] != 0, cfg[3] != 0);
    return {g.dx, g.ddt, g.da, g.db, g.dc, g.dskip, g.dz, g.ddt_bias, g.dh0, Tensor(), Tensor()};
  }
};

// x, dt, a, b, c, skip, z, dt_bias, h_initial, softplus
SsmTensors ssm_args(PyObject* const* a, const char* h_name, bool h_needed) {
  return {need(a[0], "x"), need(a[1], "dt"), need(a[2], "a"), need(a[3], "b"), need(a[4], "c"), arg(a[5], "skip"), arg(a[6], "z"), arg(a[7], "dt_bias"),
          h_needed ? need(a[8], h_name) : arg(a[8], h_name), bool_arg(a[9])};
}
// ssm_scan(..., return_last) -> (y, h_last or None)
PyObject* py_ssm_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 11);
  const SsmTensors t = ssm_args(a, "h_initial", false);
  const bool want_last = bool_arg(a[10]);
  check_ssm(kSsm, t, false);
  Tensor y, last;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::OptionalCUDAGuard guard(t.x.device());
    if (wants_grad({&t.x, &t.dt, &t.a, &t.b, &t.c, &t.skip, &t.z, &t.dt_bias, &t.h0})) {
      const auto o = ScanFn::apply(t.x, t.dt, t.a, t.b, t.c, given(t.skip), given(t.z), given(t.dt_bias), given(t.h0), t.softplus, want_last);
      y = o[0];
      if (want_last) last = o[1];
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      const Scanned o = ssm_forward(t, want_last, false);
      y = o.y; last = o.h_last;
    }
  }
  return Py_BuildValue("(NN)", wrap(y), wrap(last));
  END_HANDLE_TH_ERRORS
}
// ssm_scan_fw(..., keep, return_last) -> (y, h_last or None, checkpoints or None)
PyObject* py_ssm_scan_fw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 12);
  const SsmTensors t = ssm_args(a, "h_initial", false);
  check_ssm(kSsm, t, false);
  c10::cuda::OptionalCUDAGuard guard(t.x.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Scanned o = ssm_forward(t, bool_arg(a[11]), bool_arg(a[10]));
  return Py_BuildValue("(NNN)", wrap(o.y), wrap(o.h_last), wrap(o.ckpt));
  END_HANDLE_TH_ERRORS
}
// ssm_scan_bw(..., checkpoints, dy, dh_last) -> (dx, ddt, da, db, dc, dskip, dz, ddt_bias, dh_initial), None for what was not given
PyObject* py_ssm_scan_bw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 13);
  const SsmTensors t = ssm_args(a, "h_initial", false);
  const Tensor ckpt = need(a[10], "checkpoints"), dy = arg(a[11], "dy"), dhl = arg(a[12], "dh_last");
  check_ssm(kSsm, t, false);
  check_tensors(kSsm, {&t.x, &ckpt, &dy, &dhl});
  check_size(kSsm, "dy", dy, t.x.sizes());
  check_size(kSsm, "dh_last", dhl, {t.x.size(0), t.x.size(2), t.a.size(1)});
  const SsmSizes q = ssm_sizes(t);
  if (!ckpt.is_contiguous() || ckpt.nbytes() < mlstm_b200_ssm_checkpoint_bytes(q.B, q.S, q.D, q.N))
    C10_THROW_ERROR(ValueError, "ssm_scan__b200: checkpoints of another call");
  c10::cuda::OptionalCUDAGuard guard(t.x.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const ScanGrads g = ssm_backward(t, ckpt, dy, dhl, t.skip.defined(), t.dt_bias.defined(), t.h0.defined());
  return Py_BuildValue("(NNNNNNNNN)", wrap(g.dx), wrap(g.ddt), wrap(g.da), wrap(g.db), wrap(g.dc), wrap(g.dskip), wrap(g.dz), wrap(g.ddt_bias), wrap(g.dh0));
  END_HANDLE_TH_ERRORS
}
// ssm_step(x, dt, a, b, c, skip, z, dt_bias, h, softplus, h_new) -> (y, h_new)
PyObject* py_ssm_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 11);
  const char* const op = "ssm_step__b200";
  SsmTensors t = ssm_args(a, "h", true);
  Tensor h_new = arg(a[10], "h_new");
  check_ssm(op, t, true);
  check_tensors(op, {&t.x, &h_new});
  if (h_new.defined() && (h_new.sizes() != t.h0.sizes() || h_new.scalar_type() != at::kFloat || !h_new.is_contiguous()))
    C10_THROW_ERROR(ValueError, "ssm_step__b200: h_new must be a contiguous f32 (B, D, N) tensor");
  at::NoGradGuard no_grad;   // the step has no gradient
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const at::Device dev = t.x.device();
    c10::cuda::OptionalCUDAGuard guard(dev);
    auto c = [](const Tensor& p) { return p.defined() ? p.contiguous() : p; };
    t = SsmTensors{c(t.x), c(t.dt), f32c(t.a), c(t.b), c(t.c), f32c(t.skip), c(t.z), f32c(t.dt_bias), f32c(t.h0), t.softplus};
    y = empty(t.x.sizes(), t.x.scalar_type(), dev);
    if (h_new.defined()) check_written(op, "h_new", h_new, t.h0, {&t.x, &t.dt, &t.a, &t.b, &t.c, &t.skip, &t.z, &t.dt_bias});
    else h_new = empty(t.h0.sizes(), at::kFloat, dev);
    if (t.x.numel() > 0)
      check(mlstm_b200_ssm_step(ptr(t.x), ptr(t.dt), fptr(t.a), ptr(t.b), ptr(t.c), fptr(t.skip), ptr(t.z), fptr(t.dt_bias), fptr(t.h0),
                                y.mutable_data_ptr(), fout(h_new), (int)t.x.size(0), (int)t.x.size(1), (int)t.a.size(1),
                                t.b.dim() == 3 ? (int)t.b.size(1) : 1, t.softplus, dtype_code(t.x.scalar_type()), current_stream(dev)),
            "mlstm_b200_ssm_step");
  }
  return Py_BuildValue("(NN)", wrap(y), wrap(h_new));
  END_HANDLE_TH_ERRORS
}

}  // namespace

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef mlstm_host::kLayerMethods[] = {
    METHOD(layer_norm), METHOD(layer_norm_fw), METHOD(layer_norm_bw), METHOD(short_conv), METHOD(short_conv_bw), METHOD(short_conv_step),
    METHOD(ssm_scan), METHOD(ssm_scan_fw), METHOD(ssm_scan_bw), METHOD(ssm_step), {nullptr, nullptr, 0, nullptr}};

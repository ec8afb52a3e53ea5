// The host side of the gated linear recurrence and of dropout, in the manner of host_layers.cpp.
#include "host_layers.h"

namespace {

using namespace mlstm_host;

// ---- gated linear recurrence --------------------------------------------------------------------------
struct GatedTensors {
  Tensor x, f, i, z, rate, h0;   // i, z, rate, h0 may be undefined
  int scale;
};
void check_gated(const char* op, const GatedTensors& t, bool one_token) {
  check_tensors(op, {&t.x, &t.f, &t.i, &t.z, &t.rate, &t.h0});
  for (const Tensor* p : {&t.x, &t.rate, &t.h0}) check_kernel_dtype(*p);
  if (t.x.dim() != (one_token ? 2 : 3)) bad_shape(op, "x", t.x, one_token ? "(B, D)" : "(B, S, D)");
  check_int_sizes(op, t.x);
  struct { const char* name; const Tensor& t; } like[] = {{"f", t.f}, {"i", t.i}, {"z", t.z}};
  for (const auto& p : like) {
    if (!p.t.defined()) continue;
    if (p.t.scalar_type() != t.x.scalar_type()) C10_THROW_ERROR(ValueError, c10::str(op, ": x, f, i, z must share one dtype"));
    if (p.t.sizes() != t.x.sizes()) bad_shape(op, p.name, p.t, "of x's shape");
  }
  if (t.rate.defined() && (t.rate.dim() != 1 || t.rate.size(0) != t.x.size(-1))) bad_shape(op, "rate", t.rate, "(D,)");
  if (t.h0.defined() && t.h0.sizes() != at::IntArrayRef{t.x.size(0), t.x.size(-1)}) bad_shape(op, one_token ? "h" : "h_initial", t.h0, "(B, D)");
}
GatedTensors gated_ready(const GatedTensors& t) {   // as the kernels read them
  return {last_dense(t.x), last_dense(t.f), last_dense(t.i), last_dense(t.z), f32c(t.rate), f32c(t.h0), t.scale};
}
std::array<long long, 8> gated_strides(const GatedTensors& t) {
  std::array<long long, 8> s{};
  const Tensor* const ts[4] = {&t.x, &t.f, &t.i, &t.z};
  for (int k = 0; k < 4; ++k)
    if (ts[k]->defined()) s[2 * k] = ts[k]->stride(0), s[2 * k + 1] = token_stride(*ts[k]);
  return s;
}
struct Gated { Tensor y, h_last, ckpt; };
Gated gated_forward(const GatedTensors& t_, bool want_last, bool keep) {
  const at::Device dev = t_.x.device();
  const int B = (int)t_.x.size(0), S = (int)t_.x.size(1), D = (int)t_.x.size(2);
  Gated o;
  o.y = empty(t_.x.sizes(), t_.x.scalar_type(), dev);
  if (want_last) o.h_last = empty({B, D}, at::kFloat, dev);
  if (t_.x.numel() == 0) {   // no token: the last state is the first
    if (want_last) { if (t_.h0.defined()) o.h_last.copy_(t_.h0); else o.h_last.zero_(); }
    if (keep) o.ckpt = bytes(0, dev);
    return o;
  }
  const GatedTensors t = gated_ready(t_);
  if (keep) o.ckpt = bytes(mlstm_b200_gated_checkpoint_bytes(B, S, D), dev);
  const size_t need = mlstm_b200_gated_workspace_bytes(B, S, D, 0);
  const Tensor ws = need > 0 ? bytes(need, dev) : Tensor();
  const auto st = gated_strides(t);
  check(mlstm_b200_gated_scan_fw(ptr(t.x), ptr(t.f), ptr(t.i), ptr(t.z), fptr(t.rate), fptr(t.h0), st.data(), o.y.mutable_data_ptr(), fout(o.h_last),
                                 fout(o.ckpt), fout(ws), need, B, S, D, t.scale, dtype_code(t.x.scalar_type()), current_stream(dev)),
        "mlstm_b200_gated_scan_fw");
  return o;
}
struct GatedGrads { Tensor dx, df, di, dz, drate, dh0; };
// h0: the initial state's type, where its gradient is wanted (its values are not needed: the checkpoints have them)
GatedGrads gated_backward(const GatedTensors& t_, const Tensor& ckpt, const Tensor& dy_, const Tensor& dh_last_, bool want_rate,
                          std::optional<at::ScalarType> h0) {
  const at::Device dev = t_.x.device();
  const at::ScalarType dt = t_.x.scalar_type();
  const int B = (int)t_.x.size(0), S = (int)t_.x.size(1), D = (int)t_.x.size(2);
  GatedGrads g;
  g.dx = empty(t_.x.sizes(), dt, dev);
  g.df = empty(t_.x.sizes(), dt, dev);
  if (t_.i.defined()) g.di = empty(t_.x.sizes(), dt, dev);
  if (t_.z.defined()) g.dz = empty(t_.x.sizes(), dt, dev);
  if (want_rate) g.drate = empty({D}, at::kFloat, dev);
  if (h0) g.dh0 = empty({B, D}, at::kFloat, dev);
  if (t_.x.numel() == 0) {
    if (want_rate) g.drate.zero_();
    if (h0) { if (dh_last_.defined()) g.dh0.copy_(dh_last_); else g.dh0.zero_(); }
  } else {
    const GatedTensors t = gated_ready({t_.x, t_.f, t_.i, t_.z, t_.rate, Tensor(), t_.scale});
    const Tensor dy = dy_.defined() ? last_dense(to_dtype(dy_, dt)) : zeros(t_.x.sizes(), dt, dev);
    const Tensor dhl = f32c(dh_last_);
    const long long gs[2] = {dy.stride(0), token_stride(dy)};
    const size_t need = mlstm_b200_gated_workspace_bytes(B, S, D, 1);
    const Tensor ws = bytes(need, dev);
    const auto st = gated_strides(t);
    auto out = [](const Tensor& p) { return p.defined() ? p.mutable_data_ptr() : nullptr; };
    check(mlstm_b200_gated_scan_bw(ptr(t.x), ptr(t.f), ptr(t.i), ptr(t.z), fptr(t.rate), st.data(), fptr(ckpt), ptr(dy), gs, fptr(dhl), out(g.dx),
                                   out(g.df), out(g.di), out(g.dz), fout(g.drate), fout(g.dh0), fout(ws), need, B, S, D, t.scale, dtype_code(dt),
                                   current_stream(dev)),
          "mlstm_b200_gated_scan_bw");
  }
  if (want_rate) g.drate = to_dtype(g.drate, t_.rate.scalar_type());
  if (h0) g.dh0 = to_dtype(g.dh0, *h0);
  return g;
}

const char* const kGated = "gated_scan__b200";
class GatedFn : public torch::autograd::Function<GatedFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& f, const OptT& i, const OptT& z, const OptT& rate, const OptT& h0,
                               int64_t scale, bool want_last) {
    const GatedTensors t{x, f, i.value_or(Tensor()), z.value_or(Tensor()), rate.value_or(Tensor()), h0.value_or(Tensor()), (int)scale};
    Gated o = gated_forward(t, want_last, true);
    ctx->save_for_backward({t.x, t.f, t.i, t.z, t.rate, o.ckpt});   // (not h0: its buffer may hold the next state before the backward runs)
    ctx->set_materialize_grads(false);
    const bool want_h0 = t.h0.defined() && t.h0.requires_grad();
    ctx->saved_data["cfg"] = std::vector<int64_t>{scale, t.rate.defined() && t.rate.requires_grad(), want_h0, want_h0 ? (int64_t)t.h0.scalar_type() : 0};
    if (want_last) return {o.y, o.h_last};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative(kGated);
    const auto s = ctx->get_saved_variables();
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    c10::cuda::OptionalCUDAGuard guard(s[0].device());
    const GatedTensors t{s[0], s[1], s[2], s[3], s[4], Tensor(), (int)cfg[0]};
    const GatedGrads g = gated_backward(t, s[5], grads[0], grads.size() > 1 ? grads[1] : Tensor(), cfg[1] != 0,
                                        cfg[2] != 0 ? std::optional((at::ScalarType)cfg[3]) : std::nullopt);
    return {g.dx, g.df, g.di, g.dz, g.drate, g.dh0, Tensor(), Tensor()};
  }
};

int scale_arg(PyObject* o) {
  const long s = long_arg(o);
  if (s < 0 || s > 2) C10_THROW_ERROR(ValueError, c10::str("Unsupported input scale ", s, ": 0, 1 or 2."));
  return (int)s;
}
// x, f, i, z, rate, h_initial, scale
GatedTensors gated_args(PyObject* const* a, const char* h_name, bool h_needed) {
  return {need(a[0], "x"), need(a[1], "f"), arg(a[2], "i"), arg(a[3], "z"), arg(a[4], "rate"), h_needed ? need(a[5], h_name) : arg(a[5], h_name),
          scale_arg(a[6])};
}
// gated_scan(..., return_last) -> (y, h_last or None)
PyObject* py_gated_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 8);
  const GatedTensors t = gated_args(a, "h_initial", false);
  const bool want_last = bool_arg(a[7]);
  check_gated(kGated, t, false);
  Tensor y, last;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::OptionalCUDAGuard guard(t.x.device());
    if (wants_grad({&t.x, &t.f, &t.i, &t.z, &t.rate, &t.h0})) {
      const auto o = GatedFn::apply(t.x, t.f, given(t.i), given(t.z), given(t.rate), given(t.h0), (int64_t)t.scale, want_last);
      y = o[0];
      if (want_last) last = o[1];
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      const Gated o = gated_forward(t, want_last, false);
      y = o.y; last = o.h_last;
    }
  }
  return Py_BuildValue("(NN)", wrap(y), wrap(last));
  END_HANDLE_TH_ERRORS
}
// gated_scan_fw(..., keep, return_last) -> (y, h_last or None, checkpoints or None)
PyObject* py_gated_scan_fw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 9);
  const GatedTensors t = gated_args(a, "h_initial", false);
  check_gated(kGated, t, false);
  c10::cuda::OptionalCUDAGuard guard(t.x.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Gated o = gated_forward(t, bool_arg(a[8]), bool_arg(a[7]));
  return Py_BuildValue("(NNN)", wrap(o.y), wrap(o.h_last), wrap(o.ckpt));
  END_HANDLE_TH_ERRORS
}
// gated_scan_bw(..., checkpoints, dy, dh_last) -> (dx, df, di, dz, drate, dh_initial), None for what was not given; h_initial's values are not read
PyObject* py_gated_scan_bw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 10);
  const GatedTensors t = gated_args(a, "h_initial", false);
  const Tensor ckpt = need(a[7], "checkpoints"), dy = arg(a[8], "dy"), dhl = arg(a[9], "dh_last");
  check_gated(kGated, t, false);
  check_tensors(kGated, {&t.x, &ckpt, &dy, &dhl});
  check_size(kGated, "dy", dy, t.x.sizes());
  check_size(kGated, "dh_last", dhl, {t.x.size(0), t.x.size(2)});
  if (!ckpt.is_contiguous() || ckpt.nbytes() < mlstm_b200_gated_checkpoint_bytes((int)t.x.size(0), (int)t.x.size(1), (int)t.x.size(2)))
    C10_THROW_ERROR(ValueError, "gated_scan__b200: checkpoints of another call");
  c10::cuda::OptionalCUDAGuard guard(t.x.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const GatedGrads g = gated_backward(t, ckpt, dy, dhl, t.rate.defined(), t.h0.defined() ? std::optional(t.h0.scalar_type()) : std::nullopt);
  return Py_BuildValue("(NNNNNN)", wrap(g.dx), wrap(g.df), wrap(g.di), wrap(g.dz), wrap(g.drate), wrap(g.dh0));
  END_HANDLE_TH_ERRORS
}
// gated_step(x, f, i, z, rate, h, scale, h_new) -> (y, h_new)
PyObject* py_gated_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 8);
  const char* const op = "gated_step__b200";
  GatedTensors t = gated_args(a, "h", true);
  Tensor h_new = arg(a[7], "h_new");
  check_gated(op, t, true);
  check_tensors(op, {&t.x, &h_new});
  if (h_new.defined() && (h_new.sizes() != t.h0.sizes() || h_new.scalar_type() != at::kFloat || !h_new.is_contiguous()))
    C10_THROW_ERROR(ValueError, "gated_step__b200: h_new must be a contiguous f32 (B, D) tensor");
  at::NoGradGuard no_grad;   // the step has no gradient
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const at::Device dev = t.x.device();
    c10::cuda::OptionalCUDAGuard guard(dev);
    auto c = [](const Tensor& p) { return p.defined() ? p.contiguous() : p; };
    t = GatedTensors{c(t.x), c(t.f), c(t.i), c(t.z), f32c(t.rate), f32c(t.h0), t.scale};
    y = empty(t.x.sizes(), t.x.scalar_type(), dev);
    if (h_new.defined()) check_written(op, "h_new", h_new, t.h0, {&t.x, &t.f, &t.i, &t.z, &t.rate});
    else h_new = empty(t.h0.sizes(), at::kFloat, dev);
    if (t.x.numel() > 0)
      check(mlstm_b200_gated_step(ptr(t.x), ptr(t.f), ptr(t.i), ptr(t.z), fptr(t.rate), fptr(t.h0), y.mutable_data_ptr(), fout(h_new), (int)t.x.size(0),
                                  (int)t.x.size(1), t.scale, dtype_code(t.x.scalar_type()), current_stream(dev)),
            "mlstm_b200_gated_step");
  }
  return Py_BuildValue("(NN)", wrap(y), wrap(h_new));
  END_HANDLE_TH_ERRORS
}

// ---- dropout ------------------------------------------------------------------------------------------
const char* const kDropout = "dropout__b200";
struct Seed {
  Tensor device;     // one 64-bit number on the GPU, or undefined
  int64_t value;
};
void check_dropout(const Tensor& x, const Tensor& residual, const Seed& seed, double p, int64_t offset) {
  check_tensors(kDropout, {&x, &residual, &seed.device});
  check_kernel_dtype(x);
  if (residual.defined()) {
    if (residual.sizes() != x.sizes()) bad_shape(kDropout, "residual", residual, "of x's shape");
    if (residual.scalar_type() != x.scalar_type() && residual.scalar_type() != at::kFloat)
      C10_THROW_ERROR(ValueError, "dropout__b200: residual must have x's dtype or f32");
  }
  if (!(p >= 0 && p <= 1)) C10_THROW_ERROR(ValueError, c10::str("dropout__b200: p must be from 0 to 1, got ", p));
  if (seed.device.defined() && (seed.device.scalar_type() != at::kLong || seed.device.numel() != 1))
    C10_THROW_ERROR(ValueError, "dropout__b200: seed must be a number, or an int64 tensor with one element");
  if (seed.value < 0 || offset < 0) C10_THROW_ERROR(ValueError, "dropout__b200: seed and offset must not be negative");
}
// The axes of up to three tensors of one shape as four, the last of them of stride one; false where their strides do not allow that.
struct Axes {
  long long n[4] = {1, 1, 1, 1}, s[3][3] = {};
};
bool merge_axes(at::IntArrayRef sizes, std::initializer_list<const Tensor*> ts, Axes& a) {
  int k = 3;   // the axis that grows
  long long last[3] = {1, 1, 1};
  for (int64_t d = (int64_t)sizes.size() - 1; d >= 0; --d) {
    if (sizes[d] == 1) continue;
    bool joins = true, any = a.n[k] > 1 || k == 3;
    int j = 0;
    for (const Tensor* t : ts) {
      if (t->defined() && t->stride(d) != last[j] * a.n[k]) joins = false;
      ++j;
    }
    if (!joins && any) {
      if (k == 0) return false;
      --k;
      j = 0;
      for (const Tensor* t : ts) {
        if (t->defined()) a.s[j][k] = last[j] = t->stride(d);
        ++j;
      }
    }
    a.n[k] *= sizes[d];
  }
  return true;
}
Tensor dropout_apply(const Tensor& x_, const Tensor& residual_, const Seed& seed, double p, int64_t offset, const Tensor& out_) {
  if (x_.numel() == 0) return out_;
  Tensor x = x_.dim() > 0 ? last_dense(x_) : x_, residual = residual_.defined() && x.dim() > 0 ? last_dense(residual_) : residual_, out = out_;
  Axes a;
  if (!merge_axes(x.sizes(), {&x, &residual, &out}, a)) {
    x = x.contiguous();
    if (residual.defined()) residual = residual.contiguous();
    a = Axes();
    if (!merge_axes(x.sizes(), {&x, &residual, &out}, a)) {   // (the output lies in an order of its own)
      out = empty(x.sizes(), out.scalar_type(), x.device());
      a = Axes();
      merge_axes(x.sizes(), {&x, &residual, &out}, a);
    }
  }
  check(mlstm_b200_dropout(ptr(x), a.s[0], ptr(residual), a.s[1], out.mutable_data_ptr(), a.s[2], a.n, p, (unsigned long long)seed.value, ptr(seed.device),
                           (unsigned long long)offset, dtype_code(x.scalar_type()), dtype_code(out.scalar_type()), current_stream(x.device())),
        "mlstm_b200_dropout");
  return out;
}
Tensor dropout_forward(const Tensor& x, const Tensor& residual, const Seed& seed, double p, int64_t offset) {
  return dropout_apply(x, residual, seed, p, offset, empty(x.sizes(), residual.defined() ? residual.scalar_type() : x.scalar_type(), x.device()));
}

class DropoutFn : public torch::autograd::Function<DropoutFn> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptT& residual_opt, const OptT& seed_opt, int64_t seed_value, double p, int64_t offset) {
    const Tensor residual = residual_opt.value_or(Tensor());
    const Seed seed{seed_opt.value_or(Tensor()), seed_value};
    ctx->save_for_backward({seed.device});
    ctx->saved_data["cfg"] = std::vector<int64_t>{seed_value, offset, (int64_t)x.scalar_type(), x.requires_grad(), residual.defined() && residual.requires_grad()};
    ctx->saved_data["p"] = p;
    // the gradient lies as x does, where x covers its memory once
    ctx->saved_data["strides"] = x.is_non_overlapping_and_dense() ? x.strides().vec() : std::vector<int64_t>{};
    return dropout_forward(x, residual, seed, p, offset);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative(kDropout);
    const auto saved = ctx->get_saved_variables();
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    const auto strides = ctx->saved_data["strides"].toIntVector();
    const Tensor& dy = grads[0];
    c10::cuda::OptionalCUDAGuard guard(dy.device());
    Tensor dx;
    if (cfg[3] != 0) {
      const at::ScalarType dt = (at::ScalarType)cfg[2];
      dx = (int64_t)strides.size() == dy.dim() ? at::empty_strided(dy.sizes(), strides, dy.options().dtype(dt)) : empty(dy.sizes(), dt, dy.device());
      dx = dropout_apply(dy, Tensor(), Seed{saved[0], cfg[0]}, ctx->saved_data["p"].toDouble(), cfg[1], dx);
    }
    return {dx, cfg[4] != 0 ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// x, residual, seed (a tensor or None), seed (a number), p, offset
struct DropoutArgs { Tensor x, residual; Seed seed; double p; int64_t offset; };
DropoutArgs dropout_args(PyObject* const* a) {
  DropoutArgs d{need(a[0], "x"), arg(a[1], "residual"), Seed{arg(a[2], "seed"), long_arg(a[3])}, double_arg(a[4]), long_arg(a[5])};
  check_dropout(d.x, d.residual, d.seed, d.p, d.offset);
  return d;
}
PyObject* py_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 6);
  const DropoutArgs d = dropout_args(a);
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::OptionalCUDAGuard guard(d.x.device());
    if (wants_grad({&d.x, &d.residual})) {
      y = DropoutFn::apply(d.x, given(d.residual), given(d.seed.device), d.seed.value, d.p, d.offset);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      y = dropout_forward(d.x, d.residual, d.seed, d.p, d.offset);
    }
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}
// dropout_bw(dy, seed, seed, p, offset, dtype) -> dx, contiguous
PyObject* py_dropout_bw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  nargs_are(n, 6);
  const Tensor dy = need(a[0], "dy");
  const Seed seed{arg(a[1], "seed"), long_arg(a[2])};
  const double p = double_arg(a[3]);
  const int64_t offset = long_arg(a[4]);
  const at::ScalarType dt = dtype_arg(a[5]);
  check_dropout(dy, Tensor(), seed, p, offset);
  if (dtype_code(dt) < 0 || (dt != dy.scalar_type() && dy.scalar_type() != at::kFloat)) C10_THROW_ERROR(ValueError, "dropout__b200: dy must have x's dtype or f32");
  c10::cuda::OptionalCUDAGuard guard(dy.device());
  at::AutoDispatchBelowADInplaceOrView below;
  return wrap(dropout_apply(dy, Tensor(), seed, p, offset, empty(dy.sizes(), dt, dy.device())));
  END_HANDLE_TH_ERRORS
}

}  // namespace

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef mlstm_host::kGatedMethods[] = {METHOD(gated_scan), METHOD(gated_scan_fw), METHOD(gated_scan_bw), METHOD(gated_step), METHOD(dropout),
                                           METHOD(dropout_bw), {nullptr, nullptr, 0, nullptr}};

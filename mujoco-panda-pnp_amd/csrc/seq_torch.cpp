// seq_torch.cpp — the sequence operators' front end for torch: argument checks, outputs and workspaces
// from torch's allocator, autograd nodes, and the calls into libpnp's C entry points (include/pnp.h).
// pnp_amd/seqops.py documents the operators and is how they are reached.
//
// It is native because a call's host time is what small batches pay: the same front end in Python over
// ctypes took 17 us for an 8-bit product and 180 us for a norm with its gradient.
//
// The entry points come by address from the library that the package has loaded (`bind`), so that the
// process holds one libpnp.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <string>
#include <vector>

#include "../../include/pnp.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> MaybeTensor;

struct Api {
  const char* (*last_error)();
#define ENTRY(f) decltype(&pnp_##f) f
  ENTRY(rms_norm); ENTRY(rms_norm_bwd); ENTRY(rms_norm_bwd_workspace); ENTRY(quantize_rows); ENTRY(matmul_i8);
  ENTRY(causal_conv); ENTRY(causal_conv_bwd); ENTRY(causal_conv_bwd_workspace); ENTRY(causal_conv_step);
  ENTRY(selective_scan); ENTRY(selective_scan_bwd); ENTRY(selective_scan_step);
  ENTRY(scan_ckpt_floats); ENTRY(scan_workspace); ENTRY(scan_bwd_workspace);
#undef ENTRY
} api;

void bind(const std::map<std::string, uintptr_t>& at) {
  api.last_error = reinterpret_cast<decltype(api.last_error)>(at.at("pnp_last_error"));
#define ENTRY(f) api.f = reinterpret_cast<decltype(api.f)>(at.at("pnp_" #f))
  ENTRY(rms_norm); ENTRY(rms_norm_bwd); ENTRY(rms_norm_bwd_workspace); ENTRY(quantize_rows); ENTRY(matmul_i8);
  ENTRY(causal_conv); ENTRY(causal_conv_bwd); ENTRY(causal_conv_bwd_workspace); ENTRY(causal_conv_step);
  ENTRY(selective_scan); ENTRY(selective_scan_bwd); ENTRY(selective_scan_step);
  ENTRY(scan_ckpt_floats); ENTRY(scan_workspace); ENTRY(scan_bwd_workspace);
#undef ENTRY
}

// what an entry point refused or HIP reported (pnp_amd._lib.PnpError in Python)
struct Failed : std::runtime_error { using std::runtime_error::runtime_error; };
[[noreturn]] void fail(const char* fn, int64_t rc) {
  throw Failed(std::string(fn) + " failed (" + std::to_string(rc) + "): " + api.last_error());
}

// ---- checks
int code_of(ScalarType t) {
  switch (t) {
    case at::kFloat: return PNP_F32;
    case at::kBFloat16: return PNP_BF16;
    case at::kHalf: return PNP_F16;
    default: return -1;
  }
}

void on_device(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a device tensor (got ", t.device(), "); the sequence operators have no CPU path");
}
void same_device(const Tensor& t, const char* name, const Tensor& like) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", the other tensors on ", like.device());
}
// an activation: on a device, of a known type; of `like`'s type and device where given
void activation(const Tensor& t, const char* name, const Tensor* like = nullptr) {
  on_device(t, name);
  TORCH_CHECK_TYPE(code_of(t.scalar_type()) >= 0, name, ": dtype ", t.scalar_type(), ", expected float32, bfloat16 or float16");
  if (!like) return;
  TORCH_CHECK_TYPE(t.scalar_type() == like->scalar_type(), name, ": dtype ", t.scalar_type(), ", expected ", like->scalar_type(),
                   " as the other activations");
  same_device(t, name, *like);
}
void dims(const Tensor& t, const char* name, int64_t n) {
  TORCH_CHECK_VALUE(t.dim() == n, name, ": shape ", t.sizes(), ", expected ", n, " dimensions");
}
// what the entry points hold in 32 bits
void channels(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) > 0 && t.size(-1) <= (1 << 24), name, ": shape ", t.sizes(),
                    ", expected a last dimension from 1 to ", 1 << 24);
}
void shaped(const Tensor& t, const char* name, at::IntArrayRef want) {
  TORCH_CHECK_VALUE(t.sizes() == want, name, ": shape ", t.sizes(), ", expected ", want);
}
// values as they lie in memory (not a view that stands for their negative)
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor whole(const Tensor& t) { return plain(t).contiguous(); }
// a parameter, used in fp32 and contiguous (a differentiable cast: its gradient comes back in its own type)
Tensor parameter(const MaybeTensor& t, const char* name, at::IntArrayRef want, const Tensor& like) {
  if (!t || !t->defined()) return Tensor();
  TORCH_CHECK_TYPE(at::isFloatingType(t->scalar_type()), name, " must be a floating tensor");
  same_device(*t, name, like);
  shaped(*t, name, want);
  return whole(t->to(at::kFloat));
}
Tensor required(const MaybeTensor& t, const char* name, at::IntArrayRef want, const Tensor& like) {
  TORCH_CHECK_TYPE(t && t->defined(), name, " must be a floating tensor");
  return parameter(t, name, want, like);
}
// starts, reset: bytes or truth values
Tensor marks(const MaybeTensor& t, const char* name, at::IntArrayRef want, const Tensor& like) {
  if (!t || !t->defined()) return Tensor();
  TORCH_CHECK_TYPE(t->scalar_type() == at::kByte || t->scalar_type() == at::kBool, name, " must be a uint8 or bool tensor");
  same_device(*t, name, like);
  shaped(*t, name, want);
  return t->contiguous();
}
// a contiguous last dimension
Tensor lines(const Tensor& t_) {
  const Tensor t = plain(t_);
  return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
// a state that a call advances in place, which autograd has to hear of as of torch's own in-place calls: a graph
// that holds the state as it was refuses to go back through it
void in_place(const Tensor& state) {
  TORCH_CHECK_VALUE(state.is_contiguous() && !state.is_neg(), "state must be contiguous: it is advanced in place");
}
void advanced(const Tensor& state) {
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
}

// an input of a call that advances `state` in place, copied first where the two share memory: some of the call's
// workgroups may read it after others have written
Tensor apart(const Tensor& t, const Tensor& state) {
  if (!t.defined() || !t.numel() || !state.numel() || !t.is_alias_of(state)) return t;
  const auto end = [](const Tensor& v) {
    int64_t last = 0;
    for (int64_t i = 0; i < v.dim(); i++) last += (v.size(i) - 1) * v.stride(i);
    return (const char*)v.const_data_ptr() + (last + 1) * (int64_t)v.element_size();
  };
  const bool meet = (const char*)t.const_data_ptr() < end(state) && (const char*)state.const_data_ptr() < end(t);
  return meet ? t.clone(at::MemoryFormat::Contiguous) : t;
}

// autograd nodes take what may be missing as an optional (an undefined tensor among their inputs is an error)
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
Tensor value(const MaybeTensor& t) { return t ? *t : Tensor(); }

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const MaybeTensor& t) { return t && wants(*t); }
// the operators have gradients and no derivative forward: a tangent is refused, not dropped
bool tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool tangent(const MaybeTensor& t) { return t && tangent(*t); }
template <typename... Ts> void backward_only(const char* name, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(tangent(ts) || ...) || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), name,
                              " has no forward-mode derivative");
}
template <typename... Ts> bool training(const Ts&... ts) { return at::GradMode::is_enabled() && (wants(ts) || ...); }
template <typename... Ts> void serving(const char* name, const Ts&... ts) {
  backward_only(name, ts...);
  TORCH_CHECK_VALUE(!training(ts...), name, " has no gradient: call it under torch.no_grad()");
}

// ---- launches
const void* cptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const float* cfloat(const Tensor& t) { return (const float*)cptr(t); }
float* mfloat(const Tensor& t) { return (float*)mptr(t); }
const uint8_t* cbyte(const Tensor& t) { return (const uint8_t*)cptr(t); }

// the current stream of the tensors' device, that device current
struct Place {
  c10::DeviceGuard guard;
  void* stream;
  explicit Place(const Tensor& t)
      : guard(t.device()), stream(at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()) {}
};
template <typename F, typename... A> void call(const char* fn, F f, const Tensor& on, A... a) {
  const Place p(on);
  if (const int32_t rc = f(a..., p.stream)) fail(fn, rc);
}
#define CALL(f, ...) call("pnp_" #f, api.f, __VA_ARGS__)
template <typename D> int64_t floats(const char* fn, int64_t (*f)(const D*), const D& d) {
  const int64_t n = f(&d);
  if (n < 0) fail(fn, n);
  return n;
}
#define FLOATS(f, d) floats("pnp_" #f, api.f, d)

Tensor fresh(at::IntArrayRef shape, ScalarType t, const Tensor& like) { return at::empty(shape, like.options().dtype(t)); }
Tensor scratch(int64_t n, const Tensor& like) { return n ? fresh({n}, at::kFloat, like) : Tensor(); }

// gradients that have no gradient themselves: asked for one, they say so
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second gradient", (int64_t)grads.size());
  return (*node)(std::move(grads));
}

// ---- norm
// [..., dim] as rows
Tensor rows_of(const Tensor& t) { return t.defined() ? lines(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})) : t; }

pnp_norm_desc norm_desc(const Tensor& x, const Tensor& r, const Tensor& w, double eps) {
  pnp_norm_desc d{};
  d.rows = x.size(0); d.dim = (int32_t)x.size(1); d.type = code_of(x.scalar_type()); d.eps = (float)eps;
  d.res_type = code_of((r.defined() ? r : x).scalar_type());
  d.x = cptr(x); d.x_stride = x.stride(0); d.weight = cfloat(w);
  if (r.defined()) { d.residual = cptr(r); d.r_stride = r.stride(0); }
  return d;
}

struct NormRun { Tensor y, s, rstd; };
NormRun norm_run(const Tensor& x, const Tensor& r, const Tensor& w, double eps, bool train) {
  const Tensor x2 = rows_of(x), r2 = rows_of(r);
  NormRun o{fresh(x.sizes(), x.scalar_type(), x), x, train ? fresh({x2.size(0)}, at::kFloat, x) : Tensor()};
  if (r.defined()) o.s = fresh(x.sizes(), r.scalar_type(), x);
  pnp_norm_desc d = norm_desc(x2, r2, w, eps);
  d.y = mptr(o.y); d.rstd = mfloat(o.rstd);
  if (r.defined()) d.s = mptr(o.s);
  CALL(rms_norm, x, &d);
  return o;
}

struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& r_, const Tensor& w, double eps) {
    const Tensor r = value(r_);
    const NormRun o = norm_run(x, r, w, eps, true);
    ctx->save_for_backward({o.s, w, o.rstd});
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["flags"] = (int64_t)(r.defined() | (w.requires_grad() << 1));
    ctx->set_materialize_grads(false);
    return {o.y, o.s};   // without a residual s is x: the stream goes on through here, one rounding of dx + ds
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    backward_only("add_rms_norm", grads[0], grads[1]);
    const auto saved = ctx->get_saved_variables();
    const Tensor &s0 = saved[0], &w = saved[1], &rstd = saved[2];
    const ScalarType type = (ScalarType)ctx->saved_data["type"].toInt();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const bool added = flags & 1;
    if (!grads[0].defined()) {
      const Tensor& ds = grads[1];
      if (!ds.defined()) return variable_list(4);
      return once({ds.to(type), added ? ds : Tensor(), Tensor(), Tensor()}, "add_rms_norm");
    }
    const Tensor s = rows_of(s0), dy = rows_of(grads[0]), ds = rows_of(grads[1]);
    pnp_norm_bwd_desc d{};
    d.rows = s.size(0); d.dim = (int32_t)s.size(1); d.type = code_of(type); d.res_type = code_of(s.scalar_type());
    d.dy = cptr(dy); d.dy_stride = dy.stride(0); d.s = cptr(s); d.s_stride = s.stride(0);
    if (ds.defined()) { d.ds = cptr(ds); d.ds_stride = ds.stride(0); }
    d.weight = cfloat(w); d.rstd = cfloat(rstd);
    const Tensor dx = fresh(s0.sizes(), type, s);
    Tensor dres = dx, dw, ws;
    d.dx = mptr(dx);
    if (s.scalar_type() != type) {
      dres = fresh(s0.sizes(), s.scalar_type(), s);
      d.dres = mptr(dres);
    }
    if (flags & 2) {
      dw = fresh(w.sizes(), at::kFloat, s);
      d.workspace_floats = FLOATS(rms_norm_bwd_workspace, d);
      ws = scratch(d.workspace_floats, s);
      d.dweight = mfloat(dw); d.workspace = mfloat(ws);
    }
    CALL(rms_norm_bwd, s, &d);
    return once({dx, added ? dres : Tensor(), dw, Tensor()}, "add_rms_norm");
  }
};

struct NormIn { Tensor w, r; };
NormIn norm_in(const Tensor& x, const MaybeTensor& w, const MaybeTensor& r, double eps) {
  activation(x, "x");
  channels(x, "x");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative (got ", eps, ")");
  NormIn o;
  o.w = required(w, "weight", {x.size(-1)}, x);
  if (r && r->defined()) {
    activation(*r, "residual");
    TORCH_CHECK_TYPE(r->scalar_type() == x.scalar_type() || r->scalar_type() == at::kFloat, "residual: dtype ", r->scalar_type(), ", expected ",
                     x.scalar_type(), " or float32");
    same_device(*r, "residual", x);
    shaped(*r, "residual", x.sizes());
    o.r = *r;
  }
  return o;
}

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& residual, double eps) {
  backward_only("add_rms_norm", x, weight, residual);
  const NormIn in = norm_in(x, weight, residual, eps);
  if (training(x, in.w, in.r)) {
    const variable_list o = NormFn::apply(x, maybe(in.r), in.w, eps);
    return {o[0], o[1]};
  }
  const NormRun o = norm_run(x, in.r, in.w, eps, false);
  return {o.y, o.s};
}

// 8-bit rows, a multiple of 16 bytes apart: the product's loads want rows on such boundaries
struct Q8 { Tensor q, scale; };
Q8 q8_out(const Tensor& x) {
  return {fresh({x.size(0), (x.size(1) + 15) / 16 * 16}, at::kChar, x), fresh({x.size(0)}, at::kFloat, x)};
}
Q8 q8_view(const Q8& o, at::IntArrayRef shape) {
  if (shape.size() == 2) return {o.q.size(1) == shape[1] ? o.q : o.q.narrow(1, 0, shape[1]), o.scale};
  std::vector<int64_t> s = shape.vec();
  const Tensor scale = o.scale.view(shape.slice(0, shape.size() - 1));
  s.back() = o.q.size(1);
  return {o.q.view(s).narrow(-1, 0, shape.back()), scale};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_q8(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& residual, double eps) {
  serving("add_rms_norm_q8", x, weight, residual);
  const NormIn in = norm_in(x, weight, residual, eps);
  const Tensor x2 = rows_of(x), r2 = rows_of(in.r);
  const Q8 o = q8_out(x2);
  pnp_norm_desc d = norm_desc(x2, r2, in.w, eps);
  d.q = (int8_t*)mptr(o.q); d.q_stride = o.q.stride(0); d.scale = mfloat(o.scale);
  Tensor s = x;
  if (in.r.defined()) {
    s = fresh(x.sizes(), in.r.scalar_type(), x);
    d.s = mptr(s);
  }
  CALL(rms_norm, x, &d);
  const Q8 v = q8_view(o, x.sizes());
  return {v.q, v.scale, s};
}

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  serving("quantize_rows", x);
  activation(x, "x");
  channels(x, "x");
  const Tensor x2 = rows_of(x);
  const Q8 o = q8_out(x2);
  CALL(quantize_rows, x, cptr(x2), x2.stride(0), code_of(x.scalar_type()), x2.size(0), (int32_t)x2.size(1), (int8_t*)mptr(o.q), o.q.stride(0),
       mfloat(o.scale));
  const Q8 v = q8_view(o, x.sizes());
  return {v.q, v.scale};
}

// ---- product in 8 bits
// rows that do not overlap, contiguous each (a broadcast row is copied out)
Tensor i8_rows(const Tensor& t) {
  const Tensor l = lines(t);
  return l.size(0) <= 1 || l.stride(0) >= l.size(1) ? l : l.contiguous();
}

Tensor matmul_i8(const Tensor& q, const MaybeTensor& scale, const Tensor& wq, const MaybeTensor& wscale, const MaybeTensor& bias,
                 ScalarType out_dtype) {
  serving("matmul_i8", scale, wscale, bias);
  TORCH_CHECK_TYPE(q.scalar_type() == at::kChar, "q must be an int8 tensor");
  TORCH_CHECK_TYPE(wq.scalar_type() == at::kChar, "wq must be an int8 tensor");
  on_device(q, "q");
  on_device(wq, "wq");
  TORCH_CHECK_TYPE(code_of(out_dtype) >= 0, "out_dtype ", out_dtype, ", expected float32, bfloat16 or float16");
  TORCH_CHECK_VALUE(wq.dim() == 2 && q.dim() >= 1 && q.size(-1) == wq.size(1) && wq.numel() > 0, "q ", q.sizes(), " and wq ", wq.sizes(),
                    ": expected [..., K] and [N, K]");
  same_device(wq, "wq", q);
  const int64_t K = wq.size(1), N = wq.size(0);
  std::vector<int64_t> shape = q.sizes().vec();
  shape.back() = N;
  const Tensor s = required(scale, "scale", q.sizes().slice(0, q.dim() - 1), q), ws = required(wscale, "wscale", {N}, q),
               b = parameter(bias, "bias", {N}, q);
  const Tensor q2 = i8_rows(q.reshape({-1, K})), w2 = i8_rows(wq), out = fresh(shape, out_dtype, q);
  pnp_i8_desc d{};
  TORCH_CHECK_VALUE(N < (1 << 30) && K < (1 << 30), "wq: shape ", wq.sizes(), " is too large");
  d.M = q2.size(0); d.N = (int32_t)N; d.K = (int32_t)K; d.out_type = code_of(out_dtype);
  d.q = (const int8_t*)cptr(q2); d.wq = (const int8_t*)cptr(w2);
  d.q_stride = std::max(q2.stride(0), K); d.wq_stride = std::max(w2.stride(0), K);
  d.scale = cfloat(s); d.wscale = cfloat(ws); d.bias = cfloat(b); d.out = mptr(out);
  CALL(matmul_i8, q, &d);
  return out;
}

// ---- causal convolution
pnp_conv_desc conv_desc(const Tensor& x, const Tensor& w, const Tensor& b, bool silu, const Tensor& starts, const Tensor& state) {
  pnp_conv_desc d{};
  d.B = x.size(0); d.L = x.size(1); d.dim = (int32_t)x.size(2); d.width = (int32_t)w.size(1);
  d.type = code_of(x.scalar_type()); d.silu = silu;
  d.x = cptr(x); d.x_bstride = x.stride(0); d.x_tstride = x.stride(1);
  d.weight = cfloat(w); d.bias = cfloat(b); d.starts = cbyte(starts); d.state = cptr(state);
  return d;
}

std::tuple<Tensor, Tensor> conv_run(const Tensor& x, const Tensor& w, const Tensor& b, bool silu, const Tensor& starts, const Tensor& state) {
  const Tensor y = fresh(x.sizes(), x.scalar_type(), x), last = fresh({x.size(0), w.size(1) - 1, x.size(2)}, x.scalar_type(), x);
  pnp_conv_desc d = conv_desc(x, w, b, silu, starts, state);
  d.y = mptr(y); d.last_state = mptr(last);
  CALL(causal_conv, x, &d);
  return {y, last};
}

struct ConvFn : torch::autograd::Function<ConvFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const MaybeTensor& b_, bool silu,
                               const MaybeTensor& starts_, const MaybeTensor& state_) {
    const Tensor b = value(b_), starts = value(starts_), state = value(state_);
    const auto [y, last] = conv_run(x, w, b, silu, starts, state);
    ctx->save_for_backward({x, w, b, starts, state});
    ctx->saved_data["flags"] = (int64_t)(silu | (wants(w) << 1) | (wants(b) << 2) | (wants(state) << 3));
    ctx->set_materialize_grads(false);
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    backward_only("causal_conv", grads[0], grads[1]);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &starts = saved[3], &state = saved[4];
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(6);
    const Tensor dy = grads[0].defined() ? lines(grads[0]) : at::zeros(x.sizes(), x.options());
    const Tensor dlast = grads[1].defined() ? whole(grads[1]) : Tensor();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    pnp_conv_bwd_desc d{};
    d.f = conv_desc(x, w, b, flags & 1, starts, state);
    d.dy = cptr(dy); d.dy_bstride = dy.stride(0); d.dy_tstride = dy.stride(1); d.dlast = cptr(dlast);
    const Tensor dx = fresh(x.sizes(), x.scalar_type(), x);
    Tensor dw, db, ds, ws;
    if (flags & 2) dw = fresh(w.sizes(), at::kFloat, x);
    if (flags & 4) db = fresh(b.sizes(), at::kFloat, x);
    if (flags & 8) ds = fresh(state.sizes(), x.scalar_type(), x);
    d.dx = mptr(dx); d.dweight = mfloat(dw); d.dbias = mfloat(db); d.dstate = mptr(ds);
    if (dw.defined() || db.defined()) {
      d.workspace_floats = FLOATS(causal_conv_bwd_workspace, d);
      ws = scratch(d.workspace_floats, x);
      d.workspace = mfloat(ws);
    }
    CALL(causal_conv_bwd, x, &d);
    return once({dx, dw, db, Tensor(), Tensor(), ds}, "causal_conv");
  }
};

Tensor conv_weight(const Tensor& w, int64_t dim, const Tensor& like) {
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) >= 2 && w.size(1) <= 4, "weight: expected [dim, width] with a width of 2, 3 or 4");
  return parameter(w, "weight", {dim, w.size(1)}, like);
}
bool is_silu(const c10::optional<std::string>& a) {
  TORCH_CHECK_VALUE(!a || *a == "silu", "activation '", *a, "', expected None or 'silu'");
  return a.has_value();
}

std::tuple<Tensor, Tensor> causal_conv(const Tensor& x_, const Tensor& weight, const MaybeTensor& bias, const c10::optional<std::string>& act,
                                       const MaybeTensor& starts_, const MaybeTensor& state_) {
  backward_only("causal_conv", x_, weight, bias, state_);
  activation(x_, "x");
  dims(x_, "x", 3);
  channels(x_, "x");
  const bool silu = is_silu(act);
  const Tensor w = conv_weight(weight, x_.size(2), x_), b = parameter(bias, "bias", {x_.size(2)}, x_);
  const Tensor starts = marks(starts_, "starts", x_.sizes().slice(0, 2), x_);
  Tensor state;
  if (state_ && state_->defined()) {
    activation(*state_, "state", &x_);
    shaped(*state_, "state", {x_.size(0), w.size(1) - 1, x_.size(2)});
    state = whole(*state_);
  }
  const Tensor x = lines(x_);
  if (!training(x, w, b, state)) return conv_run(x, w, b, silu, starts, state);
  const variable_list o = ConvFn::apply(x, w, maybe(b), silu, maybe(starts), maybe(state));
  return {o[0], o[1]};
}

Tensor causal_conv_step(const Tensor& x_, const Tensor& state, const Tensor& weight, const MaybeTensor& bias,
                        const c10::optional<std::string>& act, const MaybeTensor& reset_) {
  serving("causal_conv_step", x_, state, weight, bias);
  activation(x_, "x");
  dims(x_, "x", 2);
  channels(x_, "x");
  const bool silu = is_silu(act);
  const Tensor w = conv_weight(weight, x_.size(1), x_), b = parameter(bias, "bias", {x_.size(1)}, x_);
  activation(state, "state", &x_);
  shaped(state, "state", {x_.size(0), w.size(1) - 1, x_.size(1)});
  in_place(state);
  const Tensor reset = apart(marks(reset_, "reset", x_.sizes().slice(0, 1), x_), state), x = apart(lines(x_), state);
  const Tensor wa = apart(w, state), ba = apart(b, state), y = fresh(x.sizes(), x.scalar_type(), x);
  CALL(causal_conv_step, x, cptr(x), x.stride(0), mptr(state), cfloat(wa), cfloat(ba), cbyte(reset), x.size(0), (int32_t)x.size(1),
       (int32_t)w.size(1), code_of(x.scalar_type()), (int32_t)silu, mptr(y));
  advanced(state);
  return y;
}

// ---- selective scan
struct ScanIn { Tensor u, delta, A, B, C, D, z, bias; };

// [..., N] or [..., groups, N] with what follows the leading dimensions contiguous
Tensor packed_groups(const Tensor& t_, int64_t lead) {
  const Tensor t = plain(t_);
  const bool ok = (t.size(-1) == 1 || t.stride(-1) == 1) && (t.dim() == lead + 1 || t.size(-2) == 1 || t.stride(-2) == t.size(-1));
  return ok ? t : t.contiguous();
}

// the scan's offsets within a tile are 32-bit: a tensor with tokens further apart is copied
Tensor near(const Tensor& t, int64_t lead) {
  return t.defined() && lead == 2 && t.stride(1) > PNP_SCAN_MAX_TSTRIDE ? t.contiguous() : t;
}

// lead: dimensions before the channels
ScanIn scan_in(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const MaybeTensor& D, const MaybeTensor& z,
               const MaybeTensor& bias, int64_t lead) {
  activation(u, "u");
  dims(u, "u", lead + 1);
  const int64_t dim = u.size(-1);
  channels(u, "u");
  activation(delta, "delta", &u);
  shaped(delta, "delta", u.sizes());
  if (z && z->defined()) {
    activation(*z, "z", &u);
    shaped(*z, "z", u.sizes());
  }
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(1) >= 1 && A.size(1) <= 64, "A: expected [dim, N] with N from 1 to 64");
  const Tensor A32 = parameter(A, "A", {dim, A.size(1)}, u);
  activation(B, "B", &u);
  activation(C, "C", &u);
  const int64_t groups = B.dim() == lead + 2 ? B.size(-2) : B.dim() == lead + 1 ? 1 : 0;
  std::vector<int64_t> want = u.sizes().slice(0, lead).vec();
  if (B.dim() == lead + 2) want.push_back(groups);
  want.push_back(A.size(1));
  TORCH_CHECK_VALUE(groups >= 1 && dim % groups == 0 && B.sizes() == want && C.sizes() == want, "B ", B.sizes(), " and C ", C.sizes(),
                    ": expected ", u.sizes().slice(0, lead), " and then [groups,] ", A.size(1), ", groups dividing ", dim);
  return {near(lines(u), lead), near(lines(delta), lead), A32, near(packed_groups(B, lead), lead), near(packed_groups(C, lead), lead),
          parameter(D, "D", {dim}, u), z && z->defined() ? near(lines(*z), lead) : Tensor(), parameter(bias, "delta_bias", {dim}, u)};
}

pnp_scan_desc scan_desc(const ScanIn& v, const Tensor& starts, const Tensor& state, bool step) {
  pnp_scan_desc d{};
  d.B = v.u.size(0); d.L = step ? 1 : v.u.size(1); d.dim = (int32_t)v.u.size(-1); d.N = (int32_t)v.A.size(1);
  d.groups = v.B.dim() == (step ? 3 : 4) ? (int32_t)v.B.size(-2) : 1; d.type = code_of(v.u.scalar_type());
  auto put = [&](const Tensor& t, const void*& p, int64_t& sb, int64_t& st) {
    if (!t.defined()) return;
    p = cptr(t);
    sb = t.stride(0);
    st = step ? 0 : t.stride(1);
  };
  put(v.u, d.u, d.u_bstride, d.u_tstride);
  put(v.delta, d.delta, d.delta_bstride, d.delta_tstride);
  put(v.z, d.z, d.z_bstride, d.z_tstride);
  put(v.B, d.Bm, d.B_bstride, d.B_tstride);
  put(v.C, d.Cm, d.C_bstride, d.C_tstride);
  d.A = cfloat(v.A); d.D = cfloat(v.D); d.delta_bias = cfloat(v.bias); d.state = cfloat(state); d.starts = cbyte(starts);
  return d;
}

struct ScanRun { Tensor out, last, ckpt; };
ScanRun scan_run(const ScanIn& v, const Tensor& starts, const Tensor& state, bool train) {
  ScanRun o{fresh(v.u.sizes(), v.u.scalar_type(), v.u), fresh({v.u.size(0), v.u.size(2), v.A.size(1)}, at::kFloat, v.u), Tensor()};
  pnp_scan_desc d = scan_desc(v, starts, state, false);
  d.out = mptr(o.out); d.last_state = mfloat(o.last);
  d.workspace_floats = FLOATS(scan_workspace, d);
  const Tensor ws = scratch(d.workspace_floats, v.u);
  d.workspace = mfloat(ws);
  if (train) {
    d.ckpt_floats = FLOATS(scan_ckpt_floats, d);
    o.ckpt = scratch(d.ckpt_floats, v.u);
    d.ckpt = mfloat(o.ckpt);
  }
  CALL(selective_scan, v.u, &d);
  return o;
}

struct ScanFn : torch::autograd::Function<ScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                               const MaybeTensor& D_, const MaybeTensor& z_, const MaybeTensor& bias_, const MaybeTensor& starts_,
                               const MaybeTensor& state_) {
    const Tensor D = value(D_), z = value(z_), bias = value(bias_), starts = value(starts_), state = value(state_);
    const ScanRun o = scan_run({u, delta, A, B, C, D, z, bias}, starts, state, true);
    ctx->save_for_backward({u, delta, A, B, C, D, z, bias, starts, state, o.ckpt});
    ctx->set_materialize_grads(false);
    return {o.out, o.last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    backward_only("selective_scan", grads[0], grads[1]);
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(10);
    const auto s = ctx->get_saved_variables();
    const ScanIn v{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]};
    const Tensor &starts = s[8], &state = s[9], &ckpt = s[10], &u = v.u;
    const ScalarType t = u.scalar_type();
    const Tensor dout = grads[0].defined() ? near(lines(grads[0]), 2) : at::zeros(u.sizes(), u.options());
    const Tensor dlast = grads[1].defined() ? whole(grads[1]) : Tensor();
    pnp_scan_bwd_desc d{};
    d.f = scan_desc(v, starts, state, false);
    d.f.ckpt = mfloat(ckpt); d.f.ckpt_floats = ckpt.defined() ? ckpt.numel() : 0;
    d.dout = cptr(dout); d.dout_bstride = dout.stride(0); d.dout_tstride = dout.stride(1); d.dlast = cfloat(dlast);
    const Tensor du = fresh(u.sizes(), t, u), dd = fresh(u.sizes(), t, u), dB = fresh(v.B.sizes(), t, u), dC = fresh(v.C.sizes(), t, u);
    const Tensor dz = v.z.defined() ? fresh(u.sizes(), t, u) : Tensor();
    auto like32 = [&](const Tensor& p) { return p.defined() ? fresh(p.sizes(), at::kFloat, u) : Tensor(); };
    const Tensor dA = like32(v.A), dD = like32(v.D), dbias = like32(v.bias), dstate = like32(state);
    d.du = mptr(du); d.ddelta = mptr(dd); d.dz = mptr(dz); d.dB = mptr(dB); d.dC = mptr(dC);
    d.dA = mfloat(dA); d.dD = mfloat(dD); d.ddelta_bias = mfloat(dbias); d.dstate = mfloat(dstate);
    d.workspace_floats = FLOATS(scan_bwd_workspace, d);
    const Tensor ws = scratch(d.workspace_floats, u);
    d.workspace = mfloat(ws);
    CALL(selective_scan_bwd, u, &d);
    return once({du, dd, dA, dB, dC, dD, dz, dbias, Tensor(), dstate}, "selective_scan");
  }
};

void state32(const Tensor& s, at::IntArrayRef want, const Tensor& like) {
  TORCH_CHECK_TYPE(s.scalar_type() == at::kFloat, "state must be a float32 tensor");
  same_device(s, "state", like);
  shaped(s, "state", want);
}

std::tuple<Tensor, Tensor> selective_scan(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                                          const MaybeTensor& D, const MaybeTensor& z, const MaybeTensor& bias, const MaybeTensor& starts_,
                                          const MaybeTensor& state_) {
  backward_only("selective_scan", u, delta, A, B, C, D, z, bias, state_);
  const ScanIn v = scan_in(u, delta, A, B, C, D, z, bias, 2);
  const Tensor starts = marks(starts_, "starts", u.sizes().slice(0, 2), u);
  Tensor state;
  if (state_ && state_->defined()) {
    state32(*state_, {u.size(0), u.size(2), A.size(1)}, u);
    state = whole(*state_);
  }
  if (!training(v.u, v.delta, v.A, v.B, v.C, v.D, v.z, v.bias, state)) {
    const ScanRun o = scan_run(v, starts, state, false);
    return {o.out, o.last};
  }
  const variable_list o = ScanFn::apply(v.u, v.delta, v.A, v.B, v.C, maybe(v.D), maybe(v.z), maybe(v.bias), maybe(starts), maybe(state));
  return {o[0], o[1]};
}

Tensor selective_scan_step(const Tensor& u, const Tensor& state, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                           const MaybeTensor& D, const MaybeTensor& z, const MaybeTensor& bias, const MaybeTensor& reset_) {
  serving("selective_scan_step", u, state, delta, A, B, C, D, z, bias);
  ScanIn v = scan_in(u, delta, A, B, C, D, z, bias, 1);
  state32(state, {u.size(0), u.size(1), A.size(1)}, u);
  in_place(state);
  for (Tensor* t : {&v.u, &v.delta, &v.A, &v.B, &v.C, &v.D, &v.z, &v.bias}) *t = apart(*t, state);
  const Tensor reset = apart(marks(reset_, "reset", u.sizes().slice(0, 1), u), state), out = fresh(u.sizes(), u.scalar_type(), u);
  pnp_scan_desc d = scan_desc(v, reset, state, true);
  d.out = mptr(out); d.last_state = mfloat(state);
  CALL(selective_scan_step, u, &d);
  advanced(state);
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failed& e) {
      const py::object type = py::module_::import("pnp_amd._lib").attr("PnpError");
      PyErr_SetString(type.ptr(), e.what());
    }
  });
  const py::call_guard<py::gil_scoped_release> free;
  const auto none = py::none();
  m.def("bind", &bind);
  m.def("add_rms_norm", &add_rms_norm, py::arg("x"), py::arg("weight"), py::arg("residual") = none, py::arg("eps") = 1e-6, free);
  m.def("add_rms_norm_q8", &add_rms_norm_q8, py::arg("x"), py::arg("weight"), py::arg("residual") = none, py::arg("eps") = 1e-6, free);
  m.def("quantize_rows", &quantize_rows, py::arg("x"), free);
  m.def("matmul_i8", &matmul_i8, py::arg("q"), py::arg("scale"), py::arg("wq"), py::arg("wscale"), py::arg("bias") = none,
        py::arg("out_dtype") = at::kFloat, free);
  m.def("causal_conv", &causal_conv, py::arg("x"), py::arg("weight"), py::arg("bias") = none, py::arg("activation") = none,
        py::arg("starts") = none, py::arg("state") = none, free);
  m.def("causal_conv_step", &causal_conv_step, py::arg("x"), py::arg("state"), py::arg("weight"), py::arg("bias") = none,
        py::arg("activation") = none, py::arg("reset") = none, free);
  m.def("selective_scan", &selective_scan, py::arg("u"), py::arg("delta"), py::arg("A"), py::arg("B"), py::arg("C"), py::arg("D") = none,
        py::arg("z") = none, py::arg("delta_bias") = none, py::arg("starts") = none, py::arg("state") = none, free);
  m.def("selective_scan_step", &selective_scan_step, py::arg("u"), py::arg("state"), py::arg("delta"), py::arg("A"), py::arg("B"),
        py::arg("C"), py::arg("D") = none, py::arg("z") = none, py::arg("delta_bias") = none, py::arg("reset") = none, free);
}

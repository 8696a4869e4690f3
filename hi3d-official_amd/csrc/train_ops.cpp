// torch.ops.hi3d.* of the training kernels (norm_train.hip, linear_train.hip, adamw.hip): torch tensors in, fresh tensors out (AdamW: in place),
// checks before anything is launched, the current stream of the operands' device.  Host-only C++, as torch_ops.cpp.
// The autograd face of these is hi3d_hip/train.py.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/hi3d_hip.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
void check_rc(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (rc=", rc, "): ", hi3d_last_error()); }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
void* ptr(const OptTensor& t) { return has(t) ? t->data_ptr() : nullptr; }

int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return HI3D_F32;
    case at::kBFloat16: return HI3D_BF16;
    case at::kHalf: return HI3D_F16;
    default: TORCH_CHECK(false, name, ": fp32, bf16 or fp16 required, got ", t.scalar_type());
  }
}
void want_gpu(const Tensor& t, const Tensor& on, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.layout() == at::kStrided, name, ": dense device tensor required (this framework has no CPU path)");
  TORCH_CHECK(t.device() == on.device(), name, ": on ", t.device(), ", the other operands on ", on.device());
  TORCH_CHECK(!t.is_conj() && !t.is_neg(), name, ": lazily conjugated or negated view");
}

// the rows of t (all but its last dimension) at one pitch >= their length: t itself where its strides say so, a dense copy of it otherwise
struct Rows { Tensor t; int64_t n, width, ld; };
Rows rows_of(const Tensor& t) {
  const int64_t d = t.dim(), C = t.size(-1), R = C ? t.numel() / C : 0;
  bool ok = C <= 1 || t.stride(-1) == 1;
  int64_t ld = -1, next = 0;
  for (int64_t i = d - 2; i >= 0 && ok; --i) {
    if (t.size(i) == 1) continue;
    if (ld < 0) ld = next = t.stride(i);
    else ok = t.stride(i) == next;
    next = t.stride(i) * t.size(i);
  }
  if (ld < 0) ld = C;                                   // one row
  if (ok && ld >= C) return {t, R, C, ld};
  return {t.contiguous(), R, C, C};
}
Tensor dense(const OptTensor& t) { return has(t) ? t->contiguous() : Tensor(); }

// ---- layer norm -------------------------------------------------------------------------------------------------------------------
struct NormArgs { int64_t R; int C, dtype, wdtype; };
NormArgs norm_args(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const char* name) {
  want_gpu(x, x, name);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, name, ": a last dimension of at least one element required");
  TORCH_CHECK(x.size(-1) <= HI3D_NORM_MAX_WIDTH, name, ": width ", x.size(-1), " is over ", HI3D_NORM_MAX_WIDTH);
  NormArgs a = {x.numel() / x.size(-1), (int)x.size(-1), dtype_of(x, name), HI3D_F32};
  for (const OptTensor* t : {&weight, &bias}) {
    if (!has(*t)) continue;
    want_gpu(**t, x, name);
    TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == a.C, name, ": weight and bias must be [", a.C, "]");
    a.wdtype = dtype_of(**t, name);
  }
  TORCH_CHECK(!has(weight) || !has(bias) || weight->scalar_type() == bias->scalar_type(), name, ": weight and bias must have one type");
  return a;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> norm_fwd(const Tensor& x, const OptTensor& residual, const OptTensor& weight, const OptTensor& bias, double eps,
                                                    const char* name) {
  const NormArgs a = norm_args(x, weight, bias, name);
  TORCH_CHECK(std::isfinite(eps) && eps >= 0, name, ": eps must be finite and not negative");
  if (has(residual)) {
    want_gpu(*residual, x, name);
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), name, ": residual must have x's shape and type");
  }
  const Guard guard(x.device());
  const Rows rx = rows_of(x), rr = has(residual) ? rows_of(*residual) : Rows{Tensor(), 0, 0, 0};
  const Tensor w = dense(weight), b = dense(bias);
  Tensor y = at::empty(x.sizes(), x.options()), z;
  if (has(residual)) z = at::empty(x.sizes(), x.options());
  const auto stat = x.sizes().slice(0, x.dim() - 1);
  Tensor mean = at::empty(stat, x.options().dtype(at::kFloat)), rstd = at::empty(stat, x.options().dtype(at::kFloat));
  check_rc(hi3d_layernorm_fwd(rx.t.data_ptr(), rr.t.defined() ? rr.t.data_ptr() : nullptr, w.defined() ? w.data_ptr() : nullptr,
                              b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), z.defined() ? z.data_ptr() : nullptr, mean.data_ptr<float>(),
                              rstd.data_ptr<float>(), a.R, a.C, rx.ld, rr.ld, a.dtype, a.wdtype, (float)eps, stream_of(x)), "hi3d_layernorm_fwd");
  return {y, z, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layernorm_fwd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  auto r = norm_fwd(x, c10::nullopt, weight, bias, eps, "hi3d::layernorm_fwd");
  return {std::get<0>(r), std::get<2>(r), std::get<3>(r)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> add_layernorm_fwd(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& bias, double eps) {
  return norm_fwd(x, residual, weight, bias, eps, "hi3d::add_layernorm_fwd");
}

std::tuple<Tensor, Tensor, Tensor> layernorm_bwd(const Tensor& dy, const Tensor& z, const Tensor& mean, const Tensor& rstd, const OptTensor& weight,
                                                 const OptTensor& bias, const OptTensor& dz, bool need_dw, bool need_db) {
  const char* name = "hi3d::layernorm_bwd";
  const NormArgs a = norm_args(z, weight, bias, name);
  want_gpu(dy, z, name);
  TORCH_CHECK(dy.sizes() == z.sizes() && dy.scalar_type() == z.scalar_type(), name, ": dy must have z's shape and type");
  if (has(dz)) {
    want_gpu(*dz, z, name);
    TORCH_CHECK(dz->sizes() == z.sizes() && dz->scalar_type() == z.scalar_type(), name, ": dz must have z's shape and type");
  }
  for (const Tensor* t : {&mean, &rstd}) {
    want_gpu(*t, z, name);
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->numel() == a.R && t->is_contiguous(), name, ": mean and rstd must be dense fp32, one value a row");
  }
  const Guard guard(z.device());
  const Rows ry = rows_of(dy), rz = rows_of(z), rd = has(dz) ? rows_of(*dz) : Rows{Tensor(), 0, 0, 0};
  const Tensor w = dense(weight);
  Tensor dx = at::empty(z.sizes(), z.options()), dw, db;
  if (has(weight) && need_dw) dw = at::empty({a.C}, weight->options());
  if (has(bias) && need_db) db = at::empty({a.C}, bias->options());
  const int64_t ws_n = (dw.defined() || db.defined()) ? hi3d_layernorm_bwd_workspace_floats(a.R, a.C, a.dtype) : 0;
  Tensor ws;
  if (ws_n) ws = at::empty({ws_n}, z.options().dtype(at::kFloat));
  check_rc(hi3d_layernorm_bwd(ry.t.data_ptr(), rz.t.data_ptr(), rd.t.defined() ? rd.t.data_ptr() : nullptr, w.defined() ? w.data_ptr() : nullptr,
                              mean.data_ptr<float>(), rstd.data_ptr<float>(), dx.data_ptr(), dw.defined() ? dw.data_ptr() : nullptr,
                              db.defined() ? db.data_ptr() : nullptr, ws_n ? ws.data_ptr<float>() : nullptr, a.R, a.C, ry.ld, rz.ld, rd.ld, a.dtype, a.wdtype,
                              stream_of(z)), "hi3d_layernorm_bwd");
  return {dx, dw, db};
}

// ---- linear layer -----------------------------------------------------------------------------------------------------------------
int act_of(c10::string_view a, const char* name) {
  if (a == "none") return HI3D_ACT_NONE;
  if (a == "gelu") return HI3D_ACT_GELU;
  if (a == "quick_gelu") return HI3D_ACT_QUICK_GELU;
  if (a == "silu") return HI3D_ACT_SILU;
  if (a == "relu") return HI3D_ACT_RELU;
  TORCH_CHECK(false, name, ": unknown activation '", a, "' (none, gelu, quick_gelu, silu, relu)");
}
// sizes, types and activation of a call on x [M, K], w [N, K], bias [N]
hi3d_linear_desc linear_desc(const Tensor& x, const Tensor& w, const OptTensor& bias, c10::string_view act, const char* name) {
  want_gpu(x, x, name);
  want_gpu(w, x, name);
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && x.size(1) >= 1 && w.size(0) >= 1, name, ": x [M, K] and w [N, K] of at least one column required");
  TORCH_CHECK(x.scalar_type() == w.scalar_type() && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf), name, ": x and w must both be bf16 or both fp16");
  TORCH_CHECK(w.size(0) <= 0x7fffffffLL && w.size(1) <= 0x7fffffffLL, name, ": a width does not fit 32 bits");
  hi3d_linear_desc d = {};
  d.M = x.size(0); d.N = (int32_t)w.size(0); d.K = (int32_t)w.size(1);
  d.dtype = dtype_of(x, name); d.bias_dtype = HI3D_F32; d.act = act_of(act, name);
  if (has(bias)) {
    want_gpu(*bias, x, name);
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == d.N && (bias->scalar_type() == at::kFloat || bias->scalar_type() == x.scalar_type()), name,
                ": bias must be [N], fp32 or of x's type");
    d.bias_dtype = dtype_of(*bias, name);
  }
  return d;
}
void want_like(const Tensor& t, const Tensor& x, int64_t M, int64_t N, const char* name, const char* what) {
  want_gpu(t, x, name);
  TORCH_CHECK(t.dim() == 2 && t.size(0) == M && t.size(1) == N && t.scalar_type() == x.scalar_type(), name, ": ", what, " must be [", M, ", ", N, "] of x's type");
}
Tensor workspace(hi3d_linear_desc* d, int64_t bytes, const Tensor& on) {
  Tensor ws;
  if (bytes) {
    ws = at::empty({bytes}, on.options().dtype(at::kByte));
    d->ws = ws.data_ptr(); d->ws_bytes = bytes;
  }
  return ws;
}

std::tuple<Tensor, Tensor> linear_act(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, c10::string_view act, bool save_z) {
  const char* name = "hi3d::linear_act";
  hi3d_linear_desc d = linear_desc(x, w, bias, act, name);
  if (has(residual)) want_like(*residual, x, d.M, d.N, name, "residual");
  const Guard guard(x.device());
  const Rows rx = rows_of(x), rw = rows_of(w), rr = has(residual) ? rows_of(*residual) : Rows{Tensor(), 0, 0, 0};
  const Tensor b = dense(bias);
  Tensor y = at::empty({d.M, d.N}, x.options()), z;
  if (save_z) z = at::empty({d.M, d.N}, x.options());
  d.x = rx.t.data_ptr(); d.ldx = rx.ld; d.w = rw.t.data_ptr(); d.ldw = rw.ld;
  d.bias = b.defined() ? b.data_ptr() : nullptr;
  if (rr.t.defined()) { d.residual = rr.t.data_ptr(); d.ldr = rr.ld; }
  d.y = y.data_ptr(); d.z = z.defined() ? z.data_ptr() : nullptr;
  const Tensor ws = workspace(&d, hi3d_linear_fwd_workspace_bytes(&d), x);
  check_rc(hi3d_linear_fwd(&d, stream_of(x)), "hi3d_linear_fwd");
  return {y, z};
}

std::tuple<Tensor, Tensor, Tensor> linear_act_bwd(const Tensor& dy, const Tensor& x, const Tensor& w, const OptTensor& z, const OptTensor& bias, c10::string_view act,
                                                  bool need_dx, bool need_dw) {
  const char* name = "hi3d::linear_act_bwd";
  hi3d_linear_desc d = linear_desc(x, w, bias, act, name);
  want_like(dy, x, d.M, d.N, name, "dy");
  TORCH_CHECK(d.act == HI3D_ACT_NONE || has(z), name, ": this activation's gradient needs z");
  if (has(z)) want_like(*z, x, d.M, d.N, name, "z");
  const Guard guard(x.device());
  const Rows ry = rows_of(dy), rz = d.act != HI3D_ACT_NONE ? rows_of(*z) : Rows{Tensor(), 0, 0, 0}, rx = rows_of(x), rw = rows_of(w);
  Tensor dx, dw, db;
  if (need_dx) dx = at::empty({d.M, d.K}, x.options());
  if (need_dw) dw = at::empty({d.N, d.K}, w.options());
  if (has(bias)) db = at::empty({d.N}, bias->options());
  d.x = rx.t.data_ptr(); d.ldx = rx.ld; d.w = rw.t.data_ptr(); d.ldw = rw.ld; d.dy = ry.t.data_ptr(); d.lddy = ry.ld;
  if (rz.t.defined()) { d.z = rz.t.data_ptr(); d.ldz = rz.ld; }
  d.dx = dx.defined() ? dx.data_ptr() : nullptr; d.dw = dw.defined() ? dw.data_ptr() : nullptr; d.db = db.defined() ? db.data_ptr() : nullptr;
  const Tensor ws = workspace(&d, hi3d_linear_bwd_workspace_bytes(&d), x);
  check_rc(hi3d_linear_bwd(&d, stream_of(x)), "hi3d_linear_bwd");
  return {dx, dw, db};
}

// ---- AdamW ------------------------------------------------------------------------------------------------------------------------
const float* scalar_of(const OptTensor& t, const Tensor& on, const char* what) {
  if (!has(t)) return nullptr;
  want_gpu(*t, on, what);
  TORCH_CHECK(t->scalar_type() == at::kFloat && t->numel() == 1, what, ": one fp32 value required");
  return t->data_ptr<float>();
}

using Spans = std::vector<std::pair<uintptr_t, uintptr_t>>;
void span_of(const Tensor& t, Spans& to) {
  const uintptr_t b = (uintptr_t)t.data_ptr();
  if (const int64_t n = t.numel()) to.emplace_back(b, b + n * t.element_size());
}
// whether what is written overlaps nothing else (lists of views into one buffer, or of tensors in the order of their allocation, are in order
// already and merged in linear time)
bool apart(Spans (&written)[4], Spans& read) {
  Spans all;
  for (Spans& l : written) {
    if (!std::is_sorted(l.begin(), l.end())) std::sort(l.begin(), l.end());
    Spans both(all.size() + l.size());
    std::merge(all.begin(), all.end(), l.begin(), l.end(), both.begin());
    all.swap(both);
  }
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].first < all[i - 1].second) return false;
  if (!std::is_sorted(read.begin(), read.end())) std::sort(read.begin(), read.end());
  size_t i = 0;
  for (const auto& r : read) {
    while (i < all.size() && all[i].second <= r.first) ++i;
    if (i < all.size() && all[i].first < r.second) return false;
  }
  return true;
}

void adamw_(at::TensorList params, at::TensorList grads, at::TensorList exp_avg, at::TensorList exp_avg_sq, at::TensorList copies, double lr, double beta1,
            double beta2, double eps, double weight_decay, int64_t step, const OptTensor& step_t, const OptTensor& lr_t, const OptTensor& grad_scale,
            const OptTensor& found_inf) {
  const char* name = "hi3d::adamw_";
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && exp_avg.size() == n && exp_avg_sq.size() == n && (copies.empty() || copies.size() == n), name, ": lists of different lengths");
  TORCH_CHECK(std::isfinite(lr) && lr >= 0 && std::isfinite(eps) && eps >= 0 && std::isfinite(weight_decay) && weight_decay >= 0, name,
              ": lr, eps and weight_decay must be finite and not negative");
  TORCH_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, name, ": betas must be in [0, 1)");
  TORCH_CHECK(has(step_t) || (!has(lr_t) && !has(grad_scale) && !has(found_inf)), name, ": lr, grad_scale and found_inf on the device need the step there too");
  TORCH_CHECK(has(step_t) || step >= 1, name, ": steps count from 1");
  if (!n) return;
  const Tensor& on = params[0];
  // one launch per combination of types; the tensors of a combination keep their order
  struct Kind { int p, g, c; std::vector<hi3d_adamw_tensor> t; };
  std::vector<Kind> kinds;
  Spans written[4], read;                     // parameters, both moments, copies; gradients
  for (Spans& l : written) l.reserve(n);
  read.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &g = grads[i], &m = exp_avg[i], &v = exp_avg_sq[i];
    want_gpu(p, on, name);
    const int pd = dtype_of(p, name), gd = dtype_of(g, name);
    TORCH_CHECK(p.is_non_overlapping_and_dense(), name, ": tensor ", i, ": parameters must be dense in memory (in any order of dimensions)");
    for (const Tensor* t : {&g, &m, &v}) {
      want_gpu(*t, on, name);
      TORCH_CHECK(t->sizes() == p.sizes() && t->strides() == p.strides(), name, ": tensor ", i, ": gradient and moments must have the parameter's shape and strides");
    }
    TORCH_CHECK(m.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat, name, ": tensor ", i, ": moments must be fp32");
    hi3d_adamw_tensor d = {p.data_ptr(), g.data_ptr(), m.data_ptr<float>(), v.data_ptr<float>(), nullptr, p.numel()};
    int cd = HI3D_BF16;
    span_of(p, written[0]); span_of(m, written[1]); span_of(v, written[2]); span_of(g, read);
    if (!copies.empty()) {
      const Tensor& c = copies[i];
      want_gpu(c, on, name);
      TORCH_CHECK(pd == HI3D_F32 && (c.scalar_type() == at::kBFloat16 || c.scalar_type() == at::kHalf), name, ": tensor ", i,
                  ": a working copy is bf16 or fp16, of an fp32 parameter");
      TORCH_CHECK(c.sizes() == p.sizes() && c.strides() == p.strides(), name, ": tensor ", i, ": the working copy must have the parameter's shape and strides");
      cd = dtype_of(c, name);
      d.copy = c.data_ptr();
      span_of(c, written[3]);
    }
    auto k = std::find_if(kinds.begin(), kinds.end(), [&](const Kind& q) { return q.p == pd && q.g == gd && q.c == cd; });
    if (k == kinds.end()) { kinds.push_back({pd, gd, cd, {}}); k = kinds.end() - 1; k->t.reserve(n); }
    k->t.push_back(d);
  }
  TORCH_CHECK(apart(written, read), name, ": a tensor that is written shares memory with another of the call (the same parameter twice?)");
  const Guard guard(on.device());
  hi3d_adamw_coefs_t c = {};
  c.beta1 = (float)beta1; c.one_minus_beta1 = (float)(1.0 - beta1); c.beta2 = (float)beta2; c.one_minus_beta2 = (float)(1.0 - beta2); c.eps = (float)eps;
  c.grad_scale = 1.0f;
  Tensor coefs;
  if (has(step_t)) {
    float* st = (float*)scalar_of(step_t, on, "hi3d::adamw_ step");
    coefs = at::empty({HI3D_ADAMW_COEFS}, on.options().dtype(at::kFloat).memory_format(c10::nullopt));
    const hi3d_adamw_rates rates = {lr, beta1, beta2, weight_decay};
    check_rc(hi3d_adamw_coefs(coefs.data_ptr<float>(), st, scalar_of(lr_t, on, "hi3d::adamw_ lr"), scalar_of(grad_scale, on, "hi3d::adamw_ grad_scale"),
                              scalar_of(found_inf, on, "hi3d::adamw_ found_inf"), &rates, stream_of(on)), "hi3d_adamw_coefs");
  } else {
    c.shrink = (float)(1.0 - lr * weight_decay);
    c.step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    c.inv_root = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  }
  for (const Kind& k : kinds)
    check_rc(hi3d_adamw_step(k.t.data(), (int)k.t.size(), k.p, k.g, k.c, &c, coefs.defined() ? coefs.data_ptr<float>() : nullptr, stream_of(on)), "hi3d_adamw_step");
  // a backward pass that saved these before the step has to see that they changed
  for (const at::TensorList& l : {params, copies})
    for (const Tensor& t : l)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(hi3d, m) {
  m.def("layernorm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("add_layernorm_fwd(Tensor x, Tensor residual, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("layernorm_bwd(Tensor dy, Tensor z, Tensor mean, Tensor rstd, Tensor? weight, Tensor? bias, Tensor? dz, bool need_dw=True, "
        "bool need_db=True) -> (Tensor, Tensor, Tensor)");
  m.def("linear_act(Tensor x, Tensor w, Tensor? bias, Tensor? residual, str act, bool save_z) -> (Tensor, Tensor)");
  m.def("linear_act_bwd(Tensor dy, Tensor x, Tensor w, Tensor? z, Tensor? bias, str act, bool need_dx, bool need_dw) -> (Tensor, Tensor, Tensor)");
  m.def("adamw_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_sq, Tensor(d!)[] copies, float lr, float beta1, "
        "float beta2, float eps, float weight_decay, int step, Tensor(e!)? step_t, Tensor? lr_t, Tensor? grad_scale, Tensor? found_inf) -> ()");
}

TORCH_LIBRARY_IMPL(hi3d, CUDA, m) {
  m.impl("layernorm_fwd", &layernorm_fwd);
  m.impl("add_layernorm_fwd", &add_layernorm_fwd);
  m.impl("layernorm_bwd", &layernorm_bwd);
  m.impl("linear_act", &linear_act);
  m.impl("linear_act_bwd", &linear_act_bwd);
  m.impl("adamw_", &adamw_);
}

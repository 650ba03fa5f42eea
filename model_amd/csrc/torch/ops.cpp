// The host path of layer_norm, vocab_cross_entropy and packed_attention
// (model_amd/layer_norm.py, cross_entropy.py and attention.py check the arguments
// and document them): output and workspace tensors, the calls into libmpl.so
// (include/mpl.h), and the autograd nodes; and of clip_global_norm
// (model_amd/grad_clip.py).  In C++ because a training step's small calls are bound
// by host time: torch runs backward nodes on a thread of its own, where a Python
// node of the first two took 40 to 80 us a call, several times its kernels.
//
// Host code only: built by the host compiler against torch's headers and linked
// to libmpl.so beside it.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/TracerMode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/util/ThreadLocalDebugInfo.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <functional>
#include <initializer_list>
#include <memory>
#include <numeric>
#include <optional>
#include <tuple>
#include <utility>
#include <vector>

#include "../../../include/mpl.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MPL_F32;
    case at::kHalf: return MPL_F16;
    case at::kBFloat16: return MPL_BF16;
    default: TORCH_CHECK(false, "unsupported dtype ", t.scalar_type());
  }
}

void check(int rc, const char* what) { TORCH_CHECK(rc == MPL_OK, what, " failed (code ", rc, "): ", mpl_last_error()); }

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

// The calls below read memory and launch kernels that no transform sees: a trace
// would record an empty output, and a tangent or a batch would be left out without
// a word.  `args` may hold undefined tensors.
void refuse_modes(const char* what) {
  using c10::DispatchKey;
  TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled(), what, " cannot be traced (torch.jit.trace)");
  TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode), what,
              " cannot be transformed by torch.func (vmap, grad, jvp, ...)");
  for (const auto mode : {c10::impl::TorchDispatchModeKey::PROXY, c10::impl::TorchDispatchModeKey::FAKE,
                          c10::impl::TorchDispatchModeKey::FUNCTIONAL})
    TORCH_CHECK(!c10::impl::TorchDispatchModeTLS::get_mode(mode).has_value(), what,
                " cannot be traced (make_fx, fake or functional tensors)");
}
void refuse_wrapped(const char* what, const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::FuncTorchBatched,
                                         DispatchKey::FuncTorchGradWrapper, DispatchKey::Batched,
                                         DispatchKey::Functionalize});
  TORCH_CHECK(!t.key_set().has_any(wrapped), what, " takes plain tensors, no wrappers or subclasses with their own dispatch");
  TORCH_CHECK(!t._fw_grad(0).defined(), what, " has no forward-mode derivative: an argument is a dual tensor");
}
void refuse_transforms(const char* what, std::initializer_list<Tensor> args) {
  refuse_modes(what);
  for (const Tensor& t : args)
    if (t.defined()) refuse_wrapped(what, t);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A captured backward of leaves that an eager graph holds ends the process, so
// the nodes refuse to run under capture.  `Pretended` makes one thread, and the
// backward passes that it starts (torch hands them the thread's debug information,
// on whichever thread they run), behave as under capture: for tests.
struct Pretended : c10::DebugInfoBase {};
constexpr auto kPretended = c10::DebugInfoKind::TEST_INFO;
bool capturing() {
  return dynamic_cast<Pretended*>(c10::ThreadLocalDebugInfo::get(kPretended)) != nullptr ||
         c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}
void pretend_capturing(bool on) {
  const bool now = dynamic_cast<Pretended*>(c10::ThreadLocalDebugInfo::get(kPretended)) != nullptr;
  if (on && !now) c10::ThreadLocalDebugInfo::_push(kPretended, std::make_shared<Pretended>());
  else if (!on && now) c10::ThreadLocalDebugInfo::_pop(kPretended);
}

// First derivatives only: what a node returns under create_graph raises when it
// is differentiated again.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once", 1);
    g = (*error)({g.detach().requires_grad_(true)})[0];
  }
  return grads;
}

// Contiguous, and what its memory says: torch marks some tensors as negated
// (the imaginary part of a conjugate) or as zeros without memory.
Tensor dense(const Tensor& t) {
  if (!t.defined()) return t;
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.resolve_neg().contiguous();
}

// Rows of d elements next to each other and the elements from row to row (at
// least d); copied only where they do not lie so.
struct Rows {
  Tensor t;
  int64_t pitch = 0;
  void* data() const { return t.defined() ? t.data_ptr() : nullptr; }
};
Rows rows_of(const Tensor& t, int64_t d) {
  if (!t.defined()) return {};
  if (t.is_neg() || t._is_zerotensor()) return {dense(t), d};
  if (t.is_contiguous()) return {t, d};
  Tensor r = t.reshape({-1, d});
  if ((d > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < d)) return {r.contiguous(), d};
  return {r, r.size(0) > 1 ? r.stride(0) : d};
}

// ------------------------------------------------------------- layer norm
// (y, sum or undefined, statistics [2, rows] or undefined)
std::tuple<Tensor, Tensor, Tensor> ln_forward(const Tensor& x, const Tensor& scale, const Tensor& bias, double eps,
                                              const Tensor& residual, bool stats) {
  const c10::DeviceGuard guard(x.device());
  const int64_t d = x.size(-1), rows = x.numel() / d;
  Tensor y = at::empty(x.sizes(), x.options()), total, st;
  if (residual.defined()) total = at::empty(x.sizes(), x.options());
  if (stats) st = at::empty({2, rows}, x.options().dtype(at::kFloat));
  if (rows) {
    const Rows a = rows_of(x, d), r = rows_of(residual, d);
    const Tensor w = dense(scale), b = dense(bias);
    float* mean = (float*)ptr(st);
    check(mpl_layer_norm(a.data(), a.pitch, r.data(), r.pitch, dtype_code(x), w.data_ptr(), b.data_ptr(), dtype_code(w),
                         rows, (int)d, (float)eps, y.data_ptr(), ptr(total), mean, mean ? mean + rows : nullptr,
                         stream_of(x)),
          "mpl_layer_norm");
  }
  return {y, total, st};
}

// (dx, d_scale, d_bias), undefined where not wanted
std::tuple<Tensor, Tensor, Tensor> ln_backward(const Tensor& g_y, const Tensor& s, const Tensor& scale,
                                               const float* mean, const float* rstd, const Tensor& g_residual,
                                               bool want_x, bool want_params) {
  const c10::DeviceGuard guard(s.device());
  const int64_t d = s.size(-1), rows = s.numel() / d;
  Tensor dx, ds, db;
  if (want_x) dx = at::empty(s.sizes(), s.options());
  if (want_params) {
    ds = rows ? at::empty({d}, scale.options()) : at::zeros({d}, scale.options());
    db = rows ? at::empty({d}, scale.options()) : at::zeros({d}, scale.options());
  }
  if (rows && (want_x || want_params)) {
    const Rows a = rows_of(s, d), g = rows_of(g_y, d), r = rows_of(g_residual, d);
    const Tensor w = dense(scale);
    const int code = dtype_code(s);
    const size_t n = want_params ? mpl_layer_norm_bwd_workspace_bytes(rows, (int)d, code) : 0;
    Tensor ws;
    if (n) ws = at::empty({(int64_t)n}, s.options().dtype(at::kByte));
    check(mpl_layer_norm_bwd(g.data(), g.pitch, a.data(), a.pitch, r.data(), r.pitch, code, w.data_ptr(), dtype_code(w),
                             mean, rstd, rows, (int)d, ptr(dx), ptr(ds), ptr(db), ptr(ws), n, stream_of(s)),
          "mpl_layer_norm_bwd");
  }
  return {dx, ds, db};
}

Tensor or_none(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& scale, const Tensor& bias, double eps,
                               const std::optional<Tensor>& residual) {
    auto [y, total, st] = ln_forward(x, scale, bias, eps, or_none(residual), true);
    ctx->save_for_backward({total.defined() ? total : x, scale, st});
    ctx->set_materialize_grads(false);
    if (total.defined()) return {y, total};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!capturing(), "torch autograd through layer_norm is not supported under HIP graph capture: use "
                "layer_norm_forward and layer_norm_backward, which capture");
    const bool added = grads.size() > 1;  // two outputs: there was a residual
    const bool nx = ctx->needs_input_grad(0), ns = ctx->needs_input_grad(1), nb = ctx->needs_input_grad(2),
               nr = added && ctx->needs_input_grad(3);
    const Tensor g_sum = added ? grads[1] : Tensor();
    refuse_transforms("layer_norm's gradient", {grads[0], g_sum});
    variable_list out(5);
    if (!grads[0].defined()) {  // only the sum was used
      if (nx) out[0] = g_sum;
      if (nr) out[4] = g_sum;
      return out;
    }
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &st = saved[2];
    {
      const at::AutoGradMode no_grad(false);
      const float* mean = (const float*)st.data_ptr();
      auto [dx, ds, db] = ln_backward(grads[0], s, saved[1], mean, mean + st.size(1), g_sum, nx || nr, ns || nb);
      if (nx) out[0] = dx;
      if (ns) out[1] = ds;
      if (nb) out[2] = db;
      if (nr) out[4] = dx;
    }
    return once(std::move(out), "layer_norm");
  }
};

py::object layer_norm(const Tensor& x, const Tensor& scale, const Tensor& bias, double eps,
                      const std::optional<Tensor>& residual, bool autograd) {
  const Tensor r = or_none(residual);
  refuse_transforms("layer_norm", {x, scale, bias, r});
  if (autograd) {
    const variable_list out = LayerNormFunction::apply(x, scale, bias, eps, residual);
    return r.defined() ? py::cast(std::make_tuple(out[0], out[1])) : py::cast(out[0]);
  }
  auto [y, total, st] = ln_forward(x, scale, bias, eps, r, false);
  return r.defined() ? py::cast(std::make_tuple(y, total)) : py::cast(y);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm_forward(const Tensor& x, const Tensor& scale, const Tensor& bias,
                                                              double eps, const std::optional<Tensor>& residual) {
  refuse_transforms("layer_norm_forward", {x, scale, bias, or_none(residual)});
  const at::AutoGradMode no_grad(false);
  auto [y, total, st] = ln_forward(x, scale, bias, eps, or_none(residual), true);
  return {y, total.defined() ? total : x, st.select(0, 0), st.select(0, 1)};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& g_y, const Tensor& s, const Tensor& scale,
                                                       const Tensor& mean, const Tensor& rstd,
                                                       const std::optional<Tensor>& g_residual) {
  refuse_transforms("layer_norm_backward", {g_y, s, scale, mean, rstd, or_none(g_residual)});
  const at::AutoGradMode no_grad(false);
  const Tensor m = dense(mean), r = dense(rstd);
  return ln_backward(g_y, s, scale, (const float*)m.data_ptr(), (const float*)r.data_ptr(), or_none(g_residual), true,
                     true);
}

// ---------------------------------------------------------- cross entropy
// 16-bit rows that the tiles read as they lie (d a multiple of 64) start at 16
// bytes and are less than 2^23 elements apart.
Rows operand_of(const Tensor& t, int64_t d) {
  Rows r = rows_of(t, d);
  if (t.scalar_type() != at::kFloat && d % 64 == 0 && ((uintptr_t)r.data() % 16 || r.pitch % 8 || r.pitch >= (1 << 23)))
    return {r.t.clone(at::MemoryFormat::Contiguous), d};
  return r;
}

Tensor workspace(int64_t rows, int64_t vocab, int64_t d, const Tensor& like, bool backward) {
  const size_t n = mpl_vocab_cross_entropy_workspace_bytes(rows, vocab, (int)d, dtype_code(like), backward);
  TORCH_CHECK_VALUE(n, "vocab_cross_entropy: ", rows, " rows, a vocabulary of ", vocab, " and a width of ", d,
                    " are out of range");
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

Tensor ids_of(const Tensor& targets) { return targets.to(at::kLong).contiguous(); }

std::tuple<Tensor, Tensor> ce_forward(const Tensor& hidden, const Tensor& embedding, const Tensor& ids,
                                      int64_t ignore_index) {
  const c10::DeviceGuard guard(hidden.device());
  const int64_t V = embedding.size(0), d = embedding.size(1), R = ids.numel();
  const auto f32 = hidden.options().dtype(at::kFloat);
  Tensor loss = at::empty(ids.sizes(), f32), lse = at::empty(ids.sizes(), f32);
  if (R) {
    const Rows h = operand_of(hidden, d), e = operand_of(embedding, d);
    const Tensor ws = workspace(R, V, d, hidden, false);
    check(mpl_vocab_cross_entropy(h.data(), h.pitch, e.data(), e.pitch, dtype_code(hidden), (const int64_t*)ids.data_ptr(),
                                  R, V, (int)d, ignore_index, ws.data_ptr(), ws.numel(), (float*)loss.data_ptr(),
                                  (float*)lse.data_ptr(), stream_of(hidden)),
          "mpl_vocab_cross_entropy");
  }
  return {loss, lse};
}

std::tuple<Tensor, Tensor> ce_backward(const Tensor& hidden, const Tensor& embedding, const Tensor& ids,
                                       int64_t ignore_index, const Tensor& lse, const Tensor& g_loss,
                                       const Tensor& g_lse, bool want_h, bool want_e) {
  const c10::DeviceGuard guard(hidden.device());
  const int64_t V = embedding.size(0), d = embedding.size(1), R = ids.numel();
  Tensor dh, de;
  if (want_h) dh = at::empty(hidden.sizes(), hidden.options());
  if (want_e) de = R ? at::empty({V, d}, hidden.options()) : at::zeros({V, d}, hidden.options());
  if (R && (want_h || want_e)) {
    auto row_grad = [](const Tensor& g) { return g.defined() ? dense(g.to(at::kFloat)) : g; };
    const Tensor gl = row_grad(g_loss), gs = row_grad(g_lse);
    const Rows h = operand_of(hidden, d), e = operand_of(embedding, d);
    const Tensor ws = workspace(R, V, d, hidden, true);
    check(mpl_vocab_cross_entropy_bwd(h.data(), h.pitch, e.data(), e.pitch, dtype_code(hidden),
                                      (const int64_t*)ids.data_ptr(), R, V, (int)d, ignore_index,
                                      (const float*)lse.data_ptr(), (const float*)ptr(gl), (const float*)ptr(gs),
                                      ws.data_ptr(), ws.numel(), ptr(dh), ptr(de), stream_of(hidden)),
          "mpl_vocab_cross_entropy_bwd");
  }
  return {dh, de};
}

struct CrossEntropyFunction : torch::autograd::Function<CrossEntropyFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& embedding, const Tensor& ids,
                               int64_t ignore_index) {
    auto [loss, lse] = ce_forward(hidden, embedding, ids, ignore_index);
    ctx->save_for_backward({hidden, embedding, ids, lse});
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->set_materialize_grads(false);
    return {loss, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!capturing(), "torch autograd through vocab_cross_entropy is not supported under HIP graph capture: use "
                "vocab_cross_entropy_grads, which captures");
    variable_list out(4);
    refuse_transforms("vocab_cross_entropy's gradient", {grads[0], grads[1]});
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    {
      const at::AutoGradMode no_grad(false);
      std::tie(out[0], out[1]) =
          ce_backward(s[0], s[1], s[2], ctx->saved_data["ignore_index"].toInt(), s[3], grads[0], grads[1],
                      ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    }
    return once(std::move(out), "vocab_cross_entropy");
  }
};

std::tuple<Tensor, Tensor> vocab_cross_entropy(const Tensor& hidden, const Tensor& embedding, const Tensor& targets,
                                               int64_t ignore_index, bool autograd) {
  refuse_transforms("vocab_cross_entropy", {hidden, embedding, targets});
  const Tensor ids = ids_of(targets);
  if (!autograd) return ce_forward(hidden, embedding, ids, ignore_index);
  const variable_list out = CrossEntropyFunction::apply(hidden, embedding, ids, ignore_index);
  return {out[0], out[1]};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> vocab_cross_entropy_grads(const Tensor& hidden, const Tensor& embedding,
                                                                     const Tensor& targets,
                                                                     const std::optional<Tensor>& g_loss,
                                                                     const std::optional<Tensor>& g_lse,
                                                                     int64_t ignore_index) {
  refuse_transforms("vocab_cross_entropy_grads", {hidden, embedding, targets, or_none(g_loss), or_none(g_lse)});
  const at::AutoGradMode no_grad(false);
  const Tensor ids = ids_of(targets);
  auto [loss, lse] = ce_forward(hidden, embedding, ids, ignore_index);
  auto [dh, de] = ce_backward(hidden, embedding, ids, ignore_index, lse, or_none(g_loss), or_none(g_lse), true, true);
  return {loss, lse, dh, de};
}

// ------------------------------------------------------- packed attention
// [tokens, heads, hd] with hd elements next to each other, rows at 16 bytes and not
// too far apart (mpl.h); copied only where they do not lie so.
struct Heads {
  Tensor t;
  int64_t token = 0, head = 0;
};
Heads heads_of(const Tensor& x, bool shared = false) {  // shared: k and v
  Tensor t = x._is_zerotensor() ? dense(x) : x.resolve_neg();
  const int64_t unit = 16 / t.element_size();
  constexpr int64_t kFar = 1 << 23;
  auto lies = [&](const Tensor& y) {
    return y.numel() == 0 ||
           (y.stride(2) == 1 && (uintptr_t)y.data_ptr() % 16 == 0 &&
            (y.size(0) == 1 || (y.stride(0) % unit == 0 && y.stride(0) <= kFar)) &&
            (y.size(1) == 1 || (y.stride(1) % unit == 0 &&
                                (shared || y.stride(1) * std::max<int64_t>(32, y.size(1)) <= 32 * kFar))));
  };
  if (!lies(t)) t = t.clone(at::MemoryFormat::Contiguous);
  if (t.numel() == 0) return {t, 0, 0};
  return {t, t.size(0) == 1 ? 0 : t.stride(0), t.size(1) == 1 ? 0 : t.stride(1)};
}

// The arguments of a call, and the tensors that they point into.
struct PackedCall {
  mpl_packed_attention_args a;
  Heads q, k, v;
  Tensor starts, key_starts, key_lengths;
  PackedCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& starts_, const Tensor& key_starts_,
             const Tensor& key_lengths_, double scale)
      : q(heads_of(q_)), k(heads_of(k_, true)), v(heads_of(v_, true)), starts(dense(starts_)), key_starts(dense(key_starts_)),
        key_lengths(dense(key_lengths_)) {
    a.q = ptr(q.t); a.k = ptr(k.t); a.v = ptr(v.t);
    a.q_token = q.token; a.q_head = q.head;
    a.k_token = k.token; a.k_head = k.head;
    a.v_token = v.token; a.v_head = v.head;
    a.dtype = dtype_code(q_);
    a.heads = (int)q_.size(1); a.groups = (int)k_.size(1); a.head_dim = (int)q_.size(2);
    a.tokens = q_.size(0); a.keys = k_.size(0); a.sequences = starts.numel() - 1;
    a.starts = ptr(starts);
    a.key_starts = key_starts.defined() ? ptr(key_starts) : ptr(starts);
    a.key_lengths = ptr(key_lengths);
    a.index_bytes = (int)starts.element_size();
    a.scale = (float)scale;
  }
  Tensor workspace(bool backward) const {
    const size_t n = mpl_packed_attention_workspace_bytes(&a, backward);
    TORCH_CHECK_VALUE(n, "packed_attention: ", mpl_last_error());
    return at::empty({(int64_t)n}, q.t.options().dtype(at::kByte));
  }
};

std::tuple<Tensor, Tensor> pa_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts,
                                      const Tensor& key_starts, const Tensor& key_lengths, double scale, bool want_lse) {
  const c10::DeviceGuard guard(q.device());
  const PackedCall c(q, k, v, starts, key_starts, key_lengths, scale);
  Tensor out = at::empty(q.sizes(), q.options()), lse;
  if (want_lse) lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  if (q.size(0)) {
    const Tensor ws = c.workspace(false);
    check(mpl_packed_attention(&c.a, ws.data_ptr(), ws.numel(), out.data_ptr(), (float*)ptr(lse), stream_of(q)),
          "mpl_packed_attention");
  }
  return {out, lse};
}

// (dq, dk, dv), undefined where not wanted
std::tuple<Tensor, Tensor, Tensor> pa_backward(const Tensor& g_out, const Tensor& g_lse, const Tensor& q, const Tensor& k,
                                               const Tensor& v, const Tensor& out, const Tensor& lse, const Tensor& starts,
                                               const Tensor& key_starts, const Tensor& key_lengths, double scale,
                                               bool want_q, bool want_k, bool want_v) {
  const c10::DeviceGuard guard(q.device());
  Tensor dq, dk, dv;
  if (want_q) dq = at::empty(q.sizes(), q.options());
  if (want_k) dk = at::empty(k.sizes(), k.options());
  if (want_v) dv = at::empty(v.sizes(), v.options());
  if ((q.size(0) || k.size(0)) && (want_q || want_k || want_v)) {
    const PackedCall c(q, k, v, starts, key_starts, key_lengths, scale);
    const Heads g = heads_of(g_out.defined() ? g_out : at::zeros(q.sizes(), q.options()));
    const Tensor o = heads_of(out.contiguous()).t, l = dense(lse);
    const Tensor gl = g_lse.defined() ? dense(g_lse.to(at::kFloat)) : g_lse;
    const Tensor ws = c.workspace(true);
    check(mpl_packed_attention_bwd(&c.a, ptr(g.t), g.token, g.head, ptr(o), (const float*)ptr(l), (const float*)ptr(gl),
                                   ws.data_ptr(), ws.numel(), ptr(dq), ptr(dk), ptr(dv), stream_of(q)),
          "mpl_packed_attention_bwd");
  }
  return {dq, dk, dv};
}

struct PackedAttentionFunction : torch::autograd::Function<PackedAttentionFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& starts, const std::optional<Tensor>& key_starts,
                               const std::optional<Tensor>& key_lengths, double scale) {
    auto [out, lse] = pa_forward(q, k, v, starts, or_none(key_starts), or_none(key_lengths), scale, true);
    ctx->save_for_backward({q, k, v, out, lse, starts, or_none(key_starts), or_none(key_lengths)});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!capturing(), "torch autograd through packed_attention is not supported under HIP graph capture: use "
                "packed_attention_forward and packed_attention_backward, which capture");
    variable_list out(7);
    refuse_transforms("packed_attention's gradient", {grads[0], grads[1]});
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    {
      const at::AutoGradMode no_grad(false);
      std::tie(out[0], out[1], out[2]) =
          pa_backward(grads[0], grads[1], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7],
                      ctx->saved_data["scale"].toDouble(), ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                      ctx->needs_input_grad(2));
    }
    return once(std::move(out), "packed_attention");
  }
};

// (out, lse or none)
std::tuple<Tensor, std::optional<Tensor>> packed_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                                           const Tensor& starts, const std::optional<Tensor>& key_starts,
                                                           const std::optional<Tensor>& key_lengths, double scale,
                                                           bool want_lse, bool autograd) {
  refuse_transforms("packed_attention", {q, k, v, starts, or_none(key_starts), or_none(key_lengths)});
  if (autograd) {
    const variable_list out = PackedAttentionFunction::apply(q, k, v, starts, key_starts, key_lengths, scale);
    return {out[0], want_lse ? std::optional<Tensor>(out[1]) : std::nullopt};
  }
  const at::AutoGradMode no_grad(false);
  auto [out, lse] = pa_forward(q, k, v, starts, or_none(key_starts), or_none(key_lengths), scale, want_lse);
  return {out, want_lse ? std::optional<Tensor>(lse) : std::nullopt};
}

std::tuple<Tensor, Tensor, Tensor> packed_attention_backward(const Tensor& g_out, const Tensor& q, const Tensor& k,
                                                             const Tensor& v, const Tensor& out, const Tensor& lse,
                                                             const Tensor& starts, const std::optional<Tensor>& key_starts,
                                                             const std::optional<Tensor>& key_lengths, double scale,
                                                             const std::optional<Tensor>& g_lse) {
  refuse_transforms("packed_attention_backward",
                    {g_out, q, k, v, out, lse, starts, or_none(key_starts), or_none(key_lengths), or_none(g_lse)});
  const at::AutoGradMode no_grad(false);
  return pa_backward(g_out, or_none(g_lse), q, k, v, out, lse, starts, or_none(key_starts), or_none(key_lengths), scale,
                     true, true, true);
}

// --------------------------------------------------------------- gradient clip
// The bytes from a tensor's first element to behind its last; `whole`: it takes them all.
struct Span {
  char *first, *end;
  const Tensor* t;
  bool whole;
};

// Whether two tensors have a byte in common.  With steps i and j along their axes and x
// and y within an element it is one equation, sum i s - sum j t + x - y = distance; axes of
// one stride become one unknown, and the unknowns are tried from the largest stride on as
// far as the others' sum can still make up the rest.  Views of one matrix have one or two
// values left for each; a search that does not end within kMostSteps finds nothing.
struct Meeting {
  struct Unknown {
    int64_t stride, lo, hi;  // its steps
    int64_t least, most;     // of the sum of the unknowns behind it
    int64_t divisor;         // of its stride and theirs
  };
  std::vector<Unknown> of;
  int64_t x_lo, x_hi;
  int steps = 0;
  static constexpr int kMostSteps = 100000;

  void axes(const Span& s, int sign) {
    const int64_t size = s.t->element_size();
    auto add = [&](int64_t stride, int64_t n) {
      if (n <= 1) return;
      auto at = std::find_if(of.begin(), of.end(), [&](const Unknown& u) { return u.stride == stride; });
      if (at == of.end()) at = of.insert(of.end(), Unknown{stride, 0, 0, 0, 0, 1});
      (sign > 0 ? at->hi : at->lo) += sign * (n - 1);
    };
    if (s.whole) return add(size, s.t->numel());
    for (int64_t d = 0; d < s.t->dim(); ++d) add(s.t->stride(d) * size, s.t->size(d));
  }
  bool from(size_t k, int64_t rest) {
    if (++steps > kMostSteps) return false;
    if (k == of.size()) return rest >= x_lo && rest <= x_hi;
    const Unknown& u = of[k];
    if (floor_div(rest - x_lo, u.divisor) * u.divisor < rest - x_hi) return false;  // no x - y leaves a multiple
    const int64_t lo = std::max(u.lo, -floor_div(u.most - rest, u.stride));
    const int64_t hi = std::min(u.hi, floor_div(rest - u.least, u.stride));
    for (int64_t i = lo; i <= hi && steps <= kMostSteps; ++i)
      if (from(k + 1, rest - i * u.stride)) return true;
    return false;
  }
  static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
  bool found(const Span& a, const Span& b) {
    axes(a, 1);
    axes(b, -1);
    x_lo = 1 - (int64_t)b.t->element_size();
    x_hi = (int64_t)a.t->element_size() - 1;
    std::sort(of.begin(), of.end(), [](const Unknown& p, const Unknown& q) { return p.stride > q.stride; });
    int64_t least = x_lo, most = x_hi, divisor = 0;
    for (size_t k = of.size(); k--;) {
      of[k].least = least;
      of[k].most = most;
      of[k].divisor = divisor = std::gcd(divisor, of[k].stride);
      least += of[k].lo * of[k].stride;
      most += of[k].hi * of[k].stride;
    }
    const int64_t rest = b.first - a.first;
    return rest >= least && rest <= most && from(0, rest);
  }
};

// `list` holds its tensors while the call runs: references, no copies of a thousand handles.
Tensor clip_grads(const py::list& list, double grad_clip, const std::optional<Tensor>& row_sq, bool apply,
                  const char* what) {
  std::vector<std::reference_wrapper<const Tensor>> grads;
  grads.reserve(list.size());
  for (const py::handle o : list) {
    TORCH_CHECK_TYPE(THPVariable_Check(o.ptr()), what, ": gradient ", grads.size(), " is no tensor");
    grads.emplace_back(THPVariable_Unpack(o.ptr()));
  }
  const Tensor rows = or_none(row_sq);
  TORCH_CHECK_VALUE(!grads.empty() || rows.defined(), what, ": no gradients");
  TORCH_CHECK_VALUE(grad_clip >= 0, what, ": grad_clip ", grad_clip, " must not be negative");
  refuse_modes(what);
  const auto device = (grads.empty() ? rows : grads[0].get()).device();
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& t = grads[i];
    refuse_wrapped(what, t);
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf ||
                                                     t.scalar_type() == at::kBFloat16),
                      what, ": gradient ", i, " must be a dense float32, float16 or bfloat16 tensor, got ", t.scalar_type(),
                      " ", t.layout());
    TORCH_CHECK_VALUE(t.device() == device, what, ": gradient ", i, " on ", t.device(), ", others on ", device);
    if (apply) {
      TORCH_CHECK_VALUE(!(t.requires_grad() && at::GradMode::is_enabled()), what, ": gradient ", i,
                        " requires grad itself: it cannot be scaled in place outside torch.no_grad()");
      TORCH_CHECK_VALUE(at::has_internal_overlap(t) != at::MemOverlap::Yes, what, ": gradient ", i,
                        " is expanded: its elements share memory");
    }
  }
  if (rows.defined()) {
    refuse_wrapped(what, rows);
    TORCH_CHECK_VALUE(rows.scalar_type() == at::kFloat && rows.layout() == at::kStrided && rows.device() == device, what,
                      ": row_sq must be a dense float32 tensor on ", device);
  }
  TORCH_CHECK_VALUE(device.is_cuda(), what, " runs on the GPU only (libmpl.so), gradients are on ", device);
  const at::AutoGradMode no_grad(false);
  const c10::DeviceGuard guard(device);
  std::vector<Tensor> held;                        // copies of what does not lie in one piece
  std::vector<std::pair<Tensor, Tensor>> back;     // and where they go
  std::vector<void*> x;
  std::vector<int64_t> n;
  std::vector<int> types;
  std::vector<Span> spans;
  n.reserve(grads.size());
  x.reserve(grads.size());
  types.reserve(grads.size());
  spans.reserve(grads.size());
  for (const Tensor& t : grads) {
    const int64_t m = t.numel();
    if (m == 0 || t._is_zerotensor()) continue;  // add nothing, and are scaled by being what they are
    char* at = (char*)t.data_ptr();
    const bool whole = t.is_non_overlapping_and_dense();
    if (apply) {
      int64_t last = m - 1;
      if (!whole) {
        last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
      }
      spans.push_back({at, at + (last + 1) * t.element_size(), &t, whole});
    }
    if (t.is_neg() || !whole) {
      held.push_back(dense(t));
      at = (char*)held.back().data_ptr();
      if (apply) back.emplace_back(t, held.back());
    }
    x.push_back(at);
    n.push_back(m);
    types.push_back(dtype_code(t));
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.first < b.first; });
  std::vector<const Span*> open;  // those that reach to where the next begins
  for (const Span& b : spans) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Span* a) { return a->end <= b.first; }), open.end());
    for (const Span* a : open)
      TORCH_CHECK_VALUE(!(a->whole && b.whole) && !Meeting().found(*a, b), what, ": two of the gradients share memory");
    open.push_back(&b);
  }
  const auto opt = at::TensorOptions().device(device);
  Tensor out = at::empty({2}, opt.dtype(at::kFloat));
  const Tensor r = dense(rows);
  const size_t bytes = mpl_clip_grads_workspace_bytes((int64_t)x.size());
  TORCH_CHECK_VALUE(bytes, what, ": too many gradients");
  const Tensor ws = at::empty({(int64_t)bytes}, opt.dtype(at::kByte));
  check(mpl_clip_grads(x.data(), n.data(), types.data(), (int64_t)x.size(), (const float*)ptr(r), r.defined() ? r.numel() : 0,
                       (float)grad_clip, apply, (float*)out.data_ptr(), ws.data_ptr(), bytes, stream_of(out)),
        "mpl_clip_grads");
  for (auto& [to, from] : back) to.copy_(from);
  if (apply)
    for (const Tensor& t : grads)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return out;
}

Tensor clip_global_norm(const py::list& grads, double grad_clip, const std::optional<Tensor>& row_sq) {
  return clip_grads(grads, grad_clip, row_sq, true, "clip_global_norm");
}
Tensor global_norm_scale(const py::list& grads, double grad_clip, const std::optional<Tensor>& row_sq) {
  return clip_grads(grads, grad_clip, row_sq, false, "global_norm_scale");
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("vocab_cross_entropy", &vocab_cross_entropy);
  m.def("vocab_cross_entropy_grads", &vocab_cross_entropy_grads);
  m.def("packed_attention", &packed_attention);
  m.def("packed_attention_backward", &packed_attention_backward);
  m.def("clip_global_norm", &clip_global_norm);
  m.def("global_norm_scale", &global_norm_scale);
  m.def("pretend_capturing", &pretend_capturing);
}

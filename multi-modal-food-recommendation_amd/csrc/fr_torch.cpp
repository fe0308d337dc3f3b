// torch binding of the sequence operators (engine/seq_ops.py): argument checks, allocation and autograd
// nodes in C++ around the C-ABI entry points of fr_engine.h.
//
// These operators are called one by one on small batches, where the time of a call is the host's: a
// 512 x 64 dropout with its gradient takes 47 us through this binding and 74 us through a Python
// autograd function over ctypes, of which 38 us are the autograd engine's own.  The C entry points
// are called by address (bind()), so they are those of the one library that engine/native.py loaded.
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <map>
#include <optional>
#include <sstream>
#include <string>

#include "fr_engine.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

struct EngineError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject* g_error = nullptr;  // FoodRec.engine.native.EngineError

template <typename... A>
[[noreturn]] void fail(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw EngineError(s.str());
}

// the C entry points, by the names of fr_engine.h
struct Entries {
  decltype(&::fr_last_error) last_error;
  decltype(&::fr_embedding_scaled_fwd) embedding_scaled_fwd;
  decltype(&::fr_embedding_scaled_bwd_workspace) embedding_scaled_bwd_workspace;
  decltype(&::fr_embedding_scaled_bwd) embedding_scaled_bwd;
  decltype(&::fr_dropout) dropout;
  decltype(&::fr_rms_norm_fwd) rms_norm_fwd;
  decltype(&::fr_rms_norm_bwd_workspace) rms_norm_bwd_workspace;
  decltype(&::fr_rms_norm_bwd) rms_norm_bwd;
  decltype(&::fr_item_logp_fwd_workspace) item_logp_fwd_workspace;
  decltype(&::fr_item_logp_fwd) item_logp_fwd;
  decltype(&::fr_item_logp_bwd_workspace) item_logp_bwd_workspace;
  decltype(&::fr_item_logp_bwd) item_logp_bwd;
  decltype(&::fr_preference_loss) preference_loss;
} g_fr;

void bind(const std::map<std::string, uintptr_t>& at, py::object error) {
  g_error = error.inc_ref().ptr();  // kept for the life of the process
#define FR_BIND(name) g_fr.name = reinterpret_cast<decltype(g_fr.name)>(at.at("fr_" #name))
  FR_BIND(last_error);
  FR_BIND(embedding_scaled_fwd);
  FR_BIND(embedding_scaled_bwd_workspace);
  FR_BIND(embedding_scaled_bwd);
  FR_BIND(dropout);
  FR_BIND(rms_norm_fwd);
  FR_BIND(rms_norm_bwd_workspace);
  FR_BIND(rms_norm_bwd);
  FR_BIND(item_logp_fwd_workspace);
  FR_BIND(item_logp_fwd);
  FR_BIND(item_logp_bwd_workspace);
  FR_BIND(item_logp_bwd);
  FR_BIND(preference_loss);
#undef FR_BIND
}

void done(int rc, const char* what) {
  if (rc != FR_OK) fail(what, " failed: ", g_fr.last_error());
}

// ---------------------------------------------------------------------------------- checks, layouts
void on_gpu(const Tensor& t) {
  if (!t.is_cuda())
    fail("FoodRec MI355X engine ops need tensors on a ROCm GPU device (got a tensor on ", t.device(),
         "); there is no CPU path");
}

// What a direct call of a kernel would lose in silence is refused: a tangent of forward-mode differentiation, and the
// call itself in a trace, which would hold the allocation of its result alone.
void plain_call(const char* name, const Tensor& t) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    fail(name, ": engine operators have no forward-mode derivative");
  if (torch::jit::tracer::isTracing()) fail(name, ": engine operators cannot be traced");
  if (!t.has_storage()) fail(name, ": a dense tensor required (no sparse one, and none of torch.func's transforms)");
}

// the tensors on one GPU, the first in a supported type
template <typename... O>
void check(const char* name, const Tensor& t, const O&... others) {
  const auto plain = [&](const Tensor& o) { plain_call(name, o); };
  const auto same = [&](const Tensor& o) {
    on_gpu(o);
    if (o.device() != t.device()) fail(name, ": tensors on ", t.device(), " and ", o.device());
  };
  const auto each = [&](const auto& o, const auto& f) {
    if constexpr (std::is_same_v<std::decay_t<decltype(o)>, MaybeTensor>) {
      if (o) f(*o);
    } else {
      f(o);
    }
  };
  plain(t);
  (each(others, plain), ...);
  on_gpu(t);
  (each(others, same), ...);
  if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16)
    fail(name, ": fp32 or bf16 tensors required (got ", t.scalar_type(), ")");
}

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? FR_F32 : FR_BF16; }

Tensor ids_of(const char* name, const Tensor& idx) {
  if (idx.scalar_type() != at::kLong && idx.scalar_type() != at::kInt)
    fail(name, ": int64 or int32 ids required (got ", idx.scalar_type(), ")");
  return idx.to(at::kLong).contiguous();
}

// [..., d] as [rows, d] with unit stride inside a row (a view where the strides allow it)
Tensor rows2d(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1))) r = r.contiguous();
  return r;
}

int64_t ld_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const MaybeTensor& t) { return t && t->requires_grad(); }
template <typename... A>
bool recording(const A&... a) {
  return at::GradMode::is_enabled() && (wants_grad(a) || ...);
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* data(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }
const int64_t* longs(const Tensor& t) { return static_cast<const int64_t*>(t.data_ptr()); }
float* floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor workspace(int64_t bytes, const Tensor& like) {
  return at::empty({std::max<int64_t>(bytes, 16)}, like.options().dtype(at::kByte));
}

// A backward's results when the backward itself is recorded (create_graph): usable, but an error where a
// second derivative is asked for, as torch's once_differentiable has it.
variable_list once(const variable_list& grads, variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  bool any = false;
  for (const Tensor& g : grads) any |= g.defined() && g.requires_grad();
  if (!any) return out;
  variable_list marked;
  for (Tensor& o : out) marked.push_back(o.defined() ? o.detach().requires_grad_() : o);
  return torch::autograd::DelayedError("trying to differentiate twice an engine operator that is differentiable once",
                                       (int64_t)out.size())
      .apply(std::move(marked));
}

// ---------------------------------------------------------------------------------- scaled embedding
Tensor embedding_fwd(const Tensor& idx, const Tensor& w, double scale) {
  auto size = idx.sizes().vec();
  size.push_back(w.size(1));
  Tensor out = at::empty(size, w.options());
  if (idx.numel()) {
    c10::DeviceGuard guard(w.device());
    done(g_fr.embedding_scaled_fwd(longs(idx), idx.numel(), data(w), ld_of(w), w.size(0), (int)w.size(1), dtype_of(w),
                                   (float)scale, data(out), stream_of(w)),
         "fr_embedding_scaled_fwd");
  }
  return out;
}

struct EmbeddingScaled : torch::autograd::Function<EmbeddingScaled> {
  static Tensor forward(AutogradContext* ctx, const Tensor& idx, const Tensor& w, double scale, int64_t pad) {
    ctx->save_for_backward({idx});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["rows"] = w.size(0);
    return embedding_fwd(idx, w, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor idx = ctx->get_saved_variables()[0], g = rows2d(grads[0]);
    const int64_t rows = ctx->saved_data["rows"].toInt(), d = g.size(1), n = idx.numel();
    c10::DeviceGuard guard(g.device());
    Tensor dw = at::empty({rows, d}, g.options());
    Tensor ws = workspace(g_fr.embedding_scaled_bwd_workspace(n, rows, (int)d), g);
    done(g_fr.embedding_scaled_bwd(longs(idx), n, data(g), ld_of(g), rows, (int)d, dtype_of(g),
                                   (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["pad"].toInt(), data(dw),
                                   data(ws), ws.numel(), stream_of(g)),
         "fr_embedding_scaled_bwd");
    return once(grads, {Tensor(), dw, Tensor(), Tensor()});
  }
};

Tensor embedding_scaled(const Tensor& idx, const Tensor& weight, double scale, std::optional<int64_t> padding_idx) {
  const char* name = "embedding_scaled";
  check(name, weight, idx);
  if (weight.dim() != 2 || weight.size(1) < 1 || weight.size(1) > 16384 || weight.size(0) < 1 ||
      weight.size(0) >= INT32_MAX)
    fail(name, ": unsupported table shape ", weight.sizes());
  if (idx.numel() > INT32_MAX) fail(name, ": ", idx.numel(), " ids, fewer than 2^31 required");
  const Tensor ids = ids_of(name, idx), w = rows2d(weight);
  int64_t pad = -1;
  if (padding_idx) {
    pad = *padding_idx < 0 ? *padding_idx + weight.size(0) : *padding_idx;
    if (pad < 0 || pad >= weight.size(0)) fail(name, ": padding_idx ", *padding_idx, " outside the table");
  }
  return recording(w) ? EmbeddingScaled::apply(ids, w, scale, pad) : embedding_fwd(ids, w, scale);
}

// ---------------------------------------------------------------------------------- dropout
Tensor dropout_run(const Tensor& x, const MaybeTensor& residual, double p, uint64_t seed, const Tensor& step,
                   const Tensor& used) {
  Tensor y = at::empty_like(x);
  c10::DeviceGuard guard(x.device());
  done(g_fr.dropout(data(x), data(residual), data(y), x.numel(), dtype_of(x), p, seed, longs(step),
                    static_cast<int64_t*>(data(used)), stream_of(x)),
       "fr_dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, double p, int64_t seed,
                        const Tensor& counter) {
    Tensor used = at::empty_like(counter);  // the step's value, written by the kernel
    ctx->save_for_backward({used});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["residual"] = residual.has_value();
    return dropout_run(x, residual, p, (uint64_t)seed, counter, used);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dx;
    if (ctx->needs_input_grad(0))
      dx = dropout_run(grads[0].contiguous(), std::nullopt, ctx->saved_data["p"].toDouble(),
                       (uint64_t)ctx->saved_data["seed"].toInt(), ctx->get_saved_variables()[0], Tensor());
    const bool residual = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
    return once(grads, {dx, residual ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, const Tensor& counter, const MaybeTensor& residual) {
  const char* name = "dropout";
  check(name, x, counter, residual);
  if (!(p >= 0.0 && p <= 1.0)) fail(name, ": p = ", p, " outside [0, 1]");
  if (counter.scalar_type() != at::kLong || counter.numel() != 1)
    fail(name, ": the counter is an int64 tensor of one element");
  if (residual && (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type()))
    fail(name, ": residual ", residual->sizes(), " ", residual->scalar_type(), " differs from x ", x.sizes(), " ",
         x.scalar_type());
  const Tensor xc = x.contiguous();
  MaybeTensor rc;
  if (residual) rc = residual->contiguous();
  return recording(xc, rc) ? Dropout::apply(xc, rc, p, (int64_t)seed, counter)
                           : dropout_run(xc, rc, p, seed, counter, Tensor());
}

// ---------------------------------------------------------------------------------- RMS norm
struct Normed {
  Tensor y, scale, h, rstd;
};

Normed norm_run(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight, double eps, bool quant,
                bool want_rstd) {
  const Tensor x2 = rows2d(x);
  Tensor r2;
  const int64_t rows = x2.size(0);
  Normed o;
  o.y = at::empty(x.sizes(), quant ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  if (residual) {
    r2 = rows2d(*residual);
    o.h = at::empty(x.sizes(), x.options());
  }
  const auto f32 = x.options().dtype(at::kFloat);
  if (quant) o.scale = at::empty(x.sizes().slice(0, x.dim() - 1), f32);
  if (want_rstd) o.rstd = at::empty({rows}, f32);
  if (rows) {
    c10::DeviceGuard guard(x.device());
    done(g_fr.rms_norm_fwd(data(x2), ld_of(x2), data(r2), residual ? ld_of(r2) : 0, rows, (int)x2.size(1), dtype_of(x),
                           data(weight), dtype_of(weight ? *weight : x), (float)eps, data(o.y), quant, floats(o.scale),
                           data(o.h), floats(o.rstd), stream_of(x)),
         "fr_rms_norm_fwd");
  }
  return o;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual,
                               const MaybeTensor& weight, double eps) {
    Normed o = norm_run(x, residual, weight, eps, false, true);
    ctx->set_materialize_grads(false);
    // fp32: the stored h is the forward's; bf16: x and the residual, whose sum is not rounded yet
    const bool stored = residual && x.scalar_type() == at::kFloat;
    ctx->save_for_backward({stored ? o.h : x, residual && !stored ? *residual : Tensor(), weight ? *weight : Tensor(),
                            o.rstd});
    ctx->saved_data["residual"] = residual.has_value();
    if (!residual) return {o.y};
    return {o.y, o.h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &r = saved[1], &weight = saved[2], &rstd = saved[3];
    const bool residual = ctx->saved_data["residual"].toBool();
    // the inputs' gradients that are asked for: x, the residual and the weight as far as they were given
    const bool need_x = ctx->needs_input_grad(0), need_r = residual && ctx->needs_input_grad(1);
    const bool need_w = weight.defined() && ctx->needs_input_grad(residual ? 2 : 1);
    const Tensor dy = grads[0], dh = residual ? grads[1] : Tensor();
    Tensor dx, dw;
    if (!dy.defined()) {  // only h was used, or nothing
      dx = dh;
      if (need_w) dw = at::zeros_like(weight);
    } else {
      c10::DeviceGuard guard(h.device());
      const Tensor h2 = rows2d(h), dy2 = rows2d(dy), dh2 = dh.defined() ? rows2d(dh) : Tensor(),
                   r2 = r.defined() ? rows2d(r) : Tensor();
      const int64_t rows = h2.size(0), d = h2.size(1);
      if (need_x || need_r) dx = at::empty(h.sizes(), h.options());
      if (need_w) dw = rows ? at::empty_like(weight) : at::zeros_like(weight);
      if (rows && (dx.defined() || dw.defined())) {
        const int64_t bytes = need_w ? g_fr.rms_norm_bwd_workspace(rows, (int)d) : 0;
        const Tensor ws = need_w ? workspace(bytes, h) : Tensor();
        done(g_fr.rms_norm_bwd(data(dy2), ld_of(dy2), data(dh2), dh.defined() ? ld_of(dh2) : 0, data(h2), ld_of(h2),
                               data(r2), r.defined() ? ld_of(r2) : 0, rows, (int)d, dtype_of(h), data(weight),
                               dtype_of(weight.defined() ? weight : h), floats(rstd), data(dx), data(dw), data(ws),
                               bytes, stream_of(h)),
             "fr_rms_norm_bwd");
      }
    }
    return once(grads, {need_x ? dx : Tensor(), need_r ? dx : Tensor(), dw, Tensor()});
  }
};

MaybeTensor norm_args(const char* name, const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight,
                      double eps) {
  check(name, x, residual, weight);
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 8192)
    fail(name, ": rows of 1 to 8192 required (got ", x.sizes(), ")");
  if (x.numel() / x.size(-1) > INT32_MAX) fail(name, ": fewer than 2^31 rows required");
  if (residual && (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type()))
    fail(name, ": residual ", residual->sizes(), " ", residual->scalar_type(), " differs from x ", x.sizes(), " ",
         x.scalar_type());
  if (!(eps >= 0.0 && std::isfinite((float)eps))) fail(name, ": eps = ", eps);
  if (!weight) return std::nullopt;
  if (weight->dim() != 1 || weight->size(0) != x.size(-1) ||
      (weight->scalar_type() != at::kFloat && weight->scalar_type() != x.scalar_type()))
    fail(name, ": weight ", weight->sizes(), " ", weight->scalar_type(), ": [", x.size(-1), "] in fp32 or ",
         x.scalar_type(), " required");
  return weight->contiguous();
}

Tensor rms_norm(const Tensor& x, const MaybeTensor& weight, double eps) {
  const MaybeTensor none, w = norm_args("rms_norm", x, none, weight, eps);
  return recording(x, w) ? RmsNorm::apply(x, none, w, eps)[0] : norm_run(x, none, w, eps, false, false).y;
}

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& weight,
                                        double eps) {
  if (!residual) fail("add_rms_norm: a residual is required (rms_norm takes none)");
  const MaybeTensor w = norm_args("add_rms_norm", x, residual, weight, eps);
  if (recording(x, residual, w)) {
    const variable_list o = RmsNorm::apply(x, residual, w, eps);
    return {o[0], o[1]};
  }
  const Normed o = norm_run(x, residual, w, eps, false, false);
  return {o.y, o.h};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_quant(const Tensor& x, const MaybeTensor& residual,
                                                      const MaybeTensor& weight, double eps) {
  const MaybeTensor w = norm_args("add_rms_norm_quant", x, residual, weight, eps);
  if (recording(x, residual, w)) fail("add_rms_norm_quant has no gradient: call it under torch.no_grad()");
  const Normed o = norm_run(x, residual, w, eps, true, false);
  return {o.y, o.scale, residual ? o.h : x};
}

// ---------------------------------------------------------------------------------- item log-probabilities
struct LogP {
  Tensor logp, lse, o, rest;
};

LogP logp_run(const Tensor& h, const Tensor& w, const Tensor& ids, double scale, bool for_dh, bool for_dw) {
  const auto f32 = h.options().dtype(at::kFloat);
  const int64_t n = h.size(0), d = h.size(1);
  LogP r;
  r.logp = at::empty({n}, f32);
  if (for_dw) r.lse = at::empty({2, n}, f32);
  if (for_dh || for_dw) r.rest = at::empty({n}, f32);
  if (for_dh) r.o = at::empty({n, d}, f32);
  if (n) {
    c10::DeviceGuard guard(h.device());
    const Tensor ws = workspace(g_fr.item_logp_fwd_workspace(n, w.size(0), (int)d, ld_of(w), dtype_of(h), for_dh), h);
    done(g_fr.item_logp_fwd(data(h), ld_of(h), n, data(w), ld_of(w), w.size(0), (int)d, dtype_of(h), longs(ids),
                            (float)scale, floats(r.logp), floats(r.lse), floats(r.o), floats(r.rest), data(ws),
                            ws.numel(), stream_of(h)),
         "fr_item_logp_fwd");
  }
  return r;
}

struct ItemLogProbs : torch::autograd::Function<ItemLogProbs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& ids, double scale,
                        bool for_dh, bool for_dw) {
    const LogP r = logp_run(h, w, ids, scale, for_dh, for_dw);
    ctx->save_for_backward({h, w, ids, r.lse, r.o, r.rest});
    ctx->saved_data["scale"] = scale;
    return r.logp;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &w = saved[1], &ids = saved[2], &lse = saved[3], &o = saved[4], &rest = saved[5];
    c10::DeviceGuard guard(h.device());
    const int64_t n = h.size(0);
    Tensor dh, dw, ws;
    if (ctx->needs_input_grad(0)) dh = at::empty(h.sizes(), h.options());
    if (ctx->needs_input_grad(1)) dw = n ? at::empty(w.sizes(), w.options()) : at::zeros(w.sizes(), w.options());
    if (n && (dh.defined() || dw.defined())) {
      const Tensor g = grads[0].contiguous();
      if (dw.defined())
        ws = workspace(g_fr.item_logp_bwd_workspace(n, w.size(0), (int)h.size(1), ld_of(w), dtype_of(h)), h);
      done(g_fr.item_logp_bwd(data(h), ld_of(h), n, data(w), ld_of(w), w.size(0), (int)h.size(1), dtype_of(h), longs(ids),
                              floats(lse), floats(o), floats(rest), floats(g),
                              (float)ctx->saved_data["scale"].toDouble(), data(dh), data(dw), data(ws),
                              ws.defined() ? ws.numel() : 0, stream_of(h)),
           "fr_item_logp_bwd");
    }
    return once(grads, {dh, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor item_log_probs(const Tensor& user_rows, const Tensor& item_table, const Tensor& items, double scale) {
  const char* name = "item_log_probs";
  check(name, user_rows, item_table, items);
  if (user_rows.dim() != 2 || item_table.dim() != 2 || user_rows.size(1) != item_table.size(1) ||
      user_rows.scalar_type() != item_table.scalar_type())
    fail(name, ": rows ", user_rows.sizes(), " ", user_rows.scalar_type(), " and table ", item_table.sizes(), " ",
         item_table.scalar_type(), " do not match");
  const int64_t n = user_rows.size(0), d = user_rows.size(1);
  if (d < 1 || d > 256) fail(name, ": d = ", d, ", 1 to 256 supported");
  if (item_table.size(0) < 1 || item_table.size(0) > INT32_MAX - 64 || n > INT32_MAX)
    fail(name, ": 1 to 2^31 - 65 items and fewer than 2^31 rows required");
  if (items.dim() != 1 || items.size(0) != n) fail(name, ": items ", items.sizes(), ", expected [", n, "]");
  if (!((float)scale > 0.f && scale < 1e30)) fail(name, ": scale = ", scale, ", a positive number required");
  const Tensor ids = ids_of(name, items), h = rows2d(user_rows);
  Tensor w = rows2d(item_table);
  if (reinterpret_cast<uintptr_t>(w.data_ptr()) % 16) w = w.clone();
  return recording(h, w) ? ItemLogProbs::apply(h, w, ids, scale, h.requires_grad(), w.requires_grad())
                         : logp_run(h, w, ids, scale, false, false).logp;
}

// ---------------------------------------------------------------------------------- preference loss
struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logp, const MaybeTensor& ref, const Tensor& offsets,
                        double beta, double smoothing) {
    c10::DeviceGuard guard(logp.device());
    const int64_t pairs = (offsets.numel() - 1) / 2;
    Tensor loss = at::empty({}, logp.options()), scratch = at::empty({pairs}, logp.options());
    Tensor grad = at::empty_like(logp);
    done(g_fr.preference_loss(floats(logp), static_cast<const float*>(data(ref)), longs(offsets), pairs, logp.numel(),
                              (float)beta, (float)smoothing, floats(loss), floats(scratch), floats(grad),
                              stream_of(logp)),
         "fr_preference_loss");
    ctx->save_for_backward({grad});
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return once(grads, {ctx->get_saved_variables()[0] * grads[0].detach(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor preference_loss(const Tensor& logp, const MaybeTensor& ref, const Tensor& offsets, double beta,
                       double smoothing) {
  const char* name = "preference_loss";
  check(name, logp, ref, offsets);
  if (logp.scalar_type() != at::kFloat || logp.dim() != 1)
    fail(name, ": fp32 [n] log-probabilities required (got ", logp.scalar_type(), " ", logp.sizes(), ")");
  if (ref && (ref->scalar_type() != at::kFloat || ref->sizes() != logp.sizes()))
    fail(name, ": reference ", ref->scalar_type(), " ", ref->sizes(), " differs");
  if (offsets.scalar_type() != at::kLong || offsets.dim() != 1 || offsets.numel() < 3 || offsets.numel() % 2 == 0)
    fail(name, ": offsets are int64 [2 pairs + 1]");
  if (!((float)beta > 0.f && std::isfinite((float)beta)) || !(smoothing >= 0.0 && smoothing <= 0.5))
    fail(name, ": beta = ", beta, " > 0 and label_smoothing = ", smoothing, " in [0, 1/2] required");
  MaybeTensor r;
  if (ref) r = ref->detach().contiguous();
  return PreferenceLoss::apply(logp.contiguous(), r, offsets.contiguous(), beta, smoothing);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const EngineError& e) {
      PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  const auto free_gil = py::call_guard<py::gil_scoped_release>();
  m.def("embedding_scaled", &embedding_scaled, free_gil);
  m.def("dropout", &dropout, free_gil);
  m.def("rms_norm", &rms_norm, free_gil);
  m.def("add_rms_norm", &add_rms_norm, free_gil);
  m.def("add_rms_norm_quant", &add_rms_norm_quant, free_gil);
  m.def("item_log_probs", &item_log_probs, free_gil);
  m.def("preference_loss", &preference_loss, free_gil);
}

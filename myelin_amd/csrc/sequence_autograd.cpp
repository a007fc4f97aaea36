// The sequence-model operators' host code in C++: what the Functions of
// attention.py, dropout.py, log_probs.py, gated.py, embedding.py,
// distillation.py and verification.py do (the same entry points, outputs and
// saved tensors), without Python in either direction.  Their small calls
// are host work: the training step of 12800 rows of 10 classes, 7 us of
// kernels, took 134 us with the Python Function, half of it on the autograd
// engine's device thread, which waits there for the interpreter lock that the
// caller's thread holds, and takes 37 to 60 us with this one (host work varies by
// that much from run to run).
//
// Arguments are checked in Python, before; sizes by the entry points.

#include "sequence_autograd.h"

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "../../include/myelin_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Library {
  decltype(&myelin_token_log_probs_workspace_bytes) log_probs_workspace = nullptr;
  decltype(&myelin_token_log_probs) log_probs = nullptr;
  decltype(&myelin_token_log_probs_bwd) log_probs_bwd = nullptr;
  decltype(&myelin_counter_dropout) dropout = nullptr;
  decltype(&myelin_decay_attention_workspace_elems) attention_workspace = nullptr;
  decltype(&myelin_decay_attention_fwd) attention_fwd = nullptr;
  decltype(&myelin_decay_attention_bwd) attention_bwd = nullptr;
  decltype(&myelin_decay_attention_step) attention_step = nullptr;
  decltype(&myelin_gated_recurrence_kept_elems) recurrence_kept = nullptr;
  decltype(&myelin_gated_recurrence_workspace_elems) recurrence_workspace = nullptr;
  decltype(&myelin_gated_recurrence_fwd) recurrence_fwd = nullptr;
  decltype(&myelin_gated_recurrence_bwd) recurrence_bwd = nullptr;
  decltype(&myelin_gated_recurrence_step) recurrence_step = nullptr;
  decltype(&myelin_token_embedding) embedding = nullptr;
  decltype(&myelin_token_embedding_bwd_workspace_bytes) embedding_workspace = nullptr;
  decltype(&myelin_token_embedding_bwd) embedding_bwd = nullptr;
  decltype(&myelin_distillation_loss_workspace_bytes) distillation_workspace = nullptr;
  decltype(&myelin_distillation_loss) distillation = nullptr;
  decltype(&myelin_distillation_loss_bwd) distillation_bwd = nullptr;
  decltype(&myelin_verify_draft_workspace_bytes) verify_workspace = nullptr;
  decltype(&myelin_verify_draft) verify = nullptr;
  decltype(&myelin_last_error) last_error = nullptr;
  PyObject *hip_error = nullptr;  // the class of failed launches; never released
} lib;

// as _lib.call: ValueError for a rejected argument, MyelinHipError else
void check(int rc, const char *name) {
  if (rc == MYELIN_OK) return;
  const std::string message = std::string(name) + ": " + lib.last_error();
  pybind11::gil_scoped_acquire gil;
  PyErr_SetString(rc == MYELIN_EINVAL ? PyExc_ValueError : lib.hip_error, message.c_str());
  python_error error;
  error.persist();
  throw error;
}

myelin_stream_t stream_of(const Tensor &t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void *at(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *f32(const Tensor &t) { return static_cast<float *>(at(t)); }
int64_t *i64(const Tensor &t) { return static_cast<int64_t *>(at(t)); }
int32_t *i32(const Tensor &t) { return static_cast<int32_t *>(at(t)); }
Tensor plain(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }
Tensor contiguous(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

// the library's dtype codes of the two types these operators take
int code_of(const Tensor &t) { return t.scalar_type() == torch::kFloat32 ? 0 : 2; }

// Gradients that have none themselves: under create_graph they carry a node
// that raises when it is differentiated.
variable_list once(variable_list grads) {
  if (!torch::GradMode::is_enabled()) return grads;
  for (Tensor &g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable",
      static_cast<int64_t>(grads.size()));
  return (*error)(std::move(grads));
}

bool needs(std::initializer_list<Tensor> tensors) {
  if (!torch::GradMode::is_enabled()) return false;
  for (const Tensor &t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// ---- log probabilities ---------------------------------------------------
struct LogProbs {
  Tensor log_probs, entropy, stats, top_log_probs, top_tokens;
};

// x [R, V] with rows of unit stride, targets [R] int64 or undefined
LogProbs log_probs_forward(const Tensor &x, const Tensor &targets, int64_t top, int64_t ignore) {
  const int64_t R = x.size(0), V = x.size(1);
  const auto options = x.options().dtype(torch::kFloat32);
  LogProbs r;
  if (targets.defined()) r.log_probs = torch::empty({R}, options);
  r.entropy = torch::empty({R}, options);
  r.stats = torch::empty({2, R}, options);
  if (top) {
    r.top_log_probs = torch::empty({R, top}, options);
    r.top_tokens = torch::empty({R, top}, x.options().dtype(torch::kInt64));
  }
  const int64_t need = lib.log_probs_workspace(R, V, static_cast<int>(top));
  Tensor ws;
  if (need) ws = torch::empty({need}, x.options().dtype(torch::kUInt8));
  check(lib.log_probs(at(x), code_of(x), x.stride(0), i64(targets), ignore, f32(r.log_probs), f32(r.entropy),
                      f32(r.stats), f32(r.top_log_probs), i64(r.top_tokens), R, V, static_cast<int>(top), at(ws), need,
                      stream_of(x)),
        "myelin_token_log_probs");
  return r;
}

// what there is of {log_probs, entropy, top_log_probs, top_tokens}
variable_list results(const LogProbs &r) {
  variable_list out;
  for (const Tensor &t : {r.log_probs, r.entropy, r.top_log_probs, r.top_tokens})
    if (t.defined()) out.push_back(t);
  return out;
}

struct LogProbsFunction : torch::autograd::Function<LogProbsFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &targets, int64_t top,
                               int64_t ignore) {
    const LogProbs r = log_probs_forward(x, plain(targets), top, ignore);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, plain(targets), r.stats, r.entropy});
    ctx->saved_data["ignore"] = ignore;
    if (top) ctx->mark_non_differentiable({r.top_log_probs, r.top_tokens});
    return results(r);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &targets = saved[1];
    const Tensor g_lp = targets.defined() ? contiguous(grads[0]) : Tensor(),
                 g_ent = contiguous(grads[targets.defined() ? 1 : 0]);
    variable_list out(4);
    if (!g_lp.defined() && !g_ent.defined()) return out;
    const int64_t R = x.size(0), V = x.size(1);
    const c10::DeviceGuard guard(x.device());
    out[0] = torch::empty({R, V}, x.options());
    check(lib.log_probs_bwd(at(x), code_of(x), x.stride(0), i64(targets), ctx->saved_data["ignore"].toInt(),
                            f32(saved[2]), f32(saved[3]), f32(g_lp), f32(g_ent), at(out[0]), R, V, stream_of(x)),
          "myelin_token_log_probs_bwd");
    return once(std::move(out));
  }
};

variable_list token_log_probs(const Tensor &x, const OptTensor &targets, int64_t top, int64_t ignore) {
  const c10::DeviceGuard guard(x.device());
  if (needs({x})) return LogProbsFunction::apply(x, targets, top, ignore);
  return results(log_probs_forward(x, plain(targets), top, ignore));
}

// ---- dropout -------------------------------------------------------------
struct Mask {
  int64_t steps, threshold, seed, offset;
  double scale;
};

Tensor dropped(const Tensor &x, const Tensor &residual, const Mask &m, const Tensor &offset) {
  Tensor y = torch::empty_like(x);
  check(lib.dropout(at(x), code_of(x), at(residual), at(y), m.steps, m.steps ? x.numel() / m.steps : 0, m.threshold,
                    static_cast<float>(m.scale), m.seed, m.offset, i64(offset), stream_of(x)),
        "myelin_counter_dropout");
  return y;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, const OptTensor &offset,
                        const Mask &m) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({plain(offset)});
    ctx->saved_data["m"] = std::vector<int64_t>{m.steps, m.threshold, m.seed, m.offset};
    ctx->saved_data["scale"] = m.scale;
    ctx->saved_data["residual"] = residual.has_value();
    return dropped(x, plain(residual), m, plain(offset));
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(4);
    const Tensor &g = grads[0];
    if (!g.defined()) return out;
    const Tensor offset = ctx->get_saved_variables()[0];
    if (ctx->needs_input_grad(0)) {
      const c10::DeviceGuard guard(g.device());
      const std::vector<int64_t> m = ctx->saved_data["m"].toIntVector();
      out[0] = dropped(g.contiguous(), Tensor(), Mask{m[0], m[1], m[2], m[3], ctx->saved_data["scale"].toDouble()},
                       offset);
    }
    // (inputs are counted without those that were not given)
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = g;
    return once(std::move(out));
  }
};

// x and residual contiguous; the offset on the device, or the number
Tensor counter_dropout(const Tensor &x, const OptTensor &residual, const OptTensor &offset, int64_t steps,
                       int64_t threshold, double scale, int64_t seed, int64_t number) {
  const c10::DeviceGuard guard(x.device());
  const Mask m{steps, threshold, seed, number, scale};
  if (needs({x, plain(residual)})) return DropoutFunction::apply(x, residual, offset, m);
  return dropped(x, plain(residual), m, plain(offset));
}

// ---- attention -----------------------------------------------------------
struct Sizes {
  int64_t T, B, H, Hk, Dk, Dv;
};

Sizes sizes_of(const Tensor &q, const Tensor &v) {
  return {q.size(0), q.size(1), q.size(2), v.size(2), q.size(3), v.size(3)};
}

// strides of all but each tensor's last dimension
std::vector<int64_t> strides_of(std::initializer_list<Tensor> tensors) {
  std::vector<int64_t> s;
  for (const Tensor &t : tensors)
    for (int64_t i = 0; i + 1 < t.dim(); ++i) s.push_back(t.stride(i));
  return s;
}

Tensor unit_stride(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

Tensor attention_workspace(const Tensor &q, const Sizes &z, int backward, int64_t *elems) {
  *elems = lib.attention_workspace(code_of(q), z.T, z.B, z.H, z.Hk, z.Dk, z.Dv, backward);
  return *elems ? torch::empty({*elems}, q.options().dtype(torch::kFloat32)) : Tensor();
}

// {final state, out}
variable_list attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &decay,
                                const Tensor &state, const Tensor &lengths, double scale) {
  const Sizes z = sizes_of(q, v);
  Tensor out = torch::empty({z.T, z.B, z.H, z.Dv}, q.options());
  Tensor last = torch::empty({z.B, z.H, z.Dk, z.Dv}, q.options().dtype(torch::kFloat32));
  int64_t elems;
  const Tensor ws = attention_workspace(q, z, 0, &elems);
  check(lib.attention_fwd(at(q), at(k), at(v), code_of(q), strides_of({q, k, v}).data(), f32(decay), f32(state),
                          i32(lengths), at(out), f32(last), z.T, z.B, z.H, z.Hk, z.Dk, z.Dv, static_cast<float>(scale),
                          f32(ws), elems, stream_of(q)),
        "myelin_decay_attention_fwd");
  return {last, out};
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                               const OptTensor &state, const Tensor &decay, const OptTensor &lengths, double scale) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, plain(state), decay, plain(lengths)});
    ctx->saved_data["scale"] = scale;
    return attention_forward(q, k, v, decay, plain(state), plain(lengths), scale);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2];
    const Sizes z = sizes_of(q, v);
    const c10::DeviceGuard guard(q.device());
    const Tensor g_out =
        grads[1].defined() ? unit_stride(grads[1]) : torch::zeros({z.T, z.B, z.H, z.Dv}, q.options());
    const Tensor g_last = contiguous(grads[0]);
    Tensor gq = torch::empty(q.sizes(), q.options()), gk = torch::empty(k.sizes(), q.options()),
           gv = torch::empty(v.sizes(), q.options()), gs;
    if (saved[3].defined() && ctx->needs_input_grad(3))
      gs = torch::empty({z.B, z.H, z.Dk, z.Dv}, q.options().dtype(torch::kFloat32));
    int64_t elems;
    const Tensor ws = attention_workspace(q, z, 1, &elems);
    check(lib.attention_bwd(at(q), at(k), at(v), at(g_out), code_of(q), strides_of({q, k, v, g_out}).data(),
                            f32(saved[4]), f32(saved[3]), i32(saved[5]), f32(g_last), at(gq), at(gk), at(gv), f32(gs),
                            z.T, z.B, z.H, z.Hk, z.Dk, z.Dv, static_cast<float>(ctx->saved_data["scale"].toDouble()),
                            f32(ws), elems, stream_of(q)),
          "myelin_decay_attention_bwd");
    if (ctx->needs_input_grad(0)) out[0] = gq;
    if (ctx->needs_input_grad(1)) out[1] = gk;
    if (ctx->needs_input_grad(2)) out[2] = gv;
    out[3] = gs;
    return once(std::move(out));
  }
};

// q, k, v with unit stride in their last dimension, the others contiguous
variable_list decay_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &decay,
                              const OptTensor &state, const OptTensor &lengths, double scale) {
  const c10::DeviceGuard guard(q.device());
  if (needs({q, k, v, plain(state)})) return AttentionFunction::apply(q, k, v, state, decay, lengths, scale);
  return attention_forward(q, k, v, decay, plain(state), plain(lengths), scale);
}

// {new state, out}; the new state goes to out_state, if given
variable_list decay_attention_step(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &decay,
                                   const Tensor &state, const OptTensor &out_state, double scale) {
  const c10::DeviceGuard guard(q.device());
  const int64_t B = q.size(0), H = q.size(1), Dk = q.size(2), Hk = v.size(1), Dv = v.size(2);
  Tensor out = torch::empty({B, H, Dv}, q.options());
  Tensor to = out_state.has_value() ? *out_state : torch::empty({B, H, Dk, Dv}, state.options());
  check(lib.attention_step(at(q), at(k), at(v), code_of(q), strides_of({q, k, v}).data(), f32(decay), f32(state),
                           at(out), f32(to), B, H, Hk, Dk, Dv, static_cast<float>(scale), stream_of(q)),
        "myelin_decay_attention_step");
  // autograd notices where it keeps out_state for a backward pass
  if (out_state.has_value() && !to.is_inference()) to.unsafeGetTensorImpl()->bump_version();
  return {to, out};
}

// ---- gated recurrence ----------------------------------------------------
Tensor recurrence_workspace(const Tensor &x, int backward, int64_t *elems) {
  *elems = lib.recurrence_workspace(code_of(x), x.size(0), x.size(1), x.size(2), backward);
  return *elems ? torch::empty({*elems}, x.options().dtype(torch::kFloat32)) : Tensor();
}

// unit stride in the last dimension, and batch rows near enough for the kernels
Tensor recurrence_rows(const Tensor &t) {
  const int64_t B = t.size(-2), N = t.size(-1);
  const bool near = B <= 1 || N == 0 || (64 / N + 1) * t.stride(-2) + N < int64_t{1} << 29;
  return near ? unit_stride(t) : t.contiguous();
}

// {final state, out}, and the kept states where a gradient is wanted
variable_list recurrence_forward(const Tensor &x, const Tensor &gate, const Tensor &state, const Tensor &lengths,
                                 Tensor *kept) {
  const int64_t T = x.size(0), B = x.size(1), N = x.size(2);
  const auto f32s = x.options().dtype(torch::kFloat32);
  Tensor out = torch::empty({T, B, N}, x.options()), last = torch::empty({B, N}, f32s);
  if (kept) *kept = torch::empty({lib.recurrence_kept(T, B, N)}, f32s);
  int64_t elems;
  const Tensor ws = recurrence_workspace(x, 0, &elems);
  check(lib.recurrence_fwd(at(x), at(gate), code_of(x), strides_of({x, gate}).data(), f32(state), i32(lengths), at(out),
                           f32(last), kept ? f32(*kept) : nullptr, T, B, N, f32(ws), elems, stream_of(x)),
        "myelin_gated_recurrence_fwd");
  return {last, out};
}

struct RecurrenceFunction : torch::autograd::Function<RecurrenceFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &gate, const OptTensor &state,
                               const OptTensor &lengths) {
    ctx->set_materialize_grads(false);
    Tensor kept;
    variable_list out = recurrence_forward(x, gate, plain(state), plain(lengths), &kept);
    ctx->save_for_backward({x, gate, plain(lengths), kept});
    ctx->saved_data["state"] = state.has_value();
    return out;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gate = saved[1];
    const int64_t T = x.size(0), B = x.size(1), N = x.size(2);
    const c10::DeviceGuard guard(x.device());
    const Tensor g_out = grads[1].defined() ? recurrence_rows(grads[1]) : Tensor(), g_last = contiguous(grads[0]);
    if (ctx->needs_input_grad(0)) out[0] = torch::empty({T, B, N}, x.options());
    if (ctx->needs_input_grad(1)) out[1] = torch::empty({T, B, N}, x.options());
    // (inputs are counted without those that were not given)
    if (ctx->saved_data["state"].toBool() && ctx->needs_input_grad(2))
      out[2] = torch::empty({B, N}, x.options().dtype(torch::kFloat32));
    int64_t elems;
    const Tensor ws = recurrence_workspace(x, 1, &elems);
    check(lib.recurrence_bwd(at(x), at(gate), at(g_out), code_of(x),
                             strides_of({x, gate, g_out.defined() ? g_out : x}).data(), i32(saved[2]), f32(saved[3]),
                             f32(g_last), at(out[0]), at(out[1]), f32(out[2]), T, B, N, f32(ws), elems, stream_of(x)),
          "myelin_gated_recurrence_bwd");
    return once(std::move(out));
  }
};

// state and lengths contiguous
variable_list gated_recurrence(const Tensor &given_x, const Tensor &given_gate, const OptTensor &state,
                               const OptTensor &lengths) {
  const c10::DeviceGuard guard(given_x.device());
  const Tensor x = recurrence_rows(given_x), gate = recurrence_rows(given_gate);
  if (needs({x, gate, plain(state)})) return RecurrenceFunction::apply(x, gate, state, lengths);
  return recurrence_forward(x, gate, plain(state), plain(lengths), nullptr);
}

// {new state, out}; the new state goes to out_state, if given
variable_list gated_recurrence_step(const Tensor &given_x, const Tensor &given_gate, const Tensor &given_state,
                                    const OptTensor &out_state) {
  const c10::DeviceGuard guard(given_x.device());
  const Tensor x = recurrence_rows(given_x), gate = recurrence_rows(given_gate), state = given_state.contiguous();
  const int64_t B = x.size(0), N = x.size(1);
  Tensor out = torch::empty({B, N}, x.options());
  Tensor to = out_state.has_value() ? *out_state : torch::empty({B, N}, state.options());
  check(lib.recurrence_step(at(x), at(gate), code_of(x), strides_of({x, gate}).data(), f32(state), at(out), f32(to), B,
                            N, stream_of(x)),
        "myelin_gated_recurrence_step");
  // autograd notices where it keeps out_state for a backward pass
  if (out_state.has_value() && !to.is_inference()) to.unsafeGetTensorImpl()->bump_version();
  return {to, out};
}

// ---- embedding -----------------------------------------------------------
Tensor embedded(const Tensor &weight, const Tensor &tokens, double scale, int64_t padding) {
  const int64_t M = tokens.numel(), V = weight.size(0), D = weight.size(1);
  std::vector<int64_t> shape = tokens.sizes().vec();
  shape.push_back(D);
  Tensor out = torch::empty(shape, weight.options());
  check(lib.embedding(i64(tokens), at(weight), code_of(weight), weight.stride(0), at(out), M, V, D,
                      static_cast<float>(scale), padding, stream_of(weight)),
        "myelin_token_embedding");
  return out;
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &weight, const Tensor &tokens, double scale,
                        int64_t padding) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["sizes"] = std::vector<int64_t>{padding, weight.size(0), weight.size(1)};
    return embedded(weight, tokens, scale, padding);
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const Tensor tokens = ctx->get_saved_variables()[0], g = grads[0].contiguous();
    const std::vector<int64_t> z = ctx->saved_data["sizes"].toIntVector();
    const int64_t M = tokens.numel(), V = z[1], D = z[2];
    const c10::DeviceGuard guard(g.device());
    out[0] = torch::empty({V, D}, g.options());
    const int64_t need = lib.embedding_workspace(M, V, D);
    Tensor ws;
    if (need) ws = torch::empty({need}, g.options().dtype(torch::kUInt8));
    check(lib.embedding_bwd(i64(tokens), at(g), code_of(g), at(out[0]), M, V, D,
                            static_cast<float>(ctx->saved_data["scale"].toDouble()), z[0], at(ws), need, stream_of(g)),
          "myelin_token_embedding_bwd");
    return once(std::move(out));
  }
};

// weight with rows of unit stride
Tensor token_embedding(const Tensor &weight, const Tensor &given, double scale, int64_t padding) {
  const c10::DeviceGuard guard(weight.device());
  const Tensor tokens = given.to(torch::kInt64).contiguous();
  if (needs({weight})) return EmbeddingFunction::apply(weight, tokens, scale, padding);
  return embedded(weight, tokens, scale, padding);
}

// ---- distillation --------------------------------------------------------
struct Distilled {
  Tensor loss, probs, stats;
};

// rows x [R, V]; the loss in the shape `lead` of R rows
Distilled distillation_forward(const Tensor &x, at::IntArrayRef lead, const Tensor &values, const Tensor &tokens,
                               double temperature, bool keep) {
  const int64_t R = x.size(0), V = x.size(1), K = tokens.size(1);
  const auto f32s = x.options().dtype(torch::kFloat32);
  Distilled d{torch::empty(lead, f32s), Tensor(), torch::empty({2, R}, f32s)};
  if (keep) d.probs = torch::empty({R, K}, f32s);
  const int64_t need = lib.distillation_workspace(R, V);
  Tensor ws;
  if (need) ws = torch::empty({need}, x.options().dtype(torch::kUInt8));
  check(lib.distillation(at(x), code_of(x), x.stride(0), f32(values), i64(tokens), static_cast<float>(temperature),
                         f32(d.loss), f32(d.probs), f32(d.stats), R, V, static_cast<int>(K), at(ws), need,
                         stream_of(x)),
        "myelin_distillation_loss");
  return d;
}

// [..., V] as rows [R, V] of unit stride
Tensor distillation_rows(const Tensor &logits) {
  const int64_t V = logits.size(-1);
  const Tensor x = logits.dim() == 2 ? logits : logits.reshape({-1, V});
  return (x.size(0) > 1 && x.stride(0) < V) || x.stride(1) != 1 ? x.contiguous() : x;
}

at::IntArrayRef lead_of(const Tensor &logits) { return logits.sizes().slice(0, logits.dim() - 1); }

struct DistillationFunction : torch::autograd::Function<DistillationFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &values, const Tensor &tokens,
                        double temperature) {
    const Tensor x = distillation_rows(logits);
    const Distilled d = distillation_forward(x, lead_of(logits), values, tokens, temperature, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, tokens, d.probs, d.stats});
    ctx->saved_data["temperature"] = temperature;
    return d.loss;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], g = grads[0].contiguous();
    const int64_t R = x.size(0), V = x.size(1);
    const c10::DeviceGuard guard(x.device());
    std::vector<int64_t> shape = g.sizes().vec();
    shape.push_back(V);
    out[0] = torch::empty(shape, x.options());
    check(lib.distillation_bwd(at(x), code_of(x), x.stride(0), i64(saved[1]), f32(saved[2]), f32(saved[3]), f32(g),
                               static_cast<float>(ctx->saved_data["temperature"].toDouble()), at(out[0]), R, V,
                               static_cast<int>(saved[1].size(1)), stream_of(x)),
          "myelin_distillation_loss_bwd");
    return once(std::move(out));
  }
};

Tensor distillation_loss(const Tensor &logits, const Tensor &teacher_logits, const Tensor &teacher_tokens,
                         double temperature) {
  const c10::DeviceGuard guard(logits.device());
  const int64_t K = teacher_logits.size(-1);
  const Tensor values = teacher_logits.reshape({-1, K}).to(torch::kFloat32).contiguous();
  const Tensor tokens = teacher_tokens.reshape({-1, K}).to(torch::kInt64).contiguous();
  if (needs({logits})) return DistillationFunction::apply(logits, values, tokens, temperature);
  return distillation_forward(distillation_rows(logits), lead_of(logits), values, tokens, temperature, false).loss;
}

// ---- verification --------------------------------------------------------
// {accepted, tokens}; lengths contiguous
variable_list verify_draft(const Tensor &given_target, const OptTensor &given_draft, const Tensor &given_tokens,
                           const Tensor &given_uniforms, const OptTensor &lengths) {
  const c10::DeviceGuard guard(given_target.device());
  const torch::NoGradGuard no_grad;
  const Tensor target = unit_stride(given_target), uniforms = given_uniforms.contiguous();
  const Tensor q = given_draft.has_value() ? unit_stride(*given_draft) : Tensor();
  const Tensor tokens = given_tokens.to(torch::kInt64).contiguous();
  const int64_t n = target.size(0) - 1, B = target.size(1), V = target.size(2);
  const auto whole = target.options().dtype(torch::kInt64);
  Tensor accepted = torch::empty({B}, whole), out = torch::empty({n + 1, B}, whole);
  const int64_t need = lib.verify_workspace(B, V);
  Tensor ws;
  if (need) ws = torch::empty({need}, target.options().dtype(torch::kUInt8));
  check(lib.verify(at(target), at(q), code_of(target), strides_of({target, q.defined() ? q : target}).data(),
                   i64(tokens), f32(uniforms), i32(plain(lengths)), i64(accepted), i64(out), n, B, V, at(ws), need,
                   stream_of(target)),
        "myelin_verify_draft");
  return {accepted, out};
}

template <class F>
void take(F &to, const pybind11::dict &from, const char *name) {
  to = reinterpret_cast<F>(from[name].cast<uintptr_t>());
}

}  // namespace

void register_sequence_operators(pybind11::module_ &m) {
  m.def("bind_sequence", [](const pybind11::dict &addresses, const pybind11::object &hip_error) {
    take(lib.log_probs_workspace, addresses, "myelin_token_log_probs_workspace_bytes");
    take(lib.log_probs, addresses, "myelin_token_log_probs");
    take(lib.log_probs_bwd, addresses, "myelin_token_log_probs_bwd");
    take(lib.dropout, addresses, "myelin_counter_dropout");
    take(lib.attention_workspace, addresses, "myelin_decay_attention_workspace_elems");
    take(lib.attention_fwd, addresses, "myelin_decay_attention_fwd");
    take(lib.attention_bwd, addresses, "myelin_decay_attention_bwd");
    take(lib.attention_step, addresses, "myelin_decay_attention_step");
    take(lib.recurrence_kept, addresses, "myelin_gated_recurrence_kept_elems");
    take(lib.recurrence_workspace, addresses, "myelin_gated_recurrence_workspace_elems");
    take(lib.recurrence_fwd, addresses, "myelin_gated_recurrence_fwd");
    take(lib.recurrence_bwd, addresses, "myelin_gated_recurrence_bwd");
    take(lib.recurrence_step, addresses, "myelin_gated_recurrence_step");
    take(lib.embedding, addresses, "myelin_token_embedding");
    take(lib.embedding_workspace, addresses, "myelin_token_embedding_bwd_workspace_bytes");
    take(lib.embedding_bwd, addresses, "myelin_token_embedding_bwd");
    take(lib.distillation_workspace, addresses, "myelin_distillation_loss_workspace_bytes");
    take(lib.distillation, addresses, "myelin_distillation_loss");
    take(lib.distillation_bwd, addresses, "myelin_distillation_loss_bwd");
    take(lib.verify_workspace, addresses, "myelin_verify_draft_workspace_bytes");
    take(lib.verify, addresses, "myelin_verify_draft");
    take(lib.last_error, addresses, "myelin_last_error");
    lib.hip_error = pybind11::object(hip_error).release().ptr();
  });
  // as ctypes does for the library's calls: other threads run meanwhile
  const auto nogil = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("token_log_probs", &token_log_probs, nogil);
  m.def("counter_dropout", &counter_dropout, nogil);
  m.def("decay_attention", &decay_attention, nogil);
  m.def("decay_attention_step", &decay_attention_step, nogil);
  m.def("gated_recurrence", &gated_recurrence, nogil);
  m.def("gated_recurrence_step", &gated_recurrence_step, nogil);
  m.def("token_embedding", &token_embedding, nogil);
  m.def("distillation_loss", &distillation_loss, nogil);
  m.def("verify_draft", &verify_draft, nogil);
}

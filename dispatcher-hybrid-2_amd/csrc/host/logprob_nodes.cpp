// Log-probabilities of tokens, the preference loss and the policy loss as autograd nodes in C++: what fused_logprobs.py calls in
// plain eager execution (why in C++: vocab_nodes.cpp).

#include "nodes.h"

namespace {

// the gradients as torch operations, differentiable themselves; never freed
py::object *again_logprobs = nullptr, *again_preference = nullptr, *again_policy = nullptr;

// (rows, T, V) logits and (rows, T) tokens as the entry points take them
struct Rows {
  Tensor z, tokens;
  int64_t sb = 0, st = 0, B = 1, T = 1, n = 1;
  int code, V, token_bits;
  Rows(const char* what, const Tensor& logits, const Tensor& tokens_)
      : z(unit_rows(logits)), tokens(tokens_.contiguous()), code(dtype_code(logits)), V(narrow(logits.size(-1))) {
    if (z.dim() > 3) z = unit_rows(z.flatten(0, z.dim() - 3));
    if (z.dim() == 3) {
      B = z.size(0), T = z.size(1), sb = z.stride(0), st = z.stride(1);
    } else if (z.dim() == 2) {
      T = z.size(0), st = z.stride(0);
    }
    n = B * T;
    TORCH_CHECK_VALUE(n < (1 << 22), what, ": ", n, " rows, fewer than ", 1 << 22, " possible");
    token_bits = bits(what, tokens);
    same_count(what, "tokens", tokens.numel(), n);
  }
};

Tensor workspace(int64_t bytes, const Tensor& like) {
  Tensor ws;                                                   // (refused sizes: the call says why)
  if (bytes > 0) ws = at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false));
  return ws;
}
// What a loss keeps for its backward pass, `numbers` of them, and behind them its workspace: one allocation, as long as the latter
// is small.
struct Buffer {
  Tensor kept, ws;
  float* at = nullptr;
  void* scratch = nullptr;
  Buffer(int64_t numbers, int64_t bytes, const at::TensorOptions& f32) {
    const int64_t first = (numbers + 3) / 4 * 4, more = bytes > 0 ? (bytes + 3) / 4 : 0;
    const bool together = more <= 65536;
    kept = at::empty({together ? first + more : numbers}, f32);
    at = kept.data_ptr<float>();
    if (together) {
      scratch = at + first;
    } else {
      ws = at::empty({more}, f32);
      scratch = ws.data_ptr();
    }
  }
};
void* at_(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
// fp32 on one stride
Tensor numbers(const Tensor& t) { return t.defined() ? t.to(at::kFloat).contiguous() : t; }

// kept by a saved-tensor hook in any layout
Tensor kept_rows(const char* what, const Tensor& kept, int64_t needs) {
  TORCH_CHECK_VALUE(kept.scalar_type() == at::kFloat && kept.numel() >= needs, what, ": ", kept.numel(), " numbers kept, ", needs,
                    " needed");
  return kept.is_contiguous() && reinterpret_cast<uintptr_t>(kept.data_ptr()) % 16 == 0 ? kept : fresh(kept);
}

// ---- log-probabilities ------------------------------------------------------------------------------------------------
// {log-probabilities, entropies (or none)}, kept: four numbers a row
std::pair<variable_list, Tensor> logprobs(const Tensor& logits, const Tensor& tokens, double temperature, int64_t ignore_index,
                                          bool entropy, bool keep) {
  const char* what = "token_logprobs";
  same_gpu(what, logits, {&tokens});
  const c10::DeviceGuard guard(logits.device());
  const Rows a(what, logits, tokens);
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  variable_list out{at::empty(shape, f32)};
  if (entropy) out.push_back(at::empty(shape, f32));
  Tensor kept;
  if (keep) kept = at::empty({4 * a.n}, f32);
  const int64_t bytes = lib.dh_logprob_workspace_bytes(a.code, a.n, a.V);
  const Tensor ws = workspace(bytes, logits);
  check(lib.dh_logprob_fwd(a.code, a.z.data_ptr(), a.sb, a.st, a.n ? a.B : 0, a.n ? (int)a.T : 1, a.V, a.tokens.data_ptr(),
                           a.token_bits, ignore_index, temperature, floats(out[0]), entropy ? floats(out[1]) : nullptr,
                           at_(kept), at_(ws), bytes, stream_of(logits)),
        what);
  return {out, kept};
}

// the gradients in a row's log-probability and entropy
struct Upstream {
  const float* by_lp = nullptr;
  int64_t lp_div = 1, lp_stride = 1;
  const float* by_ent = nullptr;
  int64_t ent_stride = 1;
  const float* g = nullptr;
  int64_t g_div = 1, g_mod = 1, g_stride = 0;
  const float* divisor = nullptr;
};
Tensor rows_grad(const char* what, const Rows& a, const Tensor& logits, double temperature, int64_t ignore_index, const float* kept,
                 const Upstream& u) {
  Tensor dz = at::empty(logits.sizes(), logits.options().requires_grad(false));
  if (dz.numel() == 0) return dz;
  check(lib.dh_logprob_bwd(a.code, a.z.data_ptr(), a.sb, a.st, a.B, (int)a.T, a.V, a.tokens.data_ptr(), a.token_bits,
                           ignore_index, temperature, kept, u.by_lp, u.lp_div, u.lp_stride, u.by_ent, u.ent_stride, u.g, u.g_div,
                           u.g_mod, u.g_stride, u.divisor, dz.data_ptr(), stream_of(logits)),
        what);
  return dz;
}

Tensor logprobs_grad(const Tensor& g_lp, const Tensor& g_ent, const Tensor& logits, const Tensor& tokens, const Tensor& kept_,
                     double temperature, int64_t ignore_index) {
  const char* what = "token_logprobs gradient";
  same_gpu(what, logits, {&g_lp, &g_ent, &tokens, &kept_});
  const c10::DeviceGuard guard(logits.device());
  const Rows a(what, logits, tokens);
  const Tensor kept = kept_rows(what, kept_, 4 * a.n);
  Tensor lp = g_lp.defined() ? g_lp.to(at::kFloat).reshape({-1}) : at::zeros({1}, kept.options());
  if (g_lp.defined()) same_count(what, "the log-probabilities' gradient", lp.numel(), a.n);
  const Tensor ent = g_ent.defined() ? g_ent.to(at::kFloat).reshape({-1}) : Tensor();
  if (ent.defined()) same_count(what, "the entropies' gradient", ent.numel(), a.n);
  Upstream u;
  u.by_lp = floats(lp);
  u.lp_stride = g_lp.defined() ? lp.stride(0) : 0;
  if (ent.defined()) u.by_ent = floats(ent), u.ent_stride = ent.stride(0);
  return rows_grad(what, a, logits, temperature, ignore_index, floats(kept), u);
}

// a call of a differentiable gradient in Python
template <typename... A>
Tensor by_torch(py::object* fn, A&&... args) {
  const py::gil_scoped_acquire gil;
  try {
    return (*fn)(std::forward<A>(args)...).template cast<Tensor>();
  } catch (py::error_already_set& e) {     // (it must not outlive the lock it is held under)
    TORCH_CHECK(false, e.what());
  }
}
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, double temperature,
                               int64_t ignore_index, bool entropy) {
    auto [out, kept] = logprobs(logits, tokens, temperature, ignore_index, entropy, logits.requires_grad());
    ctx->set_materialize_grads(false);
    if (logits.requires_grad()) ctx->save_for_backward({logits, savable(tokens), kept});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore_index;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    const Tensor ent = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !ent.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const double temperature = ctx->saved_data["temperature"].toDouble();
    const int64_t ignore = ctx->saved_data["ignore"].toInt();
    out[0] = at::GradMode::is_enabled()
                 ? by_torch(again_logprobs, saved[0], saved[1], temperature, ignore, maybe(grads[0]), maybe(ent))
                 : logprobs_grad(grads[0], ent, saved[0], saved[1], saved[2], temperature, ignore);
    return out;
  }
};

// the same from hidden states and the head's weight
variable_list head_logprobs(const Tensor& hidden, const Tensor& weight, const Tensor& tokens_, double temperature,
                            int64_t ignore_index, bool entropy, bool round_logits) {
  const char* what = "head_logprobs";
  same_gpu(what, hidden, {&weight, &tokens_});
  const int code = dtype_code(hidden);
  TORCH_CHECK_TYPE(weight.scalar_type() == hidden.scalar_type(), what, ": weight of another type");
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(hidden.device());
  TORCH_CHECK_VALUE(weight.dim() == 2 && hidden.dim() >= 1 && weight.size(1) == hidden.size(-1), what, ": hidden states ",
                    hidden.sizes(), " and weight ", weight.sizes());
  const Tensor h = unit_rows(hidden.dim() == 2 ? hidden : hidden.dim() == 1 ? hidden.unsqueeze(0) : hidden.flatten(0, -2)),
               w = unit_rows(weight), tokens = tokens_.contiguous();
  const int64_t n = h.size(0);
  const int token_bits = bits(what, tokens);
  same_count(what, "tokens", tokens.numel(), n);
  const auto f32 = hidden.options().dtype(at::kFloat).requires_grad(false);
  const auto shape = hidden.sizes().slice(0, hidden.dim() - 1);
  variable_list out{at::empty(shape, f32)};
  if (entropy) out.push_back(at::empty(shape, f32));
  const int V = narrow(w.size(0));
  const int64_t bytes = lib.dh_head_logprob_workspace_bytes(code, n, V);
  const Tensor ws = workspace(bytes, hidden);
  check(lib.dh_head_logprob(code, h.data_ptr(), h.stride(0), n, narrow(h.size(1)), w.data_ptr(), w.stride(0), V, tokens.data_ptr(),
                            token_bits, ignore_index, temperature, round_logits, floats(out[0]), entropy ? floats(out[1]) : nullptr,
                            at_(ws), bytes, stream_of(hidden)),
        what);
  return out;
}

// ---- preference loss ----------------------------------------------------------------------------------------------------
struct Preference {
  int64_t kind;                            // 0 sigmoid, 1 hinge, 2 squared
  bool average;
  double beta, margin, smoothing;
  int64_t ignore_index, reduction;         // reduction: 0 none, 1 mean, 2 sum
};
int64_t preference_kept(int64_t n, int64_t pairs) { return 4 * n + 2 * pairs + 1; }

struct Loss {
  Tensor loss, values, kept;
};

Loss preference(const Tensor& logits, const Tensor& tokens, const Tensor& reference_, const Preference& f) {
  const char* what = "preference_loss";
  same_gpu(what, logits, {&tokens, &reference_});
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK_VALUE(logits.dim() == 3 && logits.size(0) % 2 == 0, what, ": logits (2 n, T, V) expected, got ", logits.sizes());
  const Rows a(what, logits, tokens);
  const int64_t pairs = a.B / 2;
  Tensor reference = reference_;
  if (reference.defined()) {
    same_count(what, "the reference", reference.numel(), 2 * pairs);
    reference = (reference.scalar_type() == at::kDouble ? reference : reference.to(at::kFloat)).contiguous();
  }
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  Loss o;
  o.loss = f.reduction ? at::empty({}, f32) : at::empty({pairs}, f32);
  o.values = at::empty({2 * pairs}, f32);
  const int64_t bytes = lib.dh_preference_workspace_bytes(a.code, pairs, narrow(a.T), a.V);
  const Buffer buffer(preference_kept(a.n, pairs), bytes, f32);
  o.kept = buffer.kept;
  float* kept = buffer.at;
  check(lib.dh_preference_fwd(a.code, a.z.data_ptr(), a.sb, a.st, pairs, narrow(a.T), a.V, a.tokens.data_ptr(), a.token_bits,
                              f.ignore_index, at_(reference), reference.defined() && reference.scalar_type() == at::kDouble ? 64 : 32,
                              narrow(f.kind), f.average, f.beta, f.margin, f.smoothing, narrow(f.reduction),
                              f.reduction ? nullptr : floats(o.loss), floats(o.values), kept + 4 * a.n, kept,
                              f.reduction ? floats(o.loss) : nullptr, kept + 4 * a.n + 2 * pairs, buffer.scratch, bytes,
                              stream_of(logits)),
        what);
  return o;
}

Tensor preference_grad(const Tensor& grad, const Tensor& logits, const Tensor& tokens, const Tensor& kept_, int64_t ignore_index,
                       int64_t reduction) {
  const char* what = "preference_loss gradient";
  same_gpu(what, logits, {&grad, &tokens, &kept_});
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK_VALUE(logits.dim() == 3 && logits.size(0) % 2 == 0, what, ": logits (2 n, T, V) expected, got ", logits.sizes());
  const Rows a(what, logits, tokens);
  const int64_t pairs = a.B / 2;
  const Tensor kept = kept_rows(what, kept_, preference_kept(a.n, pairs)), g = grad.to(at::kFloat).reshape({-1});
  same_count(what, "the loss's gradient", g.numel(), reduction ? 1 : pairs);
  Upstream u;
  u.by_lp = floats(kept) + 4 * a.n;
  u.lp_div = a.T > 0 ? a.T : 1;
  u.g = floats(g);
  if (reduction) {
    u.divisor = u.by_lp + 2 * pairs;
  } else {
    u.g_div = u.lp_div, u.g_mod = pairs > 0 ? pairs : 1, u.g_stride = pairs ? g.stride(0) : 0;
  }
  return rows_grad(what, a, logits, 1.0, ignore_index, floats(kept), u);
}

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                               const std::optional<Tensor>& reference_, int64_t kind, bool average, double beta, double margin,
                               double smoothing, int64_t ignore_index, int64_t reduction) {
    const Tensor reference = reference_ ? *reference_ : Tensor();
    const Loss o = preference(logits, tokens, reference, Preference{kind, average, beta, margin, smoothing, ignore_index, reduction});
    ctx->set_materialize_grads(false);
    if (logits.requires_grad()) ctx->save_for_backward({logits, savable(tokens), savable(reference), o.kept});
    ctx->mark_non_differentiable({o.values});
    ctx->saved_data["numbers"] = std::vector<double>{beta, margin, smoothing};
    ctx->saved_data["whole"] = std::vector<int64_t>{kind, average, ignore_index, reduction};
    return {o.loss, o.values};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(10);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto f = ctx->saved_data["numbers"].toDoubleVector();
    const auto i = ctx->saved_data["whole"].toIntVector();
    out[0] = at::GradMode::is_enabled()
                 ? by_torch(again_preference, saved[0], saved[1], maybe(saved[2]), i[0], i[1] != 0, f[0], f[1], f[2], i[2], i[3],
                            grads[0])
                 : preference_grad(grads[0], saved[0], saved[1], saved[3], i[2], i[3]);
    return out;
  }
};

// ---- policy loss --------------------------------------------------------------------------------------------------------
struct Policy {
  double clip, clip_high, kl, entropy, temperature;
  int64_t ignore_index, reduction;         // reduction: 0 none, 1 mean, 2 sum, 3 mean of the sequences' means
};
int64_t policy_kept(int64_t n, double entropy) { return (entropy != 0.0 ? 6 : 5) * n + 1; }

Loss policy(const Tensor& logits, const Tensor& tokens, const Tensor& old_, const Tensor& advantages_, const Tensor& reference_,
            const Policy& f) {
  const char* what = "policy_loss";
  same_gpu(what, logits, {&tokens, &old_, &advantages_, &reference_});
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK_VALUE(logits.dim() >= 2, what, ": logits (..., T, V) expected, got ", logits.sizes());
  const Rows a(what, logits, tokens);
  const Tensor old = numbers(old_), advantages = numbers(advantages_), reference = numbers(reference_);
  same_count(what, "the old log-probabilities", old.numel(), a.n);
  if (reference.defined()) same_count(what, "the reference", reference.numel(), a.n);
  const bool per_sequence = advantages_.dim() < tokens.dim();
  same_count(what, "the advantages", advantages.numel(), per_sequence ? a.B : a.n);
  const bool ent = f.entropy != 0.0;
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  Loss o;
  o.loss = f.reduction ? at::empty({}, f32) : at::empty(shape, f32);
  o.values = at::empty(shape, f32);
  const int64_t bytes = lib.dh_policy_workspace_bytes(a.code, a.B, narrow(a.T), a.V, ent);
  const Buffer buffer(policy_kept(a.n, f.entropy), bytes, f32);
  o.kept = buffer.kept;
  float* kept = buffer.at;
  check(lib.dh_policy_fwd(a.code, a.z.data_ptr(), a.sb, a.st, a.B, narrow(a.T), a.V, a.tokens.data_ptr(), a.token_bits,
                          f.ignore_index, f.temperature, floats(old), floats(advantages), per_sequence, floats(reference), f.clip,
                          f.clip_high, f.kl, f.entropy, narrow(f.reduction), f.reduction ? nullptr : floats(o.loss),
                          floats(o.values), kept + 4 * a.n, ent ? kept + 5 * a.n : nullptr, kept,
                          f.reduction ? floats(o.loss) : nullptr, kept + (ent ? 6 : 5) * a.n, buffer.scratch, bytes, stream_of(logits)),
        what);
  return o;
}

Tensor policy_grad(const Tensor& grad, const Tensor& logits, const Tensor& tokens, const Tensor& kept_, double entropy,
                   double temperature, int64_t ignore_index, int64_t reduction) {
  const char* what = "policy_loss gradient";
  same_gpu(what, logits, {&grad, &tokens, &kept_});
  const c10::DeviceGuard guard(logits.device());
  const Rows a(what, logits, tokens);
  const Tensor kept = kept_rows(what, kept_, policy_kept(a.n, entropy)), g = grad.to(at::kFloat).reshape({-1});
  same_count(what, "the loss's gradient", g.numel(), reduction ? 1 : a.n);
  Upstream u;
  u.by_lp = floats(kept) + 4 * a.n;
  if (entropy != 0.0) u.by_ent = floats(kept) + 5 * a.n;
  u.g = floats(g);
  if (reduction) {
    u.divisor = floats(kept) + (entropy != 0.0 ? 6 : 5) * a.n;
  } else {
    u.g_mod = a.n > 0 ? a.n : 1, u.g_stride = a.n ? g.stride(0) : 0;
  }
  return rows_grad(what, a, logits, temperature, ignore_index, floats(kept), u);
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const Tensor& old,
                               const Tensor& advantages, const std::optional<Tensor>& reference_, double clip, double clip_high,
                               double kl, double entropy, double temperature, int64_t ignore_index, int64_t reduction) {
    const Tensor reference = reference_ ? *reference_ : Tensor();
    const Loss o = policy(logits, tokens, old, advantages, reference,
                          Policy{clip, clip_high, kl, entropy, temperature, ignore_index, reduction});
    ctx->set_materialize_grads(false);
    if (logits.requires_grad())
      ctx->save_for_backward({logits, savable(tokens), savable(old), savable(advantages), savable(reference), o.kept});
    ctx->mark_non_differentiable({o.values});
    ctx->saved_data["numbers"] = std::vector<double>{clip, clip_high, kl, entropy, temperature};
    ctx->saved_data["whole"] = std::vector<int64_t>{ignore_index, reduction};
    return {o.loss, o.values};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(12);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto f = ctx->saved_data["numbers"].toDoubleVector();
    const auto i = ctx->saved_data["whole"].toIntVector();
    out[0] = at::GradMode::is_enabled()
                 ? by_torch(again_policy, saved[0], saved[1], saved[2], saved[3], maybe(saved[4]), f[0], f[1], f[2], f[3], f[4], i[0],
                            i[1], grads[0])
                 : policy_grad(grads[0], saved[0], saved[1], saved[5], f[3], f[4], i[0], i[1]);
    return out;
  }
};

}  // namespace

void bind_logprobs(py::module_& m) {
  m.def("bind_logprobs", [](py::object logprobs_, py::object preference_, py::object policy_) {
    again_logprobs = new py::object(std::move(logprobs_));
    again_preference = new py::object(std::move(preference_));
    again_policy = new py::object(std::move(policy_));
  });
  using release = py::call_guard<py::gil_scoped_release>;
  using Maybe = std::optional<Tensor>;
  // the launches alone, for the registered operations
  m.def("logprobs", [](const Tensor& logits, const Tensor& tokens, double temperature, int64_t ignore_index, bool entropy) {
    return guarded([&] { return logprobs(logits, tokens, temperature, ignore_index, entropy, true); });
  }, release());
  m.def("logprobs_grad", [](const Maybe& g_lp, const Maybe& g_ent, const Tensor& logits, const Tensor& tokens, const Tensor& kept,
                            double temperature, int64_t ignore_index) {
    return guarded([&] {
      return logprobs_grad(g_lp.value_or(Tensor()), g_ent.value_or(Tensor()), logits, tokens, kept, temperature, ignore_index);
    });
  }, release());
  m.def("head_logprobs", [](const Tensor& hidden, const Tensor& weight, const Tensor& tokens, double temperature,
                            int64_t ignore_index, bool entropy, bool round_logits) {
    return guarded([&] { return head_logprobs(hidden, weight, tokens, temperature, ignore_index, entropy, round_logits); });
  }, release());
  m.def("preference", [](const Tensor& logits, const Tensor& tokens, const Maybe& reference, int64_t kind, bool average, double beta,
                         double margin, double smoothing, int64_t ignore_index, int64_t reduction) {
    return guarded([&] {
      const Loss o = preference(logits, tokens, reference.value_or(Tensor()),
                                Preference{kind, average, beta, margin, smoothing, ignore_index, reduction});
      return std::make_tuple(o.loss, o.values, o.kept);
    });
  }, release());
  m.def("preference_grad", [](const Tensor& g, const Tensor& logits, const Tensor& tokens, const Tensor& kept, int64_t ignore_index,
                              int64_t reduction) {
    return guarded([&] { return preference_grad(g, logits, tokens, kept, ignore_index, reduction); });
  }, release());
  m.def("policy", [](const Tensor& logits, const Tensor& tokens, const Tensor& old, const Tensor& advantages, const Maybe& reference,
                     double clip, double clip_high, double kl, double entropy, double temperature, int64_t ignore_index,
                     int64_t reduction) {
    return guarded([&] {
      const Loss o = policy(logits, tokens, old, advantages, reference.value_or(Tensor()),
                            Policy{clip, clip_high, kl, entropy, temperature, ignore_index, reduction});
      return std::make_tuple(o.loss, o.values, o.kept);
    });
  }, release());
  m.def("policy_grad", [](const Tensor& g, const Tensor& logits, const Tensor& tokens, const Tensor& kept, double entropy,
                          double temperature, int64_t ignore_index, int64_t reduction) {
    return guarded([&] { return policy_grad(g, logits, tokens, kept, entropy, temperature, ignore_index, reduction); });
  }, release());
  // with their nodes
  m.def("token_logprobs", [](const Tensor& logits, const Tensor& tokens, double temperature, int64_t ignore_index, bool entropy) {
    return guarded([&] { return TokenLogprobs::apply(logits, tokens, temperature, ignore_index, entropy); });
  }, release());
  m.def("preference_loss", [](const Tensor& logits, const Tensor& tokens, const Maybe& reference, int64_t kind, bool average,
                              double beta, double margin, double smoothing, int64_t ignore_index, int64_t reduction) {
    return guarded([&] {
      return PreferenceLoss::apply(logits, tokens, reference, kind, average, beta, margin, smoothing, ignore_index, reduction);
    });
  }, release());
  m.def("policy_loss", [](const Tensor& logits, const Tensor& tokens, const Tensor& old, const Tensor& advantages,
                          const Maybe& reference, double clip, double clip_high, double kl, double entropy, double temperature,
                          int64_t ignore_index, int64_t reduction) {
    return guarded([&] {
      return PolicyLoss::apply(logits, tokens, old, advantages, reference, clip, clip_high, kl, entropy, temperature, ignore_index,
                               reduction);
    });
  }, release());
}

// The vocabulary-end operators as autograd nodes in C++: what fused_vocab.py calls in plain eager execution.
//
// Their backward passes run on autograd's thread for the device, and nodes in Python hand the interpreter over twice a pass:
// lookup and gradient of 200 embedding rows took 90 us with them, of which the kernels are 9, and take 48 with these (torch's
// own 52 in the same process). The kernels are the C entry points of libdh_mixer.so, bound by address by the module that loads that library; nothing here
// computes.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <map>
#include <optional>
#include <string>

#include "dh_mixer.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

namespace {

#define ENTRIES(X)                                                                                                     \
  X(dh_embed_fwd) X(dh_embed_bwd) X(dh_embed_bwd_workspace_bytes) X(dh_top_logits) X(dh_distill_fwd) X(dh_distill_bwd) \
      X(dh_distill_workspace_bytes) X(dh_last_error)
#define MEMBER(name) decltype(&::name) name = nullptr;
struct Entries {
  ENTRIES(MEMBER)
} lib;
#undef MEMBER

// never freed: they outlive us
py::object* again = nullptr;               // the differentiable gradient as torch operations
py::object* out_of_memory = nullptr;       // torch.OutOfMemoryError

void check(int status, const char* what) {
  if (status == 0) return;
  const char* text = lib.dh_last_error();
  TORCH_CHECK_VALUE(status != DH_ERR_INVALID_ARG, what, " failed (INVALID_ARG): ", text);
  TORCH_CHECK_VALUE(status != DH_ERR_UNSUPPORTED_SHAPE, what, " failed (UNSUPPORTED_SHAPE): ", text);
  TORCH_CHECK_TYPE(status != DH_ERR_UNSUPPORTED_DTYPE, what, " failed (UNSUPPORTED_DTYPE): ", text);
  TORCH_CHECK(false, what, " failed (", status == DH_ERR_LAUNCH_FAILED ? "LAUNCH_FAILED" : "UNKNOWN", "): ", text);
}

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return DH_F32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "dispatcher kernels support float32 and bfloat16, got torch.",
                   c10::toString(t.scalar_type()));
  return DH_BF16;
}

void require_gpu(const char* what, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), what, ": tensors must be on the GPU (got device ", t.device(),
              "); the fused paths have no CPU implementation");
}
void same_gpu(const char* what, const Tensor& x, std::initializer_list<const Tensor*> others) {
  require_gpu(what, x);
  for (const Tensor* t : others)
    TORCH_CHECK(!t->defined() || t->device() == x.device(), what, ": all tensors must be on one device (got ", x.device(),
                " and ", t->device(), ")");
}

// the current stream of a device; made with that device as the current one
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int bits(const char* what, const Tensor& t) {
  if (t.scalar_type() == at::kInt) return 32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong, what, ": integers must be int32 or int64, got torch.",
                   c10::toString(t.scalar_type()));
  return 64;
}
// A kernel reads as much as the sizes say, so every launch checks them, whoever calls it (a registered operation by its name,
// a saved-tensor hook that hands back another tensor).
void same_count(const char* what, const char* which, int64_t has, int64_t needs) {
  TORCH_CHECK_VALUE(has == needs, what, ": ", which, " of ", has, " elements, ", needs, " needed");
}

// for the entry points' ints: what does not fit is -1, which they refuse
int narrow(int64_t v) { return v >= 0 && v <= INT32_MAX ? (int)v : -1; }

Tensor fresh(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
// unit-stride rows (any other layout copied); broadcast rows stay
Tensor unit_rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// ---- embedding ------------------------------------------------------------------------------------------------------
Tensor lookup(const Tensor& weight, const Tensor& tokens, double scale, int64_t zero_token) {
  const char* what = "embed_tokens";
  same_gpu(what, weight, {&tokens});
  const int code = dtype_code(weight);
  TORCH_CHECK_VALUE(weight.dim() == 2, what, ": weight (V, d) expected, got ", weight.sizes());
  const int64_t V = weight.size(0), d = weight.size(1);
  const c10::DeviceGuard guard(weight.device());
  const Tensor w = weight.stride(1) == 1 && weight.stride(0) >= d ? weight : fresh(weight);
  const Tensor ids = tokens.contiguous();
  auto shape = tokens.sizes().vec();
  shape.push_back(d);
  Tensor out = at::empty(shape, weight.options());
  const int id_bits = bits(what, ids);
  check(lib.dh_embed_fwd(code, w.data_ptr(), w.stride(0), V, narrow(d), ids.data_ptr(), id_bits, ids.numel(),
                         (float)scale, zero_token, out.data_ptr(), d, stream_of(w)),
        what);
  return out;
}

Tensor lookup_grad(const Tensor& dy, const Tensor& tokens, int64_t rows, double scale, int64_t skip_token) {
  const char* what = "embed_tokens gradient";
  same_gpu(what, dy, {&tokens});
  const int code = dtype_code(dy);
  const int64_t d = dy.size(-1);
  const c10::DeviceGuard guard(dy.device());
  const Tensor ids = tokens.contiguous();
  const int id_bits = bits(what, ids);
  same_count(what, "dy", dy.numel(), ids.numel() * d);
  TORCH_CHECK_VALUE(rows >= 1, what, ": a vocabulary of ", rows);
  Tensor y = dy.dim() == 2 ? dy : dy.reshape({-1, d});
  if (y.stride(1) != 1 || y.stride(0) < d) y = fresh(y);
  Tensor out = at::empty({rows, d}, dy.options());
  const int width = narrow(d);
  const int64_t bytes = lib.dh_embed_bwd_workspace_bytes(ids.numel(), rows, width);
  Tensor ws;                                                   // (refused sizes: the call says why)
  if (bytes > 0) ws = at::empty({bytes}, dy.options().dtype(at::kByte));
  check(lib.dh_embed_bwd(code, y.data_ptr(), y.stride(0), ids.data_ptr(), id_bits, ids.numel(), rows, width, (float)scale,
                         skip_token, out.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr, bytes, stream_of(dy)),
        what);
  return out;
}

struct Embed : torch::autograd::Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, double scale, int64_t zero_token,
                        int64_t skip_token) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["skip"] = skip_token;
    return lookup(weight, tokens, scale, zero_token);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads);
};

// linear in dy: its own gradient looks the rows of g up, zeros where positions were left out
struct EmbedGrad : torch::autograd::Function<EmbedGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dy, const Tensor& tokens, int64_t rows, double scale,
                        int64_t skip_token) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["skip"] = skip_token;
    return lookup_grad(dy, tokens, rows, scale, skip_token);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const Tensor tokens = ctx->get_saved_variables()[0], g = grads[0];
    const int64_t skip = ctx->saved_data["skip"].toInt();
    return {Embed::apply(g, tokens, ctx->saved_data["scale"].toDouble(), skip >= 0 ? skip : g.size(0), skip), Variable(),
            Variable(), Variable(), Variable()};
  }
};

variable_list Embed::backward(AutogradContext* ctx, const variable_list& grads) {
  const Tensor tokens = ctx->get_saved_variables()[0];
  const int64_t rows = ctx->saved_data["rows"].toInt(), skip = ctx->saved_data["skip"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  return {at::GradMode::is_enabled() ? EmbedGrad::apply(grads[0], tokens, rows, scale, skip)
                                     : lookup_grad(grads[0], tokens, rows, scale, skip),
          Variable(), Variable(), Variable(), Variable()};
}

// ---- a teacher's targets --------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> top_logits(const Tensor& logits, int64_t k) {
  const char* what = "top_logits";
  require_gpu(what, logits);
  const int code = dtype_code(logits);
  const int64_t V = logits.size(-1);
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(logits.device());
  const Tensor rows = unit_rows(logits.dim() == 2 ? logits : logits.reshape({-1, V}));
  auto shape = logits.sizes().vec();
  shape.back() = k;
  Tensor values = at::empty(shape, logits.options().requires_grad(false)),
         tokens = at::empty(shape, logits.options().dtype(at::kLong).requires_grad(false));
  check(lib.dh_top_logits(code, rows.data_ptr(), rows.stride(0), rows.size(0), narrow(V), narrow(k),
                          values.data_ptr(), tokens.data_ptr<int64_t>(), stream_of(logits)),
        what);
  return {values, tokens};
}

// ---- distillation loss ----------------------------------------------------------------------------------------------
struct Mix {                               // what the loss is mixed from
  double temperature, weight;
  int64_t ignore_index, reduction;         // reduction: 0 none, 1 mean, 2 sum
};

// the arguments both directions share, and the tensors they point to
struct Rows {
  Tensor z, t_logits, t_tokens, labels;
  int64_t sb = 0, st = 0, B = 1, T = 1, n = 1;
  int code, t_code, V, token_bits, label_bits = 64;
  Rows(const char* what, const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_tokens, const Tensor& lb)
      : z(unit_rows(logits)),
        t_logits(teacher_logits.contiguous()),
        t_tokens(teacher_tokens.contiguous()),
        labels(lb.defined() ? lb.contiguous() : lb),
        code(dtype_code(logits)),
        t_code(dtype_code(teacher_logits)),
        V(narrow(logits.size(-1))) {
    if (z.dim() > 3) z = unit_rows(z.reshape({-1, z.size(-1)}));
    if (z.dim() == 3) {
      B = z.size(0), T = z.size(1), sb = z.stride(0), st = z.stride(1);
    } else if (z.dim() == 2) {
      T = z.size(0), st = z.stride(0);
    }
    n = B * T;
    if (n == 0) B = 0, T = 1;
    TORCH_CHECK_VALUE(n < (1 << 22), what, ": ", n, " rows, fewer than ", 1 << 22, " possible");
    token_bits = bits(what, t_tokens);
    same_count(what, "teacher logits", t_logits.numel(), n * K());
    same_count(what, "teacher tokens", t_tokens.numel(), n * K());
    if (labels.defined()) {
      label_bits = bits(what, labels);
      same_count(what, "labels", labels.numel(), n);
    }
  }
  int64_t K() const { return t_logits.size(-1); }
  void* label_ptr() const { return labels.defined() ? labels.data_ptr() : nullptr; }
};

// (loss, kept): kept holds four numbers a row and the divisor, and behind them the rows' losses where they are no result and
// the workspace
std::tuple<Tensor, Tensor> distill(const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_tokens,
                                   const Tensor& labels, const Mix& m) {
  const char* what = "distillation_loss";
  same_gpu(what, logits, {&teacher_logits, &teacher_tokens, &labels});
  const c10::DeviceGuard guard(logits.device());
  const Rows a(what, logits, teacher_logits, teacher_tokens, labels);
  const int64_t n = a.n;
  const auto f32 = logits.options().dtype(at::kFloat);
  // the loss apart: it may be changed in place
  Tensor out = m.reduction ? at::empty({}, f32) : at::empty(logits.sizes().slice(0, logits.dim() - 1), f32);
  const int64_t bytes = lib.dh_distill_workspace_bytes(a.code, n, a.V);
  const int64_t first = 4 * n + 4, rows = m.reduction ? (n + 3) / 4 * 4 : 0;
  Tensor kept = at::empty({first + rows + (bytes + 3) / 4}, f32);
  float* at_ = kept.data_ptr<float>();
  check(lib.dh_distill_fwd(a.code, a.z.data_ptr(), a.sb, a.st, a.B, (int)a.T, a.V, a.t_code, a.t_logits.data_ptr(),
                           a.t_tokens.data_ptr(), a.token_bits, narrow(a.K()), a.label_ptr(), a.label_bits,
                           m.ignore_index, (float)m.temperature, (float)m.weight, narrow(m.reduction),
                           m.reduction ? at_ + first : out.data_ptr<float>(), at_, m.reduction ? out.data_ptr<float>() : nullptr,
                           m.reduction ? at_ + 4 * n : nullptr, at_ + first + rows, bytes, stream_of(logits)),
        what);
  return {out, kept};
}

Tensor distill_grad(const Tensor& grad, const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_tokens,
                    const Tensor& labels, const Tensor& kept_, const Mix& m) {
  const char* what = "distillation_loss gradient";
  same_gpu(what, logits, {&grad, &teacher_logits, &teacher_tokens, &labels, &kept_});
  const c10::DeviceGuard guard(logits.device());
  Tensor dz = at::empty(logits.sizes(), logits.options());
  if (dz.numel() == 0) return dz;
  const Rows a(what, logits, teacher_logits, teacher_tokens, labels);
  const Tensor g = grad.to(at::kFloat).reshape({-1});
  same_count(what, "the loss's gradient", g.numel(), m.reduction ? 1 : a.n);
  TORCH_CHECK_VALUE(kept_.numel() >= 4 * a.n + 4, what, ": ", kept_.numel(), " numbers kept of ", a.n, " rows");
  Tensor kept = kept_;                                         // (a saved-tensor hook may change the layout)
  if (!kept.is_contiguous() || reinterpret_cast<uintptr_t>(kept.data_ptr()) % 16) kept = fresh(kept);
  const float* at_ = kept.data_ptr<float>();
  check(lib.dh_distill_bwd(a.code, a.z.data_ptr(), a.sb, a.st, a.B, (int)a.T, a.V, a.t_code, a.t_logits.data_ptr(),
                           a.t_tokens.data_ptr(), a.token_bits, narrow(a.K()), a.label_ptr(), a.label_bits,
                           m.ignore_index, (float)m.temperature, (float)m.weight, at_, g.data_ptr<float>(),
                           m.reduction ? 0 : g.stride(0), m.reduction ? at_ + 4 * a.n : nullptr, dz.data_ptr(),
                           stream_of(logits)),
        what);
  return dz;
}

// targets and labels made under inference mode (a teacher's, say) cannot be saved for a backward pass: copies of them can
Tensor savable(const Tensor& t) { return t.defined() && t.is_inference() ? t.clone() : t; }

struct Distill : torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_tokens,
                        const std::optional<Tensor>& labels, double temperature, double weight, int64_t ignore_index,
                        int64_t reduction) {
    const Tensor lb = labels ? *labels : Tensor();
    auto [out, kept] = distill(logits, teacher_logits, teacher_tokens, lb, Mix{temperature, weight, ignore_index, reduction});
    ctx->set_materialize_grads(false);
    if (logits.requires_grad())
      ctx->save_for_backward({logits, savable(teacher_logits), savable(teacher_tokens), savable(lb), kept});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["weight"] = weight;
    ctx->saved_data["ignore"] = ignore_index;
    ctx->saved_data["reduction"] = reduction;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(8);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Mix m{ctx->saved_data["temperature"].toDouble(), ctx->saved_data["weight"].toDouble(),
                ctx->saved_data["ignore"].toInt(), ctx->saved_data["reduction"].toInt()};
    if (!at::GradMode::is_enabled()) {
      out[0] = distill_grad(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], m);
      return out;
    }
    const py::gil_scoped_acquire gil;
    try {
      const std::optional<Tensor> labels = saved[3].defined() ? std::optional<Tensor>(saved[3]) : std::nullopt;
      out[0] = (*again)(saved[0], saved[1], saved[2], labels, m.temperature, m.weight, m.ignore_index, m.reduction, grads[0])
                   .cast<Tensor>();
    } catch (py::error_already_set& e) {   // (it must not outlive the lock it is held under)
      TORCH_CHECK(false, e.what());
    }
    return out;
  }
};

// errors as Python's of the same kind
template <typename F>
auto guarded(F&& f) {
  try {
    return f();
  } catch (const c10::ValueError& e) {
    throw py::value_error(e.what_without_backtrace());
  } catch (const c10::TypeError& e) {
    throw py::type_error(e.what_without_backtrace());
  } catch (const c10::OutOfMemoryError& e) {                   // (what a training loop catches to try a smaller batch)
    const py::gil_scoped_acquire gil;
    PyErr_SetString(out_of_memory->ptr(), e.what_without_backtrace());
    throw py::error_already_set();
  } catch (const c10::Error& e) {
    throw std::runtime_error(e.what_without_backtrace());
  }
}

}  // namespace

PYBIND11_MODULE(_vocab_nodes, m) {
  // what this was compiled against, for the loader to compare before anything is called
  m.attr("abi_version") = DH_ABI_VERSION;
  m.attr("torch_version") = DH_TORCH_VERSION;
  m.def("bind", [](const std::map<std::string, uintptr_t>& at, py::object differentiable) {
#define ENTRY(name) lib.name = reinterpret_cast<decltype(&::name)>(at.at(#name));
    ENTRIES(ENTRY)
#undef ENTRY
    again = new py::object(std::move(differentiable));
    out_of_memory = new py::object(py::module_::import("torch").attr("OutOfMemoryError"));
  });
  using release = py::call_guard<py::gil_scoped_release>;
  // the launches alone, for the registered operations
  m.def("lookup", [](const Tensor& weight, const Tensor& tokens, double scale, int64_t zero_token) {
    return guarded([&] { return lookup(weight, tokens, scale, zero_token); });
  }, release());
  m.def("lookup_grad", [](const Tensor& dy, const Tensor& tokens, int64_t rows, double scale, int64_t skip_token) {
    return guarded([&] { return lookup_grad(dy, tokens, rows, scale, skip_token); });
  }, release());
  m.def("distill",
        [](const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_tokens, const std::optional<Tensor>& labels,
           double temperature, double weight, int64_t ignore_index, int64_t reduction) {
          return guarded([&] {
            return distill(logits, teacher_logits, teacher_tokens, labels.value_or(Tensor()),
                           Mix{temperature, weight, ignore_index, reduction});
          });
        },
        release());
  m.def("distill_grad",
        [](const Tensor& g, const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_tokens,
           const std::optional<Tensor>& labels, const Tensor& kept, double temperature, double weight, int64_t ignore_index,
           int64_t reduction) {
          return guarded([&] {
            return distill_grad(g, logits, teacher_logits, teacher_tokens, labels.value_or(Tensor()), kept,
                                Mix{temperature, weight, ignore_index, reduction});
          });
        },
        release());
  // with their nodes
  m.def("embed_tokens", [](const Tensor& weight, const Tensor& tokens, double scale, int64_t zero_token, int64_t skip_token) {
    return guarded([&] { return Embed::apply(weight, tokens, scale, zero_token, skip_token); });
  }, release());
  m.def("top_logits", [](const Tensor& logits, int64_t k) { return guarded([&] { return top_logits(logits, k); }); }, release());
  m.def("distillation_loss",
        [](const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_tokens, const std::optional<Tensor>& labels,
           double temperature, double weight, int64_t ignore_index, int64_t reduction) {
          return guarded([&] {
            return Distill::apply(logits, teacher_logits, teacher_tokens, labels, temperature, weight, ignore_index, reduction);
          });
        },
        release());
}

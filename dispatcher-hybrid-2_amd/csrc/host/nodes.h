// What the C++ nodes of this folder share: the library's entry points, its errors as torch's, the checks before a launch.
#pragma once

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

#define ENTRIES(X)                                                                                                       \
  X(dh_embed_fwd) X(dh_embed_bwd) X(dh_embed_bwd_workspace_bytes) X(dh_top_logits) X(dh_distill_fwd) X(dh_distill_bwd)   \
      X(dh_distill_workspace_bytes) X(dh_logprob_fwd) X(dh_logprob_bwd) X(dh_logprob_workspace_bytes)                    \
          X(dh_preference_fwd) X(dh_preference_workspace_bytes) X(dh_policy_fwd) X(dh_policy_workspace_bytes)            \
              X(dh_head_logprob) X(dh_head_logprob_workspace_bytes) X(dh_last_error)
#define MEMBER(name) decltype(&::name) name = nullptr;
struct Entries {
  ENTRIES(MEMBER)
};
#undef MEMBER
extern Entries lib;

// never freed: they outlive us
extern py::object* out_of_memory;          // torch.OutOfMemoryError

inline void check(int status, const char* what) {
  if (status == 0) return;
  const char* text = lib.dh_last_error();
  TORCH_CHECK_VALUE(status != DH_ERR_INVALID_ARG, what, " failed (INVALID_ARG): ", text);
  TORCH_CHECK_VALUE(status != DH_ERR_UNSUPPORTED_SHAPE, what, " failed (UNSUPPORTED_SHAPE): ", text);
  TORCH_CHECK_TYPE(status != DH_ERR_UNSUPPORTED_DTYPE, what, " failed (UNSUPPORTED_DTYPE): ", text);
  TORCH_CHECK(false, what, " failed (", status == DH_ERR_LAUNCH_FAILED ? "LAUNCH_FAILED" : "UNKNOWN", "): ", text);
}

inline int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return DH_F32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "dispatcher kernels support float32 and bfloat16, got torch.",
                   c10::toString(t.scalar_type()));
  return DH_BF16;
}

inline void require_gpu(const char* what, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), what, ": tensors must be on the GPU (got device ", t.device(),
              "); the fused paths have no CPU implementation");
}
inline void same_gpu(const char* what, const Tensor& x, std::initializer_list<const Tensor*> others) {
  require_gpu(what, x);
  for (const Tensor* t : others)
    TORCH_CHECK(!t->defined() || t->device() == x.device(), what, ": all tensors must be on one device (got ", x.device(),
                " and ", t->device(), ")");
}

// the current stream of a device; made with that device as the current one
inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

inline int bits(const char* what, const Tensor& t) {
  if (t.scalar_type() == at::kInt) return 32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong, what, ": integers must be int32 or int64, got torch.",
                   c10::toString(t.scalar_type()));
  return 64;
}
// A kernel reads as much as the sizes say, so every launch checks them, whoever calls it (a registered operation by its name,
// a saved-tensor hook that hands back another tensor).
inline void same_count(const char* what, const char* which, int64_t has, int64_t needs) {
  TORCH_CHECK_VALUE(has == needs, what, ": ", which, " of ", has, " elements, ", needs, " needed");
}

// for the entry points' ints: what does not fit is -1, which they refuse
inline int narrow(int64_t v) { return v >= 0 && v <= INT32_MAX ? (int)v : -1; }

inline Tensor fresh(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
// unit-stride rows (any other layout copied); broadcast rows stay
inline Tensor unit_rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// constants made under inference mode (a teacher's targets, say) cannot be saved for a backward pass: copies of them can
inline Tensor savable(const Tensor& t) { return t.defined() && t.is_inference() ? t.clone() : t; }

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

// bindings of the other files
void bind_logprobs(py::module_& m);

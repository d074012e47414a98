// What the host sides in C++ share: the library's entry points looked up by name, its errors as torch's, tensors as the entry
// points take them, and what their autograd nodes refuse.
#pragma once

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>

#include "cdssm_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library that the Python side has loaded (its path may be another build's).
inline decltype(&cdssm_last_error) last_error;
struct Library {
  void* handle;
  const std::string& path;
  explicit Library(const std::string& p) : handle(dlopen(p.c_str(), RTLD_NOW)), path(p) {
    TORCH_CHECK(handle, path, ": ", dlerror());
    get(last_error, "cdssm_last_error");
  }
  template <typename F>
  void get(F& f, const char* name) const {
    f = reinterpret_cast<F>(dlsym(handle, name));
    TORCH_CHECK(f, path, " has no ", name);
  }
};

inline hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
inline int code_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
inline int id_bytes(const Tensor& t) { return t.scalar_type() == at::kLong ? 8 : 4; }

inline void ok(int status, const char* name) {
  TORCH_CHECK(status == 0, name, " failed (status ", status, "): ", last_error());
}
inline int64_t bytes(int64_t n, const char* op) {
  TORCH_CHECK_VALUE(n >= 0, op, ": ", last_error());
  return n;
}

// Forward-mode derivatives are not computed, and not passed by in silence.
inline void no_tangent(const char* op, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), op, " has no forward-mode derivative");
}

// t (..., C) as (rows, C) with dense columns and a row stride of at least C, copied only where it has to be.
inline Tensor rows_of(const Tensor& t) {
  const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  if (r.is_contiguous()) return r;
  const bool dense = (r.size(1) == 1 || r.stride(1) == 1) && (r.size(0) <= 1 || r.stride(0) >= r.size(1));
  return dense ? r : r.contiguous();
}
// Any row stride will do for a single row, whose own may be beyond what the entry points take.
constexpr int64_t kRowStride = int64_t(1) << 22;
inline int64_t row_stride(const Tensor& t) {
  if (t.size(0) != 1) return t.stride(0);
  return t.stride(0) > kRowStride ? t.size(1) : std::max(t.stride(0), t.size(1));
}

inline Tensor workspace(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// The gradients of a backward, which cannot be differentiated themselves: a derivative of theirs, by what they were made
// from, raises.
inline variable_list once(const char* op, variable_list grads, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads) {
    if (!g.defined()) continue;
    variable_list in{g.requires_grad_()};
    in.insert(in.end(), from.begin(), from.end());
    const auto error =
        std::make_shared<torch::autograd::DelayedError>(std::string(op) + " has no second derivative", int64_t(in.size()));
    g = (*error)(std::move(in))[0];
  }
  return grads;
}

}  // namespace

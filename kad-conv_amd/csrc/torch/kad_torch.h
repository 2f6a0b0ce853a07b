// What the files of kadconv._native share.
#pragma once
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/FunctionsManual.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <string_view>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "kadconv_hip.h"

namespace kad_torch {


using at::Tensor;
using OptTensor = std::optional<Tensor>;

inline void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", kad_last_error()); }

inline void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KAD_F32;
    case at::kHalf: return KAD_F16;
    case at::kBFloat16: return KAD_BF16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type(), "; expected float32, float16 or bfloat16");
  }
}

inline Tensor defined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
inline Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
inline const void* pointer(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline void* mutable_pointer(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A dense channels-last map of x's shape, dtype and device.
inline Tensor map_like(const Tensor& x) {
  const int64_t n = x.size(0), c = x.size(1), h = x.size(2), w = x.size(3);
  return at::detail::empty_strided_cuda({n, c, h, w}, {h * w * c, 1, w * c, c}, x.scalar_type(), x.device());
}

inline Tensor floats(const Tensor& x, at::IntArrayRef sizes) {
  return at::detail::empty_cuda(sizes, at::kFloat, x.device(), std::nullopt);
}

// Whether calls are watched (a trace, a dispatch mode) or a tensor stands for another (fake, wrapped, or a view that
// negates what is stored): the caller then takes the registered operator, which such a program sees and which is given
// the values themselves.  What is allocated and launched here, it would not see.
inline bool observed(std::initializer_list<const Tensor*> tensors) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set()) return true;
  for (const Tensor* t : tensors)
    if (t->defined() && (!t->has_storage() || t->key_set().has(c10::DispatchKey::Python) || t->is_neg() || t->_is_zerotensor()))
      return true;
  return false;
}

// The activation's number, after its check.
inline int checked_act(const std::optional<std::string_view>& act) {
  TORCH_CHECK_VALUE(!act || *act == "relu" || *act == "silu", "act '", act.value_or(""), "' is none of None, 'relu', 'silu'");
  return !act ? KAD_ACT_NONE : *act == "relu" ? KAD_ACT_RELU : KAD_ACT_SILU;
}

// The entry points of kad_rows.cpp.
void bind_rows(py::module_& m);

}  // namespace kad_torch

using namespace kad_torch;

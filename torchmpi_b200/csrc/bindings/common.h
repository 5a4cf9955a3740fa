// What the autograd functions of autograd.cpp and experts.cpp share.
#pragma once
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <atomic>
#include <initializer_list>
#include <string>
#include <utility>
#include "tmpi_c_api.h"

namespace tmpi_bind {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

enum { LINEAR, LAYERNORM, ATTENTION, XENT, ATTENTION_BACKWARD, BATCHNORM, CONV, STEM, ACT8, EXPERTS, FP8, ADAMW, KINDS };
inline std::atomic<long long> g_launches[KINDS];      // attention: calls, and those of the backward alone

inline void* stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }
inline void launched(int what, int n) { g_launches[what].fetch_add(n, std::memory_order_relaxed); }

inline void check(int status) {
  if (!status) return;
  pybind11::gil_scoped_acquire gil;
  pybind11::module_::import("torchmpi_b200._lib").attr("check")(status);
}

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return TMPI_F16;
    case at::kBFloat16: return TMPI_BF16;
    case at::kFloat: return TMPI_F32;
    case at::kDouble: return TMPI_F64;                           // what a kernel does not take, its entry point refuses
    case at::kByte: return TMPI_U8;
    case at::kChar: return TMPI_I8;
    case at::kShort: return TMPI_I16;
    case at::kInt: return TMPI_I32;
    case at::kLong: return TMPI_I64;
    default: throw pybind11::type_error(std::string("torchmpi_b200: unsupported dtype ") + c10::toString(t));
  }
}

// Contiguous and on a 16-byte boundary, which the elementwise kernels' loads need: a view into a larger buffer may start
// anywhere.
inline Tensor packed(const Tensor& t, at::MemoryFormat format = at::MemoryFormat::Contiguous) {
  if (t.is_contiguous(format) && (uintptr_t)t.data_ptr() % 16 == 0) return t;
  Tensor c = t.contiguous(format);
  if ((uintptr_t)c.data_ptr() % 16) c = c.clone(format);
  return c;
}

// A saved tensor as it was saved: hooks (torch.autograd.graph.save_on_cpu, say) may hand it back in another layout.
inline Tensor as_saved(const Tensor& t, at::MemoryFormat format = at::MemoryFormat::Contiguous) { return t.defined() ? packed(t, format) : t; }

// An uninitialized tensor on the current device, past the dispatcher (half a microsecond for each of a small call's).
inline Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) { return Tensor(at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, c10::cuda::current_device()), c10::nullopt)); }

using OptTensor = c10::optional<Tensor>;
inline Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
inline const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline const int* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int>() : nullptr; }
// Whether a call goes by its autograd function: a gradient may be asked for, or an input has a forward-mode tangent (whatever the grad mode), which the
// function refuses; a result without one would stand for a derivative of zero.
inline bool wants_grad(std::initializer_list<Tensor> inputs) {
  const bool backward = at::GradMode::is_enabled();
  for (const Tensor& t : inputs)
    if (t.defined() && ((backward && t.requires_grad()) || t._fw_grad(/*level=*/0).defined())) return true;
  return false;
}
// all on the current device, which there is one of per process
inline bool here(std::initializer_list<const Tensor*> tensors) {
  const int64_t device = c10::cuda::current_device();
  for (const Tensor* t : tensors)
    if (t->defined() && !(t->is_cuda() && t->get_device() == device)) return false;
  return true;
}
inline bool all_of_type(std::initializer_list<const Tensor*> tensors, at::ScalarType type) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->scalar_type() != type) return false;
  return true;
}
inline bool floating(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat; }
inline bool shaped(const Tensor& t, std::initializer_list<int64_t> sizes) { return !t.defined() || t.sizes() == at::IntArrayRef(sizes); }
// [..., cols] as rows
inline Tensor rows_of(const Tensor& x) { return x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}); }
constexpr int64_t MOST = int64_t(1) << 30;                          // rows, columns and entries that the kernels count in 32 bits

// of autograd.cpp: a b^T (+ bias), and the gradients of a linear layer that are asked for
Tensor matmul_nt(const Tensor& a, const Tensor& b, const Tensor& bias);
void linear_gradients(const Tensor& dy, const Tensor& x, const Tensor& w, Tensor* dx, Tensor* dw, Tensor* db);
void register_experts(pybind11::module_& m);      // experts.cpp
void register_fp8(pybind11::module_& m);          // fp8.cpp
void register_adamw(pybind11::module_& m);        // adamw.cpp

}  // namespace tmpi_bind

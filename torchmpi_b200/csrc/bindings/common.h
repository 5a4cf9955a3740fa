// What the autograd functions of autograd.cpp and experts.cpp share.
#pragma once
#include <torch/extension.h>
#include <c10/cuda/CUDAStream.h>
#include <atomic>
#include <string>
#include <utility>
#include "tmpi_c_api.h"

namespace tmpi_bind {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

enum { LINEAR, LAYERNORM, ATTENTION, XENT, ATTENTION_BACKWARD, BATCHNORM, CONV, STEM, ACT8, EXPERTS, KINDS };
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

// of autograd.cpp: a b^T (+ bias), and the gradients of a linear layer that are asked for
Tensor matmul_nt(const Tensor& a, const Tensor& b, const Tensor& bias);
void linear_gradients(const Tensor& dy, const Tensor& x, const Tensor& w, Tensor* dx, Tensor* dw, Tensor* db);
void register_experts(pybind11::module_& m);      // experts.cpp

}  // namespace tmpi_bind

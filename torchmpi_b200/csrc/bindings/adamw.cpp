// The AdamW step over a model's tensors (ops/adamw.py).  What stays the same from step to step - the tensors, the place of their states - is held here, so that
// a step costs the host one call: weights and gradients are looked at and their addresses taken anew in every step.
#include "common.h"
#include <pybind11/stl.h>
#include <algorithm>
#include <array>
#include <cmath>

namespace tmpi_bind {
namespace {

// A tensor of p's shape in the order of its storage, of the given type.
Tensor in_order(const Tensor& g, const Tensor& p, at::ScalarType type) {
  if (g.scalar_type() == type && g.strides() == p.strides()) return g;
  Tensor c = at::empty_like(p, p.options().dtype(type));
  c.copy_(g);
  return c;
}
bool in_same_order(const Tensor& p, const std::vector<int64_t>& strides) {
  if (p.dim() != (int64_t)strides.size()) return false;
  for (int64_t d = 0; d < p.dim(); ++d)
    if (p.size(d) != 1 && p.stride(d) != strides[d]) return false;
  return true;
}
bool taken(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }
constexpr at::ScalarType TYPES[] = {at::kBFloat16, at::kHalf, at::kFloat};

struct AdamW {
  std::vector<Tensor> params;
  std::vector<int64_t> places, sizes;
  std::vector<std::vector<int64_t>> strides;                        // the order of the states
  std::vector<at::ScalarType> types;
  std::vector<int> group;
  Tensor m, v, m_top, v_top, master, steps, counter, norm;
  Tensor sums, coefficient;                                         // of a clipped step
  int bits;

  // groups: lr, beta1, beta2, eps, weight decay; rates: learning rates on the device, or None
  void step(const std::vector<std::array<double, 5>>& groups, const std::vector<OptTensor>& rates, c10::optional<double> max_norm, double scale) {
    at::NoGradGuard no_grad;
    const int64_t device = c10::cuda::current_device();
    std::vector<tmpi_adamw_group_t> g(groups.size());
    for (size_t i = 0; i < groups.size(); ++i) {
      const auto& x = groups[i];
      g[i] = {(float)x[0], (float)x[1], (float)x[2], (float)(1 - x[1]), (float)(1 - x[2]), (float)std::log(x[1]), (float)std::log(x[2]), (float)x[3], (float)x[4], nullptr};
      if (rates[i].has_value()) {
        const Tensor& r = *rates[i];
        TORCH_CHECK_VALUE(r.is_cuda() && r.get_device() == device && r.scalar_type() == at::kFloat && r.numel() == 1, "AdamW: a learning rate on the device is one fp32 number on the current one");
        g[i].device_lr = r.data_ptr<float>();
      }
    }
    std::vector<Tensor> kept;                                        // gradients that had to be copied
    std::vector<std::pair<Tensor, Tensor>> stepped;                  // parameters, and the fp32 tensors that are stepped in their place
    std::vector<tmpi_adamw_tensor_t> tables[3];
    for (size_t i = 0; i < params.size(); ++i) {
      const Tensor& p = params[i];
      const Tensor& grad = p.grad();
      if (!grad.defined() || !sizes[i]) continue;
      TORCH_CHECK_VALUE(p.is_cuda() && p.get_device() == device, "AdamW: a parameter on ", p.device(), ", but the current device is cuda:", device);
      TORCH_CHECK_VALUE(p.numel() == sizes[i] && p.scalar_type() == types[i] && in_same_order(p, strides[i]) && p.is_non_overlapping_and_dense(), "AdamW: a parameter has changed: ", p.scalar_type(), " ", p.sizes(),
                        " with strides ", p.strides());
      TORCH_CHECK_VALUE(!grad.is_sparse() && grad.layout() == at::kStrided && grad.device() == p.device() && grad.sizes() == p.sizes(), "AdamW: a gradient that is not its parameter's: ", grad.sizes());
      // A gradient of another type than its 16-bit parameter's counts as it is: the step is that of an fp32 parameter, the master or a copy, whose rounding the parameter becomes.
      const bool other = grad.scalar_type() != types[i] && types[i] != at::kFloat;
      const at::ScalarType type = other ? at::kFloat : types[i];
      const Tensor ordered = in_order(grad, p, type);
      if (!ordered.is_same(grad)) kept.push_back(ordered);
      const Tensor w = !other ? p : master.defined() ? master.slice(0, places[i], places[i] + sizes[i]).as_strided(p.sizes(), p.strides()) : in_order(p, p, type);
      if (other) stepped.emplace_back(p, w);
      const int code = type == at::kBFloat16 ? 0 : type == at::kHalf ? 1 : 2;
      tables[code].push_back({w.data_ptr(), ordered.data_ptr(), places[i], sizes[i], (int)w.element_size(), group[i], (int)i});
    }
    tmpi_adamw_states_t s{};
    s.m = m.data_ptr(); s.v = v.data_ptr();
    s.m_top = bits == 8 ? m_top.data_ptr<float>() : nullptr;
    s.v_top = bits == 8 ? v_top.data_ptr<float>() : nullptr;
    s.steps = steps.data_ptr<int>();
    s.counter = (unsigned*)counter.data_ptr<int>();
    s.scale = (float)scale;
    if (max_norm.has_value()) {
      const tmpi_norm_finish_t finish{norm.data_ptr<float>(), coefficient.data_ptr<float>(), s.counter, (float)scale, (float)*max_norm};
      int used = 0;
      for (int c = 0; c < 3; ++c) {
        if (tables[c].empty()) continue;
        const bool last = (c > 1 || tables[2].empty()) && (c > 0 || tables[1].empty());          // of the types
        check(tmpi_norm_squares(tables[c].data(), (int)tables[c].size(), dtype_code(TYPES[c]), sums.data_ptr<double>(), &used, last ? &finish : nullptr, stream()));
        launched(ADAMW, 1);
      }
      if (!used) {                                                   // no gradient at all
        check(tmpi_norm_finish(sums.data_ptr<double>(), 0, (float)scale, (float)*max_norm, norm.data_ptr<float>(), coefficient.data_ptr<float>(), stream()));
        launched(ADAMW, 1);
      }
      s.coefficient = coefficient.data_ptr<float>();
    }
    for (int c = 0; c < 3; ++c) {
      if (tables[c].empty()) continue;
      s.master = master.defined() && TYPES[c] != at::kFloat ? master.data_ptr<float>() : nullptr;
      check(tmpi_adamw_step(tables[c].data(), (int)tables[c].size(), g.data(), (int)g.size(), &s, bits, dtype_code(TYPES[c]), stream()));
      launched(ADAMW, 1);
    }
    for (auto& [p, w] : stepped) p.copy_(w);
    for (const auto& p : params)
      if (p.grad().defined()) p.unsafeGetTensorImpl()->bump_version();          // written to, as autograd has to know
  }
};

}  // namespace

void register_adamw(pybind11::module_& m) {
  pybind11::class_<AdamW>(m, "AdamW")
      .def(pybind11::init([](std::vector<Tensor> params, std::vector<int64_t> places, std::vector<int> group, Tensor m_, Tensor v, const OptTensor& m_top, const OptTensor& v_top, const OptTensor& master,
                             Tensor steps, Tensor counter, Tensor norm, int bits) {
        AdamW a;
        for (const Tensor& p : params) {
          a.sizes.push_back(p.numel());
          a.strides.push_back(p.strides().vec());
          a.types.push_back(p.scalar_type());
        }
        a.params = std::move(params); a.places = std::move(places); a.group = std::move(group);
        a.m = m_; a.v = v; a.m_top = or_none(m_top); a.v_top = or_none(v_top); a.master = or_none(master);
        a.steps = steps; a.counter = counter; a.norm = norm; a.bits = bits;
        a.sums = fresh({tmpi_norm_sums((int)a.params.size()) + 2 * tmpi_norm_sums(0)}, at::kDouble);          // of three types' launches
        a.coefficient = fresh({1}, at::kFloat);
        return a;
      }))
      .def("step", &AdamW::step);
  m.def("adamw_values", [](const Tensor& mq, const Tensor& m_top, const Tensor& vq, const Tensor& v_top, int code) {
    const auto type = code == TMPI_F32 ? at::kFloat : code == TMPI_F16 ? at::kHalf : at::kBFloat16;
    Tensor a = fresh({mq.numel()}, type), b = fresh({mq.numel()}, type);
    check(tmpi_adamw_values(mq.data_ptr(), m_top.data_ptr<float>(), vq.data_ptr(), v_top.data_ptr<float>(), a.data_ptr(), b.data_ptr(), mq.numel() / 128, code, stream()));
    launched(ADAMW, 1);
    return std::make_pair(a, b);
  });
  // the norm of all of them together, or nothing (None) for what the kernel does not take
  m.def("grad_norm", [](const std::vector<Tensor>& tensors) -> OptTensor {
    std::vector<Tensor> kept;
    std::vector<tmpi_adamw_tensor_t> tables[3];
    int total = 0, used = 0;
    const int64_t device = c10::cuda::current_device();
    for (const Tensor& t_ : tensors) {
      if (!(t_.is_cuda() && t_.get_device() == device && t_.layout() == at::kStrided && taken(t_.scalar_type()))) return c10::nullopt;
      if (!t_.numel()) continue;
      const Tensor t = t_.is_non_overlapping_and_dense() ? t_ : t_.detach().contiguous();
      kept.push_back(t);
      tables[t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : 2].push_back({nullptr, t.data_ptr(), 0, t.numel(), (int)t.element_size(), 0, 0});
    }
    if (kept.empty()) return c10::nullopt;
    for (const auto& t : tables) total += tmpi_norm_sums((int)t.size());
    const Tensor sums = fresh({total}, at::kDouble), norm = fresh({}, at::kFloat);
    for (int c = 0; c < 3; ++c)
      if (!tables[c].empty()) check(tmpi_norm_squares(tables[c].data(), (int)tables[c].size(), dtype_code(TYPES[c]), sums.data_ptr<double>(), &used, nullptr, stream()));
    check(tmpi_norm_finish(sums.data_ptr<double>(), used, 1.f, 1.f, norm.data_ptr<float>(), nullptr, stream()));
    launched(ADAMW, 2);
    return norm;
  });
}

}  // namespace tmpi_bind

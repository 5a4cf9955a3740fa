// Autograd functions of layers of experts and of 8-bit activation checkpoints (ops/experts.py, ops/act8.py).  An entry returns nothing (None) for what
// the kernels do not take, wrong arguments among it: the Python function then raises, or computes with PyTorch's operations.  So a call
// that the kernels take is looked at once, here (in Python the checks of a layer of experts took 17 us of a call of 39).  Scratch
// memory comes from PyTorch's allocator on the calling stream, per call.
#include "common.h"
#include <c10/cuda/CUDAFunctions.h>
#include <algorithm>
#include <initializer_list>

namespace tmpi_bind {
namespace {

enum { PLAIN = 0, GELU = 1, GELU_AND_Z = 2, GELU_AND_Z8 = 3, FP32 = 4 };      // tmpi_grouped_gemm's modes

using OptTensor = c10::optional<Tensor>;
Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const int* ints(const Tensor& t) { return t.defined() ? t.data_ptr<int>() : nullptr; }
// Whether a call goes by its autograd function: a gradient may be asked for, or an input has a forward-mode tangent (whatever the grad mode), which the
// function refuses; a result without one would stand for a derivative of zero.
bool wants_grad(std::initializer_list<Tensor> inputs) {
  const bool backward = at::GradMode::is_enabled();
  for (const Tensor& t : inputs)
    if (t.defined() && ((backward && t.requires_grad()) || t._fw_grad(/*level=*/0).defined())) return true;
  return false;
}

// The kernels' gradients are constants to autograd: one asked for with a graph (create_graph) would lose its part of what it enters in silence.
void refuse_graph() { TORCH_CHECK(!at::GradMode::is_enabled(), "layers of experts and 8-bit checkpoints can be differentiated once (no create_graph)"); }

// all on the current device, which there is one of per process
bool here(std::initializer_list<const Tensor*> tensors) {
  const int64_t device = c10::cuda::current_device();
  for (const Tensor* t : tensors)
    if (t->defined() && !(t->is_cuda() && t->get_device() == device)) return false;
  return true;
}
bool all_of_type(std::initializer_list<const Tensor*> tensors, at::ScalarType type) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->scalar_type() != type) return false;
  return true;
}
bool floating(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat; }
bool shaped(const Tensor& t, std::initializer_list<int64_t> sizes) { return !t.defined() || t.sizes() == at::IntArrayRef(sizes); }
// [..., cols] as rows
Tensor rows_of(const Tensor& x) { return x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}); }
constexpr int64_t MOST = int64_t(1) << 30;                          // rows, columns and entries that the kernels count in 32 bits

struct Kept { Tensor q, scale; };                                   // an 8-bit checkpoint, [..., cols] and [..., ceil(cols / 32)]

Kept empty_kept(const Tensor& like, at::IntArrayRef sizes) {
  std::vector<int64_t> blocks = sizes.vec();
  blocks.back() = (blocks.back() + 31) / 32;
  return {at::empty(sizes, like.options().dtype(at::kFloat8_e4m3fn)), at::empty(blocks, like.options().dtype(at::kByte))};
}
Kept quantize(const Tensor& x) {                                    // packed
  Kept k = empty_kept(x, x.sizes());
  const int64_t cols = x.size(-1);
  check(tmpi_act8_quantize(x.data_ptr(), k.q.data_ptr(), k.scale.data_ptr(), x.numel() / cols, (int)cols, dtype_code(x.scalar_type()), stream()));
  launched(ACT8, 1);
  return k;
}
Tensor restore(const Kept& k, at::ScalarType type) {
  Tensor x = at::empty(k.q.sizes(), k.q.options().dtype(type));
  const int64_t cols = x.size(-1);
  check(tmpi_act8_restore(k.q.data_ptr(), k.scale.data_ptr(), x.data_ptr(), x.numel() / cols, (int)cols, dtype_code(type), stream()));
  launched(ACT8, 1);
  return x;
}
// (dz, h) of tmpi_act8_gelu_gradient; h only where it is asked for
std::pair<Tensor, Tensor> gelu_gradient(const Tensor& dy, const Kept& k, bool with_h = true) {
  Tensor dz = at::empty_like(dy), h;
  if (with_h) h = at::empty_like(dy);
  const int64_t cols = dy.size(-1);
  check(tmpi_act8_gelu_gradient(dy.data_ptr(), k.q.data_ptr(), k.scale.data_ptr(), dz.data_ptr(), with_h ? h.data_ptr() : nullptr, dy.numel() / cols, (int)cols,
                                dtype_code(dy.scalar_type()), stream()));
  launched(ACT8, 1);
  return {dz, h};
}
// dz is linear in dy, with the slope at what the checkpoint stands for; h and the slope do not depend on it.
struct GeluGradientFn : public torch::autograd::Function<GeluGradientFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& dy, const Tensor& q, const Tensor& scale) {
    const Kept k{packed(q), packed(scale)};
    const auto both = gelu_gradient(packed(dy), k);
    ctx->save_for_backward({k.q, k.scale});
    ctx->mark_non_differentiable({both.second});
    ctx->set_materialize_grads(false);
    return {both.first, both.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    return {gelu_gradient(packed(grads[0]), {as_saved(saved[0]), as_saved(saved[1])}, false).first, Tensor(), Tensor()};
  }
};
bool is_kept(const Tensor& q, const Tensor& scale) {
  if (!(q.scalar_type() == at::kFloat8_e4m3fn && scale.scalar_type() == at::kByte && q.dim() >= 1 && scale.dim() == q.dim() && q.numel() > 0 && q.size(-1) <= MOST)) return false;
  for (int64_t i = 0; i + 1 < q.dim(); ++i)
    if (q.size(i) != scale.size(i)) return false;
  return scale.size(-1) == (q.size(-1) + 31) / 32 && here({&q, &scale});
}

// ---------------------------------------------------------------- products grouped by expert
// offsets undefined: one expert (w [N, K]) with all rows.  z, scale: see tmpi_grouped_gemm.
Tensor grouped(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& offsets, bool w_is_kn, int mode, const Tensor& z, const Tensor& scale) {
  const int experts = offsets.defined() ? (int)w.size(0) : 1, d = (int)w.dim();
  const int N = (int)w.size(w_is_kn ? d - 1 : d - 2), K = (int)x.size(1);
  Tensor y = mode == FP32 ? at::empty({tmpi_grouped_slices((int)x.size(0), experts, K, N) * x.size(0), N}, x.options().dtype(at::kFloat)) : at::empty({x.size(0), N}, x.options());
  check(tmpi_grouped_gemm(x.data_ptr(), w.data_ptr(), ptr(bias), ints(offsets), y.data_ptr(), z.defined() ? z.data_ptr() : nullptr,
                          scale.defined() ? scale.data_ptr() : nullptr, (int)x.size(0), experts, K, N, w_is_kn ? 1 : 0, mode, stream()));
  launched(EXPERTS, 1);
  return y;
}
// (dz, h) of tmpi_grouped_gelu_gradient; dots: an empty tensor of its sums, or undefined
std::pair<Tensor, Tensor> grouped_gelu_gradient(const Tensor& dy, const Tensor& w, const Tensor& offsets, const Kept& z, const Tensor& row_weights, const Tensor& dots) {
  const int experts = offsets.defined() ? (int)w.size(0) : 1, N = (int)w.size(-1);
  Tensor dz = at::empty({dy.size(0), N}, dy.options()), h = at::empty_like(dz);
  check(tmpi_grouped_gelu_gradient(dy.data_ptr(), w.data_ptr(), ints(offsets), z.q.data_ptr(), z.scale.defined() ? z.scale.data_ptr() : nullptr,
                                   row_weights.defined() ? row_weights.data_ptr<float>() : nullptr, dz.data_ptr(), h.data_ptr(),
                                   dots.defined() ? dots.data_ptr<float>() : nullptr, (int)dy.size(0), experts, (int)dy.size(1), N, stream()));
  launched(EXPERTS, 1);
  return {dz, h};
}
// dw and, where asked for, db
void grouped_weight_gradient(const Tensor& dy, const Tensor& x, const Tensor& offsets, const Tensor& row_weights, int64_t experts, Tensor* dw, Tensor* db) {
  *dw = at::empty({experts, dy.size(1), x.size(1)}, x.options());
  if (db) *db = at::empty({experts, dy.size(1)}, x.options());
  check(tmpi_grouped_weight_gradient(dy.data_ptr(), x.data_ptr(), ints(offsets), row_weights.defined() ? row_weights.data_ptr<float>() : nullptr,
                                     dw->data_ptr(), db ? db->data_ptr() : nullptr, (int)x.size(0), (int)experts, (int)x.size(1), (int)dy.size(1), stream()));
  launched(EXPERTS, 1);
}

struct GroupedLinearFn : public torch::autograd::Function<GroupedLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const OptTensor& bias_, const Tensor& offsets_, bool with_gelu) {
    const Tensor x = packed(x_), w = packed(w_), bias = bias_.has_value() ? packed(*bias_) : Tensor(), offsets = offsets_.contiguous();
    Tensor z;
    if (with_gelu) z = at::empty({x.size(0), w.size(1)}, x.options());
    const Tensor y = grouped(x, w, bias, offsets, false, with_gelu ? GELU_AND_Z : PLAIN, z, Tensor());
    ctx->save_for_backward({x, w, offsets, z});
    ctx->saved_data["bias"] = bias.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    const auto saved = ctx->get_saved_variables();
    const Tensor x = as_saved(saved[0]), w = as_saved(saved[1]), offsets = as_saved(saved[2]), z = as_saved(saved[3]);
    Tensor dy = packed(grads[0]), dx, dw, db;
    if (z.defined() && dy.numel()) {
      Tensor dz = at::empty_like(dy);
      check(tmpi_gelu_bwd(dy.data_ptr(), z.data_ptr(), dz.data_ptr(), (size_t)dy.numel(), dtype_code(dy.scalar_type()), stream()));
      launched(EXPERTS, 1);
      dy = dz;
    }
    const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    if (ctx->needs_input_grad(0)) dx = grouped(dy, w, Tensor(), offsets, true, PLAIN, Tensor(), Tensor());
    if (ctx->needs_input_grad(1) || need_b) grouped_weight_gradient(dy, x, offsets, Tensor(), w.size(0), &dw, need_b ? &db : nullptr);
    if (!ctx->needs_input_grad(1)) dw = Tensor();
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------- an MLP with 8-bit checkpoints
struct Mlp8Fn : public torch::autograd::Function<Mlp8Fn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w1_, const OptTensor& b1_, const Tensor& w2_, const OptTensor& b2_) {
    const Tensor x = packed(x_), w1 = packed(w1_), w2 = packed(w2_), b1 = b1_.has_value() ? packed(*b1_) : Tensor(), b2 = b2_.has_value() ? packed(*b2_) : Tensor();
    const Kept kx = quantize(x), kz = empty_kept(x, {x.size(0), w1.size(0)});
    const Tensor h = grouped(x, w1, b1, Tensor(), false, GELU_AND_Z8, kz.q, kz.scale);
    const Tensor y = matmul_nt(h, w2, b2);
    ctx->save_for_backward({kx.q, kx.scale, kz.q, kz.scale, w1, w2});
    ctx->saved_data["b1"] = b1.defined();
    ctx->saved_data["b2"] = b2.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    const auto saved = ctx->get_saved_variables();
    const Kept kx{as_saved(saved[0]), as_saved(saved[1])}, kz{as_saved(saved[2]), as_saved(saved[3])};
    const Tensor w1 = as_saved(saved[4]), w2 = as_saved(saved[5]), dy = packed(grads[0]);
    const bool has_b1 = ctx->saved_data["b1"].toBool(), has_b2 = ctx->saved_data["b2"].toBool();         // an absent bias has no number among the inputs
    const bool need_x = ctx->needs_input_grad(0), need_w1 = ctx->needs_input_grad(1), need_w2 = ctx->needs_input_grad(2 + has_b1);
    const bool need_b1 = has_b1 && ctx->needs_input_grad(2), need_b2 = has_b2 && ctx->needs_input_grad(3 + has_b1);
    Tensor dx, dw1, db1, dw2, db2;
    if (need_x || need_w1 || need_b1 || need_w2) {
      const auto both = grouped_gelu_gradient(dy, w2, Tensor(), kz, Tensor(), Tensor());
      const Tensor dz = both.first;
      if (need_w2) linear_gradients(dy, both.second, w2, nullptr, &dw2, need_b2 ? &db2 : nullptr);
      if (need_w1) linear_gradients(dz, restore(kx, dz.scalar_type()), w1, need_x ? &dx : nullptr, &dw1, need_b1 ? &db1 : nullptr);
      else if (need_x) linear_gradients(dz, kx.q, w1, &dx, nullptr, need_b1 ? &db1 : nullptr);      // kx.q: for its extents alone
      else if (need_b1) db1 = dz.sum(0);
    }
    if (need_b2 && !db2.defined()) db2 = dy.sum(0);
    return {dx, dw1, db1, dw2, db2};
  }
};

// ---------------------------------------------------------------- routing
Tensor dense_columns(const Tensor& l) { return l.stride(1) == 1 && (l.size(0) < 2 || l.stride(0) >= l.size(1)) ? l : l.contiguous(); }

// weights, chosen, order, place, offsets
variable_list route(const Tensor& logits, int64_t k, bool renormalize) {
  const int T = (int)logits.size(0), E = (int)logits.size(1);
  const auto i32 = logits.options().dtype(at::kInt);
  Tensor weights = at::empty({T, k}, logits.options().dtype(at::kFloat)), chosen = at::empty({T, k}, i32), order = at::empty({T * k}, i32),
         place = at::empty({T, k}, i32), offsets = at::empty({E + 1}, i32), ws;
  const size_t need = tmpi_route_workspace_bytes(T, E, (int)k);
  if (need) ws = at::empty({(int64_t)need}, logits.options().dtype(at::kByte));
  check(tmpi_route(logits.data_ptr(), T > 1 ? logits.stride(0) : E, T, E, (int)k, renormalize, dtype_code(logits.scalar_type()), weights.data_ptr<float>(),
                   chosen.data_ptr<int>(), order.data_ptr<int>(), place.data_ptr<int>(), offsets.data_ptr<int>(), need ? ws.data_ptr() : nullptr, need, stream()));
  launched(EXPERTS, need ? 2 : 1);
  return {weights, chosen, order, place, offsets};
}

struct RouteFn : public torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits_, int64_t k, bool renormalize) {
    const Tensor logits = dense_columns(logits_);
    variable_list r = route(logits, k, renormalize);
    ctx->save_for_backward({logits, r[0], r[1]});
    ctx->saved_data["k"] = k;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->mark_non_differentiable({r[1], r[2], r[3], r[4]});
    ctx->set_materialize_grads(false);                              // or autograd fills a tensor with zeros for each of them
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor logits = dense_columns(saved[0]);
    const Tensor weights = as_saved(saved[1]), chosen = as_saved(saved[2]), dw = packed(grads[0].to(at::kFloat));
    const int T = (int)logits.size(0), E = (int)logits.size(1);
    Tensor dl = at::empty({T, E}, logits.options());
    check(tmpi_route_gradient(logits.data_ptr(), T > 1 ? logits.stride(0) : E, T, E, (int)ctx->saved_data["k"].toInt(), ctx->saved_data["renormalize"].toBool(),
                              dtype_code(logits.scalar_type()), weights.data_ptr<float>(), chosen.data_ptr<int>(), dw.data_ptr<float>(), dl.data_ptr(), stream()));
    launched(EXPERTS, 1);
    return {dl, Tensor(), Tensor()};
  }
};

const int* last(const Tensor& offsets) { return offsets.data_ptr<int>() + offsets.numel() - 1; }      // how many places are used

// offsets undefined: rows behind the last entry are left as they are; by_place: receives the weights in the order of the places
Tensor dispatch(const Tensor& x, const Tensor& place, const Tensor& offsets, const Tensor& weights = Tensor(), const Tensor& by_place = Tensor()) {
  const int64_t T = place.size(0), k = place.size(1);
  Tensor out = at::empty({T * k, x.size(1)}, x.options());
  check(tmpi_expert_dispatch(x.data_ptr(), place.data_ptr<int>(), offsets.defined() ? last(offsets) : nullptr, weights.defined() ? weights.data_ptr<float>() : nullptr, out.data_ptr(),
                             by_place.defined() ? by_place.data_ptr<float>() : nullptr, (int)T, (int)k, (int)x.size(1),
                             dtype_code(x.scalar_type()), stream()));
  launched(EXPERTS, 1);
  return out;
}
// rows of `type`, or for bf16 in fp32, as many results as grouped() has left there
Tensor combine(const Tensor& rows, const Tensor& weights, const Tensor& place, at::ScalarType type) {
  const int slices = type == at::kBFloat16 && rows.scalar_type() == at::kFloat ? (int)(rows.size(0) / place.numel()) : 0;
  Tensor y = at::empty({place.size(0), rows.size(1)}, rows.options().dtype(type));
  check(tmpi_expert_combine(rows.data_ptr(), slices, weights.defined() ? weights.data_ptr<float>() : nullptr, place.data_ptr<int>(), y.data_ptr(), (int)place.size(0),
                            (int)place.size(1), (int)rows.size(1), dtype_code(type), stream()));
  launched(EXPERTS, 1);
  return y;
}

struct DispatchFn : public torch::autograd::Function<DispatchFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& place_, const Tensor& offsets) {
    const Tensor place = place_.contiguous();
    ctx->save_for_backward({place});
    return dispatch(packed(x), place, offsets.contiguous());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    const auto saved = ctx->get_saved_variables();
    return {combine(packed(grads[0]), Tensor(), as_saved(saved[0]), grads[0].scalar_type()), Tensor(), Tensor()};
  }
};

struct CombineFn : public torch::autograd::Function<CombineFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows_, const Tensor& weights_, const Tensor& place_, const Tensor& offsets_) {
    const Tensor rows = packed(rows_), weights = weights_.contiguous(), place = place_.contiguous();
    ctx->save_for_backward({rows, weights, place, offsets_.contiguous()});
    return combine(rows, weights, place, rows.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    const auto saved = ctx->get_saved_variables();
    const Tensor rows = as_saved(saved[0]), weights = as_saved(saved[1]), place = as_saved(saved[2]), offsets = as_saved(saved[3]), dy = packed(grads[0]);
    const bool need_w = ctx->needs_input_grad(1);
    Tensor drows = at::empty_like(rows), dw;
    if (need_w) dw = at::empty_like(weights);
    check(tmpi_expert_combine_gradient(dy.data_ptr(), need_w ? rows.data_ptr() : nullptr, weights.data_ptr<float>(), place.data_ptr<int>(), last(offsets),
                                       drows.data_ptr(), need_w ? dw.data_ptr<float>() : nullptr, (int)weights.size(0), (int)weights.size(1), (int)rows.size(1),
                                       dtype_code(rows.scalar_type()), stream()));
    launched(EXPERTS, 1);
    return {drows, dw, Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------- a layer of experts
// y_t = sum over j of weights_tj (gelu(x_t w1_e^T + b1_e) w2_e^T + b2_e), e = chosen_tj.  Kept for backward: x and the pre-activation,
// in bf16 or (act8) in 8 bits, and neither the dispatched rows nor what the experts returned: the rows are gathered again, and the weight's gradient
// dy . (w2 h + b2) is (w2^T dy) . h + dy . b2, of which the first product is there anyway.  What a token's experts return, and the gradients
// that they return to it, are handed over in fp32 and rounded once, as their sum.
// Roundings that are choices: weight gelu(z) and dz to bf16, as operands of the MMAs, and without act8 the pre-activation to bf16, as a layer of bf16
// tensors has it (fp32 would double what is kept).  15 tokens, 4 of 10 experts, 520 -> 512, errors relative to the norms: dw2 0.0017 from the rounding of the
// result alone, 0.0024 with that of weight gelu(z), 0.0030 with that of z; the weights' gradient has the last alone, 0.0020 where the result's is 0.0016.
struct Layer { Tensor x, weights, chosen, place, offsets, w1, b1, w2, b2; };

// keep: the checkpoints go to kx and kz
Tensor expert_forward(const Layer& l, bool act8, bool keep, Kept* kx, Kept* kz) {
  const int64_t T = l.place.size(0), k = l.place.size(1), H = l.w1.size(1);
  Tensor xs;
  if (keep && act8) {
    *kx = empty_kept(l.x, l.x.sizes());
    *kz = empty_kept(l.x, {T * k, H});
    xs = at::empty({T * k, l.x.size(1)}, l.x.options());
    check(tmpi_expert_dispatch_keep(l.x.data_ptr(), l.place.data_ptr<int>(), xs.data_ptr(), kx->q.data_ptr(), kx->scale.data_ptr(), (int)T, (int)k, (int)l.x.size(1), stream()));
    launched(EXPERTS, 1);
  } else {
    xs = dispatch(l.x, l.place, Tensor());
    if (keep) {
      kx->q = l.x;
      kz->q = at::empty({T * k, H}, l.x.options());
    }
  }
  const Tensor h = grouped(xs, l.w1, l.b1, l.offsets, false, !keep ? GELU : act8 ? GELU_AND_Z8 : GELU_AND_Z, kz->q, kz->scale);
  return combine(grouped(h, l.w2, l.b2, l.offsets, false, FP32, Tensor(), Tensor()), l.weights, l.place, l.x.scalar_type());
}

struct ExpertsFn : public torch::autograd::Function<ExpertsFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weights, const Tensor& chosen, const Tensor& place, const Tensor& offsets, const Tensor& w1,
                        const OptTensor& b1, const Tensor& w2, const OptTensor& b2, bool act8) {
    const Layer l{x, weights, chosen, place, offsets, w1, or_none(b1), w2, or_none(b2)};
    Kept kx, kz;
    const Tensor y = expert_forward(l, act8, true, &kx, &kz);
    ctx->save_for_backward({kx.q, kx.scale, kz.q, kz.scale, weights, chosen, place, offsets, w1, w2, l.b2});
    ctx->saved_data["b1"] = l.b1.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    const auto saved = ctx->get_saved_variables();
    const Kept kx{as_saved(saved[0]), as_saved(saved[1])}, kz{as_saved(saved[2]), as_saved(saved[3])};
    const Tensor weights = as_saved(saved[4]), chosen = as_saved(saved[5]), place = as_saved(saved[6]), offsets = as_saved(saved[7]), w1 = as_saved(saved[8]),
                 w2 = as_saved(saved[9]), b2 = as_saved(saved[10]), dy = packed(grads[0]);
    const int64_t T = place.size(0), k = place.size(1), C = dy.size(1), H = w1.size(1), E = w1.size(0);
    const bool has_b1 = ctx->saved_data["b1"].toBool();                 // an absent bias has no number among the inputs
    const bool need_x = ctx->needs_input_grad(0), need_w1 = ctx->needs_input_grad(5), need_b1 = has_b1 && ctx->needs_input_grad(6),
               need_w2 = ctx->needs_input_grad(6 + has_b1), need_b2 = b2.defined() && ctx->needs_input_grad(7 + has_b1);
    const auto f32 = dy.options().dtype(at::kFloat);
    const bool need_wt = ctx->needs_input_grad(1);
    const Tensor by_place = at::empty({T * k}, f32), g = dispatch(dy, place, Tensor(), weights, by_place);
    const int64_t slices = tmpi_grouped_dots((int)(T * k), (int)E, (int)H, kz.scale.defined());
    Tensor dots, dwt;
    if (need_wt) dots = at::empty({(slices + 3) / 4, T * k, 4}, f32);
    const auto both = grouped_gelu_gradient(g, w2, offsets, kz, by_place, dots);
    const Tensor dz = both.first, hw = both.second;
    if (need_wt) {
      dwt = at::empty({T, k}, f32);
      check(tmpi_expert_weight_gradient(dots.data_ptr<float>(), dy.data_ptr(), ptr(b2), place.data_ptr<int>(), chosen.data_ptr<int>(), dwt.data_ptr<float>(), (int)T, (int)k,
                                        (int)slices, (int)C, (int)E, stream()));
      launched(EXPERTS, 1);
    }
    Tensor dx, dw1, db1, dw2, db2;
    if (need_w2 || need_b2) grouped_weight_gradient(g, hw, offsets, by_place, E, &dw2, need_b2 ? &db2 : nullptr);
    if (need_w1 || need_b1) {
      Tensor xs;
      if (kx.scale.defined()) {
        xs = at::empty({T * k, C}, dy.options());
        check(tmpi_expert_dispatch8(kx.q.data_ptr(), kx.scale.data_ptr(), place.data_ptr<int>(), xs.data_ptr(), (int)T, (int)k, (int)C, stream()));
        launched(EXPERTS, 1);
      } else {
        xs = dispatch(kx.q, place, Tensor());
      }
      grouped_weight_gradient(dz, xs, offsets, Tensor(), E, &dw1, need_b1 ? &db1 : nullptr);
    }
    if (need_x) dx = combine(grouped(dz, w1, Tensor(), offsets, true, FP32, Tensor(), Tensor()), Tensor(), place, dy.scalar_type());
    const Tensor none;
    return {dx, dwt, none, none, none, need_w1 ? dw1 : none, db1, need_w2 ? dw2 : none, db2, none};
  }
};

}  // namespace

void register_experts(pybind11::module_& m) {
  using OptPair = c10::optional<std::pair<Tensor, Tensor>>;
  m.def("act8_quantize", [](const Tensor& x) -> OptPair {
    if (!(x.is_cuda() && floating(x) && x.dim() >= 1 && x.numel() > 0 && x.size(-1) <= MOST && here({&x}))) return c10::nullopt;
    const Kept k = quantize(packed(x.detach()));
    return std::make_pair(k.q, k.scale);
  });
  m.def("act8_restore", [](const Tensor& q, const Tensor& scale, int code) -> OptTensor {
    if (!(code == TMPI_F32 || code == TMPI_F16 || code == TMPI_BF16) || !q.is_cuda() || !is_kept(q, scale)) return c10::nullopt;
    return restore({packed(q), packed(scale)}, code == TMPI_F32 ? at::kFloat : code == TMPI_F16 ? at::kHalf : at::kBFloat16);
  });
  m.def("act8_gelu_gradient", [](const Tensor& dy, const Tensor& q, const Tensor& scale) -> OptPair {
    if (!(dy.is_cuda() && floating(dy) && dy.sizes() == q.sizes() && is_kept(q, scale) && here({&dy}))) return c10::nullopt;
    if (!wants_grad({dy})) return gelu_gradient(packed(dy), {packed(q), packed(scale)});
    const variable_list both = GeluGradientFn::apply(dy, q, scale);
    return std::make_pair(both[0], both[1]);
  });
  m.def("act8_mlp", [](const Tensor& x, const Tensor& w1, const OptTensor& b1_, const Tensor& w2, const OptTensor& b2_) -> OptTensor {
    const Tensor b1 = or_none(b1_), b2 = or_none(b2_);
    if (!(x.is_cuda() && x.dim() >= 1 && w1.dim() == 2 && w2.dim() == 2 && all_of_type({&x, &w1, &b1, &w2, &b2}, at::kBFloat16) && here({&x, &w1, &b1, &w2, &b2}))) return c10::nullopt;
    const int64_t C = w1.size(1), H = w1.size(0), D = w2.size(0), rows = x.size(-1) ? x.numel() / x.size(-1) : 0;
    if (!(x.size(-1) == C && w2.size(1) == H && shaped(b1, {H}) && shaped(b2, {D}) && C % 8 == 0 && H % 8 == 0 && D % 8 == 0 && C && H && D && rows && std::max({rows, C, H, D}) <= MOST)) return c10::nullopt;
    const Tensor x2 = rows_of(x);
    Tensor y;
    if (wants_grad({x, w1, w2, b1, b2})) {
      y = Mlp8Fn::apply(x2, w1, b1_, w2, b2_);
    } else {
      const Tensor h = grouped(packed(x2), packed(w1), b1.defined() ? packed(b1) : b1, Tensor(), false, GELU, Tensor(), Tensor());
      y = matmul_nt(h, packed(w2), b2.defined() ? packed(b2) : b2);
    }
    if (x.dim() == 2) return y;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = D;
    return y.view(shape);
  });
  m.def("grouped_linear", [](const Tensor& x, const Tensor& w, const OptTensor& bias_, const Tensor& offsets, bool gelu) -> OptTensor {
    const Tensor bias = or_none(bias_);
    if (!(x.is_cuda() && x.dim() == 2 && w.dim() == 3 && all_of_type({&x, &w, &bias}, at::kBFloat16) && offsets.scalar_type() == at::kInt && here({&x, &w, &bias, &offsets}))) return c10::nullopt;
    const int64_t E = w.size(0), N = w.size(1), K = w.size(2);
    if (!(x.size(1) == K && shaped(bias, {E, N}) && shaped(offsets, {E + 1}) && K % 8 == 0 && N % 8 == 0 && w.numel() && E <= tmpi_grouped_max_experts() && x.size(0) && std::max({x.size(0), N, K}) <= MOST)) return c10::nullopt;
    if (wants_grad({x, w, bias})) return GroupedLinearFn::apply(x, w, bias_, offsets, gelu);
    return grouped(packed(x), packed(w), bias.defined() ? packed(bias) : bias, offsets.contiguous(), false, gelu ? GELU : PLAIN, Tensor(), Tensor());
  });
  m.def("expert_route", [](const Tensor& logits, int64_t k, bool renormalize) -> c10::optional<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>> {
    if (!(logits.is_cuda() && logits.dim() == 2 && floating(logits) && here({&logits}))) return c10::nullopt;
    int experts = 0, most = 0;
    check(tmpi_route_limits(&experts, &most));
    const int64_t T = logits.size(0), E = logits.size(1);
    if (!(k >= 1 && k <= E && E <= experts && k <= most && T * k <= MOST)) return c10::nullopt;
    const variable_list r = wants_grad({logits}) ? RouteFn::apply(logits, k, renormalize) : route(dense_columns(logits), k, renormalize);
    return std::make_tuple(r[0], r[1], r[2], r[3], r[4]);
  });
  m.def("expert_dispatch", [](const Tensor& x, const Tensor& place, const Tensor& offsets) -> OptTensor {
    if (!(x.is_cuda() && x.dim() == 2 && floating(x) && x.numel() && place.dim() == 2 && offsets.dim() == 1 && offsets.size(0) >= 1 && all_of_type({&place, &offsets}, at::kInt) &&
          here({&x, &place, &offsets}) && place.size(0) == x.size(0) && place.numel() && place.numel() <= MOST && x.size(1) <= MOST)) return c10::nullopt;
    if (!wants_grad({x})) return dispatch(packed(x), place.contiguous(), offsets.contiguous());
    return DispatchFn::apply(x, place, offsets);
  });
  m.def("expert_combine", [](const Tensor& rows, const Tensor& weights, const Tensor& place, const Tensor& offsets) -> OptTensor {
    if (!(rows.is_cuda() && rows.dim() == 2 && floating(rows) && rows.numel() && place.dim() == 2 && offsets.dim() == 1 && offsets.size(0) >= 1 && all_of_type({&place, &offsets}, at::kInt) &&
          weights.scalar_type() == at::kFloat && weights.sizes() == place.sizes() && here({&rows, &weights, &place, &offsets}) && place.numel() == rows.size(0) && place.numel() <= MOST &&
          rows.size(1) <= MOST)) return c10::nullopt;
    if (!wants_grad({rows, weights})) return combine(packed(rows), weights.contiguous(), place.contiguous(), rows.scalar_type());
    return CombineFn::apply(rows, weights, place, offsets);
  });
  m.def("expert_mlp", [](const Tensor& x, const Tensor& weights, const Tensor& chosen, const Tensor& order, const Tensor& place, const Tensor& offsets,
                         const Tensor& w1, const OptTensor& b1_, const Tensor& w2, const OptTensor& b2_, bool act8) -> OptTensor {
    const Tensor b1 = or_none(b1_), b2 = or_none(b2_);
    if (!(x.is_cuda() && x.dim() >= 1 && w1.dim() == 3 && w2.dim() == 3 && place.dim() == 2 && all_of_type({&x, &w1, &b1, &w2, &b2}, at::kBFloat16) &&
          all_of_type({&chosen, &order, &place, &offsets}, at::kInt) && weights.scalar_type() == at::kFloat &&
          here({&x, &weights, &chosen, &order, &place, &offsets, &w1, &b1, &w2, &b2}))) return c10::nullopt;
    const int64_t E = w1.size(0), H = w1.size(1), C = w1.size(2), T = place.size(0), k = place.size(1);
    if (!(x.size(-1) == C && x.numel() == T * C && shaped(weights, {T, k}) && shaped(chosen, {T, k}) && shaped(order, {T * k}) && shaped(offsets, {E + 1}) && shaped(w2, {E, C, H}) &&
          shaped(b1, {E, H}) && shaped(b2, {E, C}) && C % 8 == 0 && H % 8 == 0 && w1.numel() && E <= tmpi_grouped_max_experts() && T && T * k && std::max({T * k, C, H}) <= MOST)) return c10::nullopt;
    const Layer l{packed(rows_of(x)), weights.contiguous(), chosen.contiguous(), place.contiguous(), offsets.contiguous(), packed(w1), b1.defined() ? packed(b1) : b1,
                  packed(w2), b2.defined() ? packed(b2) : b2};
    Tensor y;
    if (wants_grad({x, weights, w1, w2, b1, b2})) {
      y = ExpertsFn::apply(l.x, l.weights, l.chosen, l.place, l.offsets, l.w1, b1.defined() ? OptTensor(l.b1) : OptTensor(), l.w2, b2.defined() ? OptTensor(l.b2) : OptTensor(), act8);
    } else {
      Kept none;
      y = expert_forward(l, act8, false, &none, &none);
    }
    return x.dim() == 2 ? y : y.view(x.sizes());
  });
}

}  // namespace tmpi_bind

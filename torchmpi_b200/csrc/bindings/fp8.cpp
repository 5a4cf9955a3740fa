// Matrices in 8 bits with a scale for each block of 128, their products, and the linear layer that is made of them (ops/fp8.py).  As in experts.cpp an
// entry returns nothing (None) for what the kernels do not take, wrong arguments among it: the Python function then raises, or computes
// with PyTorch's operations.
#include "common.h"
#include <algorithm>

namespace tmpi_bind {
namespace {

struct Mat8 { Tensor q, scale; };                                   // of `rows` rows; what lies behind the columns is zero

void refuse_graph() { TORCH_CHECK(!at::GradMode::is_enabled(), "products in 8 bits can be differentiated once (no create_graph)"); }

Mat8 empty_mat(const Tensor& like, int64_t rows, int64_t cols) {
  return {at::empty({rows, tmpi_fp8_pitch(cols)}, like.options().dtype(at::kFloat8_e4m3fn)), at::empty({(int64_t)tmpi_fp8_scale_bytes(rows, cols)}, like.options().dtype(at::kByte))};
}
// rows whose elements follow each other; the rows themselves may lie apart
Tensor dense_rows(const Tensor& x) { return x.stride(1) == 1 && (x.size(0) < 2 || x.stride(0) >= x.size(1)) ? x : x.contiguous(); }
int64_t pitch(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// a, t: along the rows and the columns, each where it is given; z, sums: see tmpi_fp8_quantize
void quantize(const Tensor& x, const Tensor& z, Mat8* a, Mat8* t, const Tensor& sums) {
  const int64_t rows = x.size(0), cols = x.size(1);
  if (a) *a = empty_mat(x, rows, cols);
  if (t) *t = empty_mat(x, cols, rows);
  check(tmpi_fp8_quantize(x.data_ptr(), pitch(x), ptr(z), a ? a->q.data_ptr() : nullptr, a ? a->scale.data_ptr() : nullptr, t ? t->q.data_ptr() : nullptr,
                          t ? t->scale.data_ptr() : nullptr, sums.defined() ? sums.data_ptr<float>() : nullptr, rows, cols, dtype_code(x.scalar_type()), stream()));
  launched(FP8, 1);
}

// a b^T (+ bias) with `cols` columns of K; with gelu the GELU of it, and the rounded sums in z where it is given
Tensor product(const Mat8& a, const Mat8& b, int64_t cols, const Tensor& bias, bool gelu, Tensor* z, at::ScalarType type) {
  const int M = (int)a.q.size(0), N = (int)b.q.size(0), K = (int)cols;
  Tensor c = at::empty({M, N}, a.q.options().dtype(type)), ws;
  if (z) *z = at::empty_like(c);
  const size_t need = tmpi_fp8_product_workspace_bytes(M, N, K);
  if (need) ws = at::empty({(int64_t)need}, a.q.options().dtype(at::kByte));
  check(tmpi_fp8_product(a.q.data_ptr(), a.scale.data_ptr(), b.q.data_ptr(), b.scale.data_ptr(), ptr(bias), c.data_ptr(), z ? z->data_ptr() : nullptr, M, N, K, gelu, dtype_code(type),
                         need ? ws.data_ptr() : nullptr, need, stream()));
  launched(FP8, need ? 2 : 1);
  return c;
}

// x w^T (+ bias, GELU) without gradients
Tensor linear_kept(const Tensor& x, const Mat8& w, const Tensor& bias, bool gelu) {
  if (x.size(0) <= tmpi_fp8_few_tokens()) {
    Tensor y = at::empty({x.size(0), w.q.size(0)}, x.options());
    check(tmpi_fp8_few(x.data_ptr(), pitch(x), w.q.data_ptr(), w.scale.data_ptr(), ptr(bias), y.data_ptr(), (int)x.size(0), (int)w.q.size(0), (int)x.size(1), gelu,
                       dtype_code(x.scalar_type()), stream()));
    launched(FP8, 1);
    return y;
  }
  Mat8 a;
  quantize(x, Tensor(), &a, nullptr, Tensor());
  return product(a, w, x.size(1), bias, gelu, nullptr, x.scalar_type());
}

// Kept for backward: x and w along their columns, in 8 bits, and with a GELU the rounded pre-activation; each where a gradient needs it.
struct Linear8Fn : public torch::autograd::Function<Linear8Fn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const OptTensor& bias_, bool gelu, bool need_x, bool need_w) {
    const Tensor x = dense_rows(x_), w = dense_rows(w_), bias = bias_.has_value() ? packed(*bias_) : Tensor();
    Mat8 xr, xc, wr, wc;
    Tensor z;
    quantize(x, Tensor(), &xr, need_w ? &xc : nullptr, Tensor());
    quantize(w, Tensor(), &wr, need_x ? &wc : nullptr, Tensor());
    Tensor y = product(xr, wr, x.size(1), bias, gelu, gelu ? &z : nullptr, x.scalar_type());
    ctx->save_for_backward({xc.q, xc.scale, wc.q, wc.scale, z});
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["inputs"] = x.size(1);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    const auto saved = ctx->get_saved_variables();
    const Mat8 xc{as_saved(saved[0]), as_saved(saved[1])}, wc{as_saved(saved[2]), as_saved(saved[3])};
    const Tensor z = as_saved(saved[4]), dy = z.defined() ? packed(grads[0]) : dense_rows(grads[0]);
    const bool need_x = wc.q.defined() && ctx->needs_input_grad(0), need_w = xc.q.defined() && ctx->needs_input_grad(1),
               need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);      // an absent bias has no number among the inputs
    const int64_t T = dy.size(0), N = dy.size(1), K = ctx->saved_data["inputs"].toInt();
    const auto type = dy.scalar_type();
    Tensor dx, dw, db, sums;
    if (need_x || need_w || need_b) {
      Mat8 rows, columns;
      if (need_b) sums = at::empty({(T + 127) / 128, N}, dy.options().dtype(at::kFloat));
      quantize(dy, z, need_x ? &rows : nullptr, need_w || need_b || z.defined() ? &columns : nullptr, sums);
      if (need_x) dx = product(rows, wc, N, Tensor(), false, nullptr, type);
      if (need_w) dw = product(columns, xc, T, Tensor(), false, nullptr, type);
      if (need_b) {
        db = at::empty({N}, dy.options());
        check(tmpi_fp8_column_sums(sums.data_ptr<float>(), (int)sums.size(0), (int)N, db.data_ptr(), dtype_code(type), stream()));
        launched(FP8, 1);
      }
    }
    return {dx, dw, db, Tensor(), Tensor(), Tensor()};
  }
};

// q [rows, pitch of cols] with its scales, dense and aligned
bool is_mat(const Tensor& q, const Tensor& scale, int64_t cols) {
  return q.scalar_type() == at::kFloat8_e4m3fn && scale.scalar_type() == at::kByte && q.dim() == 2 && scale.dim() == 1 && cols >= 1 && cols <= MOST && q.size(0) >= 1 && q.size(0) <= MOST &&
         q.size(1) == tmpi_fp8_pitch(cols) && scale.size(0) == (int64_t)tmpi_fp8_scale_bytes(q.size(0), cols) && here({&q, &scale});
}
Mat8 packed_mat(const Tensor& q, const Tensor& scale) { return {packed(q), packed(scale)}; }
bool extents(int64_t M, int64_t N, int64_t K) { return M >= 1 && N >= 1 && K >= 1 && std::max({M, N, K}) <= MOST; }
Tensor shaped_as(const Tensor& y, const Tensor& x) {
  if (x.dim() == 2) return y;
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = y.size(1);
  return y.view(shape);
}

}  // namespace

void register_fp8(pybind11::module_& m) {
  // (q, scale) along the rows, and of the transpose, each where it is asked for
  m.def("fp8_quantize", [](const Tensor& x_, bool rows, bool columns) -> c10::optional<std::vector<Tensor>> {
    if (!(x_.is_cuda() && floating(x_) && x_.dim() == 2 && extents(x_.size(0), x_.size(1), 1) && here({&x_}))) return c10::nullopt;
    const Tensor x = dense_rows(x_.detach());
    Mat8 a, t;
    quantize(x, Tensor(), rows ? &a : nullptr, columns ? &t : nullptr, Tensor());
    std::vector<Tensor> out;
    if (rows) out.insert(out.end(), {a.q, a.scale});
    if (columns) out.insert(out.end(), {t.q, t.scale});
    return out;
  });
  m.def("fp8_restore", [](const Tensor& q, const Tensor& scale, int64_t cols, int code) -> OptTensor {
    if (!(code == TMPI_F32 || code == TMPI_F16 || code == TMPI_BF16) || !q.is_cuda() || !is_mat(q, scale, cols)) return c10::nullopt;
    const Mat8 a = packed_mat(q, scale);
    Tensor x = at::empty({q.size(0), cols}, q.options().dtype(code == TMPI_F32 ? at::kFloat : code == TMPI_F16 ? at::kHalf : at::kBFloat16));
    check(tmpi_fp8_restore(a.q.data_ptr(), a.scale.data_ptr(), x.data_ptr(), q.size(0), cols, code, stream()));
    launched(FP8, 1);
    return x;
  });
  m.def("fp8_matmul", [](const Tensor& qa, const Tensor& sa, const Tensor& qb, const Tensor& sb, int64_t cols, const OptTensor& bias_, int code) -> OptTensor {
    const Tensor bias = or_none(bias_);
    if (!(code == TMPI_F32 || code == TMPI_F16 || code == TMPI_BF16) || !qa.is_cuda() || !is_mat(qa, sa, cols) || !is_mat(qb, sb, cols)) return c10::nullopt;
    const auto type = code == TMPI_F32 ? at::kFloat : code == TMPI_F16 ? at::kHalf : at::kBFloat16;
    if (!(shaped(bias, {qb.size(0)}) && all_of_type({&bias}, type) && here({&bias}))) return c10::nullopt;
    return product(packed_mat(qa, sa), packed_mat(qb, sb), cols, bias.defined() ? packed(bias.detach()) : bias, false, nullptr, type);
  });
  m.def("fp8_linear_kept", [](const Tensor& x, const Tensor& q, const Tensor& scale, int64_t cols, const OptTensor& bias_, bool gelu) -> OptTensor {
    const Tensor bias = or_none(bias_);
    if (!(x.is_cuda() && floating(x) && x.dim() >= 1 && x.size(-1) == cols && is_mat(q, scale, cols) && shaped(bias, {q.size(0)}) && all_of_type({&bias}, x.scalar_type()) &&
          here({&x, &bias}) && extents(x.numel() / cols, 1, 1) && !wants_grad({x, bias}))) return c10::nullopt;
    return shaped_as(linear_kept(dense_rows(rows_of(x)), packed_mat(q, scale), bias.defined() ? packed(bias) : bias, gelu), x);
  });
  m.def("fp8_linear", [](const Tensor& x, const Tensor& w, const OptTensor& bias_, bool gelu) -> OptTensor {
    const Tensor bias = or_none(bias_);
    if (!(x.is_cuda() && floating(x) && x.dim() >= 1 && w.dim() == 2 && all_of_type({&w, &bias}, x.scalar_type()) && here({&x, &w, &bias}))) return c10::nullopt;
    const int64_t K = w.size(1), N = w.size(0);
    if (!(K >= 1 && x.size(-1) == K && shaped(bias, {N}) && extents(x.numel() / K, N, K))) return c10::nullopt;
    const Tensor x2 = rows_of(x);
    if (wants_grad({x, w, bias})) return shaped_as(Linear8Fn::apply(x2, w, bias_, gelu, x.requires_grad(), w.requires_grad()), x);
    Mat8 kept;
    quantize(dense_rows(w), Tensor(), &kept, nullptr, Tensor());
    return shaped_as(linear_kept(dense_rows(x2), kept, bias.defined() ? packed(bias) : bias, gelu), x);
  });
}

}  // namespace tmpi_bind

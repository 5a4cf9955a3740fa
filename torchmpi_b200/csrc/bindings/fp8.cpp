// Matrices in 8 bits with a scale for each block of 128, their products, and the linear layer that is made of them (ops/fp8.py).  As in experts.cpp an
// entry returns nothing (None) for what the kernels do not take, wrong arguments among it: the Python function then raises, or computes
// with PyTorch's operations.
#include "common.h"
#include <algorithm>

namespace tmpi_bind {
namespace {

struct Mat8 { Tensor q, scale; };                                   // of `rows` rows; what lies behind the columns is zero

void refuse_graph() { TORCH_CHECK(!at::GradMode::is_enabled(), "products in 8 bits can be differentiated once (no create_graph)"); }

Mat8 empty_mat(int64_t rows, int64_t cols) {
  return {fresh({rows, tmpi_fp8_pitch(cols)}, at::kFloat8_e4m3fn), fresh({(int64_t)tmpi_fp8_scale_bytes(rows, cols)}, at::kByte)};
}
// rows whose elements follow each other; the rows themselves may lie apart
Tensor dense_rows(const Tensor& x) { return x.stride(1) == 1 && (x.size(0) < 2 || x.stride(0) >= x.size(1)) ? x : x.contiguous(); }
int64_t pitch(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// The same inside a larger buffer.
struct Place8 {
  char *q = nullptr, *scale = nullptr;
  static int64_t bytes(int64_t rows, int64_t cols) { return aligned(rows * tmpi_fp8_pitch(cols)) + aligned((int64_t)tmpi_fp8_scale_bytes(rows, cols)); }
  static int64_t aligned(int64_t n) { return (n + 255) / 256 * 256; }
  Place8() = default;
  Place8(char* at, int64_t rows, int64_t cols) : q(at), scale(at + aligned(rows * tmpi_fp8_pitch(cols))) {}
  Place8(const Mat8& m) : q((char*)m.q.data_ptr()), scale((char*)m.scale.data_ptr()) {}
};
Tensor bytes(int64_t n) { return fresh({n}, at::kByte); }

// a, t: along the rows and the columns, each where it is given; z, sums: see tmpi_fp8_quantize
void quantize(const Tensor& x, const Tensor& z, const Place8& a, const Place8& t, float* sums) {
  check(tmpi_fp8_quantize(x.data_ptr(), pitch(x), ptr(z), a.q, a.scale, t.q, t.scale, sums, x.size(0), x.size(1), dtype_code(x.scalar_type()), stream()));
  launched(FP8, 1);
}

// a b^T (+ bias) of [M, K] and [N, K]; with gelu the GELU of it, and the rounded sums in z where it is given
Tensor product(const Place8& a, const Place8& b, int64_t M, int64_t N, int64_t K, const Tensor& bias, bool gelu, Tensor* z, at::ScalarType type) {
  Tensor c = fresh({M, N}, type), ws;
  if (z) *z = fresh({M, N}, type);
  const size_t need = tmpi_fp8_product_workspace_bytes((int)M, (int)N, (int)K);
  if (need) ws = bytes((int64_t)need);
  check(tmpi_fp8_product(a.q, a.scale, b.q, b.scale, ptr(bias), c.data_ptr(), z ? z->data_ptr() : nullptr, (int)M, (int)N, (int)K, gelu, dtype_code(c.scalar_type()),
                         need ? ws.data_ptr() : nullptr, need, stream()));
  launched(FP8, need ? 2 : 1);
  return c;
}

// x and w both ways
void quantize_two(const Tensor& x, const Place8& xr, const Place8& xc, const Tensor& w, const Place8& wr, const Place8& wc) {
  const tmpi_fp8_matrix_t two[2] = {{x.data_ptr(), pitch(x), xr.q, xr.scale, xc.q, xc.scale, x.size(0), x.size(1)}, {w.data_ptr(), pitch(w), wr.q, wr.scale, wc.q, wc.scale, w.size(0), w.size(1)}};
  check(tmpi_fp8_quantize_two(two, dtype_code(x.scalar_type()), stream()));
  launched(FP8, 1);
}

// x w^T (+ bias, GELU) without gradients
Tensor linear_kept(const Tensor& x, const Place8& w, int64_t rows, const Tensor& bias, bool gelu) {
  if (x.size(0) <= tmpi_fp8_few_tokens()) {
    Tensor y = fresh({x.size(0), rows}, x.scalar_type());
    check(tmpi_fp8_few(x.data_ptr(), pitch(x), w.q, w.scale, ptr(bias), y.data_ptr(), (int)x.size(0), (int)rows, (int)x.size(1), gelu,
                       dtype_code(x.scalar_type()), stream()));
    launched(FP8, 1);
    return y;
  }
  const Tensor room = bytes(Place8::bytes(x.size(0), x.size(1)));
  const Place8 a((char*)room.data_ptr(), x.size(0), x.size(1));
  quantize(x, Tensor(), a, Place8(), nullptr);
  return product(a, w, x.size(0), rows, x.size(1), bias, gelu, nullptr, x.scalar_type());
}

// Kept for backward: x and w along their columns, in 8 bits, in one buffer, and with a GELU the rounded pre-activation; each where a gradient needs it.
struct Linear8Fn : public torch::autograd::Function<Linear8Fn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const OptTensor& bias_, bool gelu, bool need_x, bool need_w) {
    const Tensor x = dense_rows(x_), w = dense_rows(w_), bias = bias_.has_value() ? packed(*bias_) : Tensor();
    const int64_t T = x.size(0), K = x.size(1), N = w.size(0), xs = Place8::bytes(T, K), xt = need_w ? Place8::bytes(K, T) : 0, wt = need_x ? Place8::bytes(K, N) : 0;
    const Tensor room = bytes(xs + Place8::bytes(N, K));
    Tensor kept, z;
    if (xt + wt) kept = bytes(xt + wt);
    char *at = (char*)room.data_ptr(), *to = xt + wt ? (char*)kept.data_ptr() : nullptr;
    const Place8 xr(at, T, K), wr(at + xs, N, K);
    const Place8 xc = need_w ? Place8(to, K, T) : Place8(), wc = need_x ? Place8(to + xt, K, N) : Place8();
    if (need_x && need_w) {
      quantize_two(x, xr, xc, w, wr, wc);
    } else {
      quantize(x, Tensor(), xr, xc, nullptr);
      quantize(w, Tensor(), wr, wc, nullptr);
    }
    Tensor y = product(xr, wr, T, N, K, bias, gelu, gelu ? &z : nullptr, x.scalar_type());
    ctx->save_for_backward({kept, z});
    ctx->saved_data["kept"] = K << 3 | (need_x ? 1 : 0) | (need_w ? 2 : 0) | (bias.defined() ? 4 : 0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_graph();
    const auto saved = ctx->get_saved_variables();
    const int64_t flags = ctx->saved_data["kept"].toInt();
    const Tensor kept = as_saved(saved[0]), z = as_saved(saved[1]), dy = z.defined() ? packed(grads[0]) : dense_rows(grads[0]);
    const bool need_x = (flags & 1) && ctx->needs_input_grad(0), need_w = (flags & 2) && ctx->needs_input_grad(1),
               need_b = (flags & 4) && ctx->needs_input_grad(2);      // an absent bias has no number among the inputs
    const int64_t T = dy.size(0), N = dy.size(1), K = flags >> 3;
    Tensor dx, dw, db;
    if (need_x || need_w || need_b) {
      const bool columns = need_w || need_b || z.defined();
      const int64_t tiles = (T + 127) / 128, rb = need_x ? Place8::bytes(T, N) : 0, cb = columns ? Place8::bytes(N, T) : 0;
      const Tensor room = bytes(rb + cb + (need_b ? tiles * N * 4 : 0));
      char *at = (char*)room.data_ptr(), *from = kept.defined() ? (char*)kept.data_ptr() : nullptr;
      const Place8 r = need_x ? Place8(at, T, N) : Place8(), c = columns ? Place8(at + rb, N, T) : Place8();
      float* sums = need_b ? (float*)(at + rb + cb) : nullptr;
      quantize(dy, z, r, c, sums);
      if (need_x) dx = product(r, Place8(from + (flags & 2 ? Place8::bytes(K, T) : 0), K, N), T, K, N, Tensor(), false, nullptr, dy.scalar_type());
      if (need_b) db = fresh({N}, dy.scalar_type());
      if (need_w && !need_b) dw = product(c, Place8(from, K, T), N, K, T, Tensor(), false, nullptr, dy.scalar_type());
      if (need_w && need_b) {                          // the bias sums ride along
        const Place8 xc(from, K, T);
        dw = fresh({N, K}, dy.scalar_type());
        const size_t need = tmpi_fp8_product_workspace_bytes((int)N, (int)K, (int)T);
        Tensor ws;
        if (need) ws = bytes((int64_t)need);
        check(tmpi_fp8_product_sums(c.q, c.scale, xc.q, xc.scale, dw.data_ptr(), sums, (int)tiles, db.data_ptr(), (int)N, (int)K, (int)T, dtype_code(dy.scalar_type()), need ? ws.data_ptr() : nullptr,
                                    need, stream()));
        launched(FP8, need ? 2 : 1);
      } else if (need_b) {
        check(tmpi_fp8_column_sums(sums, (int)tiles, (int)N, db.data_ptr(), dtype_code(dy.scalar_type()), stream()));
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
    if (!(x_.is_cuda() && floating(x_) && x_.dim() >= 1 && x_.size(-1) >= 1 && extents(x_.numel() / x_.size(-1), x_.size(-1), 1) && here({&x_}))) return c10::nullopt;
    at::AutoDispatchBelowAutograd no_graph;
    const Tensor x = dense_rows(rows_of(x_));
    Mat8 a, t;
    if (rows) a = empty_mat(x.size(0), x.size(1));
    if (columns) t = empty_mat(x.size(1), x.size(0));
    quantize(x, Tensor(), rows ? Place8(a) : Place8(), columns ? Place8(t) : Place8(), nullptr);
    std::vector<Tensor> out;
    if (rows) out.insert(out.end(), {a.q, a.scale});
    if (columns) out.insert(out.end(), {t.q, t.scale});
    return out;
  });
  m.def("fp8_restore", [](const Tensor& q, const Tensor& scale, int64_t cols, int code) -> OptTensor {
    if (!(code == TMPI_F32 || code == TMPI_F16 || code == TMPI_BF16) || !q.is_cuda() || !is_mat(q, scale, cols)) return c10::nullopt;
    const Mat8 a = packed_mat(q, scale);
    Tensor x = fresh({q.size(0), cols}, code == TMPI_F32 ? at::kFloat : code == TMPI_F16 ? at::kHalf : at::kBFloat16);
    check(tmpi_fp8_restore(a.q.data_ptr(), a.scale.data_ptr(), x.data_ptr(), q.size(0), cols, code, stream()));
    launched(FP8, 1);
    return x;
  });
  m.def("fp8_matmul", [](const Tensor& qa, const Tensor& sa, const Tensor& qb, const Tensor& sb, int64_t cols, const OptTensor& bias_, int code) -> OptTensor {
    const Tensor bias = or_none(bias_);
    if (!(code == TMPI_F32 || code == TMPI_F16 || code == TMPI_BF16) || !qa.is_cuda() || !is_mat(qa, sa, cols) || !is_mat(qb, sb, cols)) return c10::nullopt;
    const auto type = code == TMPI_F32 ? at::kFloat : code == TMPI_F16 ? at::kHalf : at::kBFloat16;
    if (!(shaped(bias, {qb.size(0)}) && all_of_type({&bias}, type) && here({&bias}))) return c10::nullopt;
    const Mat8 a = packed_mat(qa, sa), b = packed_mat(qb, sb);
    return product(a, b, qa.size(0), qb.size(0), cols, bias.defined() ? packed(bias.detach()) : bias, false, nullptr, type);
  });
  m.def("fp8_linear_kept", [](const Tensor& x, const Tensor& q, const Tensor& scale, int64_t cols, const OptTensor& bias_, bool gelu) -> OptTensor {
    const Tensor bias = or_none(bias_);
    if (!(x.is_cuda() && floating(x) && x.dim() >= 1 && x.size(-1) == cols && is_mat(q, scale, cols) && shaped(bias, {q.size(0)}) && all_of_type({&bias}, x.scalar_type()) &&
          here({&x, &bias}) && extents(x.numel() / cols, 1, 1) && !wants_grad({x, bias}))) return c10::nullopt;
    const Mat8 w = packed_mat(q, scale);
    return shaped_as(linear_kept(dense_rows(rows_of(x)), w, q.size(0), bias.defined() ? packed(bias) : bias, gelu), x);
  });
  m.def("fp8_linear", [](const Tensor& x, const Tensor& w, const OptTensor& bias_, bool gelu) -> OptTensor {
    const Tensor bias = or_none(bias_);
    if (!(x.is_cuda() && floating(x) && x.dim() >= 1 && w.dim() == 2 && all_of_type({&w, &bias}, x.scalar_type()) && here({&x, &w, &bias}))) return c10::nullopt;
    const int64_t K = w.size(1), N = w.size(0);
    if (!(K >= 1 && x.size(-1) == K && shaped(bias, {N}) && extents(x.numel() / K, N, K))) return c10::nullopt;
    const Tensor x2 = rows_of(x);
    if (wants_grad({x, w, bias})) return shaped_as(Linear8Fn::apply(x2, w, bias_, gelu, x.requires_grad(), w.requires_grad()), x);
    const Tensor room = bytes(Place8::bytes(N, K));
    const Place8 kept((char*)room.data_ptr(), N, K);
    quantize(dense_rows(w), Tensor(), kept, Place8(), nullptr);
    return shaped_as(linear_kept(dense_rows(x2), kept, N, bias.defined() ? packed(bias) : bias, gelu), x);
  });
}

}  // namespace tmpi_bind

// PyTorch side of the dense 16-bit operators (schemas and documentation: torchair_b200/dense.py): argument checks, layouts,
// workspaces and the autograd formulas around the C entry points of include/tab_api.h.
//
// Why C++: a decode step of these operators runs 5 to 20 microseconds on the GPU.  The same host path in Python took 43 us per
// call of npu_linear_act (8 x 2048 -> 7168), five times the kernel; this one takes about as long as the kernel.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <array>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/tab_api.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kBlock = 64;      // values of a row that share a scale in an 8-bit checkpoint

int64_t up(int64_t v, int64_t step) { return (v + step - 1) / step * step; }

void ok(int rc, const char* entry) { TORCH_CHECK(rc == TAB_OK, entry, " failed (", rc, "): ", tab_last_error()); }

// ---- checks (the same words as the Meta implementations) ----
int act_code(const char* op, c10::string_view a) {
  if (a == "none") return TAB_ACT_NONE;
  if (a == "relu") return TAB_ACT_RELU;
  if (a == "gelu") return TAB_ACT_GELU;
  if (a == "gelu_tanh") return TAB_ACT_GELU_TANH;
  if (a == "silu") return TAB_ACT_SILU;
  TORCH_CHECK(false, op, ": activation '", a, "' (one of none, relu, gelu, gelu_tanh, silu)");
}

int check16(const char* op, const Tensor& x) {
  if (x.scalar_type() == at::kBFloat16) return TAB_BF16;
  if (x.scalar_type() == at::kHalf) return TAB_F16;
  TORCH_CHECK_NOT_IMPLEMENTED(false, op, ": x must be bf16 or fp16, got ", x.scalar_type());
}

void same(const char* op, const Tensor& x, const char* name, const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), op, ": `", name, "` is ", t.scalar_type(), ", x is ", x.scalar_type(),
              "; all 16-bit tensors of a call have one dtype");
  TORCH_CHECK(t.device() == x.device(), op, ": `", name, "` is on ", t.device(), ", x is on ", x.device());
}
void same(const char* op, const Tensor& x, const char* name, const OptTensor& t) {
  if (t.has_value()) same(op, x, name, *t);
}

// ---- layouts ----
struct Call {
  int dtype;
  cudaStream_t stream;
  at::TensorOptions opt;
  // copies that put operands into a layout the kernels take, gathered so that one launch does them all
  mutable std::array<tab_copy, 8> copies;
  mutable int pending = 0;
  mutable std::vector<Tensor> held;      // what the gathered copies read and write lives until they are launched
  void flush() const {
    if (pending == 0) return;
    const int n = pending;
    pending = 0;
    ok(tab_copy_2d(copies.data(), n, stream), "tab_copy_2d");
    held.clear();
  }
  explicit Call(const Tensor& x, int dtype_) : dtype(dtype_), stream(c10::cuda::getCurrentCUDAStream(x.device().index()).stream()), opt(x.options().requires_grad(false)) {}
  // Set while launches run beside one another.  Memory that another host thread freed meanwhile may still be in use by a launch of its own
  // between two of these, and a launch that runs beside that one does not wait for it: what a group of such launches writes is allocated
  // before the ordinary launch that opens the group, which waits for everything that was launched before the memory was handed out.
  mutable bool group_open = false;
  Tensor empty(at::IntArrayRef sizes) const { return empty(sizes, opt); }
  Tensor empty(at::IntArrayRef sizes, at::ScalarType t) const { return empty(sizes, opt.dtype(t)); }
  Tensor workspace(size_t bytes) const { return empty({static_cast<int64_t>(bytes < 256 ? 256 : bytes)}, opt.dtype(at::kByte)); }

 private:
  Tensor empty(at::IntArrayRef sizes, const at::TensorOptions& o) const {
    TORCH_INTERNAL_ASSERT(!group_open, "memory allocated between launches that run beside one another");
    return at::empty(sizes, o);
  }
};

bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

// Columns [dst_col, dst_col + dst_cols) of dst = columns [src_col, src_col + src_cols) of src inside its shape, zero elsewhere (2-D, 16-bit,
// any strides); done by the next flush.
void copy_cols(const Call& c, const Tensor& src, int64_t src_col, int64_t src_cols, const Tensor& dst, int64_t dst_col, int64_t dst_cols) {
  if (c.pending == static_cast<int>(c.copies.size())) c.flush();
  const int64_t ss = src.stride(1), ds = dst.stride(1);
  c.copies[c.pending++] = tab_copy{static_cast<const char*>(src.data_ptr()) + 2 * src_col * ss, src.stride(0), ss, src.size(0), src_cols,
                                   static_cast<char*>(dst.data_ptr()) + 2 * dst_col * ds, dst.stride(0), ds, dst.size(0), dst_cols};
  c.held.push_back(src);
  c.held.push_back(dst);
}
void copy_2d(const Call& c, const Tensor& src, const Tensor& dst) { copy_cols(c, src, 0, src.size(1), dst, 0, dst.size(1)); }

// t as [m, n]
Tensor as_rows(const Tensor& t, int64_t m, int64_t n) { return t.dim() == 2 && t.size(0) == m && t.size(1) == n ? t : t.reshape({m, n}); }

// A matrix in memory that the tensor maps take: contiguous along its columns (row-major) or along its rows, the other stride
// a multiple of 8 elements.
struct Mat {
  Tensor t;
  int64_t ld = 0;
  bool row_major = true;
  const void* ptr() const { return t.data_ptr(); }
  // as operand [index of the product, contraction]: the rows of this matrix are the index ...
  int mn_by_rows() const { return row_major ? 0 : 1; }
  // ... or its columns are
  int mn_by_cols() const { return row_major ? 1 : 0; }
};

// t [m, n] row-major: itself where its memory allows that, else a copy with rows of `pitch` >= n elements (a multiple of 8), zero
// behind n
Mat rows_of(const Call& c, const Tensor& t, int64_t pitch) {
  const int64_t n = t.size(1);
  if ((t.stride(1) == 1 || n == 1) && aligned(t)) {
    if (t.size(0) <= 1) return {t, pitch, true};
    if (t.stride(0) % 8 == 0 && t.stride(0) >= n) return {t, t.stride(0), true};
  }
  Tensor out = c.empty({t.size(0), pitch});
  copy_2d(c, t, out);
  return {out, pitch, true};
}

// the same with zeros behind the n columns, whatever lies there in t's memory
Mat padded_rows(const Call& c, const Tensor& t, int64_t pitch) {
  Tensor out = c.empty({t.size(0), pitch});
  copy_2d(c, t, out);
  return {out, pitch, true};
}

bool col_major(const Tensor& t) { return t.stride(0) == 1 && t.stride(1) != 1; }

// a weight [r, c], copied if need be; keeps the order in memory that the weight (and so its gradient) has
Mat matrix_of(const Call& c, const Tensor& t) {
  const int64_t rows = t.size(0), cols = t.size(1);
  if (aligned(t)) {
    if (t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= cols) return {t, t.stride(0), true};
    if (t.stride(0) == 1 && t.stride(1) % 8 == 0 && t.stride(1) >= rows) return {t, t.stride(1), false};
  }
  const bool cm = col_major(t);
  const int64_t pitch = up(cm ? rows : cols, 8);
  Tensor out = cm ? c.empty({cols, pitch}).t() : c.empty({rows, pitch});
  copy_2d(c, t, out);
  return {out, pitch, !cm};
}

// weight1 [H, 2 I] with either half padded to `half` columns when I is not a multiple of 8
Mat halves_of(const Call& c, const Tensor& t, int64_t half) {
  const int64_t rows = t.size(0), inner = t.size(1) / 2;
  if (inner == half) return matrix_of(c, t);
  const bool cm = col_major(t);
  const int64_t pitch = cm ? up(rows, 8) : 2 * half;
  Tensor out = cm ? c.empty({2 * half, pitch}).t() : c.empty({rows, pitch});
  copy_cols(c, t, 0, inner, out, 0, half);
  copy_cols(c, t, inner, inner, out, half, half);
  return {out, pitch, !cm};
}

// weight2 [I, H] with zero rows behind I
Tensor padded_weight2(const Call& c, const Tensor& t, int64_t rows) {
  const int64_t cols = t.size(1);
  Tensor out = col_major(t) ? c.empty({cols, rows}).t() : c.empty({rows, up(cols, 8)}).narrow(1, 0, cols);
  copy_2d(c, t, out);
  return out;
}

// t [m, n] without gaps between rows, 16-byte aligned where that makes its rows whole pieces
Tensor dense_rows(const Call& c, const Tensor& t) {
  if (t.is_contiguous() && (aligned(t) || t.size(1) % 8 != 0)) return t;
  Tensor out = c.empty({t.size(0), t.size(1)});
  copy_2d(c, t, out);
  return out;
}

// a bias without gaps
Tensor vector_of(const Call& c, const OptTensor& t) {
  if (!t.has_value()) return Tensor();
  return dense_rows(c, t->unsqueeze(0));
}
// bias1 [2 I], either half padded to `half` values, 16-byte aligned
Tensor halves_vector(const Call& c, const OptTensor& t, int64_t half) {
  if (!t.has_value()) return Tensor();
  if (t->size(0) == 2 * half) {
    if (t->stride(0) == 1 && aligned(*t)) return *t;
    Tensor out = c.empty({1, 2 * half});
    copy_2d(c, t->unsqueeze(0), out);
    return out;
  }
  return halves_of(c, t->unsqueeze(0), half).t;
}

// the first n values of a padded row of sums
Tensor cut_row(const Call& c, const Tensor& t, int64_t n) {
  if (t.size(1) == n) return t.view({n});
  Tensor out = c.empty({1, n});
  copy_cols(c, t, 0, n, out, 0, n);
  return out.view({n});
}
// [rows, 2 I8] -> [rows, 2 I], in the same order
Tensor cut_halves(const Call& c, const Tensor& t, int64_t inner) {
  const int64_t rows = t.size(0), half = t.size(1) / 2;
  if (half == inner) return t;
  Tensor out = col_major(t) ? c.empty({2 * inner, rows}).t() : c.empty({rows, 2 * inner});
  copy_cols(c, t, 0, inner, out, 0, inner);
  copy_cols(c, t, half, inner, out, inner, inner);
  return out;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// what a forward pass keeps for its backward pass: 16-bit values, or int8 with scales
struct Kept {
  Tensor values, scale, x_q, x_scale;
  bool int8() const { return values.defined() && values.scalar_type() == at::kChar; }
  void* p16() const { return values.defined() && !int8() ? values.data_ptr() : nullptr; }
  int8_t* p8() const { return int8() ? static_cast<int8_t*>(values.data_ptr()) : nullptr; }
  float* ps() const { return int8() ? static_cast<float*>(scale.data_ptr()) : nullptr; }
  int64_t ld() const { return values.defined() ? values.size(1) : 0; }
};

// act(a b^T + bias) + residual: a [m, k], b [n, k] as operands
void matmul(const Call& c, const void* a, int64_t lda, int a_mn, const void* b, int64_t ldb, int b_mn, int64_t m, int64_t n, int64_t k, const Tensor& out,
            const Tensor& bias = Tensor(), const Tensor& residual = Tensor(), int act = 0, const Kept& kept = Kept(), bool beside = false) {
  beside = beside && c.pending == 0;           // a product does not run beside the copy that it reads
  c.flush();
  ok(tab_dense_matmul(a, lda, a_mn, b, ldb, b_mn, c.dtype, m, n, k, ptr(bias), ptr(residual), act, kept.p16(), kept.p8(), kept.ps(), kept.ld(),
                      out.data_ptr(), beside, c.stream),
     "tab_dense_matmul");
}

// memory for the gradient [k, n] of a weight, in the memory order of the weight `like`
Tensor weight_grad_memory(const Call& c, int64_t k, int64_t n, const Tensor& like) {
  return col_major(like) ? c.empty({n, k}).t() : c.empty({k, n});
}

// x^T dz (both row-major) into out [k, n], which weight_grad_memory gave for `like`
void weight_grad(const Call& c, const Mat& x, const Mat& dz, int64_t k, int64_t n, const Tensor& like, const Tensor& out, bool beside) {
  const int64_t m = x.t.size(0);
  if (col_major(like))
    matmul(c, dz.ptr(), dz.ld, 1, x.ptr(), x.ld, 1, n, k, m, out, Tensor(), Tensor(), 0, Kept(), beside);
  else
    matmul(c, x.ptr(), x.ld, 1, dz.ptr(), dz.ld, 1, k, n, m, out, Tensor(), Tensor(), 0, Kept(), beside);
}

// a weight gradient without rows to sum over
Tensor zero_grad(const Call& c, const Tensor& like) {
  return col_major(like) ? at::zeros({like.size(1), like.size(0)}, c.opt).t() : at::zeros({like.size(0), like.size(1)}, c.opt);
}

// dz = grad act'(kept) (grad itself without an activation) and, if wanted, its column sums
Mat act_grad(const Call& c, const Mat& grad, int64_t n, int act, const Kept& kept, bool want_dz, bool want_sums, Tensor& column_sums) {
  const int64_t m = grad.t.size(0);
  Tensor dz = want_dz && act ? c.empty({m, n}) : Tensor(), parts;
  if (want_sums) {
    size_t splits = 0;
    ok(tab_act_grad_splits(m, n, &splits), "tab_act_grad_splits");
    parts = c.empty({static_cast<int64_t>(splits), n}, at::kFloat);
  }
  if (dz.defined() || parts.defined()) {
    c.flush();
    ok(tab_act_grad(grad.ptr(), grad.ld, c.dtype, m, n, act, kept.p16(), kept.p8(), kept.ps(), kept.ld(), ptr(dz), static_cast<float*>(ptr(parts)),
                    c.stream),
       "tab_act_grad");
  }
  if (want_sums) {
    column_sums = c.empty({1, n});
    ok(tab_column_sums(static_cast<const float*>(parts.data_ptr()), parts.size(0), n, column_sums.data_ptr(), c.dtype, c.stream), "tab_column_sums");
  }
  return act ? Mat{dz, n, true} : grad;
}

int any_dtype(at::ScalarType t) { return t == at::kBFloat16 ? TAB_BF16 : t == at::kHalf ? TAB_F16 : t == at::kFloat ? TAB_F32 : 0; }

void quantise(cudaStream_t stream, const Tensor& x, int64_t rows, int64_t cols, int64_t ldx, const Tensor& q, const Tensor& scale) {
  ok(tab_checkpoint_quant(x.data_ptr(), any_dtype(x.scalar_type()), ldx, rows, cols, static_cast<int8_t*>(q.data_ptr()), cols,
                          static_cast<float*>(scale.data_ptr()), up(cols, kBlock) / kBlock, stream),
     "tab_checkpoint_quant");
}

// x [m, k] kept in 8 bits for the weight gradient
void keep_x(const Call& c, const Tensor& x, Kept& kept) {
  const Tensor xr = x.stride(1) == 1 && (x.size(0) <= 1 || x.stride(0) >= x.size(1)) ? x : x.contiguous();
  kept.x_q = c.empty({x.size(0), x.size(1)}, at::kChar);
  kept.x_scale = c.empty({x.size(0), up(x.size(1), kBlock) / kBlock}, at::kFloat);
  quantise(c.stream, xr, x.size(0), x.size(1), xr.stride(0), kept.x_q, kept.x_scale);
}

// memory for int8 [m, k] in 16 bits: rows of a multiple of 8 values
Mat dequantised_memory(const Call& c, const Tensor& q) {
  const int64_t pitch = up(q.size(1), 8);
  return {c.empty({q.size(0), pitch}), pitch, true};
}

// int8 [m, k] with its scales (no gaps) -> 16 bits, zero behind k
void dequantise(const Call& c, const Tensor& q, const Tensor& scale, const Mat& y, bool beside = false) {
  ok(tab_checkpoint_dequant(static_cast<const int8_t*>(q.data_ptr()), q.size(1), static_cast<const float*>(scale.data_ptr()), scale.size(1), q.size(0),
                            q.size(1), y.t.data_ptr(), c.dtype, y.ld, y.ld, beside, c.stream),
     "tab_checkpoint_dequant");
}

using Five = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

Five keep_results(const Call& c, const Tensor& y, const Kept& k) {
  auto or_empty = [&](const Tensor& t, at::ScalarType s) { return t.defined() ? t : c.empty({0}, s); };
  return Five(y, k.values, or_empty(k.scale, at::kFloat), or_empty(k.x_q, at::kChar), or_empty(k.x_scale, at::kFloat));
}

// ---- npu_gated_ffn ----
struct FfnSizes {
  int dtype, act;
  int64_t h, inner, m;
};

FfnSizes ffn_check(const Tensor& x, const Tensor& w1, const Tensor& w2, const OptTensor& b1, const OptTensor& b2, const OptTensor& r, c10::string_view act) {
  const char* op = "npu_gated_ffn";
  FfnSizes s;
  s.dtype = check16(op, x);
  TORCH_CHECK(x.dim() >= 1 && w1.dim() == 2 && w2.dim() == 2, op, ": x must be [..., H], weight1 [H, 2 I] and weight2 [I, H]");
  s.h = x.size(-1);
  s.inner = w2.size(0);
  TORCH_CHECK(s.h > 0 && s.inner > 0 && w1.size(0) == s.h && w1.size(1) == 2 * s.inner && w2.size(1) == s.h, op, ": x ", x.sizes(), ", weight1 ", w1.sizes(),
              " and weight2 ", w2.sizes(), " do not fit [..., H], [H, 2 I] and [I, H]");
  TORCH_CHECK((!b1.has_value() || (b1->dim() == 1 && b1->size(0) == 2 * s.inner)) && (!b2.has_value() || (b2->dim() == 1 && b2->size(0) == s.h)), op,
              ": bias1 must be [2 I] = [", 2 * s.inner, "] and bias2 [H] = [", s.h, "]");
  TORCH_CHECK(!r.has_value() || r->sizes() == x.sizes(), op, ": residual must have the shape of x, got ", r.has_value() ? r->sizes() : x.sizes());
  same(op, x, "weight1", w1);
  same(op, x, "weight2", w2);
  same(op, x, "bias1", b1);
  same(op, x, "bias2", b2);
  same(op, x, "residual", r);
  s.act = act_code(op, act);
  s.m = x.numel() / s.h;
  return s;
}

Tensor ffn_forward(const Call& c, const FfnSizes& s, const Tensor& x, const Tensor& weight1, const Tensor& weight2, const OptTensor& bias1,
                   const OptTensor& bias2, const OptTensor& residual, const Kept& kept) {
  const int64_t inner8 = up(s.inner, 8);
  Tensor y = c.empty(x.sizes());
  if (s.m > 0) {
    const Mat xm = rows_of(c, as_rows(x, s.m, s.h), up(s.h, 8));
    const Mat w1 = halves_of(c, weight1, inner8), w2 = matrix_of(c, weight2);
    const Tensor b1 = halves_vector(c, bias1, inner8), b2 = vector_of(c, bias2);
    const Tensor r = residual.has_value() ? dense_rows(c, as_rows(*residual, s.m, s.h)) : Tensor();
    size_t bytes = 0;
    ok(tab_gated_ffn_workspace_bytes(s.m, s.h, inner8, &bytes), "tab_gated_ffn_workspace_bytes");
    const Tensor ws = c.workspace(bytes);
    c.flush();
    ok(tab_gated_ffn(xm.ptr(), xm.ld, w1.ptr(), w1.ld, w1.mn_by_cols(), w2.ptr(), w2.ld, w2.mn_by_cols(), s.inner, c.dtype, s.m, s.h, inner8, ptr(b1),
                     ptr(b2), ptr(r), s.act, kept.p16(), kept.p8(), kept.ps(), kept.ld(), y.data_ptr(), ws.data_ptr(), ws.numel(), c.stream),
       "tab_gated_ffn");
  }
  return y;
}

Tensor ffn_cuda(const Tensor& x, const Tensor& weight1, const Tensor& weight2, const OptTensor& bias1, const OptTensor& bias2, const OptTensor& residual,
                c10::string_view activation, bool) {
  const FfnSizes s = ffn_check(x, weight1, weight2, bias1, bias2, residual, activation);
  const c10::cuda::CUDAGuard guard(x.device());
  return ffn_forward(Call(x, s.dtype), s, x, weight1, weight2, bias1, bias2, residual, Kept());
}

Five ffn_keep_cuda(const Tensor& x, const Tensor& weight1, const Tensor& weight2, const OptTensor& bias1, const OptTensor& bias2, const OptTensor& residual,
                   c10::string_view activation, bool int8) {
  const FfnSizes s = ffn_check(x, weight1, weight2, bias1, bias2, residual, activation);
  const c10::cuda::CUDAGuard guard(x.device());
  const Call c(x, s.dtype);
  Kept kept;
  if (int8) {
    keep_x(c, as_rows(x, s.m, s.h), kept);
    const int64_t width = 2 * up(s.inner, kBlock);
    kept.values = c.empty({s.m, width}, at::kChar);
    kept.scale = c.empty({s.m, width / kBlock}, at::kFloat);
  } else {
    kept.values = c.empty({s.m, 2 * up(s.inner, 8)});
  }
  const Tensor y = ffn_forward(c, s, x, weight1, weight2, bias1, bias2, residual, kept);
  return keep_results(c, y, kept);
}

Five ffn_backward_cuda(const Tensor& grad_, const Tensor& x_, const Tensor& x_scale, const Tensor& weight1, const Tensor& weight2, const Tensor& kept_values,
                       const Tensor& kept_scale, c10::string_view activation, std::array<bool, 5> want) {
  const char* op = "npu_gated_ffn_backward";
  const int dtype = check16(op, grad_), act = act_code(op, activation);
  TORCH_CHECK(weight1.dim() == 2 && weight2.dim() == 2 && grad_.dim() >= 1, op, ": grad must be [..., H], weight1 [H, 2 I] and weight2 [I, H]");
  const int64_t inner = weight2.size(0), h = weight2.size(1);
  const bool int8 = kept_values.scalar_type() == at::kChar, x8 = x_.scalar_type() == at::kChar;
  TORCH_CHECK(h > 0 && inner > 0 && grad_.size(-1) == h && weight1.size(0) == h && weight1.size(1) == 2 * inner, op, ": grad ", grad_.sizes(), ", weight1 ",
              weight1.sizes(), " and weight2 ", weight2.sizes(), " do not fit [..., H], [H, 2 I] and [I, H]");
  same(op, grad_, "weight1", weight1);
  same(op, grad_, "weight2", weight2);
  const int64_t m = grad_.numel() / h, h8 = up(h, 8), inner8 = up(inner, 8), width = 2 * up(inner, int8 ? kBlock : 8);
  TORCH_CHECK(kept_values.dim() == 2 && kept_values.size(0) == m && kept_values.size(1) == width && kept_values.is_contiguous() &&
                  (int8 ? kept_scale.numel() == m * width / kBlock && kept_scale.scalar_type() == at::kFloat && kept_scale.is_contiguous()
                        : kept_values.scalar_type() == grad_.scalar_type()) &&
                  kept_values.device() == grad_.device() && (!int8 || kept_scale.device() == grad_.device()),
              op, ": kept ", kept_values.sizes(), " does not hold the gate and up values of ", m, " rows");
  TORCH_CHECK(!want[1] || (x_.numel() == m * h && x_.device() == grad_.device() && (x8 ? x_.is_contiguous() && x_scale.is_contiguous() && x_scale.scalar_type() == at::kFloat && x_scale.numel() == m * (up(h, kBlock) / kBlock) && x_scale.device() == grad_.device() : x_.scalar_type() == grad_.scalar_type())), op,
              ": x ", x_.sizes(), " does not fit grad ", grad_.sizes());
  const c10::cuda::CUDAGuard guard(grad_.device());
  const Call c(grad_, dtype);
  Tensor none, dx, dw1, dw2, db1, db2;
  auto result = [&](const Tensor& t) -> Tensor {
    if (t.defined()) return t;
    if (!none.defined()) none = c.empty({0});
    return none;
  };
  if (m == 0) {
    if (want[0]) dx = at::zeros(grad_.sizes(), c.opt);
    if (want[1]) dw1 = zero_grad(c, weight1);
    if (want[2]) dw2 = zero_grad(c, weight2);
    if (want[3]) db1 = at::zeros({2 * inner}, c.opt);
    if (want[4]) db2 = at::zeros({h}, c.opt);
    return Five(result(dx), result(dw1), result(dw2), result(db1), result(db2));
  }
  // column sums read whole pieces of 8: a gradient whose rows are not is copied for them with zeros behind h
  const Mat dy = want[4] && h8 != h ? padded_rows(c, as_rows(grad_, m, h), h8) : rows_of(c, as_rows(grad_, m, h), h8);
  Mat w1, xm;
  if (want[0]) w1 = halves_of(c, weight1, inner8);
  if (want[1] && !x8) xm = rows_of(c, as_rows(x_, m, h), h8);
  Kept kept;
  kept.values = kept_values;
  kept.scale = kept_scale;
  Mat dz{Tensor(), 2 * inner8, true}, hidden{Tensor(), inner8, true};
  const bool any = want[0] || want[1] || want[2] || want[3];
  // Launches that run beside one another: everything that they touch is allocated before the first of them and stays so until all of them
  // are launched (see Call::group_open).
  Mat w2;
  if (any) {
    w2 = matrix_of(c, inner == inner8 ? weight2 : padded_weight2(c, weight2, inner8));
    dz.t = c.empty({m, 2 * inner8});
    hidden.t = c.empty({m, inner8});
  }
  Tensor x_q, x_s;
  if (want[1] && x8) {
    x_q = as_rows(x_, m, h);
    x_s = as_rows(x_scale, m, up(h, kBlock) / kBlock);
    xm = dequantised_memory(c, x_q);
  }
  if (want[0]) dx = c.empty(grad_.sizes());
  if (want[1]) dw1 = weight_grad_memory(c, h, 2 * inner8, weight1);
  if (want[2]) dw2 = weight_grad_memory(c, inner, h, weight2);
  if (want[3]) db1 = c.empty({1, 2 * inner8});
  if (want[4]) db2 = c.empty({1, h8});
  // both sums in slices that do not depend on which of them are wanted, and so neither do their values
  const Mat &first = want[3] ? dz : dy, &second = want[3] && want[4] ? dy : Mat();
  const int64_t n1 = want[3] ? 2 * inner8 : h8, n2 = want[3] && want[4] ? h8 : 0;
  Tensor parts;
  if (want[3] || want[4]) {
    size_t splits = 0;
    ok(tab_act_grad_splits(m, 2 * inner8 + h8, &splits), "tab_act_grad_splits");
    parts = c.empty({static_cast<int64_t>(splits), n1 + n2}, at::kFloat);
  }
  c.flush();
  c.group_open = true;
  if (any) {
    ok(tab_gated_matmul_grad(dy.ptr(), dy.ld, w2.ptr(), w2.ld, w2.mn_by_rows(), dtype, m, inner8, h, act, kept.p16(), kept.p8(), kept.ps(), kept.ld(),
                             dz.t.data_ptr(), hidden.t.data_ptr(), c.stream),
       "tab_gated_matmul_grad");
    if (want[0] && inner != inner8) {      // the product for dx runs over the columns behind I too: infinities leave NaN there
      copy_cols(c, dz.t, 0, 0, dz.t, inner, inner8 - inner);
      copy_cols(c, dz.t, 0, 0, dz.t, inner8 + inner, inner8 - inner);
      c.flush();
    }
  }
  if (want[1] && x8) dequantise(c, x_q, x_s, xm, any);
  // What is left depends on nothing but what is ordered before it: each launch may start in the SMs that the last turn of the one before
  // leaves idle.
  bool beside = false;
  if (want[2]) {
    weight_grad(c, hidden, dy, inner, h, weight2, dw2, beside);
    beside = true;
  }
  if (want[0]) {
    matmul(c, dz.ptr(), dz.ld, 0, w1.ptr(), w1.ld, w1.mn_by_rows(), m, h, 2 * inner8, dx, Tensor(), Tensor(), 0, Kept(), beside);
    beside = true;
  }
  if (want[1]) {
    weight_grad(c, xm, dz, h, 2 * inner8, weight1, dw1, beside);
    beside = true;
  }
  if (parts.defined())
    ok(tab_two_column_sums(first.ptr(), first.ld, n1, n2 ? second.ptr() : nullptr, second.ld, n2, dtype, m, static_cast<float*>(parts.data_ptr()),
                           parts.size(0), want[3] ? db1.data_ptr() : db2.data_ptr(), n2 ? db2.data_ptr() : nullptr, beside, c.stream),
       "tab_two_column_sums");
  c.group_open = false;
  if (want[1]) dw1 = cut_halves(c, dw1, inner);
  if (want[3]) db1 = cut_halves(c, db1, inner).view({2 * inner});
  if (want[4]) db2 = cut_row(c, db2, h);
  c.flush();
  return Five(result(dx), result(dw1), result(dw2), result(db1), result(db2));
}

// ---- npu_linear_act ----
struct LinearSizes {
  int dtype, act;
  int64_t k, n, m;
};

LinearSizes linear_check(const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r, c10::string_view act, at::DimVector& out_sizes) {
  const char* op = "npu_linear_act";
  LinearSizes s;
  s.dtype = check16(op, x);
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && w.size(0) == x.size(-1) && w.size(0) > 0 && w.size(1) > 0, op, ": x ", x.sizes(), " and weight ", w.sizes(),
              " do not fit [..., K] and [K, N]");
  s.k = w.size(0);
  s.n = w.size(1);
  TORCH_CHECK(!b.has_value() || (b->dim() == 1 && b->size(0) == s.n), op, ": bias must be [N] = [", s.n, "]");
  out_sizes = at::DimVector(x.sizes());
  out_sizes.back() = s.n;
  TORCH_CHECK(!r.has_value() || r->sizes() == at::IntArrayRef(out_sizes), op, ": residual must be ", at::IntArrayRef(out_sizes), ", got ",
              r.has_value() ? r->sizes() : x.sizes());
  same(op, x, "weight", w);
  same(op, x, "bias", b);
  same(op, x, "residual", r);
  s.act = act_code(op, act);
  s.m = x.numel() / s.k;
  return s;
}

Tensor linear_forward(const Call& c, const LinearSizes& s, at::IntArrayRef out_sizes, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                      const OptTensor& residual, const Kept& kept) {
  Tensor y = c.empty(out_sizes);
  if (s.m > 0) {
    const Mat xm = rows_of(c, as_rows(x, s.m, s.k), up(s.k, 8));
    const Mat w = matrix_of(c, weight);
    const Tensor b = vector_of(c, bias);
    const Tensor r = residual.has_value() ? dense_rows(c, as_rows(*residual, s.m, s.n)) : Tensor();
    matmul(c, xm.ptr(), xm.ld, 0, w.ptr(), w.ld, w.mn_by_cols(), s.m, s.n, s.k, y, b, r, s.act, kept);
  }
  return y;
}

Tensor linear_cuda(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, c10::string_view activation, bool) {
  at::DimVector out_sizes;
  const LinearSizes s = linear_check(x, weight, bias, residual, activation, out_sizes);
  const c10::cuda::CUDAGuard guard(x.device());
  return linear_forward(Call(x, s.dtype), s, out_sizes, x, weight, bias, residual, Kept());
}

Five linear_keep_cuda(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, c10::string_view activation, bool int8) {
  at::DimVector out_sizes;
  const LinearSizes s = linear_check(x, weight, bias, residual, activation, out_sizes);
  const c10::cuda::CUDAGuard guard(x.device());
  const Call c(x, s.dtype);
  Kept kept;
  if (int8) keep_x(c, as_rows(x, s.m, s.k), kept);
  // without an activation the backward pass does not need its argument
  const int64_t width = s.act ? up(s.n, int8 ? kBlock : 8) : 0;
  Kept stored;
  if (s.act) {
    stored.values = c.empty({s.m, width}, int8 ? at::kChar : x.scalar_type());
    if (int8) stored.scale = c.empty({s.m, width / kBlock}, at::kFloat);
  }
  const Tensor y = linear_forward(c, s, out_sizes, x, weight, bias, residual, stored);
  kept.values = s.act ? stored.values : c.empty({s.m, 0}, int8 ? at::kChar : x.scalar_type());
  kept.scale = stored.scale.defined() ? stored.scale : int8 ? c.empty({s.m, 0}, at::kFloat) : Tensor();
  return keep_results(c, y, kept);
}

std::tuple<Tensor, Tensor, Tensor> linear_backward_cuda(const Tensor& grad_, const Tensor& x_, const Tensor& x_scale, const Tensor& weight,
                                                        const Tensor& kept_values, const Tensor& kept_scale, c10::string_view activation,
                                                        std::array<bool, 3> want) {
  const char* op = "npu_linear_act_backward";
  const int dtype = check16(op, grad_), act = act_code(op, activation);
  TORCH_CHECK(weight.dim() == 2 && grad_.dim() >= 1 && grad_.size(-1) == weight.size(1) && weight.size(0) > 0 && weight.size(1) > 0, op, ": grad ",
              grad_.sizes(), " and weight ", weight.sizes(), " do not fit [..., N] and [K, N]");
  same(op, grad_, "weight", weight);
  const int64_t k = weight.size(0), n = weight.size(1), m = grad_.numel() / n, n8 = up(n, 8);
  const bool int8 = kept_values.scalar_type() == at::kChar, x8 = x_.scalar_type() == at::kChar;
  const int64_t width = up(n, int8 ? kBlock : 8);
  TORCH_CHECK(act == TAB_ACT_NONE ||
                  (kept_values.dim() == 2 && kept_values.size(0) == m && kept_values.size(1) == width && kept_values.is_contiguous() &&
                   (int8 ? kept_scale.numel() == m * width / kBlock && kept_scale.scalar_type() == at::kFloat && kept_scale.is_contiguous()
                         : kept_values.scalar_type() == grad_.scalar_type()) &&
                   kept_values.device() == grad_.device() && (!int8 || kept_scale.device() == grad_.device())),
              op, ": kept ", kept_values.sizes(), " does not hold the activation's arguments of ", m, " rows");
  TORCH_CHECK(!want[1] || (x_.numel() == m * k && x_.device() == grad_.device() && (x8 ? x_.is_contiguous() && x_scale.is_contiguous() && x_scale.scalar_type() == at::kFloat && x_scale.numel() == m * (up(k, kBlock) / kBlock) && x_scale.device() == grad_.device() : x_.scalar_type() == grad_.scalar_type())), op,
              ": x ", x_.sizes(), " does not fit grad ", grad_.sizes());
  at::DimVector x_sizes(grad_.sizes());
  x_sizes.back() = k;
  const c10::cuda::CUDAGuard guard(grad_.device());
  const Call c(grad_, dtype);
  Tensor dx, dw, db;
  if (m == 0) {
    if (want[0]) dx = at::zeros(x_sizes, c.opt);
    if (want[1]) dw = zero_grad(c, weight);
    if (want[2]) db = at::zeros({n}, c.opt);
  } else {
    Kept kept;
    if (act) {
      kept.values = kept_values;
      kept.scale = kept_scale;
    }
    Mat w, xm;
    if (want[0]) w = matrix_of(c, weight);
    if (want[1] && !x8) xm = rows_of(c, as_rows(x_, m, k), up(k, 8));
    // the elementwise kernel reads whole pieces of 8
    const Mat dy = n8 != n && (act || want[2]) ? padded_rows(c, as_rows(grad_, m, n), n8) : rows_of(c, as_rows(grad_, m, n), n8);
    const Mat dz = act_grad(c, dy, n8, act, kept, want[0] || want[1], want[2], db);
    if (want[1] && x8) {
      const Tensor q = as_rows(x_, m, k);
      xm = dequantised_memory(c, q);
      dequantise(c, q, as_rows(x_scale, m, up(k, kBlock) / kBlock), xm);
    }
    if (want[0]) dx = c.empty(x_sizes);
    if (want[1]) dw = weight_grad_memory(c, k, n, weight);
    c.flush();
    c.group_open = true;
    if (want[0]) matmul(c, dz.ptr(), dz.ld, 0, w.ptr(), w.ld, w.mn_by_rows(), m, k, n, dx);
    if (want[1]) weight_grad(c, xm, dz, k, n, weight, dw, want[0]);        // beside the one before: see npu_gated_ffn_backward
    c.group_open = false;
    if (want[2]) db = cut_row(c, db, n);
    c.flush();
  }
  auto result = [&](const Tensor& t) { return t.defined() ? t : c.empty({0}); };
  return {result(dx), result(dw), result(db)};
}

// ---- 8-bit checkpoints ----
void ck_check(const char* op, const Tensor& q, const Tensor& scale) {
  TORCH_CHECK(q.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat, op, ": q must be int8 and scale fp32, got ", q.scalar_type(), " and ",
              scale.scalar_type());
  bool fits = q.dim() >= 1 && scale.dim() == q.dim() && scale.size(-1) == up(q.size(-1), kBlock) / kBlock;
  for (int64_t i = 0; fits && i + 1 < q.dim(); ++i) fits = q.size(i) == scale.size(i);
  TORCH_CHECK(fits, op, ": scale ", scale.sizes(), " does not hold one value per row and 64 values of q ", q.sizes());
  TORCH_CHECK(q.device() == scale.device(), op, ": q is on ", q.device(), ", scale is on ", scale.device());
}

std::tuple<Tensor, Tensor> ck_quant_cuda(const Tensor& x) {
  const char* op = "npu_checkpoint_quant";
  TORCH_CHECK_NOT_IMPLEMENTED(any_dtype(x.scalar_type()) != 0, op, ": x must be bf16, fp16 or fp32, got ", x.scalar_type());
  TORCH_CHECK(x.dim() >= 1, op, ": x must have at least one dimension");
  const c10::cuda::CUDAGuard guard(x.device());
  const Call c(x, any_dtype(x.scalar_type()));
  const int64_t cols = x.size(-1);
  at::DimVector scale_sizes(x.sizes());
  scale_sizes.back() = up(cols, kBlock) / kBlock;
  Tensor q = c.empty(x.sizes(), at::kChar), scale = c.empty(scale_sizes, at::kFloat);
  if (x.numel() > 0) {
    const int64_t rows = x.numel() / cols;
    const bool as_is = x.dim() == 2 && x.stride(1) == 1 && (rows == 1 || x.stride(0) >= cols);
    const Tensor xc = as_is ? x : x.contiguous();
    quantise(c.stream, xc, rows, cols, as_is ? x.stride(0) : cols, q, scale);
  }
  return {q, scale};
}

Tensor ck_dequant_cuda(const Tensor& q, const Tensor& scale, int64_t output_dtype) {
  const char* op = "npu_checkpoint_dequant";
  ck_check(op, q, scale);
  TORCH_CHECK_NOT_IMPLEMENTED(output_dtype == TAB_F16 || output_dtype == TAB_F32 || output_dtype == TAB_BF16, op, ": output_dtype=", output_dtype,
                              " (5 fp16, 6 fp32 or 15 bf16)");
  const c10::cuda::CUDAGuard guard(q.device());
  const Call c(q, static_cast<int>(output_dtype));
  Tensor y = c.empty(q.sizes(), output_dtype == TAB_F16 ? at::kHalf : output_dtype == TAB_F32 ? at::kFloat : at::kBFloat16);
  if (y.numel() > 0) {
    const int64_t cols = q.size(-1);
    const Tensor qc = q.contiguous(), sc = scale.contiguous();
    ok(tab_checkpoint_dequant(static_cast<const int8_t*>(qc.data_ptr()), cols, static_cast<const float*>(sc.data_ptr()), sc.size(-1), q.numel() / cols, cols,
                              y.data_ptr(), c.dtype, cols, cols, 0, c.stream),
       "tab_checkpoint_dequant");
  }
  return y;
}

Tensor ck_weight_grad_cuda(const Tensor& q_, const Tensor& scale_, const Tensor& grad_) {
  const char* op = "npu_checkpoint_weight_grad";
  ck_check(op, q_, scale_);
  const int dtype = check16(op, grad_);
  bool fits = grad_.dim() == q_.dim() && grad_.size(-1) > 0 && q_.size(-1) > 0;
  for (int64_t i = 0; fits && i + 1 < q_.dim(); ++i) fits = q_.size(i) == grad_.size(i);
  TORCH_CHECK(fits, op, ": q ", q_.sizes(), " and grad ", grad_.sizes(), " must be [..., K] and [..., N] of the same rows");
  TORCH_CHECK(grad_.device() == q_.device(), op, ": grad is on ", grad_.device(), ", q is on ", q_.device());
  const int64_t k = q_.size(-1), n = grad_.size(-1), m = q_.numel() / k;
  const c10::cuda::CUDAGuard guard(grad_.device());
  const Call c(grad_, dtype);
  if (m == 0) return at::zeros({k, n}, c.opt);
  const Tensor q = q_.contiguous().view({m, k}), scale = scale_.contiguous().view({m, -1});
  const Mat x = dequantised_memory(c, q), dz = rows_of(c, as_rows(grad_, m, n), up(n, 8));
  dequantise(c, q, scale, x);
  Tensor out = c.empty({k, n});
  matmul(c, x.ptr(), x.ld, 1, dz.ptr(), dz.ld, 1, k, n, m, out);
  return out;
}

// ---- autograd ----
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

template <typename Sig>
c10::TypedOperatorHandle<Sig> handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const OptTensor& t) { return t.has_value() && t->requires_grad(); }

// There is no forward-mode formula: a tangent raises instead of being dropped.
void no_tangent(const char* op, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), op, ": forward-mode differentiation is not implemented");
}
void no_tangent(const char* op, const OptTensor& t) {
  if (t.has_value()) no_tangent(op, *t);
}
template <typename... Inputs>
void no_tangents(const char* op, const Inputs&... inputs) {
  (no_tangent(op, inputs), ...);
}

// Results of a backward pass that cannot be differentiated again: doing so raises, but only when it is done.  They depend on the incoming
// gradient, the weights and (through the kept values) on every input, so all are marked whichever of these require gradients.
void once_only(const char* name, variable_list& out) {
  if (!at::GradMode::is_enabled()) return;       // without create_graph nothing is differentiated again
  variable_list some;
  for (const Tensor& t : out)
    if (t.defined()) some.push_back(t.detach().set_requires_grad(true));       // (the node's results require gradients where its inputs do)
  if (some.empty()) return;
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " cannot be differentiated twice", static_cast<int64_t>(some.size()));
  variable_list marked = (*node)(std::move(some));
  size_t i = 0;
  for (Tensor& t : out)
    if (t.defined()) t = marked[i++];
}

using FfnSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, c10::string_view, bool);
using FfnKeepSig = Five(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, c10::string_view, bool);
using FfnBackSig = Five(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, c10::string_view,
                        std::array<bool, 5>);

struct GatedFfn : torch::autograd::Function<GatedFfn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w1, const Tensor& w2, const OptTensor& b1, const OptTensor& b2,
                        const OptTensor& r, const std::string& act, bool int8) {
    static const auto op = handle<FfnKeepSig>("npu::npu_gated_ffn_keep");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, kept, scale, x_q, x_scale] = op.call(x, w1, w2, b1, b2, r, act, int8);
    ctx->save_for_backward({int8 ? x_q : x, x_scale, w1, w2, kept, scale});
    ctx->saved_data["act"] = act;
    ctx->saved_data["b1"] = b1.has_value();
    ctx->saved_data["b2"] = b2.has_value();
    ctx->saved_data["r"] = r.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto op = handle<FfnBackSig>("npu::npu_gated_ffn_backward");
    const variable_list s = ctx->get_saved_variables();
    // edges exist for the tensors that were given, in their order
    size_t edge = 3;
    std::array<bool, 5> want = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), false, false};
    if (ctx->saved_data["b1"].toBool()) want[3] = ctx->needs_input_grad(edge++);
    if (ctx->saved_data["b2"].toBool()) want[4] = ctx->needs_input_grad(edge++);
    const bool want_r = ctx->saved_data["r"].toBool() && ctx->needs_input_grad(edge);
    const std::string act = ctx->saved_data["act"].toStringRef();
    variable_list out(8);
    if (!grads[0].defined()) return out;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dx, dw1, dw2, db1, db2] = op.call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], act, want);
      if (want[0]) out[0] = dx;
      if (want[1]) out[1] = dw1;
      if (want[2]) out[2] = dw2;
      if (want[3]) out[3] = db1;
      if (want[4]) out[4] = db2;
    }
    once_only("npu_gated_ffn", out);
    if (want_r) out[5] = grads[0];
    return out;
  }
};

Tensor ffn_autograd(const Tensor& x, const Tensor& w1, const Tensor& w2, const OptTensor& b1, const OptTensor& b2, const OptTensor& r,
                    c10::string_view act, bool int8) {
  no_tangents("npu_gated_ffn", x, w1, w2, b1, b2, r);
  if (at::GradMode::is_enabled() && (wants(x) || wants(w1) || wants(w2) || wants(b1) || wants(b2) || wants(r)))
    return GatedFfn::apply(x, w1, w2, b1, b2, r, std::string(act), int8);
  static const auto op = handle<FfnSig>("npu::npu_gated_ffn");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, w1, w2, b1, b2, r, act, int8);
}

using LinearSig = Tensor(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, c10::string_view, bool);
using LinearKeepSig = Five(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, c10::string_view, bool);
using LinearBackSig = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                         c10::string_view, std::array<bool, 3>);

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r, const std::string& act, bool int8) {
    static const auto op = handle<LinearKeepSig>("npu::npu_linear_act_keep");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, kept, scale, x_q, x_scale] = op.call(x, w, b, r, act, int8);
    ctx->save_for_backward({int8 ? x_q : x, x_scale, w, kept, scale});
    ctx->saved_data["act"] = act;
    ctx->saved_data["b"] = b.has_value();
    ctx->saved_data["r"] = r.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto op = handle<LinearBackSig>("npu::npu_linear_act_backward");
    const variable_list s = ctx->get_saved_variables();
    size_t edge = 2;
    std::array<bool, 3> want = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), false};
    if (ctx->saved_data["b"].toBool()) want[2] = ctx->needs_input_grad(edge++);
    const bool want_r = ctx->saved_data["r"].toBool() && ctx->needs_input_grad(edge);
    const std::string act = ctx->saved_data["act"].toStringRef();
    variable_list out(6);
    if (!grads[0].defined()) return out;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dx, dw, db] = op.call(grads[0], s[0], s[1], s[2], s[3], s[4], act, want);
      if (want[0]) out[0] = dx;
      if (want[1]) out[1] = dw;
      if (want[2]) out[2] = db;
    }
    once_only("npu_linear_act", out);
    if (want_r) out[3] = grads[0];
    return out;
  }
};

Tensor linear_autograd(const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r, c10::string_view act, bool int8) {
  no_tangents("npu_linear_act", x, w, b, r);
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r))) return LinearAct::apply(x, w, b, r, std::string(act), int8);
  static const auto op = handle<LinearSig>("npu::npu_linear_act");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, w, b, r, act, int8);
}

}  // namespace

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
  m.impl("npu_gated_ffn", TORCH_FN(ffn_cuda));
  m.impl("npu_gated_ffn_keep", TORCH_FN(ffn_keep_cuda));
  m.impl("npu_gated_ffn_backward", TORCH_FN(ffn_backward_cuda));
  m.impl("npu_linear_act", TORCH_FN(linear_cuda));
  m.impl("npu_linear_act_keep", TORCH_FN(linear_keep_cuda));
  m.impl("npu_linear_act_backward", TORCH_FN(linear_backward_cuda));
  m.impl("npu_checkpoint_quant", TORCH_FN(ck_quant_cuda));
  m.impl("npu_checkpoint_dequant", TORCH_FN(ck_dequant_cuda));
  m.impl("npu_checkpoint_weight_grad", TORCH_FN(ck_weight_grad_cuda));
}

TORCH_LIBRARY_IMPL(npu, AutogradCUDA, m) {
  m.impl("npu_gated_ffn", TORCH_FN(ffn_autograd));
  m.impl("npu_linear_act", TORCH_FN(linear_autograd));
  // not differentiable: a gradient or a tangent that is asked for raises
  for (const char* op : {"npu_gated_ffn_keep", "npu_gated_ffn_backward", "npu_linear_act_keep", "npu_linear_act_backward", "npu_checkpoint_quant",
                         "npu_checkpoint_dequant", "npu_checkpoint_weight_grad"})
    m.impl(op, torch::autograd::autogradNotImplementedFallback());
}

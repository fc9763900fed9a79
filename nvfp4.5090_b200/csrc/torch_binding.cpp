// Torch bindings of the MXFP4, clipping and sandwich-norm entry points: checks
// of arguments, allocation and the current stream, in C++ because a call's
// host time is what its smallest users wait for (a decoded token, a small
// layer): sandwich_norm 20 us through ctypes and the Python allocator calls,
// 9 us here.  ops.py documents every function; the work is the C ABI's.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/nvfp4_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check(int rc, const char* name) {
  TORCH_CHECK(rc == 0, name, " failed: ", nvfp4b200_status_string(rc), " (status ", rc, ")");
}

// The tensor's device made current, and its current stream.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

// bf16, f32, f16 as the C ABI numbers them; -1 for any other type.
int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return NVFP4B200_BF16;
    case at::kFloat: return NVFP4B200_F32;
    case at::kHalf: return NVFP4B200_F16;
    default: return -1;
  }
}

void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
bool on(const Tensor& t, const Tensor& like) { return t.is_cuda() && t.get_device() == like.get_device(); }
// Counts a write into a caller's tensor, so that autograd refuses a backward that saved it before.
void wrote(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t scale_rows(int64_t rows) { return up(rows, 128); }
int64_t scale_cols(int64_t k) { return up(k / 32, 4); }
int64_t scale_bytes(int64_t rows, int64_t k) { return scale_rows(rows) * scale_cols(k); }
int64_t operand_bytes(int64_t rows, int64_t k) { return rows * k / 2 + scale_bytes(rows, k); }

Tensor bytes(const Tensor& like, c10::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kByte)); }
Tensor floats(const Tensor& like, c10::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }

// Contiguous, on a 16-byte boundary (a slice of a flat parameter buffer may start anywhere): copied otherwise.
Tensor vector_of(const Tensor& t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

// ---- MXFP4 -----------------------------------------------------------------

// x as the quantizers read it: 2-D, unit column stride, 16-byte aligned rows;
// copied when it is laid out otherwise.
Tensor float_matrix(const Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && code_of(x) >= 0,
              "MXFP4 quantizers expect a 2-D CUDA bf16, fp16 or fp32 tensor");
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && x.stride(1) == 1 && x.stride(0) >= x.size(1) &&
      x.stride(0) % 8 == 0)
    return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

using Pair = std::pair<Tensor, Tensor>;

// (q, s) of an operand of `rows` rows along k: new, or the caller's, checked.
Pair operand(const Tensor& like, int64_t rows, int64_t k, const std::optional<Pair>& out) {
  if (!out) return {bytes(like, {rows, k / 2}), bytes(like, {scale_rows(rows), scale_cols(k)})};
  auto good = [&](const Tensor& t, int64_t a, int64_t b) {
    return on(t, like) && t.scalar_type() == at::kByte && t.is_contiguous() && t.dim() == 2 && t.size(0) == a &&
           t.size(1) == b;
  };
  TORCH_CHECK(good(out->first, rows, k / 2) && good(out->second, scale_rows(rows), scale_cols(k)),
              "out must be contiguous uint8 (q [", rows, ", ", k / 2, "], s [", scale_rows(rows), ", ", scale_cols(k),
              "]) on the input's device");
  return *out;
}

void quantize_into(const Tensor& x, const OptTensor& row, const OptTensor& gamma, void* q, void* s, void* qt, void* st,
                   void* stream) {
  if (x.size(0) == 0) return;
  check(nvfp4b200_mx_quant(x.data_ptr(), code_of(x), static_cast<float*>(ptr(row)), ptr(gamma), q, s, qt, st, x.size(0),
                           x.size(1), std::max(x.stride(0), x.size(1)), stream),
        "nvfp4b200_mx_quant");
}

std::pair<Pair, Pair> quantize(const Tensor& x_, const OptTensor& row_, const OptTensor& gamma_, bool rows, bool cols,
                               const std::optional<Pair>& out) {
  const Tensor x = float_matrix(x_);
  const int64_t r = x.size(0), c = x.size(1);
  TORCH_CHECK(!rows || c % 32 == 0, "K must be divisible by 32 for MXFP4 1x32 scaling.");
  TORCH_CHECK(c > 0 && c % 8 == 0, "MXFP4 quantizers need columns divisible by 8");
  OptTensor row, gamma;
  if (row_) {
    TORCH_CHECK(on(*row_, x) && row_->scalar_type() == at::kFloat && row_->numel() == r,
                "row_scale is float32 [R] on the input's device");
    row = row_->contiguous();
  }
  if (gamma_) {
    TORCH_CHECK(on(*gamma_, x) && gamma_->scalar_type() == at::kBFloat16 && gamma_->numel() == c,
                "gamma is bf16 [K] on the input's device");
    gamma = vector_of(*gamma_);
  }
  On at_(x);
  Pair a, b;
  if (rows) a = operand(x, r, c, out);
  if (cols) b = operand(x, c, up(r, 32), rows ? std::nullopt : out);
  quantize_into(x, row, gamma, rows ? a.first.data_ptr() : nullptr, rows ? a.second.data_ptr() : nullptr,
                cols ? b.first.data_ptr() : nullptr, cols ? b.second.data_ptr() : nullptr, at_.stream);
  if (out) {
    wrote(out->first);
    wrote(out->second);
  }
  return {a, b};
}

Pair mx_quantize(const Tensor& x, const OptTensor& row, const OptTensor& gamma, const std::optional<Pair>& out) {
  return quantize(x, row, gamma, true, false, out).first;
}
Pair mx_quantize_t(const Tensor& x, const OptTensor& row, const OptTensor& gamma, const std::optional<Pair>& out) {
  return quantize(x, row, gamma, false, true, out).second;
}
std::tuple<Tensor, Tensor, Tensor, Tensor> mx_quantize_both(const Tensor& x, const OptTensor& row, const OptTensor& gamma) {
  auto p = quantize(x, row, gamma, true, true, std::nullopt);
  return {p.first.first, p.first.second, p.second.first, p.second.second};
}

Tensor mx_dequantize(const Tensor& q_, const Tensor& s_, bool f32) {
  TORCH_CHECK(q_.is_cuda() && q_.element_size() == 1 && q_.dim() == 2, "mx_dequantize expects packed bytes [R, K/2]");
  const int64_t r = q_.size(0), k = 2 * q_.size(1);
  TORCH_CHECK(k % 32 == 0, "K must be divisible by 32 for MXFP4 1x32 scaling.");
  TORCH_CHECK(on(s_, q_) && s_.element_size() == 1 && s_.numel() == scale_bytes(r, k),
              "MXFP4 scale tensors must be the padded swizzled [round_up(rows,128), round_up(k/32,4)] layout");
  On at_(q_);
  const Tensor q = q_.contiguous(), s = s_.contiguous();
  Tensor y = at::empty({r, k}, q.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  if (r && k)
    check(nvfp4b200_mx_dequant(q.data_ptr(), s.data_ptr(), y.data_ptr(), f32 ? NVFP4B200_F32 : NVFP4B200_BF16, r, k,
                               at_.stream),
          "nvfp4b200_mx_dequant");
  return y;
}

OptTensor bias_of(const OptTensor& bias, int64_t n, const Tensor& like) {
  if (!bias) return std::nullopt;
  TORCH_CHECK(on(*bias, like) && bias->scalar_type() == at::kBFloat16 && bias->numel() == n,
              "bias is a CUDA BF16 tensor [n] on the operands' device");
  return vector_of(*bias);
}

Tensor mx_gemm(const Tensor& qa, const Tensor& sa, const Tensor& qb, const Tensor& sb, const OptTensor& bias_,
               const OptTensor& residual, const OptTensor& out_, bool f32, bool accumulate, int epilogue) {
  TORCH_CHECK(qa.is_cuda() && on(sa, qa) && on(qb, qa) && on(sb, qa), "mx_gemm requires CUDA tensors of one device");
  TORCH_CHECK(qa.element_size() == 1 && qb.element_size() == 1 && sa.element_size() == 1 && sb.element_size() == 1 &&
                  qa.dim() == 2 && qb.dim() == 2,
              "mx_gemm expects packed bytes [rows, k/2] and one-byte scales");
  const int64_t m = qa.size(0), n = qb.size(0), k = 2 * qa.size(1);
  TORCH_CHECK(qb.size(1) * 2 == k, "K mismatch: A has ", k, ", B has ", 2 * qb.size(1));
  TORCH_CHECK(k > 0 && k % 32 == 0, "K must be divisible by 32 for MXFP4 1x32 scaling.");
  TORCH_CHECK(qa.is_contiguous() && qb.is_contiguous() && sa.is_contiguous() && sb.is_contiguous(),
              "gemm operands must be contiguous");
  TORCH_CHECK(sa.numel() == scale_bytes(m, k) && sb.numel() == scale_bytes(n, k),
              "MXFP4 scale tensors must be the padded swizzled [round_up(rows,128), round_up(k/32,4)] layout");
  On at_(qa);
  Tensor out;
  if (out_) {
    out = *out_;
    TORCH_CHECK(on(out, qa) && (out.scalar_type() == at::kBFloat16 || out.scalar_type() == at::kFloat),
                "output must be bf16 or fp32 on the operands' device");
    TORCH_CHECK(out.dim() == 2 && out.size(0) == m && out.size(1) == n && out.stride(1) == 1,
                "output must be [m, n] with unit column stride");
    TORCH_CHECK(!accumulate || out.scalar_type() == at::kFloat, "accumulate needs an fp32 output");
  } else {
    TORCH_CHECK(!accumulate, "accumulate needs an existing output");
    out = at::empty({m, n}, qa.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  }
  const OptTensor bias = bias_of(bias_, n, qa);
  if (residual)
    TORCH_CHECK(on(*residual, qa) && residual->scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16 &&
                    residual->sizes() == out.sizes() && residual->strides() == out.strides(),
                "residual must be bf16 and match a bf16 output's layout");
  if (m && n)
    check(nvfp4b200_mx_gemm(qa.data_ptr(), qb.data_ptr(), sa.data_ptr(), sb.data_ptr(), ptr(bias), ptr(residual),
                            out.data_ptr(), out.scalar_type() == at::kFloat ? NVFP4B200_F32 : NVFP4B200_BF16,
                            accumulate, epilogue, m, n, k, out.stride(0), at_.stream),
          "nvfp4b200_mx_gemm");
  if (out_) wrote(out);
  return out;
}

Tensor mx_linear(const Tensor& x, const Tensor& qw, const Tensor& sw, const OptTensor& bias_) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() >= 1, "mx_linear expects a CUDA BF16 tensor.");
  TORCH_CHECK(on(qw, x) && on(sw, x) && qw.dim() == 2 && qw.element_size() == 1 && sw.element_size() == 1 &&
                  qw.is_contiguous() && sw.is_contiguous(),
              "the weight is contiguous packed bytes [n, k/2] and one-byte scales on x's device");
  const int64_t n = qw.size(0), k = 2 * qw.size(1);
  TORCH_CHECK(x.size(-1) == k, "K mismatch: x has ", x.size(-1), ", W has ", k);
  TORCH_CHECK(k > 0 && k % 32 == 0 && n % 8 == 0, "mx_linear needs K divisible by 32 and N by 8");
  TORCH_CHECK(sw.numel() == scale_bytes(n, k),
              "MXFP4 scale tensors must be the padded swizzled [round_up(rows,128), round_up(k/32,4)] layout");
  const OptTensor bias = bias_of(bias_, n, x);
  On at_(x);
  const Tensor x2 = float_matrix(x.dim() == 2 ? x : x.reshape({-1, k}));
  const int64_t m = x2.size(0);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  Tensor y = at::empty(shape, x.options());
  if (m && n) {
    Tensor ws;   // the quantized tokens, where the product does not quantize them itself
    uint8_t* q = nullptr;
    if (!nvfp4b200_mx_linear_fused(m, n, k)) {
      ws = bytes(x, {operand_bytes(m, k)});
      q = ws.data_ptr<uint8_t>();
    }
    check(nvfp4b200_mx_linear(x2.data_ptr(), qw.data_ptr(), sw.data_ptr(), ptr(bias), q, q ? q + m * k / 2 : nullptr,
                              y.data_ptr(), m, n, k, std::max(x2.stride(0), k), at_.stream),
          "nvfp4b200_mx_linear");
  }
  return y;
}

// One orientation of a matrix in one buffer: nibbles, then scales (k % 32 == 0:
// the nibbles end on a 16-byte boundary).
struct Held {
  uint8_t* q = nullptr;
  uint8_t* s = nullptr;
  Held() = default;
  Held(uint8_t* p, int64_t rows, int64_t k) : q(p), s(p + rows * k / 2) {}
};

void product(Held a, Held b, const Tensor& out, const OptTensor& bias, int64_t m, int64_t n, int64_t k, void* stream) {
  if (m && n)
    check(nvfp4b200_mx_gemm(a.q, b.q, a.s, b.s, ptr(bias), nullptr, out.data_ptr(), code_of(out), 0, NVFP4B200_EPI_NONE,
                            m, n, k, n, stream),
          "nvfp4b200_mx_gemm");
}

// Forward of the trained layer: y, and the transposed operands that the
// backward multiplies with (of x for the weight's gradient, of w for x's).
std::tuple<Tensor, OptTensor, OptTensor> linear_forward(const Tensor& x_, const Tensor& w_, const OptTensor& bias_,
                                                        bool need_x, bool need_w) {
  TORCH_CHECK(x_.is_cuda() && (x_.scalar_type() == at::kBFloat16 || x_.scalar_type() == at::kFloat) && x_.dim() >= 1,
              "mxfp4_linear expects a CUDA bf16 or fp32 input.");
  TORCH_CHECK(on(w_, x_) && w_.dim() == 2 && code_of(w_) >= 0,
              "mxfp4_linear expects a 2-D bf16, fp16 or fp32 weight on the input's device");
  const int64_t n = w_.size(0), k = w_.size(1);
  TORCH_CHECK(x_.size(-1) == k, "K mismatch: input has ", x_.size(-1), ", weight has ", k);
  TORCH_CHECK(k > 0 && k % 32 == 0, "K must be divisible by 32 for MXFP4 1x32 scaling.");
  TORCH_CHECK(n % 8 == 0, "out_features must be divisible by 8");
  TORCH_CHECK(!(need_x || need_w) || n % 32 == 0, "training needs out_features divisible by 32");
  OptTensor bias;
  if (bias_) {
    TORCH_CHECK(on(*bias_, x_) && bias_->numel() == n, "bias is a tensor [N] on the input's device");
    bias = vector_of(bias_->to(at::kBFloat16));   // the type in which the product's epilogue reads it
  }
  On at_(x_);
  const Tensor x = float_matrix(x_.dim() == 2 ? x_ : x_.reshape({-1, k})), w = float_matrix(w_);
  const int64_t t = x.size(0), tp = up(t, 32);
  std::vector<int64_t> shape = x_.sizes().vec();
  shape.back() = n;
  Tensor y = at::empty(shape, x.options());
  OptTensor xt, wt;
  if (need_w) xt = bytes(x, {operand_bytes(k, tp)});
  if (need_x) wt = bytes(x, {operand_bytes(k, n)});
  Tensor ws = bytes(x, {operand_bytes(t, k) + operand_bytes(n, k)});
  const Held a(ws.data_ptr<uint8_t>(), t, k), b(ws.data_ptr<uint8_t>() + operand_bytes(t, k), n, k);
  const Held at = xt ? Held(xt->data_ptr<uint8_t>(), k, tp) : Held(), bt = wt ? Held(wt->data_ptr<uint8_t>(), k, n) : Held();
  if (t && n) {
    quantize_into(x, std::nullopt, std::nullopt, a.q, a.s, at.q, at.s, at_.stream);
    quantize_into(w, std::nullopt, std::nullopt, b.q, b.s, bt.q, bt.s, at_.stream);
    product(a, b, y, bias, t, n, k, at_.stream);
  }
  return {y, xt, wt};
}

int64_t tokens(const std::vector<int64_t>& x_shape) {
  int64_t t = 1;
  for (size_t i = 0; i + 1 < x_shape.size(); ++i) t *= x_shape[i];
  return t;
}

// Its backward: dx in x's shape and dy's type, dw fp32 or bf16.
std::tuple<OptTensor, OptTensor> linear_backward(const Tensor& dy_, const OptTensor& xt, const OptTensor& wt,
                                                 const std::vector<int64_t>& x_shape, int64_t n, bool need_x, bool need_w,
                                                 bool dw_f32) {
  TORCH_CHECK(dy_.is_cuda() && (dy_.scalar_type() == at::kBFloat16 || dy_.scalar_type() == at::kFloat),
              "mxfp4_linear's gradient must be bf16 or fp32");
  const int64_t k = x_shape.back();
  On at_(dy_);
  const Tensor dy = float_matrix(dy_.dim() == 2 ? dy_ : dy_.reshape({tokens(x_shape), n}));
  const int64_t t = dy.size(0), tp = up(t, 32);
  TORCH_CHECK((!need_x || (wt && on(*wt, dy) && wt->numel() == operand_bytes(k, n))) &&
                  (!need_w || (xt && on(*xt, dy) && xt->numel() == operand_bytes(k, tp))),
              "the gradient does not belong to the operands that the forward kept");
  OptTensor dx, dw;
  if (need_x) dx = at::empty(x_shape, dy.options());
  if (need_w) dw = at::empty({n, k}, dy.options().dtype(dw_f32 ? at::kFloat : at::kBFloat16));
  if (t == 0 || n == 0) {
    if (dw) dw->zero_();
    if (dx) dx->zero_();
    return {dx, dw};
  }
  const int64_t rows = need_x ? operand_bytes(t, n) : 0, cols = need_w ? operand_bytes(n, tp) : 0;
  Tensor ws = bytes(dy, {rows + cols});
  const Held d = need_x ? Held(ws.data_ptr<uint8_t>(), t, n) : Held();
  const Held dt = need_w ? Held(ws.data_ptr<uint8_t>() + rows, n, tp) : Held();
  quantize_into(dy, std::nullopt, std::nullopt, d.q, d.s, dt.q, dt.s, at_.stream);
  if (need_x) product(d, Held(wt->data_ptr<uint8_t>(), k, n), *dx, std::nullopt, t, k, n, at_.stream);
  if (need_w) product(dt, Held(xt->data_ptr<uint8_t>(), k, tp), *dw, std::nullopt, n, k, tp, at_.stream);
  return {dx, dw};
}

// The differentiable layer.  Quantization counts as the identity in the
// backward; both orientations of an operand come from one read of it, and what
// the backward needs of x and w is kept in MXFP4 (17/32 byte per element).  In
// C++ so that the backward needs neither Python nor its lock (a training step
// of 777 tokens through 1024 x 2048: 95 us with a Python function, 84 so).
struct MXLinear : public torch::autograd::Function<MXLinear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias,
                        bool need_x, bool need_w) {
    auto [y, xt, wt] = linear_forward(x, w, bias, need_x, need_w);
    ctx->save_for_backward({xt.value_or(Tensor()), wt.value_or(Tensor())});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["n"] = w.size(0);
    ctx->saved_data["w"] = (int64_t)w.scalar_type();
    ctx->saved_data["b"] = bias ? (int64_t)bias->scalar_type() : (int64_t)-1;
    ctx->saved_data["need"] = (int64_t)(need_x + 2 * need_w);
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    // its gradients are no functions that autograd could differentiate
    TORCH_CHECK(!at::GradMode::is_enabled(), "mxfp4_linear has no second derivative (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t n = ctx->saved_data["n"].toInt(), need = ctx->saved_data["need"].toInt(), b = ctx->saved_data["b"].toInt();
    const auto wtype = (at::ScalarType)ctx->saved_data["w"].toInt();
    const Tensor& dy = grads[0];
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    torch::autograd::variable_list out(5);
    if (!dy.defined()) return out;
    if (need) {
      auto [dx, dw] = linear_backward(dy, opt(saved[0]), opt(saved[1]), shape, n, need & 1, need & 2, wtype != at::kBFloat16);
      if (dx) out[0] = *dx;
      if (dw) out[1] = dw->scalar_type() == wtype ? *dw : dw->to(wtype);   // fp16: from fp32, one rounding
    }
    if (b >= 0 && ctx->needs_input_grad(2))
      out[2] = dy.reshape({tokens(shape), n}).sum(at::IntArrayRef{0}, false, at::kFloat).to((at::ScalarType)b);
    return out;
  }
};

Tensor mxfp4_linear(const Tensor& x, const Tensor& w, const OptTensor& bias) {
  const bool grad = at::GradMode::is_enabled();
  return MXLinear::apply(x, w, bias, grad && x.requires_grad(), grad && w.requires_grad());
}

// ---- gradient norm and clipping ---------------------------------------------

// which: bit 0 the norm, 1 the coefficient, 2 the fp64 total.  `outs`: the
// gradients themselves where in_place.
std::tuple<OptTensor, OptTensor, OptTensor> grad_norm(const std::vector<Tensor>& grads,
                                                      const std::optional<std::vector<Tensor>>& outs, bool in_place,
                                                      double norm_type, double grad_scale, double max_norm, int which) {
  TORCH_CHECK(norm_type == 2.0 || norm_type == INFINITY, "norm_type must be 2 or inf");
  TORCH_CHECK(max_norm >= 0.0, "max_norm must not be negative");
  const size_t count = grads.size();
  const at::Device dev =
      count ? grads[0].device() : at::Device(at::kCUDA, c10::cuda::current_device());
  TORCH_CHECK(dev.is_cuda(), "gradients are bf16, fp16 or fp32 CUDA tensors of one device");
  std::vector<const void*> src(count);
  std::vector<void*> dst(count);
  std::vector<int> src_dt(count), dst_dt(count);
  std::vector<int64_t> numel(count);
  for (size_t i = 0; i < count; ++i) {
    const Tensor& t = grads[i];
    src_dt[i] = code_of(t);
    TORCH_CHECK(src_dt[i] >= 0 && t.device() == dev, "gradients are bf16, fp16 or fp32 CUDA tensors of one device");
    TORCH_CHECK(t.is_contiguous() || t.is_non_overlapping_and_dense(),
                "gradients must be dense: every element once in one stretch of memory");
    src[i] = t.data_ptr();
    numel[i] = t.numel();
  }
  const bool write = in_place || outs;
  if (outs) {
    TORCH_CHECK(outs->size() == count, "out must hold one tensor per gradient");
    for (size_t i = 0; i < count; ++i) {
      const Tensor &o = (*outs)[i], &t = grads[i];
      dst_dt[i] = code_of(o);
      TORCH_CHECK(dst_dt[i] >= 0 && o.device() == dev && o.numel() == numel[i] &&
                      ((o.is_contiguous() && t.is_contiguous()) || (o.sizes() == t.sizes() && o.strides() == t.strides())),
                  "out holds one bf16, fp16 or fp32 tensor per gradient, contiguous and of its number of elements, or of "
                  "its shape and strides");
      dst[i] = o.data_ptr();
    }
  } else if (in_place) {
    for (size_t i = 0; i < count; ++i) {
      dst[i] = const_cast<void*>(src[i]);
      dst_dt[i] = src_dt[i];
    }
  }
  c10::cuda::CUDAGuard guard(dev);
  const auto opt = at::TensorOptions().device(dev);
  const int64_t words = NVFP4B200_GRAD_WS_DOUBLES(count);
  Tensor ws = at::empty({words}, opt.dtype(at::kDouble));
  OptTensor norm, coef, total;
  if (which & 1) norm = at::empty({1}, opt.dtype(at::kFloat));
  if (which & 2) coef = at::empty({1}, opt.dtype(at::kFloat));
  if (which & 4) total = at::empty({1}, opt.dtype(at::kDouble));
  check(nvfp4b200_grad_norm(src.data(), src_dt.data(), write ? dst.data() : nullptr, write ? dst_dt.data() : nullptr,
                            numel.data(), (int)count, norm_type == 2.0 ? 2 : 0, (float)grad_scale, (float)max_norm,
                            ws.data_ptr<double>(), words, static_cast<float*>(ptr(norm)), static_cast<float*>(ptr(coef)),
                            static_cast<double*>(ptr(total)), c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
        "nvfp4b200_grad_norm");
  if (write)
    for (const Tensor& t : in_place ? grads : *outs) wrote(t);
  return {norm, coef, total};
}

std::pair<Tensor, Tensor> grad_norm_finish(const Tensor& totals, double norm_type, double grad_scale, double max_norm) {
  TORCH_CHECK(totals.is_cuda() && totals.scalar_type() == at::kDouble && totals.is_contiguous(),
              "totals are a contiguous float64 CUDA tensor");
  TORCH_CHECK(norm_type == 2.0 || norm_type == INFINITY, "norm_type must be 2 or inf");
  TORCH_CHECK(max_norm >= 0.0, "max_norm must not be negative");
  On at_(totals);
  Tensor norm = floats(totals, {1}), coef = floats(totals, {1});
  check(nvfp4b200_grad_norm_finish(totals.data_ptr<double>(), totals.numel(), norm_type == 2.0 ? 2 : 0, (float)grad_scale,
                                   (float)max_norm, norm.data_ptr<float>(), coef.data_ptr<float>(), at_.stream),
        "nvfp4b200_grad_norm_finish");
  return {norm, coef};
}

// ---- sandwich norm ------------------------------------------------------------

void norm_input(const Tensor& b) {
  TORCH_CHECK(b.is_cuda() && code_of(b) >= 0 && b.dim() == 2, "the norms expect CUDA bf16, fp16 or fp32 [T, D]");
  TORCH_CHECK(b.size(1) > 0 && b.size(1) <= 16384, "the norms take 1 to 16384 columns");
}

bool matches(const Tensor& t, const Tensor& b) {
  return on(t, b) && t.scalar_type() == b.scalar_type() && t.sizes() == b.sizes();
}

// Unit column stride (rows may be strided), copied otherwise.
Tensor rows_of(const Tensor& t) {
  if (t.is_contiguous() || (t.stride(1) == 1 && t.stride(0) >= t.size(1))) return t;
  return t.contiguous();
}
int64_t ld(const OptTensor& t) { return t ? std::max(t->stride(0), t->size(1)) : 0; }

OptTensor weight(const OptTensor& w, const Tensor& b) {
  if (!w) return std::nullopt;
  TORCH_CHECK(on(*w, b) && w->scalar_type() == b.scalar_type() && w->numel() == b.size(1),
              "gamma_post and gamma_pre must be [D] of the activations' dtype and device");
  return w->contiguous();
}

// The gate, contiguous, and its number of groups (0 without one).
OptTensor gate_of(const OptTensor& g, const Tensor& b, int64_t& groups) {
  groups = 0;
  if (!g) return std::nullopt;
  TORCH_CHECK(on(*g, b) && g->scalar_type() == b.scalar_type() && g->dim() >= 1 && g->size(-1) == b.size(1),
              "gate must be [D] or [G, D] of the activations' dtype and device");
  groups = g->numel() / b.size(1);
  TORCH_CHECK(groups > 0 && b.size(0) % groups == 0, "the rows must split evenly over the gate's groups");
  return g->contiguous();
}

std::tuple<Tensor, OptTensor, Tensor, OptTensor> sandwich_norm(const Tensor& b_, const Tensor& x_, const OptTensor& gp_,
                                                               const OptTensor& gate_, const OptTensor& gn_,
                                                               double residual_scale, double branch_scale, double eps,
                                                               std::optional<bool> pre_) {
  norm_input(b_);
  TORCH_CHECK(matches(x_, b_), "b and x must match in shape, dtype and device");
  int64_t groups;
  const OptTensor gp = weight(gp_, b_), gn = weight(gn_, b_), gate = gate_of(gate_, b_, groups);
  const bool pre = pre_.value_or(gn.has_value());
  TORCH_CHECK(pre || !gn, "gamma_pre without the norm it belongs to");
  On at_(b_);
  const Tensor b = rows_of(b_), x = rows_of(x_);
  const int64_t t = b.size(0), d = b.size(1);
  Tensor y = at::empty({t, d}, b.options()), inv_b = floats(b, {t});
  OptTensor n, inv_y;
  if (pre) {
    n = at::empty({t, d}, b.options());
    inv_y = floats(b, {t});
  }
  if (t)
    check(nvfp4b200_sandwich_norm(b.data_ptr(), x.data_ptr(), ptr(gp), ptr(gate), ptr(gn), y.data_ptr(), ptr(n),
                                  inv_b.data_ptr<float>(), static_cast<float*>(ptr(inv_y)), code_of(b), t, d, groups,
                                  ld(b), ld(x), (float)residual_scale, (float)branch_scale, (float)eps, at_.stream),
          "nvfp4b200_sandwich_norm");
  return {y, n, inv_b, inv_y};
}

// dx, db, dgamma_post, dgate, dgamma_pre
std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor> sandwich_norm_bwd(
    const OptTensor& dy_, const Tensor& b_, const Tensor& inv_b, const OptTensor& gp_, const OptTensor& gate_,
    const OptTensor& dn_, const OptTensor& y_, const OptTensor& inv_y, const OptTensor& gn_, double residual_scale,
    double branch_scale) {
  TORCH_CHECK(dy_ || dn_, "sandwich_norm_bwd needs dy or dn");
  norm_input(b_);
  TORCH_CHECK(dn_.has_value() == y_.has_value() && dn_.has_value() == inv_y.has_value(), "dn comes with y and inv_y");
  TORCH_CHECK(dn_ || !gn_, "gamma_pre without the norm it belongs to");
  for (const OptTensor* t : {&dy_, &dn_, &y_})
    TORCH_CHECK(!*t || matches(**t, b_), "dy, dn and y must match b in shape, dtype and device");
  const int64_t t = b_.size(0), d = b_.size(1);
  auto stat = [&](const Tensor& v) {
    return on(v, b_) && v.scalar_type() == at::kFloat && v.numel() == t && v.is_contiguous();
  };
  TORCH_CHECK(stat(inv_b) && (!inv_y || stat(*inv_y)), "inv_b and inv_y are contiguous float32 [T]");
  int64_t groups;
  const OptTensor gp = weight(gp_, b_), gn = weight(gn_, b_), gate = gate_of(gate_, b_, groups);
  On at_(b_);
  const Tensor b = rows_of(b_);
  OptTensor dy, dn, y;
  if (dy_) dy = rows_of(*dy_);
  if (dn_) dn = rows_of(*dn_);
  if (y_) y = rows_of(*y_);
  Tensor dx = at::empty({t, d}, b.options()), db = at::empty({t, d}, b.options()), dpost = floats(b, {d});
  OptTensor dgate, dpre;
  if (groups) dgate = floats(b, {groups, d});
  if (dn) dpre = floats(b, {d});
  if (t == 0) {
    dpost.zero_();
    if (dgate) dgate->zero_();
    if (dpre) dpre->zero_();
    return {dx, db, dpost, dgate, dpre};
  }
  int64_t words = 0;
  check(nvfp4b200_sandwich_norm_bwd_ws(t, d, groups, &words), "nvfp4b200_sandwich_norm_bwd_ws");
  Tensor ws = floats(b, {words});
  check(nvfp4b200_sandwich_norm_bwd(ptr(dy), ptr(dn), b.data_ptr(), ptr(y), inv_b.data_ptr<float>(),
                                    static_cast<float*>(ptr(inv_y)), ptr(gp), ptr(gate), ptr(gn), dx.data_ptr(),
                                    db.data_ptr(), dpost.data_ptr<float>(), static_cast<float*>(ptr(dgate)),
                                    static_cast<float*>(ptr(dpre)), ws.data_ptr<float>(), words, code_of(b), t, d, groups,
                                    ld(dy), ld(dn), ld(b), ld(y), (float)residual_scale, (float)branch_scale, at_.stream),
        "nvfp4b200_sandwich_norm_bwd");
  return {dx, db, dpost, dgate, dpre};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("mx_quantize", &mx_quantize);
  m.def("mx_quantize_t", &mx_quantize_t);
  m.def("mx_quantize_both", &mx_quantize_both);
  m.def("mx_dequantize", &mx_dequantize);
  m.def("mx_gemm", &mx_gemm);
  m.def("mx_linear", &mx_linear);
  m.def("mxfp4_linear", &mxfp4_linear);
  m.def("grad_norm", &grad_norm);
  m.def("grad_norm_finish", &grad_norm_finish);
  m.def("sandwich_norm", &sandwich_norm);
  m.def("sandwich_norm_bwd", &sandwich_norm_bwd);
}

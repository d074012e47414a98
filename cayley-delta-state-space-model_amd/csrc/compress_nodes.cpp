// The host side of the operators around a smaller model (top logits, distillation, products with 4-bit weights) in C++: the
// loss with its autograd node, for the reasons that train_nodes.cpp gives, and the decode product, whose kernel takes as long as
// a call through ctypes does.
#include <ATen/ops/full.h>
#include <ATen/ops/zeros.h>

#include "nodes_common.hpp"

namespace {

struct Entries {
  decltype(&cdssm_top_logits) top;
  decltype(&cdssm_distillation_workspace_bytes) distill_bytes;
  decltype(&cdssm_distillation_fwd) distill_fwd;
  decltype(&cdssm_distillation_bwd) distill_bwd;
  decltype(&cdssm_int4_code_bytes) code_bytes;
  decltype(&cdssm_int4_scale_bytes) scale_bytes;
  decltype(&cdssm_int4_pack) pack;
  decltype(&cdssm_int4_unpack) unpack;
  decltype(&cdssm_int4_quantize) quantize;
  decltype(&cdssm_int4_fingerprints) fingerprints;
  decltype(&cdssm_int4_linear_workspace_bytes) linear_bytes;
  decltype(&cdssm_int4_linear) linear;
  decltype(&cdssm_int4_linear_conv_step) linear_conv;
} lib;

void open_library(const std::string& path) {
  const Library from(path);
  from.get(lib.top, "cdssm_top_logits");
  from.get(lib.distill_bytes, "cdssm_distillation_workspace_bytes");
  from.get(lib.distill_fwd, "cdssm_distillation_fwd");
  from.get(lib.distill_bwd, "cdssm_distillation_bwd");
  from.get(lib.code_bytes, "cdssm_int4_code_bytes");
  from.get(lib.scale_bytes, "cdssm_int4_scale_bytes");
  from.get(lib.pack, "cdssm_int4_pack");
  from.get(lib.unpack, "cdssm_int4_unpack");
  from.get(lib.quantize, "cdssm_int4_quantize");
  from.get(lib.fingerprints, "cdssm_int4_fingerprints");
  from.get(lib.linear_bytes, "cdssm_int4_linear_workspace_bytes");
  from.get(lib.linear, "cdssm_int4_linear");
  from.get(lib.linear_conv, "cdssm_int4_linear_conv_step");
}

// A result without a gradient is not given in silence where one would be followed.
void no_gradient(const char* op, const char* name, const Tensor& t) {
  no_tangent(op, t);
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled() || !t.requires_grad(), op, " gives no gradient to ", name,
                              ": detach it, or call under torch.no_grad()");
}

// --- top logits --------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor> top_logits(const Tensor& logits, int64_t k) {
  no_gradient("top_logits", "logits", logits);
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(logits.device());
  auto shape = logits.sizes().vec();
  const int64_t V = shape.back();
  shape.back() = k;
  Tensor values = at::empty(shape, logits.options()), ids = at::empty(shape, logits.options().dtype(at::kLong));
  if (values.numel()) {
    const Tensor x = rows_of(logits);
    ok(lib.top(code_of(x), x.data_ptr(), row_stride(x), values.data_ptr(), ids.data_ptr<int64_t>(), x.size(0), V, k, stream_of(x)),
       "cdssm_top_logits");
  }
  return {values, ids};
}

// --- distillation ------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor> distill_fwd(const Tensor& logits, const Tensor& z, const Tensor& ids, double tau, int64_t reduction) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(logits.device());
  const auto fp32 = logits.options().dtype(at::kFloat);
  const auto shape = reduction == 0 ? logits.sizes().slice(0, logits.dim() - 1) : at::IntArrayRef{};
  if (z.numel() == 0) return {at::full(shape, reduction == 1 ? NAN : 0.0, fp32), Tensor()};
  const Tensor x = rows_of(logits), zs = z.contiguous(), is = ids.contiguous();
  const int64_t T = x.size(0);
  const Tensor ws = workspace(bytes(lib.distill_bytes(T), "distillation_loss"), x);
  Tensor loss = at::empty(shape, fp32);
  ok(lib.distill_fwd(code_of(x), code_of(zs), id_bytes(is), x.data_ptr(), row_stride(x), zs.data_ptr(), is.data_ptr(), float(tau),
                     int(reduction), loss.data_ptr<float>(), ws.data_ptr(), T, x.size(1), zs.size(-1), stream_of(x)),
     "cdssm_distillation_fwd");
  return {loss, ws};
}

// The gradient takes the logits' row stride where they are a slice of rows padded to whole vectors: so both sides of a row reach
// a 16-byte boundary together.
constexpr int64_t kMostPadding = 1024;

Tensor distill_bwd(const Tensor& grad, const Tensor& logits, const Tensor& z, const Tensor& ids, const Tensor& ws, double tau,
                   int64_t reduction) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(logits.device());
  if (!ws.defined()) return at::zeros(logits.sizes(), logits.options());
  const Tensor x = rows_of(logits), zs = z.contiguous(), is = ids.contiguous(), up = grad.to(at::kFloat).contiguous();
  const int64_t T = x.size(0), V = x.size(1), ld = row_stride(x);
  const bool padded = ld > V && ld <= V + kMostPadding && ld * int64_t(x.element_size()) % 16 == 0;
  const int64_t ldg = padded ? ld : V;
  Tensor out;
  if (padded) {
    std::vector<int64_t> strides(logits.dim());
    int64_t s = ldg;
    strides.back() = 1;
    for (int64_t i = logits.dim() - 2; i >= 0; --i) {
      strides[i] = s;
      s *= logits.size(i);
    }
    out = at::empty({T * ldg}, x.options()).as_strided(logits.sizes(), strides);
  } else {
    out = at::empty(logits.sizes(), x.options());
  }
  ok(lib.distill_bwd(code_of(x), code_of(zs), id_bytes(is), x.data_ptr(), ld, zs.data_ptr(), is.data_ptr(), float(tau),
                     int(reduction), up.data_ptr<float>(), ws.data_ptr(), out.data_ptr(), ldg, T, V, zs.size(-1), stream_of(x)),
     "cdssm_distillation_bwd");
  return out;
}

// The same without autograd.
std::tuple<Tensor, std::optional<Tensor>> distill_direct_fwd(const Tensor& logits, const Tensor& z, const Tensor& ids, double tau,
                                                             int64_t reduction) {
  auto [loss, ws] = distill_fwd(logits, z, ids, tau, reduction);
  return {loss, ws.defined() ? std::optional<Tensor>(ws) : std::nullopt};
}
Tensor distill_direct_bwd(const Tensor& grad, const Tensor& logits, const Tensor& z, const Tensor& ids, const std::optional<Tensor>& ws,
                          double tau, int64_t reduction) {
  const char* op = "distillation_loss_bwd";
  const int64_t T = logits.numel() / logits.size(-1);
  TORCH_CHECK_VALUE(grad.device() == logits.device() && grad.numel() == (reduction == 0 ? T : 1), op, ": the gradient of logits ",
                    logits.sizes(), " on ", logits.device(), ", got ", grad.sizes(), " on ", grad.device());
  TORCH_CHECK_VALUE(T == 0 ? !ws : ws && ws->device() == logits.device() && ws->scalar_type() == at::kByte && ws->is_contiguous() &&
                                       ws->numel() == bytes(lib.distill_bytes(T), op),
                    op, ": not the workspace of a forward over logits ", logits.sizes());
  return distill_bwd(grad, logits, z, ids, ws ? *ws : Tensor(), tau, reduction);
}

struct Distillation : torch::autograd::Function<Distillation> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& z, const Tensor& ids, double tau, int64_t reduction) {
    auto [loss, ws] = distill_fwd(logits, z, ids, tau, reduction);
    ctx->save_for_backward({logits, z, ids, ws});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    const auto saved = ctx->get_saved_variables();
    out[0] = distill_bwd(grads[0], saved[0], saved[1], saved[2], saved[3], ctx->saved_data["tau"].toDouble(),
                         ctx->saved_data["reduction"].toInt());
    return once("distillation_loss", std::move(out), {saved[0], grads[0]});
  }
};

Tensor distill(const Tensor& logits, const Tensor& z, const Tensor& ids, double tau, int64_t reduction) {
  no_tangent("distillation_loss", logits);
  no_gradient("distillation_loss", "teacher_logits", z);
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) return std::get<0>(distill_fwd(logits, z, ids, tau, reduction));
  return Distillation::apply(logits, z, ids, tau, reduction);
}

// --- 4-bit weights -----------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor> int4_pack(const Tensor& codes, const Tensor& scales, int64_t group) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(codes.device());
  const Tensor c = codes.contiguous(), s = scales.contiguous();
  const int64_t N = c.size(0), K = c.size(1);
  Tensor words = workspace(bytes(lib.code_bytes(N, K), "pack_int4"), c);
  Tensor out = at::empty({bytes(lib.scale_bytes(N, K, group), "pack_int4") / 2}, s.options());
  ok(lib.pack(c.data_ptr(), s.data_ptr(), words.data_ptr(), out.data_ptr(), N, K, group, stream_of(c)), "cdssm_int4_pack");
  return {words, out};
}

std::tuple<Tensor, Tensor> int4_quantize(const Tensor& weight, int64_t group) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(weight.device());
  const Tensor w = rows_of(weight);
  const int64_t N = w.size(0), K = w.size(1);
  bytes(lib.scale_bytes(N, K, group), "quantize_int4");
  Tensor codes = at::empty({N, K}, w.options().dtype(at::kChar));
  Tensor scales = at::empty({N, (K + group - 1) / group}, w.options().dtype(at::kBFloat16));
  ok(lib.quantize(code_of(w), w.data_ptr(), row_stride(w), codes.data_ptr(), scales.data_ptr(), N, K, group, stream_of(w)),
     "cdssm_int4_quantize");
  return {codes, scales};
}

// A number of what each weight (N, K) holds, whatever its strides.
Tensor int4_fingerprints(const std::vector<Tensor>& weights) {
  const char* op = "fingerprints";
  TORCH_CHECK_VALUE(!weights.empty(), op, ": no weights");
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(weights[0].device());
  const size_t count = weights.size();
  std::vector<Tensor> rows(count);
  std::vector<int> dtype(count);
  std::vector<const void*> at(count);
  std::vector<int64_t> ld(count), N(count), K(count);
  for (size_t i = 0; i < count; ++i) {
    const Tensor& w = weights[i];
    TORCH_CHECK(w.is_cuda() && w.device() == weights[0].device(), op, " of weights on one GPU, got ", w.device(), " and ", weights[0].device());
    TORCH_CHECK_TYPE(w.scalar_type() == at::kFloat || w.scalar_type() == at::kBFloat16, op, ": weights must be float32 or bfloat16, got ",
                     w.scalar_type());
    TORCH_CHECK_VALUE(w.dim() == 2, op, ": weights must be (N, K), got ", w.sizes());
    rows[i] = rows_of(w);
    dtype[i] = code_of(w);
    at[i] = rows[i].data_ptr();
    ld[i] = row_stride(rows[i]);
    N[i] = w.size(0);
    K[i] = w.size(1);
  }
  const Tensor sums = at::zeros({int64_t(count)}, weights[0].options().dtype(at::kLong));
  ok(lib.fingerprints(int64_t(count), dtype.data(), at.data(), ld.data(), N.data(), K.data(),
                      reinterpret_cast<uint64_t*>(sums.data_ptr<int64_t>()), stream_of(sums)),
     "cdssm_int4_fingerprints");
  return sums;
}

// A weight's tensors as they have to be for these sizes: the kernels read them whole.
void check_weight(const char* op, const Tensor& words, const Tensor& scales, int64_t N, int64_t K, int64_t group) {
  TORCH_CHECK_VALUE(words.is_cuda() && scales.device() == words.device() && words.scalar_type() == at::kByte &&
                        scales.scalar_type() == at::kBFloat16 && words.is_contiguous() && scales.is_contiguous() &&
                        words.numel() == bytes(lib.code_bytes(N, K), op) && 2 * scales.numel() == bytes(lib.scale_bytes(N, K, group), op),
                    op, ": not a 4-bit weight of ", N, " x ", K, " in groups of ", group);
}

std::tuple<Tensor, Tensor> int4_unpack(const Tensor& words, const Tensor& scales, int64_t N, int64_t K, int64_t group) {
  check_weight("dequantize", words, scales, N, K, group);
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(words.device());
  Tensor codes = at::empty({N, K}, words.options().dtype(at::kChar));
  Tensor out = at::empty({N, (K + group - 1) / group}, scales.options());
  ok(lib.unpack(words.data_ptr(), scales.data_ptr(), codes.data_ptr(), out.data_ptr(), N, K, group, stream_of(words)), "cdssm_int4_unpack");
  return {codes, out};
}

constexpr int64_t kMostStride = int64_t(1) << 24;  // of a residual's rows

// Rows (M, K) as the kernel reads them, in whole 16-byte vectors: copied, with zeros up to the next vector, where they are not.
Tensor vectors_of(const Tensor& t) {
  const int64_t M = t.size(0), K = t.size(1);
  if (K % 8 == 0 && (M == 1 || (t.stride(0) % 8 == 0 && t.stride(0) <= int64_t(1) << 32)) &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
  const Tensor wide = at::zeros({M, (K + 7) / 8 * 8}, t.options());
  Tensor whole = wide.narrow(1, 0, K);
  whole.copy_(t);
  return whole;
}

// conv: window, weight (C, taps) or (C, 1, taps), bias of a conv step on the columns from conv_col on, its result then the second.
Tensor product(const char* op, const Tensor& x, const Tensor& words, const Tensor& scales, int64_t N, int64_t K, int64_t group,
               const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, const std::optional<Tensor>& norm,
               double eps, const Tensor* window = nullptr, const Tensor* conv_weight = nullptr, const Tensor* conv_bias = nullptr,
               int64_t conv_col = 0, Tensor* conv_y = nullptr) {
  check_weight(op, words, scales, N, K, group);
  no_gradient(op, "x", x);
  TORCH_CHECK(x.is_cuda(), op, " runs on the GPU only");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16, op, ": x must be bfloat16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K, op, ": x must be (..., ", K, "), got ", x.sizes());
  TORCH_CHECK_VALUE(x.numel() <= 64 * K, op, ": x must have at most 64 rows, got ", x.sizes());
  auto shape = x.sizes().vec();
  shape.back() = N;
  const auto part = [&](const std::optional<Tensor>& t, const char* name, at::IntArrayRef want) {
    if (!t) return Tensor();
    no_gradient(op, name, *t);
    TORCH_CHECK(t->device() == x.device(), op, ": ", name, " is on ", t->device(), ", x on ", x.device());
    TORCH_CHECK_VALUE(t->sizes() == want, op, ": ", name, " must be ", want, ", got ", t->sizes());
    return t->to(at::kBFloat16);
  };
  TORCH_CHECK(words.device() == x.device(), op, ": the weight is on ", words.device(), ", x on ", x.device());
  const Tensor b = part(bias, "bias", {N}), g = part(norm, "norm_weight", {K}), r = part(residual, "residual", shape);
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(shape, x.options());
  if (y.numel() == 0) return y;
  const Tensor x2 = vectors_of(rows_of(x)), bc = b.defined() ? b.contiguous() : b,
               gc = g.defined() ? vectors_of(g.contiguous().view({1, K})) : g;
  const int64_t M = x2.size(0);
  Tensor r2 = r.defined() ? rows_of(r) : r;
  if (r2.defined() && M > 1 && r2.stride(0) > kMostStride) r2 = r2.contiguous();
  Tensor ws;
  if (const int64_t n = bytes(lib.linear_bytes(M, N, K, g.defined()), op)) ws = workspace(n, x);
  const auto at = [](const Tensor& t) -> void* { return t.defined() ? t.data_ptr() : nullptr; };
  const int64_t ldx = M == 1 ? (K + 7) / 8 * 8 : x2.stride(0);
  if (conv_y) {
    const int64_t C = conv_bias->size(0), taps = conv_weight->size(-1);
    const Tensor w = conv_weight->to(at::kBFloat16).contiguous(), cb = conv_bias->to(at::kBFloat16).contiguous();
    ok(lib.linear_conv(1, x2.data_ptr(), ldx, words.data_ptr(), scales.data_ptr(), group, at(bc), at(gc), float(eps), y.data_ptr(), N,
                       at(ws), M, N, K, conv_col, window->data_ptr(), w.data_ptr(), cb.data_ptr(), conv_y->data_ptr(), C, taps,
                       stream_of(x)),
       "cdssm_int4_linear_conv_step");
    return y;
  }
  ok(lib.linear(1, x2.data_ptr(), ldx, words.data_ptr(), scales.data_ptr(), group, at(bc), at(r2),
                r2.defined() ? (M == 1 ? N : r2.stride(0)) : 0, at(gc), float(eps), y.data_ptr(), N, at(ws), M, N, K, stream_of(x)),
     "cdssm_int4_linear");
  return y;
}

Tensor int4_linear(const Tensor& x, const Tensor& words, const Tensor& scales, int64_t N, int64_t K, int64_t group,
                   const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, const std::optional<Tensor>& norm,
                   double eps) {
  return product("int4_linear", x, words, scales, N, K, group, bias, residual, norm, eps);
}

std::tuple<Tensor, Tensor> int4_linear_conv_step(const Tensor& x, const Tensor& words, const Tensor& scales, int64_t N, int64_t K,
                                                 int64_t group, const std::optional<Tensor>& bias, const Tensor& norm, double eps,
                                                 int64_t conv_col, const Tensor& window, const Tensor& conv_weight,
                                                 const Tensor& conv_bias) {
  const char* op = "int4_linear_conv_step";
  TORCH_CHECK_VALUE(x.dim() == 2 && conv_bias.dim() == 1 && conv_weight.dim() >= 2, op, ": x must be (M, K), conv_weight (C, taps) or "
                    "(C, 1, taps) and conv_bias (C), got ", x.sizes(), ", ", conv_weight.sizes(), ", ", conv_bias.sizes());
  const int64_t M = x.size(0), C = conv_bias.size(0), taps = conv_weight.size(-1);
  TORCH_CHECK_VALUE(conv_weight.numel() == C * taps && conv_weight.size(0) == C, op, ": conv_weight must be (", C, ", taps), got ",
                    conv_weight.sizes());
  TORCH_CHECK_VALUE(window.sizes() == at::IntArrayRef({M, taps - 1, C}) && window.scalar_type() == at::kBFloat16 && window.is_contiguous(),
                    op, ": window must be a contiguous (", M, ", ", taps - 1, ", ", C, ") bfloat16 tensor");
  for (const Tensor* t : {&window, &conv_weight, &conv_bias}) {
    TORCH_CHECK(t->device() == x.device(), op, ": the conv's tensors must be on ", x.device(), ", got ", t->device());
    no_gradient(op, "the conv's tensors", *t);
  }
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(x.device());
  Tensor conv_y = at::empty({M, C}, x.options());
  Tensor y = product(op, x, words, scales, N, K, group, bias, std::nullopt, norm, eps, &window, &conv_weight, &conv_bias, conv_col,
                     &conv_y);
  return {y, conv_y};
}

}  // namespace

PYBIND11_MODULE(_compress_nodes, m) {
  m.def("open_library", torch::wrap_pybind_function(open_library));
  m.def("top_logits", torch::wrap_pybind_function(top_logits));
  m.def("distill", torch::wrap_pybind_function(distill));
  m.def("distill_fwd", torch::wrap_pybind_function(distill_direct_fwd));
  m.def("distill_bwd", torch::wrap_pybind_function(distill_direct_bwd));
  m.def("int4_pack", torch::wrap_pybind_function(int4_pack));
  m.def("int4_quantize", torch::wrap_pybind_function(int4_quantize));
  m.def("int4_fingerprints", torch::wrap_pybind_function(int4_fingerprints));
  m.def("int4_unpack", torch::wrap_pybind_function(int4_unpack));
  m.def("int4_linear", torch::wrap_pybind_function(int4_linear));
  m.def("int4_linear_conv_step", torch::wrap_pybind_function(int4_linear_conv_step));
}

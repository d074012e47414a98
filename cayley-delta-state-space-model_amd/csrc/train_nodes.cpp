// The host side of the training step's ends (token embedding, head loss, gradient clipping) in C++, with their autograd
// nodes: torch runs a backward on a thread of its own, where a Python node has to wait for the interpreter and runs its dozen
// calls on a cold core, and a list of gradients costs Python more than the kernels.  The kernels are those of
// libcdssm_hip.so, through its C entry points.  Embedding and gradient of 64 tokens: 29 us a call instead of 46 .. 90 by
// Python nodes (torch's own 28); loss and gradients of 200 x 128 tokens, 97 words, fp32: 81 instead of 151.
#include <ATen/ops/full.h>
#include <ATen/ops/zeros.h>

#include "nodes_common.hpp"

namespace {

struct Entries {
  decltype(&cdssm_token_embedding_order_bytes) order_bytes;
  decltype(&cdssm_token_embedding_fwd) emb_fwd;
  decltype(&cdssm_token_embedding_bwd_workspace_bytes) emb_bytes;
  decltype(&cdssm_token_embedding_bwd) emb_bwd;
  decltype(&cdssm_linear_cross_entropy_workspace_bytes) ce_bytes;
  decltype(&cdssm_linear_cross_entropy_fwd) ce_fwd;
  decltype(&cdssm_linear_cross_entropy_bwd_workspace_bytes) ce_bwd_bytes;
  decltype(&cdssm_linear_cross_entropy_bwd) ce_bwd;
  decltype(&cdssm_grad_norm_workspace_bytes) norm_bytes;
  decltype(&cdssm_grad_norm) norm;
  decltype(&cdssm_clip_grads) clip;
} lib;

void open_library(const std::string& path) {
  const Library from(path);
  from.get(lib.order_bytes, "cdssm_token_embedding_order_bytes");
  from.get(lib.emb_fwd, "cdssm_token_embedding_fwd");
  from.get(lib.emb_bytes, "cdssm_token_embedding_bwd_workspace_bytes");
  from.get(lib.emb_bwd, "cdssm_token_embedding_bwd");
  from.get(lib.ce_bytes, "cdssm_linear_cross_entropy_workspace_bytes");
  from.get(lib.ce_fwd, "cdssm_linear_cross_entropy_fwd");
  from.get(lib.ce_bwd_bytes, "cdssm_linear_cross_entropy_bwd_workspace_bytes");
  from.get(lib.ce_bwd, "cdssm_linear_cross_entropy_bwd");
  from.get(lib.norm_bytes, "cdssm_grad_norm_workspace_bytes");
  from.get(lib.norm, "cdssm_grad_norm");
  from.get(lib.clip, "cdssm_clip_grads");
}

// --- token embedding ---------------------------------------------------------------------------------------------

// order: where the sorted tokens go, for a backward (undefined: not asked for).
Tensor embed(const Tensor& ids, const Tensor& weight, double scale, int64_t padding, Tensor* order) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(weight.device());
  const Tensor w = rows_of(weight), i = ids.contiguous();
  auto shape = ids.sizes().vec();
  shape.push_back(w.size(1));
  Tensor y = at::empty(shape, w.options());
  if (const int64_t n = i.numel()) {
    if (order) *order = workspace(bytes(lib.order_bytes(n, w.size(0)), "token_embedding"), w);
    ok(lib.emb_fwd(code_of(w), id_bytes(i), i.data_ptr(), w.data_ptr(), row_stride(w), float(scale), padding, y.data_ptr(),
                   order ? order->data_ptr() : nullptr, n, w.size(0), w.size(1), stream_of(w)),
       "cdssm_token_embedding_fwd");
  }
  return y;
}

Tensor embedding_fwd(const Tensor& ids, const Tensor& weight, double scale) { return embed(ids, weight, scale, -1, nullptr); }

Tensor table_gradient(const Tensor& grad, const Tensor& ids, const Tensor& order, int64_t rows, double scale, int64_t padding) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(grad.device());
  const Tensor g = rows_of(grad), i = ids.contiguous();
  const int64_t T = g.size(0), C = g.size(1);
  if (T == 0) return at::zeros({rows, C}, g.options());
  const Tensor ws = workspace(
      bytes(lib.emb_bytes(T, rows, C), "token_embedding") - (order.defined() ? order.numel() : 0), g);
  Tensor dw = at::empty({rows, C}, g.options());
  ok(lib.emb_bwd(code_of(g), id_bytes(i), i.data_ptr(), g.data_ptr(), row_stride(g), float(scale), padding,
                 order.defined() ? order.data_ptr() : nullptr, dw.data_ptr(), ws.data_ptr(), T, rows, C, stream_of(g)),
     "cdssm_token_embedding_bwd");
  return dw;
}

Tensor embedding_bwd(const Tensor& grad, const Tensor& ids, int64_t rows, double scale, int64_t padding) {
  return table_gradient(grad, ids, Tensor(), rows, scale, padding);
}

// --- head loss ---------------------------------------------------------------------------------------------------

// The forward's workspace, and up to 64 KB and T bytes more: its size tells other tokens, words and columns apart, which the entry point
// rounds up (a backward with a shorter weight would read behind it, at the labels).
int64_t loss_bytes(const Tensor& w, int64_t T) {
  const uint64_t mix = (uint64_t(w.size(0)) * 0x9e3779b97f4a7c15u + uint64_t(w.size(1))) * 0xd1b54a32d192ed03u;
  return T + int64_t(mix >> 48) + bytes(lib.ce_bytes(code_of(w), w.data_ptr(), row_stride(w), T, w.size(0), w.size(1)), "linear_cross_entropy");
}

std::tuple<Tensor, std::optional<Tensor>> loss_fwd(const Tensor& x, const Tensor& weight, const Tensor& labels, int64_t ignore,
                                                   int64_t reduction) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(x.device());
  const Tensor x2 = rows_of(x), w = rows_of(weight), y = labels.contiguous();
  const int64_t T = x2.size(0), V = w.size(0), d = w.size(1);
  const auto fp32 = x.options().dtype(at::kFloat);
  const auto shape = reduction == 0 ? labels.sizes() : at::IntArrayRef{};
  if (T == 0) return {at::full(shape, reduction == 1 ? NAN : 0.0, fp32), std::nullopt};
  const Tensor ws = workspace(loss_bytes(w, T), x);
  Tensor loss = at::empty(shape, fp32);
  ok(lib.ce_fwd(code_of(w), id_bytes(y), x2.data_ptr(), row_stride(x2), w.data_ptr(), row_stride(w), y.data_ptr(), ignore,
                int(reduction), loss.data_ptr<float>(), ws.data_ptr(), T, V, d, stream_of(w)),
     "cdssm_linear_cross_entropy_fwd");
  return {loss, ws};
}

std::tuple<std::optional<Tensor>, std::optional<Tensor>> loss_bwd(const Tensor& grad, const Tensor& weight,
                                                                  const std::optional<Tensor>& fwd_ws,
                                                                  const std::vector<int64_t>& x_shape, int64_t reduction,
                                                                  bool need_x, bool need_weight) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(weight.device());
  const Tensor w = rows_of(weight);
  const int64_t V = w.size(0), d = w.size(1);
  int64_t T = 1;
  for (size_t k = 0; k + 1 < x_shape.size(); ++k) T *= x_shape[k];
  std::optional<Tensor> dx, dw;
  if (T == 0) {
    if (need_x) dx = at::empty(x_shape, w.options());
    if (need_weight) dw = at::zeros({V, d}, w.options());
    return {dx, dw};
  }
  if (need_x) dx = at::empty(x_shape, w.options());
  if (need_weight) dw = at::empty({V, d}, w.options());
  if (!dx && !dw) return {dx, dw};
  const int64_t ldw = row_stride(w);
  TORCH_CHECK_VALUE(fwd_ws && fwd_ws->defined() && fwd_ws->device() == w.device() &&
                        fwd_ws->numel() == loss_bytes(w, T),
                    "linear_cross_entropy_bwd: not the workspace of a forward over x ", at::IntArrayRef(x_shape),
                    " and this weight");
  const Tensor g = grad.to(at::kFloat).contiguous();
  const Tensor ws =
      workspace(bytes(lib.ce_bwd_bytes(code_of(w), w.data_ptr(), ldw, T, V, d), "linear_cross_entropy_bwd"), w);
  ok(lib.ce_bwd(code_of(w), w.data_ptr(), ldw, int(reduction), g.data_ptr<float>(), fwd_ws->data_ptr(),
                dx ? dx->data_ptr() : nullptr, d, dw ? dw->data_ptr() : nullptr, d, ws.data_ptr(), T, V, d, stream_of(w)),
     "cdssm_linear_cross_entropy_bwd");
  return {dx, dw};
}

// --- gradient norm and clipping ------------------------------------------------------------------------------------

// The tensors as the entry points take them.
struct Table {
  std::vector<void*> at;
  std::vector<int> code;
  std::vector<int64_t> size;
  Table(const char* op, const char* what, const std::vector<Tensor>& ts) {
    at.reserve(ts.size());
    code.reserve(ts.size());
    size.reserve(ts.size());
    for (const Tensor& t : ts) {
      TORCH_CHECK(t.is_cuda(), op, " runs on the GPU only");
      TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, op, ": ", what,
                       " must be float32 or bfloat16, got ", t.scalar_type());
      no_tangent(op, t);
      TORCH_CHECK(t.device() == ts[0].device(), op, ": tensors on ", ts[0].device(), " and ", t.device());
      TORCH_CHECK_VALUE(t.is_non_overlapping_and_dense(), op, ": ", what, " of shape ", t.sizes(), " and strides ", t.strides(),
                        " has gaps or overlaps");
      at.push_back(t.data_ptr());
      code.push_back(code_of(t));
      size.push_back(t.numel());
    }
  }
};

Tensor global_norm(const std::vector<Tensor>& ts) {
  const at::AutoGradMode off(false);
  if (ts.empty()) return at::zeros({});
  const Table in("global_grad_norm", "a gradient", ts);
  const c10::DeviceGuard guard(ts[0].device());
  const int64_t n = ts.size();
  Tensor norm = at::empty({}, ts[0].options().dtype(at::kFloat));
  const Tensor ws = workspace(lib.norm_bytes(n), ts[0]);
  ok(lib.norm(n, in.at.data(), in.code.data(), in.size.data(), norm.data_ptr<float>(), ws.data_ptr(), stream_of(norm)),
     "cdssm_grad_norm");
  return norm;
}

// Whatever is written may share no memory with what is written or read elsewhere.
void check_apart(const Table& in, const Table& out) {
  struct Range {
    uintptr_t begin, end;
    bool write;
  };
  std::vector<Range> rs;
  rs.reserve(2 * in.at.size());
  auto add = [&](const Table& t, size_t i, bool write) {
    const auto p = reinterpret_cast<uintptr_t>(t.at[i]);
    if (t.size[i]) rs.push_back({p, p + t.size[i] * (t.code[i] ? 2 : 4), write});
  };
  for (size_t i = 0; i < in.at.size(); ++i) {
    add(out, i, true);
    if (in.at[i] != out.at[i] || in.code[i] != out.code[i]) add(in, i, false);
  }
  auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  if (!std::is_sorted(rs.begin(), rs.end(), before)) std::sort(rs.begin(), rs.end(), before);
  uintptr_t read = 0, written = 0;  // the ends so far
  for (const Range& r : rs) {
    TORCH_CHECK_VALUE(!r.write || written <= r.begin, "clip_grads: a tensor is given twice, or shares memory with another");
    TORCH_CHECK_VALUE((r.write ? read : written) <= r.begin,
                      "clip_grads: an output is another gradient's tensor, or shares memory with a gradient");
    (r.write ? written : read) = std::max(r.write ? written : read, r.end);
  }
}

Tensor clip(const std::vector<Tensor>& ts, double max_norm, const std::optional<std::vector<Tensor>>& out) {
  const char* op = "clip_grads";
  const at::AutoGradMode off(false);
  TORCH_CHECK_VALUE(max_norm >= 0, op, ": max_norm must be at least 0, got ", max_norm);
  const std::vector<Tensor>& os = out ? *out : ts;
  TORCH_CHECK_VALUE(os.size() == ts.size(), op, ": ", ts.size(), " gradients, ", os.size(), " outputs");
  if (ts.empty()) return at::zeros({});
  const Table in(op, "a gradient", ts);
  std::optional<Table> other;
  if (out) {
    other.emplace(op, "an output", os);
    for (size_t i = 0; i < ts.size(); ++i) {
      const Tensor &t = ts[i], &o = os[i];
      TORCH_CHECK_VALUE(o.numel() == t.numel() && o.device() == t.device() &&
                            ((t.is_contiguous() && o.is_contiguous()) || (o.sizes() == t.sizes() && o.strides() == t.strides())),
                        op, ": an output must have its gradient's size, layout and device, got ", o.sizes(), " ", o.strides(),
                        " for ", t.sizes(), " ", t.strides());
    }
  }
  const Table& to = other ? *other : in;
  check_apart(in, to);
  const c10::DeviceGuard guard(ts[0].device());
  const int64_t n = ts.size();
  Tensor norm = at::empty({}, ts[0].options().dtype(at::kFloat));
  const Tensor ws = workspace(lib.norm_bytes(n), ts[0]);
  ok(lib.clip(n, in.at.data(), in.code.data(), to.at.data(), to.code.data(), in.size.data(), float(max_norm),
              norm.data_ptr<float>(), ws.data_ptr(), stream_of(norm)),
     "cdssm_clip_grads");
  for (const Tensor& o : os)  // a graph that saved one of them has to notice
    if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  return norm;
}

Tensor clip_parameters(const std::vector<Tensor>& ps, double max_norm) {
  std::vector<Tensor> gs;
  gs.reserve(ps.size());
  for (const Tensor& p : ps)
    if (p.grad().defined()) gs.push_back(p.grad());
  return clip(gs, max_norm, std::nullopt);
}

// --- nodes -------------------------------------------------------------------------------------------------------

struct TokenEmbedding : torch::autograd::Function<TokenEmbedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t padding) {
    Tensor order;
    const Tensor y = embed(ids, weight, scale, padding, &order);
    ctx->save_for_backward({ids, order});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(4);
    const auto saved = ctx->get_saved_variables();
    out[0] = table_gradient(grads[0], saved[0], saved[1], ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble(),
                            ctx->saved_data["padding"].toInt());
    return once("token_embedding", std::move(out), grads);
  }
};

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& labels, int64_t ignore,
                        int64_t reduction) {
    auto [loss, ws] = loss_fwd(x, weight, labels, ignore, reduction);
    ctx->save_for_backward({weight, ws ? *ws : Tensor()});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list out(5);
    const auto saved = ctx->get_saved_variables();
    auto [dx, dw] = loss_bwd(grads[0], saved[0], saved[1], ctx->saved_data["shape"].toIntVector(),
                             ctx->saved_data["reduction"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    if (dx) out[0] = *dx;
    if (dw) out[1] = *dw;
    return once("linear_cross_entropy", std::move(out), {saved[0], grads[0]});
  }
};

Tensor embedding(const Tensor& weight, const Tensor& ids, double scale, int64_t padding) {
  no_tangent("token_embedding", weight);
  if (!at::GradMode::is_enabled() || !weight.requires_grad()) return embedding_fwd(ids, weight, scale);
  return TokenEmbedding::apply(weight, ids, scale, padding);
}

Tensor loss(const Tensor& x, const Tensor& weight, const Tensor& labels, int64_t ignore, int64_t reduction) {
  no_tangent("linear_cross_entropy", x);
  no_tangent("linear_cross_entropy", weight);
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || weight.requires_grad()))
    return std::get<0>(loss_fwd(x, weight, labels, ignore, reduction));
  return LinearCrossEntropy::apply(x, weight, labels, ignore, reduction);
}

}  // namespace

PYBIND11_MODULE(_train_nodes, m) {
  m.def("open_library", torch::wrap_pybind_function(open_library));
  m.def("embedding_fwd", torch::wrap_pybind_function(embedding_fwd));
  m.def("embedding_bwd", torch::wrap_pybind_function(embedding_bwd));
  m.def("loss_fwd", torch::wrap_pybind_function(loss_fwd));
  m.def("loss_bwd", torch::wrap_pybind_function(loss_bwd));
  m.def("embedding", torch::wrap_pybind_function(embedding));
  m.def("global_norm", torch::wrap_pybind_function(global_norm));
  m.def("clip", torch::wrap_pybind_function(clip));
  m.def("clip_parameters", torch::wrap_pybind_function(clip_parameters));
  m.def("loss", torch::wrap_pybind_function(loss));
}

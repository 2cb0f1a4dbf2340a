// Python bindings of the residual-stream kernels (residual.cuh).  Shapes, dtypes and devices are
// checked here; every entry allocates its outputs and launches on the current stream of its
// tensors' device.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>

#include "residual.h"

int* cfb_err_ptr(int device);
int cfb_num_sms(int device);

// Gradients under create_graph: they have no gradient themselves, and say so when asked.
torch::autograd::variable_list cfb_once_differentiable(torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list defined;
  for (const auto& g : grads)
    if (g.defined()) defined.push_back(g.detach().requires_grad_());
  if (defined.empty()) return grads;
  const auto node = std::make_shared<torch::autograd::DelayedError>(
      "these gradients cannot be differentiated twice", static_cast<int64_t>(defined.size()));
  const torch::autograd::variable_list out = (*node)(std::move(defined));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

Tensor empty(at::IntArrayRef sizes, torch::ScalarType dtype, const Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

int type_of(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  switch (t.scalar_type()) {
    case torch::kBFloat16: return cfb::kStreamBf16;
    case torch::kHalf: return cfb::kStreamHalf;
    case torch::kFloat32: return cfb::kStreamFloat;
    default:
      TORCH_CHECK_TYPE(false, name, " must be bfloat16, float16 or float32, got ",
                       t.scalar_type());
  }
}

void like(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.get_device() == x.get_device(), name,
                    " must be on x's CUDA device");
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " must have x's dtype ",
                   x.scalar_type(), ", got ", t.scalar_type());
}

// Contiguous and 16-byte aligned; other layouts are copied.
Tensor dense(const Tensor& t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0 ? c.clone() : c;
}

Tensor rows(const Tensor& t, const Tensor& x, const char* name) {
  like(t, x, name);
  TORCH_CHECK_VALUE(t.sizes() == x.sizes(), name, " must have x's shape");
  return dense(t);
}

// A weight [H], or nothing.
OptTensor column(const OptTensor& t, const Tensor& x, const char* name) {
  if (!t.has_value()) return t;
  like(*t, x, name);
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1), name, " must be [", x.size(-1), "]");
  return dense(*t);
}
const void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

cfb::DropArgs drop_of(double p, const OptTensor& seed, int64_t seed_value, int64_t stream,
                      const Tensor& x) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be between 0 and 1");
  TORCH_CHECK_VALUE(stream >= 0 && stream <= 0xffffffffll, "stream must fit 32 bits");
  cfb::DropArgs d;
  d.threshold = static_cast<int>(std::floor(p * 65536.0 + 0.5));
  d.stream = static_cast<uint32_t>(stream);
  d.seed = static_cast<uint64_t>(seed_value);
  if (seed.has_value()) {
    TORCH_CHECK_VALUE(seed->is_cuda() && seed->get_device() == x.get_device(),
                      "seed must be on x's CUDA device");
    TORCH_CHECK_TYPE(seed->scalar_type() == torch::kInt64, "seed must be int64");
    TORCH_CHECK_VALUE(seed->numel() == 1, "seed must have one element");
    d.seed_ptr = seed->data_ptr<int64_t>();
  }
  return d;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed with code ", rc, " ",
              rc > 0 ? cudaGetErrorString(static_cast<cudaError_t>(rc)) : "");
}

// The shape, weights and dropout of a call.
cfb::JoinArgs args_of(const Tensor& x, const OptTensor& w1, const OptTensor& gate,
                      const OptTensor& w2, double scale, const cfb::DropArgs& drop, double eps) {
  cfb::JoinArgs a;
  a.type = type_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have at least one channel");
  TORCH_CHECK_VALUE(x.size(-1) <= 0x7fffffff, "rows are too wide");
  a.H = static_cast<int>(x.size(-1));
  a.T = x.numel() / a.H;
  TORCH_CHECK_VALUE(cfb::join_width_ok(a.H), "rows of ", a.H, " channels are too wide");
  TORCH_CHECK_VALUE(std::isfinite(scale), "scale must be finite");
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "eps must not be negative");
  a.w1 = ptr(w1);
  a.gate = ptr(gate);
  a.w2 = ptr(w2);
  a.drop = drop;
  a.err = cfb_err_ptr(x.get_device());
  a.scale = static_cast<float>(scale);
  a.eps = static_cast<float>(eps);
  return a;
}

// (x', y or None, 1 / rms of the branch or None, 1 / rms of x' or None); the last two only with
// `save`, for the backward pass.
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> residual_norm_fwd(
    const Tensor& x_in, const Tensor& b_in, const OptTensor& w1_in, const OptTensor& gate_in,
    const OptTensor& w2_in, double scale, double p, const OptTensor& seed, int64_t seed_value,
    int64_t stream, double eps, bool save) {
  type_of(x_in, "x");
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = dense(x_in), b = rows(b_in, x, "branch");
  const OptTensor w1 = column(w1_in, x, "branch_weight"), gate = column(gate_in, x, "gate"),
                  w2 = column(w2_in, x, "norm_weight");
  cfb::JoinArgs a = args_of(x, w1, gate, w2, scale, drop_of(p, seed, seed_value, stream, x), eps);
  Tensor xnew = empty(x.sizes(), x.scalar_type(), x);
  OptTensor y, r1, r2;
  if (w2.has_value()) y = empty(x.sizes(), x.scalar_type(), x);
  if (save && w1.has_value()) r1 = empty({a.T}, torch::kFloat32, x);
  if (save && w2.has_value()) r2 = empty({a.T}, torch::kFloat32, x);
  a.x = x.data_ptr();
  a.b = b.data_ptr();
  a.xnew = xnew.data_ptr();
  a.y = y.has_value() ? y->data_ptr() : nullptr;
  a.r1 = r1.has_value() ? r1->data_ptr<float>() : nullptr;
  a.r2 = r2.has_value() ? r2->data_ptr<float>() : nullptr;
  check_rc(cfb::join_fwd(a, cfb_num_sms(x.get_device()), at::cuda::getCurrentCUDAStream()),
           "residual_norm");
  return {xnew, y, r1, r2};
}

// (dx, dbranch, dbranch_weight, dgate, dnorm_weight), each where `need` asks for it.
std::vector<OptTensor> residual_norm_bwd(const OptTensor& dxnew_in, const OptTensor& dy_in,
                                         const Tensor& xnew, const Tensor& b_in,
                                         const OptTensor& w1_in, const OptTensor& gate_in,
                                         const OptTensor& w2_in,
                                         const OptTensor& r1, const OptTensor& r2, double scale,
                                         double p, const OptTensor& seed, int64_t seed_value,
                                         int64_t stream, const std::vector<bool>& need) {
  TORCH_CHECK(need.size() == 5, "need has five entries");
  type_of(xnew, "x");
  const c10::cuda::CUDAGuard guard(xnew.device());
  const int sms = cfb_num_sms(xnew.get_device());
  TORCH_CHECK(xnew.is_contiguous(), "saved tensors do not match");
  const Tensor b = rows(b_in, xnew, "branch");
  const OptTensor w1 = column(w1_in, xnew, "branch_weight"), gate = column(gate_in, xnew, "gate"),
                  w2 = column(w2_in, xnew, "norm_weight");
  cfb::JoinArgs a =
      args_of(xnew, w1, gate, w2, scale, drop_of(p, seed, seed_value, stream, xnew), 0.0);
  OptTensor dxnew, dy;
  if (dxnew_in.has_value()) dxnew = rows(*dxnew_in, xnew, "gradient of x'");
  if (dy_in.has_value()) dy = rows(*dy_in, xnew, "gradient of y");
  TORCH_CHECK(!w1.has_value() || (r1.has_value() && r1->numel() == a.T), "r1 is missing");
  TORCH_CHECK(!dy.has_value() || (w2.has_value() && r2.has_value() && r2->numel() == a.T),
              "r2 is missing");
  const auto make = [&](bool on, at::IntArrayRef sizes) {
    return on ? OptTensor(empty(sizes, xnew.scalar_type(), xnew)) : OptTensor();
  };
  std::vector<OptTensor> out = {make(need[0], xnew.sizes()), make(need[1], xnew.sizes()),
                                make(need[2] && w1.has_value(), {a.H}),
                                make(need[3] && gate.has_value(), {a.H}),
                                make(need[4] && w2.has_value(), {a.H})};
  const auto at = [&](int i) { return out[i].has_value() ? out[i]->data_ptr() : nullptr; };
  a.xnew = xnew.data_ptr();
  a.b = b.data_ptr();
  a.dxnew = ptr(dxnew);
  a.dy = ptr(dy);
  a.r1 = r1.has_value() ? r1->data_ptr<float>() : nullptr;
  a.r2 = r2.has_value() ? r2->data_ptr<float>() : nullptr;
  a.dx = at(0);
  a.db = at(1);
  a.dw1 = at(2);
  a.dgate = at(3);
  a.dw2 = at(4);
  const int blocks = cfb::join_bwd_blocks(a, sms);
  TORCH_CHECK(blocks > 0, "residual_norm: rows are too wide");
  Tensor ws;
  if (a.dw1 != nullptr || a.dgate != nullptr || a.dw2 != nullptr) {
    ws = empty({static_cast<int64_t>(blocks) * 2 * a.H}, torch::kFloat32, xnew);
    a.partials = ws.data_ptr<float>();
  }
  check_rc(cfb::join_bwd(a, sms, at::cuda::getCurrentCUDAStream()), "residual_norm");
  return out;
}

Tensor dropout(const Tensor& x_in, double p, const OptTensor& seed, int64_t seed_value,
               int64_t stream) {
  const int type = type_of(x_in, "x");
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = dense(x_in);
  const cfb::DropArgs d = drop_of(p, seed, seed_value, stream, x);
  Tensor y = empty(x.sizes(), x.scalar_type(), x);
  check_rc(cfb::dropout_run(x.data_ptr(), y.data_ptr(), x.numel(), type, d,
                            at::cuda::getCurrentCUDAStream()),
           "dropout");
  return y;
}

// ------------------------------------------------------------------ autograd
// The nodes are C++ ones: a Python node's backward takes the interpreter's lock on the engine's
// thread, which is more time than the kernels of a small call take.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& seed, double p,
                        int64_t seed_value, int64_t stream) {
    ctx->save_for_backward({or_none(seed)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed_value;
    ctx->saved_data["stream"] = stream;
    return dropout(x, p, seed, seed_value, stream);
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    Tensor dx = dropout(dy[0], ctx->saved_data["p"].toDouble(), opt(saved[0]),
                        ctx->saved_data["seed"].toInt(), ctx->saved_data["stream"].toInt());
    return cfb_once_differentiable({dx, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout_grad(const Tensor& x, double p, const OptTensor& seed, int64_t seed_value,
                    int64_t stream) {
  return DropoutNode::apply(x, seed, p, seed_value, stream);
}

struct ResidualNormNode : torch::autograd::Function<ResidualNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& b,
                               const OptTensor& w1, const OptTensor& gate, const OptTensor& w2,
                               const OptTensor& seed, double scale, double p, int64_t seed_value,
                               int64_t stream, double eps) {
    ctx->set_materialize_grads(false);
    auto [xnew, y, r1, r2] = residual_norm_fwd(x, b, w1, gate, w2, scale, p, seed, seed_value,
                                               stream, eps, true);
    ctx->save_for_backward({xnew, b, or_none(w1), or_none(gate), or_none(w2), or_none(r1),
                            or_none(r2), or_none(seed)});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed_value;
    ctx->saved_data["stream"] = stream;
    variable_list out = {xnew};
    if (y.has_value()) out.push_back(*y);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(11);
    const auto v = ctx->get_saved_variables();
    const bool dy = g.size() > 1 && g[1].defined();
    std::vector<bool> need(5);
    for (int i = 0, k = 0; i < 5; ++i) {
      // the graph's edges are the defined inputs' only
      const bool given = i < 2 || v[i].defined();
      need[i] = given && ctx->needs_input_grad(k);
      if (given) ++k;
    }
    need[4] = need[4] && dy;
    if ((!g[0].defined() && !dy) || !(need[0] || need[1] || need[2] || need[3] || need[4]))
      return out;
    const auto grads = residual_norm_bwd(
        opt(g[0]), dy ? OptTensor(g[1]) : OptTensor(), v[0], v[1], opt(v[2]), opt(v[3]), opt(v[4]),
        opt(v[5]), opt(v[6]), ctx->saved_data["scale"].toDouble(), ctx->saved_data["p"].toDouble(),
        opt(v[7]), ctx->saved_data["seed"].toInt(), ctx->saved_data["stream"].toInt(), need);
    for (int i = 0; i < 5; ++i) out[i] = or_none(grads[i]);
    return cfb_once_differentiable(std::move(out));
  }
};

std::tuple<Tensor, OptTensor> residual_norm_grad(const Tensor& x, const Tensor& b,
                                                 const OptTensor& w1, const OptTensor& gate,
                                                 const OptTensor& w2, double scale, double p,
                                                 const OptTensor& seed, int64_t seed_value,
                                                 int64_t stream, double eps) {
  const auto out = ResidualNormNode::apply(x, b, w1, gate, w2, seed, scale, p, seed_value, stream,
                                           eps);
  return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
}

}  // namespace

void register_stream(pybind11::module& m) {
  m.def("residual_norm_fwd", &residual_norm_fwd);
  m.def("dropout", &dropout);
  m.def("residual_norm_grad", &residual_norm_grad);
  m.def("dropout_grad", &dropout_grad);
}

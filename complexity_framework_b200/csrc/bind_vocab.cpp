// Python bindings of the cross-entropy over the vocabulary (vocab_loss.cu).
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>

#include "vocab_loss.h"

int* cfb_err_ptr(int device);
int cfb_num_sms(int device);
torch::autograd::variable_list cfb_once_differentiable(torch::autograd::variable_list grads);

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

Tensor empty(at::IntArrayRef sizes, torch::ScalarType dtype, const Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

// A bf16 matrix of contiguous, 16-byte-aligned rows; other layouts are copied.
Tensor matrix(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_TYPE(t.scalar_type() == torch::kBFloat16, name, " must be bfloat16, got ",
                   t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 2, name, " must be 2-D");
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0 ? c.clone() : c;
}
__nv_bfloat16* bf(const Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }

void check_rc(int rc) {
  TORCH_CHECK(rc == 0, "vocab_loss failed with code ", rc, " ",
              rc > 0 && rc < 1000 ? cudaGetErrorString(static_cast<cudaError_t>(rc)) : "");
}

cfb::VlCall call_of(int64_t T, const Tensor& w, double scale, double smooth, double z,
                    int64_t ignore) {
  TORCH_CHECK_VALUE(T <= (1 << 30) && w.size(0) >= 1 && w.size(0) <= (1 << 30),
                    "too many rows or words");
  TORCH_CHECK_VALUE(w.size(1) >= 8 && w.size(1) % 8 == 0 && w.size(1) <= (1 << 20),
                    "the hidden size must be a multiple of 8, got ", w.size(1));
  TORCH_CHECK_VALUE(scale > 0.0 && std::isfinite(scale), "logit_scale must be positive and finite");
  TORCH_CHECK_VALUE(smooth >= 0.0 && smooth <= 1.0, "label_smoothing must be between 0 and 1");
  TORCH_CHECK_VALUE(z >= 0.0 && std::isfinite(z), "z_loss must not be negative");
  cfb::VlCall c;
  c.T = T;
  c.V = static_cast<int>(w.size(0));
  c.H = static_cast<int>(w.size(1));
  c.scale = static_cast<float>(scale);
  c.smooth = static_cast<float>(smooth);
  c.z = static_cast<float>(z);
  c.ignore = ignore;
  c.w = bf(w);
  c.num_sms = cfb_num_sms(w.get_device());
  c.err = cfb_err_ptr(w.get_device());
  return c;
}

int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// What the backward pass needs, in one buffer: compact rows | lse2 [R] | ginv [1] | cnt [2] |
// target [R] | src [R] | pos [T].  With `base` null, its size in bytes.
int64_t place_saved(cfb::VlCall* c, char* base) {
  const int64_t R = cfb::vl_rows(c->T);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    char* p = base == nullptr ? nullptr : base + at;
    at += up16(bytes);
    return p;
  };
  c->hc = reinterpret_cast<__nv_bfloat16*>(take(R * c->H * 2));
  c->lse2 = reinterpret_cast<float*>(take(4 * R));
  c->ginv = reinterpret_cast<float*>(take(4));
  c->cnt = reinterpret_cast<int*>(take(8));
  c->target = reinterpret_cast<int*>(take(4 * R));
  c->src = reinterpret_cast<int*>(take(4 * R));
  c->pos = reinterpret_cast<int*>(take(4 * c->T));
  return at;
}

// reduction: 0 none (the row losses, times sign), 1 mean over the counted rows, 2 sum.  Returns
// the loss, what the backward pass needs, and the weight as it was read.
std::tuple<Tensor, Tensor, Tensor> vocab_loss_fwd(const Tensor& h_in, const Tensor& w_in,
                                                  const Tensor& y_in, int64_t ignore,
                                                  double smooth, double z, double scale,
                                                  int64_t reduction, double sign, bool save) {
  TORCH_CHECK(w_in.is_cuda(), "weight must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(w_in.device());
  const Tensor h = matrix(h_in, "hidden"), w = matrix(w_in, "weight");
  TORCH_CHECK(h.get_device() == w.get_device() && y_in.is_cuda() &&
                  y_in.get_device() == w.get_device(),
              "hidden, weight and targets must be on one CUDA device");
  TORCH_CHECK_VALUE(h.size(1) == w.size(1), "hidden and weight must have one hidden size");
  TORCH_CHECK_TYPE(y_in.scalar_type() == torch::kInt64, "targets must be int64");
  TORCH_CHECK_VALUE(y_in.dim() == 1 && y_in.size(0) == h.size(0), "targets must be [rows]");
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "bad reduction");
  const Tensor y = y_in.contiguous();
  const int64_t T = h.size(0);
  cfb::VlCall c = call_of(T, w, scale, smooth, z, ignore);
  c.sign = static_cast<float>(sign);
  Tensor out = reduction == 0 ? empty({T}, torch::kFloat32, w) : empty({}, torch::kFloat32, w);
  const int64_t saved_bytes = place_saved(&c, nullptr);
  if (T == 0) {
    if (reduction != 0) out.zero_();
    return {out, empty({saved_bytes}, torch::kUInt8, w), w};
  }
  // without a backward pass what it would need is workspace like the rest
  const int64_t ws_bytes =
      up16(4 * cfb::vl_forward_floats(c)) + (reduction != 0 ? up16(4 * T) : 0);
  Tensor saved = empty({saved_bytes + (save ? 0 : ws_bytes)}, torch::kUInt8, w), ws;
  char* at = static_cast<char*>(saved.data_ptr());
  place_saved(&c, at);
  if (save) {
    ws = empty({ws_bytes}, torch::kUInt8, w);
    at = static_cast<char*>(ws.data_ptr());
  } else {
    at += saved_bytes;
  }
  cfb::VlForward f;
  f.h = bf(h);
  f.targets = y.data_ptr<int64_t>();
  f.mean = reduction == 1;
  f.ws = reinterpret_cast<float*>(at);
  f.rows = reduction == 0 ? out.data_ptr<float>()
                          : reinterpret_cast<float*>(at + up16(4 * cfb::vl_forward_floats(c)));
  if (reduction != 0) f.total = out.data_ptr<float>();
  check_rc(cfb::vl_forward(c, f, at::cuda::getCurrentCUDAStream()));
  return {out, saved, w};
}

// (dhidden [T, H], dweight [V, H]), each where it is needed.
std::tuple<OptTensor, OptTensor> vocab_loss_bwd(const Tensor& gout_in, const Tensor& saved,
                                                const Tensor& w, int64_t T, double smooth, double z,
                                                double scale, bool per_row, double sign,
                                                bool need_h, bool need_w,
                                                int64_t workspace_bytes) {
  const c10::cuda::CUDAGuard guard(w.device());
  cfb::VlCall c = call_of(T, w, scale, smooth, z, 0);
  c.sign = static_cast<float>(sign);
  TORCH_CHECK(saved.numel() == place_saved(&c, nullptr), "saved tensors do not match");
  place_saved(&c, static_cast<char*>(saved.data_ptr()));
  OptTensor dh, dw;
  if (need_h) dh = empty({T, c.H}, torch::kBFloat16, w);
  if (need_w) dw = empty({c.V, c.H}, torch::kBFloat16, w);
  if (T == 0 || !(need_h || need_w)) {
    if (dw.has_value()) dw->zero_();
    return {dh, dw};
  }
  TORCH_CHECK(gout_in.is_cuda() && gout_in.get_device() == w.get_device() &&
                  gout_in.scalar_type() == torch::kFloat32 &&
                  gout_in.numel() == (per_row ? T : 1),
              "bad gradient of the loss");
  const Tensor gout = gout_in.contiguous();
  cfb::VlBackward b;
  b.gout = gout.data_ptr<float>();
  b.per_row = per_row;
  cfb::vl_backward_plan(c, workspace_bytes, &b);
  const int64_t R = cfb::vl_rows(T);
  const int64_t dl_bytes = up16(2 * R * b.piece), resid_bytes = up16(4 * R + 4);
  const Tensor ws = empty({dl_bytes + resid_bytes + (need_h ? 4 * cfb::vl_acc_floats(c, b) : 0)},
                          torch::kUInt8, w);
  char* at = static_cast<char*>(ws.data_ptr());
  b.dl = reinterpret_cast<__nv_bfloat16*>(at);
  b.resid = reinterpret_cast<float*>(at + dl_bytes);
  b.alpha = b.resid + R;
  if (need_h) {
    b.acc = reinterpret_cast<float*>(at + dl_bytes + resid_bytes);
    b.dh = bf(*dh);
  }
  if (need_w) b.dw = bf(*dw);
  check_rc(cfb::vl_backward(c, b, at::cuda::getCurrentCUDAStream()));
  return {dh, dw};
}

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// What a backward pass knows beside its tensors.
struct Options {
  int64_t rows = 0;
  double smooth = 0, z = 0, scale = 1, sign = 1;
  bool per_row = false;
  int64_t workspace = 0;
  void put(AutogradContext* ctx) const {
    ctx->saved_data["rows"] = rows;
    ctx->saved_data["smooth"] = smooth;
    ctx->saved_data["z"] = z;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["per_row"] = per_row;
    ctx->saved_data["sign"] = sign;
    ctx->saved_data["workspace"] = workspace;
  }
  static Options of(AutogradContext* ctx) {
    const auto num = [&](const char* key) { return ctx->saved_data[key].toDouble(); };
    Options o;
    o.rows = ctx->saved_data["rows"].toInt();
    o.smooth = num("smooth");
    o.z = num("z");
    o.scale = num("scale");
    o.per_row = ctx->saved_data["per_row"].toBool();
    o.sign = num("sign");
    o.workspace = ctx->saved_data["workspace"].toInt();
    return o;
  }
};

// A part of the saved buffer (see place_saved) as a tensor.
Tensor part(const Tensor& saved, const void* at, int64_t n, torch::ScalarType type) {
  const int64_t first = static_cast<const char*>(at) - static_cast<const char*>(saved.data_ptr());
  return saved.slice(0, first, first + n * static_cast<int64_t>(c10::elementSize(type))).view(type);
}

cfb::VlCall saved_call(const Tensor& saved, const Tensor& w, const Options& o) {
  cfb::VlCall c = call_of(o.rows, w, o.scale, o.smooth, o.z, 0);
  place_saved(&c, static_cast<char*>(saved.data_ptr()));
  return c;
}

// hidden as the forward pass read it, rows that do not count 0.
Tensor hidden_of(const Tensor& saved, const Tensor& w, const Options& o) {
  const cfb::VlCall c = saved_call(saved, w, o);
  const Tensor pos = part(saved, c.pos, o.rows, torch::kInt32).to(torch::kInt64);
  const Tensor compact =
      part(saved, c.hc, cfb::vl_rows(o.rows) * c.H, torch::kBFloat16).view({-1, c.H});
  return compact.index_select(0, pos.clamp_min(0)).masked_fill_((pos < 0).unsqueeze(1), 0);
}

// The gradients in ATen operations, 32 bits, with all logits: what their own derivatives are taken
// of.
std::pair<Tensor, Tensor> plain_gradients(const Tensor& gout, const Tensor& h, const Tensor& w,
                                          const Tensor& saved, const Options& o) {
  const cfb::VlCall c = saved_call(saved, w, o);
  const Tensor pos = part(saved, c.pos, o.rows, torch::kInt32).to(torch::kInt64);
  const Tensor on = (pos >= 0).unsqueeze(1);
  const Tensor target = part(saved, c.target, cfb::vl_rows(o.rows), torch::kInt32)
                            .to(torch::kInt64)
                            .index_select(0, pos.clamp_min(0))
                            .clamp_min(0)
                            .unsqueeze(1);
  const Tensor hf = h.to(torch::kFloat32).masked_fill(~on, 0), wf = w.to(torch::kFloat32);
  const Tensor z = at::matmul(hf, wf.t()) * o.scale;
  const Tensor lse = z.logsumexp({1}, true);
  Tensor g = o.per_row ? gout.unsqueeze(1)
                       : (gout * part(saved, c.ginv, 1, torch::kFloat32)).expand({o.rows, 1});
  g = (g * (o.sign * o.scale)).masked_fill(~on, 0);
  Tensor dz = (z - lse).exp() * (1 + 2 * o.z * lse) - o.smooth / static_cast<double>(c.V);
  dz = (g * dz).scatter_add(1, target, -(1 - o.smooth) * g);
  return {at::matmul(dz, wf).to(h.scalar_type()), at::matmul(dz.t(), hf).to(w.scalar_type())};
}

// The gradients as a function of the loss's gradient, hidden and weight: the kernels' values, and
// derivatives from plain_gradients.
struct VocabLossGradNode : torch::autograd::Function<VocabLossGradNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gout, const Tensor& h,
                               const Tensor& w, const Tensor& saved, const Options& o, bool need_h,
                               bool need_w) {
    ctx->save_for_backward({gout, h, w, saved});
    o.put(ctx);
    ctx->saved_data["need_h"] = need_h;
    ctx->saved_data["need_w"] = need_w;
    ctx->set_materialize_grads(false);
    const auto grads = vocab_loss_bwd(gout, saved, w, o.rows, o.smooth, o.z, o.scale, o.per_row,
                                      o.sign, need_h, need_w, o.workspace);
    variable_list out;
    if (need_h) out.push_back(*std::get<0>(grads));
    if (need_w) out.push_back(*std::get<1>(grads));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const Options o = Options::of(ctx);
    const bool need_h = ctx->saved_data["need_h"].toBool(),
               need_w = ctx->saved_data["need_w"].toBool(), again = at::GradMode::is_enabled();
    auto saved = ctx->get_saved_variables();
    variable_list out(7), outputs, factors, inputs;
    std::vector<int> which;
    at::AutoGradMode on(true);
    for (int i = 0; i < 3; ++i) {
      if (!ctx->needs_input_grad(i)) continue;
      if (!again) saved[i] = saved[i].detach().requires_grad_();
      inputs.push_back(saved[i]);
      which.push_back(i);
    }
    const auto grads = plain_gradients(saved[0], saved[1], saved[2], saved[3], o);
    const auto take = [&](const Tensor& value, const Tensor& factor) {
      if (!factor.defined()) return;
      outputs.push_back(value);
      factors.push_back(factor);
    };
    if (need_h) take(grads.first, up[0]);
    if (need_w) take(grads.second, up[need_h ? 1 : 0]);
    if (outputs.empty() || inputs.empty()) return out;
    const auto got = torch::autograd::grad(outputs, inputs, factors, again, again, true);
    for (size_t k = 0; k < which.size(); ++k) out[which[k]] = got[k];
    return out;
  }
};

struct VocabLossNode : torch::autograd::Function<VocabLossNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& y,
                        int64_t ignore, double smooth, double z, double scale, int64_t reduction,
                        double sign, int64_t workspace_bytes) {
    auto [loss, saved, read] = vocab_loss_fwd(h, w, y, ignore, smooth, z, scale, reduction, sign,
                                              true);
    // the caller's weight itself where it was read in place, so that a change to it before the
    // backward pass is noticed
    ctx->save_for_backward({saved, read.data_ptr() == w.data_ptr() ? w : read});
    Options o;
    o.rows = h.size(0);
    o.smooth = smooth;
    o.z = z;
    o.scale = scale;
    o.sign = sign;
    o.per_row = reduction == 0;
    o.workspace = workspace_bytes;
    o.put(ctx);
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gout) {
    const auto v = ctx->get_saved_variables();
    const Options o = Options::of(ctx);
    const bool need_h = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    variable_list out(10);
    // under create_graph the engine runs this node; a node that is called by itself is not known
    const auto node = std::dynamic_pointer_cast<torch::autograd::CppNode<VocabLossNode>>(
        torch::autograd::get_current_node());
    if (!at::GradMode::is_enabled() || o.rows == 0 || node == nullptr) {
      const auto grads =
          vocab_loss_bwd(gout[0].detach(), v[0], v[1].detach(), o.rows, o.smooth, o.z, o.scale,
                         o.per_row, o.sign, need_h, need_w, o.workspace);
      if (std::get<0>(grads).has_value()) out[0] = *std::get<0>(grads);
      if (std::get<1>(grads).has_value()) out[1] = *std::get<1>(grads);
      return cfb_once_differentiable(std::move(out));
    }
    // The gradients stay part of the graph: hidden, and a weight that was copied, take the edges
    // of the call's own tensors.
    const auto joined = [&](Tensor t, int i) {
      const auto edge = node->next_edge(i);
      if (edge.is_valid()) torch::autograd::impl::set_gradient_edge(t, edge);
      return t;
    };
    Tensor h, w = v[1];
    {
      at::NoGradGuard no_grad;
      h = hidden_of(v[0], w, o);
      if (need_w && !w.requires_grad()) w = w.clone();
    }
    h = joined(h, 0);
    if (need_w && !w.requires_grad()) w = joined(w, 1);
    const auto grads = VocabLossGradNode::apply(gout[0], h, w, v[0], o, need_h, need_w);
    size_t k = 0;
    if (need_h) out[0] = grads[k++];
    if (need_w) out[1] = grads[k++];
    return out;
  }
};

// The loss alone, with its gradient where `grad` asks for it.
Tensor vocab_loss(const Tensor& h, const Tensor& w, const Tensor& y, int64_t ignore, double smooth,
                  double z, double scale, int64_t reduction, double sign, int64_t workspace_bytes,
                  bool grad) {
  if (grad)
    return VocabLossNode::apply(h, w, y, ignore, smooth, z, scale, reduction, sign,
                                workspace_bytes);
  return std::get<0>(vocab_loss_fwd(h, w, y, ignore, smooth, z, scale, reduction, sign, false));
}

}  // namespace

void register_vocab(pybind11::module& m) { m.def("vocab_loss", &vocab_loss); }

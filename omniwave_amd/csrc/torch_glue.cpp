// Calls of the small operators (norms, cross-entropy) with their autograd nodes, and the optimizer's look at
// hundreds of tensors a step, as the Python module omniwave_amd._glue: host code only, over the C ABI of
// libomniwave_amd.
//
// Why: a small launch takes 4 us on the GPU, and the same call through a Python autograd function costs its
// caller 90 (cross-entropy) to 145 us (norms), most of it Python that runs cold on autograd's thread.  Here
// the node is native.  A function returns None for inputs outside its plain case (other types, shapes,
// devices, copies to make): the caller then takes the operator of torch.library, which checks everything and
// says what is wrong.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>
#include <string>
#include <utility>
#include <vector>

#include "omniwave_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxChannels = 8192;  // of the norm kernels

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc, const char* what) {
  if (rc == OW_OK) return;
  const std::string text = std::string(what) + " failed (status " + std::to_string(rc) + "): " + ow_last_error();
  if (rc == OW_ERR_INVALID) TORCH_CHECK_VALUE(false, text);
  TORCH_CHECK(false, text);
}

int32_t dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return OW_DTYPE_F32;
    case at::kBFloat16: return OW_DTYPE_BF16;
    case at::kHalf: return OW_DTYPE_F16;
    default: return -1;
  }
}

// Whether a GPU is one that the kernels are built for (looked up once per device).
bool device_ok(const Tensor& t) {
  static int8_t known[64] = {0};
  const int i = t.device().index();
  if (i < 0 || i >= 64) return false;
  if (known[i] == 0) {
    hipDeviceProp_t p;
    known[i] = hipGetDeviceProperties(&p, i) == hipSuccess && std::strncmp(p.gcnArchName, "gfx950", 6) == 0 ? 1 : -1;
  }
  return known[i] == 1;
}

// A strided GPU tensor of one of the kernels' types, without storage tricks (conjugate, negative, nested).
bool plain(const Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && dtype_code(t) >= 0 && !t.is_neg() && !t.is_nested();
}

// Distance between rows (the last dimension) that lie at one distance, value after value; -1: they do not.
int64_t row_stride(const Tensor& t) {
  const int64_t c = t.size(-1);
  if (t.is_contiguous()) return c;
  if (c != 1 && t.stride(-1) != 1) return -1;
  int64_t step = -1, span = 0;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (step < 0) {
      step = t.stride(d);
      span = step * t.size(d);
    } else if (t.stride(d) == span) {
      span *= t.size(d);
    } else {
      return -1;
    }
  }
  return step < 0 ? c : step;
}

Tensor rows_of(const Tensor& t, int64_t* stride) {
  *stride = row_stride(t);
  if (*stride >= 0) return t;
  *stride = t.size(-1);
  return t.contiguous();
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor like(const Tensor& t) { return at::empty_like(t, at::MemoryFormat::Contiguous); }

// Hooks on saved tensors may hand out others than were saved: a kernel gets only what fits.
void check_unpacked(bool ok) {
  TORCH_CHECK_VALUE(ok, "a saved tensor has come back to the backward with another type, shape or device");
}

// The gradients of a function that can be differentiated once: an error where they are differentiated again.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) defined.push_back(g);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int>(defined.size()));
  for (Tensor& g : defined) g = g.detach().requires_grad_(true);
  variable_list marked = (*node)(std::move(defined));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[k++];
  return grads;
}

// ---------------------------------------------------------------------------------------
// Norms around a block

struct Norms {
  Tensor x, delta, post, gate, scale, next;
  double eps = 0.0;
};

OwBlockNorms descriptor(const Norms& n) {
  OwBlockNorms d{};
  const int64_t c = n.x.size(-1);
  d.rows = n.x.numel() / c;
  d.rows_per_image = d.rows / n.x.size(0);
  d.x_stride = row_stride(n.x);
  d.delta_stride = n.delta.defined() ? row_stride(n.delta) : 0;
  d.x = ptr(n.x);
  d.delta = ptr(n.delta);
  d.post_weight = ptr(n.post);
  d.gate = ptr(n.gate);
  d.scale = static_cast<const float*>(ptr(n.scale));
  d.next_weight = ptr(n.next);
  d.channels = static_cast<int32_t>(c);
  d.dtype = dtype_code(n.x);
  d.post_dtype = n.post.defined() ? dtype_code(n.post) : 0;
  d.gate_dtype = n.gate.defined() ? dtype_code(n.gate) : 0;
  d.next_dtype = n.next.defined() ? dtype_code(n.next) : 0;
  d.gate_per_image = n.gate.defined() && n.gate.dim() == 2;
  d.eps = static_cast<float>(n.eps);
  return d;
}

bool weight_ok(const Tensor& w, const Tensor& x, bool per_image) {
  if (!w.defined()) return true;
  const int64_t c = x.size(-1);
  const bool shape = w.dim() == 1 ? w.size(0) == c : per_image && w.dim() == 2 && w.size(0) == x.size(0) && w.size(1) == c;
  return shape && plain(w) && w.device() == x.device() && w.is_contiguous();
}

bool plain_case(const Norms& n) {
  const Tensor& x = n.x;
  if (!x.defined() || !plain(x) || x.dim() < 2 || x.numel() == 0 || !device_ok(x)) return false;
  const int64_t c = x.size(-1);
  if (c > kMaxChannels || x.numel() / c >= (int64_t(1) << 31) || row_stride(x) < 0) return false;
  if (!(n.eps >= 0.0) || !std::isfinite(n.eps)) return false;
  if (n.delta.defined()) {
    if (!plain(n.delta) || n.delta.scalar_type() != x.scalar_type() || n.delta.device() != x.device() ||
        n.delta.sizes() != x.sizes() || row_stride(n.delta) < 0)
      return false;
  } else if (n.post.defined() || n.gate.defined() || n.scale.defined() || !n.next.defined()) {
    return false;
  }
  if (!weight_ok(n.post, x, false) || !weight_ok(n.gate, x, true) || !weight_ok(n.next, x, false)) return false;
  if (n.scale.defined() &&
      (!plain(n.scale) || n.scale.scalar_type() != at::kFloat || n.scale.device() != x.device() || n.scale.dim() != 1 ||
       n.scale.size(0) != x.size(0) || !n.scale.is_contiguous() || n.scale.requires_grad()))
    return false;
  return true;
}

variable_list run_norms(const Norms& n) {
  const c10::DeviceGuard guard(n.x.device());
  Tensor out = n.delta.defined() ? like(n.x) : Tensor();
  Tensor next = n.next.defined() ? like(n.x) : Tensor();
  const OwBlockNorms d = descriptor(n);
  check(ow_block_norms_fwd(&d, out_ptr(out), out_ptr(next), stream_of(n.x)), "ow_block_norms_fwd");
  variable_list outs;
  if (out.defined()) outs.push_back(std::move(out));
  if (next.defined()) outs.push_back(std::move(next));
  return outs;
}

class NormsNode : public torch::autograd::Function<NormsNode> {
 public:
  typedef std::optional<Tensor> Given;
  static Given given(const Tensor& t) { return t.defined() ? Given(t) : Given(); }

  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Given& delta, const Given& post,
                               const Given& gate, const Given& scale, const Given& next, double eps) {
    const auto or_none = [](const Given& t) { return t.has_value() ? *t : Tensor(); };
    const Norms n{x, or_none(delta), or_none(post), or_none(gate), or_none(scale), or_none(next), eps};
    ctx->save_for_backward({n.x, n.delta, n.post, n.gate, n.scale, n.next});
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return run_norms(n);
  }

  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    const variable_list s = ctx->get_saved_variables();
    Norms n{s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["eps"].toDouble()};
    check_unpacked(n.x.is_cuda());
    const c10::DeviceGuard guard(n.x.device());
    const bool has_out = n.delta.defined();
    Tensor dout = has_out ? ups[0] : Tensor(), dnext = n.next.defined() ? ups[has_out ? 1 : 0] : Tensor();
    for (Tensor* g : {&dout, &dnext})  // a gradient may stand for its negative (the imaginary part of a conjugate)
      if (g->defined()) *g = g->resolve_neg();
    // Hooks on saved tensors may hand out copies that lie otherwise.
    int64_t unused = 0, out_stride = 0, next_stride = 0;
    n.x = rows_of(n.x, &unused);
    if (has_out) n.delta = rows_of(n.delta, &unused);
    for (Tensor* w : {&n.post, &n.gate, &n.scale, &n.next})
      if (w->defined()) *w = w->contiguous();
    const auto fits = [&](const Tensor& g) {
      return !g.defined() || (plain(g) && g.sizes() == n.x.sizes() && g.scalar_type() == n.x.scalar_type() &&
                              g.device() == n.x.device());
    };
    check_unpacked(plain_case(n) && fits(dout) && fits(dnext));
    if (dout.defined()) dout = rows_of(dout, &out_stride);
    if (dnext.defined()) dnext = rows_of(dnext, &next_stride);

    // needs_input_grad counts the tensors that were given.
    const Tensor* inputs[6] = {&n.x, &n.delta, &n.post, &n.gate, &n.scale, &n.next};
    Tensor grads[6];
    size_t edge = 0;
    for (int i = 0; i < 6; ++i) {
      if (!inputs[i]->defined()) continue;
      if (ctx->needs_input_grad(edge++) && i != 4) grads[i] = like(*inputs[i]);
    }
    const bool any = dout.defined() || dnext.defined();
    if (!any || (grads[5].defined() && !dnext.defined())) {
      for (Tensor& g : grads)
        if (g.defined() && (!any || &g == &grads[5])) g.zero_();
    }
    if (any) {
      const OwBlockNorms d = descriptor(n);
      void* next_weight_grad = dnext.defined() ? out_ptr(grads[5]) : nullptr;
      size_t bytes = 0;
      Tensor workspace;
      if (grads[2].defined() || grads[3].defined() || next_weight_grad != nullptr) {
        bytes = ow_block_norms_bwd_workspace(&d);
        if (bytes) workspace = at::empty({static_cast<int64_t>(bytes)}, n.x.options().dtype(at::kByte));
      }
      check(ow_block_norms_bwd(&d, ptr(dout), out_stride, ptr(dnext), next_stride, out_ptr(grads[0]), out_ptr(grads[1]),
                               out_ptr(grads[2]), out_ptr(grads[3]), next_weight_grad, out_ptr(workspace), bytes,
                               stream_of(n.x)),
            "ow_block_norms_bwd");
    }
    return once({grads[0], grads[1], grads[2], grads[3], Tensor(), grads[5], Tensor()});
  }
};

// ---------------------------------------------------------------------------------------
// Layer norm

struct LayerNorm {
  Tensor x, weight, bias;
  double eps = 0.0;
};

OwLayerNorm descriptor(const LayerNorm& n) {
  OwLayerNorm d{};
  d.channels = static_cast<int32_t>(n.x.size(-1));
  d.rows = n.x.numel() / d.channels;
  d.x_stride = row_stride(n.x);
  d.x = ptr(n.x);
  d.weight = ptr(n.weight);
  d.bias = ptr(n.bias);
  d.dtype = dtype_code(n.x);
  d.weight_dtype = n.weight.defined() ? dtype_code(n.weight) : 0;
  d.bias_dtype = n.bias.defined() ? dtype_code(n.bias) : 0;
  d.eps = static_cast<float>(n.eps);
  return d;
}

bool plain_case(const LayerNorm& n) {
  const Tensor& x = n.x;
  if (!x.defined() || !plain(x) || x.dim() < 1 || x.numel() == 0 || !device_ok(x)) return false;
  const int64_t c = x.size(-1);
  if (c > kMaxChannels || x.numel() / c >= (int64_t(1) << 31) || row_stride(x) < 0) return false;
  return n.eps >= 0.0 && std::isfinite(n.eps) && weight_ok(n.weight, x, false) && weight_ok(n.bias, x, false);
}

Tensor run_layer_norm(const LayerNorm& n) {
  const c10::DeviceGuard guard(n.x.device());
  Tensor y = like(n.x);
  const OwLayerNorm d = descriptor(n);
  check(ow_layer_norm_fwd(&d, out_ptr(y), stream_of(n.x)), "ow_layer_norm_fwd");
  return y;
}

class LayerNormNode : public torch::autograd::Function<LayerNormNode> {
 public:
  typedef std::optional<Tensor> Given;

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Given& weight, const Given& bias, double eps) {
    const LayerNorm n{x, weight.value_or(Tensor()), bias.value_or(Tensor()), eps};
    ctx->save_for_backward({n.x, n.weight, n.bias});
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return run_layer_norm(n);
  }

  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    if (!ups[0].defined()) return variable_list(4);
    const variable_list s = ctx->get_saved_variables();
    LayerNorm n{s[0], s[1], s[2], ctx->saved_data["eps"].toDouble()};
    check_unpacked(n.x.is_cuda());
    const c10::DeviceGuard guard(n.x.device());
    int64_t unused = 0, dy_stride = 0;
    n.x = rows_of(n.x, &unused);
    for (Tensor* w : {&n.weight, &n.bias})
      if (w->defined()) *w = w->contiguous();
    Tensor dy = ups[0].resolve_neg();
    check_unpacked(plain_case(n) && plain(dy) && dy.sizes() == n.x.sizes() && dy.scalar_type() == n.x.scalar_type() &&
                   dy.device() == n.x.device());
    dy = rows_of(dy, &dy_stride);
    // needs_input_grad counts the tensors that were given.
    const Tensor* inputs[3] = {&n.x, &n.weight, &n.bias};
    Tensor grads[3];
    size_t edge = 0;
    bool any = false;
    for (int i = 0; i < 3; ++i)
      if (inputs[i]->defined() && ctx->needs_input_grad(edge++)) grads[i] = like(*inputs[i]), any = true;
    if (any) {
      const OwLayerNorm d = descriptor(n);
      size_t bytes = 0;
      Tensor workspace;
      if (grads[1].defined() || grads[2].defined()) {
        bytes = ow_layer_norm_bwd_workspace(&d);
        if (bytes) workspace = at::empty({static_cast<int64_t>(bytes)}, n.x.options().dtype(at::kByte));
      }
      check(ow_layer_norm_bwd(&d, ptr(dy), dy_stride, out_ptr(grads[0]), out_ptr(grads[1]), out_ptr(grads[2]),
                              out_ptr(workspace), bytes, stream_of(n.x)),
            "ow_layer_norm_bwd");
    }
    return once({grads[0], grads[1], grads[2], Tensor()});
  }
};

// ---------------------------------------------------------------------------------------
// Cross-entropy

struct Xent {
  Tensor logits, target, target_b, mix;
  double mix_value = 1.0, smoothing = 0.0;
  int64_t ignore_index = -100;
  int32_t reduction = OW_REDUCE_MEAN;
};

OwCrossEntropy descriptor(const Xent& e) {
  OwCrossEntropy d{};
  d.rows = e.target.numel();
  d.classes = e.logits.size(-1);
  d.row_stride = row_stride(e.logits);
  d.ignore_index = e.ignore_index;
  d.logits = ptr(e.logits);
  d.target = static_cast<const int64_t*>(ptr(e.target));
  d.target_b = static_cast<const int64_t*>(ptr(e.target_b));
  d.mix = static_cast<const float*>(ptr(e.mix));
  d.mix_value = static_cast<float>(e.mix_value);
  d.smoothing = static_cast<float>(e.smoothing);
  d.dtype = dtype_code(e.logits);
  d.reduction = e.reduction;
  return d;
}

bool labels_ok(const Tensor& t, const Tensor& logits) {
  return t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == at::kLong && t.device() == logits.device() &&
         t.sizes() == logits.sizes().slice(0, logits.dim() - 1) && t.is_contiguous();
}

bool plain_case(const Xent& e) {
  const Tensor& x = e.logits;
  if (!x.defined() || !e.target.defined() || !plain(x) || x.dim() < 1 || x.numel() == 0 || !device_ok(x)) return false;
  const int64_t c = x.size(-1);
  if (c >= (int64_t(1) << 30) || x.numel() / c >= (int64_t(1) << 31) || row_stride(x) < 0) return false;
  if (!(e.smoothing >= 0.0 && e.smoothing <= 1.0) || !(e.mix_value >= 0.0 && e.mix_value <= 1.0)) return false;
  if (!labels_ok(e.target, x) || (e.target_b.defined() && !labels_ok(e.target_b, x))) return false;
  if (e.mix.defined() &&
      (!e.target_b.defined() || !plain(e.mix) || e.mix.scalar_type() != at::kFloat || e.mix.device() != x.device() ||
       e.mix.sizes() != e.target.sizes() || !e.mix.is_contiguous() || e.mix.requires_grad()))
    return false;
  return true;
}

// The loss (or the rows' losses), and what the backward needs: the rows' statistics, a row's weight in the
// loss and, with a reduction, the losses.
std::pair<Tensor, Tensor> run_xent(const Xent& e) {
  const c10::DeviceGuard guard(e.logits.device());
  const OwCrossEntropy d = descriptor(e);
  const bool reduced = e.reduction != OW_REDUCE_NONE;
  const auto f32 = e.logits.options().dtype(at::kFloat);
  Tensor aux = at::empty({2 * d.rows + 1 + (reduced ? d.rows : 0)}, f32);
  Tensor loss = reduced ? at::empty({}, f32) : at::empty(e.target.sizes(), f32);
  const size_t bytes = ow_cross_entropy_workspace(&d);
  Tensor workspace = bytes ? at::empty({static_cast<int64_t>(bytes)}, f32.dtype(at::kByte)) : Tensor();
  float* stats = static_cast<float*>(out_ptr(aux));
  float* weight = stats + 2 * d.rows;
  float* out = static_cast<float*>(out_ptr(loss));
  check(ow_cross_entropy_fwd(&d, stats, reduced ? weight + 1 : out, reduced ? out : nullptr, reduced ? weight : nullptr,
                             out_ptr(workspace), bytes, stream_of(e.logits)),
        "ow_cross_entropy_fwd");
  return {std::move(loss), std::move(aux)};
}

class XentNode : public torch::autograd::Function<XentNode> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Xent& e) {
    auto [loss, aux] = run_xent(e);
    ctx->save_for_backward({logits, e.target, e.target_b, e.mix, aux});
    ctx->saved_data["mix"] = e.mix_value;
    ctx->saved_data["smoothing"] = e.smoothing;
    ctx->saved_data["ignore"] = e.ignore_index;
    ctx->saved_data["reduction"] = static_cast<int64_t>(e.reduction);
    ctx->set_materialize_grads(false);
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    if (!ups[0].defined()) return {Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    Xent e{s[0], s[1], s[2], s[3], ctx->saved_data["mix"].toDouble(), ctx->saved_data["smoothing"].toDouble(),
           ctx->saved_data["ignore"].toInt(), static_cast<int32_t>(ctx->saved_data["reduction"].toInt())};
    check_unpacked(e.logits.is_cuda());
    const c10::DeviceGuard guard(e.logits.device());
    int64_t unused = 0;  // hooks on saved tensors may hand out copies that lie otherwise
    e.logits = rows_of(e.logits, &unused);
    for (Tensor* t : {&e.target, &e.target_b, &e.mix})
      if (t->defined()) *t = t->contiguous();
    const Tensor aux = s[4].contiguous(), up = ups[0].resolve_neg().to(at::kFloat).contiguous();
    const bool reduced = e.reduction != OW_REDUCE_NONE;
    const int64_t rows = e.target.numel();
    check_unpacked(plain_case(e) && plain(aux) && aux.scalar_type() == at::kFloat && aux.device() == e.logits.device() &&
                   aux.numel() == 2 * rows + 1 + (reduced ? rows : 0) && plain(up) && up.device() == e.logits.device() &&
                   up.numel() == (reduced ? 1 : rows));
    Tensor grad = like(e.logits);
    const OwCrossEntropy d = descriptor(e);
    const float* stats = static_cast<const float*>(ptr(aux));
    check(ow_cross_entropy_bwd(&d, stats, reduced ? stats + 2 * d.rows : nullptr,
                               static_cast<const float*>(ptr(up)), out_ptr(grad), stream_of(e.logits)),
          "ow_cross_entropy_bwd");
    return once({std::move(grad), Tensor()});
  }
};

// ---------------------------------------------------------------------------------------
// Distillation

struct Distill {
  Tensor logits, teacher, indices;
  double temperature = 1.0;
  int64_t ignore_index = -100;
  int32_t reduction = OW_REDUCE_MEAN;
};

OwDistillation descriptor(const Distill& e) {
  OwDistillation d{};
  d.classes = e.logits.size(-1);
  d.rows = e.logits.numel() / d.classes;
  d.row_stride = row_stride(e.logits);
  d.ignore_index = e.ignore_index;
  d.logits = ptr(e.logits);
  d.teacher = ptr(e.teacher);
  d.indices = static_cast<const int64_t*>(ptr(e.indices));
  d.top = static_cast<int32_t>(e.teacher.size(-1));
  d.dtype = dtype_code(e.logits);
  d.teacher_dtype = dtype_code(e.teacher);
  d.reduction = e.reduction;
  d.temperature = static_cast<float>(e.temperature);
  return d;
}

constexpr int64_t kMaxEntries = 1 << 16;  // of the distillation kernels

bool plain_case(const Distill& e) {
  const Tensor& x = e.logits;
  if (!x.defined() || !e.teacher.defined() || !e.indices.defined()) return false;
  if (!plain(x) || x.dim() < 1 || x.numel() == 0 || !device_ok(x)) return false;
  const int64_t c = x.size(-1);
  if (c >= (int64_t(1) << 30) || x.numel() / c >= (int64_t(1) << 31) || row_stride(x) < 0) return false;
  const Tensor &t = e.teacher, &i = e.indices;
  if (!plain(t) || t.device() != x.device() || t.dim() != x.dim() || t.size(-1) > kMaxEntries || !t.is_contiguous() ||
      t.requires_grad() || t.sizes().slice(0, t.dim() - 1) != x.sizes().slice(0, x.dim() - 1))
    return false;
  if (!i.is_cuda() || i.layout() != at::kStrided || i.scalar_type() != at::kLong || i.device() != x.device() ||
      i.sizes() != t.sizes() || !i.is_contiguous())
    return false;
  return e.temperature >= 1e-15 && e.temperature <= 1e15;
}

// The loss (or the rows' losses), and what the backward needs: the rows' statistics, a row's weight in the
// loss and, with a reduction, the losses.
std::pair<Tensor, Tensor> run_distill(const Distill& e) {
  const c10::DeviceGuard guard(e.logits.device());
  const OwDistillation d = descriptor(e);
  const bool reduced = e.reduction != OW_REDUCE_NONE;
  const auto f32 = e.logits.options().dtype(at::kFloat);
  Tensor aux = at::empty({4 * d.rows + 1 + (reduced ? d.rows : 0)}, f32);
  Tensor loss = reduced ? at::empty({}, f32) : at::empty(e.logits.sizes().slice(0, e.logits.dim() - 1), f32);
  const size_t bytes = ow_distillation_workspace(&d);
  Tensor workspace = bytes ? at::empty({static_cast<int64_t>(bytes)}, f32.dtype(at::kByte)) : Tensor();
  float* stats = static_cast<float*>(out_ptr(aux));
  float* weight = stats + 4 * d.rows;
  float* out = static_cast<float*>(out_ptr(loss));
  check(ow_distillation_fwd(&d, stats, reduced ? weight + 1 : out, reduced ? out : nullptr, reduced ? weight : nullptr,
                            out_ptr(workspace), bytes, stream_of(e.logits)),
        "ow_distillation_fwd");
  return {std::move(loss), std::move(aux)};
}

class DistillNode : public torch::autograd::Function<DistillNode> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Distill& e) {
    auto [loss, aux] = run_distill(e);
    ctx->save_for_backward({logits, e.teacher, e.indices, aux});
    ctx->saved_data["temperature"] = e.temperature;
    ctx->saved_data["ignore"] = e.ignore_index;
    ctx->saved_data["reduction"] = static_cast<int64_t>(e.reduction);
    ctx->set_materialize_grads(false);
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    if (!ups[0].defined()) return {Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    Distill e{s[0], s[1], s[2], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["ignore"].toInt(),
              static_cast<int32_t>(ctx->saved_data["reduction"].toInt())};
    check_unpacked(e.logits.is_cuda());
    const c10::DeviceGuard guard(e.logits.device());
    int64_t unused = 0;  // hooks on saved tensors may hand out copies that lie otherwise
    e.logits = rows_of(e.logits, &unused);
    e.teacher = e.teacher.detach().contiguous();
    e.indices = e.indices.contiguous();
    const Tensor aux = s[3].contiguous(), up = ups[0].resolve_neg().to(at::kFloat).contiguous();
    const bool reduced = e.reduction != OW_REDUCE_NONE;
    check_unpacked(plain_case(e));
    const OwDistillation d = descriptor(e);
    check_unpacked(plain(aux) && aux.scalar_type() == at::kFloat && aux.device() == e.logits.device() &&
                   aux.numel() == 4 * d.rows + 1 + (reduced ? d.rows : 0) && plain(up) &&
                   up.device() == e.logits.device() && up.numel() == (reduced ? 1 : d.rows));
    Tensor grad = like(e.logits);
    const float* stats = static_cast<const float*>(ptr(aux));
    check(ow_distillation_bwd(&d, stats, reduced ? stats + 4 * d.rows : nullptr, static_cast<const float*>(ptr(up)),
                              out_ptr(grad), stream_of(e.logits)),
          "ow_distillation_bwd");
    return once({std::move(grad), Tensor()});
  }
};

// ---------------------------------------------------------------------------------------
// Gated feed-forward product

struct Gated {
  Tensor x, gate, up;
};

constexpr int64_t kMaxWidth = 1 << 20;  // channels, hidden

OwGatedLinear descriptor(const Gated& g) {
  OwGatedLinear d{};
  d.channels = static_cast<int32_t>(g.x.size(-1));
  d.rows = g.x.numel() / d.channels;
  d.x_stride = row_stride(g.x);
  d.x = ptr(g.x);
  d.gate_weight = ptr(g.gate);
  d.up_weight = ptr(g.up);
  d.hidden = static_cast<int32_t>(g.gate.size(0));
  d.dtype = dtype_code(g.x);
  return d;
}

bool plain_case(const Gated& g) {
  const Tensor& x = g.x;
  if (!x.defined() || !g.gate.defined() || !g.up.defined()) return false;
  if (!plain(x) || x.dim() < 1 || x.numel() == 0 || !device_ok(x) || row_stride(x) < 0) return false;
  const int64_t c = x.size(-1);
  if (c > kMaxWidth || x.numel() / c >= (int64_t(1) << 31)) return false;
  for (const Tensor* w : {&g.gate, &g.up})
    if (!plain(*w) || w->scalar_type() != x.scalar_type() || w->device() != x.device() || w->dim() != 2 || w->size(1) != c ||
        w->size(0) != g.gate.size(0) || w->size(0) < 1 || w->size(0) > kMaxWidth || !w->is_contiguous())
      return false;
  return true;
}

std::vector<int64_t> hidden_shape(const Gated& g) {
  std::vector<int64_t> shape = g.x.sizes().vec();
  shape.back() = g.gate.size(0);
  return shape;
}

// The result, and with `keep` what the backward needs beside the inputs (both products, or nothing).
std::pair<Tensor, Tensor> run_gated(const Gated& g, bool keep) {
  const c10::DeviceGuard guard(g.x.device());
  Tensor h = at::empty(hidden_shape(g), g.x.options()), kept;
  const OwGatedLinear d = descriptor(g);
  if (const size_t size = keep ? ow_gated_linear_kept(&d) : 0)
    kept = at::empty({static_cast<int64_t>(size / sizeof(float))}, g.x.options().dtype(at::kFloat));
  const size_t bytes = ow_gated_linear_fwd_workspace(&d);
  const Tensor workspace = bytes ? at::empty({static_cast<int64_t>(bytes)}, g.x.options().dtype(at::kByte)) : Tensor();
  check(ow_gated_linear_fwd(&d, out_ptr(h), out_ptr(kept), out_ptr(workspace), bytes, stream_of(g.x)), "ow_gated_linear_fwd");
  return {std::move(h), std::move(kept)};
}

class GatedNode : public torch::autograd::Function<GatedNode> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up) {
    auto [h, kept] = run_gated(Gated{x, gate, up}, true);
    ctx->save_for_backward({x, gate, up, kept});
    ctx->set_materialize_grads(false);
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list ups) {
    if (!ups[0].defined()) return variable_list(3);
    const variable_list s = ctx->get_saved_variables();
    Gated g{s[0], s[1], s[2]};
    check_unpacked(g.x.is_cuda());
    const c10::DeviceGuard guard(g.x.device());
    int64_t unused = 0, dh_stride = 0;  // hooks on saved tensors may hand out copies that lie otherwise
    g.x = rows_of(g.x, &unused);
    g.gate = g.gate.contiguous();
    g.up = g.up.contiguous();
    Tensor dh = ups[0].resolve_neg();
    check_unpacked(plain_case(g) && plain(dh) && dh.sizes() == at::IntArrayRef(hidden_shape(g)) &&
                   dh.scalar_type() == g.x.scalar_type() && dh.device() == g.x.device());
    dh = rows_of(dh, &dh_stride);
    const OwGatedLinear d = descriptor(g);
    Tensor kept = s[3];
    if (kept.defined()) {
      kept = kept.contiguous();
      check_unpacked(plain(kept) && kept.scalar_type() == at::kFloat && kept.device() == g.x.device() &&
                     static_cast<size_t>(kept.numel()) * sizeof(float) == ow_gated_linear_kept(&d));
    }
    const Tensor* inputs[3] = {&g.x, &g.gate, &g.up};
    Tensor grads[3];
    bool any = false;
    for (size_t i = 0; i < 3; ++i)
      if (ctx->needs_input_grad(i)) grads[i] = like(*inputs[i]), any = true;
    if (any) {
      const size_t bytes = ow_gated_linear_bwd_workspace(&d);
      const Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, g.x.options().dtype(at::kByte));
      check(ow_gated_linear_bwd(&d, ptr(kept), ptr(dh), dh_stride, out_ptr(grads[0]), out_ptr(grads[1]), out_ptr(grads[2]),
                                out_ptr(workspace), bytes, stream_of(g.x)),
            "ow_gated_linear_bwd");
    }
    return once({grads[0], grads[1], grads[2]});
  }
};

// ---------------------------------------------------------------------------------------
// The module

// A tensor argument, undefined for None; false: it is neither.
bool as_tensor(PyObject* o, Tensor* t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}

// A number argument; false: it is none (no error is left behind: the caller's checks say what is wrong).
bool as_double(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}
bool as_int(PyObject* o, int64_t* v) {
  *v = PyLong_AsLongLong(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}

PyObject* wrap_or_none(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// norms(x, delta, post_weight, gate, scale, next_weight, eps) -> (out, next) or None
PyObject* py_norms(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 7) {
    PyErr_SetString(PyExc_TypeError, "norms takes 7 arguments");
    return nullptr;
  }
  Norms n;
  Tensor* tensors[6] = {&n.x, &n.delta, &n.post, &n.gate, &n.scale, &n.next};
  bool grad = false;
  for (int i = 0; i < 6; ++i) {
    if (!as_tensor(args[i], tensors[i])) Py_RETURN_NONE;
    grad |= tensors[i]->defined() && tensors[i]->requires_grad();
  }
  if (!as_double(args[6], &n.eps) || !plain_case(n)) Py_RETURN_NONE;
  variable_list outs;
  {
    pybind11::gil_scoped_release no_gil;
    if (grad && at::GradMode::is_enabled()) {
      outs = NormsNode::apply(n.x, NormsNode::given(n.delta), NormsNode::given(n.post), NormsNode::given(n.gate),
                              NormsNode::given(n.scale), NormsNode::given(n.next), n.eps);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      outs = run_norms(n);
    }
  }
  PyObject* out = wrap_or_none(n.delta.defined() ? outs[0] : Tensor());
  PyObject* next = out ? wrap_or_none(n.next.defined() ? outs.back() : Tensor()) : nullptr;
  PyObject* pair = next ? PyTuple_Pack(2, out, next) : nullptr;
  Py_XDECREF(out);
  Py_XDECREF(next);
  return pair;
  END_HANDLE_TH_ERRORS
}

// layer_norm(x, weight, bias, eps) -> y or None
PyObject* py_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 4) {
    PyErr_SetString(PyExc_TypeError, "layer_norm takes 4 arguments");
    return nullptr;
  }
  LayerNorm n;
  Tensor* tensors[3] = {&n.x, &n.weight, &n.bias};
  bool grad = false;
  for (int i = 0; i < 3; ++i) {
    if (!as_tensor(args[i], tensors[i])) Py_RETURN_NONE;
    grad |= tensors[i]->defined() && tensors[i]->requires_grad();
  }
  if (!as_double(args[3], &n.eps) || !plain_case(n)) Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    if (grad && at::GradMode::is_enabled()) {
      y = LayerNormNode::apply(n.x, NormsNode::given(n.weight), NormsNode::given(n.bias), n.eps);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      y = run_layer_norm(n);
    }
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// cross_entropy(logits, target, target_b, mix, mix_value, label_smoothing, ignore_index, reduction) -> loss or None
PyObject* py_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 8) {
    PyErr_SetString(PyExc_TypeError, "cross_entropy takes 8 arguments");
    return nullptr;
  }
  Xent e;
  Tensor* tensors[4] = {&e.logits, &e.target, &e.target_b, &e.mix};
  for (int i = 0; i < 4; ++i)
    if (!as_tensor(args[i], tensors[i])) Py_RETURN_NONE;
  int64_t reduction = 0;
  if (!as_double(args[4], &e.mix_value) || !as_double(args[5], &e.smoothing) || !as_int(args[6], &e.ignore_index) ||
      !as_int(args[7], &reduction))
    Py_RETURN_NONE;
  e.reduction = static_cast<int32_t>(reduction);
  if (!plain_case(e)) Py_RETURN_NONE;
  Tensor loss;
  {
    pybind11::gil_scoped_release no_gil;
    if (e.logits.requires_grad() && at::GradMode::is_enabled()) {
      loss = XentNode::apply(e.logits, e);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      loss = run_xent(e).first;
    }
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// distillation(logits, teacher_logits, teacher_indices, temperature, ignore_index, reduction) -> loss or None
PyObject* py_distillation(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 6) {
    PyErr_SetString(PyExc_TypeError, "distillation takes 6 arguments");
    return nullptr;
  }
  Distill e;
  Tensor* tensors[3] = {&e.logits, &e.teacher, &e.indices};
  for (int i = 0; i < 3; ++i)
    if (!as_tensor(args[i], tensors[i])) Py_RETURN_NONE;
  int64_t reduction = 0;
  if (!as_double(args[3], &e.temperature) || !as_int(args[4], &e.ignore_index) || !as_int(args[5], &reduction)) Py_RETURN_NONE;
  e.reduction = static_cast<int32_t>(reduction);
  if (!plain_case(e)) Py_RETURN_NONE;
  Tensor loss;
  {
    pybind11::gil_scoped_release no_gil;
    if (e.logits.requires_grad() && at::GradMode::is_enabled()) {
      loss = DistillNode::apply(e.logits, e);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      loss = run_distill(e).first;
    }
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// gated_linear(x, gate_weight, up_weight) -> h or None
PyObject* py_gated_linear(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 3) {
    PyErr_SetString(PyExc_TypeError, "gated_linear takes 3 arguments");
    return nullptr;
  }
  Gated g;
  Tensor* tensors[3] = {&g.x, &g.gate, &g.up};
  bool grad = false;
  for (int i = 0; i < 3; ++i) {
    if (!as_tensor(args[i], tensors[i])) Py_RETURN_NONE;
    grad |= tensors[i]->defined() && tensors[i]->requires_grad();
  }
  if (!plain_case(g)) Py_RETURN_NONE;
  Tensor h;
  {
    pybind11::gil_scoped_release no_gil;
    if (grad && at::GradMode::is_enabled()) {
      h = GatedNode::apply(g.x, g.gate, g.up);
    } else {
      at::AutoDispatchBelowADInplaceOrView below;
      h = run_gated(g, false).first;
    }
  }
  return THPVariable_Wrap(h);
  END_HANDLE_TH_ERRORS
}

// Numbers (addresses of tensors and what lies there) as bytes, 8 each, to be compared as a whole.
class Numbers {
 public:
  explicit Numbers(Py_ssize_t n) { of_.reserve(static_cast<size_t>(n)); }
  void add(const void* p) { of_.push_back(reinterpret_cast<int64_t>(p)); }
  void add(int64_t v) { of_.push_back(v); }
  PyObject* bytes() const {
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(of_.data()), static_cast<Py_ssize_t>(of_.size() * 8));
  }

 private:
  std::vector<int64_t> of_;
};

const void* address(const Tensor& t) { return t.has_storage() ? t.const_data_ptr() : nullptr; }

// Where a tensor lies and what lies there: values, dimensions, type and whether they are dense in their order.  Values that stand
// for their negatives are refused: a kernel reads what lies there.
void add_layout(Numbers& found, const Tensor& t) {
  TORCH_CHECK_VALUE(!t.is_neg(), "a parameter or state of shape ", t.sizes(), " is a negated view");
  found.add(address(t));
  const bool dense = t.layout() == at::kStrided && t.is_contiguous();
  found.add(t.numel() << 16 | t.dim() << 9 | int64_t(dense) << 8 | static_cast<int64_t>(t.scalar_type()));
}

// addresses(tensors) -> bytes: where the tensors of a list lie
PyObject* py_addresses(PyObject*, PyObject* list) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(PyList_Check(list), "addresses takes a list");
  const Py_ssize_t n = PyList_GET_SIZE(list);
  Numbers found(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), "addresses takes tensors");
    found.add(address(THPVariable_Unpack(o)));
  }
  return found.bytes();
  END_HANDLE_TH_ERRORS
}

// layouts(tensors) -> bytes: where the tensors of a list lie, what lies there and their sizes
PyObject* py_layouts(PyObject*, PyObject* list) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(PyList_Check(list), "layouts takes a list");
  const Py_ssize_t n = PyList_GET_SIZE(list);
  Numbers found(4 * n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), "layouts takes tensors");
    const Tensor& t = THPVariable_Unpack(o);
    add_layout(found, t);
    for (const int64_t size : t.sizes()) found.add(size);
  }
  return found.bytes();
  END_HANDLE_TH_ERRORS
}

// state_addresses(entries) -> bytes: where the tensors of a list of dictionaries lie, in their order (0 for
// what is no tensor)
PyObject* py_state_addresses(PyObject*, PyObject* list) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(PyList_Check(list), "state_addresses takes a list");
  const Py_ssize_t n = PyList_GET_SIZE(list);
  Numbers found(4 * n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *entry = PyList_GET_ITEM(list, i), *key = nullptr, *value = nullptr;
    TORCH_CHECK_TYPE(PyDict_Check(entry), "state_addresses takes dictionaries");
    for (Py_ssize_t at = 0; PyDict_Next(entry, &at, &key, &value);)
      found.add(THPVariable_Check(value) ? address(THPVariable_Unpack(value)) : nullptr);
  }
  return found.bytes();
  END_HANDLE_TH_ERRORS
}

// state_layouts(entries) -> bytes: the same without sizes of the tensors of a list of dictionaries, in their order
// (-1: no tensor)
PyObject* py_state_layouts(PyObject*, PyObject* list) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(PyList_Check(list), "state_layouts takes a list");
  const Py_ssize_t n = PyList_GET_SIZE(list);
  Numbers found(8 * n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *entry = PyList_GET_ITEM(list, i), *key = nullptr, *value = nullptr;
    TORCH_CHECK_TYPE(PyDict_Check(entry), "state_layouts takes dictionaries");
    for (Py_ssize_t at = 0; PyDict_Next(entry, &at, &key, &value);) {
      if (THPVariable_Check(value)) add_layout(found, THPVariable_Unpack(value));
      else found.add(int64_t(-1));
    }
  }
  return found.bytes();
  END_HANDLE_TH_ERRORS
}

// gradients(parameters) -> bytes: where the parameters' gradients lie (0: none); None where one of them is not
// dense and contiguous in its parameter's shape, dtype and device
PyObject* py_gradients(PyObject*, PyObject* list) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(PyList_Check(list), "gradients takes a list");
  const Py_ssize_t n = PyList_GET_SIZE(list);
  Numbers found(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), "gradients takes tensors");
    const Tensor& p = THPVariable_Unpack(o);
    const Tensor& g = p.grad();
    if (!g.defined()) {
      found.add(nullptr);
      continue;
    }
    if (g.layout() != at::kStrided || !g.is_contiguous() || g.sizes() != p.sizes() || g.scalar_type() != p.scalar_type() ||
        g.device() != p.device() || g.is_neg())
      Py_RETURN_NONE;
    found.add(address(g));
  }
  return found.bytes();
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"addresses", py_addresses, METH_O, nullptr},
    {"layouts", py_layouts, METH_O, nullptr},
    {"state_addresses", py_state_addresses, METH_O, nullptr},
    {"state_layouts", py_state_layouts, METH_O, nullptr},
    {"gradients", py_gradients, METH_O, nullptr},
    {"norms", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_norms)), METH_FASTCALL, nullptr},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_layer_norm)), METH_FASTCALL, nullptr},
    {"cross_entropy", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_cross_entropy)), METH_FASTCALL, nullptr},
    {"distillation", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_distillation)), METH_FASTCALL, nullptr},
    {"gated_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_gated_linear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_glue", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__glue() { return PyModule_Create(&kModule); }

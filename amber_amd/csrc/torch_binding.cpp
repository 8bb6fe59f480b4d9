// torch binding of the activation -> LayerNorm -> dropout operators (include/amber_mpn.h): argument checks, outputs from torch's
// allocator, the call on the tensor's current stream, and the autograd node.  In C++ because a short call costs more on the host
// than on the GPU: 20736 x 64 forward + backward takes the kernels about 12 us, the same calls through ctypes and a Python
// autograd function took 84 us (dropout) and 113 us (with the norm) of host time.
//
// The library's entry points are handed in as addresses by amber_amd/norm_dropout.py (the library itself stays a plain C ABI that
// knows nothing of torch), so an alternative build of the library is honoured here too.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include "../../include/amber_mpn.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Entries {
  decltype(&amber_mpn_last_error) last_error = nullptr;
  decltype(&amber_mpn_generator_take) take = nullptr;
  decltype(&amber_mpn_keep_mask) mask = nullptr;
  decltype(&amber_mpn_tail_forward) forward = nullptr;
  decltype(&amber_mpn_tail_backward_workspace_bytes) workspace_bytes = nullptr;
  decltype(&amber_mpn_tail_backward) backward = nullptr;
} g_lib;

void bind(uintptr_t last_error, uintptr_t take, uintptr_t mask, uintptr_t forward, uintptr_t workspace_bytes, uintptr_t backward) {
  g_lib.last_error = reinterpret_cast<decltype(g_lib.last_error)>(last_error);
  g_lib.take = reinterpret_cast<decltype(g_lib.take)>(take);
  g_lib.mask = reinterpret_cast<decltype(g_lib.mask)>(mask);
  g_lib.forward = reinterpret_cast<decltype(g_lib.forward)>(forward);
  g_lib.workspace_bytes = reinterpret_cast<decltype(g_lib.workspace_bytes)>(workspace_bytes);
  g_lib.backward = reinterpret_cast<decltype(g_lib.backward)>(backward);
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "amber_amd: ", what, " failed (code ", rc, "): ", g_lib.last_error());
}

// The current stream of a device, which the guard has made the current one.
void* stream_of(const at::Device& device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

bool dtype_id(at::ScalarType t, int32_t& id) {
  switch (t) {
    case at::kFloat: id = AMBER_DTYPE_F32; return true;
    case at::kBFloat16: id = AMBER_DTYPE_BF16; return true;
    case at::kHalf: id = AMBER_DTYPE_F16; return true;
    default: return false;
  }
}

void check_device(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "amber_amd: `", name, "` is on ", t.device(),
              "; the MPN path runs on MI355X only (move the batch to 'cuda'). There is no CPU path.");
}
void check_probability(double p) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "Dropout probability has to be between 0 and 1 (got ", p, ")");
}
void check_sequence(int64_t sequence) {
  TORCH_CHECK_VALUE(sequence >= 0 && sequence < (int64_t{1} << 62), "amber_amd: sequence has to be between 0 and 2**62 (got ", sequence,
                    ")");
}
void check_state(const std::optional<Tensor>& state) {
  TORCH_CHECK_VALUE(state.has_value() && state->defined(), "amber_amd: dropout needs the generator's `state` (CounterGenerator.take())");
  TORCH_CHECK_VALUE(state->scalar_type() == at::kLong && state->dim() == 1 && state->size(0) == 2 && state->is_contiguous(),
                    "amber_amd: `state` must be a contiguous int64 tensor (seed, offset), got ", state->scalar_type(), " ", state->sizes());
}
void check_state_device(const Tensor& state, const at::Device& device) {
  TORCH_CHECK_VALUE(state.device() == device, "amber_amd: `state` is on ", state.device(), ", the data on ", device);
}

// Evenly spaced rows of adjacent features; a copy where t is not that (or, if dense, not contiguous).
struct Rows {
  Tensor t;
  int64_t stride;
};
Rows rows_of(const Tensor& t, int64_t width, bool dense) {
  if (t.is_contiguous()) return {t, width};
  if (!dense && width > 0 && t.dim() > 0) {
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});  // a view where one stride covers the leading dimensions
    if (width == 1 || r.stride(1) == 1) return {r, r.size(0) > 1 ? r.stride(0) : width};
  }
  return {t.contiguous(), width};
}

// What the kernels read through a pointer has to be there as written: negation bits and zero tensors without memory are resolved.
Tensor plain(const Tensor& t) {
  if (!t.defined()) return t;
  if (t._is_zerotensor()) return t.clone();
  return t.is_neg() ? t.resolve_neg() : t;
}

const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mutable_data(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

struct TailBackward : public torch::autograd::Node {
  AmberTailDesc desc{};
  at::ScalarType weight_type = at::kFloat;
  SavedVariable x, weight, stats, state;

  std::string name() const override { return "AmberTailBackward"; }

  // What was saved may come back from a saved tensors' hook with other strides (a copy that was on the host, say): its layout is
  // looked at here, not remembered.
  static Rows saved(const Tensor& from, const char* name, int64_t rows, int64_t width, at::ScalarType type, const at::Device& device,
                    bool dense) {
    if (!from.defined()) return {from, width};
    TORCH_CHECK(from.numel() == rows * width && (dense || from.size(-1) == width) && from.scalar_type() == type && from.device() == device,
                "amber_amd: `", name, "` was saved for the backward pass and came back as another tensor: ", from.scalar_type(), " ",
                from.sizes(), " on ", from.device());
    return rows_of(plain(from), width, dense);
  }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    stats.reset_data();
    state.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    {
      std::lock_guard<std::mutex> lock(mutex_);
      const Tensor xs = x.unpack(), ws = weight.unpack(), ss = stats.unpack(), st = state.unpack();
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(grads[0].device());
      const Tensor grad_y = plain(grads[0]);
      const bool normalize = desc.normalize != 0;
      const int64_t width = normalize ? grad_y.size(-1) : 1, rows = grad_y.numel() / width;
      const Rows g = rows_of(grad_y, width, !normalize), r = saved(xs, "x", rows, width, grad_y.scalar_type(), grad_y.device(), !normalize),
                 w = saved(ws, "weight", 1, width, weight_type, grad_y.device(), true),
                 s = saved(ss, "stats", 2, rows, at::kFloat, grad_y.device(), true),
                 t = saved(st, "state", 1, 2, at::kLong, grad_y.device(), true);
      const bool need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
      if (task_should_compute_output(0)) out[0] = at::empty(grad_y.sizes(), grad_y.options());
      c10::DataPtr workspace;  // back to the allocator at the end of this block, in stream order like any tensor
      size_t bytes = 0;
      if (need_w) out[1] = at::empty({width}, grad_y.options().dtype(weight_type));
      if (need_b) out[2] = at::empty({width}, grad_y.options().dtype(weight_type));
      if (need_w || need_b) {
        bytes = g_lib.workspace_bytes(&desc, rows, width);
        if (bytes) workspace = c10::GetAllocator(c10::DeviceType::CUDA)->allocate(bytes);
      }
      check(g_lib.backward(&desc, rows, width, data(r.t), r.stride, data(g.t), g.stride, data(w.t), static_cast<const float*>(data(s.t)),
                           static_cast<const int64_t*>(data(t.t)), mutable_data(out[0]), mutable_data(out[1]), mutable_data(out[2]),
                           workspace.get(), bytes, stream_of(grad_y.device())),
            "tail backward");
    }
    if (at::GradMode::is_enabled()) {  // recorded (create_graph): allowed, but differentiating the gradients raises
      auto error = std::make_shared<torch::autograd::DelayedError>("amber_amd: activate_norm_dropout has first derivatives only", 3);
      return (*error)(std::move(out));
    }
    return out;
  }
};

void no_forward_mode(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "amber_amd: forward-mode derivatives are not built");
}

// y = dropout(layer_norm(act(x))), any part absent.  p is 0 outside training.
Tensor tail(const Tensor& x_, const std::optional<Tensor>& weight_, const std::optional<Tensor>& bias_, const std::optional<Tensor>& state_,
            int64_t activation, bool normalize, double p, double eps, int64_t sequence) {
  AmberTailDesc desc{};
  const Tensor x = plain(x_);
  TORCH_CHECK_TYPE(dtype_id(x.scalar_type(), desc.dtype), "amber_amd: x must be float32, bfloat16 or float16, got ", x.scalar_type());
  check_probability(p);
  check_sequence(sequence);
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < 3.0e38, "amber_amd: eps must be finite and not negative (got ", eps, ")");
  const bool drops = p > 0.0;
  if (drops) check_state(state_);
  Tensor weight, bias;
  at::ScalarType weight_type = x.scalar_type();
  if (normalize) {
    const int64_t features = x.dim() ? x.size(-1) : 0;
    TORCH_CHECK_VALUE(features > 0, "amber_amd: LayerNorm over the last dimension of a tensor of shape ", x.sizes());
    const auto take = [&](const std::optional<Tensor>& from, const char* name, Tensor& to) {
      if (!from.has_value() || !from->defined()) return;
      TORCH_CHECK_VALUE(from->dim() == 1 && from->size(0) == features, "amber_amd: ", name, " of shape ", from->sizes(), " for ", features,
                        " features");
      TORCH_CHECK_VALUE(from->device() == x.device(), "amber_amd: ", name, " is on ", from->device(), ", x on ", x.device());
      TORCH_CHECK_TYPE(from->scalar_type() == x.scalar_type() || from->scalar_type() == at::kFloat, "amber_amd: ", name,
                       " must be of x's type (", x.scalar_type(), ") or float32, got ", from->scalar_type());
      to = plain(*from);
      weight_type = to.scalar_type();
    };
    take(weight_, "weight", weight);
    take(bias_, "bias", bias);
    TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "amber_amd: weight is ",
                     weight.defined() ? weight.scalar_type() : at::kFloat, ", bias ", bias.defined() ? bias.scalar_type() : at::kFloat);
  } else {
    TORCH_CHECK_VALUE(!weight_.has_value() && !bias_.has_value(), "amber_amd: weight / bias without normalize");
  }
  check_device(x, "x");
  Tensor state;
  if (drops) {
    check_state_device(*state_, x.device());
    state = *state_;
  }
  if (!normalize && !drops && activation == AMBER_ACT_NONE) return x_;
  no_forward_mode(x);
  no_forward_mode(weight);
  no_forward_mode(bias);
  dtype_id(weight_type, desc.weight_dtype);
  desc.activation = static_cast<int32_t>(activation);
  desc.normalize = normalize;
  desc.p = p;
  desc.eps = eps;
  desc.sequence = sequence;

  const bool record = at::GradMode::is_enabled() &&
                      (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad()));
  Tensor y, stats, w;
  Rows r;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    const int64_t width = normalize ? x.size(-1) : 1, rows = x.numel() / width;  // without the norm: one flat row of elements
    r = rows_of(x, width, !normalize);
    if (weight.defined()) w = weight.contiguous();
    const Tensor b = bias.defined() ? bias.contiguous() : bias;
    y = at::empty(x.sizes(), x.options());
    if (normalize && record) stats = at::empty({2 * rows}, x.options().dtype(at::kFloat));
    check(g_lib.forward(&desc, rows, width, data(r.t), r.stride, data(w), data(b), static_cast<const int64_t*>(data(state)),
                        mutable_data(y), static_cast<float*>(mutable_data(stats)), stream_of(x.device())),
          "tail forward");
  }
  if (record) {
    std::shared_ptr<TailBackward> node(new TailBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias));
    node->desc = desc;
    node->weight_type = weight_type;
    // x itself where the kernels read it in place: a change of it before the backward pass is noticed
    if (normalize || activation != AMBER_ACT_NONE)
      node->x = SavedVariable(r.t.unsafeGetTensorImpl() == x.unsafeGetTensorImpl() || r.t.is_alias_of(x) ? x : r.t, false);
    if (weight.defined()) node->weight = SavedVariable(w.is_alias_of(weight) ? weight : w, false);
    if (stats.defined()) node->stats = SavedVariable(stats, false);
    if (state.defined()) node->state = SavedVariable(state, false);
    torch::autograd::set_history(y, node);
  }
  return y;
}

Tensor keep_mask(int64_t count, double p, const std::optional<Tensor>& state, int64_t sequence) {
  TORCH_CHECK_VALUE(count >= 0, "amber_amd: a mask of ", count, " elements");
  check_probability(p);
  check_sequence(sequence);
  check_state(state);
  check_device(*state, "state");
  const c10::DeviceGuard guard(state->device());
  const Tensor out = at::empty({count}, state->options().dtype(at::kBool));
  check(g_lib.mask(state->const_data_ptr<int64_t>(), sequence, p, count, static_cast<uint8_t*>(out.mutable_data_ptr()),
                   stream_of(state->device())),
        "keep_mask");
  return out;
}

Tensor generator_take(const Tensor& state, int64_t count) {
  TORCH_CHECK_VALUE(count >= 1 && count < (int64_t{1} << 62), "amber_amd: take of ", count, " ranges");
  check_state(state);
  check_device(state, "generator state");
  const c10::DeviceGuard guard(state.device());
  const Tensor taken = at::empty_like(state);
  // a backward pass that reads the generator's own buffer instead of `taken` must notice
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  check(g_lib.take(state.mutable_data_ptr<int64_t>(), count, taken.mutable_data_ptr<int64_t>(), stream_of(state.device())),
        "generator take");
  return taken;
}

}  // namespace

PYBIND11_MODULE(amber_torch, m) {
  namespace py = pybind11;
  m.def("bind", &bind);
  m.def("tail", &tail, py::call_guard<py::gil_scoped_release>());
  m.def("keep_mask", &keep_mask, py::call_guard<py::gil_scoped_release>());
  m.def("generator_take", &generator_take, py::call_guard<py::gil_scoped_release>());
}

// nif_torch.cpp -- the head losses of libnif as autograd functions.  A head of a level fit is three launches of a few
// microseconds; written in Python, its forward and backward passes spent 150 us around them, most of it in autograd's
// own thread.  Arguments are checked in ops.py; here are buffers, streams, devices and gradients only.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <unordered_set>

#include "../../include/nif.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Optional = std::optional<Tensor>;

Tensor or_none(const Optional& t) { return t ? *t : Tensor(); }

struct NifError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject* nif_error = nullptr;  // the class that the ctypes binding raises

void check(int status, const char* what) {
  if (status != NIF_OK)
    throw NifError(std::string(what) + " failed with status " + std::to_string(status) + ": " + nif_error_string(status));
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)(n ? n : 1)}, like.options().dtype(at::kByte)); }

Tensor loss_of(int64_t rows, int reduction, const Tensor& like) {
  const auto options = like.options().dtype(at::kFloat);
  return reduction == NIF_REDUCE_NONE ? at::empty({rows}, options) : at::empty({}, options);
}

int type_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? NIF_F32 : t.scalar_type() == at::kBFloat16 ? NIF_BF16 : NIF_F16; }

int64_t ld_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }

template <class T>
const T* data(const Tensor& t) {
  return t.defined() ? (const T*)t.const_data_ptr() : nullptr;
}
void* out(Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A leaf's gradient accumulator lives as long as a graph that ends in it and stays on the stream of the pass that made it.
// Captured together with a later pass, that stream would have to wait for the capturing one, which ends the process: a
// captured backward pass that would get there is refused.
void refuse_capture_of_live_leaves(const Tensor& like) {
  hipStreamCaptureStatus status;
  if (hipStreamIsCapturing((hipStream_t)stream_of(like), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  const c10::Stream here = c10::impl::VirtualGuardImpl(like.device().type()).getStream(like.device());
  std::vector<torch::autograd::Node*> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  const auto current = torch::autograd::get_current_node();
  if (current) todo.push_back(current.get());
  while (!todo.empty()) {
    torch::autograd::Node* node = todo.back();
    todo.pop_back();
    for (size_t i = 0; i < node->num_outputs(); ++i) {
      if (!node->task_should_compute_output(i)) continue;
      torch::autograd::Node* next = node->next_edge(i).function.get();
      if (!next || !seen.insert(next).second) continue;
      todo.push_back(next);
      if (!dynamic_cast<torch::autograd::AccumulateGrad*>(next)) continue;
      const auto stream = next->stream();
      if (stream && *stream != here)
        throw NifError("an autograd graph of an earlier pass over the same leaves is alive on another stream: a backward pass cannot be "
                       "captured with it; drop that pass's loss and outputs first");
    }
  }
}

// Gradients that are differentiated again fail, instead of counting as constants.
variable_list once(variable_list grads, const Tensor& grad_loss) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (const Tensor& g : grads)
    if (g.defined()) some.push_back(g);
  auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of the head losses are differentiable once", (int)some.size());
  for (Tensor& g : some) g = g.detach().requires_grad_();
  some = (*error)(std::move(some));
  size_t at = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = some[at++];
  return grads;
}

nif_head_desc describe(const Tensor& hidden, const Tensor& weight, const Tensor& bias, const Tensor& labels, const Tensor& indices,
                       const Tensor& values, const Tensor& lse, double temperature, int64_t ignore_index, int64_t reduction,
                       bool forward_only) {
  nif_head_desc d;
  d.hidden = data<void>(hidden);
  d.ldh = ld_of(hidden);
  d.weight = data<void>(weight);
  d.ldw = ld_of(weight);
  d.bias = data<void>(bias);
  d.rows = hidden.size(0);
  d.features = (int32_t)hidden.size(1);
  d.classes = (int32_t)weight.size(0);
  d.dtype = type_of(hidden);
  d.reduction = (int32_t)reduction;
  d.labels = data<int64_t>(labels);
  d.ignore_index = ignore_index;
  d.top_indices = data<int32_t>(indices);
  d.top_values = data<float>(values);
  d.top_lse = data<float>(lse);
  d.top = indices.defined() ? (int32_t)indices.size(1) : 0;
  d.temperature = (float)temperature;
  d.forward_only = forward_only;
  return d;
}

struct LinearHead : torch::autograd::Function<LinearHead> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Optional& bias_, const Optional& labels_,
                        const Optional& indices_, const Optional& values_, const Optional& lse_, double temperature,
                        int64_t ignore_index, int64_t reduction, bool forward_only) {
    const c10::DeviceGuard guard(hidden.device());
    const Tensor bias = or_none(bias_), labels = or_none(labels_), indices = or_none(indices_), values = or_none(values_),
                 lse = or_none(lse_);
    const nif_head_desc d = describe(hidden, weight, bias, labels, indices, values, lse, temperature, ignore_index, reduction, forward_only);
    Tensor loss = loss_of(d.rows, d.reduction, hidden);
    const size_t state_bytes = nif_head_state_bytes(&d), ws_bytes = nif_head_forward_workspace_bytes(&d);
    Tensor state = bytes(state_bytes, hidden), ws = bytes(ws_bytes, hidden);
    check(nif_head_forward(&d, loss.mutable_data_ptr<float>(), state.mutable_data_ptr(), state_bytes, ws.mutable_data_ptr(), ws_bytes,
                           stream_of(hidden)),
          "nif_head_forward");
    ctx->save_for_backward({hidden, weight, bias, labels, indices, values, lse, state});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &hidden = s[0], &weight = s[1], &bias = s[2], &state = s[7];
    variable_list r(11);
    if (!grads[0].defined()) return r;
    const c10::DeviceGuard guard(hidden.device());
    refuse_capture_of_live_leaves(hidden);
    const nif_head_desc d = describe(hidden, weight, bias, s[3], s[4], s[5], s[6], ctx->saved_data["temperature"].toDouble(),
                                     ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["reduction"].toInt(), false);
    const Tensor grad = grads[0].contiguous();
    const auto like = [](const Tensor& t) { return at::empty(t.sizes(), t.options()); };
    // counted over the tensors that were given: the bias is the third where there is one
    if (ctx->needs_input_grad(0)) r[0] = like(hidden);
    if (ctx->needs_input_grad(1)) r[1] = like(weight);
    if (bias.defined() && ctx->needs_input_grad(2)) r[2] = like(bias);
    const size_t ws_bytes = nif_head_backward_workspace_bytes(&d);
    Tensor ws = bytes(ws_bytes, hidden);
    check(nif_head_backward(&d, grad.const_data_ptr<float>(), state.const_data_ptr(), state.numel(), out(r[0]), d.features, out(r[1]),
                            d.features, out(r[2]), ws.mutable_data_ptr(), ws_bytes, stream_of(hidden)),
          "nif_head_backward");
    return once(std::move(r), grads[0]);
  }
};

struct Distill : torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& indices, const Tensor& values, const Optional& lse_,
                        double temperature, int64_t reduction) {
    const c10::DeviceGuard guard(logits.device());
    const Tensor lse = or_none(lse_);
    const int64_t n = logits.size(0);
    const int k = (int)indices.size(1);
    Tensor loss = loss_of(n, (int)reduction, logits);
    const size_t state_bytes = nif_distill_state_bytes(n, k), ws_bytes = nif_distill_workspace_bytes(n);
    Tensor state = bytes(state_bytes, logits), ws = bytes(ws_bytes, logits);
    check(nif_distill_forward(data<void>(logits), ld_of(logits), n, (int)logits.size(1), type_of(logits), data<int32_t>(indices),
                              data<float>(values), data<float>(lse), k, (float)temperature, (int)reduction, loss.mutable_data_ptr<float>(),
                              state.mutable_data_ptr(), state_bytes, ws.mutable_data_ptr(), ws_bytes, stream_of(logits)),
          "nif_distill_forward");
    ctx->save_for_backward({logits, state});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["top"] = (int64_t)k;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &logits = s[0], &state = s[1];
    variable_list r(6);
    if (!grads[0].defined()) return r;
    const c10::DeviceGuard guard(logits.device());
    refuse_capture_of_live_leaves(logits);
    const Tensor grad = grads[0].contiguous();
    r[0] = at::empty(logits.sizes(), logits.options());
    check(nif_distill_backward(data<void>(logits), ld_of(logits), logits.size(0), (int)logits.size(1), type_of(logits),
                               (int)ctx->saved_data["top"].toInt(), (float)ctx->saved_data["temperature"].toDouble(),
                               (int)ctx->saved_data["reduction"].toInt(), grad.const_data_ptr<float>(), state.const_data_ptr(),
                               state.numel(), out(r[0]), logits.size(1), stream_of(logits)),
          "nif_distill_backward");
    return once(std::move(r), grads[0]);
  }
};

Tensor linear_head(const Tensor& hidden, const Tensor& weight, const Optional& bias, const Optional& labels, const Optional& indices,
                   const Optional& values, const Optional& lse, double temperature, int64_t ignore_index, int64_t reduction) {
  const bool grads = at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()));
  return LinearHead::apply(hidden, weight, bias, labels, indices, values, lse, temperature, ignore_index, reduction, !grads);
}

Tensor distill(const Tensor& logits, const Tensor& indices, const Tensor& values, const Optional& lse, double temperature,
               int64_t reduction) {
  return Distill::apply(logits, indices, values, lse, temperature, reduction);
}

std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& logits, int64_t k, double temperature) {
  const c10::DeviceGuard guard(logits.device());
  const int64_t n = logits.size(0);
  Tensor values = at::empty({n, k}, logits.options()), indices = at::empty({n, k}, logits.options().dtype(at::kInt)),
         lse = at::empty({n}, logits.options().dtype(at::kFloat));
  check(nif_top_logits(data<void>(logits), ld_of(logits), n, (int)logits.size(1), type_of(logits), (int)k, (float)temperature,
                       values.mutable_data_ptr(), indices.mutable_data_ptr<int32_t>(), lse.mutable_data_ptr<float>(), stream_of(logits)),
        "nif_top_logits");
  return {values, indices, lse};
}

}  // namespace

// The GIL is not needed in the calls: autograd takes it for the hooks and functions that are Python's
PYBIND11_MODULE(nif_torch, m) {
  m.def("set_error", [](const pybind11::object& cls) { nif_error = cls.inc_ref().ptr(); });
  pybind11::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NifError& e) {
      PyErr_SetString(nif_error ? nif_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("linear_head", &linear_head, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("distill", &distill, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("top_logits", &top_logits, pybind11::call_guard<pybind11::gil_scoped_release>());
}

// One differentiable call of an operator: what its autograd node keeps, guards and answers.  Shared by the operator surfaces
// (operators.cpp, lm_operators.cpp).
#pragma once

#include <torch/csrc/autograd/autograd.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>

#include <mutex>
#include <utility>

#include "operands.h"

namespace ssm_ext {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients that a graph is recorded through (create_graph).  The kernels' backward passes have no derivative of their own, so the values are
// right, but differentiated again they would be constants: that raises.  They hang on all they depend on, because the engine walks only
// paths that lead to what it is asked for.
struct OnceFn : torch::autograd::Function<OnceFn> {
  static variable_list forward(AutogradContext*, const variable_list& values, at::TensorList sources) {
    (void)sources;
    return values;
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "ssm_b200 operators are differentiable once: a gradient formed with create_graph=True cannot be differentiated through them");
  }
};
inline variable_list differentiable_once(const variable_list& grads, const variable_list& sources) {
  variable_list values, res;
  for (const Tensor& t : grads)
    if (t.defined()) values.push_back(t.detach());
  if (!values.empty()) values = OnceFn::apply(values, at::TensorList(sources));
  size_t next = 0;
  for (const Tensor& t : grads) res.push_back(t.defined() ? values[next++] : Tensor());
  return res;
}

// The operands of a call, kept by its autograd node.  `guarded` holds the tensors that the backward pass reads again with
// their version counters at the time of the forward pass: an in-place edit in between is an error, as for any saved tensor.  `unread` holds the
// others, which may be edited.
struct Call : torch::CustomClassHolder {
  std::vector<std::pair<Tensor, uint32_t>> guarded, unread;
  variable_list inputs;  // the defined tensor arguments, in the order backward() answers for them
  void input(const Tensor& t) { inputs.push_back(t); }
  void input(const OptTensor& t) {
    if (t.has_value() && t->defined()) inputs.push_back(*t);
  }
  // A call without a node would drop tangents in silence, so they are looked for first.
  bool needs_grad() const {
    for (const Tensor& t : inputs)
      TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "ssm_b200 operators have no forward-mode derivative");
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : inputs)
      if (t.requires_grad()) return true;
    return false;
  }
  virtual bool reads(size_t) const { return true; }  // whether backward() reads this input again
  virtual variable_list forward(bool train) = 0;
  // One gradient (or an undefined tensor) per input.  An incoming gradient is undefined where nothing flowed back to that output, and all
  // of them can be (a node downstream that returns none).
  virtual variable_list backward(const variable_list& grads) = 0;
  // Whether backward() may run again after a walk that does not retain the graph.  A whole mixer's tensors go with that walk, as those of the
  // products that it stands for would.
  virtual bool survives_its_walk() const { return true; }
  // backward() where a graph is recorded through the gradients.
  virtual variable_list backward_recorded(const variable_list& grads) {
    variable_list res, sources;
    {
      at::NoGradGuard values_only;
      res = backward(grads);
    }
    for (const auto& kept : guarded) sources.push_back(kept.first);
    for (const auto& kept : unread) sources.push_back(kept.first);
    for (const Tensor& g : grads)
      if (g.defined()) sources.push_back(g);
    return differentiable_once(res, sources);
  }
};

struct CallFn : torch::autograd::Function<CallFn> {
  static variable_list forward(AutogradContext* ctx, const c10::intrusive_ptr<Call>& call, at::TensorList inputs) {
    for (size_t i = 0; i < inputs.size(); ++i)
      if (!inputs[i].is_inference()) (call->reads(i) ? call->guarded : call->unread).emplace_back(inputs[i], inputs[i]._version());
    ctx->saved_data["call"] = c10::IValue::make_capsule(call);
    ctx->set_materialize_grads(false);
    return call->forward(true);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->saved_data.find("call");
    TORCH_CHECK(saved != ctx->saved_data.end(), torch::autograd::ERR_BACKWARD_TWICE);
    auto holder = saved->second.toCapsule();
    Call* call = static_cast<Call*>(holder.get());
    for (const auto& kept : call->guarded) {
      if (kept.first._version() == kept.second) continue;
      std::string shape;
      for (int64_t d : kept.first.sizes()) shape += (shape.empty() ? "" : ", ") + std::to_string(d);
      TORCH_CHECK(false, "one of the tensors needed for the backward pass of an ssm_b200 operator has been modified in place (shape (" + shape + "), version " +
                             std::to_string(kept.first._version()) + ", expected " + std::to_string(kept.second) + ")");
    }
    ValueErrors scope;
    const bool last_walk = !call->survives_its_walk() && !torch::autograd::get_current_graph_task_keep_graph();
    variable_list res = at::GradMode::is_enabled() ? call->backward_recorded(grads) : call->backward(grads);
    if (last_walk) ctx->saved_data.clear();
    res.insert(res.begin(), Tensor());  // the slot of `call`
    return res;
  }
};

inline variable_list invoke_call(const c10::intrusive_ptr<Call>& call) {
  if (!call->needs_grad()) return call->forward(false);
  const variable_list inputs = call->inputs;
  call->inputs.clear();
  return CallFn::apply(call, at::TensorList(inputs));
}

inline Tensor cast(const Tensor& grad, at::ScalarType t) { return grad.scalar_type() == t ? grad : grad.to(t); }

// The word a kernel sets when one of its bounded waits runs out, one per device, in pinned host memory that the kernels write
// directly: a failure is visible to the next call without a copy, an event or a synchronisation per launch.
inline Tensor ssd_status(int64_t device) {
  static std::mutex lock;
  static std::vector<Tensor> words(64);
  TORCH_CHECK(device >= 0 && device < (int64_t)words.size(), "ssd_scan: device index out of range");
  std::lock_guard<std::mutex> hold(lock);
  Tensor& w = words[device];
  if (!w.defined()) w = at::zeros({1}, at::TensorOptions().dtype(at::kInt)).pin_memory();
  return w;
}
// Raise if a launch since the last report ran out of a wait.
inline void ssd_poll(int64_t device) {
  volatile int32_t* word = ssd_status(device).data_ptr<int32_t>();
  const int32_t code = *word;
  if (code == 0) return;
  *word = 0;
  TORCH_CHECK(false, std::string() + (code < 4 ? "ssd_scan" : code < 128 ? "gated_delta_scan" : "linear_cross_entropy") + ": a bounded device-side wait ran out in an earlier launch (status " + std::to_string(code) + "); its outputs are invalid");
}

}  // namespace ssm_ext

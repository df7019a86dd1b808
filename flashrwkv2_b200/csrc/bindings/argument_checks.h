// Argument checks that raise what the Python layer documents: TypeError for wrong types, ValueError for wrong shapes,
// layouts and values.  They run before anything touches a device.
#pragma once

#include <string>

#include "bindings.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

namespace frwkv_bindings {

template <typename Text> inline void need_type(bool condition, const Text& message) {
  if (!condition) throw py::type_error(message);
}

template <typename Text> inline void need_value(bool condition, const Text& message) {
  if (!condition) throw py::value_error(message);
}

// Gradients of an operator whose backward pass has no derivative of its own: where a graph of it is being recorded, they
// carry a node that raises when that derivative is asked for.
inline torch::autograd::variable_list differentiable_once(torch::autograd::variable_list grads, const char* what) {
  if (!torch::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list given;
  for (auto& g : grads)
    if (g.defined()) given.push_back(g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once",
                                                               static_cast<int64_t>(given.size()));
  given = (*error)(std::move(given));
  size_t next = 0;
  for (auto& g : grads)
    if (g.defined()) g = given[next++];
  return grads;
}

}  // namespace frwkv_bindings

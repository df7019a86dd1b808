// Argument checks that raise what the Python layer documents: TypeError for wrong types, ValueError for wrong shapes,
// layouts and values.  They run before anything touches a device.
#pragma once

#include <string>

#include "bindings.h"

namespace frwkv_bindings {

template <typename Text> inline void need_type(bool condition, const Text& message) {
  if (!condition) throw py::type_error(message);
}

template <typename Text> inline void need_value(bool condition, const Text& message) {
  if (!condition) throw py::value_error(message);
}

}  // namespace frwkv_bindings

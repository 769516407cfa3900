// Registration of the 8-bit KV cache bindings in the extension module.
#pragma once

#include <torch/extension.h>

void register_kv8(pybind11::module& m);

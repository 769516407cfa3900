// Registration of the 8-bit KV cache bindings in the extension module.
#pragma once

#include <cuda.h>
#include <torch/extension.h>

// One layer [pages, 2, Hkv, ps, 128] as rows of 128 bytes; box (128 bytes, min(ps, 16) rows), 128B swizzle.
CUtensorMap map_kv8(const torch::Tensor& data);

void register_kv8(pybind11::module& m);

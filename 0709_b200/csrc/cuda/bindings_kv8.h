// Registration of the 8-bit KV cache bindings in the extension module.
#pragma once

#include <cuda.h>
#include <torch/extension.h>

// One layer of the 8-bit cache, `rows` rows of 128 bytes; box (128 bytes, min(ps, 16) rows), 128B swizzle.
CUtensorMap map_kv8(const void* data, int64_t rows, int64_t ps);

void register_kv8(pybind11::module& m);

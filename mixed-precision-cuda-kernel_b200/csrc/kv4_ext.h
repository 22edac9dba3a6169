// Adds the 4-bit KV cache and the attention of prompts to the `quant_cuda` module.
#pragma once
#include <pybind11/pybind11.h>
void register_kv4(pybind11::module_& m);

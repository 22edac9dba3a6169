// Adds the paged KV cache and the adjustment of logits to the `quant_cuda` module.
#pragma once
#include <pybind11/pybind11.h>
void register_pages(pybind11::module_& m);

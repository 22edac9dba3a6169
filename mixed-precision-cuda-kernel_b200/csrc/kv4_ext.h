// Adds the 4-bit KV cache and the attention of prompts to the `quant_cuda` module.
#pragma once
#include <c10/core/Device.h>
#include <pybind11/pybind11.h>
void register_kv4(pybind11::module_& m);
// the word that a device's launches report time-outs into (device_timed_out reads it)
uint32_t* device_status(const c10::Device& device);

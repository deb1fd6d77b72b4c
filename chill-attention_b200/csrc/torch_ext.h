// What the parts of the native torch module share (torch_ext.cpp, torch_cache.cpp, torch_decode.cpp).
#pragma once
#include <torch/csrc/utils/pybind.h>

#include <string>

#include "chill_b200.h"

// Mask constants as both members of the descriptor (the whole numbers as Python's int() makes them, saturated at 64 bits).
void set_mask_constants(chill_mask_desc& desc, const pybind11::tuple& mask_args);
// Throws what Python sees as chill_attention._cabi.ChillLibraryError.
[[noreturn]] void throw_chill_error(const std::string& message);
void bind_cache(pybind11::module_& m);
void bind_decode(pybind11::module_& m);

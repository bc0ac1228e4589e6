// The operators around the attention, as the module offers them (block.cpp).
#pragma once
#include "common.h"

void bind_block(pybind11::module_& m);
void bind_int8(pybind11::module_& m);           // int8.cpp
void bind_experts(pybind11::module_& m);        // experts.cpp

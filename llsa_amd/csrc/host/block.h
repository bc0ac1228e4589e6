// The operators around the attention, as the module offers them (block.cpp).
#pragma once
#include "common.h"

void bind_block(pybind11::module_& m);

// fa_native_layer.hpp — the part of the _fa_native module that fa_native_layer.cpp defines.
#pragma once

#include <torch/extension.h>

void bind_layer(py::module_& m);

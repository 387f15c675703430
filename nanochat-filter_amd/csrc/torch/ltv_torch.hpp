// The parts of the PyTorch extension, bound by its module.
#pragma once

#include <torch/extension.h>

// the paged cache, attention over it and log probabilities (ltv_serving.cpp)
void bind_serving(pybind11::module_& m);

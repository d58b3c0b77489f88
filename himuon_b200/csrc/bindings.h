// What the binding files share.
#pragma once

#include <torch/extension.h>

#include <atomic>

extern std::atomic<int64_t> autograd_launched;         // kernels launched by the autograd functions that are written in C++
void bind_layer_ops(pybind11::module& m);

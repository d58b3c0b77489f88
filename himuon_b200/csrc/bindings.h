// What the binding files share.
#pragma once

#include <torch/extension.h>

#include <atomic>

extern std::atomic<int64_t> autograd_launched;         // kernels launched by the autograd functions that are written in C++
// out = op(a) op(b) on the GEMM kernels (bindings.cpp checks the operands).
void gemm_into(const at::Tensor& a, const at::Tensor& b, at::Tensor& out, bool trans_a, bool trans_b);
void bind_layer_ops(pybind11::module& m);

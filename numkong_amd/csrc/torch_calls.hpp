/**
 *  @brief What mx_calls.cpp and dense_calls.cpp share: torch's tensors as the library takes them.
 *  @file numkong_amd/csrc/torch_calls.hpp
 */
#ifndef NUMKONG_AMD_TORCH_CALLS_HPP
#define NUMKONG_AMD_TORCH_CALLS_HPP

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "numkong_amd/dots.h"

namespace {

/** Other threads of Python may run while the work is queued. */
struct WithoutLock {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutLock() { PyEval_RestoreThread(state); }
};

/** The GPU that a call's operands are on: the first one's, and the current one. */
struct Home {
    int index = -1;
    bool has(at::Tensor const &t) {
        if (!t.is_cuda()) return false;
        if (index < 0 && t.get_device() == c10::hip::current_device()) index = t.get_device();
        return t.get_device() == index;
    }
};
/** The tensor that an argument is, if it is one on that GPU, of `dims` dimensions, its rows of adjacent values, without a tangent. */
at::Tensor const *tensor_of(PyObject *argument, int64_t dims, Home &home) {
    if (!THPVariable_CheckExact(argument)) return nullptr;
    at::Tensor const &t = THPVariable_Unpack(argument);
    if (!home.has(t) || t.layout() != at::kStrided || t.dim() != dims) return nullptr;
    if (dims && t.size(dims - 1) > 1 && t.stride(dims - 1) != 1) return nullptr;
    if (t._fw_grad(0).defined()) return nullptr; // (forward mode: the Python side refuses it)
    return &t;
}
nk_dtype_t code_of(at::ScalarType type) {
    return type == at::kFloat ? nk_f32_k : type == at::kBFloat16 ? nk_bf16_k : type == at::kHalf ? nk_f16_k : nk_dtype_t(0);
}
nk_size_t row_bytes(at::Tensor const &t) {
    return (nk_size_t)((t.size(0) > 1 ? t.stride(0) : t.size(1)) * (int64_t)t.element_size());
}
bool natural(PyObject *argument, int64_t &value) { // an int that is not negative
    if (!PyLong_CheckExact(argument)) return false;
    int overflow = 0;
    value = PyLong_AsLongLongAndOverflow(argument, &overflow);
    return !overflow && value >= 0;
}
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, at::Tensor const &like) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}
void *stream_of(Home const &home) { return (void *)c10::hip::getCurrentHIPStream((c10::DeviceIndex)home.index).stream(); }

/** Does autograd follow it? Then mx.py says what becomes of the gradient. */
bool tracked(at::Tensor const &t) { return c10::GradMode::is_enabled() && t.requires_grad(); }

} // namespace

#endif // NUMKONG_AMD_TORCH_CALLS_HPP

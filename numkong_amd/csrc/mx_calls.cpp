/**
 *  @brief The calls of numkong_amd/mx.py in their ordinary form: tensors on the current GPU, results newly made.
 *  @file numkong_amd/csrc/mx_calls.cpp
 *
 *  A call of few tokens is a few microseconds of work, and the checks, allocations and conversions that mx.py makes for it
 *  take longer than that (quantising 16 rows: 9 us through ctypes). Here they take under two, next to the launch itself.
 *  Every function returns None for what it does not take, or what the library refuses: mx.py then goes its general way, which
 *  handles the one and explains the other, so that nothing is decided here that is not decided there as well. The library's functions
 *  come as addresses (`bind`), from whichever build of it mx.py has loaded.
 */
#include "torch_calls.hpp"

#include "numkong_amd/mx.h"

namespace {

struct Library {
    decltype(&nk_amd_mx_quantize_async) quantize;
    decltype(&nk_amd_mx_dequantize_async) dequantize;
    decltype(&nk_amd_mx_dots_workspace_size) dots_room;
    decltype(&nk_amd_mx_dots_packed_async) dots;
    decltype(&nk_amd_experts_route_async) route;
    decltype(&nk_amd_experts_route_backward_async) route_backward;
    decltype(&nk_amd_experts_plan_size) plan_size;
    decltype(&nk_amd_experts_plan_async) plan;
    decltype(&nk_amd_mx_experts_workspace_size) experts_room;
    decltype(&nk_amd_mx_dots_experts_async) experts;
};
Library library;
decltype(&nk_amd_mx_packed_size) packed_size;

PyObject *bind(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    if (count != (Py_ssize_t)(sizeof(Library) / sizeof(void *))) {
        PyErr_SetString(PyExc_TypeError, "bind takes the addresses of all functions");
        return nullptr;
    }
    void *addresses[sizeof(Library) / sizeof(void *)];
    for (Py_ssize_t i = 0; i < count; ++i) {
        addresses[i] = PyLong_AsVoidPtr(arguments[i]);
        if (!addresses[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is NULL");
            return nullptr;
        }
    }
    memcpy(&library, addresses, sizeof(library));
    Py_RETURN_NONE;
}

PyObject *bind_packed_size(PyObject *, PyObject *address) {
    packed_size = (decltype(packed_size))PyLong_AsVoidPtr(address);
    if (packed_size) Py_RETURN_NONE;
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "the address is NULL");
    return nullptr;
}

/** Is the buffer as large as its sizes say (0: there are no such sizes)? */
bool holds(at::Tensor const &buffer, nk_size_t needed) { return needed && buffer.nbytes() >= needed; }

/** What a product's call says of A: a float matrix, or codes and scales. */
struct Left {
    at::Tensor const *t = nullptr, *scales = nullptr;
    int64_t depth = 0;
    nk_dtype_t dtype = nk_dtype_t(0);
    bool found(PyObject *a, PyObject *its_scales, PyObject *its_depth, Home &home) {
        if (!(t = tensor_of(a, 2, home)) || tracked(*t)) return false;
        if (its_scales == Py_None) {
            depth = t->size(1), dtype = code_of(t->scalar_type());
            return dtype != 0;
        }
        scales = tensor_of(its_scales, 2, home);
        return scales && t->scalar_type() == at::kByte && scales->scalar_type() == at::kByte && natural(its_depth, depth);
    }
    void const *scales_data() const { return scales ? scales->data_ptr() : nullptr; }
    nk_size_t scales_stride() const { return scales ? row_bytes(*scales) : 0; }
};

/** quantize(x) -> (codes, scales) */
PyObject *quantize(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    at::Tensor const *const x = count == 1 ? tensor_of(arguments[0], 2, home) : nullptr;
    nk_dtype_t const dtype = x ? code_of(x->scalar_type()) : nk_dtype_t(0);
    if (!dtype) Py_RETURN_NONE;
    int64_t const rows = x->size(0), depth = x->size(1);
    at::Tensor codes, scales;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        codes = fresh({rows, (depth + 1) / 2}, at::kByte, *x), scales = fresh({rows, (depth + 31) / 32}, at::kByte, *x);
        status = library.quantize(dtype, x->data_ptr(), rows, depth, row_bytes(*x), codes.data_ptr(), (depth + 1) / 2, scales.data_ptr(),
                                  (depth + 31) / 32, stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(scales)));
    END_HANDLE_TH_ERRORS
}

/** dequantize(codes, scales, depth, dtype) -> x */
PyObject *dequantize(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    Left m;
    if (count != 4 || arguments[1] == Py_None || !m.found(arguments[0], arguments[1], arguments[2], home) || !THPDtype_Check(arguments[3])) Py_RETURN_NONE;
    at::ScalarType const type = ((THPDtype *)arguments[3])->scalar_type;
    nk_dtype_t const dtype = code_of(type);
    if (!dtype) Py_RETURN_NONE;
    at::Tensor x;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        int64_t const rows = m.t->size(0);
        x = fresh({rows, m.depth}, type, *m.t);
        status = library.dequantize(dtype, m.t->data_ptr(), row_bytes(*m.t), m.scales_data(), m.scales_stride(), rows, m.depth, x.data_ptr(),
                                    (nk_size_t)m.depth * x.element_size(), stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(x));
    END_HANDLE_TH_ERRORS
}

/** dots(a, scales or None, depth, image, width, depth of the image, dtype) -> c */
PyObject *dots(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    Left a;
    int64_t width, depth;
    if (count != 7 || !a.found(arguments[0], arguments[1], arguments[2], home) || !natural(arguments[4], width) || !natural(arguments[5], depth) ||
        depth != a.depth || !THPDtype_Check(arguments[6]))
        Py_RETURN_NONE;
    at::Tensor const *const image = tensor_of(arguments[3], 1, home);
    at::ScalarType const type = ((THPDtype *)arguments[6])->scalar_type;
    nk_dtype_t const dtype = code_of(type);
    if (!image || !dtype || !holds(*image, packed_size(1, width, depth))) Py_RETURN_NONE;
    at::Tensor c, workspace;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        int64_t const height = a.t->size(0);
        c = fresh({height, width}, type, *a.t);
        nk_size_t const room = library.dots_room(height, width, depth, a.scales != nullptr);
        if (room) workspace = fresh({(int64_t)room}, at::kByte, *a.t);
        status = library.dots(a.dtype, a.t->data_ptr(), row_bytes(*a.t), a.scales_data(), a.scales_stride(), image->data_ptr(), dtype, c.data_ptr(),
                              (nk_size_t)width * c.element_size(), height, width, depth, room ? workspace.data_ptr() : nullptr, room, stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(c));
    END_HANDLE_TH_ERRORS
}

/** What `experts_route` and its gradient are told, from sigmoid, renormalize, scale and, where there are groups, those. */
bool route_of(PyObject *const *arguments, bool groups, nk_amd_route_t &how) {
    int64_t sigmoid, numbers[3] = {1, 1, 1};
    if (!natural(arguments[0], sigmoid) || !PyBool_Check(arguments[1]) || !PyFloat_CheckExact(arguments[2])) return false;
    for (int i = 0; groups && i < 3; ++i)
        if (!natural(arguments[3 + i], numbers[i]) || numbers[i] > 1024) return false;
    float const scale = (float)PyFloat_AS_DOUBLE(arguments[2]);
    if (!std::isfinite(scale)) return false;
    how = {(int)sigmoid, arguments[1] == Py_True, scale, (int)numbers[0], (int)numbers[1], (int)numbers[2]};
    return true;
}

/** route(logits, top_k, bias or None, sigmoid, renormalize, scale, groups, top_groups, group_top) -> (weights, experts) */
PyObject *route(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    at::Tensor const *const logits = count == 9 ? tensor_of(arguments[0], 2, home) : nullptr, *bias = nullptr;
    nk_dtype_t const dtype = logits ? code_of(logits->scalar_type()) : nk_dtype_t(0);
    int64_t top_k;
    nk_amd_route_t how;
    if (!dtype || tracked(*logits) || !natural(arguments[1], top_k) || !route_of(arguments + 3, true, how)) Py_RETURN_NONE;
    int64_t const tokens = logits->size(0), experts = logits->size(1);
    if (arguments[2] != Py_None) {
        bias = tensor_of(arguments[2], 1, home);
        if (!bias || bias->scalar_type() != at::kFloat || bias->size(0) != experts) Py_RETURN_NONE;
    }
    if (top_k > experts) Py_RETURN_NONE;
    at::Tensor weights, chosen;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        weights = fresh({tokens, top_k}, at::kFloat, *logits), chosen = fresh({tokens, top_k}, at::kInt, *logits);
        status = library.route(dtype, logits->data_ptr(), row_bytes(*logits), tokens, experts, top_k, bias ? (float const *)bias->data_ptr() : nullptr, &how,
                               (float *)weights.data_ptr(), (nk_i32_t *)chosen.data_ptr(), stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(weights)), THPVariable_Wrap(std::move(chosen)));
    END_HANDLE_TH_ERRORS
}

/** route_backward(grad_weights, logits, experts, sigmoid, renormalize, scale) -> grad_logits */
PyObject *route_backward(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    if (count != 6) Py_RETURN_NONE;
    at::Tensor const *const grad = tensor_of(arguments[0], 2, home), *const logits = tensor_of(arguments[1], 2, home),
                           *const chosen = tensor_of(arguments[2], 2, home);
    nk_dtype_t const dtype = logits ? code_of(logits->scalar_type()) : nk_dtype_t(0);
    nk_amd_route_t how;
    if (!dtype || !grad || !chosen || !route_of(arguments + 3, false, how) || grad->scalar_type() != at::kFloat || chosen->scalar_type() != at::kInt ||
        grad->sizes() != chosen->sizes() || grad->size(0) != logits->size(0) || !grad->is_contiguous() || !chosen->is_contiguous())
        Py_RETURN_NONE;
    at::Tensor result;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        result = fresh(logits->sizes(), logits->scalar_type(), *logits);
        status = library.route_backward(dtype, logits->data_ptr(), row_bytes(*logits), logits->size(0), logits->size(1), chosen->size(1), &how,
                                        (nk_i32_t const *)chosen->data_ptr(), (float const *)grad->data_ptr(), result.data_ptr(), row_bytes(result),
                                        stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(result));
    END_HANDLE_TH_ERRORS
}

/** plan(chosen, experts) -> the plan's buffer */
PyObject *plan(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    at::Tensor const *const chosen = count == 2 ? tensor_of(arguments[0], 2, home) : nullptr;
    int64_t experts;
    if (!chosen || chosen->scalar_type() != at::kInt || !chosen->is_contiguous() || !natural(arguments[1], experts)) Py_RETURN_NONE;
    nk_size_t const slots = (nk_size_t)chosen->numel(), size = library.plan_size(slots, experts);
    if (!size) Py_RETURN_NONE;
    at::Tensor buffer;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        buffer = fresh({(int64_t)size}, at::kByte, *chosen);
        status = library.plan((nk_i32_t const *)chosen->data_ptr(), slots, experts, buffer.data_ptr(), stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(buffer));
    END_HANDLE_TH_ERRORS
}

/** experts(a, scales or None, depth, image, count, width, depth of the image, plan, tokens, top_k, experts, weights or None, dtype) -> y */
PyObject *experts(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    Left a;
    int64_t matrices, width, depth, tokens, top_k, of_plan;
    if (count != 13 || !a.found(arguments[0], arguments[1], arguments[2], home) || !natural(arguments[4], matrices) || !natural(arguments[5], width) ||
        !natural(arguments[6], depth) || !natural(arguments[8], tokens) || !natural(arguments[9], top_k) || !natural(arguments[10], of_plan) ||
        matrices != of_plan || depth != a.depth || tokens < 1 || top_k < 1 || tokens >= 1 << 30 || top_k >= 1 << 30 || !THPDtype_Check(arguments[12]))
        Py_RETURN_NONE;
    at::Tensor const *const image = tensor_of(arguments[3], 1, home), *const plan_ = tensor_of(arguments[7], 1, home), *weights = nullptr;
    at::ScalarType const type = ((THPDtype *)arguments[12])->scalar_type;
    nk_dtype_t const dtype = code_of(type);
    int64_t const slots = tokens * top_k, rows = a.t->size(0);
    if (!image || !plan_ || !dtype || (rows != tokens && rows != slots) || !holds(*image, packed_size(matrices, width, depth)) ||
        !holds(*plan_, library.plan_size(slots, matrices)))
        Py_RETURN_NONE;
    if (arguments[11] != Py_None) {
        weights = tensor_of(arguments[11], 2, home);
        if (!weights || weights->scalar_type() != at::kFloat || weights->size(0) != tokens || weights->size(1) != top_k || !weights->is_contiguous() ||
            tracked(*weights))
            Py_RETURN_NONE;
    }
    at::Tensor y, workspace;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        y = weights ? fresh({tokens, width}, type, *a.t) : fresh({tokens, top_k, width}, type, *a.t);
        nk_size_t const share = rows == tokens ? top_k : 1;
        nk_size_t const room = library.experts_room(slots, share, matrices, width, depth, a.scales != nullptr, weights != nullptr);
        if (room) workspace = fresh({(int64_t)room}, at::kByte, *a.t);
        status = library.experts(a.dtype, a.t->data_ptr(), row_bytes(*a.t), a.scales_data(), a.scales_stride(), share, image->data_ptr(), plan_->data_ptr(),
                                 slots, matrices, top_k, weights ? (float const *)weights->data_ptr() : nullptr, dtype, y.data_ptr(),
                                 (nk_size_t)width * y.element_size(), width, depth, room ? workspace.data_ptr() : nullptr, room, stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

#define CALL(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef calls[] = {CALL(bind), {"bind_packed_size", bind_packed_size, METH_O, nullptr}, CALL(quantize), CALL(dequantize), CALL(dots), CALL(route), CALL(route_backward), CALL(plan), CALL(experts),
                       {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mx_calls", nullptr, -1, calls, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__mx_calls() { return PyModule_Create(&module); }

/**
 *  @brief The calls of numkong_amd/dense.py in their ordinary form: tensors on the current GPU, results newly made.
 *  @file numkong_amd/csrc/dense_calls.cpp
 *
 *  As mx_calls.cpp: every function returns None for what it does not take, or what the library refuses, and dense.py goes its general way then.
 *  (Through ctypes a product of one token takes 11 us of the host, a norm 10; its kernel may be shorter.) Operands that autograd follows are taken as well;
 *  what the backward passes do is what dense.py's do. (In Python a small norm with its gradients took 90 us of the host.)
 */
#include "torch_calls.hpp"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "numkong_amd/dense.h"
#include "numkong_amd/hip_abi.h"

namespace {

struct Library {
    decltype(&nk_amd_mx8_quantize_async) quantize;
    decltype(&nk_amd_mx8_dequantize_async) dequantize;
    decltype(&nk_amd_rms_norm_async) norm;
    decltype(&nk_amd_rms_norm_backward_workspace_size) norm_backward_room;
    decltype(&nk_amd_rms_norm_backward_async) norm_backward;
    decltype(&nk_amd_linear_workspace_size) linear_room;
    decltype(&nk_amd_linear_async) linear;
    decltype(&nk_amd_linear_backward_workspace_size) linear_backward_room;
    decltype(&nk_amd_linear_backward_async) linear_backward;
    decltype(&nk_hip_last_error) last_error;
};
Library library;

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

/** A float operand that may be missing: false, if it is not what the call takes. */
bool floats(PyObject *argument, int64_t dims, Home &home, at::Tensor const *&t) {
    t = nullptr;
    if (argument == Py_None) return true;
    t = tensor_of(argument, dims, home);
    return t && code_of(t->scalar_type());
}
/** Does autograd follow one of them? */
template <class... Tensors>
bool followed(Tensors... t) { return ((t && tracked(*t)) || ...); }
nk_dtype_t dtype_of(at::Tensor const *t) { return t ? code_of(t->scalar_type()) : nk_dtype_t(0); }
void *data_of(at::Tensor const *t) { return t ? t->data_ptr() : nullptr; }
nk_size_t stride_of(at::Tensor const *t) { return t ? row_bytes(*t) : 0; }
bool is_vector(at::Tensor const *t, int64_t length) { return !t || (t->size(0) == length && t->is_contiguous()); }
bool has_shape(at::Tensor const *t, int64_t rows, int64_t columns) { return !t || (t->size(0) == rows && t->size(1) == columns); }
bool truth(PyObject *argument, bool &value) { return value = argument == Py_True, PyBool_Check(argument); }
/** A type that may be None: then it is `otherwise`. */
bool type_of(PyObject *argument, at::ScalarType otherwise, at::ScalarType &type) {
    type = otherwise;
    if (argument == Py_None) return true;
    if (!THPDtype_Check(argument)) return false;
    type = ((THPDtype *)argument)->scalar_type;
    return code_of(type) != 0;
}
at::Tensor strided(int64_t rows, int64_t columns, int64_t step, at::ScalarType type, at::Tensor const &like) {
    return at::empty_strided({rows, columns}, {std::max<int64_t>((columns + step - 1) / step * step, 1), 1}, at::TensorOptions().dtype(type).device(like.device()));
}
PyObject *wrapped(at::Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(std::move(t));
    Py_RETURN_NONE;
}

/** A matrix of a product: floats, or codes with scales. */
struct Matrix {
    at::Tensor const *t = nullptr, *scales = nullptr;
    bool found(PyObject *values, PyObject *its_scales, Home &home) {
        if (!(t = tensor_of(values, 2, home))) return false;
        if (its_scales == Py_None) return code_of(t->scalar_type());
        scales = tensor_of(its_scales, 2, home);
        return scales && t->scalar_type() == at::kFloat8_e4m3fn && scales->scalar_type() == at::kByte && scales->size(0) == t->size(0) &&
               scales->size(1) == (t->size(1) + 31) / 32;
    }
    nk_dtype_t dtype() const { return scales ? nk_e4m3_k : code_of(t->scalar_type()); }
};

/** quantize(x) -> (codes, scales) */
PyObject *quantize(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    at::Tensor const *const x = count == 1 ? tensor_of(arguments[0], 2, home) : nullptr;
    if (!dtype_of(x)) Py_RETURN_NONE;
    int64_t const rows = x->size(0), depth = x->size(1);
    at::Tensor codes, scales;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        codes = strided(rows, depth, 16, at::kFloat8_e4m3fn, *x), scales = strided(rows, (depth + 31) / 32, 4, at::kByte, *x);
        status = library.quantize(dtype_of(x), x->data_ptr(), rows, depth, row_bytes(*x), codes.data_ptr(), row_bytes(codes), scales.data_ptr(), row_bytes(scales),
                                  stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return Py_BuildValue("NN", wrapped(codes), wrapped(scales));
    END_HANDLE_TH_ERRORS
}

/** dequantize(codes, scales, dtype) -> x */
PyObject *dequantize(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    Matrix m;
    at::ScalarType type;
    if (count != 3 || arguments[1] == Py_None || !m.found(arguments[0], arguments[1], home) || !type_of(arguments[2], at::kFloat, type)) Py_RETURN_NONE;
    at::Tensor x;
    int status;
    {
        WithoutLock unlocked;
        at::AutoDispatchBelowADInplaceOrView guard;
        x = fresh(m.t->sizes(), type, *m.t);
        status = library.dequantize(code_of(type), m.t->data_ptr(), row_bytes(*m.t), m.scales->data_ptr(), row_bytes(*m.scales), m.t->size(0), m.t->size(1), x.data_ptr(),
                                    row_bytes(x), stream_of(home));
    }
    if (status) Py_RETURN_NONE;
    return wrapped(x);
    END_HANDLE_TH_ERRORS
}

void *stream_on(at::Tensor const &t) { return (void *)c10::hip::getCurrentHIPStream((c10::DeviceIndex)t.get_device()).stream(); }
typedef std::optional<at::Tensor> Maybe;
at::Tensor const *present(at::Tensor const &t) { return t.defined() ? &t : nullptr; }
at::Tensor const *present(Maybe const &t) { return t ? &*t : nullptr; }
Maybe maybe(at::Tensor const *t) { return t ? Maybe(*t) : Maybe(); }
/** Is a gradient of input `i` asked for? (Autograd counts those that there are.) */
bool needs(torch::autograd::AutogradContext *ctx, int64_t i) {
    int64_t const there = ctx->saved_data["there"].toInt();
    return there >> i & 1 && ctx->needs_input_grad((size_t)__builtin_popcountll((uint64_t)there & ((1ull << i) - 1)));
}
void check(int status, char const *where) { TORCH_CHECK(!status, where, ": ", library.last_error()); }
/** A gradient as the kernels read it: autograd hands on expanded and transposed ones too, and ones with a tangent. */
at::Tensor rows_of(at::Tensor const &t) {
    TORCH_CHECK(!t._fw_grad(0).defined(), "the operators have no forward-mode derivatives: a gradient has a tangent");
    return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous();
}
/** Gradients that no gradient passes: asked for one, they say so. */
torch::autograd::variable_list once(torch::autograd::variable_list found) {
    if (!c10::GradMode::is_enabled()) return found;
    torch::autograd::variable_list there;
    for (auto const &t : found)
        if (t.defined()) there.push_back(t.detach().set_requires_grad(true));
    auto const error = std::make_shared<torch::autograd::DelayedError>("the gradients of the dense operators have no gradients of their own", (int)there.size());
    if (there.empty()) return found;
    there = (*error)(std::move(there));
    size_t next = 0;
    for (auto &t : found)
        if (t.defined()) t = there[next++];
    return found;
}

int run_norm(at::Tensor const &x, at::Tensor const *weight, at::Tensor const *residual, float eps, at::ScalarType type, bool mx8, at::Tensor &y, at::Tensor &scales, at::Tensor &total) {
    at::AutoDispatchBelowADInplaceOrView guard;
    int64_t const rows = x.size(0), depth = x.size(1);
    if (mx8) y = strided(rows, depth, 16, at::kFloat8_e4m3fn, x), scales = strided(rows, (depth + 31) / 32, 4, at::kByte, x);
    else y = fresh({rows, depth}, type, x);
    if (residual) total = fresh({rows, depth}, x.scalar_type(), x);
    nk_amd_rms_norm_t const n = {(nk_size_t)rows, (nk_size_t)depth, eps, dtype_of(&x), x.data_ptr(), row_bytes(x), data_of(residual),
                                 stride_of(residual), residual ? total.data_ptr() : nullptr, residual ? row_bytes(total) : 0, dtype_of(weight), data_of(weight),
                                 mx8 ? nk_e4m3_k : code_of(type), y.data_ptr(), row_bytes(y), mx8 ? scales.data_ptr() : nullptr, mx8 ? row_bytes(scales) : 0};
    return library.norm(&n, stream_on(x));
}
int run_norm_backward(at::Tensor const &grad, at::Tensor const &total, at::Tensor const *weight, at::Tensor const *grad_total, float eps, bool need_weight, at::Tensor &of_x,
                      at::Tensor &of_weight) {
    at::AutoDispatchBelowADInplaceOrView guard;
    int64_t const rows = total.size(0), depth = total.size(1);
    at::Tensor workspace;
    of_x = fresh({rows, depth}, total.scalar_type(), total);
    if (need_weight && weight) of_weight = fresh({depth}, weight->scalar_type(), total);
    nk_amd_rms_norm_backward_t const n = {(nk_size_t)rows, (nk_size_t)depth, eps, dtype_of(&total), total.data_ptr(), row_bytes(total),
                                          dtype_of(weight), data_of(weight), dtype_of(&grad), grad.data_ptr(), row_bytes(grad), data_of(grad_total),
                                          stride_of(grad_total), of_x.data_ptr(), row_bytes(of_x), of_weight.defined() ? of_weight.data_ptr() : nullptr};
    nk_size_t const room = library.norm_backward_room(&n);
    if (room) workspace = fresh({(int64_t)room}, at::kByte, total);
    return library.norm_backward(&n, room ? workspace.data_ptr() : nullptr, room, stream_on(total));
}
struct NormWithGradient : torch::autograd::Function<NormWithGradient> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, at::Tensor x, Maybe weight, Maybe residual, double eps, at::ScalarType type) {
        at::Tensor y, scales, total;
        check(run_norm(x, present(weight), present(residual), (float)eps, type, false, y, scales, total), "rms_norm");
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual ? total : x, weight ? *weight : at::Tensor()});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["there"] = int64_t(1 | (weight ? 2 : 0) | (residual ? 4 : 0));
        return residual ? torch::autograd::variable_list {y, total} : torch::autograd::variable_list {y};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        auto const saved = ctx->get_saved_variables();
        at::Tensor const &total = saved[0], &weight = saved[1];
        at::Tensor of_x, of_weight, of_total = grads.size() > 1 && grads[1].defined() ? rows_of(grads[1]) : at::Tensor();
        if (!grads[0].defined()) { // nothing came back through y
            of_x = of_total;
            if (weight.defined() && needs(ctx, 1)) of_weight = at::zeros_like(weight);
        } else
            check(run_norm_backward(rows_of(grads[0]), total, present(weight), present(of_total), (float)ctx->saved_data["eps"].toDouble(), needs(ctx, 1), of_x, of_weight),
                  "rms_norm_backward");
        return once({needs(ctx, 0) ? of_x : at::Tensor(), of_weight, needs(ctx, 2) ? of_x : at::Tensor(), at::Tensor(), at::Tensor()});
    }
};

/** norm(x, weight or None, residual or None, eps, dtype or None, mx8) -> (y, scales or None, total or None) */
PyObject *norm(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    at::Tensor const *x, *weight, *residual;
    at::ScalarType type;
    bool mx8;
    if (count != 6 || !floats(arguments[0], 2, home, x) || !x || !floats(arguments[1], 1, home, weight) || !floats(arguments[2], 2, home, residual) ||
        !PyFloat_CheckExact(arguments[3]) || !type_of(arguments[4], x->scalar_type(), type) || !truth(arguments[5], mx8))
        Py_RETURN_NONE;
    int64_t const rows = x->size(0), depth = x->size(1);
    if (!is_vector(weight, depth) || !has_shape(residual, rows, depth) || (residual && residual->scalar_type() != x->scalar_type())) Py_RETURN_NONE;
    float const eps = (float)PyFloat_AS_DOUBLE(arguments[3]);
    at::Tensor y, scales, total;
    if (followed(x, weight, residual)) {
        if (mx8 || !(eps >= 0) || eps > std::numeric_limits<float>::max() || depth > 32768) Py_RETURN_NONE;
        WithoutLock unlocked;
        auto found = NormWithGradient::apply(*x, maybe(weight), maybe(residual), (double)eps, type);
        y = found[0];
        if (residual) total = found[1];
    } else {
        int status;
        {
            WithoutLock unlocked;
            status = run_norm(*x, weight, residual, eps, type, mx8, y, scales, total);
        }
        if (status) Py_RETURN_NONE;
    }
    return Py_BuildValue("NNN", wrapped(y), wrapped(scales), wrapped(total));
    END_HANDLE_TH_ERRORS
}

/** norm_backward(grad, total, weight or None, grad_total or None, eps, need_weight) -> (of x, of weight or None) */
PyObject *norm_backward(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    at::Tensor const *grad, *total, *weight, *grad_total;
    bool need_weight;
    if (count != 6 || !floats(arguments[0], 2, home, grad) || !grad || !floats(arguments[1], 2, home, total) || !total || !floats(arguments[2], 1, home, weight) ||
        !floats(arguments[3], 2, home, grad_total) || !PyFloat_CheckExact(arguments[4]) || !truth(arguments[5], need_weight))
        Py_RETURN_NONE;
    int64_t const rows = total->size(0), depth = total->size(1);
    if (!has_shape(grad, rows, depth) || !is_vector(weight, depth) || !has_shape(grad_total, rows, depth) || (grad_total && grad_total->scalar_type() != total->scalar_type()))
        Py_RETURN_NONE;
    if (followed(grad, total, weight, grad_total)) Py_RETURN_NONE;
    at::Tensor of_x, of_weight;
    int status;
    {
        WithoutLock unlocked;
        status = run_norm_backward(*grad, *total, weight, grad_total, (float)PyFloat_AS_DOUBLE(arguments[4]), need_weight, of_x, of_weight);
    }
    if (status) Py_RETURN_NONE;
    return Py_BuildValue("NN", wrapped(of_x), wrapped(of_weight));
    END_HANDLE_TH_ERRORS
}

int run_linear(Matrix const &a, Matrix const &w, Matrix const &up, at::Tensor const *bias, int activation, at::Tensor const *residual, at::ScalarType type, bool sums, at::Tensor &c,
               at::Tensor &pre, at::Tensor &pre_up) {
    at::AutoDispatchBelowADInplaceOrView guard;
    int64_t const height = a.t->size(0), depth = a.t->size(1), width = w.t->size(0);
    bool const gated = up.t;
    at::Tensor workspace;
    c = fresh({height, width}, type, *a.t);
    if (sums) pre = fresh({height, width}, at::kFloat, *a.t);
    if (sums && gated) pre_up = fresh({height, width}, at::kFloat, *a.t);
    nk_amd_linear_t const l = {(nk_size_t)height, (nk_size_t)width, (nk_size_t)depth, gated, a.dtype(), a.t->data_ptr(), row_bytes(*a.t), data_of(a.scales), stride_of(a.scales),
                               w.dtype(), w.t->data_ptr(), row_bytes(*w.t), data_of(w.scales), stride_of(w.scales), data_of(up.t), stride_of(up.t), data_of(up.scales),
                               stride_of(up.scales), activation, dtype_of(bias), data_of(bias), dtype_of(residual), data_of(residual), stride_of(residual),
                               code_of(type), c.data_ptr(), row_bytes(c), sums ? (float *)pre.data_ptr() : nullptr, sums && gated ? (float *)pre_up.data_ptr() : nullptr,
                               sums ? (nk_size_t)width * 4 : 0};
    nk_size_t const room = library.linear_room(&l);
    if (room) workspace = fresh({(int64_t)room}, at::kByte, *a.t);
    return library.linear(&l, room ? workspace.data_ptr() : nullptr, room, stream_on(*a.t));
}
/** `up` and the sums: NULL, if there are none; of_bias: of that type, if `biased`. */
int run_linear_backward(at::Tensor const &grad, at::Tensor const &a, at::Tensor const &w, at::Tensor const *up, at::Tensor const *sums, at::Tensor const *up_sums, int activation, bool need_a,
                        bool need_w, bool need_up, bool biased, at::ScalarType bias_type, at::Tensor &of_a, at::Tensor &of_w, at::Tensor &of_up, at::Tensor &of_bias) {
    at::AutoDispatchBelowADInplaceOrView guard;
    int64_t const height = a.size(0), depth = a.size(1), width = w.size(0);
    at::Tensor workspace;
    if (need_a) of_a = fresh({height, depth}, a.scalar_type(), a);
    if (need_w) of_w = fresh({width, depth}, a.scalar_type(), a);
    if (need_up && up) of_up = fresh({width, depth}, a.scalar_type(), a);
    if (biased) of_bias = fresh({width}, bias_type, a);
    auto const data = [](at::Tensor const &t) { return t.defined() ? t.data_ptr() : nullptr; };
    nk_size_t const row = (nk_size_t)depth * 2;
    nk_amd_linear_backward_t const l = {(nk_size_t)height, (nk_size_t)width, (nk_size_t)depth, up != nullptr, dtype_of(&a), a.data_ptr(), row_bytes(a), w.data_ptr(), row_bytes(w),
                                        data_of(up), stride_of(up), activation, (float const *)data_of(sums), (float const *)data_of(up_sums), stride_of(sums),
                                        dtype_of(&grad), grad.data_ptr(), row_bytes(grad), data(of_a), row, data(of_w), row, data(of_up), row,
                                        biased ? code_of(bias_type) : nk_dtype_t(0), data(of_bias)};
    nk_size_t const room = library.linear_backward_room(&l);
    if (room) workspace = fresh({(int64_t)room}, at::kByte, a);
    return library.linear_backward(&l, room ? workspace.data_ptr() : nullptr, room, stream_on(a));
}
Matrix plain(at::Tensor const *t) {
    Matrix m;
    m.t = t;
    return m;
}
/** Both products: a, w, w_up, bias and residual are the inputs; the gradient of the residual alone does without the sums. */
struct LinearWithGradient : torch::autograd::Function<LinearWithGradient> {
    static at::Tensor forward(torch::autograd::AutogradContext *ctx, at::Tensor a, at::Tensor w, Maybe up, Maybe bias, Maybe residual, int64_t activation, at::ScalarType type) {
        bool const keeps = up || (activation && (a.requires_grad() || w.requires_grad() || (bias && bias->requires_grad())));
        at::Tensor c, pre, pre_up;
        check(run_linear(plain(&a), plain(&w), plain(present(up)), present(bias), (int)activation, present(residual), type, keeps, c, pre, pre_up), "linear");
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({a, w, up ? *up : at::Tensor(), pre, pre_up});
        ctx->saved_data["there"] = int64_t(3 | (up ? 4 : 0) | (bias ? 8 : 0) | (residual ? 16 : 0));
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["bias"] = bias ? (int64_t)bias->scalar_type() : int64_t(-1);
        ctx->saved_data["residual"] = residual ? (int64_t)residual->scalar_type() : int64_t(-1);
        return c;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        torch::autograd::variable_list found(7);
        if (!grads[0].defined()) return found;
        auto const saved = ctx->get_saved_variables();
        bool const need[4] = {needs(ctx, 0), needs(ctx, 1), needs(ctx, 2), needs(ctx, 3)};
        int64_t const bias = ctx->saved_data["bias"].toInt(), residual = ctx->saved_data["residual"].toInt();
        if (need[0] || need[1] || need[2] || need[3])
            check(run_linear_backward(rows_of(grads[0]), saved[0], saved[1], present(saved[2]), present(saved[3]), present(saved[4]), (int)ctx->saved_data["activation"].toInt(), need[0], need[1],
                                      need[2], bias >= 0 && need[3], bias >= 0 ? (at::ScalarType)bias : at::kFloat, found[0], found[1], found[2], found[3]),
                  "linear_backward");
        if (residual >= 0 && needs(ctx, 4)) found[4] = grads[0].to((at::ScalarType)residual);
        return once(std::move(found));
    }
};

/** linear(a, its scales or None, w, its or None, w_up or None, its or None, bias or None, activation, residual or None, dtype or None, sums)
 *  -> (y, sums or None, the other matrix's or None) */
PyObject *linear(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    Matrix a, w, up;
    at::Tensor const *bias, *residual;
    at::ScalarType type;
    int64_t activation;
    bool sums;
    if (count != 11 || !a.found(arguments[0], arguments[1], home) || !w.found(arguments[2], arguments[3], home)) Py_RETURN_NONE;
    bool const gated = arguments[4] != Py_None, mx8 = w.scales;
    if ((gated && !up.found(arguments[4], arguments[5], home)) || !floats(arguments[6], 1, home, bias) || !natural(arguments[7], activation) || activation > nk_amd_gelu_tanh ||
        !floats(arguments[8], 2, home, residual) || !type_of(arguments[9], a.scales || a.t->scalar_type() == at::kFloat ? at::kBFloat16 : a.t->scalar_type(), type) ||
        !truth(arguments[10], sums))
        Py_RETURN_NONE;
    int64_t const height = a.t->size(0), depth = a.t->size(1), width = w.t->size(0);
    if (w.t->size(1) != depth || (a.scales && !mx8) || (!mx8 && a.t->scalar_type() != w.t->scalar_type()) || (mx8 && type == at::kFloat) ||
        (gated && (up.t->sizes() != w.t->sizes() || up.t->scalar_type() != w.t->scalar_type())) || !is_vector(bias, width) || !has_shape(residual, height, width))
        Py_RETURN_NONE;
    at::Tensor c, pre, pre_up;
    int status = 0;
    if (followed(a.scales ? nullptr : a.t, mx8 ? nullptr : w.t, mx8 ? nullptr : up.t, bias, residual)) {
        int64_t const most = 1 << 22; // (the backward pass's)
        if (mx8 || sums || height >= most || width >= most || depth >= most || w.t->scalar_type() == at::kFloat) Py_RETURN_NONE;
        WithoutLock unlocked;
        c = LinearWithGradient::apply(*a.t, *w.t, maybe(up.t), maybe(bias), maybe(residual), activation, type);
    } else {
        WithoutLock unlocked;
        status = run_linear(a, w, up, bias, (int)activation, residual, type, sums, c, pre, pre_up);
    }
    if (status) Py_RETURN_NONE;
    return Py_BuildValue("NNN", wrapped(c), wrapped(pre), wrapped(pre_up));
    END_HANDLE_TH_ERRORS
}

/** linear_backward(grad, a, w, w_up or None, sums or None, the other's or None, activation, need_a, need_w, need_up, bias's dtype or None)
 *  -> (of a, of w, of w_up, of the bias), None where one is not needed */
PyObject *linear_backward(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    Home home;
    at::Tensor const *grad, *a, *w, *up, *sums, *up_sums;
    int64_t activation;
    bool need_a, need_w, need_up;
    at::ScalarType bias_type;
    if (count != 11 || !floats(arguments[0], 2, home, grad) || !grad || !floats(arguments[1], 2, home, a) || !a || !floats(arguments[2], 2, home, w) || !w ||
        !floats(arguments[3], 2, home, up) || !floats(arguments[4], 2, home, sums) || !floats(arguments[5], 2, home, up_sums) || !natural(arguments[6], activation) ||
        activation > nk_amd_gelu_tanh || !truth(arguments[7], need_a) || !truth(arguments[8], need_w) || !truth(arguments[9], need_up) ||
        !type_of(arguments[10], at::kFloat, bias_type))
        Py_RETURN_NONE;
    int64_t const height = a->size(0), depth = a->size(1), width = w->size(0);
    bool const gated = up, biased = arguments[10] != Py_None;
    if (a->scalar_type() == at::kFloat || a->scalar_type() != w->scalar_type() || w->size(1) != depth || !has_shape(grad, height, width) ||
        (gated && (up->sizes() != w->sizes() || up->scalar_type() != w->scalar_type())) || !has_shape(sums, height, width) || !has_shape(up_sums, height, width) ||
        (sums && sums->scalar_type() != at::kFloat) || (up_sums && (up_sums->scalar_type() != at::kFloat || !sums || row_bytes(*sums) != row_bytes(*up_sums))) ||
        ((gated || activation) && !sums) || (gated && !up_sums))
        Py_RETURN_NONE;
    if (followed(grad, a, w, up, sums, up_sums)) Py_RETURN_NONE;
    at::Tensor of_a, of_w, of_up, of_bias;
    int status;
    {
        WithoutLock unlocked;
        status = run_linear_backward(*grad, *a, *w, up, sums, up_sums, (int)activation, need_a, need_w, need_up, biased, bias_type, of_a, of_w, of_up, of_bias);
    }
    if (status) Py_RETURN_NONE;
    return Py_BuildValue("NNNN", wrapped(of_a), wrapped(of_w), wrapped(of_up), wrapped(of_bias));
    END_HANDLE_TH_ERRORS
}

#define CALL(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef calls[] = {CALL(bind), CALL(quantize), CALL(dequantize), CALL(norm), CALL(norm_backward), CALL(linear), CALL(linear_backward), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dense_calls", nullptr, -1, calls, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__dense_calls() { return PyModule_Create(&module); }

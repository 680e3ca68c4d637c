// norm_host.cpp -- layer_norm's usual call in C++: checks, allocation, launch and the autograd node.
//
// A small layer norm takes the GPU a few microseconds.  Host time of a call with a residual and of
// its backward, 2048 x 768: 24 and 59 us through a Python autograd function, 7 and 35 here (a
// product with a vector and its backward: 37 together).  layer_norm() below returns None for
// whatever is not the usual call (another device, a strided or empty tensor, a tensor subclass or
// one with a forward-mode tangent, under a trace, an argument to refuse), and mi_adamw.norm takes
// its Python path, which does or reports it.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <optional>
#include <string>

#include "mi_adamw.h"

namespace mi_adamw_host {

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    int (*forward)(const mi_adamw_layer_norm_args*, void*) = nullptr;
    int64_t (*workspace)(int64_t, int64_t) = nullptr;
    int (*grad)(const mi_adamw_layer_norm_grad_args*, void*) = nullptr;
    const char* (*strerror)(int) = nullptr;
};
Api g_api;
PyObject* g_error = nullptr;        // MiAdamwError

int32_t code_of(at::ScalarType t) {
    return t == at::kBFloat16 ? MI_ADAMW_DTYPE_BF16 : MI_ADAMW_DTYPE_F32;
}
bool type_ok(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

void* stream_of(const Tensor& t) {
    return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// MiAdamwError, as mi_adamw._lib.check raises it; a backward calls this without the GIL.
void check(int code, const char* what) {
    if (code == MI_ADAMW_OK) return;
    const std::string text = std::string(what) + " failed: " + g_api.strerror(code) + " (code " +
                             std::to_string(code) + ")";
    pybind11::gil_scoped_acquire gil;
    PyErr_SetString(g_error, text.c_str());
    python_error error;
    error.persist();
    throw error;
}

struct Results {
    Tensor y, sum, stats;       // stats: [2][rows], mean and rstd
};

Results forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias,
                double eps, at::ScalarType out, bool stats) {
    Results r;
    r.y = at::empty(x.sizes(), x.options().dtype(out));
    mi_adamw_layer_norm_args a{};
    a.x = x.data_ptr();
    a.y = r.y.data_ptr();
    a.hidden = x.size(-1);
    a.rows = x.numel() / a.hidden;
    a.x_row = a.residual_row = a.hidden;
    a.eps = static_cast<float>(eps);
    a.x_dtype = code_of(x.scalar_type());
    a.y_dtype = code_of(out);
    if (weight.defined()) a.weight = static_cast<const float*>(weight.data_ptr());
    if (bias.defined()) a.bias = static_cast<const float*>(bias.data_ptr());
    if (residual.defined()) {
        r.sum = at::empty(x.sizes(), x.options().dtype(c10::promoteTypes(
                                         x.scalar_type(), residual.scalar_type())));
        a.residual = residual.data_ptr();
        a.sum = r.sum.data_ptr();
        a.residual_dtype = code_of(residual.scalar_type());
    }
    if (stats) {
        r.stats = at::empty({2, a.rows}, x.options().dtype(at::kFloat));
        a.mean = static_cast<float*>(r.stats.data_ptr());
        a.rstd = a.mean + a.rows;
    }
    check(g_api.forward(&a, stream_of(x)), "mi_adamw_layer_norm");
    return r;
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x,
                                 const std::optional<Tensor>& residual_,
                                 const std::optional<Tensor>& weight_,
                                 const std::optional<Tensor>& bias_, double eps, int64_t out) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const Tensor residual = residual_.value_or(Tensor()), weight = weight_.value_or(Tensor()),
                     bias = bias_.value_or(Tensor());
        ctx->saved_data["weight"] = weight.defined();
        ctx->saved_data["bias"] = bias.defined();
        Results r = mi_adamw_host::forward(x, residual, weight, bias, eps,
                                           static_cast<at::ScalarType>(out), true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["x"] = static_cast<int64_t>(x.scalar_type());
        if (!residual.defined()) {
            ctx->save_for_backward({x, weight, r.stats});
            return {r.y};
        }
        ctx->saved_data["residual"] = static_cast<int64_t>(residual.scalar_type());
        ctx->save_for_backward({r.sum, weight, r.stats});
        return {r.y, r.sum};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool second = at::GradMode::is_enabled();
        variable_list out = gradients(ctx, grads);
        if (second) {
            // under create_graph: using these gradients' gradients raises
            variable_list in;
            for (Tensor& t : out)
                if (t.defined()) in.push_back(t.detach().set_requires_grad(true));
            auto error = std::make_shared<torch::autograd::DelayedError>(
                "mi_adamw.layer_norm has no second derivative", static_cast<int>(in.size()));
            in = (*error)(std::move(in));
            size_t k = 0;
            for (Tensor& t : out)
                if (t.defined()) t = in[k++];
        }
        return out;
    }

    static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
        at::AutoDispatchBelowADInplaceOrView guard;
        variable_list result(6);
        Tensor dy = grads[0], ds = grads.size() > 1 ? grads[1] : Tensor();
        if (!dy.defined() && !ds.defined()) return result;
        // a saved-tensor hook may give them back at other strides
        auto saved = ctx->get_saved_variables();
        for (Tensor& t : saved)
            if (t.defined()) t = t.contiguous();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        const auto x_type = static_cast<at::ScalarType>(ctx->saved_data["x"].toInt());
        const bool with_residual = ctx->saved_data.count("residual") != 0;
        mi_adamw_layer_norm_grad_args a{};
        a.hidden = x.size(-1);
        a.rows = x.numel() / a.hidden;
        a.x_row = a.dy_row = a.dsum_row = a.hidden;
        dy = dy.defined() ? dy.contiguous() : at::zeros(x.sizes(), x.options().dtype(at::kFloat));
        a.x = x.data_ptr();
        a.x_dtype = code_of(x.scalar_type());
        a.dy = dy.data_ptr();
        a.dy_dtype = code_of(dy.scalar_type());
        a.mean = static_cast<const float*>(stats.data_ptr());
        a.rstd = a.mean + a.rows;
        if (weight.defined()) a.weight = static_cast<const float*>(weight.data_ptr());
        if (ds.defined()) {
            ds = ds.contiguous();
            a.dsum = ds.data_ptr();
        }
        // the node's edges: the tensors that were given, in order
        size_t edge = 0;
        const bool need_x = ctx->needs_input_grad(edge++);
        const bool need_r = with_residual && ctx->needs_input_grad(edge++);
        const bool need_w = ctx->saved_data["weight"].toBool() && ctx->needs_input_grad(edge++);
        const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(edge++);
        Tensor dx, dr;
        if (need_x || need_r) {
            const auto r_type = with_residual
                ? static_cast<at::ScalarType>(ctx->saved_data["residual"].toInt()) : x_type;
            const auto first = need_x ? x_type : r_type;
            dx = at::empty(x.sizes(), x.options().dtype(first));
            a.dx = dx.data_ptr();
            a.dx_dtype = code_of(first);
            if (need_x && need_r && r_type != first) {
                dr = at::empty(x.sizes(), x.options().dtype(r_type));
                a.dresidual = dr.data_ptr();
                a.dresidual_dtype = code_of(r_type);
            }
        }
        Tensor dw, db, partials;
        if (need_w) {
            dw = at::empty({a.hidden}, x.options().dtype(at::kFloat));
            a.dweight = static_cast<float*>(dw.data_ptr());
        }
        if (need_b) {
            db = at::empty({a.hidden}, x.options().dtype(at::kFloat));
            a.dbias = static_cast<float*>(db.data_ptr());
        }
        if (dw.defined() || db.defined()) {
            partials = at::empty({g_api.workspace(a.rows, a.hidden)},
                                 x.options().dtype(at::kByte));
            a.partials = static_cast<float*>(partials.data_ptr());
        }
        if (a.dx || a.dweight || a.dbias)
            check(g_api.grad(&a, stream_of(x)), "mi_adamw_layer_norm_grad");
        // one tensor serves both addends where their types agree, as an addition's backward gives
        if (need_x) result[0] = dx;
        if (need_r) result[1] = dr.defined() ? dr : dx;
        result[2] = dw;
        result[3] = db;
        return result;
    }
};

// A tensor the usual call takes, or None for an absent one.  False: take the Python path.
bool take(PyObject* o, Tensor& t) {
    if (o == Py_None) return true;
    if (!THPVariable_CheckExact(o)) return false;
    t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == c10::kStrided && t.is_contiguous() && t.numel() > 0 &&
           !t._fw_grad(0).defined();
}

}  // namespace

// layer_norm(x, weight, bias, eps, residual, out_dtype) -> y, (y, sum) or None
PyObject* py_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 6) {
        PyErr_SetString(PyExc_TypeError, "layer_norm(x, weight, bias, eps, residual, out_dtype)");
        return nullptr;
    }
    if (!g_api.forward || !PyFloat_CheckExact(args[3]) || torch::jit::tracer::isTracing() ||
        (args[5] != Py_None && !THPDtype_Check(args[5])))
        Py_RETURN_NONE;
    // every exception keeps its type: a hook's (a checkpoint ends its recomputation by one from
    // the saving of tensors), the allocator's, the library's
    HANDLE_TH_ERRORS
    {
        Tensor x, weight, bias, residual;
        if (!take(args[0], x) || !x.defined() || !take(args[1], weight) || !take(args[2], bias) ||
            !take(args[4], residual))
            Py_RETURN_NONE;
        const double eps = PyFloat_AS_DOUBLE(args[3]);
        const auto out = args[5] == Py_None
            ? at::autocast::is_autocast_enabled(at::kCUDA) ? at::kFloat : x.scalar_type()
            : reinterpret_cast<THPDtype*>(args[5])->scalar_type;
        if (!(eps >= 0.0) || !std::isfinite(static_cast<float>(eps)) || x.dim() < 1 || !type_ok(x.scalar_type()) ||
            !type_ok(out) || x.size(-1) > (1 << 24) || x.numel() / x.size(-1) >= (1 << 23) ||
            c10::hip::getCurrentHIPStream().device_index() != x.device().index())
            Py_RETURN_NONE;
        for (const Tensor* t : {&weight, &bias})
            if (t->defined() && (t->dim() != 1 || t->size(0) != x.size(-1) ||
                                 t->scalar_type() != at::kFloat || t->device() != x.device()))
                Py_RETURN_NONE;
        if (residual.defined() && (residual.sizes() != x.sizes() ||
                                   !type_ok(residual.scalar_type()) ||
                                   residual.device() != x.device()))
            Py_RETURN_NONE;
        const bool grad = at::GradMode::is_enabled() &&
                          (x.requires_grad() || (residual.defined() && residual.requires_grad()) ||
                           (weight.defined() && weight.requires_grad()) ||
                           (bias.defined() && bias.requires_grad()));
        variable_list got;
        if (grad) {
            auto given = [](const Tensor& t) {
                return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
            };
            got = LayerNorm::apply(x, given(residual), given(weight), given(bias), eps,
                                   static_cast<int64_t>(out));
        } else {
            Results r = forward(x, residual, weight, bias, eps, out, false);
            got = {r.y, r.sum};
        }
        if (!residual.defined()) return THPVariable_Wrap(got[0]);
        PyObject* y = THPVariable_Wrap(got[0]);
        PyObject* s = y ? THPVariable_Wrap(got[1]) : nullptr;
        PyObject* both = s ? PyTuple_Pack(2, y, s) : nullptr;
        Py_XDECREF(y);
        Py_XDECREF(s);
        return both;
    }
    END_HANDLE_TH_ERRORS
}

// bind_layer_norm(forward, workspace, grad, strerror, error): addresses of the library's functions,
// and the class of its errors
PyObject* py_bind_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 5 || !PyExceptionClass_Check(args[4])) {
        PyErr_SetString(PyExc_TypeError,
                        "bind_layer_norm(forward, workspace, grad, strerror, error)");
        return nullptr;
    }
    void* p[4];
    for (int k = 0; k < 4; ++k) {
        p[k] = PyLong_AsVoidPtr(args[k]);
        if (!p[k]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a function is missing");
            return nullptr;
        }
    }
    g_api.forward = reinterpret_cast<decltype(g_api.forward)>(p[0]);
    g_api.workspace = reinterpret_cast<decltype(g_api.workspace)>(p[1]);
    g_api.grad = reinterpret_cast<decltype(g_api.grad)>(p[2]);
    g_api.strerror = reinterpret_cast<decltype(g_api.strerror)>(p[3]);
    Py_INCREF(args[4]);
    Py_XSETREF(g_error, args[4]);
    Py_RETURN_NONE;
}

}  // namespace mi_adamw_host

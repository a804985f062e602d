// autograd_adamw.h — the plain calls of the optimiser's step, a part of autograd.cpp (after autograd_paged.h).
//
// It takes Python's own lists: turned into vectors of tensors and numbers by the bindings, and looked over in
// Python before, a step of four tensors took 8.4 us, here 6.5, and one of 28, clipped, 24.2 and 20.6 (kernels and tables
// as they were then; now 6.0 to 6.2, and 14.2 to 16.5).
#pragma once

#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

// A tensor with memory of its own.
bool is_strided(const Tensor &t, const at::Device &dev) {
    return t.defined() && t.layout() == at::kStrided && t.device() == dev &&
           !t.key_set().has(c10::DispatchKey::Python) && t.unsafeGetTensorImpl()->has_storage();
}
// In one run.
bool is_dense(const Tensor &t, const at::Device &dev) {
    return is_strided(t, dev) && (t.is_contiguous() || t.is_non_overlapping_and_dense());
}
// The shape of a dense tensor, laid out alike.
bool is_like(const Tensor &t, const Tensor &p, const at::Device &dev) {
    return is_strided(t, dev) && t.sizes() == p.sizes() && t.strides() == p.strides();
}

// Item i of a list or tuple of n; of anything else, or of another length, none.
struct Items {
    PyObject *all;
    bool right;
    Items(py::handle x, Py_ssize_t n) : all(x.ptr()) {
        right = PyList_CheckExact(all) ? PyList_GET_SIZE(all) == n : PyTuple_CheckExact(all) && PyTuple_GET_SIZE(all) == n;
    }
    PyObject *operator[](Py_ssize_t i) const {
        return PyList_CheckExact(all) ? PyList_GET_ITEM(all, i) : PyTuple_GET_ITEM(all, i);
    }
};
// An ordinary tensor (no subclass's that may answer calls itself), or null.
const Tensor *tensor_in(PyObject *x) {
    return THPVariable_CheckExact(x) ? &THPVariable_Unpack(x) : nullptr;
}
// A number, or one for each of n tensors.
struct Numbers {
    Items each;
    bool one, right = true;
    double value = 0.0;
    Numbers(py::handle x, Py_ssize_t n) : each(x, n), one(!each.right) {
        if (one) right = number(x.ptr(), &value);
    }
    static bool number(PyObject *x, double *to) {
        if (PyFloat_CheckExact(x)) *to = PyFloat_AS_DOUBLE(x);
        else if (PyLong_CheckExact(x)) {
            *to = PyLong_AsDouble(x);
            if (*to == -1.0 && PyErr_Occurred()) return PyErr_Clear(), false;
        } else return false;
        return true;
    }
    bool get(Py_ssize_t i, double *to) const {
        if (one) return *to = value, right;
        return number(each[i], to);
    }
};

// (whether it was done, the norm where it is asked for): adamw.py does the other calls.
py::tuple adamw_step(py::handle params, py::handle grads, py::handle exp_avgs, py::handle exp_avg_sqs,
                     py::handle masters, py::handle step, py::handle lr, py::handle weight_decay, py::handle betas,
                     py::handle eps_, py::handle max_norm_) {
    const auto other = [] { return py::make_tuple(false, py::none()); };
    const Py_ssize_t n = PyList_CheckExact(params.ptr()) ? PyList_GET_SIZE(params.ptr())
                         : PyTuple_CheckExact(params.ptr()) ? PyTuple_GET_SIZE(params.ptr()) : 0;
    if (n < 1) return other();
    const Items ps(params, n), gs(grads, n), ms(exp_avgs, n), vs(exp_avg_sqs, n), ws(masters, n), pair(betas, 2);
    const bool mastered = !masters.is_none();
    const Tensor *counter = tensor_in(step.ptr());
    const Numbers steps(step, n), rates(lr, n), decays(weight_decay, n);
    double b1, b2, eps, max_norm = 0.0;
    if (!gs.right || !ms.right || !vs.right || (mastered && !ws.right) || !pair.right ||
        !Numbers::number(pair[0], &b1) || !Numbers::number(pair[1], &b2) || !Numbers::number(eps_.ptr(), &eps) ||
        (!max_norm_.is_none() && (!Numbers::number(max_norm_.ptr(), &max_norm) || !(max_norm > 0))) ||
        !(b1 >= 0 && b1 < 1) || !(b2 >= 0 && b2 < 1) || !(eps >= 0))
        return other();
    const Tensor *first = tensor_in(ps[0]);
    if (!first || !first->is_cuda()) return other();
    const at::Device dev = first->device();
    const c10::DeviceGuard guard(dev);
    if (counter && !is_vector(*counter, at::kInt, dev, 1)) return other();
    bool counted = true;  // all of them on the device
    std::vector<gsv_adamw_tensor> all(n);
    std::vector<Tensor> held;  // while other threads may run, and change the lists
    held.reserve(6 * n + 1);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor *p = tensor_in(ps[i]), *g = tensor_in(gs[i]), *m = tensor_in(ms[i]), *v = tensor_in(vs[i]), *w = nullptr;
        if (mastered && ws[i] != Py_None && !(w = tensor_in(ws[i]))) return other();
        const Tensor *c = counter || steps.one ? nullptr : tensor_in(steps.each[i]);
        double t = 0.0, rate, decay;
        if (!p || !g || !m || !v || !is_dense(*p, dev) || !token_type(*p) || !is_like(*g, *p, dev) || !token_type(*g) ||
            !is_like(*m, *p, dev) || m->scalar_type() != at::kFloat || !is_like(*v, *p, dev) ||
            v->scalar_type() != at::kFloat ||
            (w && (!is_like(*w, *p, dev) || w->scalar_type() != at::kFloat || p->scalar_type() == at::kFloat)) ||
            (c && !is_vector(*c, at::kInt, dev, 1)) ||
            (!counter && !c && (!PyLong_CheckExact(steps.one ? step.ptr() : steps.each[i]) || !steps.get(i, &t) ||
                          !(t >= 1 && t < 9e15))) ||
            !rates.get(i, &rate) || !(rate >= 0) || !decays.get(i, &decay) || !(decay >= 0))
            return other();
        gsv_adamw_tensor &x = all[i];
        x = gsv_adamw_tensor{};
        x.param = ptr<void>(*p), x.grad = ptr<void>(*g), x.exp_avg = ptr<float>(*m), x.exp_avg_sq = ptr<float>(*v);
        x.master = w ? ptr<float>(*w) : nullptr, x.numel = p->numel(), x.step = (int64_t)t;
        x.lr = rate, x.weight_decay = decay, x.dtype = type_code(*p), x.grad_dtype = type_code(*g);
        x.counter = c ? ptr<int32_t>(*c) : nullptr;
        counted &= counter || c;
        held.push_back(*g);  // the others are written
        for (const Tensor *t : {p, m, v, w, c})
            if (t) held.push_back(*t);
    }
    if (!counted && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) return other();
    if (counter) held.push_back(*counter);
    gsv_adamw_args a{};
    a.tensors = all.data(), a.count = (int64_t)n;
    a.beta1 = b1, a.beta2 = b2, a.eps = eps, a.max_norm = max_norm;
    a.counter = counter ? ptr<int32_t>(*counter) : nullptr;
    Tensor norm;
    if (max_norm > 0) {
        norm = empty({}, *first, at::kFloat);
        a.norm = ptr<float>(norm);
    }
    size_t bytes = 0;
    check(lib.gsv_adamw_workspace_bytes(&a, &bytes), "adamw_workspace_bytes");
    const Tensor ws_bytes = bytes ? workspace(bytes, *first) : Tensor();
    int status;
    {
        void *const stream = stream_of(*first), *const at = ptr<void>(ws_bytes);
        const py::gil_scoped_release unlocked;
        status = lib.gsv_adamw(&a, at, bytes, stream);
    }
    if (status == GSV_ERR_INVALID_ARGUMENT) return other();  // tensors share memory; nothing was launched
    check(status, "adamw");
    for (Py_ssize_t i = 0, at = 0; i < n; ++i) {
        const Py_ssize_t last = at + 3 + (all[i].master != nullptr) + (all[i].counter != nullptr);
        while (at++ < last) written(held[at]);
    }
    if (counter) written(held.back());
    if (!norm.defined()) return py::make_tuple(true, py::none());
    return py::make_tuple(true, py::reinterpret_steal<py::object>(THPVariable_Wrap(norm)));
}

}  // namespace

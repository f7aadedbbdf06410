// CPython module behind optim.py: Python lists of tensors -> the argument arrays of the C ABI (include/mbrl.h).  A step
// looks at four tensors and a counter for every parameter; asking torch for their pointers, types and layouts from
// Python takes 0.3 us a tensor and more -- longer than the launches that follow, for any list of this framework's
// policies -- and some 25 ns here: a norm of 2 or of 10 tensors, called from Python, takes the host 4.1 to 4.9 us from machine
// to machine, where torch's fill_ of one value takes 3.7 to 4.2.  Host code only; the entry points come as addresses from the
// library that lib.py has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>
#include <vector>

#include "../../include/mbrl.h"

namespace {
decltype(&mbrl_optim_workspace_bytes) workspace_bytes;
decltype(&mbrl_grad_norm) grad_norm;
decltype(&mbrl_clip_grad_norm) clip_grad_norm;
decltype(&mbrl_adam_step) adam_step;
decltype(&mbrl_last_error) last_error;
PyObject *mbrl_error;        // lib.MbrlError

struct Raised {};            // a Python error is set
[[noreturn]] void raise(PyObject *type, const std::string &text) {
    PyErr_SetString(type, text.c_str());
    throw Raised{};
}

int type_code(at::ScalarType t) {
    switch (t) {
    case at::kDouble: return MBRL_DT_DOUBLE;
    case at::kFloat: return MBRL_DT_FLOAT;
    case at::kBFloat16: return MBRL_DT_BFLOAT;
    case at::kHalf: return MBRL_DT_HALF;
    default: return -1;
    }
}

struct List;
// The GPU that all tensors of a call are on, or the first one that is not.
struct Place {
    c10::Device device{c10::DeviceType::CPU};
    const List *wrong = nullptr;
    size_t index = 0;
    bool elsewhere = false;
    void met(const List &l, size_t i, const at::Tensor &x);
    void settle() const;
};

// The tensors of a list (or any iterable), as a tuple of its own: the caller's list may change while numbers are converted.
struct List {
    PyObject *seq = nullptr;
    const char *name;
    std::vector<const at::Tensor *> t;
    std::vector<void *> ptr;
    List(PyObject *o, const char *name_) : name(name_) {
        if (THPVariable_Check(o)) raise(PyExc_TypeError, std::string(name) + ": expected a list of tensors, got one tensor");
        seq = PySequence_Tuple(o);
        if (!seq) throw Raised{};
        const Py_ssize_t n = PyTuple_GET_SIZE(seq);
        t.reserve(n);
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject *item = PyTuple_GET_ITEM(seq, i);
            if (!THPVariable_Check(item)) {
                const std::string got = Py_TYPE(item)->tp_name;
                Py_CLEAR(seq);
                raise(PyExc_TypeError, std::string(name) + ": element " + std::to_string(i) + " is not a tensor but " + got);
            }
            t.push_back(&THPVariable_Unpack(item));
        }
        ptr.resize(n);
    }
    ~List() { Py_XDECREF(seq); }
    List(const List &) = delete;
    [[noreturn]] void bad(size_t i, PyObject *type, const std::string &why) const {
        raise(type, std::string(name) + ": element " + std::to_string(i) + " " + why);
    }
    // Refuses what no operator takes, and gets the address.  A tensor off the device is refused last, by settle(): what is wrong
    // with a list is said without a GPU too.
    void check(size_t i, Place &at) {
        const at::Tensor &x = *t[i];
        if (!x.defined() || x.layout() != at::kStrided) bad(i, PyExc_ValueError, "is not a dense (strided) tensor");
        if (x.is_neg()) bad(i, PyExc_ValueError, "is a lazily negated view (resolve_neg() it)");
        if (x._fw_grad(0).defined()) bad(i, PyExc_ValueError, "has a forward-mode tangent, which these operators do not carry on");
        if (!x.is_non_overlapping_and_dense())
            bad(i, PyExc_ValueError, "has gaps or repeated values between its strides (use .contiguous())");
        if (at.device != x.device() || !x.is_cuda()) at.met(*this, i, x);
        ptr[i] = x.numel() ? x.data_ptr() : nullptr;
    }
};

inline void Place::met(const List &l, size_t i, const at::Tensor &x) {
    if (wrong) return;
    if (x.is_cuda() && device.type() != c10::DeviceType::CUDA) {
        device = x.device();
        return;
    }
    wrong = &l;
    index = i;
    elsewhere = x.is_cuda();
}
inline void Place::settle() const {
    if (!wrong) return;
    if (elsewhere) wrong->bad(index, PyExc_ValueError, "is on another GPU than the first tensor (one process per GPU)");
    wrong->bad(index, mbrl_error, "is not on a GPU (these operators run only on the HIP device; there is no CPU path)");
}

void written(const at::Tensor &x) {        // in-place changes count, for autograd and for whoever watches _version
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

struct Sizes {
    std::vector<int64_t> numel;
    std::vector<int> dtype;
    explicit Sizes(size_t n) : numel(n), dtype(n) {}
};

void type_of(const List &l, size_t i, Sizes &s) {
    const int code = type_code(l.t[i]->scalar_type());
    if (code < 0) l.bad(i, PyExc_ValueError, "is not float64, float32, bfloat16 or float16");
    s.numel[i] = l.t[i]->numel();
    s.dtype[i] = code;
}

// Device, stream, workspace and the norm's place of one call.
struct Call {
    c10::OptionalDeviceGuard guard;
    at::Tensor norm, space;
    int64_t bytes;
    void *stream;
    Call(int op, c10::Device dev, const Sizes &s, bool with_norm) {
        if (dev.type() != c10::DeviceType::CUDA) {        // an empty list: the current GPU
            c10::impl::VirtualGuardImpl impl(c10::DeviceType::CUDA);
            if (impl.deviceCount() < 1) raise(mbrl_error, "no GPU visible: these operators run only on the HIP device (no CPU path)");
            dev = impl.getDevice();
        }
        guard.reset_device(dev);
        stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
        bytes = workspace_bytes(op, s.numel.size(), s.numel.data(), s.dtype.data());
        if (bytes < 0) raise(mbrl_error, last_error());
        if (bytes) space = at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
        if (with_norm) norm = at::empty({}, at::TensorOptions().dtype(at::kDouble).device(dev));
    }
    void *space_ptr() const { return space.defined() ? space.data_ptr() : nullptr; }
    double *norm_ptr() const { return norm.defined() ? static_cast<double *>(norm.data_ptr()) : nullptr; }
    PyObject *result() const {
        if (norm.defined()) return THPVariable_Wrap(norm);
        Py_RETURN_NONE;
    }
};

void done(int rc) {
    if (rc == -7) raise(PyExc_ValueError, last_error());
    if (rc) raise(mbrl_error, std::string(last_error()) + " (code " + std::to_string(rc) + ")");
}

double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

int norm_code(PyObject *o) {
    const double p = number(o);
    if (p == 2.0) return MBRL_NORM_TWO;
    if (p == 1.0) return MBRL_NORM_ONE;
    if (std::isinf(p) && p > 0) return MBRL_NORM_INF;
    raise(PyExc_ValueError, "norm_type has to be 1, 2 or inf");
}

double limit(PyObject *o) {
    const double v = number(o);
    if (!(v >= 0.0)) raise(PyExc_ValueError, "max_norm must not be negative or NaN");
    return v;
}

// One number for all, or one for each tensor.
std::vector<double> numbers(PyObject *o, size_t n, const char *name) {
    if (PyFloat_Check(o) || !PySequence_Check(o) || THPVariable_Check(o)) {
        const double v = number(o);
        if (!std::isfinite(v) || v < 0.0) raise(PyExc_ValueError, std::string(name) + " must be finite and not negative");
        return std::vector<double>(n, v);
    }
    PyObject *seq = PySequence_Tuple(o);        // of its own, as List's
    if (!seq) throw Raised{};
    std::vector<double> out;
    bool ok = size_t(PyTuple_GET_SIZE(seq)) == n, fits = true;
    out.reserve(n);
    for (size_t i = 0; ok && i < n; i++) {
        const double v = PyFloat_AsDouble(PyTuple_GET_ITEM(seq, i));
        if (v == -1.0 && PyErr_Occurred()) {
            Py_DECREF(seq);
            throw Raised{};
        }
        fits = fits && std::isfinite(v) && v >= 0.0;
        out.push_back(v);
    }
    Py_DECREF(seq);
    if (!ok) raise(PyExc_ValueError, std::string(name) + ": one number for all tensors or one for each");
    if (!fits) raise(PyExc_ValueError, std::string(name) + " must be finite and not negative");
    return out;
}

template <class F>
PyObject *guarded(F &&f) {
    try {
        if (!adam_step) raise(PyExc_RuntimeError, "optim_bind: not connected");
        return f();
    } catch (const Raised &) {
    } catch (const std::bad_alloc &) {
        PyErr_NoMemory();
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "optim_bind: unknown error");
    }
    return nullptr;
}

bool arity(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) PyErr_SetString(PyExc_TypeError, "optim_bind: wrong number of arguments");
    return n == want;
}

// connect(MbrlError, addresses of mbrl_optim_workspace_bytes, mbrl_grad_norm, mbrl_clip_grad_norm, mbrl_adam_step, mbrl_last_error)
PyObject *py_connect(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 6)) return nullptr;
    void *at[5];
    for (int i = 0; i < 5; i++) {
        at[i] = PyLong_AsVoidPtr(a[1 + i]);
        if (!at[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "optim_bind: null entry point");
            return nullptr;
        }
    }
    Py_INCREF(a[0]);
    Py_XSETREF(mbrl_error, a[0]);
    workspace_bytes = reinterpret_cast<decltype(workspace_bytes)>(at[0]);
    grad_norm = reinterpret_cast<decltype(grad_norm)>(at[1]);
    clip_grad_norm = reinterpret_cast<decltype(clip_grad_norm)>(at[2]);
    last_error = reinterpret_cast<decltype(last_error)>(at[4]);
    adam_step = reinterpret_cast<decltype(adam_step)>(at[3]);
    Py_RETURN_NONE;
}

// grad_norm(grads, norm_type)
PyObject *py_grad_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 2)) return nullptr;
    return guarded([&] {
        List g(a[0], "grads");
        const int kind = norm_code(a[1]);
        Sizes s(g.t.size());
        Place at;
        const bool recording = c10::GradMode::is_enabled();
        for (size_t i = 0; i < g.t.size(); i++) {
            if (recording && g.t[i]->requires_grad())
                g.bad(i, PyExc_ValueError, "requires grad, which the norm does not pass on (call it under torch.no_grad(), or detach())");
            g.check(i, at);
            type_of(g, i, s);
        }
        at.settle();
        Call c(MBRL_OP_NORM, at.device, s, true);
        done(grad_norm(g.t.size(), g.ptr.data(), s.numel.data(), s.dtype.data(), kind, c.space_ptr(), c.bytes, c.norm_ptr(), c.stream));
        return c.result();
    });
}

// clip_grad_norm_(grads, max_norm, norm_type)
PyObject *py_clip_grad_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 3)) return nullptr;
    return guarded([&] {
        List g(a[0], "grads");
        const double most = limit(a[1]);
        const int kind = norm_code(a[2]);
        Sizes s(g.t.size());
        Place at;
        for (size_t i = 0; i < g.t.size(); i++) {
            g.check(i, at);
            type_of(g, i, s);
        }
        at.settle();
        Call c(MBRL_OP_CLIP, at.device, s, true);
        done(clip_grad_norm(g.t.size(), g.ptr.data(), s.numel.data(), s.dtype.data(), kind, most, c.space_ptr(), c.bytes,
                            c.norm_ptr(), c.stream));
        for (const at::Tensor *x : g.t) written(*x);
        return c.result();
    });
}

// adam_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr, beta1, beta2, eps, weight_decay, decoupled, max_norm or None, norm_type)
PyObject *py_adam_step(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (!arity(n, 13)) return nullptr;
    return guarded([&] {
        List p(a[0], "params"), g(a[1], "grads"), m(a[2], "exp_avgs"), v(a[3], "exp_avg_sqs"), t(a[4], "steps");
        const size_t count = p.t.size();
        for (const List *l : {&g, &m, &v, &t})
            if (l->t.size() != count) raise(PyExc_ValueError, std::string(l->name) + ": not as many tensors as params");
        const std::vector<double> lr = numbers(a[5], count, "lr"), wd = numbers(a[9], count, "weight_decay");
        const double b1 = number(a[6]), b2 = number(a[7]), eps = number(a[8]);
        const int decoupled = PyObject_IsTrue(a[10]);
        if (decoupled < 0) throw Raised{};
        const bool clip = a[11] != Py_None;
        const double most = clip ? limit(a[11]) : 0.0;
        const int kind = norm_code(a[12]);
        Sizes s(count);
        Place at;
        for (size_t i = 0; i < count; i++) {
            p.check(i, at);
            type_of(p, i, s);
            const at::Tensor &x = *p.t[i];
            const at::ScalarType wide = x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
            for (List *l : {&g, &m, &v}) {
                const at::Tensor &y = *l->t[i];
                if (y.scalar_type() != (l == &g ? x.scalar_type() : wide))
                    l->bad(i, PyExc_ValueError, l == &g ? "has another type than its parameter" : "is not float32 (float64 for a float64 parameter)");
                if (y.sizes() != x.sizes()) l->bad(i, PyExc_ValueError, "has another shape than its parameter");
                l->check(i, at);
                // the order of values in memory is what counts: strides of dimensions with one value say nothing of it
                if (!(x.is_contiguous() && y.is_contiguous()) && y.strides() != x.strides())
                    for (int64_t d = 0; d < x.dim(); d++)
                        if (x.size(d) > 1 && x.numel() && x.stride(d) != y.stride(d))
                            l->bad(i, PyExc_ValueError, "has its values in another order than its parameter (strides differ)");
            }
            if (t.t[i]->scalar_type() != at::kFloat || t.t[i]->numel() != 1) t.bad(i, PyExc_ValueError, "is not one float32 value");
            t.check(i, at);
        }
        at.settle();
        Call c(MBRL_OP_ADAM, at.device, s, clip);
        std::vector<float *> steps(count);
        for (size_t i = 0; i < count; i++) steps[i] = static_cast<float *>(t.ptr[i]);
        done(adam_step(count, p.ptr.data(), g.ptr.data(), m.ptr.data(), v.ptr.data(), steps.data(), s.numel.data(), s.dtype.data(), lr.data(),
                       wd.data(), b1, b2, eps, decoupled, kind, most, c.space_ptr(), c.bytes, c.norm_ptr(), c.stream));
        for (const List *l : {&p, &m, &v, &t})
            for (const at::Tensor *x : l->t) written(*x);
        return c.result();
    });
}

PyMethodDef methods[] = {
    {"connect", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_connect)), METH_FASTCALL, nullptr},
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_grad_norm)), METH_FASTCALL, nullptr},
    {"clip_grad_norm_", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_clip_grad_norm)), METH_FASTCALL, nullptr},
    {"adam_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_adam_step)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "optim_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit_optim_bind(void) { return PyModule_Create(&module); }

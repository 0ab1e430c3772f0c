/*
 * What the native calls of layers.py and losses.py share: Python arguments checked and turned into tensors, rows and numbers,
 * results wrapped, C++ exceptions turned into Python's.  Everything is local to the module that includes it.
 */
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/eri_layers.h"
#include "eri_torch_common.h"

namespace {

using eri_face::Outputs;

struct Raised : std::exception {}; // a Python error has been set

[[noreturn]] void raise(PyObject *type, const std::string &what) {
    PyErr_SetString(type, what.c_str());
    throw Raised();
}
#define ERI_VALUE(cond, what) \
    do {                      \
        if (!(cond)) raise(PyExc_ValueError, what); \
    } while (0)

/* EriError of the last failing call. */
[[noreturn]] void raise_code(int code, const char *call) {
    PyObject *module = PyImport_ImportModule("eridiffusion_amd._lib");
    PyObject *type = module ? PyObject_GetAttrString(module, "EriError") : nullptr;
    PyObject *e = type ? PyObject_CallFunction(type, "sis", call, code, eri_last_error()) : nullptr;
    if (e) PyErr_SetObject(type, e);
    Py_XDECREF(e);
    Py_XDECREF(type);
    Py_XDECREF(module);
    throw Raised();
}
void check(int code, const char *call) {
    if (code) raise_code(code, call);
}

/* Tracers record torch's operations to run them again, or run them on tensors without values.  These kernels are none: what was
 * recorded would be outputs that nobody writes.  A dispatch mode of a user's own (one that counts or logs) stays: the call runs under it. */
void not_traced() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    const bool jit = at::tracer::impl::is_dispatch_enabled();
    const bool mode = Modes::any_modes_set() && (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL));
    ERI_VALUE(!jit && !mode, "these calls cannot be traced: a recorded program would not run their kernels");
}

int tag_of(at::ScalarType t) {
    return t == at::kFloat ? ERI_DTYPE_F32 : t == at::kBFloat16 ? ERI_DTYPE_BF16 : t == at::kFloat8_e4m3fn ? ERI_DTYPE_F8E4M3 : -1;
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, std::string(name) + " is no tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    ERI_VALUE(t.defined() && t.layout() == at::kStrided && t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch(),
              std::string(name) + " is no plain tensor");
    ERI_VALUE(!t._fw_grad(0).defined(), std::string(name) + " carries a forward-mode tangent, which these kernels do not take along");
    ERI_VALUE(t.is_cuda(), std::string(name) + " is on " + t.device().str() + ": these kernels take device tensors");
    ERI_VALUE(!t.is_conj() && !t.is_neg(), std::string(name) + " is a lazy view");
    return t;
}
const at::Tensor &floats(PyObject *o, const char *name, const at::Tensor *beside = nullptr) {
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16)
        raise(PyExc_TypeError, std::string("Unsupported: ") + name + " is " + c10::toString(t.scalar_type()) + ", and these kernels take float32 or bfloat16");
    if (beside) ERI_VALUE(t.device() == beside->device(), std::string(name) + " is on another device");
    return t;
}

bool records(const at::Tensor &t) { return t.requires_grad() && at::GradMode::is_enabled(); }

/* A tensor as rows of its last dimension.  One whose rows do not lie at one distance is copied, unless it is written to. */
struct Rows {
    at::Tensor t;
    int64_t rows = 0, cols = 0;
    uint64_t stride = 0;
    bool set() {
        cols = t.dim() ? t.size(-1) : 1;
        rows = 1;
        for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
        stride = (uint64_t)cols;
        if (t.is_contiguous()) return true;
        if (t.numel() == 0) return true;
        int64_t d = t.dim() - 1;
        if (t.size(d) != 1 && t.stride(d) != 1) return false;
        int64_t step = 0; // distance of two rows, of the innermost dimension that has two
        int64_t run = 1;  // rows inside of the dimension at hand
        for (--d; d >= 0; --d) {
            if (t.size(d) == 1) continue;
            if (step == 0) {
                step = t.stride(d);
                if (step < cols) return false;
            } else if (t.stride(d) != step * run) return false;
            run *= t.size(d);
        }
        if (step) stride = (uint64_t)step;
        return true;
    }
    explicit Rows(const at::Tensor &of, const char *written = nullptr) : t(of) {
        if (set()) return;
        ERI_VALUE(!written, std::string(written) + "'s rows do not lie at one distance");
        t = t.contiguous();
        set();
    }
};

/* Bytes that rows take: `count` of them, `width` long and `step` apart. */
struct Span {
    uint64_t at, count, width, step;
    explicit Span(const Rows &r)
        : at(reinterpret_cast<uint64_t>(r.t.const_data_ptr())), count((uint64_t)r.rows), width((uint64_t)r.cols * r.t.element_size()), step(r.stride * r.t.element_size()) {
        if (step == width || count == 1) width *= count, step = width, count = 1; // without gaps: one long row
    }
    uint64_t end() const { return at + (count - 1) * step + width; }
    bool operator==(const Span &o) const { return at == o.at && count == o.count && width == o.width && step == o.step; }
    /* Rows at the same distance may lie beside each other, columns of one matrix; at different distances they are taken to meet. */
    bool meets(const Span &o) const {
        if (!count || !width || !o.count || !o.width || end() <= o.at || o.end() <= at) return false;
        if (count > 1 && o.count > 1 && step != o.step) return true;
        if (count == 1 && o.count == 1) return true;
        const uint64_t s = count > 1 ? step : o.step;
        const uint64_t from = o.at >= at ? (o.at - at) % s : (s - (at - o.at) % s) % s; // where the other's row begins, seen from the beginning of this one's
        return from < width || from + o.width > s;
    }
};
/* Refuses a given output whose memory meets an input's: some workgroups write it while others still read. */
void apart(const Rows &out, const Rows &in, const char *name) { ERI_VALUE(!Span(out).meets(Span(in)), std::string("out overlaps ") + name); }

double number(PyObject *o, const char *name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        raise(PyExc_TypeError, std::string(name) + " is no number");
    }
    return v;
}
uint64_t word(PyObject *o, const char *name) {
    PyObject *i = PyNumber_Index(o);
    if (!i) {
        PyErr_Clear();
        raise(PyExc_TypeError, std::string(name) + " is no whole number");
    }
    const uint64_t v = PyLong_AsUnsignedLongLong(i);
    Py_DECREF(i);
    if (v == (uint64_t)-1 && PyErr_Occurred()) {
        PyErr_Clear();
        raise(PyExc_ValueError, std::string(name) + " is not between 0 and 2**64 - 1");
    }
    return v;
}

/* The current stream of a tensor's device, as torch has it. */
void *stream_of(const at::Tensor &t) {
    static PyObject *get = nullptr;
    if (!get) {
        PyObject *c = PyImport_ImportModule("torch._C");
        get = c ? PyObject_GetAttrString(c, "_cuda_getCurrentRawStream") : nullptr;
        Py_XDECREF(c);
        if (!get) throw Raised();
    }
    PyObject *device = PyLong_FromLong(t.get_device());
    PyObject *got = device ? PyObject_CallOneArg(get, device) : nullptr;
    Py_XDECREF(device);
    if (!got) throw Raised();
    void *s = PyLong_AsVoidPtr(got);
    Py_DECREF(got);
    if (!s && PyErr_Occurred()) throw Raised();
    return s;
}

/* A given output, which is written in place: autograd has to know that its values change. */
const at::Tensor &written(PyObject *o, const char *name, const at::Tensor &beside) {
    const at::Tensor &t = floats(o, name, &beside);
    ERI_VALUE(!records(t), std::string(name) + " requires a gradient itself");
    return t;
}
void changed(const at::Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
    std::vector<int64_t> s(sizes.begin(), sizes.end());
    s.push_back(last);
    return s;
}

/* A tuple of tensors, None for those that are not defined. */
PyObject *wrapped(const std::vector<at::Tensor> &all) {
    PyObject *out = PyTuple_New((Py_ssize_t)all.size());
    if (!out) throw Raised();
    for (size_t i = 0; i < all.size(); ++i) {
        PyObject *o = all[i].defined() ? THPVariable_Wrap(all[i]) : Py_NewRef(Py_None);
        if (!o) {
            Py_DECREF(out);
            throw Raised();
        }
        PyTuple_SET_ITEM(out, (Py_ssize_t)i, o);
    }
    return out;
}
PyObject *wrapped(const at::Tensor &t) {
    PyObject *o = THPVariable_Wrap(t);
    if (!o) throw Raised();
    return o;
}

template <PyObject *(*F)(PyObject *const *), Py_ssize_t N> PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, and %zd are wanted", n, N);
        return nullptr;
    }
    try {
        not_traced();
        return F(args);
    } catch (const Raised &) {
        return nullptr;
    } catch (const std::exception &) { // out of memory reaches Python as torch.OutOfMemoryError, which trainers catch
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}
template <PyObject *(*F)(PyObject *const *), Py_ssize_t N> PyMethodDef method(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&entry<F, N>)), METH_FASTCALL, nullptr};
}

} // namespace

/*
 * The calls of eridiffusion_amd/layers.py in native code: arguments checked, outputs allocated, the C function of
 * include/eri_layers.h called on the current stream.  A norm of one token takes 3 us on the device; the same work in the
 * interpreter (ctypes, a dozen attribute reads of tensors) took several times that.
 *
 * Each function returns None where autograd has to record the call: layers.py then goes through its autograd functions,
 * whose forward comes here again with recording off.
 */
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
    ERI_VALUE(!jit && !mode, "these layers cannot be traced: a recorded program would not run their kernels");
}

int tag_of(at::ScalarType t) {
    return t == at::kFloat ? ERI_DTYPE_F32 : t == at::kBFloat16 ? ERI_DTYPE_BF16 : t == at::kFloat8_e4m3fn ? ERI_DTYPE_F8E4M3 : -1;
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, std::string(name) + " is no tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    ERI_VALUE(t.defined() && t.layout() == at::kStrided && t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch(),
              std::string(name) + " is no plain tensor");
    ERI_VALUE(!t._fw_grad(0).defined(), std::string(name) + " carries a forward-mode tangent, which these layers do not take along");
    ERI_VALUE(t.is_cuda(), std::string(name) + " is on " + t.device().str() + ": these layers take device tensors");
    ERI_VALUE(!t.is_conj() && !t.is_neg(), std::string(name) + " is a lazy view");
    return t;
}
const at::Tensor &floats(PyObject *o, const char *name, const at::Tensor *beside = nullptr) {
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16)
        raise(PyExc_TypeError, std::string("Unsupported: ") + name + " is " + c10::toString(t.scalar_type()) + ", and these layers take float32 or bfloat16");
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

/* p, seed and offset; the offset may be a device tensor of one int64, read when the kernel runs. */
EriDropoutKey key_of(PyObject *p, PyObject *seed, PyObject *offset, const at::Tensor &beside) {
    EriDropoutKey k = {word(seed, "seed"), 0, nullptr, number(p, "p")};
    ERI_VALUE(k.p >= 0.0 && k.p <= 1.0, "p is not between 0 and 1");
    if (THPVariable_Check(offset)) {
        const at::Tensor &t = tensor(offset, "offset");
        ERI_VALUE(t.scalar_type() == at::kLong && t.numel() == 1 && t.device() == beside.device(), "offset is no int64 of one element beside the inputs");
        k.offset_ptr = static_cast<const uint64_t *>(t.const_data_ptr());
    } else k.offset = word(offset, "offset");
    return k;
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

/* Ids are read as they lie, 32 or 64 bits each. */
at::Tensor ids_of(PyObject *o) {
    const at::Tensor &t = tensor(o, "ids");
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) raise(PyExc_TypeError, "ids are neither int32 nor int64");
    return t.is_contiguous() ? t : t.contiguous();
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

/* embedding(ids, weight, scale, out) -> rows */
PyObject *embedding(PyObject *const *args) {
    const at::Tensor &weight = floats(args[1], "weight");
    const at::Tensor ids = ids_of(args[0]);
    ERI_VALUE(ids.device() == weight.device(), "ids are on another device");
    ERI_VALUE(weight.dim() == 2, "weight is no matrix");
    if (records(weight)) {
        ERI_VALUE(args[3] == Py_None, "out is for calls that autograd does not record");
        return Py_NewRef(Py_None);
    }
    const Rows table(weight);
    EriEmbedding a = {};
    a.scale = (float)number(args[2], "scale");
    Outputs made;
    made.guard.reset_device(weight.device());
    const auto shape = with_last(ids.sizes(), weight.size(1));
    const Rows out(args[3] == Py_None ? made.empty(shape, weight.scalar_type(), weight) : written(args[3], "out", weight), "out");
    ERI_VALUE(out.t.sizes() == at::IntArrayRef(shape) && out.t.scalar_type() == weight.scalar_type(), "out has another shape or dtype than the rows");
    if (args[3] != Py_None) apart(out, table, "weight"), apart(out, Rows(ids), "ids");
    a.ids = ids.const_data_ptr();
    a.table = table.t.const_data_ptr();
    a.out = out.t.data_ptr();
    a.tokens = (uint64_t)ids.numel();
    a.vocab = (uint64_t)weight.size(0);
    a.dim = (uint64_t)weight.size(1);
    a.table_stride = table.stride;
    a.out_stride = out.stride;
    a.ids_64 = ids.scalar_type() == at::kLong;
    a.dtype_tag = tag_of(weight.scalar_type());
    changed(out.t);
    check(eri_embedding(&a, stream_of(weight)), "eri_embedding");
    return args[3] == Py_None ? wrapped(out.t) : Py_NewRef(args[3]);
}

/* embedding_grad(ids, grad, vocab, scale, padding_id, dtype, out, accumulate) -> table's gradient */
PyObject *embedding_grad(PyObject *const *args) {
    const at::Tensor &grad = floats(args[1], "grad");
    const at::Tensor ids = ids_of(args[0]);
    ERI_VALUE(ids.device() == grad.device(), "ids are on another device");
    ERI_VALUE(grad.dim() == ids.dim() + 1 && grad.sizes().slice(0, (size_t)ids.dim()) == ids.sizes(), "grad's shape is not that of ids and a row's length");
    EriEmbeddingGrad a = {};
    const uint64_t vocab = word(args[2], "vocab");
    ERI_VALUE(vocab <= 0x7fffffffull, "vocab is over 2**31 - 1");
    a.scale = (float)number(args[3], "scale");
    a.padding_id = -1;
    if (args[4] != Py_None) {
        const uint64_t pad = word(args[4], "padding_id");
        ERI_VALUE(pad < vocab, "padding_id is no row of the table");
        a.padding_id = (int64_t)pad;
    }
    at::ScalarType dtype = grad.scalar_type();
    if (args[5] != Py_None) {
        if (!THPDtype_Check(args[5])) raise(PyExc_TypeError, "dtype is no dtype");
        dtype = reinterpret_cast<THPDtype *>(args[5])->scalar_type;
        if (dtype != at::kFloat && dtype != at::kBFloat16) raise(PyExc_TypeError, "Unsupported: a gradient is float32 or bfloat16");
    }
    const int accumulate = PyObject_IsTrue(args[7]);
    if (accumulate < 0) throw Raised();
    ERI_VALUE(!accumulate || args[6] != Py_None, "accumulate adds to out, which is not given");
    Outputs made;
    made.guard.reset_device(grad.device());
    const std::vector<int64_t> shape = {(int64_t)vocab, grad.size(-1)};
    const Rows out(args[6] == Py_None ? made.empty(shape, dtype, grad) : written(args[6], "out", grad), "out");
    ERI_VALUE(out.t.sizes() == at::IntArrayRef(shape) && (args[5] == Py_None || out.t.scalar_type() == dtype), "out has another shape or dtype than the gradient");
    const Rows rows(grad);
    if (args[6] != Py_None) apart(out, rows, "grad"), apart(out, Rows(ids), "ids");
    check(eri_embedding_grad_workspace((uint64_t)ids.numel(), vocab, (uint64_t)grad.size(-1), &a.workspace_bytes), "eri_embedding_grad_workspace");
    const at::Tensor workspace = made.empty({(int64_t)a.workspace_bytes}, at::kByte, grad);
    a.ids = ids.const_data_ptr();
    a.grad = rows.t.const_data_ptr();
    a.out = out.t.data_ptr();
    a.workspace = workspace.data_ptr();
    a.tokens = (uint64_t)ids.numel();
    a.vocab = vocab;
    a.dim = (uint64_t)grad.size(-1);
    a.grad_stride = rows.stride;
    a.out_stride = out.stride;
    a.ids_64 = ids.scalar_type() == at::kLong;
    a.grad_dtype = tag_of(grad.scalar_type());
    a.out_dtype = tag_of(out.t.scalar_type());
    a.accumulate = accumulate;
    changed(out.t);
    check(eri_embedding_grad(&a, stream_of(grad)), "eri_embedding_grad");
    return args[6] == Py_None ? wrapped(out.t) : Py_NewRef(args[6]);
}

/* dropout(x, p, seed, offset, out) -> y */
PyObject *dropout(PyObject *const *args) {
    const at::Tensor &given = floats(args[0], "x");
    EriDropout a = {};
    a.key = key_of(args[1], args[2], args[3], given);
    if (records(given)) {
        ERI_VALUE(args[4] == Py_None, "out is for calls that autograd does not record");
        return Py_NewRef(Py_None);
    }
    const Rows x(given);
    Outputs made;
    made.guard.reset_device(given.device());
    const Rows out(args[4] == Py_None ? made.empty(given.sizes(), given.scalar_type(), given) : written(args[4], "out", given), "out");
    ERI_VALUE(out.t.sizes() == given.sizes() && out.t.scalar_type() == given.scalar_type(), "out has another shape or dtype than x");
    if (args[4] != Py_None) {
        if (!(Span(out) == Span(x))) apart(out, x, "x"); // over x itself: each element by the thread that has read it
        if (a.key.offset_ptr) apart(out, Rows(THPVariable_Unpack(args[3])), "offset");
    }
    a.x = x.t.const_data_ptr();
    a.y = out.t.data_ptr();
    a.rows = (uint64_t)x.rows;
    a.cols = (uint64_t)x.cols;
    a.x_stride = x.stride;
    a.y_stride = out.stride;
    a.dtype_tag = tag_of(given.scalar_type());
    changed(out.t);
    check(eri_dropout(&a, stream_of(given)), "eri_dropout");
    return args[4] == Py_None ? wrapped(out.t) : Py_NewRef(args[4]);
}

/* A vector with an element for each column. */
at::Tensor weight_of(PyObject *o, int64_t cols, const at::Tensor &beside) {
    const at::Tensor &w = floats(o, "weight", &beside);
    ERI_VALUE(w.dim() == 1 && w.size(0) == cols, "weight has not an element for each column");
    return w.is_contiguous() ? w : w.contiguous();
}

/* rms_norm(x, weight, eps, residual, p, seed, offset, dtype, scale_group) -> (y, h, rstd, scales) */
PyObject *rms_norm(PyObject *const *args) {
    const at::Tensor &given = floats(args[0], "x");
    ERI_VALUE(given.dim() >= 1, "x has no dimension to norm");
    const int64_t cols = given.size(-1);
    EriRmsNorm a = {};
    a.key = key_of(args[4], args[5], args[6], given);
    a.eps = (float)number(args[2], "eps");
    at::ScalarType dtype = given.scalar_type();
    if (args[7] != Py_None) {
        if (!THPDtype_Check(args[7])) raise(PyExc_TypeError, "dtype is no dtype");
        dtype = reinterpret_cast<THPDtype *>(args[7])->scalar_type;
        if (tag_of(dtype) < 0) raise(PyExc_TypeError, "Unsupported: the norm's output is float32, bfloat16 or float8_e4m3fn");
    }
    const uint64_t group = word(args[8], "scale_group");
    ERI_VALUE(group == 0 || (group == 128 && dtype == at::kFloat8_e4m3fn), "scale_group is 0, or 128 with float8_e4m3fn");
    const at::Tensor weight = args[1] == Py_None ? at::Tensor() : weight_of(args[1], cols, given);
    const bool add = args[3] != Py_None;
    const at::Tensor none;
    const at::Tensor &res = add ? floats(args[3], "residual", &given) : none;
    if (add) ERI_VALUE(res.sizes() == given.sizes(), "residual has another shape than x");
    if (records(given) || (weight.defined() && records(weight)) || (add && records(res))) {
        ERI_VALUE(dtype != at::kFloat8_e4m3fn, "autograd takes no gradient through 8 bits: call without gradients, and rms_norm_grad for them");
        return Py_NewRef(Py_None);
    }
    const Rows x(given), residual(add ? res : given);
    Outputs made;
    made.guard.reset_device(given.device());
    const bool f8 = dtype == at::kFloat8_e4m3fn, keeps = add || a.key.p > 0.0;
    const at::Tensor y = made.empty(given.sizes(), dtype, given);
    const at::Tensor h = keeps ? made.empty(given.sizes(), add ? res.scalar_type() : given.scalar_type(), given) : given;
    const at::Tensor rstd = made.empty(given.sizes().slice(0, (size_t)given.dim() - 1), at::kFloat, given);
    at::Tensor scales;
    if (f8) scales = made.empty(with_last(given.sizes().slice(0, (size_t)given.dim() - 1), group ? (cols + 127) / 128 : 1), at::kFloat, given);
    a.x = x.t.const_data_ptr();
    a.residual = add ? residual.t.const_data_ptr() : nullptr;
    a.weight = weight.defined() ? weight.const_data_ptr() : nullptr;
    a.y = y.data_ptr();
    a.h = keeps ? h.data_ptr() : nullptr;
    a.rstd = static_cast<float *>(rstd.data_ptr());
    a.scales = f8 ? static_cast<float *>(scales.data_ptr()) : nullptr;
    a.rows = (uint64_t)x.rows;
    a.cols = (uint64_t)cols;
    a.x_stride = x.stride;
    a.residual_stride = residual.stride;
    a.x_dtype = tag_of(given.scalar_type());
    a.residual_dtype = add ? tag_of(res.scalar_type()) : 0;
    a.weight_dtype = weight.defined() ? tag_of(weight.scalar_type()) : 0;
    a.y_dtype = tag_of(dtype);
    a.scale_group = (int32_t)group;
    check(eri_rms_norm(&a, stream_of(given)), "eri_rms_norm");
    return wrapped({y, h, rstd, scales});
}

/* rms_norm_grad(grad, h, rstd, weight, grad_h, p, seed, offset, dtype, needs) -> gradients of (x, residual, weight) */
PyObject *rms_norm_grad(PyObject *const *args) {
    const at::Tensor &grad = floats(args[0], "grad"), &h = floats(args[1], "h", &grad), &rstd = floats(args[2], "rstd", &grad);
    ERI_VALUE(grad.dim() >= 1 && h.sizes() == grad.sizes(), "h has another shape than grad");
    const int64_t cols = grad.size(-1);
    ERI_VALUE(rstd.scalar_type() == at::kFloat && rstd.sizes() == grad.sizes().slice(0, (size_t)grad.dim() - 1), "rstd is no float32 for each row");
    const at::Tensor weight = args[3] == Py_None ? at::Tensor() : weight_of(args[3], cols, grad);
    const bool more = args[4] != Py_None;
    const at::Tensor none;
    const at::Tensor &grad_h = more ? floats(args[4], "grad_h", &grad) : none;
    if (more) ERI_VALUE(grad_h.sizes() == grad.sizes() && grad_h.scalar_type() == h.scalar_type(), "grad_h has another shape or dtype than h");
    EriRmsNormGrad a = {};
    a.key = key_of(args[5], args[6], args[7], grad);
    at::ScalarType dtype = grad.scalar_type();
    if (args[8] != Py_None) {
        if (!THPDtype_Check(args[8])) raise(PyExc_TypeError, "dtype is no dtype");
        dtype = reinterpret_cast<THPDtype *>(args[8])->scalar_type;
        if (dtype != at::kFloat && dtype != at::kBFloat16) raise(PyExc_TypeError, "Unsupported: a gradient is float32 or bfloat16");
    }
    if (!PyTuple_Check(args[9]) || PyTuple_GET_SIZE(args[9]) != 3) raise(PyExc_TypeError, "needs is no tuple of three");
    bool needs[3];
    for (int i = 0; i < 3; ++i) {
        const int yes = PyObject_IsTrue(PyTuple_GET_ITEM(args[9], i));
        if (yes < 0) throw Raised();
        needs[i] = yes;
    }
    needs[2] = needs[2] && weight.defined();
    const bool same = a.key.p == 0.0 && dtype == h.scalar_type(); // x's gradient is the residual's
    const Rows g(grad), hr(h), r(more ? grad_h : grad);
    const at::Tensor q = rstd.is_contiguous() ? rstd : rstd.contiguous();
    Outputs made;
    made.guard.reset_device(grad.device());
    at::Tensor dx, dr, dw, workspace;
    if (needs[1] || (needs[0] && same)) dr = made.empty(grad.sizes(), h.scalar_type(), grad);
    if (needs[0]) dx = same ? dr : made.empty(grad.sizes(), dtype, grad);
    if (needs[2]) {
        dw = made.empty({cols}, weight.scalar_type(), grad);
        check(eri_rms_norm_grad_workspace((uint64_t)g.rows, (uint64_t)cols, &a.workspace_bytes), "eri_rms_norm_grad_workspace");
        workspace = made.empty({(int64_t)a.workspace_bytes}, at::kByte, grad);
        a.workspace = workspace.data_ptr();
        a.grad_weight = dw.data_ptr();
        a.grad_weight_dtype = tag_of(dw.scalar_type());
    }
    a.grad = g.t.const_data_ptr();
    a.h = hr.t.const_data_ptr();
    a.rstd = static_cast<const float *>(q.const_data_ptr());
    a.weight = weight.defined() ? weight.const_data_ptr() : nullptr;
    a.grad_h = more ? r.t.const_data_ptr() : nullptr;
    a.grad_x = needs[0] && !same ? dx.data_ptr() : nullptr;
    a.grad_residual = dr.defined() ? dr.data_ptr() : nullptr;
    a.rows = (uint64_t)g.rows;
    a.cols = (uint64_t)cols;
    a.grad_stride = g.stride;
    a.h_stride = hr.stride;
    a.grad_h_stride = r.stride;
    a.grad_dtype = tag_of(grad.scalar_type());
    a.h_dtype = tag_of(h.scalar_type());
    a.x_dtype = tag_of(dtype);
    a.weight_dtype = weight.defined() ? tag_of(weight.scalar_type()) : 0;
    check(eri_rms_norm_grad(&a, stream_of(grad)), "eri_rms_norm_grad");
    return wrapped({dx, needs[1] ? dr : at::Tensor(), dw});
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

PyMethodDef methods[] = {method<embedding, 4>("embedding"), method<embedding_grad, 8>("embedding_grad"), method<dropout, 5>("dropout"),
                         method<rms_norm, 9>("rms_norm"), method<rms_norm_grad, 10>("rms_norm_grad"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layers_face", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__layers_face(void) { return PyModule_Create(&module); }

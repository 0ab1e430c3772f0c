/*
 * The calls of eridiffusion_amd/losses.py in native code: arguments checked, outputs allocated, the C function of
 * include/eri_losses.h called on the current stream.
 *
 * The two losses return None where autograd has to record the call: losses.py then goes through its autograd functions, whose
 * forward comes here again with recording off.
 */
#include "../../include/eri_losses.h"
#include "eri_face_args.h"

namespace {

/* Rows of logits, and the sizes of what has one value for each. */
at::IntArrayRef rows_of(const at::Tensor &logits) {
    ERI_VALUE(logits.dim() >= 1, "logits have no dimension to normalise");
    return logits.sizes().slice(0, (size_t)logits.dim() - 1);
}
/* Float32 for each row. */
at::Tensor per_row(PyObject *o, const char *name, const at::Tensor &logits) {
    const at::Tensor &t = floats(o, name, &logits);
    ERI_VALUE(t.scalar_type() == at::kFloat && t.sizes() == rows_of(logits), std::string(name) + " is no float32 for each row");
    return t.is_contiguous() ? t : t.contiguous();
}
at::Tensor stats_of(PyObject *o, int64_t each, const at::Tensor &logits) {
    const at::Tensor &t = floats(o, "stats", &logits);
    ERI_VALUE(t.scalar_type() == at::kFloat && t.sizes() == at::IntArrayRef(with_last(rows_of(logits), each)), "stats are not what the forward call returned for such logits");
    return t.is_contiguous() ? t : t.contiguous();
}
const at::Tensor &whole_numbers(PyObject *o, const at::Tensor &beside) {
    const at::Tensor &t = tensor(o, "ids");
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) raise(PyExc_TypeError, "ids are neither int32 nor int64");
    ERI_VALUE(t.device() == beside.device(), "ids are on another device");
    return t;
}
at::Tensor token_ids(PyObject *o, const at::Tensor &logits) {
    const at::Tensor &t = whole_numbers(o, logits);
    ERI_VALUE(t.sizes() == rows_of(logits), "ids are not one for each row");
    return t.is_contiguous() ? t : t.contiguous();
}
bool truth(PyObject *o) {
    const int yes = PyObject_IsTrue(o);
    if (yes < 0) throw Raised();
    return yes;
}

/* A teacher's tokens and their values, as rows. */
struct Teacher {
    Rows ids, values;
    Teacher(PyObject *i, PyObject *v, const at::Tensor &logits) : ids(whole_numbers(i, logits)), values(floats(v, "teacher", &logits)) {
        const at::Tensor &given = THPVariable_Unpack(i), &t = THPVariable_Unpack(v);
        ERI_VALUE(given.dim() == logits.dim() && given.sizes().slice(0, (size_t)given.dim() - 1) == rows_of(logits) && given.size(-1) >= 1 && given.size(-1) <= ERI_TOP_MOST,
                  "ids are not 1 to 64 for each row");
        ERI_VALUE(t.sizes() == given.sizes(), "teacher has another shape than ids");
        ERI_VALUE(!records(t), "the teacher gets no gradient: detach it");
    }
    template <typename A> void into(A &a) const {
        a.ids = ids.t.const_data_ptr();
        a.teacher = values.t.const_data_ptr();
        a.ids_stride = ids.stride;
        a.teacher_stride = values.stride;
        a.ids_64 = ids.t.scalar_type() == at::kLong;
        a.teacher_dtype = tag_of(values.t.scalar_type());
        a.k = (int32_t)ids.cols;
    }
};

template <typename A> void logits_into(A &a, const Rows &x, PyObject *temperature) {
    a.logits = x.t.const_data_ptr();
    a.rows = (uint64_t)x.rows;
    a.vocab = (uint64_t)x.cols;
    a.logits_stride = x.stride;
    a.dtype_tag = tag_of(x.t.scalar_type());
    a.temperature = (float)number(temperature, "temperature");
}

/* token_logprobs(logits, ids, temperature, entropy, top) -> (logprob, entropy, top, top_ids, stats) */
PyObject *token_logprobs(PyObject *const *args) {
    const at::Tensor &logits = floats(args[0], "logits");
    const auto rows = rows_of(logits);
    const bool named = args[1] != Py_None, entropy = truth(args[3]);
    const uint64_t top = word(args[4], "top");
    ERI_VALUE(top <= ERI_TOP_MOST && top <= (uint64_t)logits.size(-1), "top is over 64 or over the vocabulary");
    const at::Tensor ids = named ? token_ids(args[1], logits) : at::Tensor();
    EriTokenLogprobs a = {};
    if (records(logits) && (named || entropy)) {
        number(args[2], "temperature");
        return Py_NewRef(Py_None);
    }
    const Rows x(logits);
    logits_into(a, x, args[2]);
    a.top_n = (int32_t)top;
    Outputs made;
    made.guard.reset_device(logits.device());
    check(eri_token_logprobs_workspace(a.rows, a.vocab, a.top_n, &a.workspace_bytes), "eri_token_logprobs_workspace");
    const at::Tensor stats = made.empty(with_last(rows, 2), at::kFloat, logits), workspace = made.empty({(int64_t)a.workspace_bytes}, at::kByte, logits);
    at::Tensor logprob, h, values, places;
    if (named) {
        logprob = made.empty(rows, at::kFloat, logits);
        a.ids = ids.const_data_ptr();
        a.ids_64 = ids.scalar_type() == at::kLong;
        a.logprob = static_cast<float *>(logprob.data_ptr());
    }
    if (entropy) {
        h = made.empty(rows, at::kFloat, logits);
        a.entropy = static_cast<float *>(h.data_ptr());
    }
    if (top) {
        values = made.empty(with_last(rows, (int64_t)top), at::kFloat, logits);
        places = made.empty(with_last(rows, (int64_t)top), at::kLong, logits);
        a.top = static_cast<float *>(values.data_ptr());
        a.top_ids = static_cast<int64_t *>(places.data_ptr());
    }
    a.stats = static_cast<float *>(stats.data_ptr());
    a.workspace = workspace.data_ptr();
    check(eri_token_logprobs(&a, stream_of(logits)), "eri_token_logprobs");
    return wrapped({logprob, h, values, places, stats});
}

/* The gradient's rows: new ones, or `out`, which may be the logits themselves. */
struct Gradient {
    Outputs made;
    Rows rows;
    static at::ScalarType dtype_of(PyObject *o, const at::Tensor &logits) {
        if (o == Py_None) return logits.scalar_type();
        if (!THPDtype_Check(o)) raise(PyExc_TypeError, "dtype is no dtype");
        const at::ScalarType t = reinterpret_cast<THPDtype *>(o)->scalar_type;
        if (t != at::kFloat && t != at::kBFloat16) raise(PyExc_TypeError, "Unsupported: a gradient is float32 or bfloat16");
        return t;
    }
    Outputs &on(const at::Tensor &logits) {
        made.guard.reset_device(logits.device());
        return made;
    }
    Gradient(PyObject *dtype, PyObject *out, const at::Tensor &logits)
        : rows(out == Py_None ? on(logits).empty(logits.sizes(), dtype_of(dtype, logits), logits) : (on(logits), written(out, "out", logits)), "out") {
        if (out == Py_None) return;
        ERI_VALUE(rows.t.sizes() == logits.sizes() && (dtype == Py_None || rows.t.scalar_type() == dtype_of(dtype, logits)), "out has another shape or dtype than the gradient");
    }
};
void apart_from(const Rows &out, const at::Tensor &t, const char *name) {
    if (t.defined()) apart(out, Rows(t), name);
}
/* Over the logits themselves each element is written by the thread that has read it. */
void apart_from_logits(const Rows &out, const Rows &x) {
    if (!(Span(out) == Span(x) && out.t.scalar_type() == x.t.scalar_type())) apart(out, x, "logits");
}

/* token_logprobs_grad(logits, ids, stats, grad, grad_entropy, entropy, temperature, dtype, out) -> logits' gradient */
PyObject *token_logprobs_grad(PyObject *const *args) {
    const at::Tensor &logits = floats(args[0], "logits");
    ERI_VALUE((args[1] == Py_None) == (args[3] == Py_None), "ids and grad are given together");
    ERI_VALUE((args[4] == Py_None) == (args[5] == Py_None), "grad_entropy and entropy are given together");
    ERI_VALUE(args[3] != Py_None || args[4] != Py_None, "neither grad nor grad_entropy is given");
    const at::Tensor stats = stats_of(args[2], 2, logits);
    at::Tensor ids, grad, grad_entropy, entropy;
    if (args[3] != Py_None) ids = token_ids(args[1], logits), grad = per_row(args[3], "grad", logits);
    if (args[4] != Py_None) grad_entropy = per_row(args[4], "grad_entropy", logits), entropy = per_row(args[5], "entropy", logits);
    const Rows x(logits);
    EriTokenLogprobsGrad a = {};
    logits_into(a, x, args[6]);
    const Gradient out(args[7], args[8], logits);
    if (args[8] != Py_None) {
        apart_from_logits(out.rows, x);
        apart_from(out.rows, stats, "stats"), apart_from(out.rows, ids, "ids"), apart_from(out.rows, grad, "grad");
        apart_from(out.rows, grad_entropy, "grad_entropy"), apart_from(out.rows, entropy, "entropy");
    }
    a.stats = static_cast<const float *>(stats.const_data_ptr());
    if (grad.defined()) {
        a.ids = ids.const_data_ptr();
        a.ids_64 = ids.scalar_type() == at::kLong;
        a.grad = static_cast<const float *>(grad.const_data_ptr());
    }
    if (grad_entropy.defined()) {
        a.grad_entropy = static_cast<const float *>(grad_entropy.const_data_ptr());
        a.entropy = static_cast<const float *>(entropy.const_data_ptr());
    }
    a.out = out.rows.t.data_ptr();
    a.out_stride = out.rows.stride;
    a.out_dtype = tag_of(out.rows.t.scalar_type());
    changed(out.rows.t);
    check(eri_token_logprobs_grad(&a, stream_of(logits)), "eri_token_logprobs_grad");
    return args[8] == Py_None ? wrapped(out.rows.t) : Py_NewRef(args[8]);
}

/* distill_top(logits, ids, teacher, temperature, rest) -> (loss, stats) */
PyObject *distill_top(PyObject *const *args) {
    const at::Tensor &logits = floats(args[0], "logits");
    const auto rows = rows_of(logits);
    const Teacher teacher(args[1], args[2], logits);
    const bool rest = truth(args[4]);
    if (records(logits)) {
        number(args[3], "temperature");
        return Py_NewRef(Py_None);
    }
    const Rows x(logits);
    EriDistillTop a = {};
    logits_into(a, x, args[3]);
    teacher.into(a);
    a.rest = rest;
    Outputs made;
    made.guard.reset_device(logits.device());
    check(eri_distill_top_workspace(a.rows, a.vocab, &a.workspace_bytes), "eri_distill_top_workspace");
    const at::Tensor loss = made.empty(rows, at::kFloat, logits), stats = made.empty(with_last(rows, 6), at::kFloat, logits);
    const at::Tensor workspace = made.empty({(int64_t)a.workspace_bytes}, at::kByte, logits);
    a.loss = static_cast<float *>(loss.data_ptr());
    a.stats = static_cast<float *>(stats.data_ptr());
    a.workspace = workspace.data_ptr();
    check(eri_distill_top(&a, stream_of(logits)), "eri_distill_top");
    return wrapped({loss, stats});
}

/* distill_top_grad(logits, ids, teacher, stats, grad, temperature, dtype, out) -> logits' gradient */
PyObject *distill_top_grad(PyObject *const *args) {
    const at::Tensor &logits = floats(args[0], "logits");
    const Teacher teacher(args[1], args[2], logits);
    const at::Tensor stats = stats_of(args[3], 6, logits), grad = per_row(args[4], "grad", logits);
    const Rows x(logits);
    EriDistillTopGrad a = {};
    logits_into(a, x, args[5]);
    teacher.into(a);
    const Gradient out(args[6], args[7], logits);
    if (args[7] != Py_None) {
        apart_from_logits(out.rows, x);
        apart_from(out.rows, stats, "stats"), apart_from(out.rows, grad, "grad");
        apart(out.rows, teacher.ids, "ids"), apart(out.rows, teacher.values, "teacher");
    }
    a.stats = static_cast<const float *>(stats.const_data_ptr());
    a.grad = static_cast<const float *>(grad.const_data_ptr());
    a.out = out.rows.t.data_ptr();
    a.out_stride = out.rows.stride;
    a.out_dtype = tag_of(out.rows.t.scalar_type());
    changed(out.rows.t);
    check(eri_distill_top_grad(&a, stream_of(logits)), "eri_distill_top_grad");
    return args[7] == Py_None ? wrapped(out.rows.t) : Py_NewRef(args[7]);
}

PyMethodDef methods[] = {method<token_logprobs, 5>("token_logprobs"), method<token_logprobs_grad, 9>("token_logprobs_grad"), method<distill_top, 5>("distill_top"),
                         method<distill_top_grad, 8>("distill_top_grad"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_losses_face", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__losses_face(void) { return PyModule_Create(&module); }

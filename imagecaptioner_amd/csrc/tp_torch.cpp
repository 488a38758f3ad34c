// The torch side of the calls that write replies (replies.py): argument checks, outputs and the call, as the Python module _tp_torch.
//
// A decoding loop makes these calls once per token, and for few rows the host's part of one takes longer than the GPU's.  The same checks by Python
// attribute accesses cost 3 to 5 us a call, and an output 1.4 us; here they cost 0.3 and 0.8 (a grammar step of one row: 12.2 us of host time before, 5.6 to 6.3 now,
// 0.1 of it for refusing tangents and views that negate).
// The library's functions come as addresses from whoever has loaded it.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/tagpipe.h"

namespace {

struct Refused {};                                                               // the Python error is set

struct Api {
    decltype(&tp_shape_logits) shape;
    decltype(&tp_choose_workspace) choose_workspace;
    decltype(&tp_choose_tokens) choose;
    decltype(&tp_grammar_mask) mask;
    decltype(&tp_grammar_step) step;
    decltype(&tp_lines_workspace) lines_workspace;
    decltype(&tp_grammar_lines) lines;
} api;
PyObject* failed = nullptr;                                                      // failed(rc) raises the library's error

// The calls allocate and launch without the interpreter's lock.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

void check(int rc) {
    if (rc == TP_OK) return;
    PyObject* r = PyObject_CallFunction(failed, "i", rc);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "error %d", rc);
    throw Refused{};
}

// whether something is to be differentiated by this tensor: backwards, or forwards (it carries a tangent)
bool differentiated(const at::Tensor& t) {
    return (t.requires_grad() && c10::GradMode::is_enabled()) || (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined());
}

// whether the values are not what stands in memory: a view that negates them (as the imaginary part of a conjugate does), or zeros without memory
bool lazy(const at::Tensor& t) { return t.is_neg() || t._is_zerotensor(); }

[[noreturn]] void refuse(const char* name, PyObject* o, int device, at::ScalarType dtype, int64_t rows, int64_t columns) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_ValueError, "%s must be a tensor, got %R", name, (PyObject*)Py_TYPE(o));
        throw Refused{};
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (differentiated(t)) {
        PyErr_Format(PyExc_ValueError, "%s requires a gradient, which this call does not have: detach it", name);
        throw Refused{};
    }
    if (lazy(t)) {
        PyErr_Format(PyExc_ValueError, "%s does not stand in memory as its values are (a negated view, or zeros without memory): clone or resolve it", name);
        throw Refused{};
    }
    std::string shape = "(" + std::to_string(rows) + (columns == -2 ? ",)" : ", " + std::to_string(columns) + ")");
    PyObject *is = PyObject_GetAttrString(o, "dtype"), *sizes = PyObject_GetAttrString(o, "shape"), *on = PyObject_GetAttrString(o, "device");
    if (is && sizes && on)
        PyErr_Format(PyExc_ValueError, "%s must be a %s tensor of the shape %s (-1: any) on cuda:%d, dense along its last axis, got %S %S on %S%s", name, at::toString(dtype), shape.c_str(), device,
                     is, sizes, on, t.layout() == at::kStrided && t.is_contiguous() ? "" : ", not contiguous");
    Py_XDECREF(is);
    Py_XDECREF(sizes);
    Py_XDECREF(on);
    throw Refused{};
}

bool usable(PyObject* o, int device, at::ScalarType dtype, int64_t dim) {
    if (!THPVariable_Check(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.scalar_type() == dtype && t.get_device() == device && t.layout() == at::kStrided && t.dim() == dim && !differentiated(t) && !lazy(t);
}

// A dense vector's data.
template <class E>
E* vec(const char* name, PyObject* o, int device, at::ScalarType dtype, int64_t rows) {
    if (!usable(o, device, dtype, 1)) refuse(name, o, device, dtype, rows, -2);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.size(0) != rows || !t.is_contiguous()) refuse(name, o, device, dtype, rows, -2);
    return (E*)t.data_ptr();
}

// A table's data, rows, columns and elements between rows (its columns where there is one row at most); rows or columns -1: any.
struct Table { void* p; int64_t rows, columns, stride; };
Table table(const char* name, PyObject* o, int device, at::ScalarType dtype, int64_t rows, int64_t columns, bool vector_too = false) {
    if (vector_too && usable(o, device, dtype, 1)) {                              // one row
        const at::Tensor& t = THPVariable_Unpack(o);
        if ((columns != -1 && t.size(0) != columns) || (t.size(0) > 1 && t.stride(0) != 1)) refuse(name, o, device, dtype, rows, columns);
        return Table{t.data_ptr(), 1, t.size(0), t.size(0)};
    }
    if (!usable(o, device, dtype, 2)) refuse(name, o, device, dtype, rows, columns);
    const at::Tensor& t = THPVariable_Unpack(o);
    const int64_t r = t.size(0), c = t.size(1);
    if ((rows != -1 && r != rows) || (columns != -1 && c != columns) || (c > 1 && t.stride(1) != 1)) refuse(name, o, device, dtype, rows, columns);
    return Table{t.data_ptr(), r, c, r > 1 ? t.stride(0) : c};
}

// A backward pass that has kept what a tensor held finds it changed.
void changed(PyObject* o) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

at::Tensor empty(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType dtype) { return at::empty(sizes, like.options().dtype(dtype).requires_grad(false)); }

[[noreturn]] void value_error(const char* what) {
    PyErr_SetString(PyExc_ValueError, what);
    throw Refused{};
}

enum Rule { HISTORY, HISTORY_LEN, PROMPT_LEN, REPETITION, FREQUENCY, PRESENCE, BIAS, BIAS_ROW, MASK, MASK_ROW, RULES };
const char* const rule_names[RULES] = {"history", "history_len", "prompt_len", "repetition", "frequency", "presence", "bias", "bias_row", "mask", "mask_row"};
PyObject* rule_keys[RULES];

// The rules of a call (a dict of keyword arguments) into io, whose type, rows and vocab are known.
void read_rules(PyObject* dict, int device, tp_logits& io, PyObject* (&rule)[RULES]) {
    Py_ssize_t known = 0;
    for (int k = 0; k < RULES; ++k) {
        rule[k] = dict ? PyDict_GetItemWithError(dict, rule_keys[k]) : nullptr;
        if (!rule[k] && PyErr_Occurred()) throw Refused{};
        known += rule[k] != nullptr;
        if (rule[k] == Py_None) rule[k] = nullptr;
    }
    if (dict && known != PyDict_Size(dict)) {
        PyObject *key, *value;
        for (Py_ssize_t at = 0; PyDict_Next(dict, &at, &key, &value);) {
            bool found = false;
            for (PyObject* name : rule_keys) found = found || PyUnicode_Compare(key, name) == 0;
            if (!found) PyErr_Format(PyExc_TypeError, "unexpected keyword argument %R", key);
        }
        throw Refused{};
    }
    const int64_t rows = (int64_t)io.rows, vocab = io.vocab;
    if (rule[HISTORY]) {
        const Table t = table("history", rule[HISTORY], device, at::kInt, rows, -1);
        if (t.columns > INT32_MAX) value_error("history has 2^31 columns or more");
        if (rule[HISTORY_LEN]) io.history_len = vec<int32_t>("history_len", rule[HISTORY_LEN], device, at::kInt, rows);
        if (rule[PROMPT_LEN]) io.prompt_len = vec<int32_t>("prompt_len", rule[PROMPT_LEN], device, at::kInt, rows);
        io.history = (int32_t*)t.p;
        io.history_cap = (uint32_t)t.columns;
        io.history_stride = (uint64_t)t.stride;
        if (!t.p) io.history_len = nullptr, io.prompt_len = nullptr;             // no rows, or rows of no room: there is no history, whatever the lengths say
    } else if (rule[HISTORY_LEN] || rule[PROMPT_LEN]) {
        value_error("history_len or prompt_len without a history");
    }
    if (rule[REPETITION]) io.repetition = vec<float>("repetition", rule[REPETITION], device, at::kFloat, rows);
    if (rule[FREQUENCY]) io.frequency = vec<float>("frequency", rule[FREQUENCY], device, at::kFloat, rows);
    if (rule[PRESENCE]) io.presence = vec<float>("presence", rule[PRESENCE], device, at::kFloat, rows);
    auto rows_of = [&](Rule which, Rule row, at::ScalarType dtype, int64_t columns, const void*& p, uint64_t& stride, const int32_t*& row_of, uint32_t& n) {
        if (!rule[which]) {
            if (!rule[row]) return;
            PyErr_Format(PyExc_ValueError, "%s without a %s", rule_names[row], rule_names[which]);
            throw Refused{};
        }
        const Table t = table(rule_names[which], rule[which], device, dtype, -1, columns, true);
        if (t.rows < 1 || t.rows > INT32_MAX) {
            PyErr_Format(PyExc_ValueError, "%s has %lld rows", rule_names[which], (long long)t.rows);
            throw Refused{};
        }
        if (rule[row]) row_of = vec<int32_t>(rule_names[row], rule[row], device, at::kInt, rows);
        p = t.p;
        stride = (uint64_t)t.stride;
        n = (uint32_t)t.rows;
    };
    const void *bias = nullptr, *mask = nullptr;
    rows_of(BIAS, BIAS_ROW, at::kFloat, vocab, bias, io.bias_stride, io.bias_row, io.n_bias);
    rows_of(MASK, MASK_ROW, at::kInt, (vocab + 31) / 32, mask, io.mask_stride, io.mask_row, io.n_masks);
    io.bias = (const float*)bias;
    io.mask = (const uint32_t*)mask;
}

tp_logits empty_logits(void* stream) {
    tp_logits io{};
    io.struct_size = sizeof io;
    io.type = TP_T_F32;
    io.stream = stream;
    return io;
}

tp_logits read_logits(PyObject* o, int device, void* stream, PyObject* dict, PyObject* (&rule)[RULES]) {
    tp_logits io = empty_logits(stream);
    if (!THPVariable_Check(o)) refuse("logits", o, device, at::kFloat, -1, -1);
    const at::ScalarType type = THPVariable_Unpack(o).scalar_type();
    if (type != at::kFloat && type != at::kHalf && type != at::kBFloat16) value_error("logits must be a float32, float16 or bfloat16 tensor [rows, vocab]");
    const Table t = table("logits", o, device, type, -1, -1);
    if (t.columns > UINT32_MAX) value_error("logits have 2^32 columns or more");
    io.type = type == at::kFloat ? TP_T_F32 : type == at::kHalf ? TP_T_F16 : TP_T_BF16;
    io.rows = (uint64_t)t.rows;
    io.vocab = (uint32_t)t.columns;
    io.logits = t.p;
    io.stride = (uint64_t)t.stride;
    read_rules(dict, device, io, rule);
    return io;
}

struct Sampling { const float *temperature = nullptr, *uniform = nullptr; };
Sampling read_sampling(PyObject* temperature, PyObject* uniform, int device, int64_t rows) {
    Sampling s;
    if (temperature != Py_None) s.temperature = vec<float>("temperature", temperature, device, at::kFloat, rows);
    if (uniform != Py_None) s.uniform = vec<float>("uniform", uniform, device, at::kFloat, rows);
    if (temperature != Py_None && uniform == Py_None) value_error("a temperature needs `uniform`, the random numbers of the choice");
    return s;
}

void* address(PyObject* o) {                                                     // None: 0, which the library refuses
    if (o == Py_None) return nullptr;
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw Refused{};
    return p;
}
int small(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{};
    return (int)v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused{};
    return v != 0;
}

template <class F>
PyObject* call(Py_ssize_t given, Py_ssize_t wanted, F&& f) {
    HANDLE_TH_ERRORS
    if (given != wanted) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", given, wanted);
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
    PyObject *x = THPVariable_Wrap(a), *y = THPVariable_Wrap(b), *r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
}

// (ctx, device, stream, logits, out or None, rules)
PyObject* shape(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 6, [&]() -> PyObject* {
        PyObject* rule[RULES];
        const int device = small(a[1]);
        const tp_logits io = read_logits(a[3], device, address(a[2]), a[5], rule);
        tp_ctx* ctx = (tp_ctx*)address(a[0]);
        if (a[4] != Py_None) {
            const at::ScalarType type = THPVariable_Unpack(a[3]).scalar_type();
            const Table to = table("out", a[4], device, type, (int64_t)io.rows, io.vocab);
            changed(a[4]);
            int rc;
            {
                Unlocked u;
                rc = api.shape(ctx, &io, to.p, (uint64_t)to.stride);
            }
            check(rc);
            Py_INCREF(a[4]);
            return a[4];
        }
        at::Tensor out;
        int rc;
        {
            Unlocked u;
            const at::Tensor& logits = THPVariable_Unpack(a[3]);
            out = empty(logits, {(int64_t)io.rows, (int64_t)io.vocab}, logits.scalar_type());
            rc = api.shape(ctx, &io, out.data_ptr(), io.vocab);
        }
        check(rc);
        return THPVariable_Wrap(out);
    });
}

// (ctx, device, stream, logits, temperature, uniform, rules)
PyObject* choose(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 7, [&]() -> PyObject* {
        PyObject* rule[RULES];
        const int device = small(a[1]);
        const tp_logits io = read_logits(a[3], device, address(a[2]), a[6], rule);
        const Sampling s = read_sampling(a[4], a[5], device, (int64_t)io.rows);
        tp_ctx* ctx = (tp_ctx*)address(a[0]);
        at::Tensor tokens, logprob, workspace;
        int rc;
        {
            Unlocked u;
            const at::Tensor& logits = THPVariable_Unpack(a[3]);
            const uint64_t need = api.choose_workspace(io.rows, io.vocab);
            if (need) workspace = empty(logits, {(int64_t)need}, at::kByte);       // torch's own pool keeps it apart per stream and per graph
            tokens = empty(logits, {(int64_t)io.rows}, at::kInt);
            logprob = empty(logits, {(int64_t)io.rows}, at::kFloat);
            rc = api.choose(ctx, &io, s.temperature, s.uniform, (int32_t*)tokens.data_ptr(), (float*)logprob.data_ptr(), need ? workspace.data_ptr() : nullptr, need);
        }
        check(rc);
        return pair(tokens, logprob);
    });
}

Table read_states(PyObject* o, int device) {
    const Table t = table("states", o, device, at::kInt, -1, 2);
    if (t.stride != 2) value_error("states must be dense");
    return t;
}

// (grammar, device, stream, states, words, out or None)
PyObject* mask(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 6, [&]() -> PyObject* {
        const int device = small(a[1]);
        const int64_t words = small(a[4]);
        const tp_grammar* g = (const tp_grammar*)address(a[0]);
        void* stream = address(a[2]);
        const Table states = read_states(a[3], device);
        at::Tensor made;
        Table to{};
        if (a[5] != Py_None) {
            to = table("out", a[5], device, at::kInt, states.rows, words);
            changed(a[5]);
        }
        int rc;
        {
            Unlocked u;
            if (a[5] == Py_None) {
                made = empty(THPVariable_Unpack(a[3]), {states.rows, words}, at::kInt);
                to = Table{made.data_ptr(), states.rows, words, words};
            }
            rc = api.mask(g, (const int32_t*)states.p, (uint64_t)states.rows, (uint32_t*)to.p, (uint64_t)to.stride, stream);
        }
        check(rc);
        if (a[5] == Py_None) return THPVariable_Wrap(made);
        Py_INCREF(a[5]);
        return a[5];
    });
}

// what an appending step changes
void appended(PyObject* const (&rule)[RULES], bool append) {
    if (append && rule[HISTORY] && rule[HISTORY_LEN]) {
        changed(rule[HISTORY]);
        changed(rule[HISTORY_LEN]);
    }
}

// (grammar, device, stream, states, logits, temperature, uniform, append, rules)
PyObject* step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 9, [&]() -> PyObject* {
        PyObject* rule[RULES];
        const int device = small(a[1]);
        const tp_grammar* g = (const tp_grammar*)address(a[0]);
        const Table states = read_states(a[3], device);
        const tp_logits io = read_logits(a[4], device, address(a[2]), a[8], rule);
        if ((int64_t)io.rows != states.rows) value_error("one state per row of logits");
        const Sampling s = read_sampling(a[5], a[6], device, states.rows);
        const bool append = truth(a[7]);
        changed(a[3]);
        appended(rule, append);
        at::Tensor tokens, logprob;
        int rc;
        {
            Unlocked u;
            const at::Tensor& like = THPVariable_Unpack(a[3]);
            tokens = empty(like, {states.rows}, at::kInt);
            logprob = empty(like, {states.rows}, at::kFloat);
            rc = api.step(g, &io, s.temperature, s.uniform, (int32_t*)states.p, (int32_t*)tokens.data_ptr(), (float*)logprob.data_ptr(), append);
        }
        check(rc);
        return pair(tokens, logprob);
    });
}

// (grammar, device, stream, states, n_tokens, tokens, append, rules)
PyObject* advance(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 8, [&]() -> PyObject* {
        PyObject* rule[RULES];
        const int device = small(a[1]);
        const tp_grammar* g = (const tp_grammar*)address(a[0]);
        const Table states = read_states(a[3], device);
        tp_logits io = empty_logits(address(a[2]));
        io.rows = (uint64_t)states.rows;
        io.vocab = (uint32_t)small(a[4]);
        read_rules(a[7], device, io, rule);
        int32_t* tokens = vec<int32_t>("tokens", a[5], device, at::kInt, states.rows);
        const bool append = truth(a[6]);
        changed(a[3]);
        appended(rule, append);
        int rc;
        {
            Unlocked u;
            rc = api.step(g, &io, nullptr, nullptr, (int32_t*)states.p, tokens, nullptr, append);
        }
        check(rc);
        Py_RETURN_NONE;
    });
}

// (grammar, device, stream, tokens, lengths, begin, arena or None, longest token)
PyObject* lines(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 8, [&]() -> PyObject* {
        const int device = small(a[1]);
        const tp_grammar* g = (const tp_grammar*)address(a[0]);
        void* stream = address(a[2]);
        const Table t = table("tokens", a[3], device, at::kInt, -1, -1);
        if (t.columns > INT32_MAX) value_error("tokens have 2^31 columns or more");
        const int32_t* len = a[4] == Py_None ? nullptr : vec<int32_t>("lengths", a[4], device, at::kInt, t.rows);
        const int32_t* begin = a[5] == Py_None ? nullptr : vec<int32_t>("begin", a[5], device, at::kInt, t.rows);
        const int64_t longest = small(a[7]);
        at::Tensor arena, offsets, workspace;
        if (a[6] != Py_None) {
            if (!usable(a[6], device, at::kByte, 1) || !THPVariable_Unpack(a[6]).is_contiguous()) refuse("arena", a[6], device, at::kByte, -1, -2);
            arena = THPVariable_Unpack(a[6]);
            changed(a[6]);
        }
        int rc;
        {
            Unlocked u;
            const at::Tensor& like = THPVariable_Unpack(a[3]);
            if (a[6] == Py_None) arena = empty(like, {t.rows * t.columns * longest + 16}, at::kByte);
            offsets = t.rows ? empty(like, {t.rows + 1}, at::kLong) : at::zeros({1}, like.options().dtype(at::kLong));
            const uint64_t need = api.lines_workspace((uint64_t)t.rows);
            workspace = empty(like, {(int64_t)need}, at::kByte);
            rc = api.lines(g, (const int32_t*)t.p, (uint64_t)t.stride, (uint32_t)t.columns, begin, len, (uint64_t)t.rows, (uint8_t*)arena.data_ptr(), (uint64_t)arena.numel(),
                           (uint64_t*)offsets.data_ptr(), workspace.data_ptr(), need, stream);
        }
        check(rc);
        return pair(arena, offsets);
    });
}

// (the seven functions' addresses, what raises the library's error)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 8, [&]() -> PyObject* {
        api.shape = (decltype(api.shape))address(a[0]);
        api.choose_workspace = (decltype(api.choose_workspace))address(a[1]);
        api.choose = (decltype(api.choose))address(a[2]);
        api.mask = (decltype(api.mask))address(a[3]);
        api.step = (decltype(api.step))address(a[4]);
        api.lines_workspace = (decltype(api.lines_workspace))address(a[5]);
        api.lines = (decltype(api.lines))address(a[6]);
        Py_INCREF(a[7]);
        Py_XSETREF(failed, a[7]);
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},       {"shape", (PyCFunction)(void*)shape, METH_FASTCALL, nullptr},
    {"choose", (PyCFunction)(void*)choose, METH_FASTCALL, nullptr},   {"mask", (PyCFunction)(void*)mask, METH_FASTCALL, nullptr},
    {"step", (PyCFunction)(void*)step, METH_FASTCALL, nullptr},       {"advance", (PyCFunction)(void*)advance, METH_FASTCALL, nullptr},
    {"lines", (PyCFunction)(void*)lines, METH_FASTCALL, nullptr},     {nullptr, nullptr, 0, nullptr},
};
// The torch whose headers this was compiled with: another one's tensors may be laid out otherwise, so whoever loads the module compares, and the build looks for the text
// in the file.
const char built_for[] = "torch module for " TP_TORCH_NAME;

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tp_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tp_torch() {
    for (int k = 0; k < RULES; ++k)
        if (!(rule_keys[k] = PyUnicode_InternFromString(rule_names[k]))) return nullptr;
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", built_for) < 0) Py_CLEAR(m);
    return m;
}

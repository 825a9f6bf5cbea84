// khq_paged_py.cpp -- the module khq._paged: the calls of khq/paged.py without
// the interpreter.  A decode step's calls run for 4 to 10 us each, and their
// checks in Python took 5 to 9.  A Call stands before one of that file's functions
// and takes the same arguments: where all of them are what the function would
// pass on (plain tensors of the right type, size, layout and device), it goes
// to the C entry; anything else, also what is wrong and has to be said so, is
// the Python function's, which is asked with the same arguments.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <structmember.h>
#include <torch/csrc/autograd/python_variable.h>

#include <hip/hip_runtime.h>

#include <cstring>

#include "khq_paged.h"

namespace {

PyObject* g_error = nullptr;   // KhqError(name, status)
PyObject* g_stream = nullptr;  // device index -> handle of its current stream

// ------------------------------------------------------------ arguments
// Arguments of one call by their places in `names`, null where not given.
template <int N>
struct Names {
    PyObject* at[N];
    int positional;  // the first ones may come without a name
    bool take(PyObject* const* args, Py_ssize_t n, PyObject* kw, PyObject** out) const {
        for (int i = 0; i < N; i++) out[i] = nullptr;
        if (n > positional) return false;
        for (Py_ssize_t i = 0; i < n; i++) out[i] = args[i];
        const Py_ssize_t n_kw = kw ? PyTuple_GET_SIZE(kw) : 0;
        int next = (int)n;
        for (Py_ssize_t i = 0; i < n_kw; i++) {
            PyObject* const name = PyTuple_GET_ITEM(kw, i);  // interned, as `at` is
            int k = next;
            for (int seen = 0; at[k % N] != name; k++)
                if (++seen == N) return false;
            k %= N;
            if (out[k]) return false;
            out[k] = args[n + i];
            next = k + 1;
        }
        return true;
    }
};

bool none(PyObject* o) { return !o || o == Py_None; }

bool to_int(PyObject* o, int* v) {
    if (!o || !PyLong_CheckExact(o)) return false;
    int overflow = 0;
    const long long x = PyLong_AsLongLongAndOverflow(o, &overflow);
    if (overflow || x < INT32_MIN || x > INT32_MAX) return false;
    *v = (int)x;
    return true;
}

bool to_double(PyObject* o, double* v) {
    if (!o || !PyFloat_CheckExact(o)) return false;
    *v = PyFloat_AS_DOUBLE(o);
    return true;
}

const at::Tensor* tensor(PyObject* o) {
    return o && THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

// The index of the current device, `t`'s: -1 where it is none of those.
int device_of(const at::Tensor* t) {
    int current = -1;
    if (!t || !t->is_cuda() || hipGetDevice(&current) != hipSuccess) return -1;
    return t->get_device() == current ? current : -1;
}

bool i32(PyObject* o, long long n, int device, int** p) {
    const at::Tensor* const t = tensor(o);
    if (!t || t->scalar_type() != at::kInt || t->numel() != n || !t->is_cuda() ||
        t->get_device() != device || !t->is_contiguous())
        return false;
    *p = static_cast<int*>(t->data_ptr());
    return true;
}

bool table_of(PyObject* o, int device, int** p, int* n_seq, int* width) {
    const at::Tensor* const t = tensor(o);
    if (!t || t->dim() != 2 || t->size(0) <= 0 || t->size(0) > KHQ_PAGED_MAX_SEQ ||
        t->size(1) <= 0 || t->size(1) > INT32_MAX || !i32(o, t->numel(), device, p))
        return false;
    *n_seq = (int)t->size(0);
    *width = (int)t->size(1);
    return true;
}

struct Heads {
    void* p;
    long long token, head;
};
// [n][h][d] of this type with dense dims; one that is written must not overlap itself.
bool heads(PyObject* o, int64_t n, int64_t h, int64_t d, at::ScalarType dt, int device, bool write, Heads* x) {
    const at::Tensor* const t = tensor(o);
    if (!t || t->scalar_type() != dt || t->dim() != 3 || t->size(0) != n || t->size(1) != h ||
        t->size(2) != d || !t->is_cuda() || t->get_device() != device || t->stride(2) != 1)
        return false;
    *x = Heads{t->data_ptr(), t->stride(0), t->stride(1)};
    return !write || (x->head >= d && x->token >= (h - 1) * x->head + d);
}

bool pages_of(PyObject* ok, PyObject* ov, at::ScalarType dt, int device, khq_pages* p) {
    const at::Tensor *const k = tensor(ok), *const v = tensor(ov);
    if (!k || !v || k->scalar_type() != dt || v->scalar_type() != dt || k->dim() != 4 || !k->is_cuda() ||
        !v->is_cuda() || k->get_device() != device || v->get_device() != device ||
        k->sizes() != v->sizes() || k->strides() != v->strides() || k->numel() == 0)
        return false;
    const int64_t d = k->size(3);
    if ((d != 64 && d != 128 && d != 256) || k->stride(3) != 1 || k->size(1) > INT32_MAX ||
        k->size(2) > INT32_MAX || k->size(0) > INT32_MAX / k->size(1))
        return false;
    *p = khq_pages{k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1), k->stride(2), (int)k->size(0),
                   (int)k->size(1), (int)k->size(2), (int)d, dt == at::kHalf ? KHQ_FP16 : KHQ_BF16};
    return ((p->page_stride | p->token_stride | p->head_stride) & 7) == 0 &&
           ((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15) == 0;
}

// The last arguments of each call: whether a status raises, and where to launch
// (only the current stream is taken here).
bool launch_of(PyObject* check, PyObject* stream, int device, bool* raise, hipStream_t* st) {
    if (!none(stream) || (check && check != Py_True && check != Py_False)) return false;
    *raise = check != Py_False;
    PyObject* const index = PyLong_FromLong(device);
    if (!index) return false;
    PyObject* const h = PyObject_CallOneArg(g_stream, index);
    Py_DECREF(index);
    if (!h) return false;
    *st = static_cast<hipStream_t>(PyLong_AsVoidPtr(h));
    Py_DECREF(h);
    return !PyErr_Occurred();
}

PyObject* status_of(int rc, bool raise, const char* name) {
    if (rc != 0 && raise) {
        PyObject* const e = PyObject_CallFunction(g_error, "si", name, rc);
        if (e) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
        return nullptr;
    }
    return PyLong_FromLong(rc);
}

bool dtype_ok(const at::Tensor* t) {
    return t && (t->scalar_type() == at::kHalf || t->scalar_type() == at::kBFloat16);
}

// ---------------------------------------------------------------- the calls
// Each returns false for what the Python function is to have.
enum { PL_Q, PL_KV, PL_TABLE, PL_FREE, PL_STATE, PL_SIZE, PL_CU, PL_SEQ, PL_KV_OUT, PL_STATE_OUT, PL_STATUS,
       PL_POS, PL_SLOTS, PL_CHECK, PL_STREAM, PL_N };
Names<PL_N> plan_names;

bool plan(PyObject* const* args, Py_ssize_t n, PyObject* kw, PyObject** result) {
    PyObject* o[PL_N];
    if (!plan_names.take(args, n, kw, o)) return false;
    const at::Tensor *const q = tensor(o[PL_Q]), *const free = tensor(o[PL_FREE]), *const pos = tensor(o[PL_POS]);
    const int device = device_of(q);
    int *p[PL_N], n_seq, width, page_size;
    if (device < 0 || !free || !pos || !table_of(o[PL_TABLE], device, &p[PL_TABLE], &n_seq, &width) ||
        !to_int(o[PL_SIZE], &page_size) || page_size <= 0)
        return false;
    const int64_t n_pages = free->numel(), n_tok = pos->numel();
    if (n_pages > INT32_MAX || n_tok > INT32_MAX || n_tok == 0) return false;
    const struct { int at; int64_t n; } ints[] = {
        {PL_Q, n_seq}, {PL_KV, n_seq}, {PL_FREE, n_pages}, {PL_STATE, 2}, {PL_CU, n_seq + 1}, {PL_SEQ, n_seq},
        {PL_KV_OUT, n_seq}, {PL_STATE_OUT, 2}, {PL_STATUS, 1}, {PL_POS, n_tok}, {PL_SLOTS, n_tok}};
    for (const auto& x : ints)
        if (!i32(o[x.at], x.n, device, &p[x.at])) return false;
    bool raise;
    hipStream_t st;
    if (!launch_of(o[PL_CHECK], o[PL_STREAM], device, &raise, &st)) return false;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = khq_paged_plan(p[PL_Q], p[PL_KV], p[PL_TABLE], width, p[PL_FREE], p[PL_STATE], n_seq, (int)n_pages,
                        page_size, (int)n_tok, p[PL_CU], p[PL_SEQ], p[PL_KV_OUT], p[PL_STATE_OUT],
                        p[PL_STATUS], p[PL_POS], p[PL_SLOTS], st);
    Py_END_ALLOW_THREADS
    *result = status_of(rc, raise, "khq_paged_plan");
    return true;
}

enum { RO_Q, RO_K, RO_Q_OUT, RO_POS, RO_POS0, RO_QW, RO_KW, RO_EPS, RO_THETA, RO_DIM, RO_K_OUT, RO_K_NORMED, RO_V,
       RO_KP, RO_VP, RO_SLOTS, RO_ROUND, RO_CHECK, RO_STREAM, RO_N };
Names<RO_N> rows_names;

bool weight_of(PyObject* o, int64_t d, int device, const float** w) {
    *w = nullptr;
    if (none(o)) return true;
    const at::Tensor* const t = tensor(o);
    if (!t || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != d || !t->is_cuda() ||
        t->get_device() != device || !t->is_contiguous())
        return false;
    *w = static_cast<const float*>(t->data_ptr());
    return true;
}

// (a call of queries and keys; of one of them alone it is the Python function's)
bool rows(PyObject* const* args, Py_ssize_t n, PyObject* kw, PyObject** result) {
    PyObject* o[RO_N];
    if (!rows_names.take(args, n, kw, o)) return false;
    const at::Tensor *const q = tensor(o[RO_Q]), *const k = tensor(o[RO_K]);
    const int device = device_of(q);
    if (device < 0 || !k || !dtype_ok(q) || q->dim() != 3 || k->dim() != 3 || q->numel() == 0 || k->numel() == 0 ||
        q->size(0) > INT32_MAX || q->size(1) > INT32_MAX || k->size(1) > INT32_MAX)
        return false;
    const at::ScalarType dt = q->scalar_type();
    const int64_t m = q->size(0), hq = q->size(1), hk = k->size(1), d = q->size(2);
    if (d != 64 && d != 128 && d != 256) return false;
    khq_rows r{};
    r.eps = 1e-6f;
    r.theta = 1e7;
    r.rotary_dim = 64;
    r.n = (int)m;
    r.H_q = (int)hq;
    r.H_kv = (int)hk;
    r.head_dim = (int)d;
    r.dtype = dt == at::kHalf ? KHQ_FP16 : KHQ_BF16;
    Heads qi, qo, ki, x;
    if (!heads(o[RO_Q], m, hq, d, dt, device, false, &qi) || !heads(o[RO_Q_OUT], m, hq, d, dt, device, true, &qo) ||
        !heads(o[RO_K], m, hk, d, dt, device, false, &ki))
        return false;
    r.q = qi.p, r.q_token = qi.token, r.q_head = qi.head;
    r.q_out = qo.p, r.q_out_token = qo.token, r.q_out_head = qo.head;
    r.k = ki.p, r.k_token = ki.token, r.k_head = ki.head;
    if (!none(o[RO_K_OUT])) {
        if (!heads(o[RO_K_OUT], m, hk, d, dt, device, true, &x)) return false;
        r.k_out = x.p, r.k_out_token = x.token, r.k_out_head = x.head;
    }
    if (!none(o[RO_K_NORMED])) {
        if (!heads(o[RO_K_NORMED], m, hk, d, dt, device, true, &x)) return false;
        r.k_normed = x.p, r.k_normed_token = x.token, r.k_normed_head = x.head;
    }
    if (!weight_of(o[RO_QW], d, device, &r.q_weight) || !weight_of(o[RO_KW], d, device, &r.k_weight)) return false;
    double eps;
    if (o[RO_EPS]) {
        if (!to_double(o[RO_EPS], &eps)) return false;
        r.eps = (float)eps;
    }
    if ((o[RO_THETA] && !to_double(o[RO_THETA], &r.theta)) || (o[RO_DIM] && !to_int(o[RO_DIM], &r.rotary_dim)) ||
        (o[RO_POS0] && !to_int(o[RO_POS0], &r.pos0)))
        return false;
    if (o[RO_ROUND]) {
        if (!PyBool_Check(o[RO_ROUND])) return false;
        r.round_norm = o[RO_ROUND] == Py_True;
    }
    int* ints;
    if (!none(o[RO_POS])) {
        if (!i32(o[RO_POS], m, device, &ints)) return false;
        r.positions = ints;
    }
    khq_pages pages;
    const bool paged = !none(o[RO_KP]);
    if (paged) {
        if (!pages_of(o[RO_KP], o[RO_VP], dt, device, &pages) || pages.H_kv != hk || pages.head_dim != d ||
            !heads(o[RO_V], m, hk, d, dt, device, false, &x) || !i32(o[RO_SLOTS], m, device, &ints))
            return false;
        r.v = x.p, r.v_token = x.token, r.v_head = x.head;
        r.slots = ints;
    } else if (!none(o[RO_VP]) || !none(o[RO_V]) || !none(o[RO_SLOTS]) || (!r.k_out && !r.k_normed)) {
        return false;
    }
    bool raise;
    hipStream_t st;
    if (!launch_of(o[RO_CHECK], o[RO_STREAM], device, &raise, &st)) return false;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = khq_qk_norm_rope(&r, paged ? &pages : nullptr, st);
    Py_END_ALLOW_THREADS
    *result = status_of(rc, raise, "khq_qk_norm_rope");
    return true;
}

enum { AT_Q, AT_KP, AT_VP, AT_OUT, AT_CU, AT_SEQ, AT_TABLE, AT_MAX_Q, AT_SCALE, AT_GATE, AT_WS, AT_CHECK, AT_STREAM,
       AT_N };
Names<AT_N> attn_names;

bool attn(PyObject* const* args, Py_ssize_t n, PyObject* kw, PyObject** result) {
    PyObject* o[AT_N];
    if (!attn_names.take(args, n, kw, o)) return false;
    const at::Tensor* const q = tensor(o[AT_Q]);
    const int device = device_of(q);
    if (device < 0 || !dtype_ok(q) || q->dim() != 3 || q->numel() == 0 || q->size(0) > INT32_MAX ||
        q->size(1) > INT32_MAX)
        return false;
    const at::ScalarType dt = q->scalar_type();
    const int64_t m = q->size(0), hq = q->size(1);
    khq_pages pages;
    khq_attn_rows r{};
    Heads x;
    if (!pages_of(o[AT_KP], o[AT_VP], dt, device, &pages) || hq % pages.H_kv != 0) return false;
    const int64_t d = pages.head_dim;
    if (!heads(o[AT_Q], m, hq, d, dt, device, false, &x)) return false;
    r.q = x.p, r.q_token = x.token, r.q_head = x.head;
    if (!heads(o[AT_OUT], m, hq, d, dt, device, true, &x)) return false;
    r.out = x.p, r.out_token = x.token, r.out_head = x.head;
    if (!none(o[AT_GATE])) {
        if (!heads(o[AT_GATE], m, hq, d, dt, device, false, &x)) return false;
        r.gate = x.p, r.gate_token = x.token, r.gate_head = x.head;
    }
    int *table, *cu, *kv;
    double scale;
    if (!table_of(o[AT_TABLE], device, &table, &r.n_seq, &r.table_ld) ||
        !i32(o[AT_CU], (long long)r.n_seq + 1, device, &cu) || !i32(o[AT_SEQ], r.n_seq, device, &kv) ||
        !to_int(o[AT_MAX_Q], &r.max_q) || !to_double(o[AT_SCALE], &scale))
        return false;
    r.table = table, r.cu_q = cu, r.seq_kv = kv;
    r.scale = (float)scale;
    r.n_tok = (int)m;
    r.H_q = (int)hq;
    if (!none(o[AT_WS])) {
        const at::Tensor* const w = tensor(o[AT_WS]);
        if (!w || !w->is_cuda() || w->get_device() != device || !w->is_contiguous() || w->numel() == 0) return false;
        r.ws = w->data_ptr();
        r.ws_bytes = w->nbytes();
    }
    bool raise;
    hipStream_t st;
    if (!launch_of(o[AT_CHECK], o[AT_STREAM], device, &raise, &st)) return false;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = khq_paged_attn(&r, &pages, st);
    Py_END_ALLOW_THREADS
    *result = status_of(rc, raise, "khq_paged_attn");
    return true;
}

// ------------------------------------------------------------- the objects
struct Call {
    PyObject_HEAD
    PyObject* dict;
    PyObject* func;  // the Python function
    bool (*fast)(PyObject* const*, Py_ssize_t, PyObject*, PyObject**);
    vectorcallfunc vectorcall;
};

PyObject* call(PyObject* self, PyObject* const* args, size_t nf, PyObject* kw) {
    Call* const c = reinterpret_cast<Call*>(self);
    PyObject* result = nullptr;
    if (c->fast(args, PyVectorcall_NARGS(nf), kw, &result)) return result;
    if (PyErr_Occurred()) return nullptr;
    return PyObject_Vectorcall(c->func, args, nf, kw);
}

PyObject* call_new(PyTypeObject* type, PyObject* args, PyObject* kw) {
    PyObject* func;
    if ((kw && PyDict_GET_SIZE(kw)) || !PyArg_ParseTuple(args, "O", &func)) return nullptr;
    PyObject* const name = PyObject_GetAttrString(func, "__name__");
    if (!name) return nullptr;
    const char* const s = PyUnicode_AsUTF8(name);
    auto* const fast = !s ? nullptr : !strcmp(s, "plan") ? plan : !strcmp(s, "qk_norm_rope") ? rows
                       : !strcmp(s, "attn") ? attn : nullptr;
    Py_DECREF(name);
    if (!fast) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no call of this name");
        return nullptr;
    }
    Call* const c = reinterpret_cast<Call*>(type->tp_alloc(type, 0));
    if (!c) return nullptr;
    Py_INCREF(func);
    c->func = func;
    c->fast = fast;
    c->vectorcall = call;
    return reinterpret_cast<PyObject*>(c);
}

void call_free(PyObject* self) {
    Call* const c = reinterpret_cast<Call*>(self);
    Py_XDECREF(c->dict);
    Py_XDECREF(c->func);
    Py_TYPE(self)->tp_free(self);
}

PyGetSetDef call_getset[] = {{"__dict__", PyObject_GenericGetDict, PyObject_GenericSetDict, nullptr, nullptr}, {}};

PyTypeObject CallType = {PyVarObject_HEAD_INIT(nullptr, 0) "khq._paged.Call"};

template <int N>
bool intern(Names<N>& names, int positional, const char* const (&s)[N]) {
    names.positional = positional;
    for (int i = 0; i < N; i++)
        if (!(names.at[i] = PyUnicode_InternFromString(s[i]))) return false;
    return true;
}

// init(error, stream): the class that a status raises, and the current stream's function
PyObject* init(PyObject*, PyObject* args) {
    PyObject *error, *stream;
    if (!PyArg_ParseTuple(args, "OO", &error, &stream)) return nullptr;
    Py_INCREF(error);
    Py_INCREF(stream);
    Py_XSETREF(g_error, error);
    Py_XSETREF(g_stream, stream);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"init", init, METH_VARARGS, nullptr}, {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged() {
    CallType.tp_basicsize = sizeof(Call);
    CallType.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
    CallType.tp_vectorcall_offset = offsetof(Call, vectorcall);
    CallType.tp_dictoffset = offsetof(Call, dict);
    CallType.tp_call = PyVectorcall_Call;
    CallType.tp_new = call_new;
    CallType.tp_dealloc = call_free;
    CallType.tp_getset = call_getset;
    if (PyType_Ready(&CallType) < 0 ||
        !intern(plan_names, 5, {"q_len", "kv_len", "table", "free_pages", "state", "page_size", "cu_q", "seq_kv",
                                "kv_out", "state_out", "status", "positions", "slots", "check", "stream"}) ||
        !intern(rows_names, 3, {"q", "k", "q_out", "positions", "pos0", "q_weight", "k_weight", "eps", "theta",
                                "rotary_dim", "k_out", "k_normed", "v", "k_pages", "v_pages", "slots",
                                "round_norm", "check", "stream"}) ||
        !intern(attn_names, 4, {"q", "k_pages", "v_pages", "out", "cu_q", "seq_kv", "table", "max_q", "scale",
                                "gate", "workspace", "check", "stream"}))
        return nullptr;
    PyObject* const m = PyModule_Create(&module);
    if (!m) return nullptr;
    Py_INCREF(&CallType);
    if (PyModule_AddObject(m, "Call", reinterpret_cast<PyObject*>(&CallType)) < 0) return nullptr;
    return m;
}

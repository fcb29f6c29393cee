/* The Python calls of the operators over device tensors (llm_b200/__init__.py).
 *
 * A decoding step's kernels take a few microseconds, and checking a dozen
 * tensors' types, shapes and strides in Python takes as long; here it takes
 * about a quarter.  Tensors are any objects with data_ptr(), dtype, shape and
 * stride(), is_contiguous() and numel() as torch's have them; nothing is kept
 * of them.  Built for CPython's stable ABI.
 */
#define Py_LIMITED_API 0x030C0000
#include <Python.h>

#include "../../include/llm_b200.h"

enum { T_INT8 = 10, T_E4M3 = 11, T_INT32 = 20 };  /* and LLMB_F32, LLMB_F16, LLMB_BF16; below 0: none of them */

static PyObject *s_types, *s_refuse, *s_check;  /* dtype -> code; raise for arguments; raise for a status */
static PyObject *n_data_ptr, *n_dtype, *n_shape, *n_stride, *n_contiguous, *n_numel, *n_element_size;

static PyObject *method(PyObject *o, PyObject *name) {
    PyObject *args[1] = {o};
    return PyObject_VectorcallMethod(name, args, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
}

static int refuse(PyObject *msg) {  /* takes the message; always -1, with the exception set */
    if (msg) {
        PyObject *r = PyObject_CallFunctionObjArgs(s_refuse, msg, NULL);
        Py_XDECREF(r);
        Py_DECREF(msg);
        if (r) PyErr_SetString(PyExc_RuntimeError, "llm: an argument was not refused");
    }
    return -1;
}

static int address(PyObject *t, void **p) {
    PyObject *r = method(t, n_data_ptr);
    if (!r) return -1;
    *p = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    return PyErr_Occurred() ? -1 : 0;
}

static int type_of(PyObject *t, long *code) {
    PyObject *d = PyObject_GetAttr(t, n_dtype), *c = d ? PyObject_GetItem(s_types, d) : NULL;
    Py_XDECREF(d);
    if (!c) return -1;
    *code = PyLong_AsLong(c);
    Py_DECREF(c);
    return PyErr_Occurred() ? -1 : 0;
}

/* Up to 3 integers of a sequence; *n is its length. */
static int integers(PyObject *seq, int64_t *v, int *n) {
    PyObject *t = seq ? PySequence_Tuple(seq) : NULL;
    Py_XDECREF(seq);
    if (!t) return -1;
    *n = (int)PyTuple_Size(t);
    for (int i = 0; i < *n && i < 3; i++) v[i] = PyLong_AsLongLong(PyTuple_GetItem(t, i));
    Py_DECREF(t);
    return PyErr_Occurred() ? -1 : 0;
}

static int shape_of(PyObject *t, int64_t *v, int *n) { return integers(PyObject_GetAttr(t, n_shape), v, n); }
static int stride_of(PyObject *t, int64_t *v, int *n) { return integers(method(t, n_stride), v, n); }

static int whole(PyObject *t, PyObject *name, int64_t *v) {  /* an integer or truth value that a method returns */
    PyObject *r = method(t, name);
    if (!r) return -1;
    *v = PyLong_AsLongLong(r);
    Py_DECREF(r);
    return PyErr_Occurred() ? -1 : 0;
}

/* A contiguous tensor of n elements of that type (None: NULL). */
static int flat(PyObject *t, long type, int64_t n, const char *what, void **p) {
    long code;
    int64_t have, dense;
    *p = NULL;
    if (t == Py_None) return 0;
    if (type_of(t, &code) || whole(t, n_numel, &have) || whole(t, n_contiguous, &dense)) return -1;
    if (code != type || have != n || !dense)
        return refuse(PyUnicode_FromFormat("%s must be a contiguous %s tensor of %lld elements", what,
                                           type == T_INT32 ? "int32" : "float32", (long long)n));
    return address(t, p);
}

/* Rows [rows, heads, hd] of a type of rows: their address, type and distance. */
static int rows_of(PyObject *t, int64_t rows, int64_t heads, int64_t hd, const char *what, void **p, long *type,
                   int64_t *stride) {
    int64_t shape[3] = {0}, s[3] = {0};
    int n, m;
    if (type_of(t, type) || shape_of(t, shape, &n) || stride_of(t, s, &m)) return -1;
    if (*type < LLMB_F32 || *type > LLMB_BF16)
        return refuse(PyUnicode_FromFormat("%s must be float32, float16 or bfloat16", what));
    if (n != 3 || m != 3 || shape[0] != rows || shape[1] != heads || shape[2] != hd)
        return refuse(PyUnicode_FromFormat("%s must have shape (%lld, %lld, %lld)", what, (long long)rows, (long long)heads,
                                           (long long)hd));
    if (s[2] != 1 || (s[1] != hd && heads != 1))
        return refuse(PyUnicode_FromFormat("%s must be contiguous within a row", what));
    *stride = rows > 1 || s[0] > heads * hd ? s[0] : heads * hd;
    return address(t, p);
}

static PyObject *done(int rc) {
    if (rc == LLMB_OK) Py_RETURN_NONE;
    PyObject *c = PyLong_FromLong(rc), *r = c ? PyObject_CallFunctionObjArgs(s_check, c, NULL) : NULL;
    Py_XDECREF(c);
    return r;
}

static int number(PyObject *o, int64_t *v) {
    *v = PyLong_AsLongLong(o);
    return *v == -1 && PyErr_Occurred() ? -1 : 0;
}

static int handle(PyObject *o, void **p) {
    *p = PyLong_AsVoidPtr(o);
    return PyErr_Occurred() ? -1 : 0;
}

static int count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return 0;
    PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
    return -1;
}

/* (read, cache, batch, rows, kv_heads, head_dim, k, v, stream) */
static PyObject *call_rows(PyObject *self, PyObject *const *a, Py_ssize_t na) {
    void *cache, *batch, *stream, *k = NULL, *v = NULL;
    int64_t read, rows, heads, hd, stride = 0, other = 0;
    long type = 0, type2 = 0;
    int rc;
    (void)self;
    if (count(na, 9) || number(a[0], &read) || handle(a[1], &cache) || handle(a[2], &batch) || number(a[3], &rows) ||
        number(a[4], &heads) || number(a[5], &hd) || handle(a[8], &stream))
        return NULL;
    const int has_k = a[6] != Py_None, has_v = a[7] != Py_None;
    if (!has_k && !has_v) return refuse(PyUnicode_FromString("neither k nor v")), NULL;
    if (!read && !(has_k && has_v)) return refuse(PyUnicode_FromString("append needs k and v")), NULL;
    if (has_k && rows_of(a[6], rows, heads, hd, "k", &k, &type, &stride)) return NULL;
    if (has_v && rows_of(a[7], rows, heads, hd, "v", &v, has_k ? &type2 : &type, has_k ? &other : &stride)) return NULL;
    if (has_k && has_v && (type != type2 || stride != other))
        return refuse(PyUnicode_FromString("k and v must have one type and stride")), NULL;
    PyThreadState *st = PyEval_SaveThread();
    rc = read ? llmb_kv8_read(cache, batch, k, v, (int)type, stride, stream)
              : llmb_kv8_append(cache, batch, k, v, (int)type, stride, stream);
    PyEval_RestoreThread(st);
    return done(rc);
}

/* (cache, batch, rows, head_dim, q, out, scale, window, workspace, stream) */
static PyObject *call_attention(PyObject *self, PyObject *const *a, Py_ssize_t na) {
    void *cache, *batch, *stream, *q, *out, *work = NULL;
    int64_t rows, hd, window, shape[3] = {0}, qs, os, bytes = 0, each = 0, dense = 1;
    long type, type2;
    int n, rc;
    (void)self;
    if (count(na, 10) || handle(a[0], &cache) || handle(a[1], &batch) || number(a[2], &rows) || number(a[3], &hd) ||
        number(a[7], &window) || handle(a[9], &stream))
        return NULL;
    const double scale = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred() || shape_of(a[4], shape, &n)) return NULL;
    if (n != 3) return refuse(PyUnicode_FromString("q must be [rows, heads, head_dim]")), NULL;
    if (rows_of(a[4], rows, shape[1], hd, "q", &q, &type, &qs) || rows_of(a[5], rows, shape[1], hd, "out", &out, &type2, &os))
        return NULL;
    if (type != type2) return refuse(PyUnicode_FromString("q and out must have one type")), NULL;
    if (a[8] != Py_None) {
        if (whole(a[8], n_contiguous, &dense) || whole(a[8], n_numel, &bytes) || whole(a[8], n_element_size, &each) ||
            address(a[8], &work))
            return NULL;
        if (!dense) return refuse(PyUnicode_FromString("workspace must be contiguous")), NULL;
        bytes *= each;
    }
    if (window < INT32_MIN || window > INT32_MAX || shape[1] > INT32_MAX)
        return refuse(PyUnicode_FromString("window or heads out of range")), NULL;
    PyThreadState *st = PyEval_SaveThread();
    rc = llmb_kv8_attention(cache, batch, q, qs, out, os, (int)type, (int)shape[1], (float)scale, (int)window, work, bytes,
                            stream);
    PyEval_RestoreThread(st);
    return done(rc);
}

/* A [rows, columns] tensor's columns. */
static int columns(PyObject *t, int64_t rows, const char *what, int64_t *n) {
    int64_t shape[3] = {0};
    int dims;
    if (shape_of(t, shape, &dims)) return -1;
    if (dims != 2 || shape[0] != rows || shape[1] > INT32_MAX)
        return refuse(PyUnicode_FromFormat("%s must have two dimensions and a row for each row of logits", what));
    *n = shape[1];
    return 0;
}

/* (logits, out, tokens, history, history_lens, prompt_lens, penalties, bias_ids, bias_values, bias_starts, mask, stream) */
static PyObject *call_logits(PyObject *self, PyObject *const *a, Py_ssize_t na) {
    llmb_logits_ctl c = {0};
    void *logits, *out = NULL, *tokens, *stream, *p[7];
    int64_t shape[3] = {0}, s[3] = {0}, shape2[3] = {0}, s2[3] = {0}, hist = 0, bias = 0, words = 0;
    long type, type2;
    int n, m, n2, m2, rc;
    (void)self;
    if (count(na, 12) || handle(a[11], &stream) || type_of(a[0], &type) || shape_of(a[0], shape, &n) ||
        stride_of(a[0], s, &m) || address(a[0], &logits))
        return NULL;
    if (n != 2 || m != 2 || shape[0] > INT32_MAX || shape[1] > INT32_MAX)
        return refuse(PyUnicode_FromString("logits must be [rows, vocab]")), NULL;
    const int64_t rows = shape[0], vocab = shape[1];
    if (type < LLMB_F32 || type > LLMB_BF16 || (s[1] != 1 && vocab != 1))
        return refuse(PyUnicode_FromString("logits must be float32, float16 or bfloat16, and contiguous within a row")), NULL;
    if (a[1] != Py_None) {
        if (type_of(a[1], &type2) || shape_of(a[1], shape2, &n2) || stride_of(a[1], s2, &m2) || address(a[1], &out)) return NULL;
        if (type2 != type || n2 != 2 || m2 != 2 || shape2[0] != rows || shape2[1] != vocab || (s2[1] != 1 && vocab != 1))
            return refuse(PyUnicode_FromString("out must have the type and shape of logits and be contiguous within a row")), NULL;
    }
    if (a[3] == Py_None && (a[4] != Py_None || a[5] != Py_None))
        return refuse(PyUnicode_FromString("lengths without a history")), NULL;
    if (a[7] == Py_None && (a[8] != Py_None || a[9] != Py_None))
        return refuse(PyUnicode_FromString("biases without bias_ids")), NULL;
    if (a[7] != Py_None && a[8] == Py_None) return refuse(PyUnicode_FromString("bias_ids without bias_values")), NULL;
    if ((a[3] != Py_None && columns(a[3], rows, "history", &hist)) || (a[10] != Py_None && columns(a[10], rows, "mask", &words)) ||
        (a[7] != Py_None && whole(a[7], n_numel, &bias)))
        return NULL;
    if (bias > INT32_MAX) return refuse(PyUnicode_FromString("too many biases")), NULL;
    if (flat(a[2], T_INT32, rows, "tokens", &tokens) || flat(a[3], T_INT32, rows * hist, "history", &p[0]) ||
        flat(a[4], T_INT32, rows, "history_lens", &p[1]) || flat(a[5], T_INT32, rows, "prompt_lens", &p[2]) ||
        flat(a[6], LLMB_F32, 3 * rows, "penalties", &p[3]) || flat(a[7], T_INT32, bias, "bias_ids", &p[4]) ||
        flat(a[8], LLMB_F32, bias, "bias_values", &p[5]) || flat(a[9], T_INT32, rows + 1, "bias_starts", &p[6]) ||
        flat(a[10], T_INT32, rows * words, "mask", (void **)&c.mask))
        return NULL;
    if (hist > 0) c.history = p[0], c.history_lens = p[1], c.prompt_lens = p[2], c.history_stride = (int32_t)hist;
    c.penalties = p[3];
    if (bias > 0) c.bias_ids = p[4], c.bias_values = p[5], c.bias_starts = p[6], c.n_bias = (int32_t)bias;
    c.mask_stride = (int32_t)words;
    /* (one row, or no out: any distance does) */
    const int64_t stride = rows > 1 || s[0] > vocab ? s[0] : vocab, stride2 = rows > 1 || s2[0] > vocab ? s2[0] : vocab;
    PyThreadState *st = PyEval_SaveThread();
    rc = llmb_logits_control(logits, stride, (int)type, (int)rows, (int)vocab, &c, out, stride2, tokens, stream);
    PyEval_RestoreThread(st);
    return done(rc);
}

/* (types, refuse, check): what the calls use. */
static PyObject *call_setup(PyObject *self, PyObject *const *a, Py_ssize_t na) {
    (void)self;
    if (count(na, 3)) return NULL;
    PyObject **to[3] = {&s_types, &s_refuse, &s_check};
    for (int i = 0; i < 3; i++) {
        PyObject *old = *to[i];
        *to[i] = Py_NewRef(a[i]);
        Py_XDECREF(old);
    }
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"setup", (PyCFunction)(void (*)(void))call_setup, METH_FASTCALL, NULL},
    {"rows", (PyCFunction)(void (*)(void))call_rows, METH_FASTCALL, NULL},
    {"attention", (PyCFunction)(void (*)(void))call_attention, METH_FASTCALL, NULL},
    {"logits", (PyCFunction)(void (*)(void))call_logits, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__native(void) {
    n_data_ptr = PyUnicode_InternFromString("data_ptr"), n_dtype = PyUnicode_InternFromString("dtype");
    n_shape = PyUnicode_InternFromString("shape"), n_stride = PyUnicode_InternFromString("stride");
    n_contiguous = PyUnicode_InternFromString("is_contiguous"), n_numel = PyUnicode_InternFromString("numel");
    n_element_size = PyUnicode_InternFromString("element_size");
    if (!n_data_ptr || !n_dtype || !n_shape || !n_stride || !n_contiguous || !n_numel || !n_element_size) return NULL;
    return PyModule_Create(&module);
}

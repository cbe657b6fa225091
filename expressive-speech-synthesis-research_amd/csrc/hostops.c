/* The issuing side of the paged-decoding operators in C: what ops.page_plan, ops.page_write and ops.paged_attention do between their
 * Python call and the C ABI, for the calls that are plainly in order.  A decoder step issues three of them per block, and in Python the
 * look at the tensors costs 4 to 5 us a call beside a launch of 3 (one short request's attention: 9.4 us in Python, see ops.py).
 *
 * Every function returns True if it has issued the launch, and False, with nothing done and no error set, if anything at all is out of the
 * ordinary: a type, shape, stride or device that is not what the operator takes, or an error of the C ABI.  The caller then takes
 * the Python path, whose checks say what is wrong.  So there is one place for messages, and this file only has to accept nothing
 * that ops.py would refuse.
 *
 * Only Python's own C API is used: tensors are read through their Python attributes, so that nothing here depends on torch's ABI. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>
#include <stdint.h>

#include "../../include/estts.h"

static struct {
    int (*plan)(const estts_page_plan_args*, void*);
    int (*write)(const estts_page_write_args*, void*);
    int (*attention)(const estts_paged_attention_args*, void*);
    int64_t (*plan_ws)(int32_t, int32_t);
    int64_t (*attention_ws)(int32_t, int32_t, int32_t, int32_t, int32_t);
    PyObject *scratch, *get_device, *get_stream, *i32, *types[3];     /* types: float32, bfloat16, float16 (ESTTS_KV_*) */
} host;
static PyObject *s_shape, *s_stride, *s_dtype, *s_get_device, *s_data_ptr;

/* 1 and *out, or 0 (no error left set) */
static int as_int(PyObject* o, int64_t* out) {
    if (!o) { PyErr_Clear(); return 0; }
    *out = PyLong_CheckExact(o) ? PyLong_AsLongLong(o) : -1;
    const int ok = PyLong_CheckExact(o) && !(*out == -1 && PyErr_Occurred());
    if (!ok) PyErr_Clear();
    return ok;
}

static int call_int(PyObject* t, PyObject* name, int64_t* out) {
    PyObject* o = PyObject_CallMethodNoArgs(t, name);
    const int ok = as_int(o, out);
    Py_XDECREF(o);
    return ok;
}

/* entries of a tuple of at most 4 integers: their number, or -1 */
static int tuple_of(PyObject* o, int64_t* out) {
    int n = -1;
    if (!o) PyErr_Clear();
    else if (PyTuple_Check(o) && PyTuple_GET_SIZE(o) <= 4) {
        n = (int)PyTuple_GET_SIZE(o);
        for (int i = 0; i < n; ++i)
            if (!as_int(PyTuple_GET_ITEM(o, i), out + i)) { n = -1; break; }
    }
    Py_XDECREF(o);
    return n;
}

typedef struct { int nd; int64_t n[4], s[4]; void* at; } tensor;

/* a tensor of nd dimensions (0: any up to 4) and this type on this device */
static int look(PyObject* t, PyObject* dtype, int64_t device, int nd, tensor* out) {
    int64_t x;
    PyObject* kind = PyObject_GetAttr(t, s_dtype);
    if (!kind) { PyErr_Clear(); return 0; }
    Py_DECREF(kind);                                 /* (torch's types live as long as torch) */
    if (kind != dtype || !call_int(t, s_get_device, &x) || x != device) return 0;
    out->nd = tuple_of(PyObject_GetAttr(t, s_shape), out->n);
    if (out->nd < 0 || (nd && out->nd != nd) || tuple_of(PyObject_CallMethodNoArgs(t, s_stride), out->s) != out->nd) return 0;
    if (!call_int(t, s_data_ptr, &x)) return 0;
    out->at = (void*)(intptr_t)x;
    return 1;
}

static int contiguous(const tensor* t) {
    int64_t run = 1;
    for (int i = t->nd - 1; i >= 0; --i) {
        if (t->n[i] != 1 && t->s[i] != run) return 0;
        run *= t->n[i];
    }
    return 1;
}

static int64_t numel(const tensor* t) {
    int64_t n = 1;
    for (int i = 0; i < t->nd; ++i) n *= t->n[i];
    return n;
}

/* a contiguous int32 tensor of n elements in one dimension */
static int read_i32(PyObject* t, int64_t device, int64_t n, tensor* out) {
    return look(t, host.i32, device, 1, out) && out->n[0] == n && contiguous(out);
}

/* a [rows, >= width] view with contiguous rows; *ld its row stride */
static int read_rows(PyObject* t, int64_t device, int64_t rows, int64_t width, tensor* out, int64_t* ld) {
    if (!look(t, host.types[0], device, 2, out) || out->n[0] != rows || out->n[1] < width || (out->s[1] != 1 && out->n[1] > 1)) return 0;
    *ld = rows > 1 ? out->s[0] : width;
    return 1;
}

static int read_table(PyObject* t, int64_t device, int64_t B, tensor* out, int64_t* ld) {
    if (!look(t, host.i32, device, 2, out) || out->n[0] != B || out->n[1] < 1 || (out->s[1] != 1 && out->n[1] > 1)) return 0;
    *ld = B > 1 ? out->s[0] : out->n[1];
    return 1;
}

/* a pair of caches [n_pages, heads, page, depth] of one type and the same strides; *type: ESTTS_KV_* */
static int read_caches(PyObject* k, PyObject* v, int64_t device, tensor* ko, tensor* vo, int* type) {
    PyObject* kind = PyObject_GetAttr(k, s_dtype);
    if (!kind) { PyErr_Clear(); return 0; }
    Py_DECREF(kind);
    for (*type = 0; *type < 3 && host.types[*type] != kind; ++*type) {}
    if (*type == 3 || !look(k, kind, device, 4, ko) || !look(v, kind, device, 4, vo)) return 0;
    for (int i = 0; i < 4; ++i) {
        if (ko->n[i] != vo->n[i]) return 0;
        if (ko->n[i] == 1) ko->s[i] = vo->s[i] = i < 2 ? 0 : i == 2 ? ko->n[3] : 1;      /* (nothing is multiplied with it) */
        if (ko->s[i] != vo->s[i]) return 0;
    }
    return ko->s[3] == 1;
}

/* the device of `t` if it is the current one, else -1 */
static int64_t device_of(PyObject* t) {
    int64_t mine, current;
    if (!call_int(t, s_get_device, &mine) || mine < 0) return -1;
    PyObject* o = PyObject_CallNoArgs(host.get_device);
    const int ok = as_int(o, &current);
    Py_XDECREF(o);
    return ok && current == mine ? mine : -1;
}

static int stream_of(int64_t device, void** stream) {
    PyObject* d = PyLong_FromLongLong(device);
    PyObject* o = d ? PyObject_CallOneArg(host.get_stream, d) : NULL;
    int64_t x;
    const int ok = as_int(o, &x);
    Py_XDECREF(d);
    Py_XDECREF(o);
    *stream = ok ? (void*)(intptr_t)x : NULL;
    return ok;
}

/* scratch of one launch, as a tensor that the caller drops once the launch is issued; *at its address */
static PyObject* scratch_of(int64_t bytes, PyObject* like, void** at) {
    static PyObject* s_device;
    if (!s_device && !(s_device = PyUnicode_InternFromString("device"))) { PyErr_Clear(); return NULL; }
    PyObject *device = PyObject_GetAttr(like, s_device), *n = PyLong_FromLongLong(bytes), *t = NULL;
    int64_t x;
    if (device && n) t = PyObject_CallFunctionObjArgs(host.scratch, n, device, NULL);
    if (t && call_int(t, s_data_ptr, &x)) *at = (void*)(intptr_t)x;
    else { Py_XDECREF(t); t = NULL; }
    Py_XDECREF(device);
    Py_XDECREF(n);
    PyErr_Clear();
    return t;
}

static int fits32(int64_t x) { return x >= 0 && x <= INT32_MAX; }

/* page_write(k, v, k_cache, v_cache, slots) */
static PyObject* page_write(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    tensor k, v, kc, vc, slots;
    estts_page_write_args w;
    void* stream;
    if (n != 5) Py_RETURN_FALSE;
    const int64_t d = device_of(a[0]);
    if (d < 0 || !read_caches(a[2], a[3], d, &kc, &vc, &w.type) || !look(a[4], host.i32, d, 0, &slots) || !contiguous(&slots)) Py_RETURN_FALSE;
    const int64_t T = numel(&slots), width = kc.n[1] * kc.n[3];
    if ((kc.n[0] > 1 && !kc.s[0]) || (kc.n[1] > 1 && !kc.s[1]) || !kc.s[2] || !fits32(T) || !fits32(kc.n[0])) Py_RETURN_FALSE;
    if (!read_rows(a[0], d, T, width, &k, &w.ldk) || !read_rows(a[1], d, T, width, &v, &w.ldv) || !stream_of(d, &stream)) Py_RETURN_FALSE;
    w.k = k.at; w.v = v.at; w.k_cache = kc.at; w.v_cache = vc.at; w.slots = slots.at;
    w.s_page = kc.s[0]; w.s_head = kc.s[1]; w.s_row = kc.s[2];
    w.T = (int32_t)T; w.n_pages = (int32_t)kc.n[0]; w.heads = (int32_t)kc.n[1]; w.page = (int32_t)kc.n[2]; w.depth = (int32_t)kc.n[3];
    return PyBool_FromLong(host.write(&w, stream) == 0);
}

/* page_plan(lengths, new, block_table, free_pages, n_free, page, slots, positions, lengths_out, n_free_out, refused) */
static PyObject* page_plan(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    tensor lengths, news, table, pages, n_free, slots, positions, lengths_out, n_free_out, refused;
    estts_page_plan_args w;
    int64_t page;
    void* stream;
    if (n != 11) Py_RETURN_FALSE;
    const int64_t d = device_of(a[0]);
    if (d < 0 || !look(a[0], host.i32, d, 1, &lengths) || !contiguous(&lengths)) Py_RETURN_FALSE;
    const int64_t B = lengths.n[0];
    if (!read_i32(a[1], d, B, &news) || !read_table(a[2], d, B, &table, &w.ld_table) || !look(a[3], host.i32, d, 1, &pages) || !contiguous(&pages) ||
        !read_i32(a[4], d, 1, &n_free) || !as_int(a[5], &page) || !look(a[6], host.i32, d, 0, &slots) || !contiguous(&slots) ||
        slots.nd < 1 || slots.nd > 2 || (slots.nd == 2 && slots.n[0] != B) || !read_i32(a[8], d, B, &lengths_out) || !read_i32(a[9], d, 1, &n_free_out))
        Py_RETURN_FALSE;
    positions.at = refused.at = NULL;
    if (a[7] != Py_None && (!look(a[7], host.i32, d, slots.nd, &positions) || !contiguous(&positions) || positions.n[0] != slots.n[0] ||
                            (slots.nd == 2 && positions.n[1] != slots.n[1])))
        Py_RETURN_FALSE;
    if (a[10] != Py_None && !read_i32(a[10], d, 1, &refused)) Py_RETURN_FALSE;
    const int64_t T = numel(&slots);
    if (!fits32(B) || !fits32(T) || !fits32(table.n[1]) || !fits32(pages.n[0]) || !fits32(page) || !stream_of(d, &stream)) Py_RETURN_FALSE;
    w.lengths = lengths.at; w.n_new = news.at; w.block_table = table.at; w.free_pages = pages.at; w.n_free = n_free.at; w.slots = slots.at;
    w.positions = positions.at; w.lengths_out = lengths_out.at; w.n_free_out = n_free_out.at; w.refused = refused.at;
    w.B = (int32_t)B; w.P = (int32_t)table.n[1]; w.n_pages = (int32_t)pages.n[0]; w.page = (int32_t)page; w.T = (int32_t)T;
    w.R = slots.nd == 2 ? (int32_t)slots.n[1] : 0;
    w.ws_bytes = host.plan_ws(w.B, w.T);
    w.ws = NULL;
    PyObject* ws = NULL;
    void* at = NULL;
    if (w.ws_bytes > 0 && !(ws = scratch_of(w.ws_bytes, a[0], &at))) Py_RETURN_FALSE;
    w.ws = at;
    const int rc = host.plan(&w, stream);
    Py_XDECREF(ws);
    return PyBool_FromLong(rc == 0);
}

/* paged_attention(q, k_cache, v_cache, block_table, lengths, ctx, heads, key_mask, scale, max_len) */
static PyObject* paged_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    tensor q, kc, vc, table, lengths, ctx, mask;
    estts_paged_attention_args w;
    int64_t heads, max_len;
    void* stream;
    if (n != 10) Py_RETURN_FALSE;
    const int64_t d = device_of(a[0]);
    if (d < 0 || !read_caches(a[1], a[2], d, &kc, &vc, &w.type) || !look(a[4], host.i32, d, 1, &lengths) || !contiguous(&lengths)) Py_RETURN_FALSE;
    const int64_t B = lengths.n[0];
    if (!read_table(a[3], d, B, &table, &w.ld_table) || !as_int(a[6], &heads) || heads < 1 || kc.n[1] < 1 || heads % kc.n[1]) Py_RETURN_FALSE;
    const int64_t rows = table.n[1] * kc.n[2];
    if (a[9] == Py_None) max_len = rows;
    else if (!as_int(a[9], &max_len)) Py_RETURN_FALSE;
    if (max_len > rows) max_len = rows;
    if (max_len < 1 || !fits32(max_len) || !fits32(B) || !fits32(heads) || !fits32(table.n[1]) || !fits32(kc.n[0])) Py_RETURN_FALSE;
    if (!read_rows(a[0], d, B, heads * kc.n[3], &q, &w.ldq) || !read_rows(a[5], d, B, heads * kc.n[3], &ctx, &w.ldo)) Py_RETURN_FALSE;
    w.key_mask = NULL;
    w.mask_sb = w.mask_ss = 0;
    if (a[7] != Py_None) {
        if (!look(a[7], host.types[0], d, 2, &mask) || mask.n[0] != B || mask.n[1] < max_len) Py_RETURN_FALSE;
        w.key_mask = mask.at; w.mask_sb = mask.s[0]; w.mask_ss = mask.s[1];
    }
    if (a[8] == Py_None) w.scale = (float)(1.0 / sqrt((double)kc.n[3]));
    else if (PyFloat_CheckExact(a[8])) w.scale = (float)PyFloat_AS_DOUBLE(a[8]);
    else Py_RETURN_FALSE;
    if (!stream_of(d, &stream)) Py_RETURN_FALSE;
    w.q = q.at; w.k_cache = kc.at; w.v_cache = vc.at; w.block_table = table.at; w.lengths = lengths.at; w.ctx = ctx.at;
    w.s_page = kc.s[0]; w.s_head = kc.s[1]; w.s_row = kc.s[2];
    w.B = (int32_t)B; w.H = (int32_t)heads; w.n_pages = (int32_t)kc.n[0]; w.kv_heads = (int32_t)kc.n[1]; w.page = (int32_t)kc.n[2]; w.depth = (int32_t)kc.n[3];
    w.P = (int32_t)table.n[1]; w.max_len = (int32_t)max_len;
    w.ws_bytes = host.attention_ws(w.B, w.H, w.kv_heads, w.depth, w.max_len);
    PyObject* ws = NULL;
    void* at = NULL;
    if (w.ws_bytes > 0 && !(ws = scratch_of(w.ws_bytes, a[0], &at))) Py_RETURN_FALSE;
    w.ws = at;
    const int rc = host.attention(&w, stream);
    Py_XDECREF(ws);
    return PyBool_FromLong(rc == 0);
}

/* setup(addresses of estts_page_plan, _page_write, _paged_attention, _page_plan_ws_bytes, _paged_attention_ws_bytes, scratch(nbytes, device),
 *       current device (), raw stream (device), int32, float32, bfloat16, float16) */
static PyObject* setup(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    int64_t f[5];
    if (n != 12) { PyErr_SetString(PyExc_TypeError, "setup takes 12 arguments"); return NULL; }
    for (int i = 0; i < 5; ++i)
        if (!as_int(a[i], f + i) || !f[i]) { PyErr_SetString(PyExc_TypeError, "setup: addresses must be non-zero integers"); return NULL; }
    for (int i = 5; i < 12; ++i) Py_INCREF(a[i]);
    host.plan = (int (*)(const estts_page_plan_args*, void*))(intptr_t)f[0];
    host.write = (int (*)(const estts_page_write_args*, void*))(intptr_t)f[1];
    host.attention = (int (*)(const estts_paged_attention_args*, void*))(intptr_t)f[2];
    host.plan_ws = (int64_t (*)(int32_t, int32_t))(intptr_t)f[3];
    host.attention_ws = (int64_t (*)(int32_t, int32_t, int32_t, int32_t, int32_t))(intptr_t)f[4];
    host.scratch = a[5]; host.get_device = a[6]; host.get_stream = a[7]; host.i32 = a[8];
    for (int i = 0; i < 3; ++i) host.types[i] = a[9 + i];
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, NULL},
                                {"page_plan", (PyCFunction)(void (*)(void))page_plan, METH_FASTCALL, NULL},
                                {"page_write", (PyCFunction)(void (*)(void))page_write, METH_FASTCALL, NULL},
                                {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostops", NULL, -1, methods};

PyMODINIT_FUNC PyInit__hostops(void) {
    s_shape = PyUnicode_InternFromString("shape");
    s_stride = PyUnicode_InternFromString("stride");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_get_device = PyUnicode_InternFromString("get_device");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    if (!s_shape || !s_stride || !s_dtype || !s_get_device || !s_data_ptr) return NULL;
    return PyModule_Create(&module);
}

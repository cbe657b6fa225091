/* The issuing side of the paged-decoding operators in C++: what ops.page_plan, ops.page_write and ops.paged_attention do between their
 * Python call and the C ABI, for the calls that are plainly in order.  A decoder step issues three of them per block, and in Python the
 * look at the tensors costs 4 to 5 us a call beside a launch of 2.4 (one short request's attention: 9.4 us in Python; 5.9 where this file
 * asked for the tensors' attributes through Python; 4.1 here).
 *
 * Every function returns True if it has issued the launch, and False, with nothing done and no error set, if anything at all is out of the
 * ordinary: a type, shape, stride or device that is not what the operator takes, a tensor subclass, or a call that the C ABI refuses.  The
 * caller then takes the Python path, whose checks say what is wrong.  So there is one place for messages, and this file only has to
 * accept nothing that ops.py would refuse.  An error of the runtime (the C ABI's -2) raises instead: the launch may be under way all the
 * same (the error can be one that an earlier call of another library left behind), and a plan issued twice plans its rows twice. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>
#include <stdint.h>

#include <torch/csrc/autograd/python_variable.h>

#include "../../include/estts.h"

namespace {

struct {
    int (*plan)(const estts_page_plan_args*, void*);
    int (*write)(const estts_page_write_args*, void*);
    int (*attention)(const estts_paged_attention_args*, void*);
    int64_t (*plan_ws)(int32_t, int32_t);
    int64_t (*attention_ws)(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t);
    PyObject *alloc, *free, *get_device, *get_stream, *fail;
} host;

const at::ScalarType KV_TYPES[3] = {at::kFloat, at::kBFloat16, at::kHalf};      // ESTTS_KV_*

// true and *out, or false (no error left set)
bool as_int(PyObject* o, int64_t* out) {
    if (!o) { PyErr_Clear(); return false; }
    *out = PyLong_CheckExact(o) ? PyLong_AsLongLong(o) : -1;
    const bool ok = PyLong_CheckExact(o) && !(*out == -1 && PyErr_Occurred());
    if (!ok) PyErr_Clear();
    return ok;
}

// what a call gives as an integer; takes the reference
bool as_int_of(PyObject* o, int64_t* out) {
    const bool ok = as_int(o, out);
    Py_XDECREF(o);
    return ok;
}

struct Address {
    void* p;
    template <typename T> operator T*() const { return static_cast<T*>(p); }
};
struct tensor { int nd; int64_t n[4], s[4]; Address at; };

// a plain tensor (torch.Tensor or Parameter itself, dense) of nd dimensions (0: any up to 4) and this type on this device
bool look(PyObject* o, at::ScalarType type, int64_t device, int nd, tensor* out) {
    if (!THPVariable_CheckExact(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != at::kStrided || t.scalar_type() != type || !t.is_cuda() || t.get_device() != device) return false;
    const auto n = t.sizes(), s = t.strides();
    if (n.size() > 4 || (nd && (int)n.size() != nd)) return false;
    out->nd = (int)n.size();
    for (int i = 0; i < out->nd; ++i) { out->n[i] = n[i]; out->s[i] = s[i]; }
    out->at = {t.data_ptr()};
    return true;
}

bool contiguous(const tensor* t) {
    int64_t run = 1;
    for (int i = t->nd - 1; i >= 0; --i) {
        if (t->n[i] != 1 && t->s[i] != run) return false;
        run *= t->n[i];
    }
    return true;
}

int64_t numel(const tensor* t) {
    int64_t n = 1;
    for (int i = 0; i < t->nd; ++i) n *= t->n[i];
    return n;
}

// a contiguous int32 tensor of n elements in one dimension
bool read_i32(PyObject* t, int64_t device, int64_t n, tensor* out) {
    return look(t, at::kInt, device, 1, out) && out->n[0] == n && contiguous(out);
}

// a [rows, >= width] view with contiguous rows; *ld its row stride
bool read_rows(PyObject* t, int64_t device, int64_t rows, int64_t width, tensor* out, int64_t* ld) {
    if (!look(t, at::kFloat, device, 2, out) || out->n[0] != rows || out->n[1] < width || (out->s[1] != 1 && out->n[1] > 1)) return false;
    *ld = rows > 1 ? out->s[0] : width;
    return true;
}

bool read_table(PyObject* t, int64_t device, int64_t B, tensor* out, int64_t* ld) {
    if (!look(t, at::kInt, device, 2, out) || out->n[0] != B || out->n[1] < 1 || (out->s[1] != 1 && out->n[1] > 1)) return false;
    *ld = B > 1 ? out->s[0] : out->n[1];
    return true;
}

// a pair of caches [n_pages, heads, page, depth] of one type and the same strides; *type: ESTTS_KV_*
bool read_caches(PyObject* k, PyObject* v, int64_t device, tensor* ko, tensor* vo, int* type) {
    for (*type = 0; *type < 3 && !look(k, KV_TYPES[*type], device, 4, ko); ++*type) {}
    if (*type == 3 || !look(v, KV_TYPES[*type], device, 4, vo)) return false;
    for (int i = 0; i < 4; ++i) {
        if (ko->n[i] != vo->n[i]) return false;
        if (ko->n[i] == 1) ko->s[i] = vo->s[i] = i < 2 ? 0 : i == 2 ? ko->n[3] : 1;      // (nothing is multiplied with it)
        if (ko->s[i] != vo->s[i]) return false;
    }
    return ko->s[3] == 1;
}

// the device of `o` if it is the current one, else -1
int64_t device_of(PyObject* o) {
    int64_t current;
    if (!THPVariable_CheckExact(o) || !as_int_of(PyObject_CallNoArgs(host.get_device), &current)) return -1;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.defined() && t.is_cuda() && t.get_device() == current ? current : -1;
}

bool stream_of(int64_t device, void** stream) {
    PyObject* d = PyLong_FromLongLong(device);
    int64_t x = 0;
    const bool ok = as_int_of(d ? PyObject_CallOneArg(host.get_stream, d) : nullptr, &x);
    Py_XDECREF(d);
    *stream = reinterpret_cast<void*>(x);
    return ok;
}

// Scratch of one launch: from torch's allocator and back to it once the launch is issued, so that only later work of the same stream gets
// it again (under capture it comes out of the graph's own pool).
struct Scratch {
    PyObject* address = nullptr;
    void* at = nullptr;
    bool get(int64_t bytes, void* stream) {
        PyObject *n = PyLong_FromLongLong(bytes), *s = PyLong_FromLongLong(reinterpret_cast<intptr_t>(stream));
        if (n && s) address = PyObject_CallFunctionObjArgs(host.alloc, n, s, nullptr);
        Py_XDECREF(n);
        Py_XDECREF(s);
        int64_t x = 0;
        const bool ok = as_int(address, &x) && x;
        if (!ok) Py_CLEAR(address);
        PyErr_Clear();
        at = reinterpret_cast<void*>(x);
        return ok;
    }
    ~Scratch() {
        if (!address) return;
        Py_XDECREF(PyObject_CallOneArg(host.free, address));
        Py_DECREF(address);
        PyErr_Clear();
    }
};

// What became of a call.  (false is TURNED_DOWN)
enum { TURNED_DOWN = 0, ISSUED = 1, FAILED = 2 };

// Issues a launch without the interpreter's lock: it waits where the stream's queue is full.
template <typename A>
int launch(int (*f)(const A*, void*), const A& args, void* stream) {
    PyThreadState* state = PyEval_SaveThread();
    const int rc = f(&args, stream);
    PyEval_RestoreThread(state);
    return rc == 0 ? ISSUED : rc == -1 ? TURNED_DOWN : FAILED;
}

bool fits32(int64_t x) { return x >= 0 && x <= INT32_MAX; }

// page_write(k, v, k_cache, v_cache, slots)
int page_write(PyObject* const* a, Py_ssize_t n) {
    tensor k, v, kc, vc, slots;
    estts_page_write_args w;
    void* stream;
    if (n != 5) return false;
    const int64_t d = device_of(a[0]);
    if (d < 0 || !read_caches(a[2], a[3], d, &kc, &vc, &w.type) || !look(a[4], at::kInt, d, 0, &slots) || !contiguous(&slots)) return false;
    const int64_t T = numel(&slots), width = kc.n[1] * kc.n[3];
    if ((kc.n[0] > 1 && !kc.s[0]) || (kc.n[1] > 1 && !kc.s[1]) || !kc.s[2] || !fits32(T) || !fits32(kc.n[0]) || !fits32(kc.n[2])) return false;
    if (!read_rows(a[0], d, T, width, &k, &w.ldk) || !read_rows(a[1], d, T, width, &v, &w.ldv) || !stream_of(d, &stream)) return false;
    w.k = k.at; w.v = v.at; w.k_cache = kc.at; w.v_cache = vc.at; w.slots = slots.at;
    w.s_page = kc.s[0]; w.s_head = kc.s[1]; w.s_row = kc.s[2];
    w.T = (int32_t)T; w.n_pages = (int32_t)kc.n[0]; w.heads = (int32_t)kc.n[1]; w.page = (int32_t)kc.n[2]; w.depth = (int32_t)kc.n[3];
    return launch(host.write, w, stream);
}

// page_plan(lengths, new, block_table, free_pages, n_free, page, slots, positions, lengths_out, n_free_out, refused)
int page_plan(PyObject* const* a, Py_ssize_t n) {
    tensor lengths, news, table, pages, n_free, slots, positions, lengths_out, n_free_out, refused;
    estts_page_plan_args w;
    int64_t page;
    void* stream;
    if (n != 11) return false;
    const int64_t d = device_of(a[0]);
    if (d < 0 || !look(a[0], at::kInt, d, 1, &lengths) || !contiguous(&lengths)) return false;
    const int64_t B = lengths.n[0];
    if (!read_i32(a[1], d, B, &news) || !read_table(a[2], d, B, &table, &w.ld_table) || !look(a[3], at::kInt, d, 1, &pages) || !contiguous(&pages) ||
        !read_i32(a[4], d, 1, &n_free) || !as_int(a[5], &page) || !look(a[6], at::kInt, d, 0, &slots) || !contiguous(&slots) ||
        slots.nd < 1 || slots.nd > 2 || (slots.nd == 2 && slots.n[0] != B) || !read_i32(a[8], d, B, &lengths_out) || !read_i32(a[9], d, 1, &n_free_out))
        return false;
    positions.at = refused.at = {nullptr};
    if (a[7] != Py_None && (!look(a[7], at::kInt, d, slots.nd, &positions) || !contiguous(&positions) || positions.n[0] != slots.n[0] ||
                            (slots.nd == 2 && positions.n[1] != slots.n[1])))
        return false;
    if (a[10] != Py_None && !read_i32(a[10], d, 1, &refused)) return false;
    const int64_t T = numel(&slots);
    if (!fits32(B) || !fits32(T) || !fits32(table.n[1]) || !fits32(pages.n[0]) || !fits32(page) || !stream_of(d, &stream)) return false;
    w.lengths = lengths.at; w.n_new = news.at; w.block_table = table.at; w.free_pages = pages.at; w.n_free = n_free.at; w.slots = slots.at;
    w.positions = positions.at; w.lengths_out = lengths_out.at; w.n_free_out = n_free_out.at; w.refused = refused.at;
    w.B = (int32_t)B; w.P = (int32_t)table.n[1]; w.n_pages = (int32_t)pages.n[0]; w.page = (int32_t)page; w.T = (int32_t)T;
    w.R = slots.nd == 2 ? (int32_t)slots.n[1] : 0;
    w.ws_bytes = host.plan_ws(w.B, w.T);
    Scratch ws;
    if (w.ws_bytes > 0 && !ws.get(w.ws_bytes, stream)) return false;
    w.ws = static_cast<int32_t*>(ws.at);
    return launch(host.plan, w, stream);
}

// paged_attention(q, k_cache, v_cache, block_table, lengths, ctx, heads, key_mask, scale, max_len)
int paged_attention(PyObject* const* a, Py_ssize_t n) {
    tensor q, kc, vc, table, lengths, ctx, mask;
    estts_paged_attention_args w;
    int64_t heads, max_len;
    void* stream;
    if (n != 10) return false;
    const int64_t d = device_of(a[0]);
    if (d < 0 || !read_caches(a[1], a[2], d, &kc, &vc, &w.type) || !look(a[4], at::kInt, d, 1, &lengths) || !contiguous(&lengths)) return false;
    const int64_t B = lengths.n[0];
    if (!read_table(a[3], d, B, &table, &w.ld_table) || !as_int(a[6], &heads) || heads < 1 || kc.n[1] < 1 || heads % kc.n[1]) return false;
    const int64_t rows = table.n[1] * kc.n[2];
    if (a[9] == Py_None) max_len = rows;
    else if (!as_int(a[9], &max_len)) return false;
    if (max_len > rows) max_len = rows;
    if (max_len < 1 || !fits32(max_len) || !fits32(B) || !fits32(heads) || !fits32(table.n[1]) || !fits32(kc.n[0]) || !fits32(kc.n[2])) return false;
    if (!read_rows(a[0], d, B, heads * kc.n[3], &q, &w.ldq) || !read_rows(a[5], d, B, heads * kc.n[3], &ctx, &w.ldo)) return false;
    w.key_mask = nullptr;
    w.mask_sb = w.mask_ss = 0;
    if (a[7] != Py_None) {
        if (!look(a[7], at::kFloat, d, 2, &mask) || mask.n[0] != B || mask.n[1] < max_len) return false;
        w.key_mask = mask.at; w.mask_sb = mask.s[0]; w.mask_ss = mask.s[1];
    }
    if (a[8] == Py_None) w.scale = (float)(1.0 / sqrt((double)kc.n[3]));
    else if (PyFloat_CheckExact(a[8])) w.scale = (float)PyFloat_AS_DOUBLE(a[8]);
    else return false;
    if (!stream_of(d, &stream)) return false;
    w.q = q.at; w.k_cache = kc.at; w.v_cache = vc.at; w.block_table = table.at; w.lengths = lengths.at; w.ctx = ctx.at;
    w.s_page = kc.s[0]; w.s_head = kc.s[1]; w.s_row = kc.s[2];
    w.B = (int32_t)B; w.H = (int32_t)heads; w.n_pages = (int32_t)kc.n[0]; w.kv_heads = (int32_t)kc.n[1]; w.page = (int32_t)kc.n[2]; w.depth = (int32_t)kc.n[3];
    w.P = (int32_t)table.n[1]; w.max_len = (int32_t)max_len;
    w.ws_bytes = host.attention_ws(w.B, w.H, w.kv_heads, w.depth, w.max_len, w.type);
    Scratch ws;
    if (w.ws_bytes > 0 && !ws.get(w.ws_bytes, stream)) return false;
    w.ws = ws.at;
    return launch(host.attention, w, stream);
}

// (a tensor that only looks plain, of a function transform, say, throws when its address is asked for)
const char* const NAMES[3] = {"estts_page_plan", "estts_page_write", "estts_paged_attention"};

template <int (*F)(PyObject* const*, Py_ssize_t), int NAME>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int answer = TURNED_DOWN;
    try { answer = F(a, n); } catch (...) {}
    if (answer != FAILED) return PyBool_FromLong(answer);
    Py_XDECREF(PyObject_CallFunction(host.fail, "s", NAMES[NAME]));
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed", NAMES[NAME]);
    return nullptr;
}

// setup(addresses of estts_page_plan, _page_write, _paged_attention, _page_plan_ws_bytes, _paged_attention_ws_bytes, allocate (bytes, stream),
// free (address), current device (), raw stream (device), raise the library's last error of an entry point (its name))
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    int64_t f[5];
    if (n != 10) { PyErr_SetString(PyExc_TypeError, "setup takes 10 arguments"); return nullptr; }
    for (int i = 0; i < 5; ++i)
        if (!as_int(a[i], f + i) || !f[i]) { PyErr_SetString(PyExc_TypeError, "setup: addresses must be non-zero integers"); return nullptr; }
    for (int i = 5; i < 10; ++i) Py_INCREF(a[i]);
    host.plan = reinterpret_cast<decltype(host.plan)>(f[0]);
    host.write = reinterpret_cast<decltype(host.write)>(f[1]);
    host.attention = reinterpret_cast<decltype(host.attention)>(f[2]);
    host.plan_ws = reinterpret_cast<decltype(host.plan_ws)>(f[3]);
    host.attention_ws = reinterpret_cast<decltype(host.attention_ws)>(f[4]);
    host.alloc = a[5]; host.free = a[6]; host.get_device = a[7]; host.get_stream = a[8]; host.fail = a[9];
    Py_RETURN_NONE;
}

template <typename F>
PyMethodDef method(const char* name, F f) { return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}; }

PyMethodDef methods[] = {method("setup", setup), method("page_plan", entry<page_plan, 0>), method("page_write", entry<page_write, 1>),
                         method("paged_attention", entry<paged_attention, 2>), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch whose headers this was compiled against and the C ABI of estts.h, for the loader to compare
PyMODINIT_FUNC PyInit__hostops(void) {
    PyObject* m = PyModule_Create(&module);
    PyObject* built_for = m ? Py_BuildValue("(si)", ESTTS_TORCH, ESTTS_ABI_VERSION) : nullptr;
    if (built_for && PyModule_AddObject(m, "built_for", built_for) == 0) return m;
    Py_XDECREF(built_for);
    Py_XDECREF(m);
    return nullptr;
}

// The Python entries of the cache, attention and sampling calls in native code: checks of the tensors, allocation of results, the current stream and
// the call of the C ABI, which decides everything else.  A decode step makes one such call per layer and operator, and in Python the checks alone took
// longer than the kernels (kv_append of 64 tokens: 13 us of host time for 2.5 us on the GPU).  The module holds no state but the
// addresses of the C entries, which the mirror hands over (so the library is loaded once, by the mirror).
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <string>

#include "../../include/dsuf_qmm.h"

namespace {

decltype(&dsuf_kv_append) c_kv_append;
decltype(&dsuf_attn_decode) c_attn_decode;
decltype(&dsuf_attn_prompt) c_attn_prompt;
decltype(&dsuf_sample) c_sample;
decltype(&dsuf_last_error) c_last_error;
decltype(&dsuf_attn_workspace_bytes) c_workspace_bytes;
PyObject* g_error;      // the mirror's DsufError(code, message)

struct Refused {
    int code;
    std::string what;
};
[[noreturn]] void refuse(const std::string& what) { throw Refused{DSUF_E_BADARG, what}; }

struct Call {
    const char* who;
    dsuf_ctx* ctx;
    int device;

    Call(const char* w, PyObject* h, PyObject* dev) : who(w), ctx((dsuf_ctx*)PyLong_AsVoidPtr(h)), device((int)PyLong_AsLong(dev)) {}
    std::string name(const char* what) const { return std::string(who) + ": " + what; }

    const at::Tensor& tensor(PyObject* o, const char* what, at::ScalarType type) const {
        if (!THPVariable_Check(o)) refuse(name(what) + ": a tensor is wanted");
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.scalar_type() != type || t.get_device() != device || t.layout() != at::kStrided)
            refuse(name(what) + ": a " + at::toString(type) + " tensor on device " + std::to_string(device) + " is wanted");
        return t;
    }
    // A contiguous vector of n elements (-1: any number).
    const at::Tensor& vector(PyObject* o, const char* what, at::ScalarType type, int64_t n) const {
        const at::Tensor& t = tensor(o, what, type);
        if (t.dim() != 1 || (n >= 0 && t.size(0) != n) || (t.size(0) > 1 && t.stride(0) != 1))
            refuse(name(what) + ": a contiguous vector" + (n >= 0 ? " of " + std::to_string(n) : std::string()) + " is wanted");
        return t;
    }
    // A matrix [n][w] (-1: any) whose rows may lie apart; ld: its row stride (that of a single row says nothing and is taken as its length).
    const at::Tensor& rows(PyObject* o, const char* what, at::ScalarType type, int64_t n, int64_t w, int& ld) const {
        const at::Tensor& t = tensor(o, what, type);
        if (t.dim() != 2 || (n >= 0 && t.size(0) != n) || (w >= 0 && t.size(1) != w))
            refuse(name(what) + ": a matrix [" + std::to_string(n) + "][" + std::to_string(w) + "] is wanted (-1: any)");
        const int64_t m = t.size(0), width = t.size(1), far = m < 2 || width == 0 ? width : t.stride(0);
        if ((m > 0 && width > 1 && t.stride(1) != 1) || far < width || far > 0x7fffffff || m > 0x7fffffff)
            refuse(name(what) + ": rows must be contiguous, not overlapping and fewer than 2^31 elements apart");
        ld = (int)far;
        return t;
    }
    const at::Tensor& dense(PyObject* o, const char* what, at::ScalarType type, int64_t n, int64_t w) const {
        int ld;
        const at::Tensor& t = rows(o, what, type, n, w, ld);
        if (ld != t.size(1)) refuse(name(what) + ": must be contiguous");
        return t;
    }
    at::Tensor make(at::IntArrayRef size, at::ScalarType type) const {
        return at::empty(size, at::TensorOptions().dtype(type).device(device < 0 ? at::Device(at::kCPU) : at::Device(at::kCUDA, (c10::DeviceIndex)device)));
    }
    // The cache's description, as far as sizes are worked out from it here (the C entry checks the rest).
    const dsuf_kv_cache* cache(PyObject* o) const {
        const dsuf_kv_cache* k = (const dsuf_kv_cache*)PyLong_AsVoidPtr(o);
        if ((k->head_dim != 64 && k->head_dim != 128) || k->kv_heads < 1) refuse(name("the cache has heads of 64 or 128 columns, and at least one"));
        return k;
    }
    void* stream() const { return device < 0 ? nullptr : (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
    template <typename F>
    void run(F f) const {
        void* s = stream();
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = f(s);
        Py_END_ALLOW_THREADS
        if (rc) {
            char text[512] = "";
            c_last_error(ctx, text, sizeof(text));
            throw Refused{rc, text};
        }
    }
};

uint64_t at_(const at::Tensor& t) { return (uint64_t)t.data_ptr(); }
bool given(PyObject* o) { return o != Py_None; }
PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

long whole(const Call& c, PyObject* o, const char* what) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(c.name(what) + ": a whole number is wanted");
    }
    if (v < -0x7fffffffl || v > 0x7fffffffl) refuse(c.name(what) + ": out of range");
    return v;
}
bool yes(const Call& c, PyObject* o, const char* what) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        refuse(c.name(what) + ": true or false is wanted");
    }
    return v == 1;
}
float real(const Call& c, PyObject* o, const char* what) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(c.name(what) + ": a number is wanted");
    }
    return (float)v;
}

// (ctx, device, cache, k, v, pos, block_table, seq, rope, rope_half, q, q_out, k_out)
PyObject* kv_append(PyObject* const* a) {
    Call c("kv_append", a[0], a[1]);
    const dsuf_kv_cache* cache = c.cache(a[2]);
    const int64_t d = cache->head_dim, kv = cache->kv_heads * d;
    int ldk, ldv, ldq = 0, ldqo = 0, ldko = 0, heads = 0;
    const at::Tensor& k = c.rows(a[3], "k", at::kBFloat16, -1, kv, ldk);
    const int64_t n = k.size(0);
    const at::Tensor& v = c.rows(a[4], "v", at::kBFloat16, n, kv, ldv);
    const at::Tensor& pos = c.vector(a[5], "pos", at::kInt, n);
    const at::Tensor& table = c.dense(a[6], "block_table", at::kInt, -1, -1);
    const uint64_t seq = given(a[7]) ? at_(c.vector(a[7], "seq", at::kInt, n)) : 0;
    dsuf_rope r;
    if (given(a[8])) {
        if (!PyTuple_Check(a[8]) || PyTuple_GET_SIZE(a[8]) != 3) refuse("kv_append: rope is (cos, sin, off)");
        const at::Tensor& cos = c.dense(PyTuple_GET_ITEM(a[8], 0), "cos", at::kFloat, -1, -1);
        const at::Tensor& sin = c.dense(PyTuple_GET_ITEM(a[8], 1), "sin", at::kFloat, cos.size(0), cos.size(1));
        if (cos.size(1) > 4096) refuse("kv_append: cos and sin are wider than any head");
        r = {at_(cos), at_(sin), (int32_t)cos.size(0), (int32_t)cos.size(1) * 2, (int32_t)whole(c, PyTuple_GET_ITEM(a[8], 2), "off"), yes(c, a[9], "rope_half")};
    }
    uint64_t qp = 0, qo = 0, ko = 0;
    at::Tensor q_out;
    if (given(a[11]) && !given(a[10])) refuse("kv_append: q_out without q");
    if (given(a[10])) {
        const at::Tensor& q = c.rows(a[10], "q", at::kBFloat16, n, -1, ldq);
        const int64_t w = q.size(1);
        heads = (int)(w / d);
        if (heads == 0 || heads * d != w) refuse("kv_append: q's rows must hold whole heads");
        if (given(a[11])) q_out = c.rows(a[11], "q_out", at::kBFloat16, n, w, ldqo);
        else q_out = c.make({n, w}, at::kBFloat16), ldqo = (int)w;
        qp = at_(q), qo = at_(q_out);
    }
    if (given(a[12])) ko = at_(c.rows(a[12], "k_out", at::kBFloat16, n, kv, ldko));
    c.run([&](void* s) {
        return c_kv_append(c.ctx, s, cache, at_(k), ldk, at_(v), ldv, (int)n, at_(pos), seq, at_(table), (int)table.size(0), (int)table.size(1),
                           given(a[8]) ? &r : nullptr, qp, ldq, heads, qo, ldqo, ko, ldko);
    });
    if (given(a[11])) return Py_NewRef(a[11]);
    if (q_out.defined()) return wrap(q_out);
    Py_RETURN_NONE;
}

// out and, where wanted, lse: the caller's or new ones
struct Results {
    at::Tensor out, lse;
    int ldo;
    Results(const Call& c, PyObject* o, PyObject* l, bool want, int64_t n, int64_t width, int64_t heads) {
        if (given(o)) out = c.rows(o, "out", at::kBFloat16, n, width, ldo);
        else out = c.make({n, width}, at::kBFloat16), ldo = (int)width;
        if (given(l)) lse = c.dense(l, "lse", at::kFloat, n, heads);
        else if (want) lse = c.make({n, heads}, at::kFloat);
    }
    uint64_t lse_at() const { return lse.defined() ? at_(lse) : 0; }
    PyObject* answer(PyObject* o, PyObject* l, bool want) const {
        PyObject* first = given(o) ? Py_NewRef(o) : wrap(out);
        if (!want) return first;
        PyObject* second = given(l) ? Py_NewRef(l) : wrap(lse);
        PyObject* pair = PyTuple_Pack(2, first, second);
        Py_DECREF(first);
        Py_DECREF(second);
        return pair;
    }
};

// (ctx, device, cache, q, block_table, seq_lens, scale, window, out, lse, return_lse, workspace)
PyObject* attn_decode(PyObject* const* a) {
    Call c("attn_decode", a[0], a[1]);
    const dsuf_kv_cache* cache = c.cache(a[2]);
    const int64_t d = cache->head_dim;
    int ldq;
    const at::Tensor& q = c.rows(a[3], "q", at::kBFloat16, -1, -1, ldq);
    const int64_t b = q.size(0), width = q.size(1), heads = width / d;
    if (width == 0 || width % (d * cache->kv_heads)) refuse("attn_decode: q's rows must hold a multiple of kv_heads heads");
    const at::Tensor& table = c.dense(a[4], "block_table", at::kInt, b, -1);
    const at::Tensor& lens = c.vector(a[5], "seq_lens", at::kInt, b);
    const float scale = given(a[6]) ? real(c, a[6], "scale") : (float)(1.0 / std::sqrt((double)d));
    const long window = whole(c, a[7], "window");
    const bool want = yes(c, a[10], "return_lse");
    const at::Tensor& space = c.vector(a[11], "workspace", at::kByte, (int64_t)c_workspace_bytes(c.ctx));
    Results r(c, a[8], a[9], want, b, width, heads);
    c.run([&](void* s) {
        return c_attn_decode(c.ctx, s, cache, at_(q), ldq, (int)heads, (int)b, at_(table), (int)table.size(1), at_(lens), scale, (int)window, at_(r.out), r.ldo,
                             r.lse_at(), at_(space));
    });
    return r.answer(a[8], a[9], want);
}

// (ctx, device, q, k, v, cu_seqlens, head_dim, scale, window, out, lse, return_lse)
PyObject* attn_prompt(PyObject* const* a) {
    Call c("attn_prompt", a[0], a[1]);
    int ldq, ldk, ldv;
    const long d = whole(c, a[6], "head_dim");
    if (d != 64 && d != 128) refuse("attn_prompt: head_dim is 64 or 128");
    const at::Tensor& q = c.rows(a[2], "q", at::kBFloat16, -1, -1, ldq);
    const int64_t n = q.size(0), width = q.size(1), heads = width / d;
    const at::Tensor& k = c.rows(a[3], "k", at::kBFloat16, n, -1, ldk);
    const at::Tensor& v = c.rows(a[4], "v", at::kBFloat16, n, k.size(1), ldv);
    const int64_t kv_heads = k.size(1) / d;
    if (heads * d != width || kv_heads * d != k.size(1)) refuse("attn_prompt: rows hold whole heads");
    const at::Tensor& cu = c.vector(a[5], "cu_seqlens", at::kInt, -1);
    if (cu.size(0) < 1) refuse("attn_prompt: cu_seqlens holds at least one entry");
    const float scale = given(a[7]) ? real(c, a[7], "scale") : (float)(1.0 / std::sqrt((double)d));
    const long window = whole(c, a[8], "window");
    const bool want = yes(c, a[11], "return_lse");
    Results r(c, a[9], a[10], want, n, width, heads);
    c.run([&](void* s) {
        return c_attn_prompt(c.ctx, s, at_(q), ldq, at_(k), ldk, at_(v), ldv, (int)n, (int)heads, (int)kv_heads, (int)d, at_(cu), (int)cu.size(0) - 1, scale,
                             (int)window, at_(r.out), r.ldo, r.lse_at());
    });
    return r.answer(a[9], a[10], want);
}

// (ctx, device, logits, u, temperature, top_k, top_p, min_p, ids, logprobs, return_logprobs)
PyObject* sample(PyObject* const* a) {
    Call c("sample", a[0], a[1]);
    int ld;
    const at::Tensor& x = c.rows(a[2], "logits", at::kFloat, -1, -1, ld);
    const int64_t m = x.size(0);
    if (x.size(1) > 0x7fffffff) refuse("sample: logits are too wide");
    const at::Tensor& u = c.vector(a[3], "u", at::kFloat, m);
    auto column = [&](int i, const char* what, at::ScalarType type) { return given(a[i]) ? at_(c.vector(a[i], what, type, m)) : 0; };
    const uint64_t temperature = column(4, "temperature", at::kFloat), top_k = column(5, "top_k", at::kInt), top_p = column(6, "top_p", at::kFloat),
                   min_p = column(7, "min_p", at::kFloat);
    const bool want = yes(c, a[10], "return_logprobs");
    at::Tensor ids = given(a[8]) ? c.vector(a[8], "ids", at::kInt, m) : c.make({m}, at::kInt), lp;
    if (given(a[9])) lp = c.vector(a[9], "logprobs", at::kFloat, m);
    else if (want) lp = c.make({m}, at::kFloat);
    c.run([&](void* s) {
        return c_sample(c.ctx, s, at_(x), ld, (int)m, (int)x.size(1), temperature, top_k, top_p, min_p, at_(u), at_(ids), lp.defined() ? at_(lp) : 0);
    });
    PyObject* first = given(a[8]) ? Py_NewRef(a[8]) : wrap(ids);
    if (!want) return first;
    PyObject* second = given(a[9]) ? Py_NewRef(a[9]) : wrap(lp);
    PyObject* pair = PyTuple_Pack(2, first, second);
    Py_DECREF(first);
    Py_DECREF(second);
    return pair;
}

// Every entry takes a fixed number of positional arguments; no C++ exception leaves it.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments wanted, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused& r) {
        PyObject* e = PyObject_CallFunction(g_error, "is", r.code, r.what.c_str());
        if (e) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown exception");
    }
    return nullptr;
}

// bind(error class, addresses of kv_append, attn_decode, attn_prompt, sample, last_error, workspace_bytes)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long p[6];
    PyObject* error;
    if (!PyArg_ParseTuple(args, "OKKKKKK", &error, &p[0], &p[1], &p[2], &p[3], &p[4], &p[5])) return nullptr;
    Py_XSETREF(g_error, Py_NewRef(error));
    c_kv_append = (decltype(c_kv_append))p[0];
    c_attn_decode = (decltype(c_attn_decode))p[1];
    c_attn_prompt = (decltype(c_attn_prompt))p[2];
    c_sample = (decltype(c_sample))p[3];
    c_last_error = (decltype(c_last_error))p[4];
    c_workspace_bytes = (decltype(c_workspace_bytes))p[5];
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"kv_append", (PyCFunction)(void (*)())entry<kv_append, 13>, METH_FASTCALL, nullptr},
                         {"attn_decode", (PyCFunction)(void (*)())entry<attn_decode, 12>, METH_FASTCALL, nullptr},
                         {"attn_prompt", (PyCFunction)(void (*)())entry<attn_prompt, 12>, METH_FASTCALL, nullptr},
                         {"sample", (PyCFunction)(void (*)())entry<sample, 11>, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "dsuf_hostcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dsuf_hostcall() { return PyModule_Create(&module_def); }

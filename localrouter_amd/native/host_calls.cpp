// The host side of the calls of localrouter_amd/cache.py and of ops.attention_window: torch tensors checked and unpacked, then the
// entry point of liblr_attn.so, whose addresses bind() is given. A call's ~14 tensors cost ~0.1 us each attribute that Python reads
// of them, 3 to 7 us a call; here the checks take well below 1 us, and a call little more than its launch (back to back: append of 32
// tokens 12.0 -> 4.2 us, one token's attention 10.9 -> 8.8, its kernel's time, one page's copy 7.0 -> 3.8, a row move 8.0 -> 4.0).
// Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <sstream>
#include <string>

#include "../../include/lr_cache.h"

namespace {

PyObject* lr_error = nullptr;
decltype(&lr_cache_append_bf16) f_append = nullptr;
decltype(&lr_cache_attention_bf16) f_attention = nullptr;
decltype(&lr_cache_attention_ws_bytes) f_attention_ws = nullptr;
decltype(&lr_cache_copy_pages) f_copy = nullptr;
decltype(&lr_cache_move_rows) f_move = nullptr;
decltype(&lr_attention_window_bf16) f_window = nullptr;
decltype(&lr_attention_window_ws_bytes) f_window_ws = nullptr;

struct Raised {};   // a Python error is set

[[noreturn]] void refuse(const std::string& message) {
    PyErr_SetString(PyExc_ValueError, message.c_str());
    throw Raised{};
}
std::string describe(PyObject* o) {
    if (!THPVariable_Check(o)) return Py_TYPE(o)->tp_name;
    const at::Tensor& t = THPVariable_Unpack(o);
    std::ostringstream s;
    s << t.scalar_type() << " " << t.sizes() << " / " << t.strides() << " on " << t.device();
    return s.str();
}
[[noreturn]] void refuse(const char* name, const std::string& want, PyObject* a, PyObject* b = nullptr) {
    refuse(std::string(name) + ": expected " + want + " on the current device, got " + describe(a) + (b ? ", " + describe(b) : ""));
}

bool none(PyObject* o) { return o == Py_None; }
int64_t integer(PyObject* o, const char* name) {
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) {
        if (PyErr_ExceptionMatches(PyExc_OverflowError)) {
            PyErr_Clear();
            refuse(std::string(name) + ": a 32-bit number expected");
        }
        throw Raised{};
    }
    return x;
}
int int32(PyObject* o, const char* name) {
    const int64_t x = integer(o, name);
    if (x < INT_MIN || x > INT_MAX) refuse(std::string(name) + ": a 32-bit number expected");
    return (int)x;
}
// a count that None or more than `most` makes `most` (below 1: as it is, for the entry point to refuse)
int at_most(PyObject* o, const char* name, int64_t most) {
    return (int)(none(o) ? most : std::max<int64_t>(-1, std::min(integer(o, name), most)));
}
float number(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw Raised{};
    return (float)x;
}

struct Where {
    int dev;
    void* stream;
    Where(PyObject* d, PyObject* s) : dev((int)integer(d, "device")), stream(PyLong_AsVoidPtr(s)) {
        if (!stream && PyErr_Occurred()) throw Raised{};
    }
    bool holds(const at::Tensor& t, at::ScalarType type) const {
        return t.scalar_type() == type && t.is_cuda() && t.get_device() == dev;
    }
};
const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(name, "a tensor", o);
    return THPVariable_Unpack(o);
}
int64_t size0(PyObject* o, const char* name) {
    const at::Tensor& t = tensor(o, name);
    if (t.dim() < 1) refuse(name, "a tensor with dimensions", o);
    return t.size(0);
}

// bf16 rows [>= n, heads, 128] with contiguous heads
struct Rows {
    void* p = nullptr;
    int64_t rs = 0;
    Rows() = default;
    Rows(PyObject* o, const char* name, const Where& w, int64_t n, int64_t heads) {
        const at::Tensor& t = tensor(o, name);
        if (t.dim() != 3 || t.size(0) < n || t.size(1) != heads || t.size(2) != 128 || t.stride(2) != 1 ||
            (t.stride(1) != 128 && heads != 1) || !w.holds(t, at::kBFloat16))
            refuse(name, "bf16 [" + std::to_string(n) + ", " + std::to_string(heads) + ", 128] with contiguous heads", o);
        p = t.data_ptr();
        rs = t.size(0) > 1 ? t.stride(0) : heads * 128;
    }
};

// a contiguous vector of n elements at least
void* vector(PyObject* o, const char* name, const Where& w, int64_t n, at::ScalarType type, const char* what) {
    const at::Tensor& t = tensor(o, name);
    if (t.dim() != 1 || t.size(0) < n || !t.is_contiguous() || !w.holds(t, type))
        refuse(name, std::string("contiguous ") + what + " [" + std::to_string(n) + "]", o);
    return t.data_ptr();
}
const int* ints(PyObject* o, const char* name, const Where& w, int64_t n) {
    return static_cast<const int*>(vector(o, name, w, n, at::kInt, "int32"));
}

// bf16 [[layers,] n_pages, page_size, heads, 128] of keys and values
struct Pool {
    void *k, *v;
    int64_t ls = 0, ps, rs, hs;
    int layers = 1, n_pages, page_size, heads;
    Pool(PyObject* ko, PyObject* vo, const Where& w, bool with_layers) {
        const at::Tensor &kt = tensor(ko, "k_pages"), &vt = tensor(vo, "v_pages");
        const int64_t n = kt.dim();
        if (vt.sizes() != kt.sizes() || vt.strides() != kt.strides() || (n != 4 && !(with_layers && n == 5)) ||
            kt.size(n - 1) != 128 || kt.stride(n - 1) != 1 || !w.holds(kt, at::kBFloat16) || !w.holds(vt, at::kBFloat16))
            refuse("k_pages, v_pages", std::string("bf16 [n_pages, page_size, heads, 128]") + (with_layers ? " or [layers, ...]" : "") +
                   " of the same shape and strides", ko, vo);
        const auto s = kt.sizes().slice(n - 4), st = kt.strides().slice(n - 4);
        for (int i = 0; i < 3; ++i)
            if (s[i] > INT_MAX) refuse("k_pages: too large");
        n_pages = (int)s[0]; page_size = (int)s[1]; heads = (int)s[2];
        ps = st[0]; rs = st[1]; hs = st[2];
        // (a dimension of one element has whatever stride its view left: taken as packed)
        if (heads == 1) hs = 128;
        if (page_size == 1) rs = (heads - 1) * hs + 128;
        if (n_pages == 1) ps = (page_size - 1) * rs + (heads - 1) * hs + 128;
        if (n == 5) {
            if (kt.size(0) > INT_MAX) refuse("k_pages: too large");
            layers = (int)kt.size(0);
            ls = layers > 1 ? kt.stride(0) : 0;
        }
        k = kt.data_ptr();
        v = vt.data_ptr();
    }
};

struct Table {
    const int* p;
    int64_t rs;
    int pages;
    Table(PyObject* o, const Where& w, int64_t B) {
        const at::Tensor& t = tensor(o, "page_table");
        if (t.dim() != 2 || t.size(0) < B || t.size(1) > INT_MAX || (t.stride(1) != 1 && t.size(1) != 1) || !w.holds(t, at::kInt))
            refuse("page_table", "int32 [" + std::to_string(B) + ", pages] with contiguous rows", o);
        p = static_cast<const int*>(t.data_ptr());
        pages = (int)t.size(1);
        rs = t.size(0) > 1 ? t.stride(0) : pages;
    }
};

// The rotation tables of append: rows of at least the columns that rot dims take (its own view's: a row's stride may be another
// tensor's).
struct Rotation {
    int kind = LR_TABLE_NONE, rot = 0, rows = 0;
    const at::Tensor *a = nullptr, *b = nullptr;
    Rotation() = default;
    Rotation(PyObject* k, PyObject* ao, PyObject* bo, PyObject* r) : kind(int32(k, "table_kind")), rot(int32(r, "rot")) {
        if (kind == LR_TABLE_NONE) return;
        const int64_t dims = rot == 0 ? 128 : rot;
        const int64_t columns = kind == LR_TABLE_COSSIN_F32 ? dims / 2
                                : kind == LR_TABLE_MAT2_BF16 || kind == LR_TABLE_MAT2_F32 ? 2 * dims : 0;   // (others: no kind)
        a = &checked(ao, columns);
        rows = (int)a->size(0);
        if (!none(bo)) b = &checked(bo, columns);
    }
    const at::Tensor& checked(PyObject* o, int64_t columns) const {
        const at::Tensor& t = tensor(o, "table");
        if (t.dim() != 2 || t.stride(1) != 1 || t.size(0) > INT_MAX) refuse("table", "contiguous rows", o);
        if (t.size(1) < columns)
            refuse("table: rows of " + std::to_string(t.size(1)) + " columns, rot " + std::to_string(rot) + " needs " +
                   std::to_string(columns));
        return t;
    }
    // on the device, of the kind's type
    void at(const Where& w, PyObject* ao, PyObject* bo) const {
        const at::ScalarType type = kind == LR_TABLE_MAT2_BF16 ? at::kBFloat16 : at::kFloat;
        if (a && !w.holds(*a, type)) refuse("table", kind == LR_TABLE_MAT2_BF16 ? "bf16 rows" : "fp32 rows", ao);
        if (b && (b->sizes() != a->sizes() || b->strides() != a->strides() || !w.holds(*b, type)))
            refuse("table", "two tensors of the same type, shape and strides", ao, bo);
    }
};

// The given workspace, or one allocated on torch's current stream when `need` is not 0.
struct Workspace {
    void* p = nullptr;
    size_t bytes = 0;
    at::Tensor own;
    Workspace(PyObject* o, const Where& w, size_t need, const at::Tensor& like) {
        if (!none(o)) {
            const at::Tensor& t = tensor(o, "workspace");
            bytes = t.nbytes();
            if (bytes < need || !t.is_contiguous() || !t.is_cuda() || t.get_device() != w.dev)
                refuse("workspace: " + std::to_string(need) + " contiguous bytes on the current device needed");
            p = t.data_ptr();
        } else if (need) {
            own = at::empty({(int64_t)need}, like.options().dtype(at::kByte));
            p = own.data_ptr();
            bytes = need;
        }
    }
};

// out, or a new one
PyObject* rows_like(PyObject* o, int64_t n, int64_t heads, const at::Tensor& like) {
    if (none(o)) {
        PyObject* t = THPVariable_Wrap(at::empty({n, heads, 128}, like.options()));
        if (!t) throw Raised{};
        return t;
    }
    Py_INCREF(o);
    return o;
}
struct Held {   // a reference until it is returned
    PyObject* o;
    ~Held() { Py_XDECREF(o); }
    PyObject* release() { PyObject* x = o; o = nullptr; return x; }
};

template <class F>
void call(const char* name, F&& f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    if (rc == 0) return;
    if (PyObject* e = PyObject_CallFunction(lr_error, "si", name, rc)) {
        PyErr_SetObject(lr_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

// (device, stream, q, k, v, k_pages, v_pages, page_table, starts, lens, q_out, q_norm, k_norm, kind, table_a, table_b, positions,
// pairing, rot, eps)
PyObject* append(PyObject* const* a) {
    const Where w(a[0], a[1]);
    const int64_t T = size0(a[3], "k"), B = size0(a[9], "lens");
    const Rotation tab = T > 0 ? Rotation(a[13], a[14], a[15], a[18]) : Rotation();
    const Pool pool(a[5], a[6], w, false);
    const Rows k(a[3], "k", w, T, pool.heads), v(a[4], "v", w, T, pool.heads);
    Rows q, out;
    Held held{nullptr};
    int64_t H = 0;
    if (!none(a[2])) {
        const at::Tensor& qt = tensor(a[2], "q");
        H = qt.dim() == 3 ? qt.size(1) : 0;
        q = Rows(a[2], "q", w, T, H);
        held.o = rows_like(a[10], T, H, qt);
        out = Rows(held.o, "q_out", w, T, H);
        if (qt.size(0) != T) refuse("append: q, k and v of different lengths");
    }
    if (size0(a[4], "v") != T) refuse("append: q, k and v of different lengths");
    if (B > INT_MAX || T > INT_MAX) refuse("append: too many tokens");
    if (T > 0) {
        const float *qw = nullptr, *kw = nullptr;
        if (!none(a[11])) qw = static_cast<const float*>(vector(a[11], "q_norm", w, 128, at::kFloat, "fp32"));
        if (!none(a[12])) kw = static_cast<const float*>(vector(a[12], "k_norm", w, 128, at::kFloat, "fp32"));
        tab.at(w, a[14], a[15]);
        const Table table(a[7], w, B);
        const int *starts = ints(a[8], "starts", w, B + 1), *lens = ints(a[9], "lens", w, B);
        const int* pos = none(a[16]) ? nullptr : ints(a[16], "positions", w, T);
        const int pairing = int32(a[17], "pairing");
        const float eps = number(a[19]);
        const void *ta = tab.a ? tab.a->data_ptr() : nullptr, *tb = tab.b ? tab.b->data_ptr() : nullptr;
        const int64_t stride = tab.a ? tab.a->stride(0) : 0;
        call("lr_cache_append_bf16", [&] {
            return f_append(q.p, k.p, v.p, q.rs, k.rs, v.rs, out.p, out.rs, pool.k, pool.v, pool.ps, pool.rs, pool.hs, pool.n_pages,
                            pool.page_size, table.p, table.rs, table.pages, starts, lens, pos, (int)B, (int)T, (int)H, pool.heads, qw,
                            kw, tab.kind, ta, tb, stride, tab.rows, pairing, tab.rot, eps, static_cast<lr_stream_t>(w.stream));
        });
    }
    if (held.o) return held.release();
    Py_RETURN_NONE;
}

// (device, stream, q, k_pages, v_pages, page_table, starts, lens, out, max_rows, max_keys, tree, window, sinks, scale, workspace)
PyObject* attention(PyObject* const* a) {
    const Where w(a[0], a[1]);
    const at::Tensor& qt = tensor(a[2], "q");
    const int64_t T = size0(a[2], "q"), H = qt.dim() == 3 ? qt.size(1) : 0, B = size0(a[7], "lens");
    const Rows q(a[2], "q", w, T, H);
    const Pool pool(a[3], a[4], w, false);
    Held held{rows_like(a[8], T, H, qt)};
    const Rows out(held.o, "out", w, T, H);
    if (B > INT_MAX || T > INT_MAX || H > INT_MAX) refuse("attention: too many tokens");
    if (T == 0) return held.release();
    const Table table(a[5], w, B);
    const int64_t most = std::min<int64_t>((int64_t)table.pages * pool.page_size, INT_MAX);
    int max_rows = at_most(a[9], "max_rows", T), max_keys = at_most(a[10], "max_keys", most);
    const uint64_t* tree = nullptr;
    int words = 0;
    if (!none(a[11])) {
        const at::Tensor& t = tensor(a[11], "tree");
        if (t.dim() != 2 || t.size(0) < T || t.size(1) > INT_MAX || !t.is_contiguous() || !w.holds(t, at::kLong))
            refuse("tree", "contiguous int64 [" + std::to_string(T) + ", words]", a[11]);
        words = (int)t.size(1);
        tree = static_cast<const uint64_t*>(t.data_ptr());
    }
    const int window = int32(a[12], "window"), sinks = int32(a[13], "sinks");
    const float scale = number(a[14]);
    const int *starts = ints(a[6], "starts", w, B + 1), *lens = ints(a[7], "lens", w, B);
    auto ws_need = [&](int rows, int keys) {
        return f_attention_ws((int)B, (int)T, rows, keys, (int)H, pool.heads, pool.page_size, window, sinks);
    };
    size_t need = ws_need(max_rows, max_keys);
    // A workspace for a max_rows or max_keys beyond this call's tokens or its table may be smaller (more rows fill the GPU without
    // parts): the launch is then sized as the workspace was.
    if (!none(a[15]) && tensor(a[15], "workspace").nbytes() < need) {
        constexpr int64_t MOST = 1 << 30;   // (the most rows and positions of a call)
        const int rows = none(a[9]) ? max_rows : at_most(a[9], "max_rows", MOST / std::max<int64_t>(1, H / std::max(1, pool.heads)));
        const int keys = none(a[10]) ? max_keys : at_most(a[10], "max_keys", MOST);
        const size_t given = ws_need(rows, keys);
        if (given <= tensor(a[15], "workspace").nbytes()) {
            need = given;
            max_rows = rows;
            max_keys = keys;
        }
    }
    const Workspace ws(a[15], w, need, qt);
    call("lr_cache_attention_bf16", [&] {
        return f_attention(q.p, q.rs, out.p, out.rs, pool.k, pool.v, pool.ps, pool.rs, pool.hs, pool.n_pages, pool.page_size, table.p,
                           table.rs, table.pages, starts, lens, (int)B, (int)T, max_rows, max_keys, (int)H, pool.heads, tree, words,
                           window, sinks, scale, ws.p, ws.bytes, static_cast<lr_stream_t>(w.stream));
    });
    return held.release();
}

// (device, stream, k_pages, v_pages, src, dst)
PyObject* copy_pages(PyObject* const* a) {
    const Where w(a[0], a[1]);
    const Pool pool(a[2], a[3], w, true);
    const int64_t n = size0(a[4], "src");
    if (size0(a[5], "dst") != n) refuse("copy_pages: src and dst of different lengths");
    if (n > INT_MAX) refuse("copy_pages: too many pages");
    if (n > 0) {
        const int *src = ints(a[4], "src", w, n), *dst = ints(a[5], "dst", w, n);
        call("lr_cache_copy_pages", [&] {
            return f_copy(pool.k, pool.v, pool.layers, pool.ls, pool.ps, pool.rs, pool.hs, pool.n_pages, pool.page_size, pool.heads, src,
                          dst, (int)n, static_cast<lr_stream_t>(w.stream));
        });
    }
    Py_RETURN_NONE;
}

// (device, stream, k_pages, v_pages, page_table, starts, src, dst, max_rows)
PyObject* move_rows(PyObject* const* a) {
    const Where w(a[0], a[1]);
    const Pool pool(a[2], a[3], w, true);
    const int64_t n = size0(a[6], "src"), B = size0(a[5], "starts") - 1;
    if (size0(a[7], "dst") != n) refuse("move_rows: src and dst of different lengths");
    if (n > INT_MAX || B > INT_MAX) refuse("move_rows: too many rows");
    if (n > 0) {
        const Table table(a[4], w, B);
        const int *starts = ints(a[5], "starts", w, B + 1), *src = ints(a[6], "src", w, n), *dst = ints(a[7], "dst", w, n);
        const int max_rows = at_most(a[8], "max_rows", n);
        call("lr_cache_move_rows", [&] {
            return f_move(pool.k, pool.v, pool.layers, pool.ls, pool.ps, pool.rs, pool.hs, pool.n_pages, pool.page_size, pool.heads,
                          table.p, table.rs, table.pages, starts, src, dst, (int)B, (int)n, max_rows,
                          static_cast<lr_stream_t>(w.stream));
        });
    }
    Py_RETURN_NONE;
}

// (device, stream, q, k, v, out, window, sinks, frame, p0, scale, workspace)
PyObject* attention_window(PyObject* const* a) {
    const Where w(a[0], a[1]);
    const at::Tensor &qt = tensor(a[2], "q"), &kt = tensor(a[3], "k");
    const int64_t W = size0(a[2], "q"), H = qt.dim() == 3 ? qt.size(1) : 0;
    const int64_t N = size0(a[3], "k"), HK = kt.dim() == 3 ? kt.size(1) : 0;
    const Rows q(a[2], "q", w, W, H), k(a[3], "k", w, N, HK), v(a[4], "v", w, N, HK);
    Held held{rows_like(a[5], W, H, qt)};
    const Rows out(held.o, "out", w, W, H);
    if (W > INT_MAX || N > INT_MAX || H > INT_MAX || HK > INT_MAX) refuse("attention_window: too many rows");
    if (W == 0) return held.release();
    const int window = int32(a[6], "window"), sinks = int32(a[7], "sinks"), frame = int32(a[8], "frame"), p0 = int32(a[9], "p0");
    const float scale = number(a[10]);
    const Workspace ws(a[11], w, f_window_ws((int)W, (int)H, (int)HK, (int)N, window, sinks, frame), qt);
    call("lr_attention_window_bf16", [&] {
        return f_window(q.p, k.p, v.p, out.p, p0, (int)W, (int)H, (int)HK, (int)N, window, sinks, frame, scale, q.rs, k.rs, v.rs, out.rs,
                        ws.p, ws.bytes, static_cast<lr_stream_t>(w.stream));
    });
    return held.release();
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* guarded(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != N || !lr_error) {
        PyErr_SetString(PyExc_TypeError, lr_error ? "wrong number of arguments" : "bind() first");
        return nullptr;
    }
    try {
        return F(a);
    } catch (const Raised&) {
    } catch (const std::exception& e) {   // (an allocation that torch could not make, for one)
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// bind(LrError, {name: address})
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 2 || !PyDict_Check(a[1])) {
        PyErr_SetString(PyExc_TypeError, "bind(error, addresses)");
        return nullptr;
    }
    auto get = [&](const char* name) -> void* {
        PyObject* o = PyDict_GetItemString(a[1], name);
        return o ? PyLong_AsVoidPtr(o) : nullptr;
    };
    auto take = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(get(name));
        return f != nullptr;
    };
    if (!take(f_append, "lr_cache_append_bf16") || !take(f_attention, "lr_cache_attention_bf16") ||
        !take(f_attention_ws, "lr_cache_attention_ws_bytes") || !take(f_copy, "lr_cache_copy_pages") ||
        !take(f_move, "lr_cache_move_rows") || !take(f_window, "lr_attention_window_bf16") ||
        !take(f_window_ws, "lr_attention_window_ws_bytes")) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: an address is missing");
        return nullptr;
    }
    Py_INCREF(a[0]);
    Py_XDECREF(lr_error);
    lr_error = a[0];
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", FAST(bind)},
                         {"append", FAST((&guarded<append, 20>))},
                         {"attention", FAST((&guarded<attention, 16>))},
                         {"copy_pages", FAST((&guarded<copy_pages, 6>))},
                         {"move_rows", FAST((&guarded<move_rows, 9>))},
                         {"attention_window", FAST((&guarded<attention_window, 12>))},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_calls() { return PyModule_Create(&module); }

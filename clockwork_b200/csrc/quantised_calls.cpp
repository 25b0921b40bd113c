// The common calls of the 8-bit cache's operators (ops/quantised.py) without the interpreter's share: checks, output tensor and arguments
// of a call in C++ over torch's own tensor objects, then the library's entry point.  A kernel of these takes 3 to 15 us, and a
// call through Python's checks, 60 look-ups of tensors' fields, 10 to 14.
//
// Whatever is not as it should be (a type, a shape, a device, an entry point that refuses) makes the function here return None
// without having launched anything (of a step or of portions at most what comes first, which is then made once more); the caller then takes Python's way through the same checks, which says what is wrong or has a kernel
// for it.  So every condition there is here too, and none of its words.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <exception>

namespace {

using at::Tensor;
typedef int (*Entry)(const char*);
Entry store_entry, read_entry, decode_entry, portions_entry;
typedef int (*PrefillEntry)(const void*, int, int, int, void*, const void*, const void*, const int*, const int*, const int*, const int*, const int*,
                            const int*, float*, float*, int*, int, int, int, int, int, int, int, float, int, int, int*, cudaStream_t);
PrefillEntry prefill_entry;  // (the packed form, which takes one query head to a tile as well)
PyTypeObject *e4m3_type, *plain_type;

struct Refused : std::exception {};
inline void need(bool ok) {
    if (!ok) throw Refused();
}

const Tensor& tensor(PyObject* o) {
    need(THPVariable_Check(o));
    return THPVariable_Unpack(o);
}
long long number(PyObject* o) {
    const long long x = PyLong_AsLongLong(o);
    need(x != -1 || !PyErr_Occurred());
    return x;
}
double real(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    need(x != -1.0 || !PyErr_Occurred());
    return x;
}
int truth(PyObject* o) {
    const int x = PyObject_IsTrue(o);
    need(x >= 0);
    return x;
}
long long window_of(PyObject* o) {
    if (o == Py_None) return 0;
    const long long x = number(o);
    need(x > 0);
    return x;
}

// The device that a call's first tensor is on, which must be the current one.
int cuda_device(const Tensor& t) {
    need(t.is_cuda() && t.get_device() == c10::cuda::current_device());
    return (int)t.get_device();
}
const Tensor& of_type(PyObject* o, at::ScalarType type, int64_t dim, int device) {
    const Tensor& t = tensor(o);
    need(t.scalar_type() == type && t.dim() == dim && t.is_contiguous() && t.is_cuda() && t.get_device() == device);
    return t;
}
const void* status_of(PyObject* o, int device) {
    const Tensor& t = tensor(o);
    need(t.scalar_type() == at::kInt && t.numel() >= 4 && t.is_cuda() && t.get_device() == device);
    return t.const_data_ptr();
}
int type_code(const Tensor& t) {
    need(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16);
    return t.scalar_type() == at::kBFloat16;
}

struct Pages {
    const void *k, *v, *k_exp, *v_exp;
    int64_t pages, page_size, nkv, hd;
};
Pages quantised_pages(PyObject* o, int device) {
    need(Py_TYPE(o) == e4m3_type);
    const Tensor &k = of_type(PyTuple_GET_ITEM(o, 0), at::kFloat8_e4m3fn, 4, device), &v = of_type(PyTuple_GET_ITEM(o, 1), at::kFloat8_e4m3fn, 4, device),
                 &ke = of_type(PyTuple_GET_ITEM(o, 2), at::kByte, 3, device), &ve = of_type(PyTuple_GET_ITEM(o, 3), at::kByte, 3, device);
    const Pages p = {k.const_data_ptr(), v.const_data_ptr(), ke.const_data_ptr(), ve.const_data_ptr(), k.size(0), k.size(1), k.size(2), k.size(3)};
    need(v.sizes() == k.sizes() && ve.sizes() == ke.sizes() && ke.size(0) == p.pages && ke.size(1) == p.nkv && ke.size(2) == p.page_size);
    need(p.pages * p.page_size < (1LL << 31) && ((uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0);
    return p;
}
Pages plain_pages(PyObject* o, at::ScalarType type, int device) {
    need(Py_TYPE(o) == plain_type);
    const Tensor &k = of_type(PyTuple_GET_ITEM(o, 0), type, 4, device), &v = of_type(PyTuple_GET_ITEM(o, 1), type, 4, device);
    need(v.sizes() == k.sizes());
    return {k.const_data_ptr(), v.const_data_ptr(), nullptr, nullptr, k.size(0), k.size(1), k.size(2), k.size(3)};
}

// The block of 8-byte words that an entry point reads.
struct Words {
    uint64_t w[40];
    int n = 0;
    Words& pointer(const void* p) {
        w[n++] = (uint64_t)p;
        return *this;
    }
    Words& whole(long long x) {
        w[n++] = (uint64_t)x;
        return *this;
    }
    Words& number(double x) {
        memcpy(&w[n++], &x, 8);
        return *this;
    }
    Words& stream() { return pointer(c10::cuda::getCurrentCUDAStream().stream()); }
    Words& pages(const Pages& p) { return pointer(p.k).pointer(p.v).pointer(p.k_exp).pointer(p.v_exp); }
    void call(Entry entry) {
        int result;
        Py_BEGIN_ALLOW_THREADS;
        result = entry((const char*)w);
        Py_END_ALLOW_THREADS;
        need(result == 0);
    }
};

// What norm_rotate_store and decode_step have in common.
struct Rows {
    const Tensor& qkv;
    int device;
    int64_t n, nh, nkv, hd, rot;
    Pages cache;
    const void *positions, *slots, *inv_freq = nullptr, *q_weight = nullptr, *k_weight = nullptr, *status;

    Rows(PyObject* rows, PyObject* at, PyObject* to, PyObject* freq, PyObject* pages, PyObject* heads, PyObject* kv_heads, PyObject* entries,
         PyObject* words, PyObject* wq, PyObject* wk)
        : qkv(tensor(rows)), device(cuda_device(qkv)), nh(number(heads)), nkv(number(kv_heads)), hd(number(entries)), rot(0) {
        type_code(qkv);
        need(nh > 0 && nkv > 0 && hd > 0 && hd <= 256 && nh < (1 << 20) && nkv < (1 << 20));
        need(qkv.dim() == 2 && qkv.is_contiguous() && qkv.size(1) == (nh + 2 * nkv) * hd);
        n = qkv.size(0);
        const Tensor &p = of_type(at, at::kInt, 1, device), &s = of_type(to, at::kInt, 1, device);
        need(p.size(0) == n && s.size(0) == n);
        positions = p.const_data_ptr();
        slots = s.const_data_ptr();
        cache = Py_TYPE(pages) == e4m3_type ? quantised_pages(pages, device) : plain_pages(pages, qkv.scalar_type(), device);
        need(cache.nkv == nkv && cache.hd == hd);
        if (freq != Py_None) {
            const Tensor& f = of_type(freq, at::kFloat, 1, device);
            rot = 2 * f.size(0);
            need(rot <= hd);
            if (rot > 0) inv_freq = f.const_data_ptr();
        }
        q_weight = weight(wq);
        k_weight = weight(wk);
        status = status_of(words, device);
    }
    const void* weight(PyObject* o) {
        if (o == Py_None) return nullptr;
        const Tensor& w = of_type(o, at::kFloat, 1, device);
        need(w.size(0) == hd);
        return w.const_data_ptr();
    }
};

// (pointers, the head size that it was made for, its device) of a DecodeWorkspace
struct Scratch {
    const void *floats, *words;
    Scratch(PyObject* o, int64_t hd, int device) {
        need(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4);
        floats = (const void*)number(PyTuple_GET_ITEM(o, 0));
        words = (const void*)number(PyTuple_GET_ITEM(o, 1));
        need(number(PyTuple_GET_ITEM(o, 2)) >= hd && number(PyTuple_GET_ITEM(o, 3)) == device);
    }
};

Tensor stored(const Rows& r, double eps, int early) {
    Tensor q = at::empty({r.n, r.nh * r.hd}, r.qkv.options());
    Words()
        .pointer(r.qkv.const_data_ptr()).pointer(q.const_data_ptr()).pointer(r.positions).pointer(r.slots).pointer(r.inv_freq)
        .pointer(r.q_weight).pointer(r.k_weight).pages(r.cache).pointer(r.status).stream()
        .whole(r.n).whole(r.nh).whole(r.nkv).whole(r.hd).whole(r.rot).whole(r.cache.page_size).whole(r.cache.pages)
        .whole(type_code(r.qkv)).whole(early).number(eps)
        .call(store_entry);
    return q;
}
// qkv, positions, slots, inv_freq, cache, heads, KV heads, entries, status, q_weight, k_weight, eps, early
PyObject* store(PyObject* const* a) {
    const Rows r(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10]);
    return THPVariable_Wrap(stored(r, real(a[11]), truth(a[12])));
}

// What attention of single tokens reads besides its queries and the cache.
struct Tokens {
    const Tensor &tables, &ctx;
    int64_t s, nh;
    double scale;
    const void* status;
    long long window, sms;
    Scratch scratch;
    Tokens(PyObject* table, PyObject* lens, PyObject* heads, PyObject* factor, PyObject* words, PyObject* seen, PyObject* room, PyObject* count,
           const Pages& cache, int device)
        : tables(of_type(table, at::kInt, 2, device)), ctx(of_type(lens, at::kInt, 1, device)), s(tables.size(0)), nh(number(heads)),
          scale(real(factor)), status(status_of(words, device)), window(window_of(seen)), sms(number(count)), scratch(room, cache.hd, device) {
        need(nh > 0 && nh < (1 << 20) && cache.nkv > 0 && nh % cache.nkv == 0 && cache.hd % 32 == 0 && cache.hd <= 256 && ctx.size(0) == s);
    }
    Tensor attended(const Tensor& q, const Pages& cache, int early) const {
        Tensor out = at::empty({s, nh * cache.hd}, q.options());
        Words()
            .pointer(q.const_data_ptr()).pointer(out.const_data_ptr()).pages(cache).pointer(tables.const_data_ptr()).pointer(ctx.const_data_ptr())
            .pointer(nullptr).pointer(scratch.floats).pointer(scratch.words).pointer(status).stream()
            .whole(s > 1 ? q.stride(0) : nh * cache.hd).whole(s).whole(nh).whole(cache.nkv).whole(cache.hd).whole(cache.page_size)
            .whole(tables.size(1)).whole(cache.pages).whole(window).whole(1).whole(sms).whole(early).number(scale)  // (early: 0, 1 or 2)
            .call(decode_entry);
        return out;
    }
};
// q, cache, block tables, ctx_lens, heads, scale, status, window, workspace, SMs, early
PyObject* decode(PyObject* const* a) {
    const Tensor& q = tensor(a[0]);
    const int device = cuda_device(q);
    const Pages cache = quantised_pages(a[1], device);
    const Tokens t(a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], cache, device);
    need(type_code(q) == 1 && q.dim() == 2 && q.size(0) == t.s && q.size(1) >= t.nh * cache.hd && q.stride(1) == 1);
    return THPVariable_Wrap(t.attended(q, cache, truth(a[10])));
}
// store's arguments, then block tables, ctx_lens, scale, window, workspace, SMs
PyObject* step(PyObject* const* a) {
    const Rows r(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10]);
    const double eps = real(a[11]);
    const int early = truth(a[12]);
    need(r.cache.k_exp != nullptr && type_code(r.qkv) == 1);
    const Tokens t(a[13], a[14], a[5], a[15], a[8], a[16], a[17], a[18], r.cache, r.device);
    need(t.s == r.n);
    // (what the attention could still refuse, sizes beyond its counters, is refused again by the caller's way, behind the same store)
    return THPVariable_Wrap(t.attended(stored(r, eps, early), r.cache, early ? 1 : 2));
}

// cache, block tables, ctx_lens, out_k, out_v, status, window, blocks
PyObject* read(PyObject* const* a) {
    need(Py_TYPE(a[0]) == e4m3_type);
    const int device = cuda_device(tensor(PyTuple_GET_ITEM(a[0], 0)));
    const Pages cache = quantised_pages(a[0], device);
    const Tensor &tables = of_type(a[1], at::kInt, 2, device), &ctx = of_type(a[2], at::kInt, 1, device);
    const at::ScalarType type = tensor(a[3]).scalar_type();
    const Tensor &k = of_type(a[3], type, 4, device), &v = of_type(a[4], type, 4, device);
    const int code = type_code(k);
    need(k.sizes() == v.sizes() && k.size(0) == cache.pages && k.size(1) == cache.page_size && k.size(2) == cache.nkv && k.size(3) == cache.hd);
    need(((uintptr_t)k.const_data_ptr() | (uintptr_t)v.const_data_ptr()) % 16 == 0 && cache.hd % 16 == 0 && ctx.size(0) == tables.size(0));
    Words()
        .pages(cache).pointer(k.const_data_ptr()).pointer(v.const_data_ptr()).pointer(tables.const_data_ptr()).pointer(ctx.const_data_ptr())
        .pointer(nullptr).pointer(status_of(a[5], device)).stream().whole(tables.size(0)).whole(cache.nkv).whole(cache.hd)
        .whole(cache.page_size).whole(tables.size(1)).whole(cache.pages).whole(window_of(a[6])).whole(1).whole(number(a[7])).whole(code)
        .call(read_entry);
    Py_RETURN_TRUE;
}

// q, cache, block tables, q_start, ctx_lens, plan, heads, scale, status, window, workspace, SMs, blocks, then for portions that are read
// back (or None): k pages, v pages, (part_o, part_ml, counters: addresses; or None)
// The plan's fields go by their places in ops/quantised.py's PortionPlan.
enum { Q_LENS, CTX_LENS, SHAPE, SHORT, LEAST_ROWS, MOST_ROWS, ITEMS, EACH, ITEM_SEQ, ITEM_Q0, ITEM_SPLIT, TOK_SEQ, POSITIONS, FIELDS };
PyObject* portions(PyObject* const* a) {
    const Tensor& q = tensor(a[0]);
    const int device = cuda_device(q);
    const Pages cache = quantised_pages(a[1], device);
    const Tensor &tables = of_type(a[2], at::kInt, 2, device), &starts = of_type(a[3], at::kInt, 1, device), &ctx = of_type(a[4], at::kInt, 1, device);
    PyObject* plan = a[5];
    need(PyTuple_Check(plan) && PyTuple_GET_SIZE(plan) == FIELDS);
    auto field = [&](int i) { return PyTuple_GET_ITEM(plan, i); };
    const int64_t nh = number(a[6]), s = tables.size(0), rows = q.size(0);
    const Tensor& tok_seq = of_type(field(TOK_SEQ), at::kInt, 1, device);
    need(PyTuple_Check(field(Q_LENS)) && PyTuple_GET_SIZE(field(Q_LENS)) == s && tok_seq.size(0) <= rows);
    PyObject* shape = field(SHAPE);
    need(PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) == 4 && number(PyTuple_GET_ITEM(shape, 0)) == nh && number(PyTuple_GET_ITEM(shape, 1)) == cache.nkv &&
         number(PyTuple_GET_ITEM(shape, 2)) == cache.hd && number(PyTuple_GET_ITEM(shape, 3)) == cache.page_size);
    const long long items = number(field(ITEMS)), least = number(field(LEAST_ROWS)), most = number(field(MOST_ROWS)), few = number(field(SHORT)),
                    each = number(field(EACH));
    need(type_code(q) == 1 && nh > 0 && nh < (1 << 20) && cache.nkv > 0 && nh % cache.nkv == 0 && (cache.hd == 64 || cache.hd == 128));
    need(q.dim() == 2 && q.size(1) >= nh * cache.hd && q.stride(1) == 1 && ctx.size(0) == s && starts.size(0) == s + 1);
    need(cache.page_size >= 8 && cache.page_size <= 128 && (cache.page_size & (cache.page_size - 1)) == 0);
    const double scale = real(a[7]);
    const void* status = status_of(a[8], device);
    const long long window = window_of(a[9]), sms = number(a[11]), blocks = number(a[12]);
    const int64_t q_stride = rows > 1 ? q.stride(0) : nh * cache.hd, unit = items > 0 ? 16 : few > 0 ? 4 : 1;
    need((uintptr_t)q.const_data_ptr() % unit == 0 && 2 * q.stride(0) % unit == 0);
    need(q.stride(0) < (1LL << 31) && rows < (1LL << 31) && window < (1LL << 31) && tables.size(1) < (1LL << 31));
    const void *floats = nullptr, *words = nullptr;
    if (few > 0) {
        const Scratch scratch(a[10], cache.hd, device);
        floats = scratch.floats;
        words = scratch.words;
    }
    Tensor out = at::empty({rows, nh * cache.hd}, q.options());
    if (items > 0) {
        const Tensor &k = of_type(a[13], at::kBFloat16, 4, device), &v = of_type(a[14], at::kBFloat16, 4, device);
        const Tensor &seq = of_type(field(ITEM_SEQ), at::kInt, 1, device), &q0 = of_type(field(ITEM_Q0), at::kInt, 1, device);
        need(k.sizes() == v.sizes() && k.size(0) == cache.pages && k.size(1) == cache.page_size && k.size(2) == cache.nkv && k.size(3) == cache.hd);
        need(seq.size(0) == items && q0.size(0) == items);
        const int* split = nullptr;
        const void* scratch[3] = {nullptr, nullptr, nullptr};
        if (field(ITEM_SPLIT) != Py_None) {
            const Tensor& cut = of_type(field(ITEM_SPLIT), at::kInt, 1, device);
            need(cut.size(0) == items && PyTuple_Check(a[15]) && PyTuple_GET_SIZE(a[15]) == 3);
            split = (const int*)cut.const_data_ptr();
            for (int i = 0; i < 3; ++i) scratch[i] = (const void*)number(PyTuple_GET_ITEM(a[15], i));
        }
        Words()
            .pages(cache).pointer(k.const_data_ptr()).pointer(v.const_data_ptr()).pointer(tables.const_data_ptr()).pointer(ctx.const_data_ptr())
            .pointer(starts.const_data_ptr()).pointer(status).stream().whole(s).whole(cache.nkv).whole(cache.hd).whole(cache.page_size)
            .whole(tables.size(1)).whole(cache.pages).whole(window).whole(most + 1 > least ? most + 1 : least).whole(blocks).whole(1)
            .call(read_entry);
        int result;
        Py_BEGIN_ALLOW_THREADS;
        result = prefill_entry(q.const_data_ptr(), (int)q.stride(0), (int)q.size(1), (int)rows, out.mutable_data_ptr(), k.const_data_ptr(), v.const_data_ptr(),
                               (const int*)tables.const_data_ptr(), (const int*)starts.const_data_ptr(), (const int*)ctx.const_data_ptr(),
                               (const int*)seq.const_data_ptr(), (const int*)q0.const_data_ptr(), split, (float*)scratch[0], (float*)scratch[1],
                               (int*)scratch[2], (int)items, (int)nh, (int)cache.nkv, (int)cache.hd, (int)cache.page_size, (int)tables.size(1),
                               (int)cache.pages, (float)scale, (int)window, (int)each, (int*)status, c10::cuda::getCurrentCUDAStream().stream());
        Py_END_ALLOW_THREADS;
        need(result == 0);
    }
    if (few > 0) {
        Words()
            .pointer(q.const_data_ptr()).pointer(out.const_data_ptr()).pages(cache).pointer(tables.const_data_ptr()).pointer(ctx.const_data_ptr())
            .pointer(starts.const_data_ptr()).pointer(floats).pointer(words).pointer(status).stream().whole(q_stride).whole(s)
            .whole(nh).whole(cache.nkv).whole(cache.hd).whole(cache.page_size).whole(tables.size(1)).whole(cache.pages).whole(window).whole(sms)
            .whole(few).whole(least).whole(most).number(scale)
            .call(portions_entry);
    }
    return THPVariable_Wrap(std::move(out));
}

template <PyObject* (*CALL)(PyObject* const*), int ARGUMENTS>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n == ARGUMENTS && store_entry != nullptr) return CALL(args);
    } catch (const std::exception&) {
    }
    PyErr_Clear();
    Py_RETURN_NONE;
}

// addresses of the entry points (store, read, decode, portions of few rows, packed prefill), E4M3Pages, PlainPages
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long s, r, d, w, t;
    PyObject *e, *p;
    if (!PyArg_ParseTuple(args, "KKKKKO!O!", &s, &r, &d, &w, &t, &PyType_Type, &e, &PyType_Type, &p)) return nullptr;
    Py_INCREF(e);
    Py_INCREF(p);
    store_entry = (Entry)s;
    read_entry = (Entry)r;
    decode_entry = (Entry)d;
    portions_entry = (Entry)w;
    prefill_entry = (PrefillEntry)t;
    e4m3_type = (PyTypeObject*)e;
    plain_type = (PyTypeObject*)p;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"store", (PyCFunction)(void*)guarded<store, 13>, METH_FASTCALL, nullptr},
                         {"step", (PyCFunction)(void*)guarded<step, 19>, METH_FASTCALL, nullptr},
                         {"decode", (PyCFunction)(void*)guarded<decode, 11>, METH_FASTCALL, nullptr},
                         {"portions", (PyCFunction)(void*)guarded<portions, 16>, METH_FASTCALL, nullptr},
                         {"read", (PyCFunction)(void*)guarded<read, 8>, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "quantised_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_quantised_calls() { return PyModule_Create(&module); }

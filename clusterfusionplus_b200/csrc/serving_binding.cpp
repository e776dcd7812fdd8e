// Python binding of the serving calls (clusterfusionplus_b200/serving.py).
//
// These calls run for a few microseconds on the GPU, and a decoding server makes several of them for each layer or token: through ctypes, with
// the checks and the allocation of the results in Python, a call took 13 to 20 us of the host.  Here the checks read the tensors directly
// and the results are allocated and cut by ATen.  The library itself stays free of torch: this module gets the addresses of its entry
// points from the Python side (bind), which has loaded it.  No C++ exception leaves a function: torch's own translation makes it a Python one
// (RuntimeError; torch.OutOfMemoryError where memory ran out).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>
#include <sstream>
#include <stdexcept>
#include <string>

#include "../../include/clusterfusion_b200.h"

namespace {

struct Entries {
    decltype(&cf_last_error) last_error;
    decltype(&cf_paged_kv_plan) plan;
    decltype(&cf_paged_kv_release) release;
    decltype(&cf_kv4_append) append;
    decltype(&cf_kv4_read) read;
    decltype(&cf_kv4_attention) attention;
    decltype(&cf_kv4_attention_workspace) workspace;
    decltype(&cf_token_logprobs) logprobs;
} cf;

template <class... A> [[noreturn]] void complain(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw std::runtime_error(s.str());
}

struct Shape {
    const at::Tensor& t;
};
std::ostream& operator<<(std::ostream& s, const Shape& v) { return s << v.t.sizes() << " with strides " << v.t.strides(); }

const char* type_name(at::ScalarType t) {
    switch (t) {
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kFloat: return "torch.float32";
        case at::kByte: return "torch.uint8";
        default: return c10::toString(t);
    }
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) complain(name, ": expected a torch.Tensor");
    return THPVariable_Unpack(o);
}

// a tensor on the current device (which the first tensor of a call asks for)
struct Call {
    int device = -1;
    const at::Tensor& on_device(PyObject* o, const char* name, int64_t dims) {
        const at::Tensor& t = tensor(o, name);
        if (!t.is_cuda()) complain(name, ": expected a CUDA tensor, got ", t.device());
        if (device < 0) device = c10::cuda::current_device();
        if (t.get_device() != device) complain(name, ": tensor is on ", t.device(), " but the current device is cuda:", device);
        if (t.dim() != dims) complain(name, ": expected ", dims, dims > 1 ? " dimensions" : " dimension", ", got shape ", t.sizes());
        return t;
    }
    const at::Tensor& ints(PyObject* o, const char* name, int64_t n = -1) {
        const at::Tensor& t = on_device(o, name, 1);
        if (t.scalar_type() != at::kInt) complain(name, ": expected dtype torch.int32, got ", type_name(t.scalar_type()));
        if (!t.is_contiguous()) complain(name, ": expected a contiguous tensor, got shape ", Shape{t});
        if (n >= 0 && t.numel() != n) complain(name, ": expected ", n, " entries, got ", t.numel());
        return t;
    }
    const at::Tensor& table(PyObject* o, int64_t batch, int64_t* width, int64_t* apart) {
        const at::Tensor& t = on_device(o, "block_table", 2);
        if (t.scalar_type() != at::kInt) complain("block_table: expected dtype torch.int32, got ", type_name(t.scalar_type()));
        *width = t.size(1);
        *apart = batch > 1 ? t.stride(0) : *width;
        if (t.size(0) != batch || (t.stride(1) != 1 && *width > 1) || *apart < *width)
            complain("block_table: expected [", batch, ", pages] rows of consecutive entries, got shape ", Shape{t});
        return t;
    }
    // elements from one entry of axis d to the next; where there is but one, its stride says nothing
    static int64_t apart(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
    // rows of 16-bit numbers whose last axis is contiguous and whose other strides are multiples of `step` elements
    const at::Tensor& rows(PyObject* o, const char* name, int64_t step) {
        const at::Tensor& t = on_device(o, name, 3);
        half(t.scalar_type(), name);
        if (t.stride(2) != 1 || apart(t, 0) % step || apart(t, 1) % step)
            complain(name, ": expected a contiguous last axis and strides in multiples of ", step, " elements, got shape ", Shape{t});
        return t;
    }
    static int half(at::ScalarType t, const char* name) {
        if (t != at::kHalf && t != at::kBFloat16) complain(name, ": expected dtype torch.float16 or torch.bfloat16, got ", type_name(t));
        return t == at::kHalf ? CF_DTYPE_FP16 : CF_DTYPE_BF16;
    }
    // a 4-bit cache of `heads` heads (any if negative)
    const at::Tensor& cache(PyObject* o, int64_t heads, int64_t head_dim) {
        const at::Tensor& t = on_device(o, "cache", 4);
        const int64_t width = 40 * ((head_dim + 31) / 32);
        if (t.scalar_type() != at::kByte || !t.is_contiguous() || t.size(3) != width || (heads >= 0 && t.size(1) != heads))
            complain("cache: expected contiguous uint8 [pages, ", heads >= 0 ? std::to_string(heads) : std::string("kv_heads"), ", page_size, ", width, "] for heads of ", head_dim,
                     " (see kv4_cache), got ", type_name(t.scalar_type()), " ", Shape{t});
        return t;
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }
};

int64_t number(PyObject* o, const char* name) {
    const int64_t v = PyLong_AsLongLong(o);  // takes __index__ too
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        complain(name, ": expected a whole number");
    }
    return v;
}

void check(int rc) {
    if (rc != 0) complain("clusterfusion_b200: ", cf.last_error(), " (code ", rc, ")");
}

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

template <int N> PyObject* tuple_of(at::Tensor (&t)[N]) {
    PyObject* r = PyTuple_New(N);
    for (int i = 0; r && i < N; ++i) {
        PyObject* o = wrap(std::move(t[i]));
        if (!o) Py_CLEAR(r);
        else PyTuple_SET_ITEM(r, i, o);
    }
    return r;
}

at::Tensor empty(at::IntArrayRef shape, const at::Tensor& like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }
at::Tensor piece(const at::Tensor& t, int64_t from, int64_t n) { return t.as_strided({n}, {1}, from); }

// results that no gradient flows through, made while other Python threads run: a launch may wait for room in the stream's queue
struct Aside {
    at::AutoDispatchBelowADInplaceOrView below;
    PyThreadState* state = PyEval_SaveThread();
    ~Aside() { PyEval_RestoreThread(state); }
};

template <class F> PyObject* guarded(const char* name, Py_ssize_t n, Py_ssize_t want, F f) {
    HANDLE_TH_ERRORS
    if (n != want) complain(name, ": ", want, " arguments, got ", n);
    return f();
    END_HANDLE_TH_ERRORS
}

// (cached_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens, max_rows)
PyObject* py_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("paged_kv_plan", n, 8, [&] {
        Call c;
        const at::Tensor& cached = c.ints(a[0], "cached_lens");
        const int64_t batch = cached.numel();
        const at::Tensor& fresh = c.ints(a[1], "new_lens", batch);
        int64_t width, apart;
        const at::Tensor& table = c.table(a[2], batch, &width, &apart);
        const at::Tensor &free_pages = c.ints(a[3], "free_pages"), &count = c.ints(a[4], "free_count", 1);
        const int64_t page = number(a[5], "page_size"), max_tokens = number(a[6], "max_tokens"), max_rows = number(a[7], "max_rows");
        if (max_tokens < 0 || max_rows < 0 || max_tokens > INT32_MAX || max_rows > INT32_MAX)
            complain("max_tokens ", max_tokens, " and max_rows ", max_rows, " must not be negative, nor 2^31 or more");
        at::Tensor r[8];
        {
            Aside aside;
            // one allocation, each piece 16-byte aligned (as the calls that read them ask): rows, slots, lengths, both indptr arrays, count, status
            auto after = [](int64_t at, int64_t n) { return at + (n + 3) / 4 * 4; };
            const int64_t slots = after(0, max_rows), lens = after(slots, max_tokens), qo = after(lens, batch), kv = after(qo, batch + 1), left = after(kv, batch + 1), status = after(left, 1);
            const at::Tensor buf = empty({status + 1}, cached, at::kInt), positions = empty({max_tokens}, cached, at::kLong);
            int* p = buf.data_ptr<int>();
            check(cf.plan(cached.data_ptr<int>(), fresh.data_ptr<int>(), batch, table.data_ptr<int>(), width, apart, free_pages.data_ptr<int>(), free_pages.numel(), count.data_ptr<int>(), p + left,
                          page, p + lens, p + qo, positions.data_ptr<int64_t>(), p + slots, max_tokens, p + kv, p, max_rows, p + status, c.stream()));
            r[0] = piece(buf, lens, batch), r[1] = piece(buf, qo, batch + 1), r[2] = positions, r[3] = piece(buf, slots, max_tokens), r[4] = piece(buf, kv, batch + 1);
            r[5] = piece(buf, 0, max_rows), r[6] = piece(buf, left, 1), r[7] = piece(buf, status, 1);
        }
        return tuple_of(r);
    });
}

// (finished, kv_lens, block_table, free_pages, free_count, page_size)
PyObject* py_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("paged_kv_release", n, 6, [&] {
        Call c;
        const at::Tensor& lens = c.ints(a[1], "kv_lens");
        const int64_t batch = lens.numel();
        const at::Tensor& finished = c.ints(a[0], "finished", batch);
        int64_t width, apart;
        const at::Tensor& table = c.table(a[2], batch, &width, &apart);
        const at::Tensor &free_pages = c.ints(a[3], "free_pages"), &count = c.ints(a[4], "free_count", 1);
        const int64_t page = number(a[5], "page_size");
        at::Tensor r[2];
        {
            Aside aside;
            const at::Tensor buf = empty({2}, lens, at::kInt);
            int* p = buf.data_ptr<int>();
            check(cf.release(finished.data_ptr<int>(), lens.data_ptr<int>(), batch, table.data_ptr<int>(), width, apart, free_pages.data_ptr<int>(), free_pages.numel(), count.data_ptr<int>(), p,
                             page, p + 1, c.stream()));
            r[0] = piece(buf, 0, 1), r[1] = piece(buf, 1, 1);
        }
        return tuple_of(r);
    });
}

// (key, value, slot_map, cache)
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("kv4_append", n, 4, [&]() -> PyObject* {
        Call c;
        const at::Tensor &key = c.rows(a[0], "key", 4), &value = c.rows(a[1], "value", 4);
        if (!value.sizes().equals(key.sizes()) || value.scalar_type() != key.scalar_type())
            complain("value: expected ", key.sizes(), " of ", type_name(key.scalar_type()), " like key, got ", value.sizes(), " of ", type_name(value.scalar_type()));
        const int64_t tokens = key.size(0), heads = key.size(1), dim = key.size(2);
        const at::Tensor& cache = c.cache(a[3], heads, dim);
        const at::Tensor& slots = c.ints(a[2], "slot_map", tokens);
        {
            Aside aside;
            check(cf.append(key.data_ptr(), value.data_ptr(), Call::half(key.scalar_type(), "key"), tokens, heads, dim, Call::apart(key, 0), Call::apart(key, 1), Call::apart(value, 0), Call::apart(value, 1),
                            slots.data_ptr<int>(), cache.data_ptr(), cache.size(0), cache.size(2), c.stream()));
        }
        Py_RETURN_NONE;
    });
}

// (cache, slot_map, head_dim, bf16)
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("kv4_read", n, 4, [&] {
        Call c;
        const at::Tensor& slots = c.ints(a[1], "slot_map");
        const int64_t dim = number(a[2], "head_dim"), tokens = slots.numel();
        const at::Tensor& cache = c.cache(a[0], -1, dim);
        const at::ScalarType type = a[3] == Py_True ? at::kBFloat16 : at::kHalf;
        const int64_t heads = cache.size(1);
        at::Tensor r[2];
        {
            Aside aside;
            for (at::Tensor& t : r) t = empty({tokens, heads, dim}, cache, type);
            check(cf.read(cache.data_ptr(), cache.size(0), cache.size(2), heads, dim, slots.data_ptr<int>(), tokens, r[0].data_ptr(), r[1].data_ptr(), Call::half(type, "dtype"), c.stream()));
        }
        return tuple_of(r);
    });
}

// (query, cache, block_table, kv_lens, qo_indptr or None, max_q_len, scale or None, out or None, workspace bytes or None)
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("kv4_attention", n, 9, [&] {
        Call c;
        const at::Tensor& query = c.rows(a[0], "query", 8);
        const int64_t rows = query.size(0), heads = query.size(1), dim = query.size(2);
        const at::Tensor& lens = c.ints(a[3], "kv_lens");
        const int64_t batch = lens.numel(), max_q = number(a[5], "max_q_len");
        const int* indptr = a[4] == Py_None ? nullptr : c.ints(a[4], "qo_indptr", batch + 1).data_ptr<int>();
        int64_t width, apart;
        const at::Tensor& table = c.table(a[2], batch, &width, &apart);
        const at::Tensor& cache = c.cache(a[1], -1, dim);
        const int64_t kv_heads = cache.size(1), page = cache.size(2);
        const double scale = a[6] == Py_None ? 1.0 / std::sqrt(static_cast<double>(dim)) : PyFloat_AsDouble(a[6]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            complain("scale: expected a number");
        }
        const int64_t asked = a[8] == Py_None ? -1 : number(a[8], "workspace");
        at::Tensor out;
        if (a[7] != Py_None) {
            out = c.on_device(a[7], "out", 3);
            if (!out.sizes().equals(query.sizes()) || out.scalar_type() != query.scalar_type() || !out.is_contiguous())
                complain("out: expected a contiguous ", query.sizes(), " of ", type_name(query.scalar_type()), ", got ", type_name(out.scalar_type()), " ", Shape{out});
        }
        {
            Aside aside;
            if (a[7] == Py_None) out = empty({rows, heads, dim}, query, query.scalar_type());
            const int64_t need = asked < 0 ? cf.workspace(batch, heads, kv_heads, dim, width * page, max_q) : asked;
            at::Tensor work;  // of this call alone: graphs and streams share nothing
            if (need > 0) work = empty({need}, query, at::kByte);
            check(cf.attention(query.data_ptr(), Call::half(query.scalar_type(), "query"), rows, heads, dim, Call::apart(query, 0), Call::apart(query, 1), cache.data_ptr(), cache.size(0), page, kv_heads,
                               table.data_ptr<int>(), width, apart, lens.data_ptr<int>(), indptr, batch, max_q, static_cast<float>(scale), need > 0 ? work.data_ptr() : nullptr, need,
                               out.data_ptr(), c.stream()));
        }
        if (a[7] != Py_None) return Py_NewRef(a[7]);
        return wrap(out);
    });
}

// (logits, tokens, top_k)
PyObject* py_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("token_logprobs", n, 3, [&] {
        Call c;
        at::Tensor logits = tensor(a[0], "logits");
        if (logits.is_cuda() && logits.dim() == 1) {
            if (c.device < 0) c.device = c10::cuda::current_device();
            if (logits.get_device() != c.device) complain("logits: tensor is on ", logits.device(), " but the current device is cuda:", c.device);
            at::AutoDispatchBelowADInplaceOrView below;
            logits = logits.unsqueeze(0);
        } else {
            c.on_device(a[0], "logits", 2);
        }
        const at::ScalarType type = logits.scalar_type();
        if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat)
            complain("logits: expected dtype torch.float16, torch.bfloat16 or torch.float32, got ", type_name(type));
        const int64_t rows = logits.size(0), vocab = logits.size(1), k = number(a[2], "top_k");
        if (logits.stride(1) != 1 && vocab > 1) complain("logits: expected a contiguous last axis, got shape ", Shape{logits});
        const at::Tensor& tokens = c.on_device(a[1], "tokens", 1);
        if ((tokens.scalar_type() != at::kInt && tokens.scalar_type() != at::kLong) || tokens.numel() != rows || !tokens.is_contiguous())
            complain("tokens: expected ", rows, " contiguous entries of torch.int32 or torch.int64, got ", type_name(tokens.scalar_type()), " ", Shape{tokens});
        if (k < 0 || k > 32 || k > vocab) complain("top_k ", k, " outside 0..", vocab < 32 ? vocab : 32);
        at::Tensor r[4];
        {
            Aside aside;
            const at::Tensor buf = empty({rows * (2 + k)}, logits, at::kFloat), ids = empty({rows, k}, logits, at::kLong);
            float* p = buf.data_ptr<float>();
            check(cf.logprobs(logits.data_ptr(), type == at::kHalf ? CF_DTYPE_FP16 : type == at::kBFloat16 ? CF_DTYPE_BF16 : CF_DTYPE_FP32, rows, vocab, logits.stride(0), tokens.data_ptr(),
                              static_cast<int>(tokens.element_size()), k, p, p + rows, p + 2 * rows, ids.data_ptr<int64_t>(), c.stream()));
            r[0] = piece(buf, 0, rows), r[1] = piece(buf, rows, rows), r[2] = buf.as_strided({rows, k}, {k, 1}, 2 * rows), r[3] = ids;
        }
        return tuple_of(r);
    });
}

// addresses of the library's entry points, in the order of Entries
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    constexpr Py_ssize_t COUNT = sizeof(Entries) / sizeof(void*);
    void* at[COUNT];
    if (n != COUNT) {
        PyErr_SetString(PyExc_RuntimeError, "bind: another number of entry points");
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < n; ++i) {
        at[i] = PyLong_AsVoidPtr(a[i]);
        if (!at[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "bind: no address");
            return nullptr;
        }
    }
    static_assert(sizeof(Entries) == sizeof(at), "");
    std::memcpy(&cf, at, sizeof(cf));
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)> PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<py_bind>("bind"),           method<py_plan>("plan"),           method<py_release>("release"), method<py_append>("append"), method<py_read>("read"),
                         method<py_attention>("attention"), method<py_logprobs>("logprobs"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) {
    return PyModule_Create(&module);
}

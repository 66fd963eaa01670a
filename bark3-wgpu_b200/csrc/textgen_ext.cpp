// textgen_ext.cpp — the torch side of the text-generation calls: checks the
// tensors, allocates the outputs and the workspace from torch's allocator and
// calls the C ABI (b3_kv_append, b3_kv_attend, b3_sample) on torch's current
// stream.  textgen.py gives it the ABI's addresses and builds KvCache on Cache.
//
// In C++ because a decode step's calls are short: checking a dozen tensors and
// making the call took 15 us of Python around 3 to 5 us of launches.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/GradMode.h>

#include <exception>
#include <initializer_list>
#include <string>
#include <utility>

#include "../../include/bark3_b200.h"

namespace {

struct Abi {
    decltype(&b3_kv_append) append;
    decltype(&b3_kv_attend_workspace) workspace;
    decltype(&b3_kv_attend) attend;
    decltype(&b3_sample) sample;
    decltype(&b3_last_error) last_error;
} g_abi;
PyObject* g_error = nullptr;   // B3Error(code, message)

struct Raised {};   // the Python exception is set

[[noreturn]] void raise(int code, const std::string& msg) {
    PyObject* e = PyObject_CallFunction(g_error, "is", code, msg.c_str());
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

std::string describe(const at::Tensor& t) {
    std::string s = std::string("(");
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    s += std::string(") ") + at::toString(t.scalar_type()) + " on " + t.device().str() + ", strides (";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.stride(i));
    return s + ")";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) raise(B3_EINVAL, std::string(name) + " must be a torch tensor");
    return THPVariable_Unpack(o);
}

// These calls have no backward: where a gradient would be lost, it is said.
void no_gradient(const char* call, std::initializer_list<std::pair<const char*, PyObject*>> inputs) {
    if (!c10::GradMode::is_enabled()) return;
    for (const auto& [name, o] : inputs)
        if (o && o != Py_None && THPVariable_Check(o) && THPVariable_Unpack(o).requires_grad())
            raise(B3_EINVAL, std::string(call) + " has no backward and " + name +
                                 " requires a gradient: call it under torch.no_grad(), or detach " + name);
}

bool on(const at::Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }

// Address of a contiguous (n,) tensor, null for None.
template <typename P>
P* vector(PyObject* o, const char* name, at::ScalarType type, int64_t n, int device) {
    if (!o || o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !on(t, device) || !t.is_contiguous())
        raise(B3_EINVAL, std::string(name) + " must be a contiguous " + at::toString(type) + " tensor of " + std::to_string(n) +
                             " on cuda:" + std::to_string(device) + ", got " + describe(t));
    return static_cast<P*>(t.data_ptr());
}

int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return B3_DTYPE_F32;
        case at::kHalf: return B3_DTYPE_F16;
        case at::kBFloat16: return B3_DTYPE_BF16;
        default: return -1;
    }
}

// New rows (tokens, heads, head_dim) with adjacent channels.
const void* rows(const at::Tensor& t, const char* name, int64_t tokens, int64_t heads, int64_t dim, at::ScalarType type,
                 int device) {
    if (t.scalar_type() != type || t.dim() != 3 || t.size(0) != tokens || (heads >= 0 && t.size(1) != heads) ||
        t.size(2) != dim || t.stride(2) != 1 || !on(t, device))
        raise(B3_EINVAL, std::string(name) + " must be (" + std::to_string(tokens) + ", " +
                             (heads >= 0 ? std::to_string(heads) : std::string("heads")) + ", " + std::to_string(dim) + ") " +
                             at::toString(type) + " on cuda:" + std::to_string(device) + " with adjacent channels, got " +
                             describe(t));
    return t.data_ptr();
}

at::Tensor output(PyObject* o, at::IntArrayRef shape, const at::Tensor& like, at::ScalarType type, int device) {
    if (!o || o == Py_None) return at::empty(shape, like.options().dtype(type));
    const at::Tensor& t = tensor(o, "out");
    if (t.sizes() != shape || t.scalar_type() != type || !on(t, device) || !t.is_contiguous())
        raise(B3_EINVAL, std::string("out must be a contiguous ") + at::toString(type) + " tensor of the queries' shape, got " +
                             describe(t));
    return t;
}

// Elements from row to row of a tensor with adjacent columns.  That of a single row is any number in torch;
// 0 (an expanded tensor: every row the same) and what else there is goes to the ABI's checks.
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

int i32(int64_t v, const char* name) {
    if (v < 0 || v > 0x7fffffff) raise(B3_EINVAL, std::string(name) + " " + std::to_string(v) + " is out of range");
    return static_cast<int>(v);
}

// Runs f(stream) on torch's current stream of `device`, that device being current.
template <typename F>
void call(int device, F f) {
    const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() == device
                                                 ? std::optional<c10::Device>()
                                                 : std::optional<c10::Device>(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device))));
    const int64_t rc = f(static_cast<void*>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream()));
    if (rc < 0) raise(static_cast<int>(rc), g_abi.last_error());
}

template <typename F>
PyObject* guarded(F f) {
    try {
        const at::AutoDispatchBelowADInplaceOrView below;   // plain memory: nothing here is differentiated (no_gradient)
        return f();
    } catch (const Raised&) {
    } catch (...) {   // torch's own: each as the Python type that torch gives it (out of memory among them)
        if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

struct Cache {
    PyObject_HEAD
    b3_kv_cache c;
    int device;
    PyObject* held;   // the tensors, as a tuple
};

b3_kv_batch batch(const Cache* self, int64_t tokens, PyObject* cu_q, PyObject* kv_lens, PyObject* page_table) {
    const at::Tensor& lens = tensor(kv_lens, "kv_lens");
    const int64_t n = lens.dim() == 1 ? lens.size(0) : -1;
    b3_kv_batch b{};
    b.cu_q = vector<int32_t>(cu_q, "cu_q", at::kInt, n + 1, self->device);
    b.kv_lens = vector<int32_t>(kv_lens, "kv_lens", at::kInt, n, self->device);
    const at::Tensor& table = tensor(page_table, "page_table");
    if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != n || !on(table, self->device) || table.stride(1) != 1)
        raise(B3_EINVAL, "page_table must be a (" + std::to_string(n) + ", width) Int tensor with adjacent entries, got " +
                             describe(table));
    b.page_table = static_cast<const int32_t*>(table.data_ptr());
    b.table_width = i32(table.size(1), "page_table's width");
    b.table_stride = row_stride(table);
    b.n_seq = i32(n, "the number of sequences");
    b.tokens = i32(tokens, "the number of tokens");
    return b;
}

PyObject* cache_hold(PyObject* o, PyObject* args) {
    Cache* self = reinterpret_cast<Cache*>(o);
    PyObject *k, *v, *ks, *vs, *status;
    if (!PyArg_ParseTuple(args, "OOOOO", &k, &v, &ks, &vs, &status)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& t = tensor(k, "k");
        if (t.dim() != 4 || !t.is_cuda()) raise(B3_EINVAL, "k must be a (pages, kv_heads, page_tokens, head_dim) tensor on a GPU");
        const int device = t.get_device();
        auto pool = [&](PyObject* x, const char* name) {
            const at::Tensor& y = tensor(x, name);
            if (y.scalar_type() != at::kFloat8_e4m3fn || y.sizes() != t.sizes() || !on(y, device) || !y.is_contiguous())
                raise(B3_EINVAL, std::string(name) + " must be a contiguous Float8_e4m3fn tensor of k's shape, got " + describe(y));
            return static_cast<uint8_t*>(y.data_ptr());
        };
        auto scale = [&](PyObject* x, const char* name) {
            const at::Tensor& y = tensor(x, name);
            if (y.scalar_type() != at::kFloat || y.dim() != 2 || y.size(0) != t.size(0) || y.size(1) != t.size(1) || !on(y, device) ||
                !y.is_contiguous())
                raise(B3_EINVAL, std::string(name) + " must be a contiguous (pages, kv_heads) Float tensor, got " + describe(y));
            return static_cast<float*>(y.data_ptr());
        };
        b3_kv_cache c{};
        c.k = pool(k, "k"), c.v = pool(v, "v");
        c.k_scale = scale(ks, "k_scale"), c.v_scale = scale(vs, "v_scale");
        c.status = vector<int32_t>(status, "status", at::kInt, 1, device);
        c.pages = i32(t.size(0), "pages"), c.kv_heads = i32(t.size(1), "kv_heads");
        c.page_tokens = i32(t.size(2), "page_tokens"), c.head_dim = i32(t.size(3), "head_dim");
        self->c = c;
        self->device = device;
        Py_INCREF(args);
        Py_XSETREF(self->held, args);
        Py_RETURN_NONE;
    });
}

bool ready(const Cache* self) {
    if (!self->held) PyErr_SetString(PyExc_RuntimeError, "the cache has no tensors");
    return self->held != nullptr;
}

PyObject* cache_append(PyObject* o, PyObject* args, PyObject* kwargs) {
    Cache* self = reinterpret_cast<Cache*>(o);
    static const char* names[] = {"q", "k", "v", "cu_q", "kv_lens", "page_table", "q_norm", "k_norm", "eps", "cos", "sin",
                                  "interleaved", "positions", "out", nullptr};
    PyObject *q_, *k_, *v_, *cu, *lens, *table, *qn = nullptr, *kn = nullptr, *cos = nullptr, *sin = nullptr, *pos = nullptr,
                                                *out_ = nullptr;
    float eps = 1e-6f;
    int interleaved = 0;
    if (!PyArg_ParseTupleAndKeywords(args, kwargs, "OOOOOO|$OOfOOpOO:append", const_cast<char**>(names), &q_, &k_, &v_, &cu,
                                     &lens, &table, &qn, &kn, &eps, &cos, &sin, &interleaved, &pos, &out_) ||
        !ready(self))
        return nullptr;
    return guarded([&]() -> PyObject* {
        no_gradient("append", {{"q", q_}, {"k", k_}, {"v", v_}, {"q_norm", qn}, {"k_norm", kn}, {"cos", cos}, {"sin", sin}});
        const at::Tensor &q = tensor(q_, "q"), &k = tensor(k_, "k"), &v = tensor(v_, "v");
        const int device = self->device, dim = self->c.head_dim;
        b3_kv_append_args a{};
        a.dtype = dtype_of(q);
        if (a.dtype < 0) raise(B3_EINVAL, "q must be Float, Half or BFloat16, got " + describe(q));
        const int64_t tokens = q.dim() ? q.size(0) : 0;
        a.q = rows(q, "q", tokens, -1, dim, q.scalar_type(), device);
        a.k = rows(k, "k", tokens, self->c.kv_heads, dim, q.scalar_type(), device);
        a.v = rows(v, "v", tokens, self->c.kv_heads, dim, q.scalar_type(), device);
        a.q_token_stride = q.stride(0), a.q_head_stride = q.stride(1);
        a.k_token_stride = k.stride(0), a.k_head_stride = k.stride(1);
        a.v_token_stride = v.stride(0), a.v_head_stride = v.stride(1);
        const b3_kv_batch b = batch(self, tokens, cu, lens, table);
        a.q_norm = vector<float>(qn, "q_norm", at::kFloat, dim, device);
        a.k_norm = vector<float>(kn, "k_norm", at::kFloat, dim, device);
        a.positions = vector<int32_t>(pos, "positions", at::kInt, tokens, device);
        const bool turn = cos && cos != Py_None;
        if (turn != (sin && sin != Py_None)) raise(B3_EINVAL, "cos and sin come together");
        if (turn) {
            const at::Tensor& c = tensor(cos, "cos");
            const float* at_[2];
            for (int i = 0; i < 2; ++i) {
                const at::Tensor& t = tensor(i ? sin : cos, i ? "sin" : "cos");
                if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.sizes() != c.sizes() || !on(t, device) || !t.is_contiguous())
                    raise(B3_EINVAL, std::string(i ? "sin" : "cos") + " must be a contiguous Float (positions, rot_dim / 2) tensor, got " +
                                         describe(t));
                at_[i] = static_cast<const float*>(t.data_ptr());
            }
            a.cos = at_[0], a.sin = at_[1];
            a.rot_rows = i32(c.size(0), "the cos table's length");
            a.rot_dim = i32(2 * c.size(1), "rot_dim");
        }
        a.eps = eps;
        a.interleaved = interleaved;
        a.q_heads = i32(q.size(1), "q's heads");
        a.out_dtype = a.dtype == B3_DTYPE_F32 ? B3_DTYPE_F16 : a.dtype;
        at::Tensor out = output(out_, q.sizes(), q, a.dtype == B3_DTYPE_F32 ? at::kHalf : q.scalar_type(), device);
        a.q_out = out.data_ptr();
        call(device, [&](void* st) { return g_abi.append(&self->c, &b, &a, st); });
        return THPVariable_Wrap(std::move(out));
    });
}

PyObject* cache_attend(PyObject* o, PyObject* args, PyObject* kwargs) {
    Cache* self = reinterpret_cast<Cache*>(o);
    static const char* names[] = {"q", "cu_q", "kv_lens", "page_table", "max_q", "scale", "causal", "window", "out", "return_lse",
                                  nullptr};
    PyObject *q_, *cu, *lens, *table, *max_q = nullptr, *scale = nullptr, *out_ = nullptr;
    int causal = 1, window = 0, return_lse = 0;
    if (!PyArg_ParseTupleAndKeywords(args, kwargs, "OOOO|$OOpiOp:attend", const_cast<char**>(names), &q_, &cu, &lens, &table,
                                     &max_q, &scale, &causal, &window, &out_, &return_lse) ||
        !ready(self))
        return nullptr;
    if (!max_q) {
        PyErr_SetString(PyExc_TypeError, "attend() missing 1 required keyword-only argument: 'max_q'");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        no_gradient("attend", {{"q", q_}});
        const at::Tensor& q = tensor(q_, "q");
        const int device = self->device;
        b3_kv_attend_args a{};
        a.dtype = dtype_of(q);
        if (a.dtype != B3_DTYPE_F16 && a.dtype != B3_DTYPE_BF16) raise(B3_EINVAL, "q must be Half or BFloat16, got " + describe(q));
        const int64_t tokens = q.dim() ? q.size(0) : 0;
        a.q = rows(q, "q", tokens, -1, self->c.head_dim, q.scalar_type(), device);
        a.q_token_stride = q.stride(0), a.q_head_stride = q.stride(1);
        const b3_kv_batch b = batch(self, tokens, cu, lens, table);
        const long most = PyLong_AsLong(max_q);
        if (most == -1 && PyErr_Occurred()) throw Raised{};
        a.max_q = i32(most, "max_q");
        a.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(self->c.head_dim)));
        if (scale && scale != Py_None) {
            const double s = PyFloat_AsDouble(scale);
            if (s == -1.0 && PyErr_Occurred()) throw Raised{};
            a.scale = static_cast<float>(s);
        }
        a.causal = causal;
        a.window = window;
        a.q_heads = i32(q.size(1), "q's heads");
        at::Tensor out = output(out_, q.sizes(), q, q.scalar_type(), device), lse, work;
        a.out = out.data_ptr();
        if (return_lse) {
            lse = at::empty({tokens, q.size(1)}, q.options().dtype(at::kFloat));
            a.lse = static_cast<float*>(lse.data_ptr());
        }
        call(device, [&](void* st) -> int64_t {
            const int64_t need = g_abi.workspace(&self->c, &b, &a);
            if (need < 0) return need;
            // from torch's allocator on the current stream: calls on other streams get other memory
            work = at::empty({need}, q.options().dtype(at::kByte));
            return g_abi.attend(&self->c, &b, &a, work.data_ptr(), need, st);
        });
        if (!return_lse) return THPVariable_Wrap(std::move(out));
        return Py_BuildValue("NN", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(lse)));
    });
}

PyObject* sample(PyObject*, PyObject* args, PyObject* kwargs) {
    static const char* names[] = {"logits", "uniform", "temperature", "top_k", "top_p", "min_p", nullptr};
    PyObject *x_, *u, *t = nullptr, *k = nullptr, *p = nullptr, *m = nullptr;
    if (!PyArg_ParseTupleAndKeywords(args, kwargs, "OO|$OOOO:sample", const_cast<char**>(names), &x_, &u, &t, &k, &p, &m))
        return nullptr;
    return guarded([&]() -> PyObject* {
        no_gradient("sample", {{"logits", x_}});
        const at::Tensor& x = tensor(x_, "logits");
        b3_sample_args a{};
        a.dtype = dtype_of(x);
        if (a.dtype < 0 || x.dim() != 2 || !x.is_cuda() || x.stride(1) != 1)
            raise(B3_EINVAL, "logits must be a (rows, vocab) Float, Half or BFloat16 tensor on a GPU with adjacent columns, got " +
                                 describe(x));
        const int device = x.get_device();
        const int64_t n = x.size(0);
        if (u == Py_None) raise(B3_EINVAL, "uniform is missing");
        a.logits = x.data_ptr();
        a.uniform = vector<float>(u, "uniform", at::kFloat, n, device);
        a.temperature = vector<float>(t, "temperature", at::kFloat, n, device);
        a.top_k = vector<int32_t>(k, "top_k", at::kInt, n, device);
        a.top_p = vector<float>(p, "top_p", at::kFloat, n, device);
        a.min_p = vector<float>(m, "min_p", at::kFloat, n, device);
        a.rows = i32(n, "the number of rows");
        a.vocab = i32(x.size(1), "the vocabulary");
        a.row_stride = row_stride(x);
        at::Tensor ids = at::empty({n}, x.options().dtype(at::kInt)), logprob = at::empty({n}, x.options().dtype(at::kFloat));
        a.ids = static_cast<int32_t*>(ids.data_ptr());
        a.logprob = static_cast<float*>(logprob.data_ptr());
        call(device, [&](void* st) { return g_abi.sample(&a, st); });
        return Py_BuildValue("NN", THPVariable_Wrap(std::move(ids)), THPVariable_Wrap(std::move(logprob)));
    });
}

PyObject* bind(PyObject*, PyObject* args) {
    PyObject* error;
    unsigned long long p[5];
    if (!PyArg_ParseTuple(args, "OKKKKK", &error, p, p + 1, p + 2, p + 3, p + 4)) return nullptr;
    g_abi = {reinterpret_cast<decltype(g_abi.append)>(p[0]), reinterpret_cast<decltype(g_abi.workspace)>(p[1]),
             reinterpret_cast<decltype(g_abi.attend)>(p[2]), reinterpret_cast<decltype(g_abi.sample)>(p[3]),
             reinterpret_cast<decltype(g_abi.last_error)>(p[4])};
    Py_INCREF(error);
    Py_XSETREF(g_error, error);
    Py_RETURN_NONE;
}

void cache_dealloc(PyObject* o) {
    PyTypeObject* type = Py_TYPE(o);
    Py_XDECREF(reinterpret_cast<Cache*>(o)->held);
    type->tp_free(o);
    Py_DECREF(type);
}

PyMethodDef cache_methods[] = {
    {"_hold", cache_hold, METH_VARARGS, nullptr},
    {"append", reinterpret_cast<PyCFunction>(cache_append), METH_VARARGS | METH_KEYWORDS,
     "append(q, k, v, cu_q, kv_lens, page_table, *, q_norm=None, k_norm=None, eps=1e-6, cos=None, sin=None,\n"
     "       interleaved=False, positions=None, out=None) -> queries\n\n"
     "Norms and rotates the new tokens' q (tokens, q_heads, head_dim) and k (tokens, kv_heads, head_dim),\n"
     "stores k and v in the cache and returns the queries, ready for attend(): in q's own type, or float16\n"
     "for float32 input.  kv_lens counts the new tokens already.  q, k and v may be views of one\n"
     "projection's output."},
    {"attend", reinterpret_cast<PyCFunction>(cache_attend), METH_VARARGS | METH_KEYWORDS,
     "attend(q, cu_q, kv_lens, page_table, *, max_q, scale=None, causal=True, window=0, out=None,\n"
     "       return_lse=False) -> out or (out, lse)\n\n"
     "Attention of the new tokens' queries (tokens, q_heads, head_dim), float16 or bfloat16, over the cached\n"
     "keys and values of their sequences.  max_q: an upper bound of any sequence's new tokens.  scale:\n"
     "1 / sqrt(head_dim) by default.  out has q's type; lse is the (tokens, q_heads) float32 log-sum-exp."},
    {nullptr, nullptr, 0, nullptr}};

PyType_Slot cache_slots[] = {{Py_tp_methods, cache_methods},
                             {Py_tp_dealloc, reinterpret_cast<void*>(cache_dealloc)},
                             {Py_tp_new, reinterpret_cast<void*>(PyType_GenericNew)},
                             {0, nullptr}};
PyType_Spec cache_spec = {"_textgen.Cache", sizeof(Cache), 0, Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE, cache_slots};

PyMethodDef functions[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(sample), METH_VARARGS | METH_KEYWORDS,
     "sample(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None) -> (ids, logprob)\n\n"
     "The next token of every row of logits (rows, vocab), float32, float16 or bfloat16: ids int32, logprob\n"
     "float32, each (rows,).  uniform and the settings are (rows,) tensors on the logits' GPU (top_k int32, the\n"
     "others float32); None leaves a setting off (temperature: 1)."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_textgen", nullptr, -1, functions, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__textgen() {
    PyObject* m = PyModule_Create(&module);
    if (!m) return nullptr;
    PyObject* type = PyType_FromSpec(&cache_spec);
    if (!type || PyModule_AddObject(m, "Cache", type) < 0) {
        Py_XDECREF(type);
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}

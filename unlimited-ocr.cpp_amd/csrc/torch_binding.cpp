// Torch tensors -> libuocr_hip's rotary and paged-attention entry points: the checks of
// uocr_hip.paged in native code. A call of these takes a few us on the GPU when it decodes for a few requests;
// reading 4 to 12 tensors' attributes through Python alone took 7 to 10 us, here well under one.
// The module holds no state but the entry points' addresses (bind), which the
// ctypes loader gives, so that both work on one library.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include "uocr_hip/moe_capi.h"

namespace {

decltype(&uocr_hip_rope) f_rope;
decltype(&uocr_hip_rope_append_paged) f_append;
decltype(&uocr_hip_paged_attention_decode) f_decode;
decltype(&uocr_hip_paged_attention_prefill) f_prefill;

struct Refused {};  // a Python error is set

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
    va_list args;
    va_start(args, format);
    PyErr_FormatV(type, format, args);
    va_end(args);
    throw Refused{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", name);
    return THPVariable_Unpack(o);
}

int integer(PyObject* o, const char* name) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{};
    if (v != (int)v) refuse(PyExc_OverflowError, "%s does not fit an int", name);
    return (int)v;
}
float real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused{};
    return (float)v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Refused{};
    return v != 0;
}
void* address(PyObject* o) {
    if (o == Py_None) return nullptr;
    void* p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw Refused{};
    return p;
}

// [rows, heads, head_dim] of a call's first tensor
struct Shape {
    int n, h, d, gpu;
};
Shape shape(const at::Tensor& t, const char* name) {
    const int gpu = (int)t.get_device();
    if (gpu < 0) refuse(PyExc_ValueError, "%s must be on a GPU", name);
    if (t.dim() != 3) refuse(PyExc_ValueError, "%s must be [rows, heads, head_dim]", name);
    for (int i = 0; i < 3; ++i)
        if (t.size(i) > INT_MAX) refuse(PyExc_ValueError, "%s is too large", name);
    return Shape{(int)t.size(0), (int)t.size(1), (int)t.size(2), gpu};
}

// Rows of heads of that shape on that GPU, the dims of a head contiguous
uocr_hip_rows rows(const at::Tensor& t, const char* name, const Shape& s) {
    if (t.get_device() != s.gpu) refuse(PyExc_ValueError, "%s is not on GPU %d", name, s.gpu);
    if (t.dim() != 3 || t.size(0) != s.n || t.size(1) != s.h || t.size(2) != s.d || (t.stride(2) != 1 && s.d > 1))
        refuse(PyExc_ValueError, "%s must be [%d, %d, %d] with contiguous dims of a head", name, s.n, s.h, s.d);
    int dt = -1;
    if (t.scalar_type() == at::kFloat) dt = UOCR_HIP_DTYPE_F32;
    else if (t.scalar_type() == at::kBFloat16) dt = UOCR_HIP_DTYPE_BF16;
    else if (t.scalar_type() == at::kHalf) dt = UOCR_HIP_DTYPE_F16;
    else refuse(PyExc_TypeError, "%s must be f32, bf16 or f16", name);
    return uocr_hip_rows{t.data_ptr(), dt, t.stride(0), t.stride(1)};
}

// Contiguous vector of n entries on that GPU (None: null)
void* vector(PyObject* o, const char* name, int64_t n, int gpu, at::ScalarType type) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != type || t.get_device() != gpu || t.numel() != n || !t.is_contiguous())
        refuse(PyExc_ValueError, "%s must be a contiguous %s tensor of %lld entries on GPU %d", name,
               type == at::kInt ? "int32" : "f32", (long long)n, gpu);
    return t.data_ptr();
}
const int* ints(PyObject* o, const char* name, int64_t n, int gpu) { return (const int*)vector(o, name, n, gpu, at::kInt); }
const float* floats(PyObject* o, const char* name, int64_t n, int gpu) {
    return (const float*)vector(o, name, n, gpu, at::kFloat);
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
        return nullptr;
    }
    try {
        return PyLong_FromLong(f());
    } catch (const Refused&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}
template <typename F>
int call(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

// q, k, positions, inv_freq, q_out, k_out, interleaved, factor, stream
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 9, [&] {
        const at::Tensor& q = tensor(a[0], "q");
        const Shape s = shape(q, "q");
        const uocr_hip_rows qi = rows(q, "q", s), qo = rows(tensor(a[4], "q_out"), "q_out", s);
        uocr_hip_rows ki{}, ko{};
        Shape ks{s.n, 0, s.d, s.gpu};
        if ((a[1] == Py_None) != (a[5] == Py_None)) refuse(PyExc_ValueError, "k and k_out go together");
        if (a[1] != Py_None) {
            const at::Tensor& k = tensor(a[1], "k");
            ks.h = shape(k, "k").h;
            ki = rows(k, "k", ks);
            ko = rows(tensor(a[5], "k_out"), "k_out", ks);
        }
        const int64_t half = tensor(a[3], "inv_freq").numel();
        if (half > 1 << 20) refuse(PyExc_ValueError, "inv_freq is too long");
        const int* pos = ints(a[2], "positions", s.n, s.gpu);
        const float* freq = floats(a[3], "inv_freq", half, s.gpu);
        const bool pairs = truth(a[6]);
        const float factor = real(a[7]);
        void* stream = address(a[8]);
        return call([&] {
            return f_rope(&qi, ks.h ? &ki : nullptr, s.n, s.h, ks.h, s.d, pos, freq, (int)(2 * half), pairs, factor, &qo,
                          ks.h ? &ko : nullptr, stream);
        });
    });
}

// q, k, v, positions, inv_freq, cache address, GPU, seqs, rows, q_out, interleaved, factor, stream
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 13, [&] {
        const auto* cache = (const uocr_hip_paged_cache*)address(a[5]);
        const int gpu = integer(a[6], "GPU");
        const at::Tensor& q = tensor(a[0], "q");
        Shape s = shape(q, "q");
        if (s.gpu != gpu || s.d != cache->head_dim)
            refuse(PyExc_ValueError, "q must be on GPU %d with heads of %d", gpu, cache->head_dim);
        const Shape ks{s.n, cache->kv_heads, s.d, gpu};
        const uocr_hip_rows qi = rows(q, "q", s), ki = rows(tensor(a[1], "k"), "k", ks), vi = rows(tensor(a[2], "v"), "v", ks);
        const uocr_hip_rows qo = rows(tensor(a[9], "q_out"), "q_out", s);
        const int64_t half = a[4] == Py_None ? 0 : tensor(a[4], "inv_freq").numel();
        if (half > 1 << 20) refuse(PyExc_ValueError, "inv_freq is too long");
        const int* pos = half ? ints(a[3], "positions", s.n, gpu) : nullptr;
        const float* freq = half ? floats(a[4], "inv_freq", half, gpu) : nullptr;
        const int *seqs = ints(a[7], "seqs", s.n, gpu), *at = ints(a[8], "rows", s.n, gpu);
        const bool pairs = truth(a[10]);
        const float factor = real(a[11]);
        void* stream = address(a[12]);
        return call([&] {
            return f_append(&qi, &ki, &vi, s.n, s.h, pos, freq, (int)(2 * half), pairs, factor, cache, seqs, at, &qo, stream);
        });
    });
}

// q, cache address, GPU, q_start (None: one new token per sequence), kv_len, out, seqs, causal, scale, softcap, slopes,
// window, prefix_len, prefix_both_ways, key_begin, key_end, max_kv_len, workspace, stream
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 19, [&] {
        const auto* cache = (const uocr_hip_paged_cache*)address(a[1]);
        const int gpu = integer(a[2], "GPU");
        const at::Tensor& q = tensor(a[0], "q");
        const Shape s = shape(q, "q");
        if (s.gpu != gpu || s.d != cache->head_dim)
            refuse(PyExc_ValueError, "q must be on GPU %d with heads of %d", gpu, cache->head_dim);
        const uocr_hip_rows qi = rows(q, "q", s), oi = rows(tensor(a[5], "out"), "out", s);
        int batch = s.n;
        const int* start = nullptr;
        if (a[3] != Py_None) {
            const int64_t entries = tensor(a[3], "q_start").numel();
            if (entries < 1 || entries > INT_MAX) refuse(PyExc_ValueError, "q_start needs batch + 1 entries");
            batch = (int)entries - 1;
            start = ints(a[3], "q_start", entries, gpu);
        }
        if (a[4] == Py_None) refuse(PyExc_ValueError, "kv_len is missing");
        const int* kv_len = ints(a[4], "kv_len", cache->n_seqs, gpu);
        const int* seqs = ints(a[6], "seqs", batch, gpu);
        uocr_hip_attention_opts o{};
        o.heads = s.h;
        o.causal = truth(a[7]);
        o.scale = a[8] == Py_None ? 0.0f : real(a[8]);
        o.softcap = real(a[9]);
        o.slopes = floats(a[10], "slopes", s.h, gpu);
        o.window = integer(a[11], "window");
        o.prefix_len = ints(a[12], "prefix_len", cache->n_seqs, gpu);
        o.prefix_both_ways = truth(a[13]);
        o.key_begin = ints(a[14], "key_begin", s.n, gpu);
        o.key_end = ints(a[15], "key_end", s.n, gpu);
        const int most = integer(a[16], "max_kv_len");
        void* ws = nullptr;
        size_t size = 0;
        if (a[17] != Py_None) {
            const at::Tensor& w = tensor(a[17], "workspace");
            if (w.get_device() != gpu || !w.is_contiguous())
                refuse(PyExc_ValueError, "workspace must be a contiguous tensor on GPU %d", gpu);
            ws = w.data_ptr();
            size = w.nbytes();
        }
        void* stream = address(a[18]);
        return call([&] {
            return start ? f_prefill(cache, &o, &qi, s.n, batch, start, seqs, kv_len, most, &oi, ws, size, stream)
                         : f_decode(cache, &o, &qi, batch, seqs, kv_len, most, &oi, ws, size, stream);
        });
    });
}

// addresses of uocr_hip_rope, _rope_append_paged, _paged_attention_decode, _paged_attention_prefill
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 4, [&] {
        f_rope = (decltype(f_rope))address(a[0]);
        f_append = (decltype(f_append))address(a[1]);
        f_decode = (decltype(f_decode))address(a[2]);
        f_prefill = (decltype(f_prefill))address(a[3]);
        return 0;
    });
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
                         {"rope", (PyCFunction)(void (*)())rope, METH_FASTCALL, nullptr},
                         {"rope_append", (PyCFunction)(void (*)())rope_append, METH_FASTCALL, nullptr},
                         {"attention", (PyCFunction)(void (*)())attention, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_uocr_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__uocr_torch() { return PyModule_Create(&module); }

// PyTorch side of the 8-bit paged cache's calls (kv8.py): reads the tensors' pointers, strides and types
// and calls the C entry points of libbreeze.so, whose addresses kv8.py hands over at load. The same
// through ctypes costs 5 to 10 us a call, more than a decode step's kernels take.
//
// A Python module of its own (not part of libbreeze.so, which knows nothing of Python or PyTorch).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/bzb_ext.h"

namespace {

decltype(&bzb_kv8_append) f_append;
decltype(&bzb_kv8_read) f_read;
decltype(&bzb_kv8_attention) f_attention;
decltype(&bzb_kv8_attention_workspace) f_workspace;
decltype(&breeze_last_error) f_error;

struct Refused {};  // a Python exception is set

// kv8.py's batch: the C struct and the device its arrays are on
struct Batch : bzb_kv8_batch {
    int device;
};

[[noreturn]] void value_error(const std::string & what) {
    PyErr_SetString(PyExc_ValueError, what.c_str());
    throw Refused{};
}

// a new reference, given back at the end of its scope (at::empty may throw)
struct Ref {
    PyObject * o;
    explicit Ref(PyObject * p) : o(p) {
        if (!o) throw Refused{};
    }
    ~Ref() { Py_DECREF(o); }
    Ref(const Ref &) = delete;
    Ref & operator=(const Ref &) = delete;
};

template <typename T>
T * address(PyObject * o) {
    T * p = static_cast<T *>(PyLong_AsVoidPtr(o));
    if (!p && !PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null handle");
    if (PyErr_Occurred()) throw Refused{};
    return p;
}

const bzb_kv8_batch & batch(PyObject * o, const bzb_kv8_cache & c) {
    const Batch & b = *address<Batch>(o);
    if (b.device != c.device) value_error("the batch is on another device than the cache");
    return b;
}

const at::Tensor & tensor(PyObject * o, const char * name, int device) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: a tensor expected", name);
        throw Refused{};
    }
    const at::Tensor & t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != device) value_error(std::string(name) + ": a tensor on cuda:" + std::to_string(device) + " expected");
    return t;
}

bzb_kv8_rows rows(PyObject * o, const char * name, const bzb_kv8_cache & c, const bzb_kv8_batch & b) {
    const at::Tensor & t = tensor(o, name, c.device);
    if (t.dim() != 3 || t.size(0) != b.n_tok || t.size(2) != c.head_dim)
        value_error(std::string(name) + ": [" + std::to_string(b.n_tok) + ", heads, " + std::to_string(c.head_dim) + "] expected");
    if (t.stride(2) != 1) value_error(std::string(name) + ": contiguous heads expected");
    const auto k = t.scalar_type();
    const int type = k == at::kFloat ? BZB_F32 : k == at::kHalf ? BZB_F16 : k == at::kBFloat16 ? BZB_BF16 : -1;
    return { t.data_ptr(), t.stride(0), t.stride(1), (int) t.size(1), type };
}

// a contiguous f32 tensor of the given sizes (-1: any), or NULL for None
float * floats(PyObject * o, const char * name, int device, std::initializer_list<int64_t> sizes) {
    if (o == Py_None) return nullptr;
    const at::Tensor & t = tensor(o, name, device);
    bool ok = t.scalar_type() == at::kFloat && t.is_contiguous() && t.dim() == (int64_t) sizes.size();
    int64_t d = 0;
    for (int64_t n : sizes) {
        ok = ok && (n < 0 || t.size(d) == n);
        d++;
    }
    if (!ok) {
        std::string s;
        for (int64_t n : sizes) s += (s.empty() ? "" : ", ") + (n < 0 ? std::string("n") : std::to_string(n));
        value_error(std::string(name) + ": contiguous float32 [" + s + "] expected");
    }
    return static_cast<float *>(t.data_ptr());
}

PyObject * done(int rc) {
    if (rc < 0) {
        PyErr_SetString(PyExc_RuntimeError, f_error());
        return nullptr;
    }
    Py_RETURN_NONE;
}

template <typename F>
PyObject * guarded(Py_ssize_t n, Py_ssize_t want, F && f) {
    HANDLE_TH_ERRORS
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
        return nullptr;
    }
    try {
        return f();
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

double number(PyObject * o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw Refused{};
    return x;
}
int integer(PyObject * o) {
    const long x = PyLong_AsLong(o);
    if (x == -1 && PyErr_Occurred()) throw Refused{};
    if (x != (int) x) value_error("an argument is out of range");
    return (int) x;
}

// append(cache, batch, q, k, v, q_out, q_norm, k_norm, eps, rope)
PyObject * append(PyObject *, PyObject * const * a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject * {
        const auto & c = *address<bzb_kv8_cache>(a[0]);
        const bzb_kv8_batch & b = batch(a[1], c);
        const bzb_kv8_rows k = rows(a[3], "k", c, b), v = rows(a[4], "v", c, b);
        bzb_kv8_rows q, o;
        if (a[2] != Py_None) q = rows(a[2], "q", c, b);
        if (a[5] != Py_None) o = rows(a[5], "q_out", c, b);
        const float * wq = floats(a[6], "q_norm", c.device, { c.head_dim }), * wk = floats(a[7], "k_norm", c.device, { c.head_dim });
        const float * rope = floats(a[9], "rope", c.device, { -1, c.head_dim / 2, 2 });
        const int64_t rope_len = rope ? THPVariable_Unpack(a[9]).size(0) : 0;
        return done(f_append(&c, &b, a[2] != Py_None ? &q : nullptr, &k, &v, a[5] != Py_None ? &o : nullptr, wq, wk,
                             (float) number(a[8]), rope, (int) std::min<int64_t>(rope_len, INT_MAX),
                             c10::cuda::getCurrentCUDAStream(c.device).stream()));
    });
}

// read(cache, batch, k_out, v_out)
PyObject * read(PyObject *, PyObject * const * a, Py_ssize_t n) {
    return guarded(n, 4, [&]() -> PyObject * {
        const auto & c = *address<bzb_kv8_cache>(a[0]);
        const bzb_kv8_batch & b = batch(a[1], c);
        const bzb_kv8_rows k = rows(a[2], "k_out", c, b), v = rows(a[3], "v_out", c, b);
        return done(f_read(&c, &b, &k, &v, c10::cuda::getCurrentCUDAStream(c.device).stream()));
    });
}

// attention(cache, batch, workspaces, q, out, scale, causal, window, lse); workspaces: a dict of this function's
PyObject * attention(PyObject *, PyObject * const * a, Py_ssize_t n) {
    return guarded(n, 9, [&]() -> PyObject * {
        const auto & c = *address<bzb_kv8_cache>(a[0]);
        const bzb_kv8_batch & b = batch(a[1], c);
        const bzb_kv8_rows q = rows(a[3], "q", c, b), o = rows(a[4], "out", c, b);
        const int causal = PyObject_IsTrue(a[6]), window = integer(a[7]);
        if (causal < 0) return nullptr;
        float * lse = floats(a[8], "lse", c.device, { b.n_tok, q.n_head });
        const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.device).stream();
        const long long need = f_workspace(&c, &b, q.n_head, causal, window);
        if (need < 0) return done(-1);
        void * space = nullptr;
        if (need > 0) {
            // One for each stream and size, kept as long as the batch, and one for each capture: a graph runs on
            // whatever stream it is launched on, beside other graphs that were captured on the same one.
            cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
            unsigned long long graph = 0;
            if (cudaStreamGetCaptureInfo(stream, &capture, &graph) != cudaSuccess) {
                (void) cudaGetLastError();
                PyErr_SetString(PyExc_RuntimeError, "kv8_attention: the stream's capture is not valid");
                throw Refused{};
            }
            const Ref key(Py_BuildValue("(KLK)", (unsigned long long) reinterpret_cast<uintptr_t>(stream), need,
                                        capture == cudaStreamCaptureStatusNone ? 0ull : graph + 1));
            PyObject * held = PyDict_GetItemWithError(a[2], key.o);  // (borrowed)
            if (!held && PyErr_Occurred()) throw Refused{};
            if (held) {
                space = THPVariable_Unpack(held).data_ptr();
            } else {
                const at::Tensor t = at::empty({ (int64_t) need }, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, c.device));
                space = t.data_ptr();
                const Ref py(THPVariable_Wrap(t));
                if (PyDict_SetItem(a[2], key.o, py.o) != 0) throw Refused{};
            }
        }
        return done(f_attention(&c, &b, &q, &o, lse, (float) number(a[5]), causal, window, space, need, stream));
    });
}

// bind(append, read, attention, attention_workspace, last_error): the entry points' addresses
PyObject * bind(PyObject *, PyObject * const * a, Py_ssize_t n) {
    return guarded(n, 5, [&]() -> PyObject * {
        void * p[5];
        for (int i = 0; i < 5; i++) p[i] = address<void>(a[i]);
        f_append = reinterpret_cast<decltype(f_append)>(p[0]);
        f_read = reinterpret_cast<decltype(f_read)>(p[1]);
        f_attention = reinterpret_cast<decltype(f_attention)>(p[2]);
        f_workspace = reinterpret_cast<decltype(f_workspace)>(p[3]);
        f_error = reinterpret_cast<decltype(f_error)>(p[4]);
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {
    { "append", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(append)), METH_FASTCALL, nullptr },
    { "read", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(read)), METH_FASTCALL, nullptr },
    { "attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(attention)), METH_FASTCALL, nullptr },
    { "bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(bind)), METH_FASTCALL, nullptr },
    { nullptr, nullptr, 0, nullptr },
};
PyModuleDef module = { PyModuleDef_HEAD_INIT, "_kv8_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr };

}  // namespace

PyMODINIT_FUNC PyInit__kv8_torch() { return PyModule_Create(&module); }

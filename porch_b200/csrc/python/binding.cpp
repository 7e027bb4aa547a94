// The part of the Python binding where a call's own cost counts: tensor handles
// and the decode-step operators, whose kernels take a few microseconds. A
// ctypes call of such an operator cost 2 to 5 us more than the operator, and
// handing a result to another library 2 us more; everything else stays with
// ctypes (porch_b200/api.py). Interpreters that this module was not built for use
// porch_b200/ctypes_binding.py in its place.
//
// The native library is not linked: importing the module does not load it, and
// porch_b200/_lib.py hands it over (connect) once the first use has.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "porch_b200.h"

#include <array>
#include <dlfcn.h>

namespace {

    // The library's functions that are called here.
#define PB_CALLS(X)                                                                                          \
    X(pb_tensor_release)                                                                                     \
    X(pb_tensor_interface)                                                                                   \
    X(pb_qk_norm_rope)                                                                                       \
    X(pb_qk_norm_rope_backward)                                                                              \
    X(pb_paged_attention)                                                                                    \
    X(pb_paged_attention_scored)                                                                             \
    X(pb_kv_evict)
#define PB_POINTER(name) decltype(&::name) name = nullptr;
    struct {
        PB_CALLS(PB_POINTER)
    } native;
#undef PB_POINTER
    bool g_connected = false;
    PyObject* g_load = nullptr; // loads the library and connects it

    PyObject* g_tensor_type = nullptr; // api.Tensor, the type of results
    PyObject* g_realise = nullptr;     // realises an expression
    PyObject* g_check = nullptr;       // raises what a status means

    struct handle_object {
        PyObject_HEAD
        pb_tensor* tensor;
        PyObject* face; // __cuda_array_interface__, once asked for
    };

    void release(pb_tensor* t) {
        if (t == nullptr || !g_connected) return; // a tensor exists only once the library does
        Py_BEGIN_ALLOW_THREADS // it may have to wait for other streams' readers
        native.pb_tensor_release(t);
        Py_END_ALLOW_THREADS
    }

    // Whether the library is there; loads it, or sets the exception.
    bool ready() {
        if (g_connected) return true;
        PyObject* r = g_load == nullptr ? nullptr : PyObject_CallNoArgs(g_load);
        Py_XDECREF(r);
        if (g_connected) return true;
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ImportError, "the native library is not connected");
        return false;
    }

    void handle_dealloc(PyObject* self) {
        auto* h = reinterpret_cast<handle_object*>(self);
        release(h->tensor);
        Py_XDECREF(h->face);
        Py_TYPE(self)->tp_free(self);
    }

    int handle_init(PyObject* self, PyObject* args, PyObject*) {
        PyObject* value = nullptr;
        if (!PyArg_ParseTuple(args, "O", &value)) return -1;
        void* p = value == Py_None ? nullptr : PyLong_AsVoidPtr(value);
        if (p == nullptr && PyErr_Occurred()) return -1;
        auto* h = reinterpret_cast<handle_object*>(self);
        release(h->tensor);
        Py_CLEAR(h->face);
        h->tensor = static_cast<pb_tensor*>(p);
        return 0;
    }

    // For ctypes: an int, or None.
    PyObject* handle_address(PyObject* self, void*) {
        auto* h = reinterpret_cast<handle_object*>(self);
        if (h->tensor == nullptr) Py_RETURN_NONE;
        return PyLong_FromVoidPtr(h->tensor);
    }

    // True when `status` is PB_OK; else sets the exception that it means.
    bool checked(int status) {
        if (status == PB_OK) return true;
        PyObject* r = PyObject_CallFunction(g_check, "i", status);
        if (r != nullptr) {
            Py_DECREF(r);
            PyErr_SetString(PyExc_RuntimeError, "unknown status");
        }
        return false;
    }

    // A call of the library that returns a status, without the interpreter's lock.
    template <typename F>
    bool call(F&& f) {
        if (!ready()) return false;
        int status = 0;
        Py_BEGIN_ALLOW_THREADS // a first call compiles its kernel
        status = f();
        Py_END_ALLOW_THREADS
        return checked(status);
    }

    // The address of a realised tensor's values stays what it is once it was
    // handed out, so consumers that ask twice cost one call.
    PyObject* handle_interface(PyObject* self, void*) {
        auto* h = reinterpret_cast<handle_object*>(self);
        if (h->face == nullptr) {
            int64_t v[19];
            pb_tensor* t = h->tensor;
            // A lazy tensor is realised, which may compile its kernel.
            if (!call([&] { return native.pb_tensor_interface(t, v, 19); })) return nullptr;
            PyObject* shape = PyTuple_New(static_cast<Py_ssize_t>(v[0]));
            if (shape == nullptr) return nullptr;
            for (int64_t i = 0; i < v[0]; ++i) PyTuple_SET_ITEM(shape, i, PyLong_FromLongLong(v[3 + i]));
            PyObject* face = Py_BuildValue("{s:N,s:s,s:(KO),s:i,s:K}", "shape", shape, "typestr", "<f4", "data",
                                           static_cast<unsigned long long>(v[1]), Py_False, "version", 3, "stream",
                                           static_cast<unsigned long long>(v[2]));
            if (h->face == nullptr)
                h->face = face;
            else
                Py_XDECREF(face); // another thread was first
        }
        return Py_XNewRef(h->face);
    }

    PyGetSetDef handle_getset[] = {
        {"_h", handle_address, nullptr, "the native handle's address", nullptr},
        {"__cuda_array_interface__", handle_interface, nullptr,
         "The values in place, for another library on the same GPU (as device_data(): a raw handle, so a consumer "
         "that does not order its work behind `stream` calls synchronize() first).",
         nullptr},
        {nullptr, nullptr, nullptr, nullptr, nullptr},
    };

    PyTypeObject handle_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

    PyObject* wrap(pb_tensor* t) {
        auto* type = reinterpret_cast<PyTypeObject*>(g_tensor_type);
        PyObject* self = type->tp_alloc(type, 0);
        if (self == nullptr) {
            release(t);
            return nullptr;
        }
        reinterpret_cast<handle_object*>(self)->tensor = t;
        return self;
    }

    template <size_t N>
    PyObject* wrap_all(const std::array<pb_tensor*, N>& t) {
        PyObject* out = PyTuple_New(N);
        bool good = out != nullptr;
        for (size_t i = 0; i < N; ++i) {
            if (!good) {
                release(t[i]);
                continue;
            }
            PyObject* x = wrap(t[i]);
            good = x != nullptr;
            if (good) PyTuple_SET_ITEM(out, static_cast<Py_ssize_t>(i), x);
        }
        if (good) return out;
        Py_XDECREF(out);
        return nullptr;
    }

    // An operator's tensor arguments; expressions are realised and kept.
    struct tensors {
        std::array<pb_tensor*, 9> value{};
        std::array<PyObject*, 9> kept{};
        ~tensors() {
            for (PyObject* k : kept) Py_XDECREF(k);
        }
        bool take(PyObject* const* args, size_t count) {
            for (size_t i = 0; i < count; ++i) {
                PyObject* x = args[i];
                if (!PyObject_TypeCheck(x, &handle_type)) {
                    kept[i] = PyObject_CallOneArg(g_realise, x);
                    if (kept[i] == nullptr) return false;
                    x = kept[i];
                    if (!PyObject_TypeCheck(x, &handle_type)) {
                        PyErr_SetString(PyExc_TypeError, "expected a tensor");
                        return false;
                    }
                }
                value[i] = reinterpret_cast<handle_object*>(x)->tensor;
            }
            return true;
        }
    };

    bool expect(Py_ssize_t given, Py_ssize_t wanted) {
        if (given == wanted) return true;
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, given);
        return false;
    }

    // Batch handles and sizes arrive as ints.
    bool integer(PyObject* x, int64_t& out) {
        out = PyLong_AsLongLong(x);
        return !(out == -1 && PyErr_Occurred());
    }
    bool number(PyObject* x, float& out) {
        const double v = PyFloat_AsDouble(x);
        out = static_cast<float>(v);
        return !(v == -1.0 && PyErr_Occurred());
    }

    PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
        tensors t;
        float eps = 0;
        std::array<pb_tensor*, 2> out{};
        if (!expect(n, 9) || !t.take(args, 7) || !number(args[7], eps)) return nullptr;
        const int interleaved = PyObject_IsTrue(args[8]);
        if (interleaved < 0) return nullptr;
        const auto& v = t.value;
        if (!call([&] {
                return native.pb_qk_norm_rope(v[0], v[1], v[2], v[3], v[4], v[5], v[6], eps, interleaved, &out[0], &out[1]);
            }))
            return nullptr;
        return wrap_all(out);
    }

    PyObject* qk_norm_rope_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
        tensors t;
        float eps = 0;
        std::array<pb_tensor*, 4> out{};
        if (!expect(n, 11) || !t.take(args, 9) || !number(args[9], eps)) return nullptr;
        const int interleaved = PyObject_IsTrue(args[10]);
        if (interleaved < 0) return nullptr;
        const auto& v = t.value;
        if (!call([&] {
                return native.pb_qk_norm_rope_backward(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], eps, interleaved,
                                                out.data());
            }))
            return nullptr;
        return wrap_all(out);
    }

    // (q, batch, scale)
    PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
        tensors t;
        int64_t batch = 0;
        float scale = 0;
        pb_tensor* out = nullptr;
        if (!expect(n, 3) || !t.take(args, 1) || !integer(args[1], batch) || !number(args[2], scale)) return nullptr;
        if (!call([&] { return native.pb_paged_attention(t.value[0], reinterpret_cast<pb_kv_batch*>(batch), scale, &out); }))
            return nullptr;
        return wrap(out);
    }

    // (q, batch, scores or None, scale)
    PyObject* paged_attention_scored(PyObject*, PyObject* const* args, Py_ssize_t n) {
        tensors t, scores;
        int64_t batch = 0;
        float scale = 0;
        std::array<pb_tensor*, 2> out{};
        if (!expect(n, 4) || !t.take(args, 1) || !integer(args[1], batch) ||
            (args[2] != Py_None && !scores.take(args + 2, 1)) || !number(args[3], scale))
            return nullptr;
        if (!call([&] {
                return native.pb_paged_attention_scored(t.value[0], reinterpret_cast<pb_kv_batch*>(batch), scores.value[0],
                                                 scale, &out[0], &out[1]);
            }))
            return nullptr;
        return wrap_all(out);
    }

    // (batch, scores, positions or None, budget, recent, sinks)
    PyObject* kv_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
        tensors scores, places;
        int64_t batch = 0, budget = 0, recent = 0, sinks = 0;
        std::array<pb_tensor*, 2> out{};
        if (!expect(n, 6) || !integer(args[0], batch) || !scores.take(args + 1, 1) ||
            (args[2] != Py_None && !places.take(args + 2, 1)) || !integer(args[3], budget) ||
            !integer(args[4], recent) || !integer(args[5], sinks))
            return nullptr;
        if (!call([&] {
                return native.pb_kv_evict(reinterpret_cast<pb_kv_batch*>(batch), scores.value[0], places.value[0], budget,
                                   recent, sinks, &out[0], &out[1]);
            }))
            return nullptr;
        return wrap_all(out);
    }

    // (path of the library, loaded)
    PyObject* connect(PyObject*, PyObject* const* args, Py_ssize_t n) {
        if (!expect(n, 1)) return nullptr;
        const char* path = PyUnicode_AsUTF8(args[0]);
        if (path == nullptr) return nullptr;
        void* library = dlopen(path, RTLD_NOW | RTLD_LOCAL);
        if (library == nullptr) {
            PyErr_SetString(PyExc_ImportError, dlerror());
            return nullptr;
        }
#define PB_FIND(name)                                                                                        \
    native.name = reinterpret_cast<decltype(native.name)>(dlsym(library, #name));                            \
    if (native.name == nullptr) {                                                                            \
        PyErr_SetString(PyExc_ImportError, "the native library lacks " #name);                               \
        return nullptr;                                                                                      \
    }
        PB_CALLS(PB_FIND)
#undef PB_FIND
        g_connected = true;
        Py_RETURN_NONE;
    }

    // (tensor type, realise, check, load)
    PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
        if (!expect(n, 4)) return nullptr;
        if (!PyType_Check(args[0]) || !PyType_IsSubtype(reinterpret_cast<PyTypeObject*>(args[0]), &handle_type)) {
            PyErr_SetString(PyExc_TypeError, "the tensor type must derive from Handle");
            return nullptr;
        }
        Py_XSETREF(g_tensor_type, Py_NewRef(args[0]));
        Py_XSETREF(g_realise, Py_NewRef(args[1]));
        Py_XSETREF(g_check, Py_NewRef(args[2]));
        Py_XSETREF(g_load, Py_NewRef(args[3]));
        Py_RETURN_NONE;
    }

    PyMethodDef method(const char* name, PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
        return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr};
    }
    PyMethodDef methods[] = {
        method("qk_norm_rope", qk_norm_rope),
        method("qk_norm_rope_backward", qk_norm_rope_backward),
        method("paged_attention", paged_attention),
        method("paged_attention_scored", paged_attention_scored),
        method("kv_evict", kv_evict),
        method("bind", bind),
        method("connect", connect),
        {nullptr, nullptr, 0, nullptr},
    };

    PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__binding(void) {
    handle_type.tp_name = "porch_b200._binding.Handle";
    handle_type.tp_basicsize = sizeof(handle_object);
    handle_type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE;
    handle_type.tp_doc = "A native tensor handle, released with the object.";
    handle_type.tp_new = PyType_GenericNew;
    handle_type.tp_init = handle_init;
    handle_type.tp_dealloc = handle_dealloc;
    handle_type.tp_getset = handle_getset;
    if (PyType_Ready(&handle_type) < 0) return nullptr;
    PyObject* m = PyModule_Create(&module);
    if (m == nullptr) return nullptr;
    if (PyModule_AddObjectRef(m, "Handle", reinterpret_cast<PyObject*>(&handle_type)) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}

// Python binding of the paged cache's operators on arrays of another framework
// (metellus_b200.api.paged): a decode step calls them once a layer, and the ctypes
// structures that the other entry points are called with cost more than a small kernel.
//
// Arrays are read, and new ones made, through DLPack's C exchange API, which their type
// offers as `__dlpack_c_exchange_api__`: pointers, shapes and strides without temporary
// objects, the type's own allocator and its current stream. The structures below are that
// interface's, version 1.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "../../include/metellus_b200.h"

namespace {

struct DLDevice {
    int32_t type, id;
};
struct DLDataType {
    uint8_t code, bits;
    uint16_t lanes;
};
struct DLTensor {
    void* data;
    DLDevice device;
    int32_t ndim;
    DLDataType dtype;
    int64_t* shape;
    int64_t* strides;
    uint64_t byte_offset;
};
struct DLPackVersion {
    uint32_t major, minor;
};
struct DLManagedTensorVersioned {
    DLPackVersion version;
    void* manager_ctx;
    void (*deleter)(DLManagedTensorVersioned*);
    uint64_t flags;
    DLTensor dl_tensor;
};
struct DLPackExchangeAPI {
    DLPackVersion version;
    void* prev_api;
    int (*managed_tensor_allocator)(DLTensor* prototype, DLManagedTensorVersioned** out, void* error_ctx,
                                    void (*set_error)(void* error_ctx, const char* kind, const char* message));
    int (*managed_tensor_from_py_object_no_sync)(void* object, DLManagedTensorVersioned** out);
    int (*managed_tensor_to_py_object_no_sync)(DLManagedTensorVersioned* tensor, void** out);
    int (*dltensor_from_py_object_no_sync)(void* object, DLTensor* out);
    int (*current_work_stream)(int32_t device_type, int32_t device_id, void** out);
};

constexpr int kCuda = 2;
enum { kInt = 0, kFloat = 2, kBfloat = 4, kFloat8E4M3fn = 10 };

PyObject* g_api_name;       // "__dlpack_c_exchange_api__"
PyObject* g_requires_grad;  // "requires_grad"

const DLPackExchangeAPI* api_of(PyObject* x, const char* name) {
    // a call's arrays are nearly always of one type
    static PyTypeObject* last_type = nullptr;
    static const DLPackExchangeAPI* last_api = nullptr;
    if (Py_TYPE(x) == last_type) return last_api;
    PyObject* capsule = PyObject_GetAttr((PyObject*)Py_TYPE(x), g_api_name);
    const DLPackExchangeAPI* api = nullptr;
    if (capsule && PyCapsule_IsValid(capsule, "dlpack_exchange_api"))
        api = (const DLPackExchangeAPI*)PyCapsule_GetPointer(capsule, "dlpack_exchange_api");
    Py_XDECREF(capsule);
    PyErr_Clear();
    if (!api || api->version.major != 1) {
        if (PyObject_HasAttrString(x, "__dlpack__"))
            PyErr_Format(PyExc_TypeError, "%s is a %s, whose type does not offer DLPack's C exchange API, version 1 "
                         "(__dlpack_c_exchange_api__; torch tensors do as of torch 2.11, perhaps earlier)", name, Py_TYPE(x)->tp_name);
        else
            PyErr_Format(PyExc_TypeError, "%s must be a CUDA tensor, not %s", name, Py_TYPE(x)->tp_name);
        return nullptr;
    }
    Py_INCREF(Py_TYPE(x));  // the type stays, and its API with it
    Py_XDECREF(last_type);
    last_type = Py_TYPE(x);
    last_api = api;
    return api;
}

int dtype_of(DLDataType t) {
    if (t.lanes != 1) return -1;
    if (t.code == kFloat) return t.bits == 32 ? MT_F32 : t.bits == 16 ? MT_F16 : -1;
    if (t.code == kBfloat && t.bits == 16) return MT_BF16;
    if (t.code == kFloat8E4M3fn && t.bits == 8) return MT_E4M3;
    if (t.code == kInt) return t.bits == 8 ? MT_I8 : t.bits == 32 ? MT_I32 : t.bits == 64 ? MT_I64 : -1;
    return -1;
}

DLDataType dl_type(int dtype) {
    switch (dtype) {
        case MT_F16: return {kFloat, 16, 1};
        case MT_BF16: return {kBfloat, 16, 1};
        default: return {kFloat, 32, 1};
    }
}

// The call's device and the arrays' interface, from its first array.
struct Call {
    const DLPackExchangeAPI* api = nullptr;
    DLDevice device{0, -1};

    // `x` as the C entry points take it; checks that it is on the call's device.
    bool array(PyObject* x, const char* name, mt_array* out) {
        const DLPackExchangeAPI* its = api_of(x, name);
        if (!its) return false;
        DLTensor t;
        if (its->dltensor_from_py_object_no_sync(x, &t)) return false;
        if (!api) {
            api = its;
            device = t.device;
        }
        if (t.device.type != kCuda || t.device.type != device.type || t.device.id != device.id) {
            PyErr_Format(PyExc_ValueError, "%s must be on a CUDA device, and every array on the same one", name);
            return false;
        }
        const int dtype = dtype_of(t.dtype);
        if (dtype < 0) {
            PyErr_Format(PyExc_ValueError, "%s has a type that the paged cache's operators do not take", name);
            return false;
        }
        if (t.ndim > 4) {
            PyErr_Format(PyExc_ValueError, "%s has %d dimensions", name, (int)t.ndim);
            return false;
        }
        out->ptr = (char*)t.data + t.byte_offset;
        out->dtype = dtype;
        out->ndim = t.ndim;
        int64_t packed = 1;
        for (int i = t.ndim - 1; i >= 0; --i) {
            out->shape[i] = t.shape[i];
            out->strides[i] = t.strides ? t.strides[i] : packed;
            packed *= t.shape[i];
        }
        return true;
    }

    // A new packed array.
    DLManagedTensorVersioned* make(int dtype, int ndim, const int64_t* shape) {
        DLTensor like{};
        int64_t extents[4];
        memcpy(extents, shape, sizeof(int64_t) * ndim);
        like.device = device;
        like.ndim = ndim;
        like.dtype = dl_type(dtype);
        like.shape = extents;
        DLManagedTensorVersioned* out = nullptr;
        auto set_error = [](void*, const char*, const char* message) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, message);
        };
        if (api->managed_tensor_allocator(&like, &out, nullptr, set_error) && !PyErr_Occurred())
            PyErr_SetString(PyExc_RuntimeError, "the array could not be allocated");
        return PyErr_Occurred() ? nullptr : out;
    }
    PyObject* object(DLManagedTensorVersioned* t) {
        void* out = nullptr;
        return api->managed_tensor_to_py_object_no_sync(t, &out) ? nullptr : (PyObject*)out;
    }
    PyObject* make_object(int dtype, int ndim, const int64_t* shape) {
        DLManagedTensorVersioned* t = make(dtype, ndim, shape);
        return t ? object(t) : nullptr;
    }

    // The framework's current stream; its default stream by the handle that does not mean this
    // library's own.
    bool stream(void** out) {
        *out = nullptr;
        if (api->current_work_stream(device.type, device.id, out)) return false;
        if (!*out) *out = (void*)1;  // cudaStreamLegacy
        return true;
    }
};

bool check(int rc) {
    if (rc == 0) return true;
    char message[2048];
    mt_last_error(message, sizeof message);
    PyErr_SetString(rc == 2 ? PyExc_ValueError : PyExc_RuntimeError, message);
    return false;
}

// What the binding asks of a framework that tracks gradients, if one is loaded: its tensors' type,
// whether it is tracking, a function that counts a tensor's writes, and, while forward-mode derivatives
// are computed (else None), one that takes a tensor and its tangent apart.
struct Autograd {
    PyObject *type, *grad_enabled, *count_write, *unpack_dual;
    bool read(PyObject* x) {
        type = nullptr;
        return x == Py_None || PyArg_ParseTuple(x, "OOOO", &type, &grad_enabled, &count_write, &unpack_dual);
    }

    // The operators have no derivatives: refuse to drop one silently. `grad_enabled` is asked only
    // where an array requires a gradient.
    bool allows(PyObject* x, const char* name) {
        if (!type || x == Py_None || !PyObject_TypeCheck(x, (PyTypeObject*)type)) return true;
        if (unpack_dual != Py_None) {
            PyObject* pair = PyObject_CallOneArg(unpack_dual, x);
            PyObject* tangent = pair ? PySequence_GetItem(pair, 1) : nullptr;
            Py_XDECREF(pair);
            if (!tangent) return false;
            Py_DECREF(tangent);
            if (tangent != Py_None) {
                PyErr_Format(PyExc_ValueError, "%s has a tangent; the paged cache's operators have no derivatives", name);
                return false;
            }
        }
        PyObject* r = PyObject_GetAttr(x, g_requires_grad);
        if (!r) return false;
        const int requires_grad = PyObject_IsTrue(r);
        Py_DECREF(r);
        if (requires_grad <= 0) return requires_grad == 0;
        PyObject* e = PyObject_CallNoArgs(grad_enabled);
        if (!e) return false;
        const int on = PyObject_IsTrue(e);
        Py_DECREF(e);
        if (on > 0)
            PyErr_Format(PyExc_ValueError,
                         "%s requires a gradient; the paged cache's operators have none (use torch.no_grad() or detach it)", name);
        return on == 0;
    }
    bool allows(PyObject* const* x, std::initializer_list<const char*> names) {
        for (const char* name : names)
            if (!allows(*x++, name)) return false;
        return true;
    }

    // A tensor that something keeps for its own backward pass must not change behind its back.
    // (One call for all of them: a write then takes 3.4 us on the host, 3.05 uncounted, 3.7 with a call each.)
    bool written(PyObject* const* x, int n) {
        if (!type) return true;
        PyObject* all = PyList_New(0);
        for (int i = 0; all && i < n; ++i)
            if (PyObject_TypeCheck(x[i], (PyTypeObject*)type) && PyList_Append(all, x[i])) Py_CLEAR(all);
        if (!all) return false;
        PyObject* r = PyList_GET_SIZE(all) ? PyObject_CallOneArg(count_write, all) : Py_NewRef(Py_None);
        Py_DECREF(all);
        Py_XDECREF(r);
        return r != nullptr;
    }
};

bool read_cache(Call& call, PyObject* const* args, mt_paged_cache* c) {
    memset(c, 0, sizeof *c);
    return call.array(args[0], "k_cache", &c->k) && call.array(args[1], "v_cache", &c->v) &&
           (args[2] == Py_None || call.array(args[2], "k_scale", &c->k_scale)) &&
           (args[3] == Py_None || call.array(args[3], "v_scale", &c->v_scale));
}

bool count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd are wanted", n, want);
    return false;
}

// (autograd, k, v, k_cache, v_cache, k_scale, v_scale, slots)
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!count(n, 8)) return nullptr;
    Call call;
    Autograd autograd;
    if (!autograd.read(args[0])) return nullptr;
    mt_array k, v, slots;
    mt_paged_cache c;
    void* stream;
    if (!call.array(args[1], "k", &k) || !call.array(args[2], "v", &v) || !read_cache(call, args + 3, &c) ||
        !call.array(args[7], "slots", &slots))
        return nullptr;
    if (!autograd.allows(args + 1, {"k", "v", "k_cache", "v_cache", "k_scale", "v_scale"})) return nullptr;
    if (!call.stream(&stream) || !check(mt_cache_write(call.device.id, &k, &v, &c, &slots, stream)) ||
        !autograd.written(args + 3, 4))
        return nullptr;
    Py_RETURN_NONE;
}

// (autograd, k_cache, v_cache, k_scale, v_scale, slots, dtype code or -1, out_k, out_v) -> (k, v)
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!count(n, 9)) return nullptr;
    Call call;
    Autograd autograd;
    if (!autograd.read(args[0])) return nullptr;
    mt_array k, v, slots;
    mt_paged_cache c;
    void* stream;
    if (!read_cache(call, args + 1, &c) || !call.array(args[5], "slots", &slots)) return nullptr;
    if (!autograd.allows(args + 1, {"k_cache", "v_cache", "k_scale", "v_scale"}) || !autograd.allows(args + 7, {"out[0]", "out[1]"}))
        return nullptr;
    long dtype = PyLong_AsLong(args[6]);
    if (dtype == -1 && PyErr_Occurred()) return nullptr;
    PyObject *ok = args[7], *ov = args[8];
    if (ok == Py_None) {
        if (c.k.ndim != 4 || slots.ndim != 1) {
            PyErr_SetString(PyExc_ValueError, "cache_read: k_cache must have 4 dimensions and slots 1");
            return nullptr;
        }
        if (dtype < 0) dtype = c.k.dtype <= MT_BF16 ? c.k.dtype : MT_F32;
        const int64_t shape[3] = {slots.shape[0], c.k.shape[2], c.k.shape[3]};
        ok = call.make_object((int)dtype, 3, shape);
        ov = ok ? call.make_object((int)dtype, 3, shape) : nullptr;
    } else {
        Py_INCREF(ok);
        Py_INCREF(ov);
    }
    PyObject* result = nullptr;
    if (ok && ov && call.array(ok, "out[0]", &k) && call.array(ov, "out[1]", &v) && call.stream(&stream) &&
        check(mt_cache_read(call.device.id, &c, &slots, &k, &v, stream)) && autograd.written(args + 7, 2))
        result = PyTuple_Pack(2, ok, ov);
    Py_XDECREF(ok);
    Py_XDECREF(ov);
    return result;
}

// (autograd, q, k_cache, v_cache, k_scale, v_scale, tables, lengths, scale or None, window, out or None, return_lse)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!count(n, 12)) return nullptr;
    Call call;
    Autograd autograd;
    if (!autograd.read(args[0])) return nullptr;
    mt_array q, tables, lengths, out, lse;
    mt_paged_cache c;
    void* stream;
    if (!call.array(args[1], "q", &q) || !read_cache(call, args + 2, &c) || !call.array(args[6], "tables", &tables) ||
        !call.array(args[7], "lengths", &lengths))
        return nullptr;
    if (!autograd.allows(args + 1, {"q", "k_cache", "v_cache", "k_scale", "v_scale"}) || !autograd.allows(args[10], "out"))
        return nullptr;
    if (q.ndim != 3) return PyErr_Format(PyExc_ValueError, "paged_attention: q must have 3 dimensions, not %d", q.ndim);
    double scale;
    if (args[8] == Py_None) {
        scale = q.shape[2] > 0 ? 1.0 / __builtin_sqrt((double)q.shape[2]) : 1.0;
    } else {
        scale = PyFloat_AsDouble(args[8]);
        if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    }
    const int64_t window = PyLong_AsLongLong(args[9]);
    if (window == -1 && PyErr_Occurred()) return nullptr;
    const int with_lse = PyObject_IsTrue(args[11]);
    if (with_lse < 0) return nullptr;
    uint64_t bytes = 0;
    if (!check(mt_paged_attention_workspace(call.device.id, &q, &c, &tables, window, &bytes))) return nullptr;

    PyObject *result = nullptr, *o = args[10], *z = nullptr;
    DLManagedTensorVersioned* space = nullptr;
    if (o == Py_None) o = call.make_object(q.dtype, 3, q.shape);
    else Py_INCREF(o);
    if (!o || !call.array(o, "out", &out)) goto done;
    if (with_lse) {
        z = call.make_object(MT_F32, 2, q.shape);
        if (!z || !call.array(z, "lse", &lse)) goto done;
    }
    if (bytes) {
        const int64_t words = (int64_t)((bytes + 3) / 4);
        space = call.make(MT_F32, 1, &words);
        if (!space) goto done;
    }
    if (!call.stream(&stream) ||
        !check(mt_paged_attention(call.device.id, &q, &c, &tables, &lengths, &out, with_lse ? &lse : nullptr, scale, window,
                                  space ? (char*)space->dl_tensor.data + space->dl_tensor.byte_offset : nullptr, bytes,
                                  stream)) ||
        !autograd.written(args + 10, 1))
        goto done;
    result = with_lse ? PyTuple_Pack(2, o, z) : Py_NewRef(o);
done:
    if (space) space->deleter(space);  // the allocator hands it out again in the stream's order
    Py_XDECREF(o);
    Py_XDECREF(z);
    return result;
}

PyMethodDef methods[] = {
    {"cache_write", (PyCFunction)(void (*)(void))cache_write, METH_FASTCALL, nullptr},
    {"cache_read", (PyCFunction)(void (*)(void))cache_read, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_metellus_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__metellus_paged(void) {
    g_api_name = PyUnicode_InternFromString("__dlpack_c_exchange_api__");
    g_requires_grad = PyUnicode_InternFromString("requires_grad");
    if (!g_api_name || !g_requires_grad) return nullptr;
    return PyModule_Create(&module);
}

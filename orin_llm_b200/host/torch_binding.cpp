// Calls of the 4-bit cache for torch callers (module _q4_binding): checks the tensors and forwards to the C ABI.
//
// A decode step over a short cache is 6 to 10 microseconds of GPU time, and most of its calls in a program are of that kind;
// checking six tensors in Python and passing eighteen arguments through ctypes costs as much again.  Here the same checks are
// a few loads each.  The C ABI stays the product: nothing is launched or allocated in this file.
#include <Python.h>

#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/orin_attn_b200.h"

namespace {

struct Refused {};                       // a Python exception is set
struct Code { int rc; };                 // a status of the C ABI

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw Refused();
}

int to_int(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    if (v < -2147483648LL || v > 2147483647LL) refuse(PyExc_ValueError, "%lld does not fit in an int", v);
    return (int)v;
}

float to_float(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return (float)v;
}

const at::Tensor& tensor(const char* name, PyObject* o) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: a tensor is needed, got %s", name, Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

const char* name_of(at::ScalarType t) {
    return t == at::kFloat ? "float32" : t == at::kHalf ? "float16" : t == at::kByte ? "uint8" : t == at::kInt ? "int32" : t == at::kChar ? "int8" : c10::toString(t);
}

// Address of a contiguous tensor of that type with at least `numel` elements on CUDA device `dev`.
void* address(const char* name, PyObject* o, at::ScalarType type, long long numel, int dev) {
    const at::Tensor& t = tensor(name, o);
    if (t.scalar_type() != type || t.numel() < numel || !t.is_contiguous())
        refuse(PyExc_ValueError, "%s: a contiguous %s tensor of at least %lld elements is needed, got %s of %lld%s", name, name_of(type), numel,
               name_of(t.scalar_type()), (long long)t.numel(), t.is_contiguous() ? "" : ", not contiguous");
    if (t.get_device() != dev) refuse(PyExc_ValueError, "%s: on %s, the cache on device %d", name, t.device().str().c_str(), dev);
    return t.data_ptr();
}

struct Cache { uint8_t* ptr; int dev; };

// A cache of `layers` layers on the current device.
Cache cache_of(PyObject* o, int layers, int n_kv, int head_dim, int n_ctx) {
    const at::Tensor& t = tensor("cache", o);
    const size_t bytes = oattn_kv_q4_bytes(n_kv, head_dim, n_ctx);
    if (bytes == 0) throw Code{OATTN_ERR_UNSUPPORTED};
    Cache c;
    c.dev = t.is_cuda() ? (int)t.get_device() : -1;
    c.ptr = static_cast<uint8_t*>(address("cache", o, at::kByte, (long long)bytes * (layers > 0 ? layers : 1), c.dev));
    if (c.dev < 0 || c.dev != c10::cuda::current_device()) refuse(PyExc_ValueError, "cache: on %s, not on the current CUDA device", t.device().str().c_str());
    return c;
}

// The stream given to ops.set_stream, or torch's current one.
void* stream_of(PyObject* o, int dev) {
    if (o == Py_None) return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    void* s = PyLong_AsVoidPtr(o);
    if (!s && PyErr_Occurred()) throw Refused();
    return s;
}

const oattn_rope_params* rope_of(PyObject* o, oattn_rope_params& r, int dev) {
    if (o == Py_None) return nullptr;
    PyObject* f[4];
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse(PyExc_TypeError, "rope: (rope_type, n_rot, theta, freq_factors) is needed");
    for (int i = 0; i < 4; ++i) f[i] = PyTuple_GET_ITEM(o, i);
    r.rope_type = to_int(f[0]);
    r.n_rot = to_int(f[1]);
    r.theta = to_float(f[2]);
    r.freq_factors = f[3] == Py_None ? nullptr : static_cast<const float*>(address("freq_factors", f[3], at::kFloat, r.n_rot / 2, dev));
    return &r;
}

// Device of the cache, whatever it is: what comes with it is checked against that before it is itself (cache_of).
int device_of(PyObject* o) { return (int)tensor("cache", o).get_device(); }

// The extras of the attention calls, a dict of the C struct's members, for `batch` tokens.
const oattn_ext* ext_of(PyObject* o, oattn_ext& e, int n_head, int n_kv, int hd, int batch, int dev) {
    if (o == Py_None) return nullptr;
    if (!PyDict_Check(o)) refuse(PyExc_TypeError, "ext: a dict is needed, got %s", Py_TYPE(o)->tp_name);
    if (PyDict_GET_SIZE(o) == 0) return nullptr;
    e = oattn_ext();
    Py_ssize_t known = 0;
    auto get = [&](const char* name) {
        PyObject* v = PyDict_GetItemString(o, name);         // borrowed
        if (v) ++known;
        return v && v != Py_None ? v : nullptr;
    };
    auto member = [&](const char* name, at::ScalarType type, long long numel) {
        PyObject* v = get(name);
        return v ? address(name, v, type, numel, dev) : nullptr;
    };
    const long long nq = (long long)n_head * hd, nk = (long long)n_kv * hd;
    e.bias_q = static_cast<const float*>(member("bias_q", at::kFloat, nq));
    e.bias_k = static_cast<const float*>(member("bias_k", at::kFloat, nk));
    e.bias_v = static_cast<const float*>(member("bias_v", at::kFloat, nk));
    e.norm_q = static_cast<const float*>(member("norm_q", at::kFloat, hd));
    e.norm_k = static_cast<const float*>(member("norm_k", at::kFloat, hd));
    e.out_qs = static_cast<int8_t*>(member("out_qs", at::kChar, nq));
    e.out_scales = static_cast<float*>(member("out_scales", at::kFloat, nq / 32));
    e.out_mmq = member("out_mmq", at::kByte, (long long)batch * n_head * 144);       // one block of 128 values per token and head
    if (PyObject* v = get("norm_eps")) e.norm_eps = to_float(v);
    if (PyObject* v = get("out_mmq_ds4")) {
        e.out_mmq_ds4 = PyObject_IsTrue(v);
        if (e.out_mmq_ds4 < 0) throw Refused();
    }
    if (known != PyDict_GET_SIZE(o)) refuse(PyExc_ValueError, "unknown extension keys in %R", o);
    return &e;
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    try {
        if (n != want) refuse(PyExc_TypeError, "%zd arguments are needed, got %zd", want, n);
        return PyLong_FromLong(f());
    } catch (const Code& c) {
        return PyLong_FromLong(c.rc);
    } catch (const Refused&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// (cache, k, v, heads, head_dim, n_ctx, pos_base, batch, d_pos | None, stream | None)
PyObject* kv_store_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&] {
        const int heads = to_int(a[3]), hd = to_int(a[4]), n_ctx = to_int(a[5]), base = to_int(a[6]), batch = to_int(a[7]);
        const Cache c = cache_of(a[0], 1, heads, hd, n_ctx);
        const long long numel = (long long)batch * heads * hd;
        const float* k = static_cast<const float*>(address("k", a[1], at::kFloat, numel, c.dev));
        const float* v = static_cast<const float*>(address("v", a[2], at::kFloat, numel, c.dev));
        const int* d_pos = a[8] == Py_None ? nullptr : static_cast<const int*>(address("d_pos", a[8], at::kInt, 1, c.dev));
        return oattn_kv_store_q4(c.ptr, k, v, heads, hd, n_ctx, base, batch, d_pos, stream_of(a[9], c.dev));
    });
}

// (cache, kc, vc, heads, head_dim, n_ctx, row_base, rows, dst_ctx, dst_base, stream | None)
PyObject* kv_load_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&] {
        const int heads = to_int(a[3]), hd = to_int(a[4]), n_ctx = to_int(a[5]), dst_ctx = to_int(a[8]);
        const Cache c = cache_of(a[0], 1, heads, hd, n_ctx);
        const long long numel = (long long)heads * dst_ctx * hd;
        uint16_t* kc = static_cast<uint16_t*>(address("kc", a[1], at::kHalf, numel, c.dev));
        uint16_t* vc = static_cast<uint16_t*>(address("vc", a[2], at::kHalf, numel, c.dev));
        return oattn_kv_load_q4(c.ptr, kc, vc, heads, hd, n_ctx, to_int(a[6]), to_int(a[7]), dst_ctx, to_int(a[9]), stream_of(a[10], c.dev));
    });
}

// (cache, n_layer, n_kv, head_dim, n_ctx, n_keep, shift, stream | None)
PyObject* kv_shift_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const int layers = to_int(a[1]), n_kv = to_int(a[2]), hd = to_int(a[3]), n_ctx = to_int(a[4]);
        const Cache c = cache_of(a[0], layers, n_kv, hd, n_ctx);
        return oattn_kv_shift_q4(c.ptr, layers, n_kv, hd, n_ctx, to_int(a[5]), to_int(a[6]), stream_of(a[7], c.dev));
    });
}

// (q, k_new, v_new, cache, out | None, n_head, n_kv, head_dim, n_ctx, d_pos, scale, fuse, rope | None, ext | None, workspace,
//  stream | None)
PyObject* decode_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 16, [&] {
        const int n_head = to_int(a[5]), n_kv = to_int(a[6]), hd = to_int(a[7]), n_ctx = to_int(a[8]), fuse = to_int(a[11]);
        oattn_ext x;
        const oattn_ext* ext = ext_of(a[13], x, n_head, n_kv, hd, 1, device_of(a[3]));
        const Cache c = cache_of(a[3], 1, n_kv, hd, n_ctx);
        const float* q = static_cast<const float*>(address("q", a[0], at::kFloat, (long long)n_head * hd, c.dev));
        const float *k = nullptr, *v = nullptr;
        if (fuse & OATTN_FUSE_KV_APPEND) {
            k = static_cast<const float*>(address("k_new", a[1], at::kFloat, (long long)n_kv * hd, c.dev));
            v = static_cast<const float*>(address("v_new", a[2], at::kFloat, (long long)n_kv * hd, c.dev));
        }
        float* out = nullptr;
        if (a[4] != Py_None || !ext || !ext->out_qs) out = static_cast<float*>(address("out", a[4], at::kFloat, (long long)n_head * hd, c.dev));
        const int* d_pos = static_cast<const int*>(address("d_pos", a[9], at::kInt, 1, c.dev));
        oattn_rope_params r;
        const oattn_rope_params* rope = rope_of(a[12], r, c.dev);
        void* ws = address("workspace", a[14], at::kByte, 0, c.dev);
        return oattn_decode_q4(q, k, v, c.ptr, out, n_head, n_kv, hd, n_ctx, d_pos, to_float(a[10]), fuse, rope, ext, ws,
                               (size_t)tensor("workspace", a[14]).numel(), stream_of(a[15], c.dev));
    });
}

// (q, k_new, v_new, cache, out | None, n_head, n_kv, head_dim, n_ctx, n_past, batch, scale, fuse, rope | None, ext | None,
//  workspace, stream | None); out: fp32 or fp16
PyObject* prefill_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 17, [&] {
        const int n_head = to_int(a[5]), n_kv = to_int(a[6]), hd = to_int(a[7]), n_ctx = to_int(a[8]), batch = to_int(a[10]), fuse = to_int(a[12]);
        oattn_ext x;
        const oattn_ext* ext = ext_of(a[14], x, n_head, n_kv, hd, batch, device_of(a[3]));
        const Cache c = cache_of(a[3], 1, n_kv, hd, n_ctx);
        const long long nq = (long long)batch * n_head * hd, nk = (long long)batch * n_kv * hd;
        const float* q = static_cast<const float*>(address("q", a[0], at::kFloat, nq, c.dev));
        const float *k = nullptr, *v = nullptr;
        if (fuse & OATTN_FUSE_KV_APPEND) {
            k = static_cast<const float*>(address("k_new", a[1], at::kFloat, nk, c.dev));
            v = static_cast<const float*>(address("v_new", a[2], at::kFloat, nk, c.dev));
        }
        float* out = nullptr;
        uint16_t* out16 = nullptr;
        if (a[4] != Py_None || !ext || !ext->out_mmq) {
            if (tensor("out", a[4]).scalar_type() == at::kHalf) out16 = static_cast<uint16_t*>(address("out", a[4], at::kHalf, nq, c.dev));
            else out = static_cast<float*>(address("out", a[4], at::kFloat, nq, c.dev));
        }
        oattn_rope_params r;
        const oattn_rope_params* rope = rope_of(a[13], r, c.dev);
        void* ws = address("workspace", a[15], at::kByte, 0, c.dev);
        return oattn_prefill_q4(q, k, v, c.ptr, out, out16, n_head, n_kv, hd, n_ctx, to_int(a[9]), batch, to_float(a[11]), fuse, rope, ext, ws,
                                (size_t)tensor("workspace", a[15]).numel(), stream_of(a[16], c.dev));
    });
}

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(kv_store_q4), ENTRY(kv_load_q4), ENTRY(kv_shift_q4), ENTRY(decode_q4), ENTRY(prefill_q4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_q4_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__q4_binding(void) { return PyModule_Create(&module); }

// The attention operators' calls from torch tensors to the C ABI: argument
// checks, strides, the current stream and the workspaces, in C++ because a
// decoding step's kernels take a few microseconds each and the same checks in
// Python took 15 to 20 per call (2 to 4 here).  A plain extension module;
// the library's entry points are handed in as addresses at import, so that it
// links against torch alone.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <map>
#include <mutex>
#include <stdexcept>
#include <string>

#include "wlq_b200.h"

namespace {

struct Entries {
    decltype(&wlq_rope_kv_write) rope_kv_write;
    decltype(&wlq_kv_read) kv_read;
    decltype(&wlq_prompt_attention) prompt_attention;
    decltype(&wlq_paged_attention_workspace_bytes) workspace_bytes;
    decltype(&wlq_paged_attention) paged_attention;
    decltype(&wlq_last_error) last_error;
} lib{};
PyObject* wlq_error = nullptr;  // the package's WLQError

// Raises RuntimeError("wlq: <function>: ...") at the Python call.
[[noreturn]] void refuse(const char* fn, const char* fmt, ...) {
    char msg[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    throw std::runtime_error(std::string("wlq: ") + fn + ": " + msg);
}
struct PyFailed {};  // a Python error is set already

std::string shape_of(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}
const char* name_of(at::ScalarType t) { return c10::toString(t); }

// One call's arguments.
struct Args {
    const char* fn;
    PyObject* const* a;
    at::Device dev{at::kCPU};
    at::ScalarType act = at::kFloat;

    const at::Tensor& tensor(int i, const char* nm) const {
        if (!THPVariable_Check(a[i])) refuse(fn, "%s must be a tensor", nm);
        return THPVariable_Unpack(a[i]);
    }
    bool none(int i) const { return a[i] == Py_None; }
    int64_t integer(int i) const {
        const long long v = PyLong_AsLongLong(a[i]);
        if (v == -1 && PyErr_Occurred()) throw PyFailed{};
        return v;
    }
    float scale(int i, int64_t D) const {
        if (none(i)) return (float)(1.0 / std::sqrt((double)D));
        const double v = PyFloat_AsDouble(a[i]);
        if (v == -1.0 && PyErr_Occurred()) throw PyFailed{};
        return (float)v;
    }
    bool truth(int i) const {
        const int v = PyObject_IsTrue(a[i]);
        if (v < 0) throw PyFailed{};
        return v != 0;
    }
    // The tensor whose device and (activation) type the others go by.
    const at::Tensor& lead(int i, const char* nm) {
        const at::Tensor& t = tensor(i, nm);
        if (!t.is_cuda()) refuse(fn, "%s must be a CUDA tensor", nm);
        act = t.scalar_type();
        if (act != at::kHalf && act != at::kBFloat16)
            refuse(fn, "activations must be float16 or bfloat16, got %s", name_of(act));
        dev = t.device();
        return t;
    }
    int dtype() const { return act == at::kHalf ? WLQ_DTYPE_F16 : WLQ_DTYPE_BF16; }
    void on(const at::Tensor& t, const char* nm, at::ScalarType type) const {
        if (t.device() != dev) refuse(fn, "%s must be on %s", nm, dev.str().c_str());
        if (t.scalar_type() != type) refuse(fn, "%s must be %s, got %s", nm, name_of(type), name_of(t.scalar_type()));
    }
    // [tokens, heads, head size] with contiguous heads; -1: any number
    const at::Tensor& heads(int i, const char* nm, int64_t T, int64_t H, int64_t D) const {
        const at::Tensor& t = tensor(i, nm);
        on(t, nm, act);
        if (t.dim() != 3 || (T >= 0 && t.size(0) != T) || (H >= 0 && t.size(1) != H) || (D >= 0 && t.size(2) != D))
            refuse(fn, "%s must be [tokens, heads, head_size] = [%lld, %lld, %lld] (-1: any), got %s", nm, (long long)T,
                   (long long)H, (long long)D, shape_of(t).c_str());
        if (t.size(2) > 1 && t.stride(2) != 1) refuse(fn, "the values of a head of %s must be contiguous", nm);
        return t;
    }
    const at::Tensor& vec(int i, const char* nm, at::ScalarType type, int64_t n = -1) const {
        const at::Tensor& t = tensor(i, nm);
        on(t, nm, type);
        if (!t.is_contiguous()) refuse(fn, "%s must be contiguous", nm);
        if (n >= 0 && t.numel() != n) refuse(fn, "%s must have %lld values, got %lld", nm, (long long)n, (long long)t.numel());
        return t;
    }
    struct Cache {
        const at::Tensor *k, *v;
        uint8_t *ke = nullptr, *ve = nullptr;
        int64_t pages, Hkv, ps, D;
    };
    Cache cache(int k, int v, int ke, int ve) const {
        Cache c;
        c.k = &tensor(k, "k_cache");
        c.v = &tensor(v, "v_cache");
        if (c.k->dim() != 4 || c.k->sizes() != c.v->sizes())
            refuse(fn, "k_cache and v_cache must be [pages, kv_heads, page_size, head_size], got %s and %s",
                   shape_of(*c.k).c_str(), shape_of(*c.v).c_str());
        if (none(ke) != none(ve)) refuse(fn, "give k_exp and v_exp, or neither");
        const at::ScalarType want = none(ke) ? act : at::kFloat8_e4m3fn;
        for (const auto& [t, nm] : {std::pair<const at::Tensor*, const char*>{c.k, "k_cache"}, {c.v, "v_cache"}}) {
            if (t->scalar_type() != want)
                refuse(fn, "%s must be %s, got %s%s", nm, name_of(want), name_of(t->scalar_type()),
                       none(ke) ? " (an 8-bit cache needs k_exp and v_exp)" : "");
            if (t->device() != dev || !t->is_contiguous()) refuse(fn, "%s must be contiguous on %s", nm, dev.str().c_str());
        }
        c.pages = c.k->size(0), c.Hkv = c.k->size(1), c.ps = c.k->size(2), c.D = c.k->size(3);
        if (!none(ke)) {
            for (const auto& [i, nm] : {std::pair<int, const char*>{ke, "k_exp"}, {ve, "v_exp"}}) {
                const at::Tensor& t = vec(i, nm, at::kByte);
                if (t.dim() != 3 || t.size(0) != c.pages || t.size(1) != c.Hkv || t.size(2) != c.ps)
                    refuse(fn, "%s must be [pages, kv_heads, page_size], got %s", nm, shape_of(t).c_str());
            }
            c.ke = static_cast<uint8_t*>(tensor(ke, "k_exp").data_ptr());
            c.ve = static_cast<uint8_t*>(tensor(ve, "v_exp").data_ptr());
        }
        return c;
    }
};

// Strides of a [tokens, heads, head size] tensor.  Those of a single token or
// head are never used, and torch may have anything there.
int64_t token_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }
int64_t head_stride(const at::Tensor& t) { return t.size(1) > 1 ? t.stride(1) : t.size(2); }

template <typename T>
T* ptr(const at::Tensor& t) {
    return static_cast<T*>(t.data_ptr());
}

void status(const char* what, int rc) {
    if (rc == WLQ_OK) return;
    PyErr_Format(wlq_error, "%s failed with status %d: %s", what, rc, lib.last_error());
    throw PyFailed{};
}

// Runs a call's body; a C++ exception becomes a Python one.
template <typename Body>
PyObject* guarded(const char* fn, Py_ssize_t want, Py_ssize_t got, Body body) {
    if (want != got) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", fn, want, got);
        return nullptr;
    }
    try {
        body();
    } catch (const PyFailed&) {
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "wlq: unknown C++ exception");
        return nullptr;
    }
    Py_RETURN_NONE;
}

// q, k, v, positions, cos_sin, slots, k_cache, v_cache, q_out, k_out, k_exp, v_exp, interleaved
PyObject* rope_kv_write(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
    return guarded("rope_kv_write", 13, argc, [&] {
        Args x{"rope_kv_write", argv};
        const at::Tensor& q0 = x.lead(0, "q");
        const Args::Cache c = x.cache(6, 7, 10, 11);
        const at::Tensor& q = x.heads(0, "q", -1, -1, c.D);
        const int64_t T = q0.size(0), Hq = q0.size(1);
        const at::Tensor &k = x.heads(1, "k", T, c.Hkv, c.D), &v = x.heads(2, "v", T, c.Hkv, c.D);
        const at::Tensor& qo = x.heads(8, "q_out", T, Hq, c.D);
        const at::Tensor* ko = x.none(9) ? nullptr : &x.heads(9, "k_out", T, c.Hkv, c.D);
        const at::Tensor &pos = x.vec(3, "positions", at::kLong, T), &slots = x.vec(5, "slots", at::kLong, T);
        const at::Tensor& cs = x.vec(4, "cos_sin", at::kFloat);
        if (cs.dim() != 2) refuse(x.fn, "cos_sin must be [positions, rot]");
        const c10::cuda::CUDAGuard guard(x.dev);
        status("wlq_rope_kv_write",
               lib.rope_kv_write(q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr<int64_t>(pos), ptr<float>(cs),
                                 ptr<int64_t>(slots), c.k->data_ptr(), c.v->data_ptr(), c.ke, c.ve, qo.data_ptr(),
                                 ko ? ko->data_ptr() : nullptr, token_stride(q), head_stride(q), token_stride(k), head_stride(k),
                                 token_stride(v), head_stride(v), token_stride(qo), head_stride(qo), ko ? token_stride(*ko) : 0,
                                 ko ? head_stride(*ko) : 0, T, cs.size(0), c.pages, (int)Hq, (int)c.Hkv, (int)c.D,
                                 (int)cs.size(1), (int)c.ps, x.truth(12), x.dtype(),
                                 c10::cuda::getCurrentCUDAStream(x.dev.index()).stream()));
    });
}

// k_cache, v_cache, block_table, cu_lens, k_out, v_out, k_exp, v_exp
PyObject* kv_read(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
    return guarded("kv_read", 8, argc, [&] {
        Args x{"kv_read", argv};
        const at::Tensor& ko = x.lead(4, "k_out");
        const Args::Cache c = x.cache(0, 1, 6, 7);
        x.heads(4, "k_out", -1, c.Hkv, c.D);
        const at::Tensor& vo = x.heads(5, "v_out", ko.size(0), c.Hkv, c.D);
        if (!ko.is_contiguous() || !vo.is_contiguous()) refuse(x.fn, "k_out and v_out must be contiguous");
        const at::Tensor &table = x.vec(2, "block_table", at::kInt), &cu = x.vec(3, "cu_lens", at::kInt);
        if (table.dim() != 2 || cu.numel() != table.size(0) + 1)
            refuse(x.fn, "block_table must be [B, pages] and cu_lens [B + 1], got %s and %s", shape_of(table).c_str(),
                   shape_of(cu).c_str());
        const c10::cuda::CUDAGuard guard(x.dev);
        status("wlq_kv_read",
               lib.kv_read(c.k->data_ptr(), c.v->data_ptr(), c.ke, c.ve, ptr<int32_t>(table), ptr<int32_t>(cu),
                           ko.data_ptr(), vo.data_ptr(), ko.size(0), (int)table.size(0), c.pages, table.size(1),
                           (int)c.Hkv, (int)c.D, (int)c.ps, x.dtype(),
                           c10::cuda::getCurrentCUDAStream(x.dev.index()).stream()));
    });
}

// q, k, v, cu_seqlens, out, scale, causal
PyObject* prompt_attention(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
    return guarded("prompt_attention", 7, argc, [&] {
        Args x{"prompt_attention", argv};
        x.lead(0, "q");
        const at::Tensor& q = x.heads(0, "q", -1, -1, -1);
        const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
        const at::Tensor& k = x.heads(1, "k", T, -1, D);
        const at::Tensor &v = x.heads(2, "v", T, k.size(1), D), &o = x.heads(4, "out", T, Hq, D);
        const at::Tensor& cu = x.vec(3, "cu_seqlens", at::kInt);
        if (cu.numel() < 1) refuse(x.fn, "cu_seqlens must have a value more than there are sequences");
        const c10::cuda::CUDAGuard guard(x.dev);
        status("wlq_prompt_attention",
               lib.prompt_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr<int32_t>(cu), o.data_ptr(),
                                    token_stride(q), head_stride(q), token_stride(k), head_stride(k), token_stride(v), head_stride(v),
                                    token_stride(o), head_stride(o), T, (int)(cu.numel() - 1), (int)Hq, (int)k.size(1), (int)D,
                                    x.scale(5, D), x.truth(6), x.dtype(),
                                    c10::cuda::getCurrentCUDAStream(x.dev.index()).stream()));
    });
}

// Workspaces of paged_attention, one per device and stream (calls on several
// streams may overlap), grown when a call needs more and kept for the
// process.  While a CUDA graph is captured the graph gets one of its own, from
// its memory pool: a replay may overlap later calls on the stream that
// captured it.
auto* kept = new std::map<std::pair<int, cudaStream_t>, at::Tensor>;  // never destroyed: CUDA may be gone by then
std::mutex lock;

at::Tensor workspace(at::Device dev, c10::cuda::CUDAStream stream, size_t bytes) {
    auto make = [&] {
        at::Tensor t = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
        t.narrow(0, 0, WLQ_ATTENTION_ZERO_BYTES).zero_();
        return t;
    };
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return make();
    const std::lock_guard<std::mutex> hold(lock);
    at::Tensor& t = (*kept)[{dev.index(), stream.stream()}];
    if (!t.defined() || (size_t)t.numel() < bytes) t = make();
    return t;
}

// q, k_cache, v_cache, block_table, kv_lens, out, cu_q, max_q, k_exp, v_exp, scale
PyObject* paged_attention(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
    return guarded("paged_attention", 11, argc, [&] {
        Args x{"paged_attention", argv};
        x.lead(0, "q");
        const Args::Cache c = x.cache(1, 2, 8, 9);
        const at::Tensor& q = x.heads(0, "q", -1, -1, c.D);
        const int64_t T = q.size(0), Hq = q.size(1);
        const at::Tensor& o = x.heads(5, "out", T, Hq, c.D);
        const at::Tensor& table = x.vec(3, "block_table", at::kInt);
        if (table.dim() != 2) refuse(x.fn, "block_table must be [B, pages], got %s", shape_of(table).c_str());
        const int64_t B = table.size(0), max_q = x.integer(7);
        const at::Tensor& lens = x.vec(4, "kv_lens", at::kInt, B);
        const int32_t* cu = x.none(6) ? nullptr : ptr<int32_t>(x.vec(6, "cu_q", at::kInt, B + 1));
        if (max_q < 1 || max_q > 0x7fffffff) refuse(x.fn, "max_q must be at least 1");
        const c10::cuda::CUDAGuard guard(x.dev);
        const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(x.dev.index());
        const at::Tensor ws = workspace(x.dev, stream, lib.workspace_bytes((int)Hq, (int)c.Hkv, (int)c.D, (int)max_q));
        status("wlq_paged_attention",
               lib.paged_attention(q.data_ptr(), c.k->data_ptr(), c.v->data_ptr(), c.ke, c.ve, ptr<int32_t>(table),
                                   ptr<int32_t>(lens), cu, o.data_ptr(), token_stride(q), head_stride(q), token_stride(o),
                                   head_stride(o), T, (int)B, (int)Hq, (int)c.Hkv, (int)c.D, (int)c.ps, c.pages,
                                   table.size(1), (int)max_q, x.scale(10, c.D), x.dtype(), ws.data_ptr(),
                                   (size_t)ws.numel(), stream.stream()));
    });
}

// The kept workspaces, and their end: the next calls begin with fresh ones.
// (Memory goes back to its stream's pool, behind the calls that still use it.)
PyObject* kept_workspaces(PyObject*, PyObject*) {
    std::map<std::pair<int, cudaStream_t>, at::Tensor> all;
    {
        const std::lock_guard<std::mutex> hold(lock);  // (not while Python runs)
        all = *kept;
    }
    PyObject* list = PyList_New(0);
    for (const auto& entry : all) {
        PyObject* t = list ? THPVariable_Wrap(entry.second) : nullptr;
        if (!t || PyList_Append(list, t) < 0) Py_CLEAR(list);
        Py_XDECREF(t);
    }
    return list;
}
PyObject* drop_workspaces(PyObject*, PyObject*) {
    std::map<std::pair<int, cudaStream_t>, at::Tensor> gone;
    {
        const std::lock_guard<std::mutex> hold(lock);
        gone.swap(*kept);
    }
    Py_RETURN_NONE;
}

// setup((addresses in the order of Entries), WLQError)
PyObject* setup(PyObject*, PyObject* args) {
    PyObject* addresses;
    PyObject* error;
    if (!PyArg_ParseTuple(args, "O!O", &PyTuple_Type, &addresses, &error)) return nullptr;
    void** slots = reinterpret_cast<void**>(&lib);
    if (PyTuple_GET_SIZE(addresses) != (Py_ssize_t)(sizeof(lib) / sizeof(void*))) {
        PyErr_SetString(PyExc_TypeError, "setup: wrong number of entry points");
        return nullptr;
    }
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(addresses); ++i) {
        slots[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, i));
        if (!slots[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "setup: an entry point is missing");
            return nullptr;
        }
    }
    Py_INCREF(error);
    wlq_error = error;
    Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"rope_kv_write", fast(rope_kv_write), METH_FASTCALL, nullptr},
                         {"kv_read", fast(kv_read), METH_FASTCALL, nullptr},
                         {"prompt_attention", fast(prompt_attention), METH_FASTCALL, nullptr},
                         {"paged_attention", fast(paged_attention), METH_FASTCALL, nullptr},
                         {"kept_workspaces", kept_workspaces, METH_NOARGS, nullptr},
                         {"drop_workspaces", drop_workspaces, METH_NOARGS, nullptr},
                         {"setup", setup, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Attention operator calls over the C ABI", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__calls() { return PyModule_Create(&module); }

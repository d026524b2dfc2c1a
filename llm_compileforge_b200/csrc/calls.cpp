// The feed-forward calls from Python without a descriptor built in Python: a small call costs the GPU three to ten microseconds,
// and made through ctypes it costs the host eleven to eighteen.
//
// Each function takes the tensors of an ops.py call, checks that they are the usual ones - CUDA tensors of the current device, one
// type, shapes that fit, rows contiguous - allocates the result and makes the library call.  It answers with the result; with None
// for anything else, which the Python code beside it then handles or refuses in words; or with the library's status, an int.
// The library's functions come as addresses (bind), so this module works with whichever build of it the process has loaded.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/sfb.h"

namespace {

struct Library {
    decltype(&sfb_fused_linear) fused_linear;
    decltype(&sfb_grouped_linear) grouped_linear;
    decltype(&sfb_grouped_linear_workspace_bytes) grouped_bytes;
    decltype(&sfb_moe_route) route;
    decltype(&sfb_moe_route_workspace_bytes) route_bytes;
    decltype(&sfb_moe_combine) combine;
} lib;

using at::Tensor;

// An argument: absent (None), a tensor, or something else.
struct Arg {
    bool fine = true, given = false;
    Tensor t;
    explicit Arg(PyObject* o) {
        if (o == Py_None) return;
        fine = given = THPVariable_Check(o);
        if (given) t = THPVariable_Unpack(o);
    }
    bool is(int device, at::ScalarType type, int64_t dim) const {
        return fine && (!given || (t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.dim() == dim));
    }
};

struct Desc {
    SFBTensor d;
    const SFBTensor* ptr = nullptr;
    SFBTensor* out = nullptr;
    void set(void* data, int elem, int rank, const int64_t* sizes, const int64_t* strides) {
        d.device = SFB_DEVICE_CUDA;
        d.rank = rank;
        d.elem_size = elem;
        d.r4.allocated = d.r4.aligned = data;
        d.r4.offset = 0;
        int64_t* tail = d.r4.sizes;  // sizes[rank], then strides[rank], whatever the rank
        for (int i = 0; i < rank; ++i) { tail[i] = sizes[i]; tail[rank + i] = strides[i]; }
        ptr = out = &d;
    }
    void set(const Tensor& t) { set(t.data_ptr(), (int)t.element_size(), (int)t.dim(), t.sizes().data(), t.strides().data()); }
    // [.., n] as rows
    void rows(const Tensor& t, int64_t rows, int64_t n) {
        const int64_t sizes[2] = {rows, n}, strides[2] = {t.dim() == 2 ? t.stride(0) : n, 1};
        set(t.data_ptr(), (int)t.element_size(), 2, sizes, strides);
    }
    // [.., K, N] with K contiguous, as the [.., N, K] that is stored
    void transposed(const Tensor& t) {
        int64_t sizes[3], strides[3];
        const int r = (int)t.dim();
        for (int i = 0; i < r; ++i) { sizes[i] = t.size(i); strides[i] = t.stride(i); }
        std::swap(sizes[r - 1], sizes[r - 2]);
        std::swap(strides[r - 1], strides[r - 2]);
        set(t.data_ptr(), (int)t.element_size(), r, sizes, strides);
    }
};

int type_code(at::ScalarType t) { return t == at::kBFloat16 ? SFB_BF16 : t == at::kHalf ? SFB_F16 : t == at::kFloat ? SFB_F32 : -1; }
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
bool rows_contiguous(const Tensor& t) { return t.dim() == 2 ? t.stride(1) == 1 : t.is_contiguous(); }
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int device) {
    return at::empty(sizes, at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, (c10::DeviceIndex)device)));
}
PyObject* none() { Py_RETURN_NONE; }

// C++ exceptions (out of memory, for one) become Python's.
template <typename F>
PyObject* guarded(F f) {
    try {
        return f();
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        if (type) PyErr_SetString(type, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// Weight and up weight of one layout -> descriptors; false where there is no such layout.
bool weights(const Arg& w, const Arg& u, Desc* dw, Desc* du, int* layout) {
    const int64_t r = w.t.dim();
    if (w.t.stride(r - 1) == 1) {
        *layout = SFB_WEIGHT_KN;
        dw->set(w.t);
        if (u.given) { if (u.t.stride(r - 1) != 1) return false; du->set(u.t); }
    } else if (w.t.stride(r - 2) == 1) {
        *layout = SFB_WEIGHT_NK;
        dw->transposed(w.t);
        if (u.given) { if (u.t.stride(r - 2) != 1) return false; du->transposed(u.t); }
    } else {
        return false;
    }
    return !u.given || u.t.sizes() == w.t.sizes();
}

bool status_of(const Arg& status, int device, int32_t** p) {
    *p = nullptr;
    if (!status.given) return status.fine;
    if (!status.t.is_cuda() || status.t.get_device() != device || status.t.scalar_type() != at::kInt || status.t.numel() < 1) return false;
    *p = static_cast<int32_t*>(status.t.data_ptr());
    return true;
}

// linear(x, weight, bias, up_weight, up_bias, residual, out, status, activation, fp32_out)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (n_args != 10 || !lib.fused_linear) return none();
    return guarded([&]() -> PyObject* {
        const Arg x(a[0]), w(a[1]), b(a[2]), u(a[3]), ub(a[4]), r(a[5]), out(a[6]), status(a[7]);
        if (!x.given || !w.given || !x.t.is_cuda()) return none();
        const int device = x.t.get_device();
        const at::ScalarType type = x.t.scalar_type();
        const long act = PyLong_AsLong(a[8]);
        const bool wide = PyObject_IsTrue(a[9]) == 1;
        if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
        if (act < 0 || type_code(type) < 0 || device != c10::cuda::current_device() || x.t.dim() < 2 || x.t.dim() > 4 || !rows_contiguous(x.t)) return none();
        const int64_t K = x.t.size(-1);
        if (!w.is(device, type, 2) || !u.is(device, type, 2) || !b.is(device, type, 1) || !ub.is(device, type, 1) || w.t.size(0) != K || K < 1) return none();
        const int64_t N = w.t.size(1), M = x.t.numel() / K;
        if (N < 1 || M < 1 || (ub.given && !u.given) || (out.given && wide)) return none();
        for (const Arg* v : {&b, &ub})
            if (v->given && (v->t.size(0) != N || v->t.stride(0) != 1)) return none();
        const at::ScalarType out_type = out.given ? (out.fine ? out.t.scalar_type() : type) : wide ? at::kFloat : type;
        if (!out.fine || (out_type != type && out_type != at::kFloat)) return none();
        for (const Arg* v : {&r, &out})
            if (v->given && (!v->is(device, out_type, x.t.dim()) || v->t.size(-1) != N || v->t.numel() != M * N || !rows_contiguous(v->t))) return none();
        for (const Arg* v : {&r, &out})
            for (int64_t i = 0; v->given && i + 1 < x.t.dim(); ++i)
                if (v->t.size(i) != x.t.size(i)) return none();
        if (!r.fine) return none();
        int32_t* st;
        if (!status_of(status, device, &st)) return none();
        Desc dx, dw, du, db, dub, dr, dout;
        int layout;
        if (!weights(w, u, &dw, &du, &layout)) return none();
        dx.rows(x.t, M, K);
        if (b.given) db.set(b.t);
        if (ub.given) dub.set(ub.t);
        if (r.given) dr.rows(r.t, M, N);
        Tensor o = out.t;
        if (!out.given) {
            at::DimVector sizes(x.t.sizes());
            sizes.back() = N;
            o = empty(sizes, out_type, device);
        }
        dout.rows(o, M, N);
        const int rc = lib.fused_linear(dx.ptr, dw.ptr, db.ptr, du.ptr, dub.ptr, dr.ptr, dout.out, layout, type_code(type), type_code(out_type), (int)act, st,
                                        stream_of(device));
        if (rc != SFB_OK) return PyLong_FromLong(rc);
        if (out.given) { Py_INCREF(a[6]); return a[6]; }
        return THPVariable_Wrap(std::move(o));
    });
}

// grouped(x, weight, group_offsets, bias, up_weight, up_bias, row_index, out, workspace, status, activation, fp32_out)
PyObject* grouped(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (n_args != 12 || !lib.grouped_linear) return none();
    return guarded([&]() -> PyObject* {
        const Arg x(a[0]), w(a[1]), off(a[2]), b(a[3]), u(a[4]), ub(a[5]), index(a[6]), out(a[7]), ws(a[8]), status(a[9]);
        if (!x.given || !w.given || !off.given || !x.t.is_cuda() || ws.given || !ws.fine) return none();
        const int device = x.t.get_device();
        const at::ScalarType type = x.t.scalar_type();
        const long act = PyLong_AsLong(a[10]);
        const bool wide = PyObject_IsTrue(a[11]) == 1;
        if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
        if (act < 0 || type_code(type) < 0 || device != c10::cuda::current_device() || x.t.dim() != 2 || x.t.stride(1) != 1) return none();
        const int64_t K = x.t.size(1);
        if (!w.is(device, type, 3) || !u.is(device, type, 3) || !b.is(device, type, 2) || !ub.is(device, type, 2) || !off.is(device, at::kInt, 1) ||
            !index.is(device, at::kInt, 1) || !index.fine || w.t.size(1) != K || K < 1)
            return none();
        const int64_t E = w.t.size(0), N = w.t.size(2), M = index.given ? index.t.size(0) : x.t.size(0);
        if (E < 1 || N < 1 || M < 1 || off.t.size(0) != E + 1 || off.t.stride(0) != 1 || (index.given && index.t.stride(0) != 1) || (ub.given && !u.given) ||
            (out.given && wide))
            return none();
        for (const Arg* v : {&b, &ub})
            if (v->given && (v->t.size(0) != E || v->t.size(1) != N || v->t.stride(1) != 1)) return none();
        const at::ScalarType out_type = out.given ? (out.fine ? out.t.scalar_type() : type) : wide ? at::kFloat : type;
        if (!out.fine || (out_type != type && out_type != at::kFloat) || !out.is(device, out_type, 2) ||
            (out.given && (out.t.size(0) != M || out.t.size(1) != N || out.t.stride(1) != 1)))
            return none();
        int32_t* st;
        if (!status_of(status, device, &st)) return none();
        Desc dx, dw, du, db, dub, doff, dindex, dout;
        int layout;
        if (!weights(w, u, &dw, &du, &layout)) return none();
        dx.set(x.t);
        doff.set(off.t);
        if (b.given) db.set(b.t);
        if (ub.given) dub.set(ub.t);
        if (index.given) dindex.set(index.t);
        Tensor o = out.given ? out.t : empty({M, N}, out_type, device), room;
        dout.set(o);
        int64_t bytes = index.given && type != at::kFloat ? lib.grouped_bytes(M, K, E, 1) : 0;
        if (bytes > 0) room = empty({bytes}, at::kByte, device);
        const int rc = lib.grouped_linear(dx.ptr, dw.ptr, db.ptr, du.ptr, dub.ptr, doff.ptr, dindex.ptr, dout.out, layout, type_code(type), type_code(out_type),
                                          (int)act, st, bytes > 0 ? room.data_ptr() : nullptr, bytes > 0 ? bytes : 0, stream_of(device));
        if (rc != SFB_OK) return PyLong_FromLong(rc);
        if (out.given) { Py_INCREF(a[7]); return a[7]; }
        return THPVariable_Wrap(std::move(o));
    });
}

// route(logits, top_k, renormalize, workspace) -> (ids, weights, offsets, token_rows, positions)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (n_args != 4 || !lib.route) return none();
    return guarded([&]() -> PyObject* {
        const Arg l(a[0]), ws(a[3]);
        if (!l.given || !l.t.is_cuda() || ws.given || !ws.fine || !PyLong_CheckExact(a[1])) return none();
        const int64_t k = PyLong_AsLongLong(a[1]);
        const bool renormalize = PyObject_IsTrue(a[2]) == 1;
        if (PyErr_Occurred()) { PyErr_Clear(); return none(); }
        const int device = l.t.get_device();
        if (device != c10::cuda::current_device() || l.t.dim() != 2 || type_code(l.t.scalar_type()) < 0 || l.t.stride(1) != 1) return none();
        const int64_t T = l.t.size(0), E = l.t.size(1);
        if (T < 1 || k < 1 || k > E || k > 32) return none();
        const Tensor results[5] = {empty({T, k}, at::kInt, device), empty({T, k}, at::kFloat, device), empty({E + 1}, at::kInt, device),
                                   empty({T * k}, at::kInt, device), empty({T, k}, at::kInt, device)};
        Desc dl, d[5];
        dl.set(l.t);
        for (int i = 0; i < 5; ++i) d[i].set(results[i]);
        const int64_t bytes = lib.route_bytes(T, E);
        Tensor room;
        if (bytes > 0) room = empty({bytes}, at::kByte, device);
        const int rc = lib.route(dl.ptr, d[0].out, d[1].out, d[2].out, d[3].out, d[4].out, type_code(l.t.scalar_type()), renormalize,
                                 bytes > 0 ? room.data_ptr() : nullptr, bytes > 0 ? bytes : 0, stream_of(device));
        if (rc != SFB_OK) return PyLong_FromLong(rc);
        PyObject* all = PyTuple_New(5);
        if (!all) return nullptr;
        for (int i = 0; i < 5; ++i) {
            PyObject* o = THPVariable_Wrap(results[i]);
            if (!o) { Py_DECREF(all); return nullptr; }
            PyTuple_SET_ITEM(all, i, o);
        }
        return all;
    });
}

// combine(y, positions, weights, residual, out, status)
PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (n_args != 6 || !lib.combine) return none();
    return guarded([&]() -> PyObject* {
        const Arg y(a[0]), p(a[1]), w(a[2]), r(a[3]), out(a[4]), status(a[5]);
        if (!y.given || !p.given || !w.given || !r.fine || !out.fine || !y.t.is_cuda()) return none();
        const int device = y.t.get_device();
        const at::ScalarType type = y.t.scalar_type();
        if (device != c10::cuda::current_device() || type_code(type) < 0 || !y.is(device, type, 2) || !p.is(device, at::kInt, 2) || !w.is(device, at::kFloat, 2) ||
            !r.is(device, type, 2) || !out.is(device, type, 2))
            return none();
        const int64_t T = p.t.size(0), k = p.t.size(1), H = y.t.size(1);
        if (T < 1 || H < 1 || w.t.sizes() != p.t.sizes() || y.t.stride(1) != 1 || (k > 1 && (p.t.stride(1) != 1 || w.t.stride(1) != 1))) return none();
        for (const Arg* v : {&r, &out})
            if (v->given && (v->t.size(0) != T || v->t.size(1) != H || v->t.stride(1) != 1)) return none();
        int32_t* st;
        if (!status_of(status, device, &st)) return none();
        Tensor o = out.given ? out.t : empty({T, H}, type, device);
        Desc dy, dp, dw, dr, dout;
        dy.set(y.t); dp.set(p.t); dw.set(w.t); dout.set(o);
        if (r.given) dr.set(r.t);
        const int rc = lib.combine(dy.ptr, dp.ptr, dw.ptr, dr.ptr, dout.out, type_code(type), st, stream_of(device));
        if (rc != SFB_OK) return PyLong_FromLong(rc);
        if (out.given) { Py_INCREF(a[4]); return a[4]; }
        return THPVariable_Wrap(std::move(o));
    });
}

// bind(addresses of the library's functions, in the order of Library)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    static_assert(sizeof(Library) == 6 * sizeof(void*), "six functions");
    if (n_args != 6) { PyErr_SetString(PyExc_TypeError, "bind takes six addresses"); return nullptr; }
    void* p[6];
    for (int i = 0; i < 6; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    memcpy(&lib, p, sizeof(lib));
    return none();
}

#define SFB_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {SFB_METHOD(linear), SFB_METHOD(grouped), SFB_METHOD(route), SFB_METHOD(combine), SFB_METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", SFB_TORCH_VERSION) < 0) Py_CLEAR(m);  // of the headers above
    return m;
}

// Host side of the batched-cache operators as one CPython call each: argument checks, output and workspace allocation, launch.  A single-token step is a
// handful of kernels of 3 .. 10 us; the same steps in Python over ctypes took 11 .. 16 us of host time a call, so the host decided its speed.  Nothing is
// decided here that fastvideo_amd/ops.py does not decide as well: an argument that is not what a call needs makes it return None, and the Python front end
// names what is wrong.  The C entries of libfvk_amd.so come in as addresses (init), so that this module is bound to the library that Python has loaded.
#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/fvk_amd.h"

namespace {

decltype(&fvk_paged_plan) paged_plan = nullptr;
decltype(&fvk_rmsnorm_rope_paged_bf16) rmsnorm_rope_paged = nullptr;
decltype(&fvk_attn_ragged_workspace_bytes) workspace_bytes = nullptr;
decltype(&fvk_attn_ragged_bf16) attn_ragged = nullptr;
decltype(&fvk_last_error) last_error = nullptr;

constexpr long MOST = 0x7fffffff;

const at::Tensor* tensor(PyObject* o, at::ScalarType type, long device) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == device && t.scalar_type() == type && t.layout() == at::kStrided ? &t : nullptr;
}
const at::Tensor* ints(PyObject* o, long device) { return tensor(o, at::kInt, device); }
const at::Tensor* bf16(PyObject* o, long device) { return tensor(o, at::kBFloat16, device); }
bool vector_of(const at::Tensor* t, int64_t n) { return t && t->dim() == 1 && t->size(0) == n && t->is_contiguous(); }
bool same_shape(const at::Tensor& a, const at::Tensor& b) { return a.sizes() == b.sizes(); }

// whole number in [lo, hi]
bool number(PyObject* o, long& v, long lo = 0, long hi = MOST) {
    v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return v >= lo && v <= hi;
}
int shift_of(int64_t page) {
    for (int s = 4; s <= 8; ++s)
        if (page == int64_t(1) << s) return s;
    return -1;
}
bool window_ok(PyObject* w, PyObject* s, long& window, long& sink) { return number(w, window) && number(s, sink) && (window > 0 || sink == 0); }

PyObject* refused(const char* what, int rc) {
    const char* msg = last_error();
    return PyErr_Format(PyExc_RuntimeError, "%s failed (rc=%d): %s", what, rc, msg ? msg : "?");
}

#define DECLINE_UNLESS(cond) \
    if (!(cond)) Py_RETURN_NONE;

PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* p[5];
    for (int i = 0; i < 5; ++i) {
        p[i] = n == 5 ? PyLong_AsVoidPtr(a[i]) : nullptr;
        if (!p[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_TypeError, "init takes five addresses");
    }
    paged_plan = reinterpret_cast<decltype(paged_plan)>(p[0]);
    rmsnorm_rope_paged = reinterpret_cast<decltype(rmsnorm_rope_paged)>(p[1]);
    workspace_bytes = reinterpret_cast<decltype(workspace_bytes)>(p[2]);
    attn_ragged = reinterpret_cast<decltype(attn_ragged)>(p[3]);
    last_error = reinterpret_cast<decltype(last_error)>(p[4]);
    Py_RETURN_NONE;
}

// plan(device, stream, starts, new_lens, block_table, pages_held, free_pages, free_count, page_size, n_tokens, grid_hw, window, sink, causal) -> nine tensors
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    long device, stream, page, n_tokens, gh, gw, window, sink;
    DECLINE_UNLESS(paged_plan && n == 14 && number(a[0], device) && number(a[1], stream, 0, LONG_MAX));
    const at::Tensor *starts = ints(a[2], device), *lens = ints(a[3], device), *table = ints(a[4], device), *held = ints(a[5], device), *free = ints(a[6], device),
                     *count = ints(a[7], device);
    DECLINE_UNLESS(table && table->dim() == 2 && table->is_contiguous() && free && free->dim() == 1 && free->is_contiguous());
    const int64_t R = table->size(0), W = table->size(1), F = free->size(0);
    DECLINE_UNLESS(vector_of(starts, R) && vector_of(lens, R) && vector_of(held, R) && vector_of(count, 1));
    DECLINE_UNLESS(number(a[8], page) && shift_of(page) >= 0 && number(a[9], n_tokens) && window_ok(a[11], a[12], window, sink));
    DECLINE_UNLESS(PyTuple_Check(a[10]) && PyTuple_GET_SIZE(a[10]) == 2 && number(PyTuple_GET_ITEM(a[10], 0), gh, 1) && number(PyTuple_GET_ITEM(a[10], 1), gw, 1) &&
                   gh * gw <= MOST && R <= MOST && W <= MOST && F <= MOST);
    const int causal = PyObject_IsTrue(a[13]);
    if (causal < 0) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    // one allocation: the nine outputs in turn, then the scratch that the kernels leave for each other
    const int64_t sizes[10] = {R * W, R, F, 1, R + 1, R, n_tokens, n_tokens * 3, R, 2 * R + 1};
    int64_t total = 0;
    for (int64_t s : sizes) total += s;
    const at::Tensor buf = at::empty({total}, table->options());
    int32_t* p[10];
    int32_t* at_ = static_cast<int32_t*>(buf.data_ptr());
    for (int i = 0; i < 10; ++i) {
        p[i] = at_;
        at_ += sizes[i];
    }
    auto in = [](const at::Tensor* t) { return static_cast<const int32_t*>(t->data_ptr()); };
    const int rc = paged_plan(in(starts), in(lens), in(table), in(held), in(free), in(count), p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], (int)R,
                              (int)W, (int)F, (int)page, (int)n_tokens, (int)gh, (int)gw, (int)window, (int)sink, causal, reinterpret_cast<void*>(stream));
    if (rc != 0) return refused("fvk_paged_plan", rc);
    PyObject* out = PyTuple_New(9);
    if (!out) return nullptr;
    int64_t offset = 0;
    for (int i = 0; i < 9; ++i) {
        // a tensor over its part of the storage (whole numbers: no gradient, so no view to record; half the time of as_strided)
        at::Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
        c10::TensorImpl* impl = v.unsafeGetTensorImpl();
        impl->set_storage_offset(offset);
        const int64_t rows = i == 0 ? R : i == 7 ? n_tokens : sizes[i], columns = i == 0 ? W : 3;
        const int64_t size[2] = {rows, columns}, stride[2] = {columns, 1};
        if (i == 0 || i == 7) impl->set_sizes_and_strides(at::IntArrayRef(size, 2), at::IntArrayRef(stride, 2));
        else impl->set_sizes_and_strides(at::IntArrayRef(size, 1), at::IntArrayRef(stride + 1, 1));
        offset += sizes[i];
        PyObject* o = THPVariable_Wrap(v);
        if (!o) {
            Py_DECREF(out);
            return nullptr;
        }
        PyTuple_SET_ITEM(out, i, o);
    }
    return out;
    END_HANDLE_TH_ERRORS
}

bool three(PyObject* o, long (&v)[3]) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3) return false;
    for (int i = 0; i < 3; ++i)
        if (!number(PyTuple_GET_ITEM(o, i), v[i])) return false;
    return true;
}

bool pages_ok(const at::Tensor* k, const at::Tensor* v) {
    return k && v && k->dim() == 4 && same_shape(*k, *v) && k->size(3) == 128 && k->stride(3) == 1 && v->stride(3) == 1 && shift_of(k->size(1)) >= 0;
}

// write(device, stream, q, k, v, q_weight, k_weight, positions, rope, slot_map, k_pages, v_pages, eps, round_norm, out) -> out
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    long device, stream, sizes[3] = {0, 0, 0}, dims[3] = {0, 0, 0};
    DECLINE_UNLESS(rmsnorm_rope_paged && n == 15 && number(a[0], device) && number(a[1], stream, 0, LONG_MAX));
    const at::Tensor *q = bf16(a[2], device), *k = bf16(a[3], device), *v = bf16(a[4], device), *kp = bf16(a[10], device), *vp = bf16(a[11], device);
    DECLINE_UNLESS(pages_ok(kp, vp) && q && k && v && q->dim() == 2 && k->dim() == 2 && same_shape(*k, *v));
    const int64_t T = q->size(0), width = q->size(1), Hkv = kp->size(2);
    DECLINE_UNLESS(width > 0 && width % 128 == 0 && k->size(0) == T && k->size(1) == Hkv * 128 && q->stride(1) == 1 && k->stride(1) == 1 && v->stride(1) == 1);
    const void* w[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i)
        if (a[5 + i] != Py_None) {
            const at::Tensor* t = bf16(a[5 + i], device);
            DECLINE_UNLESS(t && t->numel() == (i == 0 ? width : Hkv * 128) && t->is_contiguous());
            w[i] = t->data_ptr();
        }
    const at::Tensor* slots = ints(a[9], device);
    DECLINE_UNLESS(vector_of(slots, T) && T <= MOST && kp->size(0) <= MOST);
    const int32_t* positions = nullptr;
    const float* table = nullptr;
    if (a[8] != Py_None) {
        DECLINE_UNLESS(PyTuple_Check(a[8]) && PyTuple_GET_SIZE(a[8]) == 3);
        const at::Tensor *t = tensor(PyTuple_GET_ITEM(a[8], 0), at::kFloat, device), *p = ints(a[7], device);
        DECLINE_UNLESS(t && p && three(PyTuple_GET_ITEM(a[8], 1), sizes) && three(PyTuple_GET_ITEM(a[8], 2), dims));
        DECLINE_UNLESS(p->dim() == 2 && p->size(0) == T && p->size(1) == 3 && p->is_contiguous());
        const long most = std::max(dims[0], std::max(dims[1], dims[2]));
        DECLINE_UNLESS(t->dim() == 3 && t->size(0) == sizes[0] + sizes[1] + sizes[2] && t->size(1) == most / 2 && t->size(2) == 2 && t->is_contiguous() &&
                       dims[0] + dims[1] + dims[2] == 128 && ((dims[0] | dims[1] | dims[2]) & 1) == 0);
        positions = static_cast<const int32_t*>(p->data_ptr());
        table = static_cast<const float*>(t->data_ptr());
    }
    const double eps = PyFloat_AsDouble(a[12]);
    const int round_norm = PyObject_IsTrue(a[13]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    at::Tensor out;
    if (a[14] == Py_None) {
        out = at::empty({T, width}, q->options());
    } else {
        const at::Tensor* t = bf16(a[14], device);
        DECLINE_UNLESS(t && same_shape(*t, *q) && t->stride(1) == 1);
        out = *t;
    }
    if (T > 0) {
        const int rc = rmsnorm_rope_paged(q->data_ptr(), k->data_ptr(), v->data_ptr(), w[0], w[1], positions, table, static_cast<const int32_t*>(slots->data_ptr()),
                                          out.data_ptr(), kp->data_ptr(), vp->data_ptr(), (int)T, (int)(width / 128), (int)Hkv, q->stride(0), k->stride(0),
                                          v->stride(0), out.stride(0), kp->stride(0), kp->stride(1), kp->stride(2), vp->stride(0), vp->stride(1), vp->stride(2),
                                          (int)kp->size(0), (int)kp->size(1), (int)sizes[0], (int)sizes[1], (int)sizes[2], (int)dims[0], (int)dims[1], (int)dims[2],
                                          round_norm, (float)eps, reinterpret_cast<void*>(stream));
        if (rc != 0) return refused("fvk_rmsnorm_rope_paged_bf16", rc);
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// attn(device, stream, q, k, v, lens, cu_q, block_table or None, max_q, max_kv, scale, causal, window, sink, out, return_lse) -> out, or (out, lse)
PyObject* attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    long device, stream, max_q, max_kv, window, sink;
    DECLINE_UNLESS(attn_ragged && n == 16 && number(a[0], device) && number(a[1], stream, 0, LONG_MAX));
    const at::Tensor *q = bf16(a[2], device), *k = bf16(a[3], device), *v = bf16(a[4], device), *lens = ints(a[5], device), *cu = ints(a[6], device);
    const bool paged = a[7] != Py_None;
    const at::Tensor* table = paged ? ints(a[7], device) : nullptr;
    DECLINE_UNLESS(q && k && v && lens && cu && q->dim() == 3 && q->size(2) == 128 && q->stride(2) == 1 && cu->dim() == 1 && cu->is_contiguous());
    const int64_t T = q->size(0), H = q->size(1), R = cu->size(0) - 1;
    DECLINE_UNLESS(R >= 1 && vector_of(lens, paged ? R : R + 1));
    if (paged) {
        DECLINE_UNLESS(pages_ok(k, v) && table && table->dim() == 2 && table->is_contiguous() && table->size(0) == R && table->size(1) >= 1);
    } else {
        DECLINE_UNLESS(k->dim() == 3 && same_shape(*k, *v) && k->size(2) == 128 && k->stride(2) == 1 && v->stride(2) == 1);
    }
    const int64_t Hkv = k->size(paged ? 2 : 1), top = paged ? table->size(1) * k->size(1) : k->size(0);
    DECLINE_UNLESS(Hkv > 0 && H % Hkv == 0 && T <= MOST && H <= MOST && R <= MOST && k->size(0) <= MOST && top <= MOST);
    max_q = T;
    max_kv = top;
    DECLINE_UNLESS((a[8] == Py_None || number(a[8], max_q)) && (a[9] == Py_None || number(a[9], max_kv)) && window_ok(a[12], a[13], window, sink));
    if (paged && max_kv > top) max_kv = top;
    const double scale = a[10] == Py_None ? 0.08838834764831845 : PyFloat_AsDouble(a[10]);  // 128^-1/2
    const int causal = PyObject_IsTrue(a[11]), want_lse = PyObject_IsTrue(a[15]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    at::Tensor out, lse, ws;
    if (a[14] == Py_None) {
        out = at::empty({T, H, 128}, q->options());
    } else {
        const at::Tensor* t = bf16(a[14], device);
        DECLINE_UNLESS(t && same_shape(*t, *q) && t->stride(2) == 1);
        out = *t;
    }
    if (want_lse) lse = at::empty({H, T}, q->options().dtype(at::kFloat));
    if (T > 0) {
        fvk_ragged_args g{};
        g.q = q->data_ptr();
        g.k = k->data_ptr();
        g.v = v->data_ptr();
        g.o = out.data_ptr();
        g.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
        g.cu_q = static_cast<const int32_t*>(cu->data_ptr());
        g.kv_lens = static_cast<const int32_t*>(lens->data_ptr());
        g.q_ts = q->stride(0);
        g.q_hs = q->stride(1);
        g.o_ts = out.stride(0);
        g.o_hs = out.stride(1);
        if (paged) {
            g.block_table = static_cast<const int32_t*>(table->data_ptr());
            g.k_ps = k->stride(0);
            g.v_ps = v->stride(0);
            g.table_width = (int)table->size(1);
            g.page_shift = shift_of(k->size(1));
            g.n_pages = (int)k->size(0);
        } else {
            g.total_k = (int)k->size(0);
        }
        g.k_rs = k->stride(paged ? 1 : 0);
        g.k_hs = k->stride(paged ? 2 : 1);
        g.v_rs = v->stride(paged ? 1 : 0);
        g.v_hs = v->stride(paged ? 2 : 1);
        g.T = (int)T;
        g.R = (int)R;
        g.H = (int)H;
        g.Hkv = (int)Hkv;
        g.max_q = (int)max_q;
        g.max_kv = (int)max_kv;
        g.scale = (float)scale;
        g.causal = causal;
        g.window = (int)window;
        g.sink = (int)sink;
        const long need = workspace_bytes(&g);
        if (need < 0) return refused("fvk_attn_ragged_workspace_bytes", -1);
        // a buffer of this call alone (the caching allocator hands it on in stream order; a captured graph keeps its own)
        if (need > 0) ws = at::empty({need}, q->options().dtype(at::kByte));
        const int rc = attn_ragged(&g, need > 0 ? ws.data_ptr() : nullptr, need, reinterpret_cast<void*>(stream));
        if (rc != 0) return refused("fvk_attn_ragged_bf16", rc);
    }
    PyObject* o = THPVariable_Wrap(out);
    if (!o || !want_lse) return o;
    PyObject* l = THPVariable_Wrap(lse);
    PyObject* both = l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_DECREF(o);
    Py_XDECREF(l);
    return both;
    END_HANDLE_TH_ERRORS
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(init), METHOD(plan), METHOD(write), METHOD(attn), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_launch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__launch() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "made_for", FVK_MADE_FOR) != 0) Py_CLEAR(m);  // neither torch's C++ interface nor CPython's has a stable ABI
    return m;
}

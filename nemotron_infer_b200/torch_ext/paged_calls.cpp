// The tensor-level calls of the paged cache and of prompt attention, compiled: a step of a few microseconds on the GPU should
// not wait for ten of argument checks in the interpreter (one paged attention call: 17 us of host time through ctypes).
//
// Each function takes the arguments of the operator of the same name in nemotron_infer_b200/ops.py, all positional, makes
// the checks that ops.py makes and calls the C ABI on torch's current stream.  It returns the operator's result, an int (the
// nmt_status of a call that was refused), or Ellipsis: something about the arguments is unusual or wrong - another
// device than the current one, a type, shape or layout it does not take - and ops.py goes through them one by one,
// with its messages.
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <torch/headeronly/version.h>

#include "nemotron_b200.h"

namespace {

using at::Tensor;

PyObject* unusual() { Py_INCREF(Py_Ellipsis); return Py_Ellipsis; }

struct View { void* p = nullptr; int64_t rows = 0, heads = 0, row_stride = 0, head_stride = 0; };

// A tensor argument: false when it is something else.
bool tensor(PyObject* o, const Tensor*& t) {
    if (!THPVariable_CheckExact(o)) return false;
    t = &THPVariable_Unpack(o);
    return true;
}
bool optional(PyObject* o, const Tensor*& t) {
    t = nullptr;
    return o == Py_None || tensor(o, t);
}
bool view(const Tensor& t, c10::Device dev, int64_t rows, int64_t heads, int64_t dim, View& v) {
    if (t.scalar_type() != at::kBFloat16 || t.dim() != 3 || t.device() != dev || t.size(0) != rows || t.size(1) != heads || t.size(2) != dim || t.stride(2) != 1)
        return false;
    v = {t.data_ptr(), rows, heads, t.stride(0), t.stride(1)};
    return true;
}
// A result: a new tensor, or the given one when it is contiguous (others may overlap: ops.py looks closer).
bool result(PyObject* given, const Tensor* t, const Tensor& like, c10::Device dev, View& v, PyObject*& out) {
    if (!t) {
        Tensor fresh = at::empty(like.sizes(), like.options());
        v = {fresh.data_ptr(), like.size(0), like.size(1), like.size(1) * like.size(2), like.size(2)};
        out = THPVariable_Wrap(std::move(fresh));
        return true;
    }
    if (!t->is_contiguous() || !view(*t, dev, like.size(0), like.size(1), like.size(2), v)) return false;
    Py_INCREF(given);
    out = given;
    return true;
}
bool ints(const Tensor* t, c10::Device dev, int64_t n, const int32_t*& p) {
    p = nullptr;
    if (!t) return true;
    if (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != n || !t->is_contiguous() || t->device() != dev) return false;
    p = static_cast<const int32_t*>(t->data_ptr());
    return true;
}
bool inner_contiguous(const Tensor& t) {
    return t.stride(3) == 1 && t.stride(2) == t.size(3) && t.stride(1) == t.size(2) * t.size(3);
}
bool scales(const Tensor* t, c10::Device dev, int64_t heads, const float*& p, int64_t& count) {
    p = nullptr;
    if (!t) return true;
    if (t->scalar_type() != at::kFloat || t->device() != dev || !t->is_contiguous() || (t->numel() != 1 && t->numel() != heads) ||
        (count && t->numel() != count))
        return false;
    count = t->numel();
    p = static_cast<const float*>(t->data_ptr());
    return true;
}
bool cache(PyObject* const* a, PyObject* k_scale, PyObject* v_scale, c10::Device dev, nmt_paged_cache& c) {
    const Tensor *k, *v, *table, *lens, *ks, *vs;
    if (!tensor(a[0], k) || !tensor(a[1], v) || !tensor(a[2], table) || !tensor(a[3], lens) || !optional(k_scale, ks) || !optional(v_scale, vs)) return false;
    if (k->dim() != 4 || v->dim() != 4 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() || k->device() != dev || v->device() != dev) return false;
    if (k->scalar_type() == at::kBFloat16) c.dtype = NMT_CACHE_BF16;
    else if (k->scalar_type() == at::kFloat8_e4m3fn) c.dtype = NMT_CACHE_E4M3;
    else return false;
    if (!inner_contiguous(*k) || !inner_contiguous(*v)) return false;
    if (table->scalar_type() != at::kInt || table->dim() != 2 || !table->is_contiguous() || table->device() != dev) return false;
    c.batch = table->size(0);
    c.max_pages = table->size(1);
    c.page_table = static_cast<const int32_t*>(table->data_ptr());
    if (!ints(lens, dev, c.batch, c.seq_lens)) return false;
    c.k = k->data_ptr();
    c.v = v->data_ptr();
    c.k_page_stride = k->stride(0);
    c.v_page_stride = v->stride(0);
    c.num_pages = k->size(0);
    c.kv_heads = k->size(1);
    c.page_size = k->size(2);
    c.head_dim = k->size(3);
    c.scale_count = 0;
    if (!scales(ks, dev, c.kv_heads, c.k_scale, c.scale_count) || !scales(vs, dev, c.kv_heads, c.v_scale, c.scale_count)) return false;
    if (!c.scale_count) c.scale_count = 1;
    return true;
}
bool number(PyObject* o, int64_t head_dim, float& scale) {
    if (o == Py_None) {
        scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(head_dim)));
        return true;
    }
    if (!PyFloat_CheckExact(o)) return false;
    scale = static_cast<float>(PyFloat_AS_DOUBLE(o));
    return true;
}
bool here(const Tensor& t) { return t.is_cuda() && t.device().index() == c10::cuda::current_device(); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
bool workspace(const Tensor* given, Tensor& own, const Tensor& like, int64_t need, void*& p) {
    p = nullptr;
    if (need <= 0) return true;
    if (!given) {
        own = at::empty({need}, like.options().dtype(at::kByte));
        given = &own;
    }
    if (given->device() != like.device() || !given->is_contiguous() || static_cast<int64_t>(given->nbytes()) < need) return false;
    p = given->data_ptr();
    return true;
}
PyObject* finish(int status, PyObject* out) {
    if (status == NMT_OK) return out;
    Py_DECREF(out);
    return PyLong_FromLong(status);
}

// (k, v, k_cache, v_cache, page_table, seq_lens, cu_new, q, rope, interleaved, k_scale, v_scale, q_out, err_flag)
PyObject* kv_append_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *k, *v, *cu, *q, *rope, *q_out, *err;
    nmt_paged_cache c;
    if (n != 14 || !tensor(a[0], k) || !tensor(a[1], v) || !optional(a[6], cu) || !optional(a[7], q) || !optional(a[8], rope) || !optional(a[12], q_out) ||
        !optional(a[13], err) || !here(*k) || !PyBool_Check(a[9]))
        return unusual();
    const c10::Device dev = k->device();
    if (!cache(a + 2, a[10], a[11], dev, c) || k->dim() != 3) return unusual();
    const int64_t T = k->size(0);
    View kv, vv, qv, ov;
    const int32_t *cu_p, *err_p;
    if (!view(*k, dev, T, c.kv_heads, c.head_dim, kv) || !view(*v, dev, T, c.kv_heads, c.head_dim, vv) || !ints(cu, dev, c.batch + 1, cu_p) ||
        !ints(err, dev, 1, err_p) || (!cu && T != c.batch) || (!q && q_out) || (q && !rope))
        return unusual();
    int64_t rows = 0, rot = 0;
    if (rope) {
        if (rope->scalar_type() != at::kFloat || rope->dim() != 2 || !rope->is_contiguous() || rope->device() != dev) return unusual();
        rows = rope->size(0);
        rot = rope->size(1);
    }
    PyObject* out = nullptr;
    if (q) {
        if (q->dim() != 3 || !view(*q, dev, T, q->size(1), c.head_dim, qv) || !result(a[12], q_out, *q, dev, ov, out)) return unusual();
    } else {
        Py_INCREF(Py_None);
        out = Py_None;
    }
    return finish(nmt_kv_append_paged_bf16(&c, cu_p, T, kv.p, kv.row_stride, kv.head_stride, vv.p, vv.row_stride, vv.head_stride,
                                           rope ? static_cast<const float*>(rope->data_ptr()) : nullptr, rows, rot, a[9] == Py_True, qv.p, qv.row_stride,
                                           qv.head_stride, qv.heads, ov.p, ov.row_stride, ov.head_stride, const_cast<int32_t*>(err_p), stream_of(*k)),
                  out);
    END_HANDLE_TH_ERRORS
}

// (q, k_cache, v_cache, page_table, seq_lens, scale, k_scale, v_scale, out, workspace, err_flag)
PyObject* sdpa_decode_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *given, *ws, *err;
    nmt_paged_cache c;
    if (n != 11 || !tensor(a[0], q) || !optional(a[8], given) || !optional(a[9], ws) || !optional(a[10], err) || !here(*q)) return unusual();
    const c10::Device dev = q->device();
    View qv, ov;
    const int32_t* err_p;
    float scale;
    if (!cache(a + 1, a[6], a[7], dev, c) || q->dim() != 3 || !view(*q, dev, c.batch, q->size(1), c.head_dim, qv) || !ints(err, dev, 1, err_p) ||
        !number(a[5], c.head_dim, scale))
        return unusual();
    Tensor own;
    void* ws_p;
    PyObject* out = nullptr;
    if (!workspace(ws, own, *q, nmt_sdpa_decode_paged_workspace_bytes(c.batch, qv.heads, c.kv_heads, c.head_dim), ws_p) || !result(a[8], given, *q, dev, ov, out))
        return unusual();
    return finish(nmt_sdpa_decode_paged_bf16(&c, qv.p, qv.row_stride, qv.head_stride, ov.p, ov.row_stride, ov.head_stride, qv.heads, scale,
                                             const_cast<int32_t*>(err_p), ws_p, stream_of(*q)),
                  out);
    END_HANDLE_TH_ERRORS
}

// (q, k, v, cu_seqlens, cu_seqlens_k, causal, scale, out, workspace)
PyObject* sdpa_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *q, *k, *v, *cu, *cu_k, *given, *ws;
    if (n != 9 || !tensor(a[0], q) || !tensor(a[1], k) || !tensor(a[2], v) || !optional(a[3], cu) || !optional(a[4], cu_k) || !optional(a[7], given) ||
        !optional(a[8], ws) || !here(*q) || !PyBool_Check(a[5]) || q->dim() != 3 || k->dim() != 3 || (!cu && cu_k))
        return unusual();
    if (cu && cu->numel() < 1) return unusual();
    const c10::Device dev = q->device();
    const int64_t T = q->size(0), T_k = k->size(0), heads = q->size(1), kv_heads = k->size(1), dim = q->size(2), batch = cu ? cu->numel() - 1 : 1;
    View qv, kv, vv, ov;
    const int32_t *cu_p, *cu_k_p;
    float scale;
    if (!view(*q, dev, T, heads, dim, qv) || !view(*k, dev, T_k, kv_heads, dim, kv) || !view(*v, dev, T_k, kv_heads, dim, vv) || !ints(cu, dev, batch + 1, cu_p) ||
        !ints(cu_k, dev, batch + 1, cu_k_p) || (cu && !cu_k && T != T_k) || !number(a[6], dim, scale))
        return unusual();
    Tensor own;
    void* ws_p;
    PyObject* out = nullptr;
    if (!workspace(ws, own, *q, nmt_sdpa_prefill_workspace_bytes(batch, T, T_k, heads, kv_heads, dim), ws_p) || !result(a[7], given, *q, dev, ov, out)) return unusual();
    return finish(nmt_sdpa_prefill_bf16(qv.p, qv.row_stride, qv.head_stride, kv.p, kv.row_stride, kv.head_stride, vv.p, vv.row_stride, vv.head_stride, ov.p,
                                        ov.row_stride, ov.head_stride, cu_p, cu_k_p, batch, T, T_k, heads, kv_heads, dim, scale, a[5] == Py_True, ws_p,
                                        stream_of(*q)),
                  out);
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"kv_append_paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(kv_append_paged)), METH_FASTCALL, nullptr},
    {"sdpa_decode_paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sdpa_decode_paged)), METH_FASTCALL, nullptr},
    {"sdpa_prefill", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sdpa_prefill)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged_calls() {
    PyObject* m = PyModule_Create(&module);
    if (m) PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION);  // of the headers: ops.py compares it with the torch that runs
    return m;
}

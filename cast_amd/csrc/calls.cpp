// cast_amd._calls: the paged cache's per-layer calls from torch tensors, for
// arguments that the kernels take as they lie.
//
// A decode step makes two of these calls a layer, and its kernels take 3 to 12 us
// where few requests run; with some ten tensors checked and 50 arguments
// converted in Python a call took 17.5 us of the host (the tree attention 22.8),
// here it takes 6 (append) and 9 to 10 (attention, 6.5 of them two launches).
// Each function repeats the conditions
// of its wrapper in cast_amd/paged.py and either makes the call, or returns
// None: the wrapper then converts what can be converted and words the error
// for what cannot.  The result is the wrapper's, or the cast_status of a call
// that the library refused.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <cmath>

#include "cast_amd.h"

namespace {

constexpr int64_t kInt32 = INT32_MAX;

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return CAST_BF16;
        case at::kHalf: return CAST_FP16;
        case at::kFloat: return CAST_FP32;
        default: return -1;
    }
}

// What Python hands over: a tensor, or None (nullptr).
struct Arg {
    const at::Tensor *t = nullptr;
    bool ok = true;
    explicit Arg(PyObject *o) {
        if (o == Py_None) return;
        if (THPVariable_CheckExact(o)) t = &THPVariable_Unpack(o);
        else ok = false;
    }
    explicit operator bool() const { return t != nullptr; }
    const at::Tensor *operator->() const { return t; }
    const at::Tensor &operator*() const { return *t; }
};

bool aligned(const at::Tensor &t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// The pools of a layer: what the other tensors have to agree with.
struct Pools {
    const at::Tensor &k, &v;
    c10::DeviceIndex index;
    at::ScalarType dtype;
    int code;
    int64_t pages, H_kv, page_size, D, esz;
    bool ok;

    Pools(const at::Tensor &k_, const at::Tensor &v_)
        : k(k_), v(v_), index(-1), dtype(k.scalar_type()), code(code_of(dtype)), ok(false) {
        if (k.dim() != 4 || code < 0 || v.scalar_type() != dtype || !k.is_cuda() || v.device() != k.device() ||
            v.sizes() != k.sizes() || k.numel() == 0)
            return;
        index = k.device().index();
        pages = k.size(0), H_kv = k.size(1), page_size = k.size(2), D = k.size(3);
        esz = k.element_size();
        // (the launch goes to the current device)
        if (c10::impl::VirtualGuardImpl(at::kCUDA).getDevice().index() != index) return;
        if (pages > kInt32 || page_size > kInt32) return;
        int64_t low = 0;
        for (const at::Tensor *t : {&k, &v}) {
            if (t->stride(3) != 1) return;
            for (int i = 0; i < 3; ++i) low |= t->stride(i);
        }
        ok = (low * esz & 15) == 0 && aligned(k) && aligned(v);
    }
    // [n, heads, D] of the pools' type, as it lies
    bool rows(const at::Tensor &t, int64_t n, int64_t heads) const {
        return t.dim() == 3 && t.scalar_type() == dtype && t.is_cuda() && t.device().index() == index && t.size(0) == n &&
               t.size(1) == heads && t.size(2) == D && t.stride(2) == 1 && ((t.stride(0) | t.stride(1)) * esz & 15) == 0 &&
               aligned(t);
    }
    // and written: no element twice
    bool output(const at::Tensor &t, int64_t n, int64_t heads) const {
        return rows(t, n, heads) && (n <= 1 || t.stride(0)) && (heads <= 1 || t.stride(1));
    }
    // int32 values side by side
    bool ints(const at::Tensor &t, int64_t n) const {
        return t.dim() == 1 && t.scalar_type() == at::kInt && t.is_cuda() && t.device().index() == index && t.size(0) == n &&
               t.is_contiguous();
    }
    bool table(const at::Tensor &t) const {
        return t.dim() == 2 && t.scalar_type() == at::kInt && t.is_cuda() && t.device().index() == index && t.numel() &&
               (t.stride(1) == 1 || t.size(1) == 1) && t.size(0) <= kInt32 && t.size(1) <= kInt32;
    }
};

template <typename T>
T *at_of(const Arg &a) {
    return a ? static_cast<T *>(a->data_ptr()) : nullptr;
}

// (a, b), whose references it takes; null where one is.
PyObject *pair(PyObject *a, PyObject *b) {
    PyObject *r = a && b ? PyTuple_Pack(2, a, b) : nullptr;
    Py_XDECREF(a);
    Py_XDECREF(b);
    return r;
}

// paged_append(k, v, k_pages, v_pages, page_table, seq_len, cu_q, q, cos, sin,
//              positions, interleaved, q_out, k_out, new_len, stream)
PyObject *paged_append(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 16) {
        PyErr_SetString(PyExc_TypeError, "paged_append takes 16 arguments");
        return nullptr;
    }
    const Arg k(o[0]), v(o[1]), kp(o[2]), vp(o[3]), table(o[4]), len(o[5]), cu(o[6]), q(o[7]), cos(o[8]), sin(o[9]), pos(o[10]),
        q_out(o[12]), k_out(o[13]), new_len(o[14]);
    for (const Arg *a : {&k, &v, &kp, &vp, &table, &len, &cu, &q, &cos, &sin, &pos, &q_out, &k_out, &new_len})
        if (!a->ok) Py_RETURN_NONE;
    if (!k || !v || !kp || !vp || !table || !len) Py_RETURN_NONE;
    const Pools pools(*kp, *vp);
    if (!pools.ok || !pools.table(*table) || k->dim() != 3) Py_RETURN_NONE;
    const int64_t B = table->size(0), total = k->size(0);
    if (!total || total > kInt32 || !pools.ints(*len, B) || !pools.rows(*k, total, pools.H_kv) ||
        !pools.rows(*v, total, pools.H_kv))
        Py_RETURN_NONE;
    if (cu ? !pools.ints(*cu, B + 1) : total != B) Py_RETURN_NONE;
    int64_t H_q = 0;
    if (q) {
        if (q->dim() != 3) Py_RETURN_NONE;
        H_q = q->size(1);
        if (!H_q || H_q % pools.H_kv || H_q > kInt32 || !pools.rows(*q, total, H_q)) Py_RETURN_NONE;
        if (q_out && !pools.output(*q_out, total, H_q)) Py_RETURN_NONE;
    } else if (q_out) {
        Py_RETURN_NONE;
    }
    if (k_out && !pools.output(*k_out, total, pools.H_kv)) Py_RETURN_NONE;
    int64_t rot = 0, max_pos = 0, ld = 0;
    if (cos || sin) {
        if (!cos || !sin || cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->strides() != sin->strides())
            Py_RETURN_NONE;
        for (const Arg *a : {&cos, &sin})
            if ((*a)->scalar_type() != at::kFloat || !(*a)->is_cuda() || (*a)->device().index() != pools.index || !aligned(**a))
                Py_RETURN_NONE;
        max_pos = cos->size(0), rot = 2 * cos->size(1), ld = max_pos > 1 ? cos->stride(0) : rot / 2;
        if (!max_pos || max_pos > kInt32 || rot <= 0 || rot > pools.D || rot % (32 / pools.esz) || cos->stride(1) != 1 ||
            ld % 4 || ld < rot / 2)
            Py_RETURN_NONE;
        if (pos && !pools.ints(*pos, total)) Py_RETURN_NONE;
    }
    if (new_len && !pools.ints(*new_len, B)) Py_RETURN_NONE;
    const int interleaved = PyObject_IsTrue(o[11]);
    if (interleaved < 0) return nullptr;
    const auto stream = reinterpret_cast<cast_stream_t>(PyLong_AsVoidPtr(o[15]));
    if (PyErr_Occurred()) return nullptr;

    at::Tensor made_q, made_len;
    const at::Tensor *qo = q_out.t, *nl = new_len.t;
    if (q && !qo) qo = &(made_q = at::empty(q->sizes(), q->options()));
    if (!nl) nl = &(made_len = at::empty({B}, len->options()));
    const void *kk = k->data_ptr(), *vv = v->data_ptr();
    void *kkp = kp->data_ptr(), *vvp = vp->data_ptr();
    const int64_t *sk = kp->strides().data(), *sv = vp->strides().data();
    int st;
    Py_BEGIN_ALLOW_THREADS;
    st = cast_paged_append(&kk, &vv, &kkp, &vvp, 1, at_of<int32_t>(table), table->stride(0), (int32_t)table->size(1),
                           (int32_t)pools.pages, (int32_t)pools.page_size, at_of<int32_t>(len),
                           static_cast<int32_t *>(nl->data_ptr()), (int32_t)B, (int32_t)total, at_of<int32_t>(cu), nullptr, 0,
                           nullptr, q ? q->data_ptr() : nullptr, qo ? qo->data_ptr() : nullptr, at_of<void>(k_out),
                           at_of<float>(cos), at_of<float>(sin), ld, (int32_t)max_pos, (int32_t)rot, interleaved,
                           cos ? at_of<int32_t>(pos) : nullptr, (int32_t)H_q, (int32_t)pools.H_kv, (int32_t)pools.D,
                           k->stride(0), k->stride(1), v->stride(0), v->stride(1), sk[0], sk[1], sk[2], sv[0], sv[1], sv[2],
                           q ? q->stride(0) : 0, q ? q->stride(1) : 0, qo ? qo->stride(0) : 0, qo ? qo->stride(1) : 0,
                           k_out ? k_out->stride(0) : 0, k_out ? k_out->stride(1) : 0, pools.code, nullptr, stream);
    Py_END_ALLOW_THREADS;
    if (st) return PyLong_FromLong(st);
    return pair(made_q.defined() ? THPVariable_Wrap(made_q) : Py_NewRef(o[q ? 12 : 7]),
                made_len.defined() ? THPVariable_Wrap(made_len) : Py_NewRef(o[14]));
    END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_pages, v_pages, page_table, seq_len, sm_scale, softcap,
//                 window, kv_split, return_lse, out, workspace, stream)
PyObject *paged_attention(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 13) {
        PyErr_SetString(PyExc_TypeError, "paged_attention takes 13 arguments");
        return nullptr;
    }
    const Arg q(o[0]), kp(o[1]), vp(o[2]), table(o[3]), len(o[4]), out(o[10]), ws(o[11]);
    for (const Arg *a : {&q, &kp, &vp, &table, &len, &out, &ws})
        if (!a->ok) Py_RETURN_NONE;
    if (!q || !kp || !vp || !table || !len) Py_RETURN_NONE;
    const Pools pools(*kp, *vp);
    if (!pools.ok || !pools.table(*table) || q->dim() != 3) Py_RETURN_NONE;
    const int64_t B = table->size(0), H_q = q->size(1);
    if (!H_q || H_q % pools.H_kv || H_q > kInt32 || !pools.rows(*q, B, H_q) || !pools.ints(*len, B)) Py_RETURN_NONE;
    if (out && !pools.output(*out, B, H_q)) Py_RETURN_NONE;
    if (!PyFloat_Check(o[6]) || !PyLong_Check(o[7]) || !PyLong_Check(o[8]) || (o[5] != Py_None && !PyFloat_Check(o[5])))
        Py_RETURN_NONE;
    const double cap = PyFloat_AS_DOUBLE(o[6]);
    const double scale = o[5] == Py_None ? 1.0 / std::sqrt((double)pools.D) : PyFloat_AS_DOUBLE(o[5]);
    int past;
    const long long window = PyLong_AsLongLongAndOverflow(o[7], &past);
    if (past || window < 0 || window > kInt32) Py_RETURN_NONE;
    const long long split = PyLong_AsLongLongAndOverflow(o[8], &past);
    if (past || split < -1 || split > kInt32) Py_RETURN_NONE;
    if (!(cap >= 0.0 && cap < HUGE_VAL)) Py_RETURN_NONE;
    const int lse_too = PyObject_IsTrue(o[9]);
    if (lse_too < 0) return nullptr;
    const auto stream = reinterpret_cast<cast_stream_t>(PyLong_AsVoidPtr(o[12]));
    if (PyErr_Occurred()) return nullptr;
    const int32_t max_pages = (int32_t)table->size(1);
    const size_t need = cast_paged_attn_workspace_size((int32_t)B, max_pages, (int32_t)pools.page_size, (int32_t)H_q,
                                                       (int32_t)pools.H_kv, (int32_t)pools.D, (int32_t)window, pools.code,
                                                       (int32_t)split);
    if (ws && (!ws->is_cuda() || ws->device().index() != pools.index || !ws->is_contiguous() || ws->nbytes() < need))
        Py_RETURN_NONE;

    at::Tensor made, lse, made_ws;
    const at::Tensor *to = out.t;
    void *space = need && ws ? ws->data_ptr() : nullptr;
    if (!to) to = &(made = at::empty({B, H_q, pools.D}, q->options()));
    if (lse_too) lse = at::empty({B, H_q}, q->options().dtype(at::kFloat));
    if (need && !ws) space = (made_ws = at::empty({(int64_t)need}, q->options().dtype(at::kByte))).data_ptr();
    const int64_t *sk = kp->strides().data(), *sv = vp->strides().data();
    int st;
    Py_BEGIN_ALLOW_THREADS;
    st = cast_paged_attn_fwd(q->data_ptr(), kp->data_ptr(), vp->data_ptr(), to->data_ptr(),
                             lse_too ? static_cast<float *>(lse.data_ptr()) : nullptr, at_of<int32_t>(table), table->stride(0),
                             max_pages, (int32_t)pools.pages, (int32_t)pools.page_size, at_of<int32_t>(len), (int32_t)B,
                             (int32_t)H_q, (int32_t)pools.H_kv, (int32_t)pools.D, q->stride(0), q->stride(1), sk[0], sk[1],
                             sk[2], sv[0], sv[1], sv[2], to->stride(0), to->stride(1), pools.code, (float)scale, (float)cap,
                             (int32_t)window, (int32_t)split, space, need, nullptr, stream);
    Py_END_ALLOW_THREADS;
    if (st) return PyLong_FromLong(st);
    PyObject *r = made.defined() ? THPVariable_Wrap(made) : Py_NewRef(o[10]);
    return lse_too ? pair(r, THPVariable_Wrap(lse)) : r;
    END_HANDLE_TH_ERRORS
}

// paged_tree_attention(q, k_pages, v_pages, page_table, k_pack, v_pack, cu_q,
//                      prefix_len, pack_len, ancestor_mask, sm_scale, total_kv,
//                      return_lse, kv_split, out, workspace, stream)
PyObject *paged_tree_attention(PyObject *, PyObject *const *o, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 17) {
        PyErr_SetString(PyExc_TypeError, "paged_tree_attention takes 17 arguments");
        return nullptr;
    }
    const Arg q(o[0]), kp(o[1]), vp(o[2]), table(o[3]), kn(o[4]), vn(o[5]), cu(o[6]), pre(o[7]), pack(o[8]), mask(o[9]),
        out(o[14]), ws(o[15]);
    for (const Arg *a : {&q, &kp, &vp, &table, &kn, &vn, &cu, &pre, &pack, &mask, &out, &ws})
        if (!a->ok) Py_RETURN_NONE;
    if (!q || !kp || !vp || !table || !kn || !vn || !cu || !pre || !pack || !mask) Py_RETURN_NONE;
    const Pools pools(*kp, *vp);
    if (!pools.ok || !pools.table(*table) || q->dim() != 3) Py_RETURN_NONE;
    const int64_t B = table->size(0), max_pages = table->size(1), total_q = q->size(0), H_q = q->size(1);
    if (!total_q || total_q > kInt32 || !H_q || H_q % pools.H_kv || H_q > kInt32 || !pools.rows(*q, total_q, H_q)) Py_RETURN_NONE;
    if (pools.page_size % 64 && max_pages > 1) Py_RETURN_NONE;
    for (const Arg *a : {&kn, &vn})
        if (!pools.rows(**a, pools.H_kv, total_q)) Py_RETURN_NONE;   // (head-major)
    if (!pools.ints(*cu, B + 1) || !pools.ints(*pre, B) || !pools.ints(*pack, B)) Py_RETURN_NONE;
    if (mask->scalar_type() != at::kLong || !mask->is_cuda() || mask->device().index() != pools.index ||
        !mask->is_contiguous() || mask->dim() < 1 || mask->dim() > 2 || mask->size(0) != total_q)
        Py_RETURN_NONE;
    const int64_t words = mask->dim() == 1 ? 1 : mask->size(1);
    if (words < 1 || words > 2) Py_RETURN_NONE;
    if (out && !pools.output(*out, total_q, H_q)) Py_RETURN_NONE;
    if ((o[10] != Py_None && !PyFloat_Check(o[10])) || (o[11] != Py_None && !PyLong_Check(o[11])) || !PyLong_Check(o[13]))
        Py_RETURN_NONE;
    const double scale = o[10] == Py_None ? 1.0 / std::sqrt((double)pools.D) : PyFloat_AS_DOUBLE(o[10]);
    int past = 0, past2;
    if (o[11] == Py_None && max_pages * pools.page_size > kInt32) Py_RETURN_NONE;
    const int64_t total_kv =
        o[11] == Py_None ? B * max_pages * pools.page_size + total_q : PyLong_AsLongLongAndOverflow(o[11], &past);
    const long long split = PyLong_AsLongLongAndOverflow(o[13], &past2);
    if (past || past2 || total_kv < 0 || total_kv > kInt32 || split < -kInt32 || split > kInt32) Py_RETURN_NONE;
    const int lse_too = PyObject_IsTrue(o[12]);
    if (lse_too < 0) return nullptr;
    const auto stream = reinterpret_cast<cast_stream_t>(PyLong_AsVoidPtr(o[16]));
    if (PyErr_Occurred()) return nullptr;
    const size_t need =
        cast_tree_attn_paged_workspace_size((int32_t)B, (int32_t)total_q, (int32_t)total_kv, (int32_t)H_q, (int32_t)pools.H_kv,
                                            (int32_t)pools.D, pools.code, (int32_t)split);
    if (ws && (!ws->is_cuda() || ws->device().index() != pools.index || !ws->is_contiguous() || ws->nbytes() < need))
        Py_RETURN_NONE;

    at::Tensor made, lse, made_ws;
    const at::Tensor *to = out.t;
    if (!to) to = &(made = at::empty({total_q, H_q, pools.D}, q->options()));
    if (lse_too) lse = at::empty({total_q, H_q}, q->options().dtype(at::kFloat));
    void *space = ws ? ws->data_ptr() : (made_ws = at::empty({(int64_t)need}, q->options().dtype(at::kByte))).data_ptr();
    const int64_t *sk = kp->strides().data(), *sv = vp->strides().data();
    int st;
    Py_BEGIN_ALLOW_THREADS;
    st = cast_tree_attn_paged_fwd(
        q->data_ptr(), kp->data_ptr(), vp->data_ptr(), at_of<int32_t>(table), table->stride(0), (int32_t)max_pages,
        (int32_t)pools.pages, (int32_t)pools.page_size, kn->data_ptr(), vn->data_ptr(), to->data_ptr(),
        lse_too ? static_cast<float *>(lse.data_ptr()) : nullptr, at_of<int32_t>(cu), at_of<int32_t>(pre), at_of<int32_t>(pack),
        static_cast<const uint64_t *>(mask->data_ptr()), (int32_t)words, (int32_t)B, (int32_t)total_q, (int32_t)total_kv,
        (int32_t)H_q, (int32_t)pools.H_kv, (int32_t)pools.D, q->stride(0), q->stride(1), sk[0], sk[1], sk[2], sv[0], sv[1],
        sv[2], kn->stride(1), kn->stride(0), vn->stride(1), vn->stride(0), to->stride(0), to->stride(1), pools.code,
        (float)scale, (int32_t)split, space, need, nullptr, stream);
    Py_END_ALLOW_THREADS;
    if (st) return PyLong_FromLong(st);
    PyObject *r = made.defined() ? THPVariable_Wrap(made) : Py_NewRef(o[14]);
    return lse_too ? pair(r, THPVariable_Wrap(lse)) : r;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(paged_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(paged_attention)), METH_FASTCALL, nullptr},
    {"paged_tree_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(paged_tree_attention)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }

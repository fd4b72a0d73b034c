// CPython front end of the C ABI for torch tensors: reads the tensors' addresses, shapes and strides,
// allocates the result and calls libws_tp.so, all natively.
//
// Filling a ctypes struct, torch.empty, torch.cuda.current_stream() and the ctypes call itself cost
// ~12 us of host time per step (B200 host, measured), more than a decode step of a tensor-parallel shard
// takes on the device (6 us).  A function here returns None for arguments outside the plain form
// (non-CUDA tensors, unexpected types or layouts); tp.py then takes its own path, which explains what is
// wrong.  A negative status of the C ABI is returned as an int.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include <vector>

#include "../../include/ws_tp.h"

namespace {

const at::Tensor *tensor(PyObject *o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() ? &t : nullptr;
}

bool act_dtype(const at::Tensor &t, int32_t *out) {
    if (t.scalar_type() == at::kBFloat16) *out = WS_ACT_BF16;
    else if (t.scalar_type() == at::kFloat) *out = WS_ACT_F32;
    else return false;
    return true;
}

// What a kernel reads or writes has to be there: all rows of scale blocks, a result of m x n floats.  (Block shapes and
// offsets that make no sense are the C ABI's to refuse.)
bool covers(const at::Tensor &scales, int64_t row0, int64_t n, int64_t bn) {
    return bn <= 0 || row0 < 0 || n < 1 || (row0 + n - 1) / bn < scales.size(0);
}
bool holds(const at::Tensor &out, int64_t m, int64_t n) {
    return out.scalar_type() == at::kFloat && out.is_contiguous() && out.numel() >= m * n;
}

// Everything of a step but its result; false: not the plain form.
bool fill_fp8(ws_fp8_gemm_args_t &a, PyObject *ox, PyObject *ow, PyObject *os, int32_t bn, int32_t bk, int64_t row0, int64_t k0) {
    const at::Tensor *x = tensor(ox), *w = tensor(ow), *s = tensor(os);
    if (!x || !w || !s || x->dim() != 2 || w->dim() != 2 || s->dim() != 2) return false;
    if (w->scalar_type() != at::kByte && w->scalar_type() != at::kFloat8_e4m3fn) return false;
    if (s->scalar_type() == at::kFloat) a.scale_kind = WS_SCALE_F32;
    else if (s->scalar_type() == at::kByte) a.scale_kind = WS_SCALE_UE8M0;
    else return false;
    if (!act_dtype(*x, &a.x_dtype) || x->stride(1) != 1 || w->stride(1) != 1 || !s->is_contiguous() || w->size(1) != x->size(1)) return false;
    const int64_t m = x->size(0), n = w->size(0), k = x->size(1);
    if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX || !covers(*s, row0, n, bn)) return false;
    a.m = (int32_t)m; a.n = (int32_t)n; a.k = (int32_t)k;
    a.x = x->data_ptr(); a.ldx = m > 1 ? x->stride(0) : k;
    a.w = static_cast<const uint8_t *>(w->data_ptr()); a.ldw = w->stride(0);
    a.scales = s->data_ptr(); a.scale_ld = s->size(1);
    a.block_n = bn; a.block_k = bk; a.row0 = row0; a.k0 = k0;
    return true;
}

bool fill_moe(ws_moe_down_args_t &a, PyObject *oh, PyObject *oids, PyObject *orw, PyObject *ow, PyObject *os, int32_t e_start) {
    const at::Tensor *h = tensor(oh), *ids = tensor(oids), *rw = tensor(orw), *w = tensor(ow), *s = tensor(os);
    if (!h || !ids || !rw || !w || !s || w->dim() != 3 || s->dim() != 3 || ids->dim() != 2 || h->dim() != 2) return false;
    if (!w->is_contiguous() || !s->is_contiguous() || !ids->is_contiguous() || !rw->is_contiguous()) return false;
    if (ids->scalar_type() != at::kInt || rw->scalar_type() != at::kFloat || !act_dtype(*h, &a.h_dtype)) return false;
    const int64_t k = w->size(2) * 2, routes = ids->numel();
    if (w->element_size() != 1 || s->element_size() != 1 || s->numel() * 16 < w->numel()) return false;
    if (h->size(0) < routes || h->size(1) < k || h->stride(1) != 1 || rw->numel() < routes) return false;
    a.h = h->data_ptr(); a.ldh = h->size(0) > 1 ? h->stride(0) : k;
    a.m = (int32_t)ids->size(0); a.top_k = (int32_t)ids->size(1); a.n = (int32_t)w->size(1); a.k = (int32_t)k;
    a.route_ids = ids->data_ptr<int32_t>(); a.route_w = rw->data_ptr<float>();
    a.w2 = static_cast<const uint8_t *>(w->data_ptr()); a.s2 = static_cast<const uint8_t *>(s->data_ptr());
    a.e_start = e_start; a.e_len = (int32_t)w->size(0);
    return true;
}

at::Tensor new_f32(const at::Tensor &like, int64_t m, int64_t n) { return at::empty({m, n}, like.options().dtype(at::kFloat).requires_grad(false)); }

bool stream_of(PyObject *o, void **out) {  // None: torch's current stream of the current device
    if (o == Py_None) {
        *out = c10::cuda::getCurrentCUDAStream().stream();
        return true;
    }
    *out = PyLong_AsVoidPtr(o);
    return !PyErr_Occurred();
}

// A status, or the result: `result` is the caller's `out` or a tensor made here.
PyObject *answer(ws_status_t st, PyObject *result) {
    if (st == WS_OK) return result;
    Py_XDECREF(result);
    return PyLong_FromLong(st);
}

#define WS_CALL(st, expr)            \
    ws_status_t st;                  \
    Py_BEGIN_ALLOW_THREADS           \
    st = expr;                       \
    Py_END_ALLOW_THREADS

// fp8(handle, x, w, scales, block_n, block_k, row0, k0, out, stream)
PyObject *py_fp8(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 10) { PyErr_SetString(PyExc_TypeError, "fp8 takes 10 arguments"); return nullptr; }
    ws_fp8_gemm_args_t a{};
    ws_tp_t *const tp = static_cast<ws_tp_t *>(PyLong_AsVoidPtr(v[0]));
    const long bn = PyLong_AsLong(v[4]), bk = PyLong_AsLong(v[5]);
    const int64_t row0 = PyLong_AsLongLong(v[6]), k0 = PyLong_AsLongLong(v[7]);
    void *stream;
    if (PyErr_Occurred() || !stream_of(v[9], &stream)) return nullptr;
    if (!fill_fp8(a, v[1], v[2], v[3], (int32_t)bn, (int32_t)bk, row0, k0)) Py_RETURN_NONE;
    PyObject *res;
    if (v[8] == Py_None) {
        at::Tensor out = new_f32(THPVariable_Unpack(v[1]), a.m, a.n);
        a.out = out.data_ptr<float>();
        res = THPVariable_Wrap(std::move(out));
    } else {
        const at::Tensor *out = tensor(v[8]);
        if (!out || !holds(*out, a.m, a.n)) Py_RETURN_NONE;
        a.out = static_cast<float *>(out->data_ptr());
        Py_INCREF(v[8]);
        res = v[8];
    }
    WS_CALL(st, ws_fp8_rowpar_gemm_allreduce(tp, &a, stream))
    return answer(st, res);
    END_HANDLE_TH_ERRORS
}

// fp8_host(handle, x_host, w, scales, block_n, block_k, row0, k0, x_dtype, out_host) -> status: x_host and out_host are
// C-contiguous buffers (numpy arrays) of at least m * k activations and m * n floats.
PyObject *py_fp8_host(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 10) { PyErr_SetString(PyExc_TypeError, "fp8_host takes 10 arguments"); return nullptr; }
    ws_tp_t *const tp = static_cast<ws_tp_t *>(PyLong_AsVoidPtr(v[0]));
    const at::Tensor *w = tensor(v[2]), *s = tensor(v[3]);
    ws_fp8_gemm_args_t a{};
    a.block_n = (int32_t)PyLong_AsLong(v[4]); a.block_k = (int32_t)PyLong_AsLong(v[5]);
    a.row0 = PyLong_AsLongLong(v[6]); a.k0 = PyLong_AsLongLong(v[7]); a.x_dtype = (int32_t)PyLong_AsLong(v[8]);
    if (PyErr_Occurred()) return nullptr;
    if (!w || !s || w->dim() != 2 || s->dim() != 2 || w->stride(1) != 1 || w->element_size() != 1) Py_RETURN_NONE;
    if (!s->is_contiguous() || !covers(*s, a.row0, w->size(0), a.block_n)) Py_RETURN_NONE;
    if (s->scalar_type() == at::kFloat) a.scale_kind = WS_SCALE_F32;
    else if (s->scalar_type() == at::kByte) a.scale_kind = WS_SCALE_UE8M0;
    else Py_RETURN_NONE;
    Py_buffer x, out;
    if (PyObject_GetBuffer(v[1], &x, PyBUF_ND) != 0) { PyErr_Clear(); Py_RETURN_NONE; }
    if (PyObject_GetBuffer(v[9], &out, PyBUF_ND | PyBUF_WRITABLE) != 0) { PyBuffer_Release(&x); PyErr_Clear(); Py_RETURN_NONE; }
    a.n = (int32_t)w->size(0); a.k = (int32_t)w->size(1);
    a.m = x.ndim > 0 ? (int32_t)x.shape[0] : 0;
    a.ldx = a.k; a.w = static_cast<const uint8_t *>(w->data_ptr()); a.ldw = w->stride(0);
    a.scales = s->data_ptr(); a.scale_ld = s->size(1);
    const int64_t es = a.x_dtype == WS_ACT_BF16 ? 2 : 4;
    const bool fits = x.len >= es * a.m * a.k && out.len >= (int64_t)4 * a.m * a.n;
    ws_status_t st = WS_OK;
    if (fits) {
        Py_BEGIN_ALLOW_THREADS
        st = ws_fp8_rowpar_gemm_allreduce_host(tp, &a, x.buf, static_cast<float *>(out.buf));
        Py_END_ALLOW_THREADS
    }
    PyBuffer_Release(&x);
    PyBuffer_Release(&out);
    if (!fits) Py_RETURN_NONE;
    return PyLong_FromLong(st);
    END_HANDLE_TH_ERRORS
}

// moe(handle, h, route_ids, route_w, w2, s2, e_start, out, stream)
PyObject *py_moe(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 9) { PyErr_SetString(PyExc_TypeError, "moe takes 9 arguments"); return nullptr; }
    ws_moe_down_args_t a{};
    ws_tp_t *const tp = static_cast<ws_tp_t *>(PyLong_AsVoidPtr(v[0]));
    const long e_start = PyLong_AsLong(v[6]);
    void *stream;
    if (PyErr_Occurred() || !stream_of(v[8], &stream)) return nullptr;
    if (!fill_moe(a, v[1], v[2], v[3], v[4], v[5], (int32_t)e_start)) Py_RETURN_NONE;
    PyObject *res;
    if (v[7] == Py_None) {
        at::Tensor out = new_f32(THPVariable_Unpack(v[1]), a.m, a.n);
        a.out = out.data_ptr<float>();
        res = THPVariable_Wrap(std::move(out));
    } else {
        const at::Tensor *out = tensor(v[7]);
        if (!out || !holds(*out, a.m, a.n)) Py_RETURN_NONE;
        a.out = static_cast<float *>(out->data_ptr());
        Py_INCREF(v[7]);
        res = v[7];
    }
    WS_CALL(st, ws_moe_down_combine_allreduce(tp, &a, stream))
    return answer(st, res);
    END_HANDLE_TH_ERRORS
}

// head(handle, x, w, scales, block_n, block_k, row0, vocab_row0, vocab, want_logits, stream) -> (logits | None, argmax)
PyObject *py_head(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 11) { PyErr_SetString(PyExc_TypeError, "head takes 11 arguments"); return nullptr; }
    ws_lm_head_args_t a{};
    ws_tp_t *const tp = static_cast<ws_tp_t *>(PyLong_AsVoidPtr(v[0]));
    const long bn = PyLong_AsLong(v[4]), bk = PyLong_AsLong(v[5]), vocab = PyLong_AsLong(v[8]);
    const int64_t row0 = PyLong_AsLongLong(v[6]);
    a.vocab_row0 = PyLong_AsLongLong(v[7]);
    a.vocab = (int32_t)vocab;
    const int want = PyObject_IsTrue(v[9]);
    void *stream;
    if (PyErr_Occurred() || !stream_of(v[10], &stream)) return nullptr;
    if (vocab < 0 || vocab > INT32_MAX || !fill_fp8(a.g, v[1], v[2], v[3], (int32_t)bn, (int32_t)bk, row0, 0)) Py_RETURN_NONE;
    const at::Tensor &x = THPVariable_Unpack(v[1]);
    at::Tensor logits, arg = at::empty({a.g.m}, x.options().dtype(at::kInt).requires_grad(false));
    a.argmax = reinterpret_cast<uint32_t *>(arg.data_ptr<int32_t>());
    if (want) {
        logits = new_f32(x, a.g.m, vocab);
        a.logits = logits.data_ptr<float>();
    }
    WS_CALL(st, ws_lm_head_allgather_argmax(tp, &a, stream))
    if (st != WS_OK) return PyLong_FromLong(st);
    PyObject *first = Py_None;
    if (want) first = THPVariable_Wrap(std::move(logits));
    else Py_INCREF(Py_None);
    PyObject *second = THPVariable_Wrap(std::move(arg));
    PyObject *pair = PyTuple_Pack(2, first, second);
    Py_DECREF(first);
    Py_DECREF(second);
    return pair;
    END_HANDLE_TH_ERRORS
}

// fp8_group(handles, devices, xs, ws, scales, block_n, block_k, row0s | None, k0s | None) -> [out of every rank]
PyObject *py_fp8_group(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 9) { PyErr_SetString(PyExc_TypeError, "fp8_group takes 9 arguments"); return nullptr; }
    if (!PyTuple_Check(v[0]) || !PyTuple_Check(v[1])) Py_RETURN_NONE;
    const Py_ssize_t world = PyTuple_GET_SIZE(v[0]);
    for (int i = 2; i < 5; ++i)
        if (!PyList_Check(v[i]) || PyList_GET_SIZE(v[i]) != world) Py_RETURN_NONE;
    for (int i = 7; i < 9; ++i)
        if (v[i] != Py_None && (!PyList_Check(v[i]) || PyList_GET_SIZE(v[i]) != world)) Py_RETURN_NONE;
    if (world < 1 || world > WS_MAX_WORLD) Py_RETURN_NONE;
    const long bn = PyLong_AsLong(v[5]), bk = PyLong_AsLong(v[6]);
    ws_fp8_gemm_args_t a[WS_MAX_WORLD] = {};
    ws_tp_t *tps[WS_MAX_WORLD];
    void *streams[WS_MAX_WORLD];
    at::Tensor outs[WS_MAX_WORLD];
    for (Py_ssize_t r = 0; r < world; ++r) {
        tps[r] = static_cast<ws_tp_t *>(PyLong_AsVoidPtr(PyTuple_GET_ITEM(v[0], r)));
        const int64_t row0 = v[7] == Py_None ? 0 : PyLong_AsLongLong(PyList_GET_ITEM(v[7], r));
        const int64_t k0 = v[8] == Py_None ? 0 : PyLong_AsLongLong(PyList_GET_ITEM(v[8], r));
        const long dev = PyLong_AsLong(PyTuple_GET_ITEM(v[1], r));
        if (PyErr_Occurred()) return nullptr;
        if (!fill_fp8(a[r], PyList_GET_ITEM(v[2], r), PyList_GET_ITEM(v[3], r), PyList_GET_ITEM(v[4], r), (int32_t)bn, (int32_t)bk, row0, k0))
            Py_RETURN_NONE;
        streams[r] = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
        outs[r] = new_f32(THPVariable_Unpack(PyList_GET_ITEM(v[2], r)), a[r].m, a[r].n);
        a[r].out = outs[r].data_ptr<float>();
    }
    WS_CALL(st, ws_fp8_rowpar_gemm_allreduce_group(tps, (int32_t)world, a, streams))
    if (st != WS_OK) return PyLong_FromLong(st);
    PyObject *list = PyList_New(world);
    for (Py_ssize_t r = 0; list && r < world; ++r) PyList_SET_ITEM(list, r, THPVariable_Wrap(std::move(outs[r])));
    return list;
    END_HANDLE_TH_ERRORS
}

// ---- operators between the steps.  An error's text is the Python layer's to give: it gets None and makes the same call.
//
// Device and stream of a call.  What is allocated meanwhile belongs to the stream that writes it.
struct CallOn {
    c10::cuda::CUDAGuard device;
    std::optional<c10::cuda::CUDAStreamGuard> guard;
    void *stream;
    CallOn(const at::Tensor &t, PyObject *o) : device(t.device()) {
        if (o != Py_None) {
            stream = PyLong_AsVoidPtr(o);
            guard.emplace(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream), t.device().index()));
        } else {
            stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
        }
    }
};

// A [m, n] tensor of rows that are stored one value after the other, on the device of `like`.
bool rows(const at::Tensor *t, const at::Tensor &like, int64_t m, int64_t n, int64_t *ld) {
    if (!t || t->dim() != 2 || t->size(0) != m || t->size(1) != n || t->device() != like.device()) return false;
    if ((n > 1 && t->stride(1) != 1) || (m > 1 && t->stride(0) < n)) return false;
    *ld = m > 1 ? t->stride(0) : n;
    return true;
}
bool vec(const at::Tensor *t, const at::Tensor &like, int64_t n) {
    return t && t->dim() == 1 && t->size(0) == n && t->is_contiguous() && t->device() == like.device();
}
// A result type as Python names it; None stands for `otherwise`.
bool result_dtype(PyObject *o, at::ScalarType otherwise, at::ScalarType *out, int32_t *code) {
    if (o != Py_None && !THPDtype_Check(o)) return false;
    *out = o == Py_None ? otherwise : reinterpret_cast<THPDtype *>(o)->scalar_type;
    *code = *out == at::kFloat ? WS_ACT_F32 : WS_ACT_BF16;
    return *out == at::kFloat || *out == at::kBFloat16;
}
// (the dispatcher's way to the same takes three times as long)
at::Tensor new_like(const at::Tensor &like, at::IntArrayRef sizes, at::ScalarType t) {
    return at::detail::empty_cuda(sizes, t, like.device(), std::nullopt);
}

// block_norm(y, residual, post_weight, next_weight, gate, gate_act, eps, weight_offset, residual_scale, block_scale, out,
//            out_dtype, normed_dtype, stream) -> (hidden, normed | None)
PyObject *py_block_norm(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 14) { PyErr_SetString(PyExc_TypeError, "block_norm takes 14 arguments"); return nullptr; }
    const at::Tensor *y = tensor(v[0]);
    if (!y || y->dim() != 2) Py_RETURN_NONE;
    ws_block_norm_args_t a{};
    const int64_t m = y->size(0), n = y->size(1);
    if (m > INT32_MAX || n > INT32_MAX || !rows(y, *y, m, n, &a.ldy) || !act_dtype(*y, &a.y_dtype)) Py_RETURN_NONE;
    a.m = (int32_t)m; a.n = (int32_t)n; a.y = y->data_ptr();
    at::ScalarType hidden_type = at::kBFloat16, normed_type;
    if (v[1] != Py_None) {
        const at::Tensor *r = tensor(v[1]);
        if (!rows(r, *y, m, n, &a.ldr) || !act_dtype(*r, &a.residual_dtype)) Py_RETURN_NONE;
        a.residual = r->data_ptr();
        hidden_type = r->scalar_type();
    }
    const void **weights[2] = {&a.post_weight, &a.next_weight};
    int32_t seen = -1;
    for (int i = 0; i < 2; ++i) {
        if (v[2 + i] == Py_None) continue;
        const at::Tensor *w = tensor(v[2 + i]);
        if (!vec(w, *y, n) || !act_dtype(*w, &a.weight_dtype) || (seen >= 0 && seen != a.weight_dtype)) Py_RETURN_NONE;
        seen = a.weight_dtype;
        *weights[i] = w->data_ptr();
    }
    a.gate_act = (int32_t)PyLong_AsLong(v[5]);
    if (v[4] != Py_None) {
        const at::Tensor *g = tensor(v[4]);
        if (!g || g->device() != y->device() || g->dim() < 1 || g->dim() > 2 || !act_dtype(*g, &a.gate_dtype)) Py_RETURN_NONE;
        const bool two = g->dim() == 2;
        const int64_t gm = two ? g->size(0) : 1, gn = g->size(two ? 1 : 0), inc = g->stride(two ? 1 : 0);
        if ((gm != 1 && gm != m) || (gn != 1 && gn != n) || (gn > 1 && inc != 0 && inc != 1)) Py_RETURN_NONE;
        a.gate = g->data_ptr();
        a.ldg = gm > 1 ? g->stride(0) : 0;
        a.gate_inc = gn > 1 ? (int32_t)inc : 0;
    }
    a.eps = (float)PyFloat_AsDouble(v[6]); a.weight_offset = (float)PyFloat_AsDouble(v[7]);
    a.residual_scale = (float)PyFloat_AsDouble(v[8]); a.block_scale = (float)PyFloat_AsDouble(v[9]);
    if (PyErr_Occurred()) return nullptr;
    if (!result_dtype(v[11], hidden_type, &hidden_type, &a.hidden_dtype) || !result_dtype(v[12], at::kBFloat16, &normed_type, &a.normed_dtype))
        Py_RETURN_NONE;
    CallOn on(*y, v[13]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor hidden, normed;
    if (v[10] != Py_None) {
        const at::Tensor *out = tensor(v[10]);
        if (!rows(out, *y, m, n, &a.ldh) || !act_dtype(*out, &a.hidden_dtype)) Py_RETURN_NONE;
        a.hidden = out->data_ptr();
    } else {
        hidden = new_like(*y, {m, n}, hidden_type);
        a.hidden = hidden.data_ptr();
        a.ldh = n;
    }
    if (a.next_weight) {
        normed = new_like(*y, {m, n}, normed_type);
        a.normed = normed.data_ptr();
        a.ldn = n;
    }
    WS_CALL(st, ws_block_norm(&a, on.stream, nullptr, 0))
    if (st != WS_OK) Py_RETURN_NONE;
    PyObject *first = v[10], *second = Py_None;
    if (hidden.defined()) first = THPVariable_Wrap(std::move(hidden));
    else Py_INCREF(first);
    if (normed.defined()) second = THPVariable_Wrap(std::move(normed));
    else Py_INCREF(second);
    PyObject *pair = PyTuple_Pack(2, first, second);
    Py_DECREF(first);
    Py_DECREF(second);
    return pair;
    END_HANDLE_TH_ERRORS
}

// token_logprobs(logits, tokens, top, stream) -> (logprobs, entropy, rank, top_ids | None, top_logprobs | None)
PyObject *py_token_logprobs(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 4) { PyErr_SetString(PyExc_TypeError, "token_logprobs takes 4 arguments"); return nullptr; }
    const at::Tensor *x = tensor(v[0]), *tok = tensor(v[1]);
    const long top = PyLong_AsLong(v[2]);
    if (PyErr_Occurred()) return nullptr;
    if (!x || !tok || x->dim() != 2 || top < 0 || top > WS_MAX_TOP) Py_RETURN_NONE;
    ws_token_logprobs_args_t a{};
    const int64_t m = x->size(0), vocab = x->size(1);
    if (m > INT32_MAX || vocab > INT32_MAX || !rows(x, *x, m, vocab, &a.ld) || !act_dtype(*x, &a.dtype) || !vec(tok, *x, m)) Py_RETURN_NONE;
    if (tok->scalar_type() != at::kInt && tok->scalar_type() != at::kLong) Py_RETURN_NONE;
    a.logits = x->data_ptr(); a.tokens = tok->data_ptr(); a.token_bytes = (int32_t)tok->element_size();
    a.m = (int32_t)m; a.vocab = (int32_t)vocab; a.top = (int32_t)top;
    CallOn on(*x, v[3]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor out[5];
    out[0] = new_like(*x, {m}, at::kFloat); out[1] = new_like(*x, {m}, at::kFloat); out[2] = new_like(*x, {m}, at::kInt);
    a.logprob = out[0].data_ptr<float>(); a.entropy = out[1].data_ptr<float>(); a.rank = out[2].data_ptr<int32_t>();
    if (top) {
        out[3] = new_like(*x, {m, top}, at::kInt); out[4] = new_like(*x, {m, top}, at::kFloat);
        a.top_id = out[3].data_ptr<int32_t>(); a.top_logprob = out[4].data_ptr<float>();
    }
    WS_CALL(st, ws_token_logprobs(&a, on.stream, nullptr, 0))
    if (st != WS_OK) Py_RETURN_NONE;
    PyObject *res = PyTuple_New(5);
    for (int i = 0; res && i < 5; ++i) {
        PyObject *o = Py_None;
        if (out[i].defined()) o = THPVariable_Wrap(std::move(out[i]));
        else Py_INCREF(o);
        PyTuple_SET_ITEM(res, i, o);
    }
    return res;
    END_HANDLE_TH_ERRORS
}

// lora(what, y, x, a, b, ids, scale, shrunk, out, stream) -> out | shrunk; what: 0 add (y x a b), 1 shrink (x a), 2 expand (y b shrunk)
PyObject *py_lora(PyObject *, PyObject *const *v, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 10) { PyErr_SetString(PyExc_TypeError, "lora takes 10 arguments"); return nullptr; }
    const long what = PyLong_AsLong(v[0]);
    if (PyErr_Occurred()) return nullptr;
    const bool shrinks = what != 2, expands = what != 1;
    const at::Tensor *ids = tensor(v[5]);
    if (!ids || ids->dim() != 1 || !ids->is_contiguous() || ids->scalar_type() != at::kInt) Py_RETURN_NONE;
    const int64_t m = ids->size(0);
    int64_t adapters = 0, rank = 0, k = 0, n = 0;
    ws_lora_args_t a{};
    a.ids = ids->data_ptr<int32_t>();
    if (shrinks) {
        const at::Tensor *x = tensor(v[2]), *w = tensor(v[3]);
        if (!x || !w || w->dim() != 3 || !w->is_contiguous() || w->scalar_type() != at::kBFloat16 || w->device() != ids->device()) Py_RETURN_NONE;
        adapters = w->size(0); rank = w->size(1); k = w->size(2);
        if (!rows(x, *ids, m, k, &a.ldx) || !act_dtype(*x, &a.x_dtype)) Py_RETURN_NONE;
        a.x = x->data_ptr(); a.a = w->data_ptr();
    }
    const at::Tensor *y = nullptr;
    if (expands) {
        const at::Tensor *w = tensor(v[4]);
        y = tensor(v[1]);
        if (!y || !w || w->dim() != 3 || !w->is_contiguous() || w->scalar_type() != at::kBFloat16 || w->device() != ids->device()) Py_RETURN_NONE;
        if (shrinks && (w->size(0) != adapters || w->size(2) != rank)) Py_RETURN_NONE;
        adapters = w->size(0); n = w->size(1); rank = w->size(2);
        if (!rows(y, *ids, m, n, &a.ldy) || !act_dtype(*y, &a.y_dtype)) Py_RETURN_NONE;
        a.y = y->data_ptr(); a.b = w->data_ptr();
        if (v[6] != Py_None) {
            const at::Tensor *s = tensor(v[6]);
            if (!vec(s, *ids, adapters) || s->scalar_type() != at::kFloat) Py_RETURN_NONE;
            a.scale = s->data_ptr<float>();
        }
    }
    if (m > INT32_MAX || adapters > INT32_MAX || rank > INT32_MAX || k > INT32_MAX || n > INT32_MAX) Py_RETURN_NONE;
    a.m = (int32_t)m; a.adapters = (int32_t)adapters; a.rank = (int32_t)rank; a.k = (int32_t)k; a.n = (int32_t)n;
    if (what == 2) {
        const at::Tensor *s = tensor(v[7]);
        if (!s || s->dim() != 2 || s->size(0) != m || s->size(1) != rank || !s->is_contiguous() || s->scalar_type() != at::kFloat ||
            s->device() != ids->device())
            Py_RETURN_NONE;
        a.shrunk = s->data_ptr<float>();
    }
    CallOn on(*ids, v[9]);
    if (PyErr_Occurred()) return nullptr;
    at::Tensor made;
    if (expands && v[8] != Py_None) {
        const at::Tensor *out = tensor(v[8]);
        if (!rows(out, *ids, m, n, &a.ldo) || out->scalar_type() != y->scalar_type()) Py_RETURN_NONE;
        a.out = out->data_ptr();
    } else if (expands) {
        made = new_like(*y, {m, n}, y->scalar_type());
        a.out = made.data_ptr();
        a.ldo = n;
    } else {
        made = new_like(*ids, {m, rank}, at::kFloat);
        a.shrunk = made.data_ptr<float>();
    }
    at::Tensor work;
    a.workspace_bytes = ws_lora_workspace(a.m, a.adapters, a.rank);
    if (a.workspace_bytes > 0) {
        work = new_like(*ids, {a.workspace_bytes}, at::kByte);
        a.workspace = work.data_ptr();
    }
    WS_CALL(st, what == 0 ? ws_lora_add(&a, on.stream, nullptr, 0) : what == 1 ? ws_lora_shrink(&a, on.stream, nullptr, 0)
                                                                                : ws_lora_expand(&a, on.stream, nullptr, 0))
    if (st != WS_OK) Py_RETURN_NONE;
    if (made.defined()) return THPVariable_Wrap(std::move(made));
    Py_INCREF(v[8]);
    return v[8];
    END_HANDLE_TH_ERRORS
}

#define WS_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {WS_METHOD(fp8), WS_METHOD(fp8_host), WS_METHOD(moe), WS_METHOD(head), WS_METHOD(fp8_group), WS_METHOD(block_norm), WS_METHOD(lora), WS_METHOD(token_logprobs),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_ws_torch", "torch tensors -> libws_tp.so", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ws_torch(void) { return PyModule_Create(&module_def); }

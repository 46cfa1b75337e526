// Host side of the operators of include/fa_ops.h in the host module: outputs and
// workspace from torch, the argument struct, the library call.  The Python layer
// has checked shapes, dtypes and devices; layouts that the kernels cannot read
// are copied here.  Every call is self-contained and runs with the tensors'
// device current.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "fa_host_util.hpp"
#include "fa_ops.h"

namespace {

using fa_host::dtype_code;
using fa_host::prepare;
using fa_host::put_strides;

decltype(&fa_scored_fwd_workspace_size) p_fwd_size;
decltype(&fa_scored_fwd) p_fwd;
decltype(&fa_scored_bwd_workspace_size) p_bwd_size;
decltype(&fa_scored_bwd) p_bwd;
decltype(&fa_prefix_workspace_size) p_prefix_size;
decltype(&fa_prefix_fwd) p_prefix;
decltype(&fa_rotary) p_rotary;

bool check_count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return false;
}
bool bound() {
    if (p_fwd) return true;
    PyErr_SetString(PyExc_RuntimeError, "the host module is not bound to the kernel library");
    return false;
}
bool all_tensors(PyObject* const* x, Py_ssize_t n) {
    for (Py_ssize_t i = 0; i < n; ++i)
        if (!THPVariable_Check(x[i])) {
            PyErr_SetString(PyExc_TypeError, "expected a tensor");
            return false;
        }
    return true;
}
bool none(PyObject* o) { return o == Py_None; }
int32_t i32(int64_t n) {
    TORCH_CHECK(n <= INT32_MAX, "size ", n, " exceeds the operators' limit of 2^31 - 1");
    return (int32_t)n;
}

// an optional integer array as contiguous int32 (held by `keep`), or null
const int32_t* lengths(PyObject* o, at::Tensor& keep) {
    if (none(o)) return nullptr;
    keep = THPVariable_Unpack(o);
    if (keep.scalar_type() == at::kLong) keep = keep.clamp(INT32_MIN, INT32_MAX);  // out of range stays so
    if (keep.scalar_type() != at::kInt || !keep.is_contiguous()) keep = keep.to(at::kInt).contiguous();
    return (const int32_t*)keep.data_ptr();
}
// document ids (B, S) as int32 with token stride 1 and any batch stride
const int32_t* documents(PyObject* o, at::Tensor& keep, int64_t& stride) {
    stride = 0;
    if (none(o)) return nullptr;
    keep = THPVariable_Unpack(o);
    // an id past int32 must not become another one's: it counts as padding
    if (keep.scalar_type() == at::kLong) keep = at::where(keep.gt(INT32_MAX), -1, keep.clamp_min(-1));
    if (keep.scalar_type() != at::kInt || (keep.size(1) > 1 && keep.stride(1) != 1)) keep = keep.to(at::kInt).contiguous();
    stride = keep.size(0) > 1 ? keep.stride(0) : 0;
    return (const int32_t*)keep.data_ptr();
}
const float* slopes_of(PyObject* o, at::Tensor& keep, int64_t& stride) {
    stride = 0;
    if (none(o)) return nullptr;
    keep = THPVariable_Unpack(o).contiguous();
    stride = keep.dim() == 2 ? keep.size(1) : 0;
    return (const float*)keep.data_ptr();
}

// tensors that an argument struct points into
struct Held {
    at::Tensor t[8];
};

// the rules, from (causal, scale, softcap, slopes, prefix, lens, offsets,
// offset0, q_docs, k_docs)
bool put_rules(fa_scored_args& a, Held& h, PyObject* const* x) {
    a.causal = PyObject_IsTrue(x[0]);
    a.scale = (float)PyFloat_AsDouble(x[1]);
    a.softcap = (float)PyFloat_AsDouble(x[2]);
    a.slopes = slopes_of(x[3], h.t[0], a.slopes_batch_stride);
    a.prefix_lengths = lengths(x[4], h.t[1]);
    a.key_lengths = lengths(x[5], h.t[2]);
    a.query_offsets = lengths(x[6], h.t[3]);
    a.query_offset = (int32_t)PyLong_AsLong(x[7]);
    a.q_documents = documents(x[8], h.t[4], a.q_documents_stride);
    if (x[9] == x[8]) {
        a.k_documents = a.q_documents;
        a.k_documents_stride = a.q_documents_stride;
    } else {
        a.k_documents = documents(x[9], h.t[5], a.k_documents_stride);
    }
    return !PyErr_Occurred();
}
constexpr int kRules = 10;

void put_sizes(fa_scored_args& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    put_strides(a.q_stride, q);
    put_strides(a.k_stride, k);
    put_strides(a.v_stride, v);
    a.batch = i32(q.size(0));
    a.seqlen_q = i32(q.size(1));
    a.seqlen_k = i32(k.size(1));
    a.num_heads = i32(q.size(2));
    a.num_heads_kv = i32(k.size(2));
    a.head_dim = i32(q.size(3));
    a.dtype = dtype_code(q.scalar_type());
}

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

PyObject* wrap_or_none(const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

// What the Python entry points look at before every call, in one: False sends them
// to their own checks, which name what is wrong.
bool element_type(const at::Tensor& t) { return dtype_code(t.scalar_type()) >= 0; }

// A tensor of forward-mode differentiation, whose tangent a kernel would drop.  (It
// need not require grad; torch has one level of them.)
bool dual(const at::Tensor& t) {
    return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined();
}

// dual(tensor or None, ...): whether one of them is
PyObject* any_dual(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    for (Py_ssize_t i = 0; i < n; ++i)
        if (THPVariable_Check(x[i]) && dual(THPVariable_Unpack(x[i]))) Py_RETURN_TRUE;
    Py_RETURN_FALSE;
    END_HANDLE_TH_ERRORS
}

// qkv_ok(q, k, v, largest head dim)
PyObject* qkv_ok(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 4)) return nullptr;
    const int64_t most = PyLong_AsLongLong(x[3]);
    if (PyErr_Occurred()) return nullptr;
    for (int i = 0; i < 3; ++i)
        if (!THPVariable_Check(x[i]) || THPVariable_Unpack(x[i]).dim() != 4) Py_RETURN_FALSE;
    const at::Tensor &q = THPVariable_Unpack(x[0]), &k = THPVariable_Unpack(x[1]), &v = THPVariable_Unpack(x[2]);
    const int64_t H = q.size(2), Hkv = k.size(2), D = q.size(3);
    const bool ok = q.is_cuda() && k.device() == q.device() && v.device() == q.device() && element_type(q) &&
                    k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
                    k.size(0) == q.size(0) && k.size(3) == D && k.sizes() == v.sizes() && Hkv > 0 && H > 0 &&
                    H % Hkv == 0 && D > 0 && D <= most && !dual(q) && !dual(k) && !dual(v);
    return PyBool_FromLong(ok);
    END_HANDLE_TH_ERRORS
}

// rotary_ok(q, k or None, table, positions or None): positions of shape (B, S)
PyObject* rotary_ok(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 4)) return nullptr;
    for (int i = 0; i < 4; ++i)
        if (!THPVariable_Check(x[i]) && !((i & 1) && none(x[i]))) Py_RETURN_FALSE;
    const at::Tensor &q = THPVariable_Unpack(x[0]), &t = THPVariable_Unpack(x[2]);
    if (q.dim() != 4 || t.dim() != 2) Py_RETURN_FALSE;
    const int64_t B = q.size(0), S = q.size(1), D = q.size(3), R = t.size(1);
    bool ok = q.is_cuda() && element_type(q) && q.size(2) > 0 && D <= 256 && t.device() == q.device() &&
              t.scalar_type() == at::kFloat && !t.requires_grad() && R >= 2 && R % 2 == 0 && R <= D && t.size(0) > 0 &&
              !dual(q) && !dual(t);
    if (ok && !none(x[1])) {
        const at::Tensor& k = THPVariable_Unpack(x[1]);
        ok = k.dim() == 4 && k.device() == q.device() && k.scalar_type() == q.scalar_type() && k.size(0) == B &&
             k.size(1) == S && k.size(2) > 0 && k.size(3) == D && !dual(k);
    }
    if (ok && !none(x[3])) {
        const at::Tensor& p = THPVariable_Unpack(x[3]);
        ok = p.dim() == 2 && p.size(0) == B && p.size(1) == S && p.device() == q.device() &&
             (p.scalar_type() == at::kInt || p.scalar_type() == at::kLong);
    }
    return PyBool_FromLong(ok);
    END_HANDLE_TH_ERRORS
}

// Whether the backward needs lse_near beside lse: slopes, and a query may stand so far
// off the keys that the rounding of its lse counts (up to 512: 2^-16 of P times the slope)
bool wants_near(const fa_scored_args& a) {
    const int64_t first = a.query_offset, end = first + a.seqlen_q;
    const bool off = a.key_lengths || first < 0 || end > a.seqlen_k;
    return a.slopes && (a.query_offsets || (off && (first < -512 || end > 512)));
}

// scored_fwd(q, k, v, <rules>, want_lse, for a backward, stream)
//   -> (status, o, lse or None, lse_near or None)
PyObject* scored_fwd(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 3 + kRules + 3) || !bound() || !all_tensors(x, 3)) return nullptr;
    c10::DeviceGuard guard(THPVariable_Unpack(x[0]).device());
    const at::Tensor q = prepare(THPVariable_Unpack(x[0])), k = prepare(THPVariable_Unpack(x[1])),
                     v = prepare(THPVariable_Unpack(x[2]));
    fa_scored_args a = {};
    Held h;
    if (!put_rules(a, h, x + 3)) return nullptr;
    const bool want = PyObject_IsTrue(x[3 + kRules]) == 1, back = PyObject_IsTrue(x[3 + kRules + 1]) == 1;
    void* const stream = PyLong_AsVoidPtr(x[3 + kRules + 2]);
    if (PyErr_Occurred()) return nullptr;
    put_sizes(a, q, k, v);
    const at::Tensor o = at::empty(q.sizes(), q.options());
    const at::Tensor lse =
        want ? at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat)) : at::Tensor();
    a.o = o.data_ptr();
    put_strides(a.o_stride, o);
    a.lse = (float*)ptr(lse);
    const at::Tensor near = back && wants_near(a) ? at::empty_like(lse) : at::Tensor();
    a.lse_near = (float*)ptr(near);
    const size_t bytes = p_fwd_size(&a);
    const at::Tensor ws = workspace(bytes, q);
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_fwd(&a, ptr(ws), bytes, stream);
    }
    return Py_BuildValue("(iNNN)", (int)st, THPVariable_Wrap(o), wrap_or_none(lse), wrap_or_none(near));
    END_HANDLE_TH_ERRORS
}

// scored_bwd(q, k, v, o, do, lse, lse_near or None, <rules>, want_dslopes, stream)
//   -> (status, dq, dk, dv, dslopes or None)
PyObject* scored_bwd(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 7 + kRules + 2) || !bound() || !all_tensors(x, 6)) return nullptr;
    if (!none(x[6]) && !all_tensors(x + 6, 1)) return nullptr;
    c10::DeviceGuard guard(THPVariable_Unpack(x[0]).device());
    const at::Tensor q = prepare(THPVariable_Unpack(x[0])), k = prepare(THPVariable_Unpack(x[1])),
                     v = prepare(THPVariable_Unpack(x[2])), o = prepare(THPVariable_Unpack(x[3])),
                     dout = prepare(THPVariable_Unpack(x[4]));
    const at::Tensor lse = THPVariable_Unpack(x[5]).contiguous();
    fa_scored_args a = {};
    Held h;
    if (!put_rules(a, h, x + 7)) return nullptr;
    const bool want = PyObject_IsTrue(x[7 + kRules]) == 1;
    void* const stream = PyLong_AsVoidPtr(x[7 + kRules + 1]);
    if (PyErr_Occurred()) return nullptr;
    put_sizes(a, q, k, v);
    const at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
                     dv = at::empty(v.sizes(), v.options());
    const at::Tensor ds = want && a.slopes ? at::empty(h.t[0].sizes(), h.t[0].options()) : at::Tensor();
    a.o = o.data_ptr();
    a.dout = dout.data_ptr();
    a.lse = (float*)lse.data_ptr();
    const at::Tensor near = none(x[6]) ? at::Tensor() : THPVariable_Unpack(x[6]).contiguous();
    a.lse_near = (float*)ptr(near);
    a.dq = dq.data_ptr();
    a.dk = dk.data_ptr();
    a.dv = dv.data_ptr();
    a.dslopes = (float*)ptr(ds);
    put_strides(a.o_stride, o);
    put_strides(a.do_stride, dout);
    put_strides(a.dq_stride, dq);
    put_strides(a.dk_stride, dk);
    put_strides(a.dv_stride, dv);
    const size_t bytes = p_bwd_size(&a);
    const at::Tensor ws = workspace(bytes, q);
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_bwd(&a, ptr(ws), bytes, stream);
    }
    return Py_BuildValue("(iNNNN)", (int)st, THPVariable_Wrap(dq), THPVariable_Wrap(dk), THPVariable_Wrap(dv),
                         wrap_or_none(ds));
    END_HANDLE_TH_ERRORS
}

// prefix_fwd(q, k_prefix, v_prefix, k, v, scale, softcap, slopes, lens, want_lse,
//     stream) -> (status, o, lse or None)
PyObject* prefix_fwd(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 11) || !bound() || !all_tensors(x, 5)) return nullptr;
    c10::DeviceGuard guard(THPVariable_Unpack(x[0]).device());
    at::Tensor t[5];
    for (int i = 0; i < 5; ++i) t[i] = prepare(THPVariable_Unpack(x[i]));
    fa_prefix_args a = {};
    Held h;
    a.scale = (float)PyFloat_AsDouble(x[5]);
    a.softcap = (float)PyFloat_AsDouble(x[6]);
    a.slopes = slopes_of(x[7], h.t[0], a.slopes_batch_stride);
    a.key_lengths = lengths(x[8], h.t[1]);
    const bool want = PyObject_IsTrue(x[9]) == 1;
    void* const stream = PyLong_AsVoidPtr(x[10]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor& q = t[0];
    a.q = q.data_ptr();
    a.k_prefix = t[1].data_ptr();
    a.v_prefix = t[2].data_ptr();
    a.k = t[3].data_ptr();
    a.v = t[4].data_ptr();
    put_strides(a.q_stride, q);
    for (int d = 0; d < 3; ++d) {
        a.kp_stride[d] = t[1].stride(d);
        a.vp_stride[d] = t[2].stride(d);
    }
    put_strides(a.k_stride, t[3]);
    put_strides(a.v_stride, t[4]);
    a.batch = i32(q.size(0));
    a.seqlen_q = i32(q.size(1));
    a.prefix_len = i32(t[1].size(0));
    a.seqlen_k = i32(t[3].size(1));
    a.num_heads = i32(q.size(2));
    a.num_heads_kv = i32(t[3].size(2));
    a.head_dim = i32(q.size(3));
    a.dtype = dtype_code(q.scalar_type());
    const at::Tensor o = at::empty(q.sizes(), q.options());
    const at::Tensor lse =
        want ? at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat)) : at::Tensor();
    a.o = o.data_ptr();
    put_strides(a.o_stride, o);
    a.lse = (float*)ptr(lse);
    const size_t bytes = p_prefix_size(&a);
    const at::Tensor ws = workspace(bytes, q);
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_prefix(&a, ptr(ws), bytes, stream);
    }
    return Py_BuildValue("(iNN)", (int)st, THPVariable_Wrap(o), wrap_or_none(lse));
    END_HANDLE_TH_ERRORS
}

// rotary(q, k or None, table, positions or None, interleaved, inverse, inplace,
//     stream) -> (status, q_out, k_out or None)
PyObject* rotary(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 8) || !bound() || !all_tensors(x, 1) || !all_tensors(x + 2, 1)) return nullptr;
    const at::Tensor& q0 = THPVariable_Unpack(x[0]);
    c10::DeviceGuard guard(q0.device());
    const bool inplace = PyObject_IsTrue(x[6]) == 1;
    // the d stride is 1 (in place: the Python layer has checked)
    auto unit = [](const at::Tensor& t) {
        bool ok = t.size(3) == 1 || t.stride(3) == 1;
        for (int d = 0; d < 3; ++d) ok = ok && t.stride(d) >= 0;
        return ok ? t : t.contiguous();
    };
    const at::Tensor q = inplace ? q0 : unit(q0);
    const at::Tensor k = none(x[1]) ? at::Tensor() : inplace ? THPVariable_Unpack(x[1]) : unit(THPVariable_Unpack(x[1]));
    const at::Tensor table = THPVariable_Unpack(x[2]).contiguous();
    const at::Tensor qo = inplace ? q : at::empty(q.sizes(), q.options());
    const at::Tensor ko = !k.defined() ? at::Tensor() : inplace ? k : at::empty(k.sizes(), k.options());
    fa_rotary_args a = {};
    auto strides = [](int64_t (&dst)[4], const at::Tensor& t) {
        put_strides(dst, t);
        dst[3] = 1;
    };
    a.q = q.data_ptr();
    a.q_out = qo.data_ptr();
    strides(a.q_stride, q);
    strides(a.q_out_stride, qo);
    if (k.defined()) {
        a.k = k.data_ptr();
        a.k_out = ko.data_ptr();
        strides(a.k_stride, k);
        strides(a.k_out_stride, ko);
        a.num_heads_k = i32(k.size(2));
    }
    a.table = (const float*)table.data_ptr();
    a.table_positions = table.size(0);
    a.rotary_dim = i32(table.size(1));
    if (!none(x[3])) {
        const at::Tensor& p = THPVariable_Unpack(x[3]);  // (B, S), int32 or int64
        a.positions = p.data_ptr();
        a.positions_stride[0] = p.size(0) > 1 ? p.stride(0) : 0;
        a.positions_stride[1] = p.size(1) > 1 ? p.stride(1) : 0;
        a.positions_64 = p.scalar_type() == at::kLong;
    }
    a.interleaved = PyObject_IsTrue(x[4]);
    a.inverse = PyObject_IsTrue(x[5]);
    void* const stream = PyLong_AsVoidPtr(x[7]);
    if (PyErr_Occurred()) return nullptr;
    a.batch = i32(q.size(0));
    a.seqlen = i32(q.size(1));
    a.num_heads = i32(q.size(2));
    a.head_dim = i32(q.size(3));
    a.dtype = dtype_code(q.scalar_type());
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_rotary(&a, stream);
    }
    if (inplace && !st) {
        fa_host::written(q);
        if (k.defined()) fa_host::written(k);
    }
    return Py_BuildValue("(iNN)", (int)st, THPVariable_Wrap(qo), wrap_or_none(ko));
    END_HANDLE_TH_ERRORS
}

// on_other_stream(tensor or None, ...): whether the gradient of one of them would be
// handed on to a stream other than its device's current one: the stream that its
// node (a leaf's accumulator, if an older graph keeps it alive) was made on
PyObject* on_other_stream(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (none(x[i])) continue;
        if (!all_tensors(x + i, 1)) return nullptr;
        const at::Tensor& t = THPVariable_Unpack(x[i]);
        if (!t.requires_grad()) continue;
        const std::shared_ptr<torch::autograd::Node> node =
            t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
        const auto st = node ? node->stream() : std::nullopt;
        if (st && *st != c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device())) Py_RETURN_TRUE;
    }
    Py_RETURN_FALSE;
    END_HANDLE_TH_ERRORS
}

// bind_ops(fa_ops_version, sizeof(fa_scored_args), sizeof(fa_prefix_args),
//     sizeof(fa_rotary_args), then the addresses of the functions above in their
//     order); refused for another version or other struct sizes, as bind is
PyObject* bind_ops(PyObject*, PyObject* const* x, Py_ssize_t n) {
    if (!check_count(n, 11)) return nullptr;
    void* p[8];
    for (int i = 0; i < 8; ++i) {
        p[i] = PyLong_AsVoidPtr(x[i == 0 ? 0 : i + 3]);
        if (PyErr_Occurred()) return nullptr;
        if (!p[i]) {
            PyErr_SetString(PyExc_ValueError, "bind_ops: null address");
            return nullptr;
        }
    }
    const size_t sizes[3] = {PyLong_AsSize_t(x[1]), PyLong_AsSize_t(x[2]), PyLong_AsSize_t(x[3])};
    if (PyErr_Occurred()) return nullptr;
    const int32_t version = ((decltype(&fa_ops_version))p[0])();
    if (version != FA_OPS_VERSION || sizes[0] != sizeof(fa_scored_args) || sizes[1] != sizeof(fa_prefix_args) ||
        sizes[2] != sizeof(fa_rotary_args)) {
        PyErr_Format(PyExc_RuntimeError,
                     "fa_host was built for operator version %d with argument structs of %zu, %zu and %zu bytes; the "
                     "library has version %d, the binding %zu, %zu and %zu bytes",
                     FA_OPS_VERSION, sizeof(fa_scored_args), sizeof(fa_prefix_args), sizeof(fa_rotary_args), (int)version,
                     sizes[0], sizes[1], sizes[2]);
        return nullptr;
    }
    p_fwd_size = (decltype(p_fwd_size))p[1];
    p_fwd = (decltype(p_fwd))p[2];
    p_bwd_size = (decltype(p_bwd_size))p[3];
    p_bwd = (decltype(p_bwd))p[4];
    p_prefix_size = (decltype(p_prefix_size))p[5];
    p_prefix = (decltype(p_prefix))p[6];
    p_rotary = (decltype(p_rotary))p[7];
    Py_RETURN_NONE;
}

}  // namespace

PyMethodDef fa_host::ops_methods[] = {
    {"bind_ops", (PyCFunction)(void*)bind_ops, METH_FASTCALL, nullptr},
    {"dual", (PyCFunction)(void*)any_dual, METH_FASTCALL, nullptr},
    {"qkv_ok", (PyCFunction)(void*)qkv_ok, METH_FASTCALL, nullptr},
    {"rotary_ok", (PyCFunction)(void*)rotary_ok, METH_FASTCALL, nullptr},
    {"scored_fwd", (PyCFunction)(void*)scored_fwd, METH_FASTCALL, nullptr},
    {"scored_bwd", (PyCFunction)(void*)scored_bwd, METH_FASTCALL, nullptr},
    {"prefix_fwd", (PyCFunction)(void*)prefix_fwd, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void*)rotary, METH_FASTCALL, nullptr},
    {"on_other_stream", (PyCFunction)(void*)on_other_stream, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

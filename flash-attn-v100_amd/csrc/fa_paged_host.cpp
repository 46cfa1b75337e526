// Host side of the operators of include/fa_paged.h in the host module: outputs and
// workspace from torch, the argument struct, the library call.  The Python layer
// has checked shapes, dtypes, devices and the pools' layout, which is never copied.
// Every call is self-contained and runs with the pools' device current.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>

#include "fa_host_util.hpp"
#include "fa_paged.h"

namespace {

using fa_host::dtype_code;
using fa_host::prepare;
using fa_host::put_strides;

decltype(&fa_paged_workspace_size) p_paged_size;
decltype(&fa_paged_fwd) p_paged;
decltype(&fa_cache_write) p_write;
decltype(&fa_cache_accept) p_accept;
decltype(&fa_cache_fork_workspace_size) p_fork_size;
decltype(&fa_cache_fork) p_fork;
decltype(&fa_cache_compact_workspace_size) p_compact_size;
decltype(&fa_cache_compact) p_compact;

// the arguments' number, and that the first `tensors` of them are tensors
bool check(Py_ssize_t n, Py_ssize_t want, PyObject* const* x, int tensors) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
        return false;
    }
    if (!p_paged) {
        PyErr_SetString(PyExc_RuntimeError, "the host module is not bound to the kernel library");
        return false;
    }
    for (int i = 0; i < tensors; ++i)
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
// an integer array as int32 with column stride 1 (held by the result); values past int32
// stay out of every range
at::Tensor ints(const at::Tensor& t) {
    at::Tensor x = t.scalar_type() == at::kLong ? t.clamp(INT32_MIN, INT32_MAX).to(at::kInt) : t;
    const int64_t d = x.dim() - 1;
    return x.size(d) <= 1 || x.stride(d) == 1 ? x : x.contiguous();
}
at::Tensor ints(PyObject* o) { return none(o) ? at::Tensor() : ints(THPVariable_Unpack(o)); }
template <typename P>
P* ptr(const at::Tensor& t) {
    return t.defined() && t.numel() ? (P*)t.data_ptr() : nullptr;
}
int64_t row_stride(const at::Tensor& t) { return t.defined() && t.dim() == 2 && t.size(0) > 1 ? t.stride(0) : 0; }

// the pool struct of k, v (pages, rows, heads, d) or with a leading dimension of layers
struct Pool {
    at::Tensor table, lens;
    void put(fa_page_pool& c, const at::Tensor& k, const at::Tensor& v, PyObject* o_table, PyObject* o_lens, int64_t batch) {
        table = ints(o_table);
        lens = ints(o_lens);
        if (lens.defined()) lens = lens.contiguous();
        const int64_t x = k.dim() - 4;
        c.k = k.data_ptr();
        c.v = v.data_ptr();
        for (int64_t i = 0; i < 5; ++i) {
            c.k_stride[i] = i + x >= 1 ? k.stride(i + x - 1) : 0;
            c.v_stride[i] = i + x >= 1 ? v.stride(i + x - 1) : 0;
        }
        c.layers = x ? i32(k.size(0)) : 1;
        c.pages = i32(k.size(x));
        c.page_size = i32(k.size(x + 1));
        c.num_heads_kv = i32(k.size(x + 2));
        c.head_dim = i32(k.size(x + 3));
        c.dtype = dtype_code(k.scalar_type());
        c.batch = i32(batch);
        c.table_cols = table.defined() ? i32(table.size(1)) : 1;
        c.page_table = ptr<const int32_t>(table);
        c.table_stride = row_stride(table);
        c.key_lengths = ptr<const int32_t>(lens);
    }
};

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

bool dual(const at::Tensor& t) {
    return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined();
}
bool wants_grad(const at::Tensor& t) { return t.requires_grad() && c10::GradMode::is_enabled(); }

// Whether two tensors share an element.  One of a and one of b are the same if, counted from
// the first of a, sum s_i x_i = (last of b) - sum t_j y_j with 0 <= x_i < n_i, 0 <= y_j < m_j: a
// sum of non-negative terms (those of one stride are one), tried from the longest stride
// down, whose rest must be within the reach of the shorter ones.  A tensor's strides mostly
// hold what is inside them, so that few multiples of each are left to try; where it takes
// too many, false: what the caller has to see to.
struct Terms {
    struct Term {
        int64_t stride, n;  // bytes; the largest multiple
    } at[16];
    int64_t reach[17];  // of terms from i on
    int count = 0, work = 10000;
    void add(const at::Tensor& t) {
        for (int64_t d = 0; d < t.dim(); ++d)
            if (t.size(d) > 1 && t.stride(d) != 0) at[count++] = {t.stride(d) * t.element_size(), t.size(d) - 1};
    }
    void order() {
        std::sort(at, at + count, [](const Term& a, const Term& b) { return a.stride > b.stride; });
        int m = 0;
        for (int i = 0; i < count; ++i)
            if (m && at[m - 1].stride == at[i].stride)
                at[m - 1].n += at[i].n;
            else
                at[m++] = at[i];
        count = m;
        reach[m] = 0;
        for (int i = m; i-- > 0;) reach[i] = reach[i + 1] + at[i].stride * at[i].n;
    }
    bool meets(int i, int64_t rest) {
        if (rest < 0 || rest > reach[i] || --work < 0) return false;
        if (rest == 0) return true;
        const int64_t low = rest - reach[i + 1];
        for (int64_t x = std::min(at[i].n, rest / at[i].stride); x >= 0 && x * at[i].stride >= low; --x)
            if (meets(i + 1, rest - x * at[i].stride)) return true;
        return false;
    }
};
bool share(const at::Tensor& a, const at::Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0 || a.dim() > 8 || b.dim() > 8 || a.device() != b.device()) return false;
    auto last = [](const at::Tensor& t) {  // (torch has no negative strides)
        intptr_t x = (intptr_t)t.data_ptr();
        for (int64_t d = 0; d < t.dim(); ++d) x += (t.size(d) - 1) * t.stride(d) * t.element_size();
        return x;
    };
    const intptr_t a0 = (intptr_t)a.data_ptr(), a1 = last(a), b0 = (intptr_t)b.data_ptr(), b1 = last(b);
    if (a1 < b0 || b1 < a0) return false;
    Terms t;
    t.add(a);
    t.add(b);
    t.order();
    return t.meets(0, b1 - a0);
}

// What the Python entry points look at before every call, in one: False sends them to
// their own checks, which name what is wrong.
bool integer(PyObject* o, const at::Tensor& k, int64_t dim) {
    if (!THPVariable_Check(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.dim() == dim && t.device() == k.device() && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong);
}
// a cache and its table and lengths (or None) of `batch` sequences (below 0: of the table's)
bool cache_ok(PyObject* ok, PyObject* ov, PyObject* table, PyObject* lens, int64_t batch, bool written) {
    if (!THPVariable_Check(ok) || !THPVariable_Check(ov)) return false;
    const at::Tensor &k = THPVariable_Unpack(ok), &v = THPVariable_Unpack(ov);
    const int64_t d = k.dim();
    if ((d != 4 && !(written && d == 5)) || !k.is_cuda() || k.sizes() != v.sizes() || v.device() != k.device() ||
        v.scalar_type() != k.scalar_type() || dtype_code(k.scalar_type()) < 0 || dual(k) || dual(v) || wants_grad(k) || wants_grad(v))
        return false;
    const int64_t es = k.element_size(), D = k.size(d - 1);
    if (D <= 0 || D > 128 || D * es % 16 != 0 || k.size(d - 2) <= 0 || (d == 5 && k.size(0) <= 0)) return false;
    for (const at::Tensor* t : {&k, &v}) {
        if ((uintptr_t)t->data_ptr() & 15 || t->stride(d - 1) != 1) return false;
        for (int64_t i = 0; i + 1 < d; ++i)
            if (t->stride(i) < 0 || t->stride(i) * es % 16 != 0) return false;
        if (written && !t->is_contiguous()) return false;
    }
    if (written && share(k, v)) return false;
    if (!none(table)) {
        if (!integer(table, k, 2) || k.size(d - 3) % 16 != 0 || k.size(d - 3) == 0) return false;
        const int64_t n = THPVariable_Unpack(table).size(0);
        if (batch >= 0 && n != batch) return false;
        batch = n;
    } else if (batch < 0 || k.size(d - 4) != batch) {
        return false;
    }
    return none(lens) || (integer(lens, k, 1) && THPVariable_Unpack(lens).size(0) == batch);
}
// new rows or queries (.., batch, tokens, heads, d) beside a cache
bool rows_ok(PyObject* o, const at::Tensor& k, int64_t dim) {
    if (!THPVariable_Check(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.dim() == dim && t.device() == k.device() && t.scalar_type() == k.scalar_type() && t.size(dim - 1) == k.size(k.dim() - 1) &&
           !dual(t) && !wants_grad(t);
}
bool check_count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return false;
}

// shares(a, b): whether two tensors share an element
PyObject* shares(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 2)) return nullptr;
    if (!THPVariable_Check(x[0]) || !THPVariable_Check(x[1])) {
        PyErr_SetString(PyExc_TypeError, "expected a tensor");
        return nullptr;
    }
    return PyBool_FromLong(share(THPVariable_Unpack(x[0]), THPVariable_Unpack(x[1])));
    END_HANDLE_TH_ERRORS
}
// pool_ok(k, v, table or None, lengths or None, batch or None, written)
PyObject* pool_ok(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 6)) return nullptr;
    const int64_t batch = none(x[4]) ? -1 : PyLong_AsLongLong(x[4]);
    if (PyErr_Occurred()) return nullptr;
    return PyBool_FromLong(cache_ok(x[0], x[1], x[2], x[3], batch, PyObject_IsTrue(x[5]) == 1));
    END_HANDLE_TH_ERRORS
}
// paged_ok(q, k, v, lengths, table (or None each))
PyObject* paged_ok(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 5)) return nullptr;
    if (!THPVariable_Check(x[0]) || THPVariable_Unpack(x[0]).dim() != 4) Py_RETURN_FALSE;
    const at::Tensor& q = THPVariable_Unpack(x[0]);
    if (!cache_ok(x[1], x[2], x[4], x[3], q.size(0), false)) Py_RETURN_FALSE;
    const at::Tensor& k = THPVariable_Unpack(x[1]);
    return PyBool_FromLong(rows_ok(x[0], k, 4) && q.size(2) > 0 && q.size(2) % k.size(2) == 0);
    END_HANDLE_TH_ERRORS
}
// write_ok(k_new, v_new, k, v, lengths, table (or None each))
PyObject* write_ok(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 6)) return nullptr;
    if (!THPVariable_Check(x[0]) || !THPVariable_Check(x[2])) Py_RETURN_FALSE;
    const at::Tensor &kn = THPVariable_Unpack(x[0]), &k = THPVariable_Unpack(x[2]);
    const int64_t d = kn.dim();
    if (d != k.dim() || d < 4 || !cache_ok(x[2], x[3], x[5], x[4], kn.size(d - 4), true)) Py_RETURN_FALSE;
    if (!rows_ok(x[0], k, d) || !rows_ok(x[1], k, d) || kn.sizes() != THPVariable_Unpack(x[1]).sizes() ||
        kn.size(d - 2) != k.size(d - 2) || (d == 5 && kn.size(0) != k.size(0)))
        Py_RETURN_FALSE;
    for (int i = 0; i < 2; ++i)
        for (int j = 2; j < 4; ++j)
            if (share(THPVariable_Unpack(x[i]), THPVariable_Unpack(x[j]))) Py_RETURN_FALSE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}
// accept_ok(k, v, path, lengths, table (or None each))
PyObject* accept_ok(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 5)) return nullptr;
    if (!THPVariable_Check(x[2]) || THPVariable_Unpack(x[2]).dim() != 2) Py_RETURN_FALSE;
    return PyBool_FromLong(cache_ok(x[0], x[1], x[4], x[3], THPVariable_Unpack(x[2]).size(0), true) &&
                           integer(x[2], THPVariable_Unpack(x[0]), 2));
    END_HANDLE_TH_ERRORS
}
// fork_ok(k, v, table, sources, lengths or None, new tokens): an int is for the caller to look at
PyObject* fork_ok(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check_count(n, 6)) return nullptr;
    if (none(x[2]) || !cache_ok(x[0], x[1], x[2], x[4], -1, true)) Py_RETURN_FALSE;
    const at::Tensor& k = THPVariable_Unpack(x[0]);
    if (!integer(x[3], k, 1)) Py_RETURN_FALSE;
    return PyBool_FromLong(!THPVariable_Check(x[5]) ||
                           (integer(x[5], k, 1) && THPVariable_Unpack(x[5]).size(0) == THPVariable_Unpack(x[3]).size(0)));
    END_HANDLE_TH_ERRORS
}

// paged_fwd(q, k, v, lengths, table, parents, slopes (or None each), scale, softcap,
//     want_lse, stream) -> (status, o, lse or None)
PyObject* paged_fwd(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check(n, 11, x, 3)) return nullptr;
    c10::DeviceGuard guard(THPVariable_Unpack(x[0]).device());
    const at::Tensor q = prepare(THPVariable_Unpack(x[0]));
    const at::Tensor &k = THPVariable_Unpack(x[1]), &v = THPVariable_Unpack(x[2]);
    fa_paged_args a = {};
    Pool pool;
    pool.put(a.pool, k, v, x[4], x[3], q.size(0));
    const at::Tensor parents = ints(x[5]);
    const at::Tensor slopes = none(x[6]) ? at::Tensor() : THPVariable_Unpack(x[6]).contiguous();
    a.scale = (float)PyFloat_AsDouble(x[7]);
    a.softcap = (float)PyFloat_AsDouble(x[8]);
    const bool want = PyObject_IsTrue(x[9]) == 1;
    void* const stream = PyLong_AsVoidPtr(x[10]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor o = at::empty(q.sizes(), q.options());
    const at::Tensor lse =
        want ? at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat)) : at::Tensor();
    a.q = q.data_ptr();
    a.o = o.data_ptr();
    a.lse = ptr<float>(lse);
    put_strides(a.q_stride, q);
    put_strides(a.o_stride, o);
    a.seqlen_q = i32(q.size(1));
    a.num_heads = i32(q.size(2));
    a.slopes = ptr<const float>(slopes);
    a.slopes_batch_stride = slopes.defined() && slopes.dim() == 2 ? slopes.size(1) : 0;
    a.parents = ptr<const int32_t>(parents);
    a.parents_stride = row_stride(parents);
    const size_t bytes = p_paged_size(&a);
    const at::Tensor ws = workspace(bytes, q);
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_paged(&a, ptr<void>(ws), bytes, stream);
    }
    PyObject* const l = lse.defined() ? THPVariable_Wrap(lse) : Py_NewRef(Py_None);
    return Py_BuildValue("(iNN)", (int)st, THPVariable_Wrap(o), l);
    END_HANDLE_TH_ERRORS
}

void changed(const at::Tensor& k, const at::Tensor& v) {
    fa_host::written(k);
    fa_host::written(v);
}

// cache_write(k_new, v_new, k, v, lengths, table (or None each), stream) -> status
PyObject* cache_write(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check(n, 7, x, 4)) return nullptr;
    const at::Tensor &k = THPVariable_Unpack(x[2]), &v = THPVariable_Unpack(x[3]);
    c10::DeviceGuard guard(k.device());
    const at::Tensor in[2] = {prepare(THPVariable_Unpack(x[0])), prepare(THPVariable_Unpack(x[1]))};
    const int64_t d = in[0].dim();
    fa_cache_write_args a = {};
    Pool pool;
    pool.put(a.pool, k, v, x[5], x[4], in[0].size(d - 4));
    void* const stream = PyLong_AsVoidPtr(x[6]);
    if (PyErr_Occurred()) return nullptr;
    a.k = in[0].data_ptr();
    a.v = in[1].data_ptr();
    for (int64_t i = 0; i < 5; ++i) {
        a.k_stride[i] = i + d - 5 >= 0 ? in[0].stride(i + d - 5) : 0;
        a.v_stride[i] = i + d - 5 >= 0 ? in[1].stride(i + d - 5) : 0;
    }
    a.tokens = i32(in[0].size(d - 3));
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_write(&a, stream);
    }
    if (!st) changed(k, v);
    return PyLong_FromLong(st);
    END_HANDLE_TH_ERRORS
}

// cache_accept(k, v, path, lengths, table (or None each), tokens, stream) -> (status, lengths)
PyObject* cache_accept(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check(n, 7, x, 3)) return nullptr;
    const at::Tensor &k = THPVariable_Unpack(x[0]), &v = THPVariable_Unpack(x[1]);
    c10::DeviceGuard guard(k.device());
    const at::Tensor path = ints(x[2]);
    fa_cache_accept_args a = {};
    Pool pool;
    pool.put(a.pool, k, v, x[4], x[3], path.size(0));
    a.tokens = (int32_t)PyLong_AsLong(x[5]);
    void* const stream = PyLong_AsVoidPtr(x[6]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor lens = at::empty({path.size(0)}, k.options().dtype(at::kInt));
    a.path = ptr<const int32_t>(path);
    a.path_stride = row_stride(path);
    a.path_cols = i32(path.size(1));
    a.new_lengths = ptr<int32_t>(lens);
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_accept(&a, stream);
    }
    if (!st) changed(k, v);
    return Py_BuildValue("(iN)", (int)st, THPVariable_Wrap(lens));
    END_HANDLE_TH_ERRORS
}

// cache_fork(k, v, table, sources, lengths or None, new tokens (an int or a tensor),
//     stream) -> (status, table, lengths)
PyObject* cache_fork(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check(n, 7, x, 4)) return nullptr;
    const at::Tensor &k = THPVariable_Unpack(x[0]), &v = THPVariable_Unpack(x[1]);
    c10::DeviceGuard guard(k.device());
    fa_cache_fork_args a = {};
    Pool pool;
    pool.put(a.pool, k, v, x[2], x[4], THPVariable_Unpack(x[2]).size(0));
    const at::Tensor sources = ints(x[3]).contiguous();
    at::Tensor more;
    if (THPVariable_Check(x[5]))
        more = ints(x[5]).contiguous();
    else
        a.more_all = (int32_t)PyLong_AsLong(x[5]);
    void* const stream = PyLong_AsVoidPtr(x[6]);
    if (PyErr_Occurred()) return nullptr;
    const auto i = k.options().dtype(at::kInt);
    const at::Tensor table = at::empty({sources.size(0), pool.table.size(1)}, i), lens = at::empty({sources.size(0)}, i);
    a.sources = ptr<const int32_t>(sources);
    a.more = ptr<const int32_t>(more);
    a.new_batch = i32(sources.size(0));
    a.new_table = ptr<int32_t>(table);
    a.new_lengths = ptr<int32_t>(lens);
    const size_t bytes = p_fork_size(&a);
    const at::Tensor ws = workspace(bytes, k);
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_fork(&a, ptr<void>(ws), bytes, stream);
    }
    if (!st) changed(k, v);
    return Py_BuildValue("(iNN)", (int)st, THPVariable_Wrap(table), THPVariable_Wrap(lens));
    END_HANDLE_TH_ERRORS
}

// cache_compact(k, v, table, lengths or None, stream) -> (status, table, used)
PyObject* cache_compact(PyObject*, PyObject* const* x, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!check(n, 5, x, 3)) return nullptr;
    const at::Tensor &k = THPVariable_Unpack(x[0]), &v = THPVariable_Unpack(x[1]);
    c10::DeviceGuard guard(k.device());
    fa_cache_compact_args a = {};
    Pool pool;
    pool.put(a.pool, k, v, x[2], x[3], THPVariable_Unpack(x[2]).size(0));
    void* const stream = PyLong_AsVoidPtr(x[4]);
    if (PyErr_Occurred()) return nullptr;
    const auto i = k.options().dtype(at::kInt);
    const at::Tensor table = at::empty(pool.table.sizes(), i), used = at::empty({}, i);
    a.new_table = ptr<int32_t>(table);
    a.used = ptr<int32_t>(used);
    const size_t bytes = p_compact_size(&a);
    const at::Tensor ws = workspace(bytes, k);
    int32_t st;
    {
        pybind11::gil_scoped_release no_gil;
        st = p_compact(&a, ptr<void>(ws), bytes, stream);
    }
    if (!st) changed(k, v);
    return Py_BuildValue("(iNN)", (int)st, THPVariable_Wrap(table), THPVariable_Wrap(used));
    END_HANDLE_TH_ERRORS
}

// bind_paged(fa_paged_version, the sizes of the five argument structs in the header's
//     order, then the addresses of the functions above in their order); refused for
//     another version or other struct sizes, as bind is
PyObject* bind_paged(PyObject*, PyObject* const* x, Py_ssize_t n) {
    constexpr int kSizes = 5, kFunctions = 8;
    if (n != 1 + kSizes + kFunctions) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", 1 + kSizes + kFunctions, n);
        return nullptr;
    }
    void* p[1 + kFunctions];
    for (int i = 0; i <= kFunctions; ++i) {
        p[i] = PyLong_AsVoidPtr(x[i == 0 ? 0 : i + kSizes]);
        if (PyErr_Occurred()) return nullptr;
        if (!p[i]) {
            PyErr_SetString(PyExc_ValueError, "bind_paged: null address");
            return nullptr;
        }
    }
    const size_t mine[kSizes] = {sizeof(fa_paged_args), sizeof(fa_cache_write_args), sizeof(fa_cache_accept_args),
                                 sizeof(fa_cache_fork_args), sizeof(fa_cache_compact_args)};
    const int32_t version = ((decltype(&fa_paged_version))p[0])();
    bool same = version == FA_PAGED_VERSION;
    for (int i = 0; i < kSizes; ++i) same = same && PyLong_AsSize_t(x[1 + i]) == mine[i];
    if (PyErr_Occurred()) return nullptr;
    if (!same) {
        PyErr_Format(PyExc_RuntimeError,
                     "fa_host was built for paged cache version %d; the library has version %d, or the binding other argument "
                     "structs",
                     FA_PAGED_VERSION, (int)version);
        return nullptr;
    }
    p_paged_size = (decltype(p_paged_size))p[1];
    p_paged = (decltype(p_paged))p[2];
    p_write = (decltype(p_write))p[3];
    p_accept = (decltype(p_accept))p[4];
    p_fork_size = (decltype(p_fork_size))p[5];
    p_fork = (decltype(p_fork))p[6];
    p_compact_size = (decltype(p_compact_size))p[7];
    p_compact = (decltype(p_compact))p[8];
    Py_RETURN_NONE;
}

}  // namespace

PyMethodDef fa_host::paged_methods[] = {
    {"bind_paged", (PyCFunction)(void*)bind_paged, METH_FASTCALL, nullptr},
    {"shares", (PyCFunction)(void*)shares, METH_FASTCALL, nullptr},
    {"pool_ok", (PyCFunction)(void*)pool_ok, METH_FASTCALL, nullptr},
    {"paged_ok", (PyCFunction)(void*)paged_ok, METH_FASTCALL, nullptr},
    {"write_ok", (PyCFunction)(void*)write_ok, METH_FASTCALL, nullptr},
    {"accept_ok", (PyCFunction)(void*)accept_ok, METH_FASTCALL, nullptr},
    {"fork_ok", (PyCFunction)(void*)fork_ok, METH_FASTCALL, nullptr},
    {"paged_fwd", (PyCFunction)(void*)paged_fwd, METH_FASTCALL, nullptr},
    {"cache_write", (PyCFunction)(void*)cache_write, METH_FASTCALL, nullptr},
    {"cache_accept", (PyCFunction)(void*)cache_accept, METH_FASTCALL, nullptr},
    {"cache_fork", (PyCFunction)(void*)cache_fork, METH_FASTCALL, nullptr},
    {"cache_compact", (PyCFunction)(void*)cache_compact, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

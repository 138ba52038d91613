// The host side of a packed linear's call, as a Python extension: checks, output, stream and launch in one call from Python.
// Through ctypes and torch's Python functions the same takes 7 us, more than the kernel of a 2048 x 2048 layer; here 4, of which
// the launch is 3.  Anything out of the ordinary (another type, a subclass, a transform, a layout, a device) is left to the
// Python path: the call returns None.
#include <Python.h>
#include <structmember.h>

#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

namespace {

using gemv_fn = int (*)(const void *, const void *, int64_t, const void *, void *, int, void *, size_t, void *);
using rows_fn = int (*)(const void *, const void *, int64_t, const void *, void *, int, void *);
gemv_fn g_gemv = nullptr;
rows_fn g_rows = nullptr;
PyObject *g_check = nullptr;                             // raises the library's error for a status

// The interpreter's lock, given up while torch allocates (which may wait for the device) and while a launch is made (which waits
// where the queue is full): another thread may be the one that would end the wait.
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked &) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

struct P6Call {
    PyObject_HEAD
    vectorcallfunc call;
    const void *tensor;                                  // the ixb_p6 structure (of the object that holds this one)
    int64_t out_f, in_f;
    int index;
    void *scratch;                                       // of ixb_p6_gemv
    size_t scratch_bytes;
    PyObject *keep;                                      // the scratch's tensor
};

// (x, bias or None, many): y = x W^T for 1..8 rows, and with `many` 9..64 rows of a layer whose in_f is a multiple of 64
PyObject *p6_call(PyObject *self_, PyObject *const *args, size_t nargsf, PyObject *kw)
{
    const P6Call *self = (const P6Call *)self_;
    if (PyVectorcall_NARGS(nargsf) != 3 || kw) {
        PyErr_SetString(PyExc_TypeError, "expected (x, bias, many)");
        return nullptr;
    }
    try {
        if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
        const at::Tensor x = THPVariable_Unpack(args[0]);            // (held: other threads run below)
        if (x.scalar_type() != at::kBFloat16 || x.layout() != at::kStrided || !x.is_cuda() || x.get_device() != self->index ||
            at::isTensorSubclassLike(x) || x.is_neg() || x.dim() < 1 || x.size(-1) != self->in_f || !x.is_contiguous())
            Py_RETURN_NONE;
        const int64_t m = x.numel() / self->in_f;
        if (m < 1 || m > 64 || (m > 8 && (self->in_f % 64 || args[2] != Py_True))) Py_RETURN_NONE;
        const void *bias = nullptr;
        at::Tensor b;
        if (args[1] != Py_None) {
            if (!THPVariable_Check(args[1])) Py_RETURN_NONE;
            b = THPVariable_Unpack(args[1]);
            if (b.scalar_type() != at::kBFloat16 || b.numel() != self->out_f || !b.is_cuda() || b.get_device() != self->index || !b.is_contiguous())
                Py_RETURN_NONE;
            bias = b.data_ptr();
        }
        at::DimVector shape(x.sizes().begin(), x.sizes().end());
        shape.back() = self->out_f;
        at::Tensor y;
        int rc = 0;
        bool plain;
        {
            const Unlocked unlocked;
            c10::cuda::OptionalCUDAGuard guard;
            if (c10::cuda::current_device() != self->index) guard.set_index((c10::DeviceIndex)self->index);
            y = at::empty(shape, at::TensorOptions().dtype(at::kBFloat16).device(at::Device(at::kCUDA, (c10::DeviceIndex)self->index)));
            plain = !at::isTensorSubclassLike(y);
            if (plain) {
                void *stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)self->index).stream();
                rc = m <= 8 ? g_gemv(self->tensor, x.data_ptr(), m, bias, y.data_ptr(), 0, self->scratch, self->scratch_bytes, stream)
                            : g_rows(self->tensor, x.data_ptr(), m, bias, y.data_ptr(), 0, stream);
            }
        }
        if (!plain) Py_RETURN_NONE;
        if (rc) {
            PyObject *r = PyObject_CallFunction(g_check, "i", rc);
            Py_XDECREF(r);
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "packed linear failed");
            return nullptr;
        }
        return THPVariable_Wrap(std::move(y));
    } catch (...) {                                      // as torch's functions raise it: out of memory, an error of Python code
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

void p6_dealloc(PyObject *self_)
{
    Py_XDECREF(((P6Call *)self_)->keep);
    Py_TYPE(self_)->tp_free(self_);
}

PyMemberDef p6_members[] = {{"__vectorcalloffset__", T_PYSSIZET, offsetof(P6Call, call), READONLY, nullptr}, {nullptr, 0, 0, 0, nullptr}};
PyTypeObject P6CallType = {PyVarObject_HEAD_INIT(nullptr, 0)};

// p6(structure address, out_f, in_f, device index, scratch tensor)
PyObject *new_p6(PyObject *, PyObject *args)
{
    unsigned long long tensor;
    long long out_f, in_f;
    int index;
    PyObject *scratch;
    if (!PyArg_ParseTuple(args, "KLLiO", &tensor, &out_f, &in_f, &index, &scratch)) return nullptr;
    if (!g_gemv || !THPVariable_Check(scratch) || out_f <= 0 || in_f <= 0) {
        PyErr_SetString(PyExc_ValueError, "p6: not bound, or bad arguments");
        return nullptr;
    }
    P6Call *c = PyObject_New(P6Call, &P6CallType);
    if (!c) return nullptr;
    c->call = p6_call;
    c->tensor = (const void *)(uintptr_t)tensor;
    c->out_f = out_f;
    c->in_f = in_f;
    c->index = index;
    const at::Tensor &s = THPVariable_Unpack(scratch);
    c->scratch = s.data_ptr();
    c->scratch_bytes = (size_t)s.numel() * s.element_size();
    c->keep = scratch;
    Py_INCREF(scratch);
    return (PyObject *)c;
}

// bind(address of ixb_p6_gemv, of ixb_p6_rows, check)
PyObject *bind(PyObject *, PyObject *args)
{
    unsigned long long gemv, rows;
    PyObject *check;
    if (!PyArg_ParseTuple(args, "KKO", &gemv, &rows, &check)) return nullptr;
    g_gemv = (gemv_fn)(uintptr_t)gemv;
    g_rows = (rows_fn)(uintptr_t)rows;
    Py_XDECREF(g_check);
    g_check = check;
    Py_INCREF(check);
    Py_RETURN_NONE;
}

// empty(device index, (n, type), (n, type), ...): uninitialised one-dimensional tensors (n < 0: of no dimension);
// type 'B' uint8, 'b' int8, 'i' int32, 'h' bfloat16
PyObject *empty(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    if (nargs < 1) {
        PyErr_SetString(PyExc_TypeError, "empty(index, (n, type), ...)");
        return nullptr;
    }
    const long index = PyLong_AsLong(args[0]);
    if (index < 0) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "expected a CUDA device");
        return nullptr;
    }
    struct Spec {
        long long n;
        int type;
    };
    try {
        c10::SmallVector<Spec, 8> specs((size_t)(nargs - 1));
        c10::SmallVector<at::Tensor, 8> tensors;
        for (Py_ssize_t i = 1; i < nargs; ++i)
            if (!PyArg_ParseTuple(args[i], "LC", &specs[i - 1].n, &specs[i - 1].type)) return nullptr;
        {
            const Unlocked unlocked;
            for (const Spec &s : specs) {
                const auto dt = s.type == 'B' ? at::kByte : s.type == 'b' ? at::kChar : s.type == 'i' ? at::kInt : at::kBFloat16;
                const int64_t size[1] = {s.n};
                tensors.push_back(at::empty(at::IntArrayRef(size, s.n < 0 ? 0 : 1), at::TensorOptions().dtype(dt).device(at::Device(at::kCUDA, (c10::DeviceIndex)index))));
            }
        }
        PyObject *out = PyTuple_New(nargs - 1);
        for (Py_ssize_t i = 0; out && i < nargs - 1; ++i) {
            PyObject *o = THPVariable_Wrap(std::move(tensors[i]));
            if (!o) {
                Py_DECREF(out);
                return nullptr;
            }
            PyTuple_SET_ITEM(out, i, o);
        }
        return out;
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

// ---------------------------------------------------------------- the calls of a serving step
// The same for the paged cache's calls and the rules on logits (paged.py, logits.py): what they check there, and the launch.  None where
// anything is out of the ordinary, a refusal included: the Python path then says what.
using page_step_fn = int (*)(const int32_t *, const int32_t *, int32_t *, const int32_t *, const int32_t *, int64_t, int64_t, int64_t, int64_t, int64_t,
                             int32_t *, int32_t *, int32_t *, int32_t *, int32_t *, int32_t *, int32_t *, void *);
using rope_paged_fn = int (*)(const void *, const void *, const void *, const int32_t *, const int32_t *, void *, void *, const void *, const void *,
                              const float *, const float *, void *, int64_t, int64_t, int64_t, int64_t, int64_t, float, int64_t, int64_t, int64_t, int64_t,
                              int64_t, int64_t, int64_t, int64_t, void *);
using attn_paged_fn = int (*)(const void *, const void *, const void *, const int32_t *, const int32_t *, const int32_t *, void *, int64_t, int64_t, int64_t,
                              int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, float, void *, size_t, void *);
using logits_fn = int (*)(const void *, int, int64_t, const int32_t *, int64_t, int64_t, const int32_t *, const int32_t *, const float *, const float *,
                          const float *, const int32_t *, const float *, int64_t, const void *, int64_t, int64_t, const int32_t *, float *, int64_t, int64_t *,
                          int64_t, int64_t, void *);
page_step_fn g_page_step = nullptr;
rope_paged_fn g_rope_paged = nullptr;
attn_paged_fn g_attn_paged = nullptr;
logits_fn g_logits = nullptr;

// A plain strided CUDA tensor of this type on device `index` (-1: any, and index becomes its device)
bool take(PyObject *o, at::Tensor &t, at::ScalarType type, int &index)
{
    if (!THPVariable_Check(o)) return false;
    t = THPVariable_Unpack(o);
    if (t.scalar_type() != type || t.layout() != at::kStrided || !t.is_cuda() || at::isTensorSubclassLike(t) || t.is_neg()) return false;
    if (index < 0) index = t.get_device();
    return t.get_device() == index;
}
bool take_ints(PyObject *o, at::Tensor &t, int64_t n, int &index)      // contiguous int32, n of them (-1: any number)
{
    return take(o, t, at::kInt, index) && t.is_contiguous() && (n < 0 || t.numel() == n);
}
// a matrix with contiguous columns (a vector: one row)
struct Rows {
    int64_t rows, cols, pitch;
};
bool rows_of(const at::Tensor &t, Rows &r)
{
    if (t.dim() == 1) {
        r = {1, t.size(0), t.size(0)};
        return t.stride(0) == 1;
    }
    if (t.dim() != 2 || t.stride(1) != 1) return false;
    r = {t.size(0), t.size(1), t.size(0) > 1 ? t.stride(0) : t.size(1)};
    return true;
}
// what the entry points refuse in Python (paged.PAGES, paged.MAX_REQUESTS)
bool page_holds(int64_t page) { return page == 16 || page == 32 || page == 64 || page == 128 || page == 256; }
constexpr int64_t kMaxRequests = 4096;
// [pages, page, heads, dimensions] whose pages are contiguous and may lie apart
bool pool_of(const at::Tensor &t, int64_t heads, int64_t d, int64_t &pages, int64_t &page, int64_t &pitch)
{
    if (t.dim() != 4 || t.size(0) < 1 || t.size(2) != heads || t.size(3) != d || t.stride(3) != 1 || t.stride(2) != d || t.stride(1) != heads * d) return false;
    pages = t.size(0);
    page = t.size(1);
    pitch = pages > 1 ? t.stride(0) : page * heads * d;
    return page_holds(page) && pitch >= page * heads * d && pitch % 8 == 0;
}
bool number(PyObject *o, int64_t &v)
{
    v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
    if (v == -1 && PyErr_Occurred()) PyErr_Clear();
    return v >= 0;
}
const int32_t *ints(const at::Tensor &t) { return t.defined() && t.numel() ? (const int32_t *)t.data_ptr() : nullptr; }
const float *floats(const at::Tensor &t) { return t.defined() && t.numel() ? (const float *)t.data_ptr() : nullptr; }

// launch(stream) with the device current and without the interpreter's lock; false: an exception is set
template <class F>
bool launched(int index, F launch)
{
    int rc;
    {
        const Unlocked unlocked;
        c10::cuda::OptionalCUDAGuard guard;
        if (c10::cuda::current_device() != index) guard.set_index((c10::DeviceIndex)index);
        rc = launch(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream());
    }
    if (!rc) return true;
    PyObject *r = PyObject_CallFunction(g_check, "i", rc);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "the launch failed");
    return false;
}
#define IXB_HOST_TRY try {
#define IXB_HOST_END                                                                 \
    }                                                                                \
    catch (...)                                                                      \
    {                                                                                \
        torch::translate_exception_to_python(std::current_exception());              \
        return nullptr;                                                              \
    }

// (q_len, length, table, free, n_free, page, rows, cu_rows, length, n_free, slot, pos, owner, status)
PyObject *page_step(PyObject *, PyObject *const *a, Py_ssize_t nargs)
{
    IXB_HOST_TRY
    int dev = -1;
    int64_t page, rows;
    at::Tensor q, len, table, free_, n_free, cu, nl, nf, slot, pos, owner, status;
    if (nargs != 14 || !g_page_step || !take_ints(a[0], q, -1, dev)) Py_RETURN_NONE;
    const int64_t r = q.numel();
    if (r < 1 || r > kMaxRequests || !take_ints(a[1], len, r, dev) || !take_ints(a[2], table, -1, dev) || !take_ints(a[3], free_, -1, dev) || !take_ints(a[4], n_free, 1, dev) ||
        !number(a[5], page) || !page_holds(page) || !number(a[6], rows) || table.dim() != 2 || table.size(0) != r || !take_ints(a[7], cu, r + 1, dev) || !take_ints(a[8], nl, r, dev) ||
        !take_ints(a[9], nf, 1, dev) || !take_ints(a[10], slot, rows, dev) || !take_ints(a[11], pos, rows, dev) || !take_ints(a[12], owner, rows, dev) ||
        !take_ints(a[13], status, 2, dev) || rows < 1 || free_.numel() < 1 || table.numel() < 1)
        Py_RETURN_NONE;
    auto i = [](const at::Tensor &t) { return (int32_t *)t.data_ptr(); };
    if (!launched(dev, [&](void *st) {
            return g_page_step(i(q), i(len), i(table), i(free_), i(n_free), r, table.size(1), free_.numel(), page, rows, i(cu), i(nl), i(nf), i(slot), i(pos),
                               i(owner), i(status), st);
        }))
        return nullptr;
    Py_RETURN_TRUE;
    IXB_HOST_END
}

// (q, k, v, pos, slot, k_pages, v_pages, cos, sin, hq, hkv, head_dim, rot_dim, q_norm, k_norm, eps, out)
PyObject *rope_paged(PyObject *, PyObject *const *a, Py_ssize_t nargs)
{
    IXB_HOST_TRY
    int dev = -1;
    int64_t hq, hkv, d, rot, pages, page, kp, vp, n2, p2;
    at::Tensor q, k, v, pos, slot, kpool, vpool, cs, sn, qn, kn, out;
    Rows rq, rk, rv, ro;
    const auto bf = at::kBFloat16;
    if (nargs != 17 || !g_rope_paged || !number(a[9], hq) || !number(a[10], hkv) || !number(a[11], d) || !number(a[12], rot) || !PyFloat_Check(a[15]) ||
        !take(a[0], q, bf, dev) || !take(a[1], k, bf, dev) || !take(a[2], v, bf, dev) || !rows_of(q, rq) || !rows_of(k, rk) || !rows_of(v, rv))
        Py_RETURN_NONE;
    if (!take_ints(a[3], pos, -1, dev) || !take_ints(a[4], slot, -1, dev) || !take(a[5], kpool, bf, dev) || !take(a[6], vpool, bf, dev) ||
        !take(a[7], cs, at::kFloat, dev) || !take(a[8], sn, at::kFloat, dev) || !take(a[16], out, bf, dev) || !rows_of(out, ro) ||
        !pool_of(kpool, hkv, d, pages, page, kp) || !pool_of(vpool, hkv, d, n2, p2, vp))
        Py_RETURN_NONE;
    if (a[13] != Py_None && (!take(a[13], qn, bf, dev) || !qn.is_contiguous() || qn.numel() != d)) Py_RETURN_NONE;
    if (a[14] != Py_None && (!take(a[14], kn, bf, dev) || !kn.is_contiguous() || kn.numel() != d)) Py_RETURN_NONE;
    if (rq.rows < 1 || rk.rows != rq.rows || rv.rows != rq.rows || ro.rows != rq.rows || rk.cols != hkv * d || rv.cols != rk.cols || rv.pitch != rk.pitch ||
        rq.cols < hq * d || (a[16] != a[0] && ro.cols != hq * d) || pos.numel() < rq.rows || slot.numel() < rq.rows || n2 != pages || p2 != page || !cs.is_contiguous() ||
        !sn.is_contiguous() || cs.dim() != 2 || sn.dim() != 2 || cs.size(1) != rot / 2 || cs.size(0) < 1 || cs.sizes() != sn.sizes())
        Py_RETURN_NONE;
    const float eps = (float)PyFloat_AS_DOUBLE(a[15]);
    if (!launched(dev, [&](void *st) {
            return g_rope_paged(q.data_ptr(), k.data_ptr(), v.data_ptr(), ints(pos), ints(slot), kpool.data_ptr(), vpool.data_ptr(),
                                qn.defined() ? qn.data_ptr() : nullptr, kn.defined() ? kn.data_ptr() : nullptr, floats(cs), floats(sn), out.data_ptr(), rq.rows, hq,
                                hkv, d, rot, eps, rq.pitch, rk.pitch, ro.pitch, cs.size(0), pages, page, kp, vp, st);
        }))
        return nullptr;
    Py_RETURN_TRUE;
    IXB_HOST_END
}

// (hq, hkv, head_dim, scratch, q, k_pages, v_pages, table, length, cu_rows, max_q or None, out or None, scale or None): out
PyObject *attn_paged(PyObject *, PyObject *const *a, Py_ssize_t nargs)
{
    IXB_HOST_TRY
    int dev = -1;
    int64_t hq, hkv, d, pages, page, kp, vp, n2, p2, max_q;
    at::Tensor scratch, q, kpool, vpool, table, len, cu, out;
    Rows rq;
    const auto bf = at::kBFloat16;
    if (nargs != 13 || !g_attn_paged || !number(a[0], hq) || !number(a[1], hkv) || !number(a[2], d) || !take(a[4], q, bf, dev) || !take(a[3], scratch, at::kByte, dev) ||
        !take(a[5], kpool, bf, dev) || !take(a[6], vpool, bf, dev) || !take_ints(a[7], table, -1, dev) || !take_ints(a[8], len, -1, dev) || !rows_of(q, rq))
        Py_RETURN_NONE;
    const int64_t r = len.numel();
    if (r < 1 || r > kMaxRequests || !take_ints(a[9], cu, r + 1, dev) || table.dim() != 2 || table.size(0) != r || table.size(1) < 1 || rq.rows < 1 || rq.cols < hq * d ||
        !pool_of(kpool, hkv, d, pages, page, kp) || !pool_of(vpool, hkv, d, n2, p2, vp) || n2 != pages || p2 != page)
        Py_RETURN_NONE;
    max_q = rq.rows;
    if (a[10] != Py_None) {
        if (!number(a[10], max_q) || max_q < 1) Py_RETURN_NONE;
        if (max_q > rq.rows) max_q = rq.rows;
    }
    double scale = 1.0 / std::sqrt((double)d);
    if (a[12] != Py_None) {
        if (!PyFloat_Check(a[12])) Py_RETURN_NONE;
        scale = PyFloat_AS_DOUBLE(a[12]);
        if (!(scale > 0.0) || std::isinf(scale)) Py_RETURN_NONE;
    }
    if (a[11] != Py_None && (!take(a[11], out, bf, dev) || !out.is_contiguous() || out.numel() != rq.rows * hq * d)) Py_RETURN_NONE;
    const bool given = out.defined();
    bool plain = true;
    if (!launched(dev, [&](void *st) {
            if (!given) {
                out = at::empty({rq.rows, hq * d}, q.options());
                if (!(plain = !at::isTensorSubclassLike(out))) return 0;
            }
            return g_attn_paged(q.data_ptr(), kpool.data_ptr(), vpool.data_ptr(), ints(table), ints(len), ints(cu), out.data_ptr(), r, table.size(1), rq.rows, max_q,
                                hq, hkv, d, pages, page, rq.pitch, kp, vp, (float)scale, scratch.data_ptr(), (size_t)scratch.numel(), st);
        }))
        return nullptr;
    if (!plain) Py_RETURN_NONE;
    if (given) {
        Py_INCREF(a[11]);
        return a[11];
    }
    return THPVariable_Wrap(std::move(out));
    IXB_HOST_END
}

// a matrix [rows, cols] (cols -1: any) of this type with contiguous rows that do not overlap; false with None is up to the caller
bool take_rows(PyObject *o, at::Tensor &t, at::ScalarType type, int64_t rows, int64_t cols, int &dev, int64_t &pitch)
{
    if (!take(o, t, type, dev) || t.dim() != 2 || t.size(0) != rows || (cols >= 0 && t.size(1) != cols) || (t.size(1) > 1 && t.stride(1) != 1)) return false;
    pitch = rows > 1 ? t.stride(0) : t.size(1);
    return pitch >= t.size(1);
}

// (logits, history, n_tokens, n_prompt, repetition, presence, frequency, bias_ids, bias_values, mask, mask_row, out, token): all but logits and
// out may be None
PyObject *logits(PyObject *, PyObject *const *a, Py_ssize_t nargs)
{
    IXB_HOST_TRY
    int dev = -1;
    if (nargs != 13 || !g_logits || !THPVariable_Check(a[0])) Py_RETURN_NONE;
    const auto type = THPVariable_Unpack(a[0]).scalar_type();
    if ((type != at::kBFloat16 && type != at::kFloat) || THPVariable_Unpack(a[0]).dim() != 2) Py_RETURN_NONE;
    const int64_t b = THPVariable_Unpack(a[0]).size(0), v = THPVariable_Unpack(a[0]).size(1);
    at::Tensor x, hist, row_i[2], row_f[3], ids, vals, mask, mask_row, out, token;
    int64_t pitch, hist_pitch = 0, out_pitch, mask_pitch = 0, bp, n_bias = 0, n_masks = 0;
    if (b < 1 || v < 1 || !take_rows(a[0], x, type, b, v, dev, pitch) || !take_rows(a[11], out, at::kFloat, b, v, dev, out_pitch)) Py_RETURN_NONE;
    auto per_row = [&](PyObject *o, at::Tensor &t, at::ScalarType ty) { return o == Py_None || (take(o, t, ty, dev) && t.dim() == 1 && t.size(0) == b && t.is_contiguous()); };
    if (a[1] == Py_None) {
        for (int i = 2; i <= 6; ++i)
            if (a[i] != Py_None) Py_RETURN_NONE;
    } else {
        if (!take_rows(a[1], hist, at::kInt, b, -1, dev, hist_pitch) || a[2] == Py_None || !per_row(a[2], row_i[0], at::kInt) || !per_row(a[3], row_i[1], at::kInt))
            Py_RETURN_NONE;
        for (int i = 0; i < 3; ++i)
            if (!per_row(a[4 + i], row_f[i], at::kFloat)) Py_RETURN_NONE;
    }
    if ((a[7] == Py_None) != (a[8] == Py_None)) Py_RETURN_NONE;
    if (a[7] != Py_None) {
        if (!take_rows(a[7], ids, at::kInt, b, -1, dev, bp) || !ids.is_contiguous()) Py_RETURN_NONE;
        n_bias = ids.size(1);
        if (!take_rows(a[8], vals, at::kFloat, b, n_bias, dev, bp) || !vals.is_contiguous()) Py_RETURN_NONE;
    }
    if (a[9] != Py_None) {
        if (!THPVariable_Check(a[9]) || THPVariable_Unpack(a[9]).dim() != 2) Py_RETURN_NONE;
        n_masks = THPVariable_Unpack(a[9]).size(0);
        if (n_masks < 1 || (a[10] == Py_None && n_masks != b) || !take_rows(a[9], mask, at::kInt, n_masks, (v + 31) / 32, dev, mask_pitch)) Py_RETURN_NONE;
    } else if (a[10] != Py_None) {
        Py_RETURN_NONE;
    }
    if (!per_row(a[10], mask_row, at::kInt) || !per_row(a[12], token, at::kLong)) Py_RETURN_NONE;
    if (!launched(dev, [&](void *st) {
            return g_logits(x.data_ptr(), type == at::kFloat, pitch, ints(hist), hist.defined() ? hist.size(1) : 0, hist_pitch, ints(row_i[0]), ints(row_i[1]),
                            floats(row_f[0]), floats(row_f[1]), floats(row_f[2]), ints(ids), floats(vals), n_bias, ints(mask), n_masks, mask_pitch, ints(mask_row),
                            (float *)out.data_ptr(), out_pitch, token.defined() ? (int64_t *)token.data_ptr() : nullptr, b, v, st);
        }))
        return nullptr;
    Py_RETURN_TRUE;
    IXB_HOST_END
}

// bind_serve(addresses of ixb_page_step, ixb_rope_paged, ixb_attn_paged, ixb_logits)
PyObject *bind_serve(PyObject *, PyObject *args)
{
    unsigned long long p[4];
    if (!PyArg_ParseTuple(args, "KKKK", &p[0], &p[1], &p[2], &p[3])) return nullptr;
    g_page_step = (page_step_fn)(uintptr_t)p[0];
    g_rope_paged = (rope_paged_fn)(uintptr_t)p[1];
    g_attn_paged = (attn_paged_fn)(uintptr_t)p[2];
    g_logits = (logits_fn)(uintptr_t)p[3];
    Py_RETURN_NONE;
}

#define IXB_FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"page_step", IXB_FAST(page_step)},
                         {"rope_paged", IXB_FAST(rope_paged)},
                         {"attn_paged", IXB_FAST(attn_paged)},
                         {"logits", IXB_FAST(logits)},
                         {"bind_serve", bind_serve, METH_VARARGS, nullptr},
                         {"p6", new_p6, METH_VARARGS, nullptr},
                         {"bind", bind, METH_VARARGS, nullptr},
                         {"empty", (PyCFunction)(void (*)(void))empty, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ixbhost", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ixbhost()
{
    P6CallType.tp_name = "ixrun_b200._ixbhost.P6Call";
    P6CallType.tp_basicsize = sizeof(P6Call);
    P6CallType.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
    P6CallType.tp_vectorcall_offset = offsetof(P6Call, call);
    P6CallType.tp_call = PyVectorcall_Call;
    P6CallType.tp_dealloc = p6_dealloc;
    P6CallType.tp_members = p6_members;
    P6CallType.tp_free = PyObject_Free;
    if (PyType_Ready(&P6CallType) < 0) return nullptr;
    return PyModule_Create(&module);
}

// Launch path of the eager calls (module mlora._host): checks the tensors of a call, collects their addresses and
// calls the C ABI of libmlora_hip.so on torch's current stream.
//
// Why it is native: an eager decode or prefill step is a few calls per layer, each checking up to fourteen tensors.
// In Python that took 6 to 22 us a call on top of the launches themselves (2.6 us each), more than the kernels of a
// small batch run.  Host time per call, launches included, in Python -> here: plan_decode 9.2 -> 4.5 us, bgmv over seven
// projections in two launches 19.4 -> 9.1 us (0.5 of it the allocation of its intermediate), sgmv_multi over seven (three
// launches) 34.5 -> 10.7 us.
// The reference's q, k and v calls of a layer, outputs included (deltas_ref and Lora_GPU._invoke): 21 -> 16 us, a step of four layers
// that the host bounds 86 -> 65 us (66 since results are kept for one thread, stream and capture).
// Nothing is kept from one call for the next: every tensor is checked and every slab looked up on every call.  A negative
// code of the C ABI is returned, and raised by the caller.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/mlora.h"

namespace {

struct PyFail {};   // a Python exception is set

[[noreturn]] void raise(PyObject *type, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw PyFail();
}

// ---------------------------------------------------------------- arguments
const at::Tensor &tensor(PyObject *o)
{
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "expected a tensor, got %.100s", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

struct Ref {        // an owned reference
    PyObject *o;
    explicit Ref(PyObject *p) : o(p) { if (!o) throw PyFail(); }
    ~Ref() { Py_DECREF(o); }
    Ref(const Ref &) = delete;
    Ref &operator=(const Ref &) = delete;
};

PyObject *s_page_tbl, *s_rank, *s_scaling, *s_work, *s_group, *s_perm, *s_seg_start, *s_seg_len, *s_seg_adapter,
    *s_chunk_start, *s_chunk_len, *s_chunk_adapter, *s_counters, *s_row_off, *s_tok_rank, *s_tok_scale, *s_T, *s_workspace,
    *s_n_slots, *s_max_pages, *s_page_rows, *s_n_pages, *s_max_rank, *s_tok_adapter, *s_dtype_code, *s_projections, *s_a_rows, *s_b_rows, *s_buf,
    *s_packed, *s_hin, *s_hout, *s_has_zeros, *s_tok_req, *s_tok_pos, *s_pages, *s_req_prefix, *s_prefix_pages, *s_prefix_len, *s_k, *s_v,
    *s_cos_sin, *s_interleaved, *s_batch, *s_n_q_heads, *s_n_kv_heads, *s_page_tokens, *s_n_req, *s_n_prefix, *s_rows,
    *s_state, *s_scratch, *s_cache;

void *attr_ptr(PyObject *o, PyObject *name)          // data pointer of a tensor attribute, null for None
{
    Ref a(PyObject_GetAttr(o, name));
    return a.o == Py_None ? nullptr : tensor(a.o).data_ptr();
}

long long as_int(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PyFail();
    return v;
}

bool is_true(PyObject *o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PyFail();
    return v != 0;
}

long long attr_int(PyObject *o, PyObject *name)
{
    Ref a(PyObject_GetAttr(o, name));
    return as_int(a.o);
}

void need_device(const at::Tensor &t)
{
    if (!t.is_cuda()) raise(PyExc_ValueError, "mlora kernels take device tensors; got a CPU tensor");
}

void need_contiguous(const at::Tensor &t)
{
    if (!t.is_contiguous()) raise(PyExc_ValueError, "mlora kernels take contiguous tensors");
}

struct List {       // a list or tuple of the caller
    PyObject *o;
    explicit List(PyObject *seq) : o(PySequence_Fast(seq, "expected a sequence")) { if (!o) throw PyFail(); }
    ~List() { Py_DECREF(o); }
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(o); }
    const at::Tensor &operator[](Py_ssize_t i) const { return tensor(PySequence_Fast_GET_ITEM(o, i)); }
};

void *stream() { return c10::hip::getCurrentHIPStream().stream(); }

// Other Python threads run while a launch is made (it waits when the device's queue is full).
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    Unlocked() = default;
    ~Unlocked() { PyEval_RestoreThread(state); }
    Unlocked(const Unlocked &) = delete;
    Unlocked &operator=(const Unlocked &) = delete;
};

template <typename F, typename... A>
int launch(F entry_point, A... args)                 // args are read before the lock goes
{
    const Unlocked u;
    return entry_point(args...);
}

// ---------------------------------------------------------------- a call over projections of one pool layer
struct Call {
    int n = 0, dtype = 0;
    at::ScalarType type = at::kHalf;
    void *y[MLORA_MAX_PROJ];
    const void *x[MLORA_MAX_PROJ], *a[MLORA_MAX_PROJ], *b[MLORA_MAX_PROJ];
    int32_t hin[MLORA_MAX_PROJ], hout[MLORA_MAX_PROJ];
};

// Address of a layer of the slab tensor [n_layers, rows, width] that `slabs` (a dict) holds for a projection.
const void *slab_of(PyObject *slabs, PyObject *name, int64_t layer)
{
    Ref o(PyObject_GetItem(slabs, name));
    const at::Tensor &t = tensor(o.o);
    const int64_t l = layer < 0 ? layer + t.size(0) : layer;
    if (l < 0 || l >= t.size(0)) raise(PyExc_IndexError, "layer %lld outside the pool's %lld layers", (long long)layer, (long long)t.size(0));
    return static_cast<const char *>(t.data_ptr()) + l * t.stride(0) * t.element_size();
}

// The call's widths, slabs, y and x, after every check of their placement, type and shape.
Call call_of(PyObject *pool, PyObject *projs, int64_t layer, const List &ys, const List &xs, int64_t T)
{
    Call c;
    const Ref names(PySequence_Fast(projs, "expected the projections' names"));
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(names.o);
    if (n < 1 || n > MLORA_MAX_PROJ || ys.size() != n || xs.size() != n)
        raise(PyExc_ValueError, "need 1..%d projections with one y and one x each", MLORA_MAX_PROJ);
    for (Py_ssize_t i = 0; i < n; i++) { need_device(ys[i]); need_device(xs[i]); }
    for (Py_ssize_t i = 0; i < n; i++) { need_contiguous(ys[i]); need_contiguous(xs[i]); }
    c.n = (int)n;
    c.dtype = (int)attr_int(pool, s_dtype_code);
    c.type = c.dtype == MLORA_F16 ? at::kHalf : at::kBFloat16;
    const Ref widths(PyObject_GetAttr(pool, s_projections)), a_rows(PyObject_GetAttr(pool, s_a_rows)), b_rows(PyObject_GetAttr(pool, s_b_rows));
    for (Py_ssize_t i = 0; i < n; i++) {
        PyObject *name = PySequence_Fast_GET_ITEM(names.o, i);
        const Ref w(PyObject_GetItem(widths.o, name)), hi(PySequence_GetItem(w.o, 0)), ho(PySequence_GetItem(w.o, 1));
        c.hin[i] = (int32_t)as_int(hi.o);
        c.hout[i] = (int32_t)as_int(ho.o);
        const at::Tensor &yt = ys[i], &xt = xs[i];
        if (yt.scalar_type() != c.type || xt.scalar_type() != c.type)
            raise(PyExc_TypeError, "x and y must have the pool dtype %s", c.type == at::kHalf ? "torch.float16" : "torch.bfloat16");
        if (xt.dim() != 2 || yt.dim() != 2 || xt.size(0) != T || xt.size(1) != c.hin[i] || yt.size(0) != T || yt.size(1) != c.hout[i])
            raise(PyExc_ValueError, "projection %S: expected x [%lld, %d] and y [%lld, %d]", name, (long long)T, (int)c.hin[i],
                  (long long)T, (int)c.hout[i]);
        c.y[i] = yt.data_ptr();
        c.x[i] = xt.data_ptr();
        c.a[i] = slab_of(a_rows.o, name, layer);
        c.b[i] = slab_of(b_rows.o, name, layer);
    }
    return c;
}

struct Tables {
    const int32_t *page_tbl, *rank;
    const float *scaling;
    int n_slots, max_pages, page_rows, max_rank;
    int64_t n_pages;
};

Tables tables(PyObject *pool)
{
    return {static_cast<const int32_t *>(attr_ptr(pool, s_page_tbl)), static_cast<const int32_t *>(attr_ptr(pool, s_rank)),
            static_cast<const float *>(attr_ptr(pool, s_scaling)), (int)attr_int(pool, s_n_slots), (int)attr_int(pool, s_max_pages),
            (int)attr_int(pool, s_page_rows), (int)attr_int(pool, s_max_rank), attr_int(pool, s_n_pages)};
}

// ---------------------------------------------------------------- decode
// A plan's buffer: data pointer (null for None), after a check that a launch on `like` may write `n` values of its type there.
void *buffer(PyObject *plan, PyObject *name, at::ScalarType type, int64_t n, const at::Tensor &like)
{
    Ref a(PyObject_GetAttr(plan, name));
    if (a.o == Py_None) return nullptr;
    const at::Tensor &t = tensor(a.o);
    if (t.numel() < n)
        raise(PyExc_ValueError, "the plan's %U holds %lld values, %lld needed: it was made for a smaller batch or pool", name,
              (long long)t.numel(), (long long)n);
    if (t.scalar_type() != type || !t.is_contiguous() || t.device() != like.device())
        raise(PyExc_ValueError, "the plan's %U must be a contiguous buffer of its type on the batch's device", name);
    return t.data_ptr();
}

// gather(pool, plan, tok_adapter, group)
PyObject *gather(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 4) raise(PyExc_TypeError, "gather takes 4 arguments");
    PyObject *pool = v[0], *plan = v[1];
    const at::Tensor &tok = tensor(v[2]);
    const Tables tb = tables(pool);
    const int64_t T = tok.numel(), segs = T < tb.n_slots ? T : tb.n_slots;
    auto i32 = [&](PyObject *name, int64_t n) { return static_cast<int32_t *>(buffer(plan, name, at::kInt, n, tok)); };
    // the per-token view, which is None unless the caller asked for it
    int32_t *row_off = i32(s_row_off, T * tb.max_pages), *tok_rank = i32(s_tok_rank, T);
    float *tok_scale = static_cast<float *>(buffer(plan, s_tok_scale, at::kFloat, T, tok));
    int32_t *perm = i32(s_perm, T), *seg_start = i32(s_seg_start, segs), *seg_len = i32(s_seg_len, segs), *seg_adapter = i32(s_seg_adapter, segs);
    int32_t *chunk_start = i32(s_chunk_start, T), *chunk_len = i32(s_chunk_len, T), *chunk_adapter = i32(s_chunk_adapter, T);
    int32_t *counters = i32(s_counters, MLORA_CNT_WORDS), *work = i32(s_work, (int64_t)MLORA_WORK_CAP(T) * MLORA_WORK_WORDS);
    need_device(tok);
    const int rc = launch(mlora_pool_gather, static_cast<const int32_t *>(tok.data_ptr()), (int)T, tb.page_tbl, tb.rank, tb.scaling, tb.n_slots,
                          tb.max_pages, tb.page_rows, tb.n_pages, row_off, tok_rank, tok_scale, perm, seg_start, seg_len, seg_adapter,
                          chunk_start, chunk_len, chunk_adapter, (int)as_int(v[3]), counters, work, stream());
    return PyLong_FromLong(rc);
}

// bgmv(pool, layer, projs, ys, xs, tok_adapter, plan or None, fused: True, False or None (by the sizes), accumulate)
PyObject *bgmv(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 9) raise(PyExc_TypeError, "bgmv takes 9 arguments");
    PyObject *pool = v[0], *plan = v[6] == Py_None ? nullptr : v[6];
    const List ys(v[3]), xs(v[4]);
    const at::Tensor &tok = tensor(v[5]);
    const bool accumulate = v[8] == Py_True;
    bool fused = v[7] != Py_None && is_true(v[7]);
    need_device(tok);
    need_contiguous(tok);
    if (tok.scalar_type() != at::kInt) raise(PyExc_TypeError, "tok_adapter must be int32");
    const int64_t T = tok.numel();
    const Call c = call_of(pool, v[2], as_int(v[1]), ys, xs, T);
    if (plan) {
        Ref made_for(PyObject_GetAttr(plan, s_tok_adapter));
        if (tensor(made_for.o).numel() != T) raise(PyExc_ValueError, "plan was built for a different batch size");
    } else if (v[7] == Py_None) {
        fused = true;
    } else if (!fused) {
        raise(PyExc_ValueError, "the two-launch form needs a plan");
    }
    const Tables tb = tables(pool);
    const int group = plan ? (int)attr_int(plan, s_group) : 1;
    // The intermediate of the two-launch forms is this call's own, from torch's allocator: calls that share a plan may
    // overlap on several streams or threads, and a captured graph keeps what its launches write.  It may be given back
    // when the launches are queued (the allocator hands it out again in stream order).
    at::Tensor room;
    int64_t ws_bytes = 0;
    int form = MLORA_FORM_FUSED;
    if (!fused && T > 0) {
        form = mlora_bgmv_form(c.n, c.hin, c.hout, (int)T, tb.n_slots, tb.max_rank, group, &ws_bytes);
        if (form < 0) return PyLong_FromLong(form);
        if (v[7] != Py_None) form = MLORA_FORM_PAIR;
        if (form != MLORA_FORM_FUSED) room = at::empty({ws_bytes}, tok.options().dtype(at::kByte));
    }
    const int rc = launch(
        mlora_bgmv_multi_form, form, c.n, c.y, c.x, c.a, c.b, c.hin, c.hout, static_cast<const int32_t *>(tok.data_ptr()), (int)T, tb.page_tbl, tb.rank, tb.scaling,
        tb.n_slots, tb.max_pages, tb.page_rows, tb.n_pages, tb.max_rank, plan ? static_cast<const int32_t *>(attr_ptr(plan, s_work)) : nullptr,
        group, room.defined() ? room.data_ptr() : nullptr, ws_bytes, c.dtype, accumulate, stream());
    return PyLong_FromLong(rc);
}

// A reference-layout decode call over n projections: every check, then the launch.  y, x, a, b give the tensors of a projection.
template <typename Y, typename X, typename A, typename B>
int ref_call(PyObject *plan, int n, Y y_of, X x_of, A a_of, B b_of, int layer, float scale, bool accumulate, int64_t T, int64_t N, int64_t L, int64_t r)
{
    for (int i = 0; i < n; i++) { need_device(y_of(i)); need_device(x_of(i)); need_device(a_of(i)); need_device(b_of(i)); }
    for (int i = 0; i < n; i++) { need_contiguous(y_of(i)); need_contiguous(x_of(i)); need_contiguous(a_of(i)); need_contiguous(b_of(i)); }
    void *y[MLORA_MAX_PROJ];
    const void *x[MLORA_MAX_PROJ], *a[MLORA_MAX_PROJ], *b[MLORA_MAX_PROJ];
    int32_t hin[MLORA_MAX_PROJ], hout[MLORA_MAX_PROJ];
    const at::ScalarType type = y_of(0).scalar_type();
    int max_hin = 0;
    for (int i = 0; i < n; i++) {
        const at::Tensor &yt = y_of(i), &xt = x_of(i), &at = a_of(i), &bt = b_of(i);
        if (at.dim() != 4 || bt.dim() != 4) raise(PyExc_ValueError, "wa_T_all must be [N, L, r, Hin] and wb_T_all [N, L, Hout, r]");
        if (at.size(0) != N || at.size(1) != L || at.size(2) != r || bt.size(0) != N || bt.size(1) != L || bt.size(3) != r)
            raise(PyExc_ValueError, "pool tensors disagree with each other or with the plan on N, L or r");
        if (xt.dim() != 2 || yt.dim() != 2 || xt.size(0) != T || xt.size(1) != at.size(3) || yt.size(0) != T || yt.size(1) != bt.size(2))
            raise(PyExc_ValueError, "x must be [B, Hin] and y [B, Hout] for the plan's batch");
        if (yt.scalar_type() != type || xt.scalar_type() != type || at.scalar_type() != type || bt.scalar_type() != type)
            raise(PyExc_TypeError, "y, x and the pools must share one 16-bit dtype");
        y[i] = yt.data_ptr(); x[i] = xt.data_ptr(); a[i] = at.data_ptr(); b[i] = bt.data_ptr();
        hin[i] = (int32_t)at.size(3); hout[i] = (int32_t)bt.size(2);
        max_hin = hin[i] > max_hin ? hin[i] : max_hin;
    }
    if (type != at::kHalf && type != at::kBFloat16) raise(PyExc_TypeError, "mlora kernels take float16 or bfloat16 tensors");
    const int64_t bytes = mlora_bgmv_workspace_bytes(n, (int)T, max_hin, (int)r);
    // this call's own, as in bgmv; straight from torch's allocator, a tensor takes longer to make
    at::DataPtr room;
    if (bytes > 0) {
        const c10::DeviceGuard device(y_of(0).device());
        room = c10::GetAllocator(at::kCUDA)->allocate((size_t)bytes);
    }
    void *ws = room.get();
    return launch(mlora_bgmv_reflayout_multi, n, y, x, a, b, hin, hout, attr_ptr(plan, s_buf), (int)T, (int)N, (int)L, (int)r,
                  layer, scale, (int)attr_int(plan, s_group), type == at::kHalf ? MLORA_F16 : MLORA_BF16, accumulate, ws, bytes, stream());
}

// bgmv_ref(plan, ys, xs, was, wbs, layer, scale, accumulate, T, N, L, r)
PyObject *bgmv_ref(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 12) raise(PyExc_TypeError, "bgmv_ref takes 12 arguments");
    const List ys(v[1]), xs(v[2]), was(v[3]), wbs(v[4]);
    const int n = (int)ys.size();
    if (n < 1 || n > MLORA_MAX_PROJ || xs.size() != n || was.size() != n || wbs.size() != n)
        raise(PyExc_ValueError, "need 1..%d projections with one y, x, wa and wb each", MLORA_MAX_PROJ);
    return PyLong_FromLong(ref_call(v[0], n, [&](int i) -> const at::Tensor & { return ys[i]; }, [&](int i) -> const at::Tensor & { return xs[i]; },
                                    [&](int i) -> const at::Tensor & { return was[i]; }, [&](int i) -> const at::Tensor & { return wbs[i]; },
                                    (int)as_int(v[5]), (float)PyFloat_AsDouble(v[6]), v[7] == Py_True, as_int(v[8]), as_int(v[9]),
                                    as_int(v[10]), as_int(v[11])));
}

// deltas_ref(plan, x, weights (wa, wb of every projection in turn), layer, T, N, L, r): the deltas alone, in new tensors of x's
// type; a tuple of them, or the C ABI's negative code
PyObject *deltas_ref(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 8) raise(PyExc_TypeError, "deltas_ref takes 8 arguments");
    const at::Tensor &x = tensor(v[1]);
    const List w(v[2]);
    const int n = (int)w.size() / 2;
    if (n < 1 || n > MLORA_MAX_PROJ || w.size() != 2 * n) raise(PyExc_ValueError, "need 1..%d projections with one wa and wb each", MLORA_MAX_PROJ);
    need_device(x);
    at::Tensor y[MLORA_MAX_PROJ];
    for (int i = 0; i < n; i++) {
        if (w[2 * i + 1].dim() != 4) raise(PyExc_ValueError, "wa_T_all must be [N, L, r, Hin] and wb_T_all [N, L, Hout, r]");
        y[i] = at::empty({x.size(0), w[2 * i + 1].size(2)}, x.options());
    }
    const int rc = ref_call(v[0], n, [&](int i) -> const at::Tensor & { return y[i]; }, [&](int) -> const at::Tensor & { return x; },
                            [&](int i) -> const at::Tensor & { return w[2 * i]; }, [&](int i) -> const at::Tensor & { return w[2 * i + 1]; },
                            (int)as_int(v[3]), 1.0f, false, as_int(v[4]), as_int(v[5]), as_int(v[6]), as_int(v[7]));
    if (rc) return PyLong_FromLong(rc);
    Ref out(PyTuple_New(n));
    for (int i = 0; i < n; i++) {
        PyObject *t = THPVariable_Wrap(y[i]);
        if (!t) throw PyFail();
        PyTuple_SET_ITEM(out.o, i, t);
    }
    Py_INCREF(out.o);
    return out.o;
}

// What orders a program's work: thread, device, stream and capture number (0 outside a capture).  What is queued under equal values
// runs in the order it is queued.
struct Order {
    int64_t v[4];
    Order()
    {
        const c10::hip::HIPStream s = c10::hip::getCurrentHIPStream();
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        unsigned long long id = 0;
        // the null stream cannot be captured, and asking it during another stream's capture is an error
        if (s.stream() && hipStreamGetCaptureInfo(s.stream(), &status, &id) != hipSuccess)
            raise(PyExc_RuntimeError, "the capture state of the current stream is not known: %s", hipGetErrorString(hipGetLastError()));
        v[0] = (int64_t)PyThread_get_thread_ident();
        v[1] = s.device_index();
        v[2] = (int64_t)(uintptr_t)s.stream();
        v[3] = status == hipStreamCaptureStatusNone ? 0 : (int64_t)id;
    }
};

PyObject *bytes_of(const int64_t *v, Py_ssize_t n) { return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(v), n * (Py_ssize_t)sizeof(int64_t)); }

// order(): it, as bytes to compare
PyObject *order(PyObject *const *, Py_ssize_t nargs)
{
    if (nargs != 0) raise(PyExc_TypeError, "order takes no arguments");
    const Order o;
    return bytes_of(o.v, 4);
}

// state(x, weights): the order, and which objects x and the weights are at which torch versions, as bytes to compare while the
// objects are alive.  One call for all of it: the q, k and v calls of a layer ask for it every time.
PyObject *state(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 2) raise(PyExc_TypeError, "state takes 2 arguments");
    const List w(v[1]);
    if (w.size() > 2 * MLORA_MAX_PROJ) raise(PyExc_ValueError, "at most %d weights", 2 * MLORA_MAX_PROJ);
    int64_t out[4 + 2 * (1 + 2 * MLORA_MAX_PROJ)];
    const Order o;
    for (int i = 0; i < 4; i++) out[i] = o.v[i];
    Py_ssize_t n = 4;
    auto add = [&](PyObject *t) { out[n++] = (int64_t)(uintptr_t)t; out[n++] = tensor(t)._version(); };
    add(v[0]);
    for (Py_ssize_t i = 0; i < w.size(); i++) add(PySequence_Fast_GET_ITEM(w.o, i));
    return bytes_of(out, n);
}

// ---------------------------------------------------------------- prefill
struct Segments { const int32_t *start, *len, *adapter; int64_t n; };

Segments segments(const at::Tensor &start, const at::Tensor &len, const at::Tensor &adapter)
{
    const at::Tensor *all[3] = {&start, &len, &adapter};
    for (const at::Tensor *t : all) need_device(*t);
    for (const at::Tensor *t : all) need_contiguous(*t);
    for (const at::Tensor *t : all)
        if (t->scalar_type() != at::kInt) raise(PyExc_TypeError, "segment arrays must be int32");
    const int64_t n = start.numel();
    if (len.numel() != n || adapter.numel() != n) raise(PyExc_ValueError, "seg_start, seg_len and seg_adapter must have the same length");
    return {static_cast<const int32_t *>(start.data_ptr()), static_cast<const int32_t *>(len.data_ptr()),
            static_cast<const int32_t *>(adapter.data_ptr()), n};
}

// prefill_plan(pool, seg_start, seg_len, seg_adapter, T, workspace, aligned)
PyObject *prefill_plan(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 7) raise(PyExc_TypeError, "prefill_plan takes 7 arguments");
    PyObject *pool = v[0];
    const Segments sg = segments(tensor(v[1]), tensor(v[2]), tensor(v[3]));
    const at::Tensor &ws = tensor(v[5]);
    need_device(ws);
    need_contiguous(ws);
    const Tables tb = tables(pool);
    const auto plan = v[6] == Py_True ? mlora_sgmv_plan_aligned : mlora_sgmv_plan;
    const int rc = launch(plan, sg.start, sg.len, sg.adapter, (int)sg.n, tb.page_tbl, tb.rank, tb.scaling, (int)as_int(v[4]),
                        tb.n_slots, tb.max_pages, tb.page_rows, tb.n_pages, tb.max_rank, ws.data_ptr(), ws.numel(), stream());
    return PyLong_FromLong(rc);
}

// sgmv_multi(pool, layer, projs, ys, xs, plan, accumulate)
PyObject *sgmv_multi(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 7) raise(PyExc_TypeError, "sgmv_multi takes 7 arguments");
    PyObject *pool = v[0], *plan = v[5];
    const List ys(v[3]), xs(v[4]);
    const int64_t T = attr_int(plan, s_T);
    const Call c = call_of(pool, v[2], as_int(v[1]), ys, xs, T);
    Ref start(PyObject_GetAttr(plan, s_seg_start)), len(PyObject_GetAttr(plan, s_seg_len)), adapter(PyObject_GetAttr(plan, s_seg_adapter)),
        wsp(PyObject_GetAttr(plan, s_workspace));
    const Segments sg = segments(tensor(start.o), tensor(len.o), tensor(adapter.o));
    const at::Tensor &ws = tensor(wsp.o);
    need_device(ws);
    need_contiguous(ws);
    const Tables tb = tables(pool);
    const int rc = launch(mlora_sgmv_multi_planned, c.n, c.y, c.x, c.a, c.b, c.hin, c.hout, sg.start, sg.len, sg.adapter, (int)sg.n, tb.page_tbl,
                                            tb.rank, tb.scaling, (int)T, tb.n_slots, tb.max_pages, tb.page_rows, tb.n_pages, tb.max_rank,
                                            c.dtype, v[6] == Py_True, ws.data_ptr(), ws.numel(), stream());
    return PyLong_FromLong(rc);
}

// ---------------------------------------------------------------- the decode step around the LoRA apply
// A launch goes to the current device's current stream, so every tensor of the call has to be there.
void need_here(const at::Tensor &t)
{
    need_device(t);
    if (t.get_device() != c10::hip::current_device())
        raise(PyExc_ValueError, "a tensor is on device %d, the current device is %d", (int)t.get_device(), (int)c10::hip::current_device());
}

int dtype_of(const at::Tensor &t)
{
    if (t.scalar_type() == at::kHalf) return MLORA_F16;
    if (t.scalar_type() == at::kBFloat16) return MLORA_BF16;
    raise(PyExc_TypeError, "mlora kernels take float16 or bfloat16 tensors");
}

struct Attr {       // an attribute that is a tensor, or None
    Ref r;
    Attr(PyObject *o, PyObject *name) : r(PyObject_GetAttr(o, name)) {}
    bool none() const { return r.o == Py_None; }
    const at::Tensor &t() const { return tensor(r.o); }
};

// w4_gemv(ys, xs, weights, accumulate)
PyObject *w4_gemv(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 4) raise(PyExc_TypeError, "w4_gemv takes 4 arguments");
    const List ys(v[0]), xs(v[1]);
    const Ref ws(PySequence_Fast(v[2], "expected a sequence of W4Weight"));
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(ws.o);
    if (n < 1 || n > MLORA_MAX_PROJ || ys.size() != n || xs.size() != n)
        raise(PyExc_ValueError, "need 1..%d projections with one y, one x and one weight each", MLORA_MAX_PROJ);
    for (Py_ssize_t i = 0; i < n; i++) { need_device(ys[i]); need_device(xs[i]); }
    for (Py_ssize_t i = 0; i < n; i++) { need_contiguous(ys[i]); need_contiguous(xs[i]); }
    const at::ScalarType type = xs[0].scalar_type();
    const int dtype = dtype_of(xs[0]);
    if (xs[0].dim() != 2) raise(PyExc_ValueError, "x must be [T, hin]");
    const int64_t T = xs[0].size(0);
    void *y[MLORA_MAX_PROJ];
    const void *x[MLORA_MAX_PROJ], *packed[MLORA_MAX_PROJ];
    int32_t hin[MLORA_MAX_PROJ], hout[MLORA_MAX_PROJ], group[MLORA_MAX_PROJ], zeros[MLORA_MAX_PROJ];
    for (Py_ssize_t i = 0; i < n; i++) {
        PyObject *w = PySequence_Fast_GET_ITEM(ws.o, i);
        const Attr buf(w, s_packed);
        const at::Tensor &b = buf.t(), &yt = ys[i], &xt = xs[i];
        hin[i] = (int32_t)attr_int(w, s_hin);
        hout[i] = (int32_t)attr_int(w, s_hout);
        group[i] = (int32_t)attr_int(w, s_group);
        const Ref has(PyObject_GetAttr(w, s_has_zeros));
        zeros[i] = is_true(has.o);
        if (yt.scalar_type() != type || xt.scalar_type() != type || attr_int(w, s_dtype_code) != dtype)
            raise(PyExc_TypeError, "x, y and the weights' scales must share one 16-bit dtype");
        if (xt.dim() != 2 || yt.dim() != 2 || xt.size(0) != T || xt.size(1) != hin[i] || yt.size(0) != T || yt.size(1) != hout[i])
            raise(PyExc_ValueError, "projection %d: expected x [%lld, %d] and y [%lld, %d]", (int)i, (long long)T, (int)hin[i], (long long)T, (int)hout[i]);
        if (b.scalar_type() != at::kByte || !b.is_contiguous() || b.numel() < mlora_w4_packed_bytes(hin[i], hout[i], group[i], zeros[i]))
            raise(PyExc_ValueError, "projection %d: the packed weight is not what its sizes need", (int)i);
        need_here(xt);
        need_here(yt);
        need_here(b);
        y[i] = yt.data_ptr(); x[i] = xt.data_ptr(); packed[i] = b.data_ptr();
    }
    if (T > (1 << 20)) raise(PyExc_ValueError, "at most 2^20 tokens");
    return PyLong_FromLong(launch(mlora_w4_gemv_multi, (int)n, y, x, packed, hin, hout, group, zeros, (int)T, dtype, (int)is_true(v[3]), stream()));
}

// The tables and token lists of a KVBatch.
struct Batch {
    const int32_t *tok_req, *tok_pos, *page_tbl, *req_prefix = nullptr, *prefix_tbl = nullptr, *prefix_len = nullptr;
    int T, n_req, max_pages, n_prefix = 0, max_prefix_pages = 0;
};

const int32_t *int_table(const at::Tensor &t, PyObject *name, int dims)
{
    need_device(t);
    if (t.scalar_type() != at::kInt) raise(PyExc_TypeError, "%U must be int32", name);
    if (t.dim() != dims) raise(PyExc_ValueError, "%U must have %d dimension(s)", name, dims);
    need_contiguous(t);
    need_here(t);
    for (int d = 0; d < dims; d++)
        if (t.size(d) > 0x7fffffffLL) raise(PyExc_ValueError, "%U is too large", name);
    return static_cast<const int32_t *>(t.data_ptr());
}

Batch batch_of(PyObject *o)
{
    Batch b;
    const Attr req(o, s_tok_req), pos(o, s_tok_pos), pages(o, s_pages), of(o, s_req_prefix), ppages(o, s_prefix_pages), plen(o, s_prefix_len);
    b.tok_req = int_table(req.t(), s_tok_req, 1);
    b.tok_pos = int_table(pos.t(), s_tok_pos, 1);
    b.page_tbl = int_table(pages.t(), s_pages, 2);
    b.T = (int)req.t().size(0);
    b.n_req = (int)pages.t().size(0);
    b.max_pages = (int)pages.t().size(1);
    if (pos.t().size(0) != b.T) raise(PyExc_ValueError, "tok_req and tok_pos must have the same length");
    if (of.none() != plen.none()) raise(PyExc_ValueError, "req_prefix and prefix_len go together");
    if (of.none()) {
        if (!ppages.none()) raise(PyExc_ValueError, "prefix_pages without req_prefix");
        return b;
    }
    b.req_prefix = int_table(of.t(), s_req_prefix, 1);
    b.prefix_len = int_table(plen.t(), s_prefix_len, 1);
    b.n_prefix = (int)plen.t().size(0);
    if (of.t().size(0) != b.n_req) raise(PyExc_ValueError, "req_prefix must have one entry for every row of pages");
    if (!ppages.none()) {
        b.prefix_tbl = int_table(ppages.t(), s_prefix_pages, 2);
        b.max_prefix_pages = (int)ppages.t().size(1);
        if (ppages.t().size(0) != b.n_prefix) raise(PyExc_ValueError, "prefix_pages and prefix_len must have the same length");
    }
    return b;
}

struct Cache {
    void *k, *v;
    int64_t n_pages;
    int page_tokens, n_kv_heads, head_dim, dtype;
    at::ScalarType type;
};

Cache cache_of(PyObject *o, int64_t layer)
{
    const Attr ka(o, s_k), va(o, s_v);
    const at::Tensor &k = ka.t(), &v = va.t();
    need_here(k);
    need_here(v);
    if (k.dim() != 5 || v.dim() != 5 || !k.is_contiguous() || !v.is_contiguous() || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
        raise(PyExc_ValueError, "the cache's k and v must be contiguous [n_layers, n_pages, n_kv_heads, page_tokens, head_dim] tensors of one type");
    if (layer < 0 || layer >= k.size(0)) raise(PyExc_IndexError, "layer %lld outside the cache's %lld layers", (long long)layer, (long long)k.size(0));
    const int64_t at = layer * k.stride(0) * k.element_size();
    return {static_cast<char *>(k.data_ptr()) + at, static_cast<char *>(v.data_ptr()) + at, k.size(1), (int)k.size(3), (int)k.size(2), (int)k.size(4),
            dtype_of(k), k.scalar_type()};
}

// Data pointer of [T, heads, head_dim] with only the tokens apart, and the elements from token to token.
void *token_rows(const char *name, const at::Tensor &t, int64_t T, int64_t heads, const Cache &c, int64_t &stride)
{
    need_device(t);
    if (t.scalar_type() != c.type) raise(PyExc_TypeError, "%s must have the cache's dtype", name);
    if (t.dim() != 3 || t.size(0) != T || t.size(1) != heads || t.size(2) != c.head_dim)
        raise(PyExc_ValueError, "%s must be [%lld, %lld, %d]", name, (long long)T, (long long)heads, c.head_dim);
    if (t.stride(2) != 1 || (heads > 1 && t.stride(1) != c.head_dim)) raise(PyExc_ValueError, "the heads of a token of %s must lie one behind the other", name);
    need_here(t);
    stride = T > 1 ? t.stride(0) : heads * c.head_dim;
    return t.data_ptr();
}

// kv_append(q or None, k, v, q_out or None, cache, layer, batch, rope or None, bad or None)
PyObject *kv_append(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 9) raise(PyExc_TypeError, "kv_append takes 9 arguments");
    const Cache c = cache_of(v[4], as_int(v[5]));
    const Batch b = batch_of(v[6]);
    int64_t q_stride = 0, o_stride = 0, k_stride, v_stride, q_heads = c.n_kv_heads;
    const void *q = nullptr;
    void *q_out = nullptr;
    if (v[0] != Py_None) {
        const at::Tensor &qt = tensor(v[0]);
        q_heads = qt.dim() == 3 ? qt.size(1) : 0;
        q = token_rows("q", qt, b.T, q_heads, c, q_stride);
        q_out = v[3] == Py_None ? const_cast<void *>(q) : token_rows("q_out", tensor(v[3]), b.T, q_heads, c, o_stride);
        if (v[3] == Py_None) o_stride = q_stride;
    } else if (v[3] != Py_None) {
        raise(PyExc_ValueError, "q_out without q");
    }
    const void *k = token_rows("k", tensor(v[1]), b.T, c.n_kv_heads, c, k_stride), *val = token_rows("v", tensor(v[2]), b.T, c.n_kv_heads, c, v_stride);
    const float *cos_sin = nullptr;
    int n_pos = 0, rot = 0, interleaved = 0;
    if (v[7] != Py_None) {
        const Attr table(v[7], s_cos_sin);
        const at::Tensor &t = table.t();
        need_here(t);
        if (t.scalar_type() != at::kFloat || t.dim() != 2 || !t.is_contiguous()) raise(PyExc_ValueError, "the rotation's table must be contiguous float32 [n_pos, rot]");
        const Ref inter(PyObject_GetAttr(v[7], s_interleaved));
        cos_sin = static_cast<const float *>(t.data_ptr());
        n_pos = (int)(t.size(0) < 0x7fffffffLL ? t.size(0) : 0x7fffffffLL);
        rot = (int)t.size(1);
        interleaved = is_true(inter.o);
    }
    int32_t *bad = nullptr;
    if (v[8] != Py_None) {
        const at::Tensor &t = tensor(v[8]);
        need_here(t);
        if (t.scalar_type() != at::kInt || t.numel() < 1) raise(PyExc_ValueError, "bad must be an int32 tensor of one value");
        bad = static_cast<int32_t *>(t.data_ptr());
    }
    return PyLong_FromLong(launch(mlora_kv_append, q, q_stride, q_out, o_stride, k, k_stride, val, v_stride, c.k, c.v, c.n_pages, c.page_tokens, (int)q_heads,
                                  c.n_kv_heads, c.head_dim, b.tok_req, b.tok_pos, b.T, b.page_tbl, b.n_req, b.max_pages, b.req_prefix, b.prefix_len,
                                  b.n_prefix, cos_sin, n_pos, rot, interleaved, bad, c.dtype, stream()));
}

void need_prefix_pages(const Batch &b)
{
    if (b.n_prefix > 0 && !b.prefix_tbl) raise(PyExc_ValueError, "attention over shared prefixes needs prefix_pages");
}

void *plan_buf(const at::Tensor &t)
{
    need_here(t);
    if (t.scalar_type() != at::kByte || !t.is_contiguous()) raise(PyExc_ValueError, "the plan's buf must be a contiguous uint8 buffer");
    return t.data_ptr();
}

// attn_plan(batch, buf, page_tokens, n_q_heads, n_kv_heads, head_dim)
PyObject *attn_plan(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 6) raise(PyExc_TypeError, "attn_plan takes 6 arguments");
    const Batch b = batch_of(v[0]);
    need_prefix_pages(b);
    const at::Tensor &buf = tensor(v[1]);
    return PyLong_FromLong(launch(mlora_attn_plan, b.tok_req, b.tok_pos, b.T, b.n_req, b.max_pages, b.req_prefix, b.prefix_len, b.n_prefix,
                                  b.max_prefix_pages, (int)as_int(v[2]), (int)as_int(v[3]), (int)as_int(v[4]), (int)as_int(v[5]), plan_buf(buf), buf.numel(), stream()));
}

// prefix_attention(q, out, cache, layer, plan, scale)
PyObject *prefix_attention(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 6) raise(PyExc_TypeError, "prefix_attention takes 6 arguments");
    PyObject *plan = v[4];
    const Cache c = cache_of(v[2], as_int(v[3]));
    const Ref batch(PyObject_GetAttr(plan, s_batch));
    const Batch b = batch_of(batch.o);
    need_prefix_pages(b);
    const int64_t q_heads = attr_int(plan, s_n_q_heads);
    if (attr_int(plan, s_n_kv_heads) != c.n_kv_heads || attr_int(plan, s_page_tokens) != c.page_tokens || attr_int(plan, s_T) != b.T ||
        attr_int(plan, s_n_req) != b.n_req || attr_int(plan, s_n_prefix) != b.n_prefix)
        raise(PyExc_ValueError, "the plan was made for another cache layout, batch size or number of requests or prefixes");
    int64_t q_stride, o_stride;
    const void *q = token_rows("q", tensor(v[0]), b.T, q_heads, c, q_stride);
    void *out = token_rows("out", tensor(v[1]), b.T, q_heads, c, o_stride);
    const Attr bufa(plan, s_buf);
    const at::Tensor &buf = bufa.t();
    const void *pb = plan_buf(buf);
    const double scale = PyFloat_AsDouble(v[5]);
    if (scale == -1.0 && PyErr_Occurred()) throw PyFail();
    // this call's own, as in bgmv_ref
    const int64_t bytes = mlora_attn_workspace_bytes(b.T, b.n_prefix, (int)q_heads, c.n_kv_heads, c.head_dim);
    at::DataPtr room;
    if (b.T > 0 && bytes > 0) {
        const c10::DeviceGuard device(buf.device());
        room = c10::GetAllocator(at::kCUDA)->allocate((size_t)bytes);
    }
    return PyLong_FromLong(launch(mlora_prefix_attention, out, o_stride, q, q_stride, static_cast<const void *>(c.k), static_cast<const void *>(c.v), c.n_pages, c.page_tokens, (int)q_heads, c.n_kv_heads,
                                  c.head_dim, b.tok_req, b.tok_pos, b.T, b.page_tbl, b.n_req, b.max_pages, b.req_prefix, b.prefix_tbl, b.prefix_len, b.n_prefix,
                                  b.max_prefix_pages, (float)scale, pb, buf.numel(), room.get(), bytes, c.dtype, stream()));
}

// ---------------------------------------------------------------- microscaled operands
struct Packed {     // an MX4Tensor
    const at::Tensor t;
    int rows, k;
    explicit Packed(PyObject *o) : t(Attr(o, s_packed).t()), rows((int)attr_int(o, s_rows)), k((int)attr_int(o, s_k))
    {
        need_here(t);
        if (t.scalar_type() != at::kByte || !t.is_contiguous() || t.numel() < mlora_mx4_bytes(rows, k))
            raise(PyExc_ValueError, "the packed operand is not what its sizes need");
    }
};

// Rows of `k` elements next to each other, and the elements from row to row.
void *rows_of(const char *name, const at::Tensor &t, int64_t k, int64_t &stride)
{
    need_device(t);
    if (t.dim() != 2 || (k >= 0 && t.size(1) != k)) raise(PyExc_ValueError, "%s must be [rows, k]", name);
    if (t.size(0) > 0x7fffffffLL || t.size(1) > 0x7fffffffLL) raise(PyExc_ValueError, "%s is too large", name);
    if (t.stride(1) != 1 && t.size(1) > 1) raise(PyExc_ValueError, "the elements of a row of %s must lie one behind the other", name);
    need_here(t);
    stride = t.size(0) > 1 ? t.stride(0) : t.size(1);
    return t.data_ptr();
}

at::Tensor new_bytes(int64_t n, const at::Tensor &like)
{
    const c10::DeviceGuard device(like.device());
    return at::empty({n}, like.options().dtype(at::kByte));
}

// mx4_quantize(x, packed or None) -> (packed, rows, k): the caller's buffer, which must have the room that x needs, or a new one
PyObject *mx4_quantize(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 2) raise(PyExc_TypeError, "mx4_quantize takes 2 arguments");
    const at::Tensor &x = tensor(v[0]);
    const int dtype = dtype_of(x);
    int64_t stride;
    const void *rows = rows_of("x", x, -1, stride);
    const int64_t need = mlora_mx4_bytes((int)x.size(0), (int)x.size(1));
    if (need < 0) return PyLong_FromLong((long)need);
    at::Tensor b = v[1] == Py_None ? new_bytes(need, x) : tensor(v[1]);
    need_here(b);
    if (b.scalar_type() != at::kByte || !b.is_contiguous()) raise(PyExc_ValueError, "packed must be a contiguous uint8 buffer");
    const int rc = launch(mlora_mx4_quantize, rows, stride, (int)x.size(0), (int)x.size(1), dtype, b.data_ptr(), b.numel(), stream());
    if (rc) return PyLong_FromLong(rc);
    PyObject *packed = v[1] == Py_None ? THPVariable_Wrap(std::move(b)) : Py_NewRef(v[1]);
    if (!packed) throw PyFail();
    return Py_BuildValue("(Nii)", packed, (int)x.size(0), (int)x.size(1));
}

// mx4_values(packed operand, out or None, dtype code for a new one) -> out
PyObject *mx4_values(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 3) raise(PyExc_TypeError, "mx4_values takes 3 arguments");
    const Packed p(v[0]);
    at::Tensor out;
    if (v[1] == Py_None) {
        const c10::DeviceGuard device(p.t.device());
        out = at::empty({p.rows, p.k}, p.t.options().dtype(as_int(v[2]) == MLORA_F16 ? at::kHalf : at::kBFloat16));
    } else {
        out = tensor(v[1]);
    }
    const int dtype = dtype_of(out);
    int64_t stride;
    void *rows = rows_of("out", out, p.k, stride);
    if (out.size(0) != p.rows) raise(PyExc_ValueError, "out must have %d rows", p.rows);
    const int rc = launch(mlora_mx4_values, p.t.data_ptr(), p.t.numel(), p.rows, p.k, rows, stride, dtype, stream());
    if (rc) return PyLong_FromLong(rc);
    if (v[1] != Py_None) return Py_NewRef(v[1]);
    PyObject *o = THPVariable_Wrap(std::move(out));
    if (!o) throw PyFail();
    return o;
}

// mx4_gemm(ys, xs, weights, accumulate)
PyObject *mx4_gemm(PyObject *const *v, Py_ssize_t nargs)
{
    if (nargs != 4) raise(PyExc_TypeError, "mx4_gemm takes 4 arguments");
    const List ys(v[0]);
    const Ref xs(PySequence_Fast(v[1], "expected a sequence of MX4Tensor")), ws(PySequence_Fast(v[2], "expected a sequence of MX4Tensor"));
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(ws.o);
    if (n < 1 || n > MLORA_MAX_PROJ || ys.size() != n || PySequence_Fast_GET_SIZE(xs.o) != n)
        raise(PyExc_ValueError, "need 1..%d projections with one y, one x and one weight each", MLORA_MAX_PROJ);
    const at::ScalarType type = ys[0].scalar_type();
    const int dtype = dtype_of(ys[0]);
    void *y[MLORA_MAX_PROJ];
    const void *x[MLORA_MAX_PROJ], *w[MLORA_MAX_PROJ];
    int32_t hin[MLORA_MAX_PROJ], hout[MLORA_MAX_PROJ];
    int T = 0;
    for (Py_ssize_t i = 0; i < n; i++) {
        const Packed px(PySequence_Fast_GET_ITEM(xs.o, i)), pw(PySequence_Fast_GET_ITEM(ws.o, i));
        const at::Tensor &yt = ys[i];
        need_here(yt);
        need_contiguous(yt);
        if (i == 0) T = px.rows;
        if (yt.scalar_type() != type) raise(PyExc_TypeError, "all y must share one 16-bit dtype");
        if (px.rows != T || px.k != pw.k || yt.dim() != 2 || yt.size(0) != T || yt.size(1) != pw.rows)
            raise(PyExc_ValueError, "projection %d: expected x [%d, %d] and y [%d, %d]", (int)i, T, pw.k, T, pw.rows);
        y[i] = yt.data_ptr(); x[i] = px.t.data_ptr(); w[i] = pw.t.data_ptr();
        hin[i] = pw.k; hout[i] = pw.rows;
    }
    return PyLong_FromLong(launch(mlora_mx4_gemm_multi, (int)n, y, x, w, hin, hout, T, dtype, (int)is_true(v[3]), stream()));
}

// ---------------------------------------------------------------- page tables
struct Pages {      // a KVPages
    const at::Tensor state, scratch;
    const Cache c;
    int64_t n_layers;
    int n_req, max_pages;
    Pages(PyObject *o, PyObject *cache, PyObject *k) : state(Attr(o, s_state).t()), scratch(Attr(o, s_scratch).t()), c(cache_of(cache, 0)),
        n_layers(tensor(k).size(0)), n_req((int)attr_int(o, s_n_req)), max_pages((int)attr_int(o, s_max_pages))
    {
        for (const at::Tensor &t : {state, scratch}) {
            need_here(t);
            if (t.scalar_type() != at::kInt || !t.is_contiguous()) raise(PyExc_ValueError, "the tables' state and scratch must be contiguous int32 buffers");
        }
    }
};

template <typename F>
PyObject *with_pages(PyObject *const *v, Py_ssize_t nargs, bool wants, F call)
{
    if (nargs != (wants ? 2 : 1)) raise(PyExc_TypeError, "pages calls take the tables and, but for compact, the rows' values");
    const Ref cache(PyObject_GetAttr(v[0], s_cache)), k(PyObject_GetAttr(cache.o, s_k));
    const Pages p(v[0], cache.o, k.o);
    const int32_t *want = nullptr;
    if (wants) {
        const at::Tensor &t = tensor(v[1]);
        need_here(t);
        if (t.scalar_type() != at::kInt) raise(PyExc_TypeError, "the rows' values must be int32");
        if (t.dim() != 1 || t.size(0) != p.n_req || !t.is_contiguous()) raise(PyExc_ValueError, "expected one contiguous value for each of the %d rows", p.n_req);
        want = static_cast<const int32_t *>(t.data_ptr());
    }
    return PyLong_FromLong(call(p, want));
}

// pages_resize(pages, want)
PyObject *pages_resize(PyObject *const *v, Py_ssize_t nargs)
{
    return with_pages(v, nargs, true, [](const Pages &p, const int32_t *want) {
        return launch(mlora_pages_resize, p.state.data_ptr(), p.state.numel(), p.scratch.data_ptr(), p.scratch.numel(), want, p.n_req, p.max_pages, p.c.k,
                      p.c.v, (int)p.n_layers, p.c.n_pages, p.c.n_kv_heads, p.c.page_tokens, p.c.head_dim, stream());
    });
}

// pages_fork(pages, parent)
PyObject *pages_fork(PyObject *const *v, Py_ssize_t nargs)
{
    return with_pages(v, nargs, true, [](const Pages &p, const int32_t *parent) {
        return launch(mlora_pages_fork, p.state.data_ptr(), p.state.numel(), p.scratch.data_ptr(), p.scratch.numel(), parent, p.n_req, p.max_pages,
                      p.c.n_pages, p.c.page_tokens, stream());
    });
}

// pages_compact(pages)
PyObject *pages_compact(PyObject *const *v, Py_ssize_t nargs)
{
    return with_pages(v, nargs, false, [](const Pages &p, const int32_t *) {
        return launch(mlora_pages_compact, p.state.data_ptr(), p.state.numel(), p.scratch.data_ptr(), p.scratch.numel(), p.n_req, p.max_pages, p.c.k,
                      p.c.v, (int)p.n_layers, p.c.n_pages, p.c.n_kv_heads, p.c.page_tokens, p.c.head_dim, stream());
    });
}

// ---------------------------------------------------------------- module
template <PyObject *(*F)(PyObject *const *, Py_ssize_t)>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    try {
        return F(args, nargs);
    } catch (const PyFail &) {
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

#define MLORA_FN(name) {#name, (PyCFunction)(void (*)())entry<name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MLORA_FN(gather), MLORA_FN(bgmv), MLORA_FN(bgmv_ref), MLORA_FN(deltas_ref), MLORA_FN(order), MLORA_FN(state), MLORA_FN(prefill_plan),
                         MLORA_FN(sgmv_multi), MLORA_FN(w4_gemv), MLORA_FN(kv_append), MLORA_FN(attn_plan), MLORA_FN(prefix_attention),
                         MLORA_FN(mx4_quantize), MLORA_FN(mx4_values), MLORA_FN(mx4_gemm), MLORA_FN(pages_resize), MLORA_FN(pages_fork), MLORA_FN(pages_compact), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Native launch path of mlora's eager calls.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host()
{
    const std::pair<PyObject **, const char *> names[] = {
        {&s_page_tbl, "page_tbl"}, {&s_rank, "rank"}, {&s_scaling, "scaling"}, {&s_work, "work"}, {&s_group, "group"},
        {&s_perm, "perm"}, {&s_seg_start, "seg_start"}, {&s_seg_len, "seg_len"}, {&s_seg_adapter, "seg_adapter"},
        {&s_chunk_start, "chunk_start"}, {&s_chunk_len, "chunk_len"}, {&s_chunk_adapter, "chunk_adapter"}, {&s_counters, "counters"},
        {&s_row_off, "row_off"}, {&s_tok_rank, "tok_rank"}, {&s_tok_scale, "tok_scale"}, {&s_T, "T"}, {&s_workspace, "workspace"},
        {&s_n_slots, "n_slots"}, {&s_max_pages, "max_pages"}, {&s_page_rows, "page_rows"}, {&s_n_pages, "n_pages"},
        {&s_max_rank, "max_rank"}, {&s_tok_adapter, "tok_adapter"}, {&s_dtype_code, "dtype_code"}, {&s_projections, "projections"},
        {&s_a_rows, "a_rows"}, {&s_b_rows, "b_rows"}, {&s_buf, "buf"},
        {&s_packed, "packed"}, {&s_hin, "hin"}, {&s_hout, "hout"}, {&s_has_zeros, "has_zeros"}, {&s_tok_req, "tok_req"},
        {&s_tok_pos, "tok_pos"}, {&s_pages, "pages"}, {&s_req_prefix, "req_prefix"}, {&s_prefix_pages, "prefix_pages"},
        {&s_prefix_len, "prefix_len"}, {&s_k, "k"}, {&s_v, "v"}, {&s_cos_sin, "cos_sin"}, {&s_interleaved, "interleaved"},
        {&s_batch, "batch"}, {&s_n_q_heads, "n_q_heads"}, {&s_n_kv_heads, "n_kv_heads"}, {&s_page_tokens, "page_tokens"},
        {&s_n_req, "n_req"}, {&s_n_prefix, "n_prefix"}, {&s_rows, "rows"}, {&s_state, "state"}, {&s_scratch, "scratch"}, {&s_cache, "cache"}};
    for (const auto &p : names)
        if (!(*p.first = PyUnicode_InternFromString(p.second))) return nullptr;
    return PyModule_Create(&module);
}

// Native call path of the Python op interface (tileinfer_hip/backend.py): reads the tensors,
// checks them as backend.py does and calls the C ABI, without building ctypes structures.
//
// Every function returns the ti_status of the call, or -1 where it takes the arguments not to
// be plain ones (a tensor subclass, a CPU or non-contiguous tensor, a shape or type that does
// not fit): backend.py then runs its own checks, which raise, or make the call. So what is
// accepted and what is raised is defined there alone.
//
// Why: attention_inputs_ and paged_attention_ of a short step took 20.8 us a pair through
// Python checks and ctypes, whatever the GPU needed (its three kernels 8 to 12); here 9.3 us,
// and one float32 token (16 / 8 heads, 1024 positions) 23.8 -> 11.3 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "tileinfer_hip.h"

namespace {

decltype(&ti_attention) f_attention;
decltype(&ti_attention_inputs) f_inputs;
decltype(&ti_store_kv) f_store_kv;
decltype(&ti_rope) f_rope;
decltype(&ti_rmsnorm) f_rmsnorm;
decltype(&ti_update_key_bounds) f_bounds;
decltype(&ti_select_pages) f_select;
decltype(&ti_sparse_attention) f_sparse;
decltype(&ti_verify_draft) f_verify;
decltype(&ti_window_attention) f_window;
decltype(&ti_reserve_pages) f_reserve;
decltype(&ti_release_pages) f_release;
PyObject *int8_pages, *key_bounds, *fp8_pages, *page_pool;   // Int8Pages, KeyBounds, Fp8Pages, PagePool
PyObject *n_free, *n_free_count, *n_tables, *n_lengths, *n_behind, *n_ticket, *n_window, *n_sinks;
PyObject *n_layer_q, *n_layer_scale, *n_smooth, *n_half, *n_cos_sin, *n_bounds, *n_scale, *n_channel, *n_page_size;   // attribute names

struct NotPlain {};   // leave the call to backend.py

// A plain GPU tensor of contiguous elements.
const at::Tensor &dev(PyObject *o) {
    if (!THPVariable_CheckExact(o)) throw NotPlain{};
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous()) throw NotPlain{};
    return t;
}
const at::Tensor *dev_or_none(PyObject *o) { return o == Py_None ? nullptr : &dev(o); }
void require(bool ok) {
    if (!ok) throw NotPlain{};
}
const int32_t *i32(const at::Tensor &t) {
    require(t.scalar_type() == at::kInt);
    return static_cast<const int32_t *>(t.data_ptr());
}
int dtype_of(const at::Tensor &t) {
    if (t.scalar_type() == at::kBFloat16) return TI_BF16;
    require(t.scalar_type() == at::kFloat);
    return TI_F32;
}
float number(PyObject *o) {
    require(PyFloat_CheckExact(o) || PyLong_CheckExact(o));
    const double x = PyFloat_AsDouble(o);
    require(!PyErr_Occurred());
    return (float)x;
}
long integer(PyObject *o) {
    require(PyLong_CheckExact(o));
    const long x = PyLong_AsLong(o);
    require(!PyErr_Occurred());
    return x;
}
void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// An attribute held for the scope of a call.
struct Attr {
    PyObject *o;
    Attr(PyObject *of, PyObject *name) : o(PyObject_GetAttr(of, name)) { require(o != nullptr); }
    ~Attr() { Py_DECREF(o); }
    Attr(const Attr &) = delete;
};

// An 8-bit block layer, on the current GPU (as OneGpu below).
ti_kv_cache fp8_cache_of(PyObject *k, PyObject *v) {
    require(Py_TYPE(k) == Py_TYPE(v));
    Attr lq(k, n_layer_q), lq2(v, n_layer_q), ls(k, n_layer_scale), ls2(v, n_layer_scale), h0(k, n_half), h1(v, n_half);
    require(lq.o == lq2.o && ls.o == ls2.o && integer(h0.o) == 0 && integer(h1.o) == 1);
    const at::Tensor &q = dev(lq.o), &s = dev(ls.o);
    require(q.dim() == 5 && q.size(0) == 2 && q.element_size() == 1 && s.scalar_type() == at::kFloat && s.sizes() == q.sizes().slice(0, 3));
    require(q.device() == s.device() && q.device().index() == c10::hip::current_device());
    ti_kv_cache c{};
    c.kind = TI_KV_FP8;
    c.layer_q = static_cast<int8_t *>(q.data_ptr());
    c.layer_scale = static_cast<float *>(s.data_ptr());
    c.num_pages = (int32_t)q.size(1), c.kv_heads = (int32_t)q.size(2);
    c.page_size = (int32_t)q.size(3), c.head_dim = (int32_t)q.size(4);
    return c;
}

// The layer's cache: dense pools [pages][H][P][D] of element type `like`, an Int8Pages or an Fp8Pages pair.
ti_kv_cache cache_of(PyObject *k, PyObject *v, at::ScalarType like) {
    if ((PyObject *)Py_TYPE(k) == fp8_pages || (PyObject *)Py_TYPE(v) == fp8_pages) return fp8_cache_of(k, v);
    ti_kv_cache c{};
    if ((PyObject *)Py_TYPE(k) == int8_pages || (PyObject *)Py_TYPE(v) == int8_pages) {
        require(Py_TYPE(k) == Py_TYPE(v));
        Attr lq(k, n_layer_q), lq2(v, n_layer_q), ls(k, n_layer_scale), sm(k, n_smooth), h0(k, n_half), h1(v, n_half);
        require(lq.o == lq2.o && integer(h0.o) == 0 && integer(h1.o) == 1);
        const at::Tensor &q = dev(lq.o);
        require(q.dim() == 5);
        c.kind = TI_KV_INT8;
        c.layer_q = static_cast<int8_t *>(q.data_ptr());
        c.layer_scale = static_cast<float *>(dev(ls.o).data_ptr());
        c.smooth = static_cast<const float *>(dev(sm.o).data_ptr());
        c.num_pages = (int32_t)q.size(1), c.kv_heads = (int32_t)q.size(2);
        c.page_size = (int32_t)q.size(3), c.head_dim = (int32_t)q.size(4);
        return c;
    }
    const at::Tensor &kt = dev(k), &vt = dev(v);
    require(kt.dim() == 4 && kt.sizes() == vt.sizes() && kt.scalar_type() == like && vt.scalar_type() == like);
    c.kind = TI_KV_DENSE;
    c.k_pages = kt.data_ptr();
    c.v_pages = vt.data_ptr();
    c.num_pages = (int32_t)kt.size(0), c.kv_heads = (int32_t)kt.size(1);
    c.page_size = (int32_t)kt.size(2), c.head_dim = (int32_t)kt.size(3);
    return c;
}

// The GPU that the calls below launch on: the current one, and that of all their tensors (backend.py
// makes another one current).
struct OneGpu {
    c10::Device d;
    OneGpu(const at::Tensor &t) : d(t.device()) { require(d.index() == c10::hip::current_device()); }
    const at::Tensor &operator()(PyObject *o) const {
        const at::Tensor &t = dev(o);
        require(t.device() == d);
        return t;
    }
    const at::Tensor *or_none(PyObject *o) const { return o == Py_None ? nullptr : &(*this)(o); }
    // The layer's cache with its tensors on this GPU.
    ti_kv_cache cache(PyObject *k, PyObject *v, at::ScalarType like) const {
        const ti_kv_cache c = cache_of(k, v, like);
        if (c.kind == TI_KV_DENSE) {
            (*this)(k), (*this)(v);
        } else if (c.kind == TI_KV_FP8) {
            Attr q(k, n_layer_q), s(k, n_layer_scale);
            (*this)(q.o), (*this)(s.o);
        } else {
            Attr q(k, n_layer_q), s(k, n_layer_scale), m(k, n_smooth);
            (*this)(q.o), (*this)(s.o), (*this)(m.o);
        }
        return c;
    }
};

// The tensors of a KeyBounds; its shape is (pages, kv_heads, page_size, D).
struct Bounds {
    Attr b, s, c;
    ti_key_bounds ptr;
    int64_t pages, heads, page, D;
    Bounds(PyObject *o, const OneGpu &gpu)
        : b((require((PyObject *)Py_TYPE(o) == key_bounds), o), n_bounds), s(o, n_scale), c(o, n_channel) {
        const at::Tensor &bt = gpu(b.o), &st = gpu(s.o), *ct = gpu.or_none(c.o);
        const Attr p(o, n_page_size);
        require(bt.dim() == 4 && bt.scalar_type() == at::kChar && st.scalar_type() == at::kFloat && bt.size(2) == 2);
        require(st.dim() == 2 && st.size(0) == bt.size(0) && st.size(1) == bt.size(1));
        pages = bt.size(0), heads = bt.size(1), page = integer(p.o), D = bt.size(3);
        require(!ct || (ct->scalar_type() == at::kFloat && ct->dim() == 2 && ct->size(0) == heads && ct->size(1) == D));
        ptr = {static_cast<int8_t *>(bt.data_ptr()), static_cast<float *>(st.data_ptr()),
               ct ? static_cast<const float *>(ct->data_ptr()) : nullptr};
    }
};

// The step of query tokens that block_tables, positions, query_start_loc and max_query_len give.
struct StepArgs {
    const int32_t *tables, *positions, *qsl;
    int seqs, n, total, stride;
    StepArgs(const OneGpu &gpu, PyObject *o_tables, PyObject *o_positions, PyObject *o_qsl, PyObject *o_n) {
        const at::Tensor &bt = gpu(o_tables), &pos = gpu(o_positions), *q = gpu.or_none(o_qsl);
        tables = i32(bt), positions = i32(pos), qsl = q ? i32(*q) : nullptr;
        require(bt.dim() == 1 || bt.dim() == 2);
        const int64_t B = bt.dim() == 2 ? bt.size(0) : 1;
        require(B > 0 && (!q || (o_n != Py_None && q->numel() == B + 1)));
        seqs = (int)B, total = (int)pos.numel(), stride = (int)bt.size(-1);
        n = (int)(o_n != Py_None ? integer(o_n) : total / B);
    }
};

// Runs `body` (checks, then the call without the interpreter lock) and returns its status.
template <typename F>
PyObject *guarded(Py_ssize_t nargs, Py_ssize_t want, F &&body) {
    long status = -1;
    if (nargs == want && f_attention) {
        try {
            status = body();
        } catch (...) {
            status = -1;
        }
    }
    PyErr_Clear();
    return PyLong_FromLong(status);
}
template <typename F>
long unlocked(F &&call) {
    long status;
    Py_BEGIN_ALLOW_THREADS
    status = call();
    Py_END_ALLOW_THREADS
    return status;
}

// (out, workspace, q, k_pages, v_pages, block_tables, positions, scale, causal,
//  query_start_loc, max_query_len, path, one_sequence)
PyObject *py_attention(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 13, [&]() -> long {
        const at::Tensor &out = dev(a[0]), &q = dev(a[2]), &bt = dev(a[5]), &pos = dev(a[6]);
        const at::Tensor *ws = dev_or_none(a[1]), *qsl = dev_or_none(a[9]);
        require(q.dim() == 3 && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type());
        const ti_kv_cache c = cache_of(a[3], a[4], q.scalar_type());
        ti_attention_args g{};
        g.dtype = dtype_of(q);
        g.positions = i32(pos);
        g.block_tables = i32(bt);
        require(c.kind != TI_KV_FP8 || q.device().index() == c10::hip::current_device());
        require(pos.numel() == q.size(0) && q.size(2) == c.head_dim && PyBool_Check(a[8]));
        const bool rows = bt.dim() == 2 && a[12] != Py_True;
        const int64_t B = rows ? bt.size(0) : 1;
        require(B > 0 && (!qsl || a[10] != Py_None));
        g.q_heads = (int32_t)q.size(1);
        g.num_seqs = (int32_t)B;
        g.max_query_len = (int32_t)(a[10] != Py_None ? integer(a[10]) : q.size(0) / B);
        g.total_tokens = (int32_t)q.size(0);
        g.block_table_stride = (int32_t)(rows ? bt.size(1) : bt.numel());
        g.q = q.data_ptr();
        g.out = out.data_ptr();
        g.query_start_loc = qsl ? i32(*qsl) : nullptr;
        g.scale = number(a[7]);
        g.causal = a[8] == Py_True;
        g.path = (int32_t)integer(a[11]);
        g.workspace = ws ? ws->data_ptr() : nullptr;
        g.workspace_bytes = ws ? (size_t)ws->nbytes() : 0;
        void *s = stream_of(q);
        return unlocked([&] { return f_attention(&g, &c, s); });
    });
}

// (q, k_pages, v_pages, qkv, q_norm, k_norm, table, positions, slots, eps)
PyObject *py_inputs(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 10, [&]() -> long {
        const Attr table(a[6], n_cos_sin);
        const at::Tensor &q = dev(a[0]), &qkv = dev(a[3]), &cs = dev(table.o), &pos = dev(a[7]), &slots = dev(a[8]);
        const at::Tensor *qn = dev_or_none(a[4]), *kn = dev_or_none(a[5]);
        require(q.dim() == 3 && !qn == !kn);
        const int64_t n = q.size(0), nq = q.size(1), D = q.size(2);
        const ti_kv_cache c = cache_of(a[1], a[2], q.scalar_type());
        require(c.kind != TI_KV_FP8 || q.device().index() == c10::hip::current_device());
        require(qkv.scalar_type() == q.scalar_type() && qkv.numel() == n * (nq + 2 * (int64_t)c.kv_heads) * D && D == c.head_dim);
        require(cs.scalar_type() == q.scalar_type() && cs.dim() == 3 && cs.size(1) == 2 && cs.size(2) == D);
        require(pos.numel() == n && slots.numel() == n);
        const int dtype = dtype_of(q);
        const int32_t *p = i32(pos), *sl = i32(slots);
        const float eps = number(a[9]);
        void *s = stream_of(q), *qo = q.data_ptr();
        const void *x = qkv.data_ptr(), *w1 = qn ? qn->data_ptr() : nullptr, *w2 = kn ? kn->data_ptr() : nullptr, *t = cs.data_ptr();
        const int len = (int)cs.size(0);
        return unlocked([&] { return f_inputs(dtype, qo, &c, x, w1, w2, t, len, p, sl, (int)n, (int)nq, eps, s); });
    });
}

// (k_pages, v_pages, k, v, slots)
PyObject *py_store_kv(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 5, [&]() -> long {
        const at::Tensor &k = dev(a[2]), &v = dev(a[3]), &slots = dev(a[4]);
        require(k.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type());
        const ti_kv_cache c = cache_of(a[0], a[1], k.scalar_type());
        require(c.kind != TI_KV_FP8 || k.device().index() == c10::hip::current_device());
        require(k.size(1) == c.kv_heads && k.size(2) == c.head_dim && slots.numel() == k.size(0));
        const int dtype = dtype_of(k);
        const int32_t *sl = i32(slots);
        void *s = stream_of(k);
        const void *kp = k.data_ptr(), *vp = v.data_ptr();
        const int n = (int)k.size(0);
        return unlocked([&] { return f_store_kv(dtype, &c, kp, vp, sl, n, s); });
    });
}

// (y, x, cos, sin, positions)
PyObject *py_rope(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 5, [&]() -> long {
        const at::Tensor &y = dev(a[0]), &x = dev(a[1]), &c = dev(a[2]), &s = dev(a[3]), &pos = dev(a[4]);
        const auto T = x.scalar_type();
        require(x.dim() == 3 && y.sizes() == x.sizes() && y.scalar_type() == T && c.scalar_type() == T && s.scalar_type() == T);
        require(c.dim() == 2 && c.sizes() == s.sizes() && c.size(1) == x.size(2) && pos.numel() == x.size(0));
        const int dtype = dtype_of(x);
        const int32_t *p = i32(pos);
        void *st = stream_of(x), *yp = y.data_ptr();
        const void *xp = x.data_ptr(), *cp = c.data_ptr(), *sp = s.data_ptr();
        const int len = (int)c.size(0), n = (int)x.size(0), H = (int)x.size(1), D = (int)x.size(2);
        return unlocked([&] { return f_rope(dtype, yp, xp, cp, sp, len, p, n, H, D, st); });
    });
}

// (y, x, w, eps)
PyObject *py_rmsnorm(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 4, [&]() -> long {
        const at::Tensor &y = dev(a[0]), &x = dev(a[1]), &w = dev(a[2]);
        require(x.dim() >= 1 && y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type() && w.scalar_type() == x.scalar_type());
        const int64_t H = x.size(-1);
        require(H > 0 && w.dim() == 1 && w.size(0) == H);
        const int dtype = dtype_of(x);
        const float eps = number(a[3]);
        void *s = stream_of(x), *yp = y.data_ptr();
        const void *xp = x.data_ptr(), *wp = w.data_ptr();
        const int rows = (int)(x.numel() / H);
        return unlocked([&] { return f_rmsnorm(dtype, yp, xp, wp, rows, (int)H, eps, s); });
    });
}

// (bounds, k_pages, v_pages, block_tables, positions, query_start_loc, max_query_len)
PyObject *py_bounds(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 7, [&]() -> long {
        const at::Tensor &pos = dev(a[4]);
        const OneGpu gpu(pos);
        const Bounds b(a[0], gpu);
        const bool dense = THPVariable_CheckExact(a[1]);
        const at::ScalarType like = dense ? THPVariable_Unpack(a[1]).scalar_type() : at::kBFloat16;
        const ti_kv_cache c = gpu.cache(a[1], a[2], like);
        require(b.pages == c.num_pages && b.heads == c.kv_heads && b.page == c.page_size && b.D == c.head_dim);
        const int dtype = dense ? dtype_of(THPVariable_Unpack(a[1])) : TI_BF16;
        const StepArgs t(gpu, a[3], a[4], a[5], a[6]);
        void *s = stream_of(pos);
        return unlocked([&] { return f_bounds(dtype, &c, &b.ptr, t.tables, t.stride, t.positions, t.qsl, t.seqs, t.n, t.total, s); });
    });
}

// (tables, lengths, workspace, q, bounds, block_tables, positions, sinks, window, causal, query_start_loc, max_query_len)
PyObject *py_select(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 12, [&]() -> long {
        const at::Tensor &q = dev(a[3]);
        const OneGpu gpu(q);
        const at::Tensor &tables = gpu(a[0]), &lengths = gpu(a[1]), &ws = gpu(a[2]);
        const Bounds b(a[4], gpu);
        const StepArgs t(gpu, a[5], a[6], a[10], a[11]);
        require(q.dim() == 3 && q.size(2) == b.D && t.total == q.size(0) && PyBool_Check(a[9]));
        require(tables.dim() == 3 && tables.size(0) == q.size(0) && tables.size(1) == b.heads);
        require(lengths.dim() == 2 && lengths.size(0) == q.size(0) && lengths.size(1) == b.heads);
        ti_select_args g{};
        g.dtype = dtype_of(q);
        g.q_heads = (int32_t)q.size(1), g.kv_heads = (int32_t)b.heads, g.head_dim = (int32_t)b.D;
        g.page_size = (int32_t)b.page, g.num_pages = (int32_t)b.pages;
        g.num_seqs = t.seqs, g.max_query_len = t.n, g.total_tokens = t.total, g.block_table_stride = t.stride;
        g.keep = (int32_t)tables.size(2), g.sinks = (int32_t)integer(a[7]), g.window = (int32_t)integer(a[8]), g.causal = a[9] == Py_True;
        g.q = q.data_ptr(), g.bounds = b.ptr;
        g.positions = t.positions, g.query_start_loc = t.qsl, g.block_tables = t.tables;
        g.tables = const_cast<int32_t *>(i32(tables)), g.lengths = const_cast<int32_t *>(i32(lengths));
        g.workspace = ws.data_ptr(), g.workspace_bytes = (size_t)ws.nbytes();
        void *s = stream_of(q);
        return unlocked([&] { return f_select(&g, s); });
    });
}

// (out, workspace, q, k_pages, v_pages, tables, lengths, scale, query_start_loc, max_query_len)
PyObject *py_sparse(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 10, [&]() -> long {
        const at::Tensor &q = dev(a[2]);
        const OneGpu gpu(q);
        const at::Tensor &out = gpu(a[0]), *ws = gpu.or_none(a[1]), &tables = gpu(a[5]), &lengths = gpu(a[6]), *qsl = gpu.or_none(a[8]);
        require(q.dim() == 3 && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type());
        const ti_kv_cache c = gpu.cache(a[3], a[4], q.scalar_type());
        require(q.size(2) == c.head_dim && (!qsl || a[9] != Py_None));
        require(tables.dim() == 3 && tables.size(0) == q.size(0) && tables.size(1) == c.kv_heads);
        require(lengths.dim() == 2 && lengths.size(0) == q.size(0) && lengths.size(1) == c.kv_heads);
        ti_sparse_attention_args g{};
        g.dtype = dtype_of(q);
        g.max_query_len = a[9] == Py_None ? 1 : (int32_t)integer(a[9]);
        require(g.max_query_len > 0 && (qsl || q.size(0) % g.max_query_len == 0));
        g.num_seqs = (int32_t)(qsl ? qsl->numel() - 1 : q.size(0) / g.max_query_len);
        g.q_heads = (int32_t)q.size(1), g.total_tokens = (int32_t)q.size(0), g.table_width = (int32_t)tables.size(2);
        g.q = q.data_ptr(), g.out = out.data_ptr();
        g.tables = i32(tables), g.lengths = i32(lengths), g.query_start_loc = qsl ? i32(*qsl) : nullptr;
        g.scale = number(a[7]);
        g.workspace = ws ? ws->data_ptr() : nullptr, g.workspace_bytes = ws ? (size_t)ws->nbytes() : 0;
        void *s = stream_of(q);
        return unlocked([&] { return f_sparse(&g, &c, s); });
    });
}

// (accepted, tokens, workspace, draft_tokens, target, draft, uniforms, draft_lens)
PyObject *py_verify(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 8, [&]() -> long {
        const at::Tensor &p = dev(a[4]);
        const OneGpu gpu(p);
        const at::Tensor &acc = gpu(a[0]), &tok = gpu(a[1]), &ws = gpu(a[2]), &x = gpu(a[3]), *q = gpu.or_none(a[5]), &u = gpu(a[6]),
                         *n = gpu.or_none(a[7]);
        require(p.dim() == 3 && p.size(1) > 0);
        const int64_t B = p.size(0), N = p.size(1) - 1, V = p.size(2);
        require(x.dim() == 2 && x.size(0) == B && x.size(1) == N && tok.dim() == 2 && tok.size(0) == B && tok.size(1) == N + 1);
        require(acc.dim() == 1 && acc.size(0) == B && u.dim() == 2 && u.size(0) == B && u.size(1) == N + 1 && u.scalar_type() == at::kFloat);
        require(!q || (q->dim() == 3 && q->size(0) == B && q->size(1) == N && q->size(2) == V && q->scalar_type() == p.scalar_type()));
        require(!n || (n->dim() == 1 && n->size(0) == B));
        ti_verify_args g{};
        g.dtype = dtype_of(p);
        g.num_seqs = (int32_t)B, g.max_drafts = (int32_t)N, g.vocab = (int32_t)V;
        g.draft_tokens = i32(x), g.draft_lens = n ? i32(*n) : nullptr;
        g.target = p.data_ptr(), g.draft = q ? q->data_ptr() : nullptr;
        g.uniforms = static_cast<const float *>(u.data_ptr());
        g.accepted = const_cast<int32_t *>(i32(acc)), g.tokens = const_cast<int32_t *>(i32(tok));
        g.workspace = ws.data_ptr(), g.workspace_bytes = (size_t)ws.nbytes();
        void *s = stream_of(p);
        return unlocked([&] { return f_verify(&g, s); });
    });
}

// (out, workspace, q, k_pages, v_pages, block_tables, positions, scale, window, sinks, query_start_loc, max_query_len)
PyObject *py_window(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 12, [&]() -> long {
        const at::Tensor &q = dev(a[2]);
        const OneGpu gpu(q);
        const at::Tensor &out = gpu(a[0]), *ws = gpu.or_none(a[1]);
        require(q.dim() == 3 && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type());
        const ti_kv_cache c = gpu.cache(a[3], a[4], q.scalar_type());
        const StepArgs t(gpu, a[5], a[6], a[10], a[11]);
        require(t.total == q.size(0) && q.size(2) == c.head_dim);
        ti_attention_args g{};
        g.dtype = dtype_of(q);
        g.q_heads = (int32_t)q.size(1);
        g.num_seqs = t.seqs, g.max_query_len = t.n, g.total_tokens = t.total, g.block_table_stride = t.stride;
        g.q = q.data_ptr(), g.out = out.data_ptr();
        g.positions = t.positions, g.query_start_loc = t.qsl, g.block_tables = t.tables;
        g.scale = number(a[7]);
        g.causal = 1;
        g.workspace = ws ? ws->data_ptr() : nullptr, g.workspace_bytes = ws ? (size_t)ws->nbytes() : 0;
        const long window = integer(a[8]), sinks = integer(a[9]);
        require(window >= 1 && window <= 0x7fffffff && sinks >= 0 && sinks <= 0x7fffffff);
        void *s = stream_of(q);
        return unlocked([&] { return f_window(&g, (int)window, (int)sinks, &c, s); });
    });
}

// A PagePool's arrays, and its GPU.
struct Pool {
    Attr free, count, tables, lengths, behind, ticket;
    OneGpu gpu;
    ti_page_pool p{};
    Pool(PyObject *o)
        : free((require((PyObject *)Py_TYPE(o) == page_pool), o), n_free), count(o, n_free_count), tables(o, n_tables),
          lengths(o, n_lengths), behind(o, n_behind), ticket(o, n_ticket), gpu(dev(free.o)) {
        const Attr size(o, n_page_size), window(o, n_window), sinks(o, n_sinks);
        const at::Tensor &t = gpu(tables.o), &f = gpu(free.o), *b = gpu.or_none(behind.o);
        require(t.dim() == 2 && f.numel() <= 0x7fffffff);
        const int64_t S = t.size(0);
        require(gpu(lengths.o).numel() == S && gpu(count.o).numel() == 1 && gpu(ticket.o).numel() == 1 && (!b || b->numel() == S));
        p.num_pages = (int32_t)f.numel(), p.page_size = (int32_t)integer(size.o), p.num_seqs = (int32_t)S, p.table_width = (int32_t)t.size(1);
        p.window = (int32_t)integer(window.o), p.sinks = (int32_t)integer(sinks.o);
        p.free = out(free.o), p.free_count = out(count.o), p.tables = out(tables.o), p.lengths = out(lengths.o);
        p.behind = b ? out(behind.o) : nullptr, p.ticket = out(ticket.o);
    }
    int32_t *out(PyObject *o) const { return const_cast<int32_t *>(i32(gpu(o))); }
};

// (pool, counts, positions, slots, query_start_loc, short)
PyObject *py_reserve(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 6, [&]() -> long {
        const Pool pool(a[0]);
        const at::Tensor &counts = pool.gpu(a[1]), &pos = pool.gpu(a[2]), &slots = pool.gpu(a[3]);
        const int64_t S = pool.p.num_seqs, T = pos.numel();
        require(counts.dim() == 1 && counts.numel() == S && pos.dim() == 1 && slots.dim() == 1 && slots.numel() == T && T <= 0x7fffffff);
        require(pool.gpu(a[4]).dim() == 1 && pool.gpu(a[4]).numel() == S + 1 && pool.gpu(a[5]).numel() == 1);
        const int32_t *n = i32(counts);
        int32_t *x = pool.out(a[2]), *y = pool.out(a[3]), *z = pool.out(a[4]), *w = pool.out(a[5]);
        void *s = stream_of(counts);
        return unlocked([&] { return f_reserve(&pool.p, n, (int)T, x, y, z, w, s); });
    });
}

// (pool, lengths)
PyObject *py_release(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded(nargs, 2, [&]() -> long {
        const Pool pool(a[0]);
        const at::Tensor &keep = pool.gpu(a[1]);
        require(keep.dim() == 1 && keep.numel() == pool.p.num_seqs);
        const int32_t *n = i32(keep);
        void *s = stream_of(keep);
        return unlocked([&] { return f_release(&pool.p, n, s); });
    });
}

void hold(PyObject *&to, PyObject *o) {
    Py_INCREF(o);
    Py_XDECREF(to);
    to = o;
}

// bind(Int8Pages, KeyBounds, Fp8Pages, PagePool, addresses of ti_attention, ti_attention_inputs, ti_store_kv, ti_rope,
//      ti_rmsnorm, ti_update_key_bounds, ti_select_pages, ti_sparse_attention, ti_verify_draft, ti_window_attention,
//      ti_reserve_pages, ti_release_pages)
PyObject *py_bind(PyObject *, PyObject *args) {
    PyObject *pages, *bounds, *fp8, *pool;
    unsigned long long f[12];
    if (!PyArg_ParseTuple(args, "OOOOKKKKKKKKKKKK", &pages, &bounds, &fp8, &pool, &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6], &f[7],
                          &f[8], &f[9], &f[10], &f[11]))
        return nullptr;
    hold(int8_pages, pages);
    hold(key_bounds, bounds);
    hold(fp8_pages, fp8);
    hold(page_pool, pool);
    f_window = reinterpret_cast<decltype(f_window)>(f[9]);
    f_reserve = reinterpret_cast<decltype(f_reserve)>(f[10]);
    f_release = reinterpret_cast<decltype(f_release)>(f[11]);
    f_bounds = reinterpret_cast<decltype(f_bounds)>(f[5]);
    f_select = reinterpret_cast<decltype(f_select)>(f[6]);
    f_sparse = reinterpret_cast<decltype(f_sparse)>(f[7]);
    f_verify = reinterpret_cast<decltype(f_verify)>(f[8]);
    f_attention = reinterpret_cast<decltype(f_attention)>(f[0]);
    f_inputs = reinterpret_cast<decltype(f_inputs)>(f[1]);
    f_store_kv = reinterpret_cast<decltype(f_store_kv)>(f[2]);
    f_rope = reinterpret_cast<decltype(f_rope)>(f[3]);
    f_rmsnorm = reinterpret_cast<decltype(f_rmsnorm)>(f[4]);
    Py_RETURN_NONE;
}

#define FAST(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST("attention", py_attention), FAST("attention_inputs", py_inputs), FAST("store_kv", py_store_kv),
                         FAST("rope", py_rope), FAST("rmsnorm", py_rmsnorm), FAST("update_key_bounds", py_bounds),
                         FAST("select_pages", py_select), FAST("sparse_attention", py_sparse), FAST("verify_draft", py_verify),
                         FAST("window_attention", py_window), FAST("reserve_pages", py_reserve), FAST("release_pages", py_release),
                         {"bind", py_bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
    n_layer_q = PyUnicode_InternFromString("layer_q");
    n_layer_scale = PyUnicode_InternFromString("layer_scale");
    n_smooth = PyUnicode_InternFromString("smooth");
    n_half = PyUnicode_InternFromString("half");
    n_cos_sin = PyUnicode_InternFromString("cos_sin");
    n_bounds = PyUnicode_InternFromString("bounds");
    n_scale = PyUnicode_InternFromString("scale");
    n_channel = PyUnicode_InternFromString("channel");
    n_page_size = PyUnicode_InternFromString("page_size");
    n_free = PyUnicode_InternFromString("free");
    n_free_count = PyUnicode_InternFromString("free_count");
    n_tables = PyUnicode_InternFromString("tables");
    n_lengths = PyUnicode_InternFromString("lengths");
    n_behind = PyUnicode_InternFromString("behind");
    n_ticket = PyUnicode_InternFromString("ticket");
    n_window = PyUnicode_InternFromString("window");
    n_sinks = PyUnicode_InternFromString("sinks");
    PyObject *m = PyModule_Create(&module);
    // the torch and Python whose layouts this was compiled for; _lib.py compares
    if (m && PyModule_AddStringConstant(m, "built_for", BUILT_FOR) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}

// host.cpp - the Python entry points' way to the C ABI in native code
// (_sqahost.so). A decode step's node took 12 us of host time per call in Python
// (a ctypes descriptor per tensor at 1.5 to 2.2 us each, the ctypes call and the
// stream lookup), more than its kernels take on the GPU at short contexts; the
// same call takes about 1 us here beside its launches.
//
// Each function takes the tensors of one entry point, with the output and the
// workspace given, and the current stream. It checks what the Python wrapper
// checks and returns the library's status; anything it does not take as it is (a
// tensor subclass, another rank or type, a stream argument, an int that is not
// an int) it answers with None before any work, and the wrapper takes its general
// path, which raises what it always raised. Nothing is kept between calls.
#include <Python.h>

#include <cmath>
#include <initializer_list>

#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/sqattn.h"
#include "call.hpp"

namespace {

using sqa_py::answer;
using sqa_py::General;
using sqa_py::without_gil;

const at::Tensor &tensor(PyObject *o) {
    if (!THPVariable_CheckExact(o)) throw General();
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject *o) {
    if (!PyLong_CheckExact(o)) throw General();
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &over);
    if (over) throw General();
    return v;
}

double real(PyObject *o);

// the softmax scale, or head dim ** -0.5 for None
float scale_of(PyObject *o, const at::Tensor &q) {
    return (float)(o == Py_None ? std::pow((double)q.size(2), -0.5) : real(o));
}

double real(PyObject *o) {
    if (!PyFloat_CheckExact(o)) throw General();
    return PyFloat_AS_DOUBLE(o);
}

void need(bool ok) {
    if (!ok) throw General();
}

sqa_tensor make(int type, const at::Tensor &t, int64_t ne0, int64_t ne1, int64_t ne2, int64_t nb0, int64_t nb1,
                int64_t nb2, int64_t nb3) {
    sqa_tensor d{};
    d.type = type;
    d.ne[0] = ne0, d.ne[1] = ne1, d.ne[2] = ne2, d.ne[3] = 1;
    d.nb[0] = (uint64_t)nb0, d.nb[1] = (uint64_t)nb1, d.nb[2] = (uint64_t)nb2, d.nb[3] = (uint64_t)nb3;
    d.data = t.data_ptr();
    return d;
}

// (n0, n1) rows of 4-byte values, the row stride as it is
sqa_tensor rows2(const at::Tensor &t, int64_t n0, int64_t n1) {
    const int64_t s = t.stride(0) * 4;
    return make(SQA_TYPE_F32, t, n0, n1, 1, 4, s, s * n1, s * n1);
}

sqa_tensor cache_rows(const at::Tensor &c, int64_t ne0) {
    need(c.dim() >= 1 && c.size(0) > 0);
    const int64_t rows = c.size(0), rb = c.numel() / rows;
    need(rb == ne0 / SQA_QK4_0 * SQA_Q4_0_BLOCK_BYTES);
    return make(SQA_TYPE_Q4_0, c, ne0, rows, 1, SQA_Q4_0_BLOCK_BYTES, rb, rb * rows, rb * rows);
}

sqa_tensor index(const at::Tensor &t, int type, int64_t nb0) {
    need(t.dim() >= 1);
    const int64_t n = t.size(0);
    return make(type, t, n, 1, 1, nb0, nb0 * n, nb0 * n, nb0 * n);
}

sqa_tensor q_view(const at::Tensor &q) {  // (n_q, H, D) -> [D, n_q, H]
    need(q.dim() == 3);
    return make(SQA_TYPE_F32, q, q.size(2), q.size(0), q.size(1), 4, q.stride(0) * 4, q.stride(1) * 4,
                q.stride(1) * 4 * q.size(1));
}

sqa_tensor cache_view(const at::Tensor &c, int64_t n_kv) {  // (rows, Hkv, bytes) -> [D, n_kv, Hkv]
    need(c.dim() == 3 && c.scalar_type() == at::kByte && c.is_contiguous() && n_kv <= c.size(0));
    const int64_t Hkv = c.size(1), rb = c.size(2);
    return make(SQA_TYPE_Q4_0, c, rb / SQA_Q4_0_BLOCK_BYTES * SQA_QK4_0, n_kv, Hkv, SQA_Q4_0_BLOCK_BYTES, Hkv * rb, rb,
                rb * Hkv);
}

sqa_tensor out_view(const at::Tensor &o) {  // (n_q, H, D) -> [D, H, n_q]
    need(o.dim() == 3 && o.is_contiguous());
    const int64_t n_q = o.size(0), H = o.size(1), D = o.size(2);
    return make(SQA_TYPE_F32, o, D, H, n_q, 4, D * 4, H * D * 4, H * D * 4 * n_q);
}

sqa_tensor mask_view(const at::Tensor &m) {
    need(m.dim() == 2 && m.scalar_type() == at::kHalf && m.stride(1) == 1);
    const int64_t s = m.stride(0) * 2;
    return make(SQA_TYPE_F16, m, m.size(1), m.size(0), 1, 2, s, s * m.size(0), s * m.size(0));
}

void *stream() { return c10::hip::getCurrentHIPStream().stream(); }

// q, k_cache, v_cache, n_kv, mask, scale, max_bias, softcap, out, workspace
PyObject *fa(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 10);
        const at::Tensor &q = tensor(a[0]), &ws = tensor(a[9]);
        const int64_t n_kv = integer(a[3]);
        const sqa_tensor tq = q_view(q), tk = cache_view(tensor(a[1]), n_kv), tv = cache_view(tensor(a[2]), n_kv),
                         to = out_view(tensor(a[8]));
        sqa_tensor tm;
        const bool mask = a[4] != Py_None;
        if (mask) tm = mask_view(tensor(a[4]));
        const float scale = scale_of(a[5], q), bias = (float)real(a[6]), cap = (float)real(a[7]);
        void *wp = ws.data_ptr(), *st = stream();
        const size_t wb = (size_t)ws.numel();
        return without_gil([&] {
            return sqa_flash_attn_ext(&tq, &tk, &tv, mask ? &tm : nullptr, scale, bias, cap, &to, wp, wb, st);
        });
    });
}

// q, k_cache, v_cache, n_kv, q_pos0, gate, scale, out, workspace
PyObject *fa_causal(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 9);
        const at::Tensor &q = tensor(a[0]), &ws = tensor(a[8]);
        const int64_t n_kv = integer(a[3]), pos0 = integer(a[4]);
        const sqa_tensor tq = q_view(q), tk = cache_view(tensor(a[1]), n_kv), tv = cache_view(tensor(a[2]), n_kv),
                         to = out_view(tensor(a[7]));
        sqa_tensor tg;
        const bool gate = a[5] != Py_None;
        if (gate) {
            const at::Tensor &t = tensor(a[5]);
            need(t.dim() >= 2);
            tg = make(SQA_TYPE_F32, t, q.size(2), q.size(1), q.size(0), 4, t.stride(1) * 4, t.stride(0) * 4,
                      t.stride(0) * 4 * q.size(0));
        }
        const float scale = scale_of(a[6], q);
        void *wp = ws.data_ptr(), *st = stream();
        const size_t wb = (size_t)ws.numel();
        return without_gil([&] {
            return sqa_flash_attn_ext_causal(&tq, &tk, &tv, pos0, gate ? &tg : nullptr, scale, &to, wp, wb, st);
        });
    });
}

// mask, step_start
PyObject *fill_mask(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 2);
        const sqa_tensor tm = mask_view(tensor(a[0]));
        const int64_t start = integer(a[1]);
        void *st = stream();
        return without_gil([&] { return sqa_fill_causal_mask(&tm, start, st); });
    });
}

// cache, src, idx
PyObject *set_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 3);
        const at::Tensor &src = tensor(a[1]), &idx = tensor(a[2]);
        need(src.dim() == 2 && idx.dim() >= 1);
        const int64_t ne0 = src.size(1);
        const sqa_tensor td = cache_rows(tensor(a[0]), ne0), ts = rows2(src, ne0, src.size(0)),
                         ti = index(idx, SQA_TYPE_I64, idx.stride(0) * 8);
        void *st = stream();
        return without_gil([&] { return sqa_set_rows_q4_0(&td, &ts, &ti, st); });
    });
}

// every tensor of a call on the current device (the general path switches to theirs)
void here(std::initializer_list<PyObject *> ts) {
    const int dev = (int)c10::hip::current_device();
    for (PyObject *o : ts) {
        if (o == Py_None) continue;
        const at::Tensor &t = tensor(o);
        need(t.is_cuda() && t.get_device() == dev);
    }
}

// (n,) row indices
sqa_tensor places(const at::Tensor &t) {
    need(t.dim() == 1 && t.scalar_type() == at::kLong);
    return index(t, SQA_TYPE_I64, t.stride(0) * 8);
}

// cache, idx, out
PyObject *get_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 3);
        here({a[0], a[1], a[2]});
        const at::Tensor &c = tensor(a[0]), &o = tensor(a[2]);
        need(c.dim() >= 2 && c.scalar_type() == at::kByte && c.is_contiguous() && o.dim() == 2 &&
             (o.scalar_type() == at::kFloat || o.scalar_type() == at::kHalf) && (o.size(1) <= 1 || o.stride(1) == 1));
        const int64_t ne0 = o.size(1), e = (int64_t)o.element_size(), s = o.stride(0) * e;
        const sqa_tensor ts = cache_rows(c, ne0), ti = places(tensor(a[1])),
                         to = make(e == 4 ? SQA_TYPE_F32 : SQA_TYPE_F16, o, ne0, o.size(0), 1, e, s, s * o.size(0), s * o.size(0));
        void *st = stream();
        return without_gil([&] { return sqa_get_rows_q4_0(&to, &ts, &ti, st); });
    });
}

// dst, src, to, from, delta, rope (both or neither None)
PyObject *move_rows(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Py_buffer view{};
    PyObject *r = answer([&]() -> int {
        need(n == 6);
        here({a[0], a[1], a[2], a[3], a[4]});
        auto heads = [](const at::Tensor &t) {
            need(t.dim() == 3 && t.scalar_type() == at::kByte && t.is_contiguous() && t.size(2) % SQA_Q4_0_BLOCK_BYTES == 0);
            const int64_t rb = t.size(2), row = rb * t.size(1);
            return make(SQA_TYPE_Q4_0, t, rb / SQA_Q4_0_BLOCK_BYTES * SQA_QK4_0, t.size(1), t.size(0), SQA_Q4_0_BLOCK_BYTES, rb,
                        row, row * t.size(0));
        };
        const sqa_tensor td = heads(tensor(a[0])), ts = heads(tensor(a[1])), tt = places(tensor(a[2])), tf = places(tensor(a[3]));
        sqa_tensor tl;
        const bool turn = a[4] != Py_None;
        need(turn == (a[5] != Py_None));
        if (turn) {
            const at::Tensor &d = tensor(a[4]);
            need(d.dim() == 1 && d.scalar_type() == at::kInt && d.is_contiguous());
            tl = index(d, SQA_TYPE_I32, 4);
            need(PyObject_GetBuffer(a[5], &view, PyBUF_SIMPLE) == 0 && view.len == (Py_ssize_t)sizeof(sqa_rope));
        }
        const sqa_rope *rope = turn ? (const sqa_rope *)view.buf : nullptr;
        void *st = stream();
        return without_gil([&] { return sqa_move_rows_q4_0(&td, &ts, &tt, &tf, turn ? &tl : nullptr, rope, st); });
    });
    if (view.obj) PyBuffer_Release(&view);
    return r;
}

// cache or out, src, norm_w, eps, pos, rope, idx (None: F32 output)
PyObject *rope_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Py_buffer view{};
    PyObject *r = answer([&]() -> int {
        need(n == 7);
        const at::Tensor &dst = tensor(a[0]), &src = tensor(a[1]), &pos = tensor(a[4]);
        need(src.dim() == 3);
        const int64_t n_tok = src.size(0), n_head = src.size(1), D = src.size(2);
        const sqa_tensor ts = make(SQA_TYPE_F32, src, D, n_head, n_tok, 4, src.stride(1) * 4, src.stride(0) * 4,
                                   src.stride(0) * 4 * n_tok),
                         tp = index(pos, SQA_TYPE_I32, 4);
        sqa_tensor tw;
        const bool norm = a[2] != Py_None;
        if (norm) tw = make(SQA_TYPE_F32, tensor(a[2]), D, 1, 1, 4, 4 * D, 4 * D, 4 * D);
        const float eps = (float)real(a[3]);
        need(PyObject_GetBuffer(a[5], &view, PyBUF_SIMPLE) == 0 && view.len == (Py_ssize_t)sizeof(sqa_rope));
        const sqa_rope *rope = (const sqa_rope *)view.buf;
        void *st = stream();
        if (a[6] == Py_None) {
            const sqa_tensor to = make(SQA_TYPE_F32, dst, D, n_head, n_tok, 4, D * 4, n_head * D * 4, n_head * D * 4 * n_tok);
            return without_gil([&] { return sqa_rope_norm_f32(&to, &ts, norm ? &tw : nullptr, eps, &tp, rope, st); });
        }
        const at::Tensor &idx = tensor(a[6]);
        need(idx.dim() >= 1);
        const sqa_tensor td = cache_rows(dst, n_head * D), ti = index(idx, SQA_TYPE_I64, idx.stride(0) * 8);
        return without_gil([&] {
            return sqa_rope_norm_set_rows_q4_0(&td, &ts, norm ? &tw : nullptr, eps, &tp, rope, &ti, st);
        });
    });
    if (view.obj) PyBuffer_Release(&view);
    return r;
}

// w, x, gate, out, workspace
PyObject *out_proj(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 5);
        const at::Tensor &w = tensor(a[0]), &x = tensor(a[1]), &o = tensor(a[3]), &ws = tensor(a[4]);
        need(x.dim() == 2 && w.dim() >= 1 && o.dim() >= 1);
        const int64_t M = x.size(0), K = x.size(1), N = w.size(0), wn = w.stride(0);
        const sqa_tensor tw = make(SQA_TYPE_Q4_K, w, K, N, 1, 144, wn, wn * N, wn * N), tx = rows2(x, K, M),
                         to = rows2(o, N, M);
        sqa_tensor tg;
        const bool gate = a[2] != Py_None;
        if (gate) {
            need(tensor(a[2]).dim() >= 1);
            tg = rows2(tensor(a[2]), K, M);
        }
        void *wp = ws.data_ptr(), *st = stream();
        const size_t wb = (size_t)ws.numel();
        return without_gil([&] { return sqa_out_proj(&tw, &tx, gate ? &tg : nullptr, &to, wp, wb, st); });
    });
}

// handle, slot, k_cur, v_cur, idx
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 5);
        sqa_kv_cache *kv = (sqa_kv_cache *)(uintptr_t)integer(a[0]);
        const int64_t slot = integer(a[1]);
        need(slot == (int64_t)(int32_t)slot);
        const at::Tensor &k = tensor(a[2]), &v = tensor(a[3]);
        need(k.dim() == 2 && v.dim() >= 1);
        const int64_t n_tok = k.size(0), ne0 = k.size(1);
        const sqa_tensor tk = rows2(k, ne0, n_tok), tv = rows2(v, ne0, n_tok),
                         ti = make(SQA_TYPE_I64, tensor(a[4]), n_tok, 1, 1, 8, 8 * n_tok, 8 * n_tok, 8 * n_tok);
        void *st = stream();
        return without_gil([&] { return sqa_kv_cache_append(kv, (int32_t)slot, &tk, &tv, &ti, st); });
    });
}

// one-dimensional contiguous tensor
sqa_tensor vec(const at::Tensor &t, at::ScalarType dtype, int type) {
    need(t.dim() == 1 && t.scalar_type() == dtype && t.is_contiguous());
    const int64_t n = t.size(0), e = (int64_t)t.element_size();
    return make(type, t, n, 1, 1, e, e * n, e * n, e * n);
}
sqa_tensor ints(const at::Tensor &t) { return vec(t, at::kInt, SQA_TYPE_I32); }

sqa_tensor table_view(const at::Tensor &t) {  // (B, W) -> [W, B]
    need(t.dim() == 2 && t.scalar_type() == at::kInt && (t.size(1) <= 1 || t.stride(1) == 1));
    const int64_t s = t.stride(0) * 4;
    return make(SQA_TYPE_I32, t, t.size(1), t.size(0), 1, 4, s, s * t.size(0), s * t.size(0));
}

sqa_tensor pool_view(const at::Tensor &t) {  // (n_pages, page, Hkv, bytes) -> [D, Hkv, page, n_pages]
    need(t.dim() == 4 && t.scalar_type() == at::kByte);
    const int64_t n = t.size(0), page = t.size(1), Hkv = t.size(2), rb = t.size(3);
    need(n >= 1 && rb % SQA_Q4_0_BLOCK_BYTES == 0 && t.stride(3) == 1 && (Hkv == 1 || t.stride(2) == rb) &&
         (page == 1 || t.stride(1) == Hkv * rb) && (n == 1 || t.stride(0) > 0));
    sqa_tensor d = make(SQA_TYPE_Q4_0, t, rb / SQA_Q4_0_BLOCK_BYTES * SQA_QK4_0, Hkv, page, SQA_Q4_0_BLOCK_BYTES, rb,
                        Hkv * rb, n == 1 ? page * Hkv * rb : t.stride(0));
    d.ne[3] = n;
    return d;
}

// state, ring, table, n_past, n_new, page, then the step: state, n_past, q_start, kv_len, slots, pos
PyObject *plan(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 12);
        here({a[0], a[1], a[2], a[3], a[4], a[6], a[7], a[8], a[9], a[10], a[11]});
        const sqa_tensor st = ints(tensor(a[0])), ring = ints(tensor(a[1])), tab = table_view(tensor(a[2])),
                         past = ints(tensor(a[3])), fresh = ints(tensor(a[4])), so = ints(tensor(a[6])),
                         po = ints(tensor(a[7])), qs = ints(tensor(a[8])), kl = ints(tensor(a[9])),
                         sl = vec(tensor(a[10]), at::kLong, SQA_TYPE_I64), pos = ints(tensor(a[11]));
        const int64_t page = integer(a[5]);
        need(page == (int64_t)(int32_t)page);
        void *s = stream();
        return without_gil([&] {
            return sqa_paged_plan(&past, &fresh, &tab, &ring, &st, (int32_t)page, &so, &po, &qs, &kl, &sl, &pos, s);
        });
    });
}

// q_start, kv_len, group, shared_len, members, m_start, m_pos, token_group, pos
PyObject *share(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 9);
        here({a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8]});
        sqa_tensor t[9];
        for (int i = 0; i < 8; ++i) t[i] = ints(tensor(a[i]));
        const bool pos = a[8] != Py_None;
        if (pos) t[8] = ints(tensor(a[8]));
        void *s = stream();
        return without_gil([&] {
            return sqa_paged_share(&t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6], &t[7], pos ? &t[8] : nullptr, s);
        });
    });
}

sqa_tensor gate_view(const at::Tensor &t, const at::Tensor &q) {
    need(t.dim() == 3 && t.scalar_type() == at::kFloat && t.sizes() == q.sizes() && (t.size(2) <= 1 || t.stride(2) == 1));
    return make(SQA_TYPE_F32, t, q.size(2), q.size(1), q.size(0), 4, t.stride(1) * 4, t.stride(0) * 4, t.stride(0) * 4 * q.size(0));
}

// q, k_pool, v_pool, table, q_start, kv_len, prefix, shared_table, shared_len, members, m_start, m_pos, token_group,
// max_q, scale, max_bias, softcap, gate, out, workspace
PyObject *attn_shared(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 20);
        here({a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12], a[17], a[18], a[19]});
        const at::Tensor &q = tensor(a[0]), &o = tensor(a[18]), &ws = tensor(a[19]);
        need(q.dim() == 3 && q.scalar_type() == at::kFloat && o.scalar_type() == at::kFloat && ws.is_contiguous() &&
             (q.size(2) <= 1 || q.stride(2) == 1));
        const sqa_tensor tq = q_view(q), tk = pool_view(tensor(a[1])), tv = pool_view(tensor(a[2])),
                         tt = table_view(tensor(a[3])), ts = ints(tensor(a[4])), tl = ints(tensor(a[5])),
                         st = table_view(tensor(a[7])), sl = ints(tensor(a[8])), me = ints(tensor(a[9])),
                         ms = ints(tensor(a[10])), mp = ints(tensor(a[11])), tr = ints(tensor(a[12])), to = out_view(o);
        sqa_tensor tp, tg;
        const bool prefix = a[6] != Py_None, gate = a[17] != Py_None;
        if (prefix) tp = ints(tensor(a[6]));
        if (gate) tg = gate_view(tensor(a[17]), q);
        const int64_t max_q = integer(a[13]);
        const float scale = scale_of(a[14], q), bias = (float)real(a[15]), cap = (float)real(a[16]);
        void *wp = ws.data_ptr(), *s = stream();
        const size_t wb = (size_t)ws.nbytes();
        return without_gil([&] {
            return sqa_paged_attn_shared(&tq, &tk, &tv, &tt, &ts, &tl, prefix ? &tp : nullptr, &st, &sl, &me, &ms, &mp, &tr,
                                         max_q, scale, bias, cap, gate ? &tg : nullptr, &to, wp, wb, s);
        });
    });
}

// q, k_pool, v_pool, table, q_start, kv_len, prefix, max_q, scale, max_bias, softcap, gate, out, workspace
PyObject *paged_attn(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 14);
        here({a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[11], a[12], a[13]});
        const at::Tensor &q = tensor(a[0]), &o = tensor(a[12]), &ws = tensor(a[13]);
        need(q.dim() == 3 && q.scalar_type() == at::kFloat && o.scalar_type() == at::kFloat && ws.is_contiguous() &&
             (q.size(2) <= 1 || q.stride(2) == 1));
        const sqa_tensor tq = q_view(q), tk = pool_view(tensor(a[1])), tv = pool_view(tensor(a[2])),
                         tt = table_view(tensor(a[3])), ts = ints(tensor(a[4])), tl = ints(tensor(a[5])), to = out_view(o);
        sqa_tensor tp, tg;
        const bool prefix = a[6] != Py_None, gate = a[11] != Py_None;
        if (prefix) tp = ints(tensor(a[6]));
        if (gate) tg = gate_view(tensor(a[11]), q);
        const int64_t max_q = integer(a[7]);
        const float scale = scale_of(a[8], q), bias = (float)real(a[9]), cap = (float)real(a[10]);
        void *wp = ws.data_ptr(), *st = stream();
        const size_t wb = (size_t)ws.nbytes();
        return without_gil([&] {
            return sqa_paged_attn(&tq, &tk, &tv, &tt, &ts, &tl, prefix ? &tp : nullptr, max_q, scale, bias, cap,
                                  gate ? &tg : nullptr, &to, wp, wb, st);
        });
    });
}

// base, x, a, b, ids, scale, gate, out
PyObject *lora(PyObject *, PyObject *const *p, Py_ssize_t n) {
    return answer([&]() -> int {
        need(n == 8);
        here({p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]});
        auto rows = [](const at::Tensor &t) {
            need(t.dim() == 2 && t.scalar_type() == at::kFloat && (t.size(1) <= 1 || t.stride(1) == 1));
            return rows2(t, t.size(1), t.size(0));
        };
        auto half3 = [](const at::Tensor &t) {
            need(t.dim() == 3 && t.scalar_type() == at::kHalf && t.is_contiguous());
            const int64_t n0 = t.size(2), n1 = t.size(1), n2 = t.size(0);
            return make(SQA_TYPE_F16, t, n0, n1, n2, 2, 2 * n0, 2 * n0 * n1, 2 * n0 * n1 * n2);
        };
        const sqa_tensor td = rows(tensor(p[0])), tx = rows(tensor(p[1])), ta = half3(tensor(p[2])), tb = half3(tensor(p[3])),
                         ti = ints(tensor(p[4])), to = rows(tensor(p[7]));
        sqa_tensor ts, tg;
        const bool scale = p[5] != Py_None, gate = p[6] != Py_None;
        if (scale) ts = vec(tensor(p[5]), at::kFloat, SQA_TYPE_F32);
        if (gate) tg = rows(tensor(p[6]));
        void *st = stream();
        return without_gil([&] {
            return sqa_lora_add(&td, &tx, gate ? &tg : nullptr, &ta, &tb, &ti, scale ? &ts : nullptr, &to, st);
        });
    });
}

PyMethodDef methods[] = {
#define SQA_FN(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
    SQA_FN(fa),        SQA_FN(fa_causal), SQA_FN(fill_mask), SQA_FN(set_rows),
    SQA_FN(rope_norm), SQA_FN(out_proj),  SQA_FN(append),    SQA_FN(plan),
    SQA_FN(paged_attn), SQA_FN(lora),     SQA_FN(get_rows),  SQA_FN(move_rows),
    SQA_FN(share),     SQA_FN(attn_shared), {nullptr, nullptr, 0, nullptr},
#undef SQA_FN
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_sqahost", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__sqahost() { return PyModule_Create(&module); }

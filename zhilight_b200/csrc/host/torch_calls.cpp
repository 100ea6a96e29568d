// The calls that a program makes once per layer and token, from Python tensors to launches in one step: ops.py's general path costs 10 to 30 us of
// interpreter and ctypes per call, more than many of the kernels behind it.  Host time of a call, us, there / here: one row through a 4096 x 4096
// 4-bit Linear 12.9 / 6.6 (the GPU works 4.7), an int8 Linear 30 / 13, an fp8 one 35 / 18, a bf16 one 16 / 8, an attention step over 32 caches
// 88 / 19, a masked prompt portion 37 / 16.  Each function does what the Python function of its name does, on the same stream and with
// the same entry points of the library, and returns the result, the library's error code as an int, or None for anything out of the ordinary (CPU
// tensors, tensor subclasses, wrapped or strided tensors where plain ones are asked for, active torch modes, memory of other owners):
// ops.py then takes its general path, which serves or refuses it.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../../include/zhilight_b200.h"

namespace {

// Entry points of the loaded library, by address (the library is found and opened by _lib.py)
struct {
    decltype(&zl_w4a16_gemm_fused) w4;
    decltype(&zl_dense_gemm_skinny) dense;
    decltype(&zl_int8_quant_per_token) int8_quant;
    decltype(&zl_fp8_quant_per_tensor) fp8_quant;
    decltype(&zl_w8a8_gemm) w8;
    decltype(&zl_decode_attention_workspace_bytes) attn_bytes;
    decltype(&zl_decode_attention_host) attn;
    decltype(&zl_qkv_axes_rope_append) axes_rope;
    decltype(&zl_paged_attention_workspace_bytes) paged_bytes;
    decltype(&zl_paged_attention) paged;
    decltype(&zl_verify_drafts) verify;
    decltype(&zl_qkv_axes_rope_append_int4) axes_rope4;
    decltype(&zl_int4_cache_values) values4;
    decltype(&zl_paged_attention_int4_workspace_bytes) paged4_bytes;
    decltype(&zl_paged_attention_int4) paged4;
    decltype(&zl_adjust_logits) adjust;
} zl;

struct NotPlain {};   // the general path's

const at::Tensor& plain(PyObject* o, bool contiguous) {
    if (!THPVariable_CheckExact(o)) throw NotPlain{};
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || !t.has_storage() || t.layout() != at::kStrided || t.is_neg() || t.unsafeGetTensorImpl()->is_python_dispatch() ||
        (contiguous && !t.is_contiguous()))
        throw NotPlain{};
    return t;
}
void* optional(PyObject* o, bool contiguous) { return o == Py_None ? nullptr : plain(o, contiguous).data_ptr(); }
int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kHalf: return ZL_F16;
        case at::kBFloat16: return ZL_BF16;
        case at::kFloat: return ZL_F32;
        default: throw NotPlain{};
    }
}
int to_int(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw NotPlain{};
    }
    if (v != (int)v) throw NotPlain{};
    return (int)v;
}
int truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        throw NotPlain{};
    }
    return v;
}
void args(Py_ssize_t n, Py_ssize_t want) {
    if (n != want || c10::impl::dispatch_mode_enabled() || at::impl::torch_function_mode_enabled()) throw NotPlain{};
}
zl_stream_t stream() { return (zl_stream_t)c10::cuda::getCurrentCUDAStream().stream(); }
at::Tensor empty(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type).requires_grad(false)); }

// as ctypes does, the library's calls run without the interpreter's lock
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
int unlocked(F&& f) {
    Unlocked u;
    return f();
}
// pdl of a call: early reads, or a dependent that waits for everything earlier first
int launched(PyObject* pdl) { return truth(pdl) ? 1 : 2; }
PyObject* result(int rc, const at::Tensor& out) { return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out); }

PyObject* pair_of(const at::Tensor& x, const at::Tensor& y) {
    PyObject *first = THPVariable_Wrap(x), *second = THPVariable_Wrap(y), *pair = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return pair;
}

template <typename F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS   // what torch throws here becomes what its own calls raise, torch.OutOfMemoryError for one
    try {
        return f();
    } catch (const NotPlain&) {
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// x, packed, n, k, group_size, bias, residual, epilogue, pdl, out, variant
PyObject* w4a16_gemm_fused(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 11);
        if (!zl.w4) throw NotPlain{};
        const at::Tensor& x = plain(a[0], false);
        if (x.scalar_type() != at::kHalf || x.dim() != 2) throw NotPlain{};
        zl_w4_fused_args_t p = {};
        p.x = x.data_ptr();
        p.M = (int)x.size(0);
        p.ldx = (int)x.stride(0);
        p.packed = plain(a[1], false).data_ptr();
        p.N = to_int(a[2]);
        p.K = to_int(a[3]);
        p.group_size = to_int(a[4]);
        p.bias = optional(a[5], false);
        p.residual = optional(a[6], false);
        p.epilogue = to_int(a[7]);
        p.pdl = launched(a[8]);
        p.variant = to_int(a[10]);
        if (p.epilogue == ZL_EPI_QKV_ROPE || p.N < 0) throw NotPlain{};
        const at::Tensor y = a[9] == Py_None ? empty(x, {x.size(0), p.epilogue == ZL_EPI_SWIGLU ? p.N / 2 : p.N}, at::kHalf) : plain(a[9], false);
        p.y = y.data_ptr();
        const zl_stream_t s = stream();
        return result(unlocked([&] { return zl.w4(&p, s); }), y);
    });
}

// x, w, bias, out_dtype (ZL_F16 ..., or None: x's), pdl
PyObject* dense_gemm_skinny(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 5);
        if (!zl.dense) throw NotPlain{};
        const at::Tensor &x = plain(a[0], true), &w = plain(a[1], true);
        if (x.dim() != 2 || w.dim() < 1) throw NotPlain{};
        void* const bias = optional(a[2], true);
        const int dt = dtype_of(x), od = a[3] == Py_None ? dt : to_int(a[3]), pdl = launched(a[4]);
        if (od != ZL_F16 && od != ZL_BF16 && od != ZL_F32) throw NotPlain{};
        const at::Tensor y = empty(x, {x.size(0), w.size(0)}, od == ZL_F16 ? at::kHalf : od == ZL_BF16 ? at::kBFloat16 : at::kFloat);
        const zl_stream_t s = stream();
        return result(unlocked([&] {
                          return zl.dense(x.data_ptr(), (int)x.stride(0), w.data_ptr(), bias, y.data_ptr(), (int)x.size(0), (int)w.size(0), (int)x.size(1), dt,
                                          od, pdl, s);
                      }),
                      y);
    });
}

// x, w, w_scale, bias, kind (ZL_W8_INT8, ZL_W8_FP8), pdl: quantisation of the rows and the product
PyObject* w8_linear(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 6);
        if (!zl.w8 || !zl.int8_quant || !zl.fp8_quant) throw NotPlain{};
        const at::Tensor &x = plain(a[0], true), &w = plain(a[1], true), &ws = plain(a[2], true);
        if (x.dim() != 2 || w.dim() < 1) throw NotPlain{};
        void* const bias = optional(a[3], true);
        const int kind = to_int(a[4]), pdl = launched(a[5]), dt = dtype_of(x), ws_dt = dtype_of(ws);
        const int64_t m = x.size(0), k = x.size(1), scale_at = (m * k + 15) / 16 * 16;
        const at::Tensor y = empty(x, {m, w.size(0)}, x.scalar_type());
        const at::Tensor room = empty(x, {scale_at + 4 * m}, at::kByte);   // the 8-bit rows, then their scales
        uint8_t* const q = static_cast<uint8_t*>(room.data_ptr());
        float* const scale = reinterpret_cast<float*>(q + scale_at);
        const zl_stream_t s = stream();
        return result(unlocked([&] {
                          const int rc = kind == ZL_W8_INT8 ? zl.int8_quant(x.data_ptr(), (int)x.stride(0), q, scale, (int)m, (int)k, dt, pdl, s)
                                                            : zl.fp8_quant(x.data_ptr(), q, scale, (size_t)(m * k), dt, pdl, s);
                          // the GEMM may start on its weights during the quantisation, which itself is behind everything earlier
                          return rc ? rc
                                    : zl.w8(q, scale, w.data_ptr(), ws.data_ptr(), ws_dt, bias, y.data_ptr(), (int)m, (int)w.size(0), (int)k, kind, dt, 1, s);
                      }),
                      y);
    });
}

// q, buf_lens, k_bufs, v_bufs, mask, scale, max_len_buf, num_kv_heads, bshd, pdl (which changes nothing: the call is behind everything earlier)
PyObject* decode_attention(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 10);
        if (!zl.attn || !zl.attn_bytes) throw NotPlain{};
        const at::Tensor &q = plain(a[0], true), &lens = plain(a[1], true);
        if (q.dim() != 4) throw NotPlain{};
        void* const mask = optional(a[4], true);
        const double scale = PyFloat_AsDouble(a[5]);
        if (scale == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            throw NotPlain{};
        }
        const int max_len = to_int(a[6]), kv_heads = to_int(a[7]), bshd = truth(a[8]), dt = dtype_of(q);
        truth(a[9]);
        const int b = (int)q.size(0), len_q = (int)q.size(1), heads = (int)q.size(2), dim = (int)q.size(3);
        // every tensor whose memory the launches below use; what torch cannot resize belongs to another owner and has to be waited for
        std::vector<const at::Tensor*> used{&q, &lens};
        if (mask) used.push_back(&THPVariable_Unpack(a[4]));
        std::vector<uint64_t> at_;
        for (int i = 2; i < 4; ++i) {
            if (!PyList_CheckExact(a[i]) && !PyTuple_CheckExact(a[i])) throw NotPlain{};
            const Py_ssize_t n = PySequence_Fast_GET_SIZE(a[i]);
            if (n != b) throw NotPlain{};
            for (Py_ssize_t j = 0; j < n; ++j) {
                const at::Tensor& t = plain(PySequence_Fast_GET_ITEM(a[i], j), false);
                used.push_back(&t);
                at_.push_back(reinterpret_cast<uint64_t>(t.data_ptr()));
            }
        }
        for (const at::Tensor* t : used)
            if (!t->storage().resizable()) throw NotPlain{};
        if (b == 0) throw NotPlain{};
        // the caller's lists may change hands once the lock is gone: keep the storages, not the tensors
        std::vector<c10::Storage> storages;
        storages.reserve(used.size());
        for (const at::Tensor* t : used) storages.push_back(t->storage());
        const at::Tensor out = at::empty_like(q);
        const size_t ws_bytes = zl.attn_bytes(b, len_q, heads, dim, max_len), table_at = (ws_bytes + 15) / 16 * 16;
        const at::Tensor room = empty(q, {(int64_t)(table_at + 16 * b)}, at::kByte);   // the kernels' workspace, then the table of addresses
        uint8_t* const ws = static_cast<uint8_t*>(room.data_ptr());
        void* const table = ws + table_at;
        const c10::cuda::CUDAStream cs = c10::cuda::getCurrentCUDAStream();
        const int rc = unlocked([&] {
            return zl.attn(q.data_ptr(), static_cast<const int32_t*>(lens.data_ptr()), at_.data(), table, static_cast<const int8_t*>(mask), (float)scale, max_len,
                           out.data_ptr(), b, len_q, heads, kv_heads, dim, bshd, ws, ws_bytes, dt, (zl_stream_t)cs.stream());
        });
        if (rc == 0)
            for (const c10::Storage& s : storages) c10::cuda::CUDACachingAllocator::recordStream(s.data_ptr(), cs);
        return result(rc, out);
    });
}

// ---- a step of new tokens over a paged cache: what ops.py checks of shapes, types, strides and devices has to hold here, else ops.py refuses it
void must(bool ok) {
    if (!ok) throw NotPlain{};
}
double to_double(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw NotPlain{};
    }
    return v;
}
// a tensor on the current device
const at::Tensor& here(PyObject* o, bool contiguous) {
    const at::Tensor& t = plain(o, contiguous);
    must(t.device().index() == c10::cuda::current_device());
    return t;
}
const int32_t* ints(PyObject* o, int64_t n) {   // (n)
    const at::Tensor& t = here(o, true);
    must(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n);
    return static_cast<const int32_t*>(t.data_ptr());
}
struct Paged {
    void *k, *v;
    const int32_t* table;
    long long pages, step[3];
    int page_size, kv_heads, dim, ld_table, max_pages, seqs;
};
// int4: bytes, 5 dim / 8 a row, whose rows were written from `type`
void caches(Paged& p, const at::Tensor& k, const at::Tensor& v, at::ScalarType type, bool int4) {
    const at::ScalarType held = int4 ? at::kByte : type;
    must(k.dim() == 4 && v.sizes() == k.sizes() && k.scalar_type() == held && v.scalar_type() == held && (type == at::kHalf || type == at::kBFloat16));
    must(k.numel() > 0 && k.size(3) > 1 && k.stride(3) == 1 && v.stride(3) == 1 && (!int4 || k.size(3) == 40 || k.size(3) == 80));
    p.k = k.data_ptr(), p.v = v.data_ptr(), p.pages = k.size(0);
    for (int i = 0; i < 3; ++i) {
        p.step[i] = k.size(i) == 1 ? 0 : k.stride(i);
        must(p.step[i] == (k.size(i) == 1 ? 0 : v.stride(i)) && (p.step[i] > 0 || k.size(i) == 1));
    }
    must(k.size(1) < 1 << 30 && k.size(2) < 1 << 16 && k.size(3) < 1 << 16);
    p.page_size = (int)k.size(1), p.kv_heads = (int)k.size(2), p.dim = (int)(int4 ? k.size(3) / 5 * 8 : k.size(3));
}
Paged paged_cache(PyObject* k_cache, PyObject* v_cache, PyObject* page_table, at::ScalarType type, bool int4) {
    const at::Tensor &k = here(k_cache, false), &v = here(v_cache, false), &t = here(page_table, false);
    must(t.dim() == 2 && t.scalar_type() == at::kInt && t.numel() > 0 && t.stride(1) == 1);
    Paged p = {};
    caches(p, k, v, type, int4);
    must(t.size(0) < 1 << 30 && t.size(1) < 1 << 30 && t.stride(0) < 1ll << 31);
    p.table = static_cast<const int32_t*>(t.data_ptr());
    p.seqs = (int)t.size(0), p.max_pages = (int)t.size(1), p.ld_table = p.seqs > 1 ? (int)t.stride(0) : p.max_pages;
    return p;
}

// qkv, pos, inv_freq, axis, token_seq, placement, page_table, k_cache, v_cache, heads, layout, mscale, pdl
template <bool INT4>
PyObject* axes_rope_append(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 13);
        const auto entry = INT4 ? zl.axes_rope4 : zl.axes_rope;
        must(entry);
        const at::Tensor& x = here(a[0], false);
        const Paged c = paged_cache(a[7], a[8], a[6], x.scalar_type(), INT4);
        const int heads = to_int(a[9]), layout = to_int(a[10]), pdl = truth(a[12]);
        const double mscale = to_double(a[11]);
        must(x.dim() == 2 && heads > 0 && heads < 1 << 16 && x.size(1) == (int64_t)(heads + 2 * c.kv_heads) * c.dim && x.stride(1) == 1);
        const int64_t t = x.size(0);
        must(t > 0 && t < 1ll << 31);
        const at::Tensor &pos = here(a[1], true), &freq = here(a[2], true);
        must(pos.scalar_type() == at::kInt && pos.dim() == 2 && pos.size(0) > 0 && pos.size(0) < 1 << 16 && pos.size(1) == t);
        must(freq.scalar_type() == at::kDouble && freq.dim() == 1 && 2 * freq.size(0) <= c.dim);
        const int32_t *axis = ints(a[3], freq.size(0)), *seq = ints(a[4], t), *place = ints(a[5], t);
        const at::Tensor q = empty(x, {t, (int64_t)heads * c.dim}, x.scalar_type());
        const long long ld = t > 1 ? x.stride(0) : x.size(1);
        const int dt = dtype_of(x);
        const zl_stream_t s = stream();
        return result(unlocked([&] {
                          return entry(x.data_ptr(), ld, static_cast<const int32_t*>(pos.data_ptr()), t, (int)pos.size(0),
                                         static_cast<const double*>(freq.data_ptr()), axis, (int)freq.size(0), layout, (float)mscale, seq, place, c.table,
                                         c.ld_table, c.max_pages, c.seqs, c.k, c.v, c.pages, c.page_size, c.step[0], c.step[1], c.step[2], q.data_ptr(), (int)t,
                                         heads, c.kv_heads, c.dim, dt, pdl, s);
                      }),
                      q);
    });
}

// q, k_cache, v_cache, page_table, seq_lens, q_starts, scale, window, max_new, out, pdl
template <bool INT4>
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 11);
        const auto entry = INT4 ? zl.paged4 : zl.paged;
        const auto room_of = INT4 ? zl.paged4_bytes : zl.paged_bytes;
        must(entry && room_of);
        const at::Tensor& q = here(a[0], true);
        const Paged c = paged_cache(a[1], a[2], a[3], q.scalar_type(), INT4);
        must((q.dim() == 2 || q.dim() == 3) && (q.dim() == 2 || q.size(2) == c.dim));
        const int64_t t = q.size(0), width = q.size(1) * (q.dim() == 3 ? c.dim : 1);
        must(t > 0 && t < 1ll << 31 && width > 0 && width < 1 << 24 && width % ((int64_t)c.kv_heads * c.dim) == 0);
        const int32_t *lens = ints(a[4], c.seqs), *starts = ints(a[5], (int64_t)c.seqs + 1);
        const double scale = to_double(a[6]);
        const int window = to_int(a[7]), most = a[8] == Py_None ? (int)t : to_int(a[8]), pdl = truth(a[10]);
        must(most > 0);
        if (a[9] != Py_None) {
            const at::Tensor& o = here(a[9], true);
            must(o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type());
        }
        const at::Tensor out = a[9] == Py_None ? empty(q, q.sizes(), q.scalar_type()) : THPVariable_Unpack(a[9]);
        const int heads = (int)(width / c.dim), new_ = (int)std::min<int64_t>(most, t);
        const size_t bytes = room_of((int)t, new_, c.seqs, (int)std::min<long long>((long long)c.max_pages * c.page_size, (1ll << 31) - 256), heads, c.kv_heads, c.dim);
        at::Tensor room;
        if (bytes) room = empty(q, {(int64_t)bytes}, at::kByte);
        void* const ws = bytes ? room.data_ptr() : nullptr;
        const int dt = dtype_of(q);
        const zl_stream_t s = stream();
        return result(unlocked([&] {
                          return entry(q.data_ptr(), c.k, c.v, c.pages, c.page_size, c.step[0], c.step[1], c.step[2], c.table, c.ld_table, c.max_pages, lens, starts,
                                       c.seqs, (float)scale, window, out.data_ptr(), (int)t, new_, heads, c.kv_heads, c.dim, ws, bytes, dt, pdl, s);
                      }),
                      out);
    });
}

// target, draft, drafted, accept, sample, count, pdl: a pair of tensors
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 7);
        must(zl.verify);
        const at::Tensor &p = here(a[0], false), &words = here(a[2], true), &accept = here(a[3], true), &sample = here(a[4], true);
        must(p.dim() == 3 && p.scalar_type() == at::kFloat && p.size(1) > 0 && p.size(2) > 0 && p.stride(2) == 1);
        const int64_t b = p.size(0), k = p.size(1) - 1, vocab = p.size(2);
        must(b > 0 && b < 1 << 30 && k < 1 << 30 && vocab <= 1 << 30);
        long long d_seq = 0, d_row = 0;
        const float* draft = nullptr;
        if (a[1] != Py_None) {
            const at::Tensor& d = here(a[1], false);
            must(d.dim() == 3 && d.size(0) == b && d.size(1) == k && d.size(2) == vocab && d.scalar_type() == at::kFloat && d.stride(2) == 1);
            draft = static_cast<const float*>(d.data_ptr()), d_seq = d.stride(0), d_row = d.stride(1);
        }
        must(words.scalar_type() == at::kInt && words.dim() == 2 && words.size(0) == b && words.size(1) == k);
        must(accept.scalar_type() == at::kFloat && accept.dim() == 2 && accept.size(0) == b && accept.size(1) == k);
        must(sample.scalar_type() == at::kFloat && sample.dim() == 1 && sample.size(0) == b);
        const int32_t* count = a[5] == Py_None ? nullptr : ints(a[5], b);
        const int pdl = truth(a[6]);
        const at::Tensor accepted = empty(p, {b}, at::kInt), tokens = empty(p, {b, k + 1}, at::kInt);
        const zl_stream_t s = stream();
        const int rc = unlocked([&] {
            return zl.verify(static_cast<const float*>(p.data_ptr()), p.stride(0), p.stride(1), draft, d_seq, d_row, static_cast<const int32_t*>(words.data_ptr()),
                             static_cast<const float*>(accept.data_ptr()), static_cast<const float*>(sample.data_ptr()), count, static_cast<int32_t*>(accepted.data_ptr()),
                             static_cast<int32_t*>(tokens.data_ptr()), (int)b, (int)k, (int)vocab, pdl, s);
        });
        return rc ? PyLong_FromLong(rc) : pair_of(accepted, tokens);
    });
}

// k_cache, v_cache, dtype, pages, pdl: a pair of tensors, or one where v_cache is None
PyObject* int4_cache_values(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 5);
        must(zl.values4 && THPDtype_Check(a[2]));
        const at::ScalarType type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
        const at::Tensor &k = here(a[0], false), &v = a[1] == Py_None ? k : here(a[1], false);
        Paged c = {};
        caches(c, k, v, type, true);
        const int32_t* pages = nullptr;
        int64_t n = c.pages;
        if (a[3] != Py_None) {
            const at::Tensor& t = here(a[3], true);
            must(t.scalar_type() == at::kInt && t.dim() == 1);
            pages = static_cast<const int32_t*>(t.data_ptr()), n = t.size(0);
        }
        must(n > 0);
        const int pdl = truth(a[4]);
        const at::Tensor k_out = empty(k, {n, c.page_size, c.kv_heads, c.dim}, type);
        at::Tensor v_out;
        if (a[1] != Py_None) v_out = empty(k, k_out.sizes(), type);
        void* const second = a[1] != Py_None ? v_out.data_ptr() : nullptr;
        const int dt = dtype_of(k_out);
        const zl_stream_t s = stream();
        const int rc = unlocked([&] {
            return zl.values4(c.k, second ? c.v : nullptr, c.pages, c.page_size, c.step[0], c.step[1], c.step[2], pages, n, k_out.data_ptr(), second, c.kv_heads, c.dim, dt,
                              pdl, s);
        });
        if (rc || !second) return result(rc, k_out);
        return pair_of(k_out, v_out);
    });
}

// logits, tokens, token_seq, token_lens, prompt_lens, repetition, frequency, presence, bias_starts, bias_words, bias, temperature, mask, mask_row, out_dtype, out, pdl
PyObject* adjust_logits(PyObject*, PyObject* const* a, Py_ssize_t na) {
    return guarded([&]() -> PyObject* {
        args(na, 17);
        must(zl.adjust);
        const at::Tensor& x = here(a[0], false);
        must(x.dim() == 2 && x.size(0) > 0 && x.size(0) < 1 << 30 && x.size(1) > 0 && x.size(1) <= 1 << 24 && x.stride(1) == 1);
        const int64_t r = x.size(0), vocab = x.size(1);
        const int dt = dtype_of(x);
        at::ScalarType type = x.scalar_type();
        if (a[14] != Py_None) {
            must(THPDtype_Check(a[14]));
            type = reinterpret_cast<THPDtype*>(a[14])->scalar_type;
        } else if (a[15] != Py_None) {
            type = here(a[15], false).scalar_type();
        }
        must(type == x.scalar_type() || type == at::kFloat);
        const long long ld = r > 1 ? x.stride(0) : vocab;
        must(ld >= vocab);
        auto rows = [&](PyObject* o) { return o == Py_None ? nullptr : ints(o, r); };
        auto floats = [&](PyObject* o, int64_t n) -> const float* {
            if (o == Py_None) return nullptr;
            const at::Tensor& t = here(o, true);
            must(t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == n);
            return static_cast<const float*>(t.data_ptr());
        };
        struct Table {
            const int32_t* at;
            long long ld;
            int rows, cols;
        };
        auto table = [&](PyObject* o) -> Table {   // (rows, columns) int32
            const at::Tensor& t = here(o, false);
            must(t.scalar_type() == at::kInt && t.dim() == 2 && t.numel() > 0 && t.size(0) < 1 << 30 && t.size(1) < 1 << 23 && (t.stride(1) == 1 || t.size(1) == 1));
            const long long step = t.size(0) > 1 ? t.stride(0) : t.size(1);
            must(step >= t.size(1));
            return {static_cast<const int32_t*>(t.data_ptr()), step, (int)t.size(0), (int)t.size(1)};
        };
        Table words = {}, mask = {};
        if (a[1] != Py_None) {
            words = table(a[1]);
            must(a[3] != Py_None && (a[2] != Py_None || words.rows >= r));
        } else {
            for (int i = 2; i < 8; ++i) must(a[i] == Py_None);
        }
        const int32_t *seq = rows(a[2]), *lens = rows(a[3]), *prompt = rows(a[4]);
        const float *rep = floats(a[5], r), *freq = floats(a[6], r), *pres = floats(a[7], r), *heat = floats(a[11], r);
        const int32_t *starts = nullptr, *bias_words = nullptr;
        const float* bias = nullptr;
        int64_t n = 0;
        if (a[8] != Py_None) {
            starts = ints(a[8], r + 1);
            const at::Tensor& w = here(a[9], true);
            must(w.dim() == 1 && w.size(0) < 1ll << 31 && a[10] != Py_None);
            n = w.size(0);
            bias_words = ints(a[9], n), bias = floats(a[10], n);
            if (n == 0) starts = nullptr;
        } else {
            must(a[9] == Py_None && a[10] == Py_None);
        }
        const int32_t* mask_row = nullptr;
        if (a[12] != Py_None) {
            mask = table(a[12]), mask_row = rows(a[13]);
            must(mask.cols * 32ll >= vocab && (mask_row || mask.rows >= r));
        } else {
            must(a[13] == Py_None);
        }
        if (a[15] != Py_None) {
            const at::Tensor& o = here(a[15], false);
            must(o.sizes() == x.sizes() && o.scalar_type() == type && o.stride(1) == 1);
        }
        const at::Tensor out = a[15] == Py_None ? empty(x, {r, vocab}, type) : THPVariable_Unpack(a[15]);
        const long long ld_out = r > 1 ? out.stride(0) : vocab;
        must(ld_out >= vocab);
        const int out_dt = dtype_of(out), pdl = truth(a[16]);
        const zl_stream_t s = stream();
        return result(unlocked([&] {
                          return zl.adjust(x.data_ptr(), ld, dt, out.data_ptr(), ld_out, out_dt, (int)r, (int)vocab, words.at, words.ld, words.rows, words.cols, seq, lens,
                                           prompt, rep, freq, pres, starts, bias_words, bias, (int)n, heat, mask.at, mask.ld, mask.rows, mask_row, pdl, s);
                      }),
                      out);
    });
}

// {name of an entry point: its address}
PyObject* bind(PyObject*, PyObject* d) {
    if (!PyDict_Check(d)) {
        PyErr_SetString(PyExc_TypeError, "a dict of addresses");
        return nullptr;
    }
    auto set = [&](auto& f, const char* name) {
        PyObject* v = PyDict_GetItemString(d, name);   // borrowed
        f = reinterpret_cast<std::decay_t<decltype(f)>>(v ? PyLong_AsVoidPtr(v) : nullptr);
    };
    set(zl.w4, "zl_w4a16_gemm_fused");
    set(zl.dense, "zl_dense_gemm_skinny");
    set(zl.int8_quant, "zl_int8_quant_per_token");
    set(zl.fp8_quant, "zl_fp8_quant_per_tensor");
    set(zl.w8, "zl_w8a8_gemm");
    set(zl.attn_bytes, "zl_decode_attention_workspace_bytes");
    set(zl.attn, "zl_decode_attention_host");
    set(zl.axes_rope, "zl_qkv_axes_rope_append");
    set(zl.paged_bytes, "zl_paged_attention_workspace_bytes");
    set(zl.paged, "zl_paged_attention");
    set(zl.verify, "zl_verify_drafts");
    set(zl.axes_rope4, "zl_qkv_axes_rope_append_int4");
    set(zl.values4, "zl_int4_cache_values");
    set(zl.paged4_bytes, "zl_paged_attention_int4_workspace_bytes");
    set(zl.paged4, "zl_paged_attention_int4");
    set(zl.adjust, "zl_adjust_logits");
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

#define ZL_FAST_AS(name, ...) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(__VA_ARGS__)), METH_FASTCALL, nullptr}
#define ZL_FAST(name) ZL_FAST_AS(#name, name)
PyMethodDef methods[] = {ZL_FAST(w4a16_gemm_fused), ZL_FAST(dense_gemm_skinny), ZL_FAST(w8_linear), ZL_FAST(decode_attention),
                         ZL_FAST_AS("qkv_axes_rope_append", axes_rope_append<false>), ZL_FAST_AS("paged_attention", attend<false>), ZL_FAST(verify_drafts),
                         ZL_FAST_AS("qkv_axes_rope_append_int4", axes_rope_append<true>), ZL_FAST_AS("paged_attention_int4", attend<true>),
                         ZL_FAST(int4_cache_values), ZL_FAST(adjust_logits),
                         {"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }

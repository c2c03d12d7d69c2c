// The decoder-attention calls from PyTorch tensors: ops.py hands its arguments over as they are, and a call
// whose operands are all in order goes straight to the C ABI. Anything else returns kNotInOrder and nothing has
// happened; ops.py then looks for what is wrong and raises. Through attributes and ctypes the checks and the
// call of these operators took 7 to 16 us, longer than their kernels at the smallest sizes (3 to 7 us).
//
// Every function takes its tensors (or None) first and ends in the current device's index and its current
// stream's handle; it returns the C ABI's status, or kNotInOrder.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "forge_amd.h"

#include <initializer_list>

namespace {

constexpr long kNotInOrder = -1000;

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// A device tensor of this type on this device.
bool on(const at::Tensor* t, at::ScalarType type, long device) {
    return t && t->scalar_type() == type && t->is_cuda() && t->get_device() == device && t->has_storage() &&
           !t->is_conj() && !t->is_neg() && !t->_is_zerotensor();
}
bool dense(const at::Tensor* t, at::ScalarType type, long device, std::initializer_list<int64_t> shape) {
    return on(t, type, device) && t->is_contiguous() && t->sizes().equals(c10::IntArrayRef(shape));
}
template <class T>
T* at_(const at::Tensor* t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }
template <class T>
T* at_(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

int code(at::ScalarType t) { return t == at::kHalf ? FORGE_FP16 : t == at::kBFloat16 ? FORGE_BF16 : -1; }

// (tokens, heads, D) with contiguous heads, and its token and head strides (0 along a dimension of one element).
struct Heads {
    const at::Tensor* t;
    int64_t tokens, heads, D, token, head;
    bool take(PyObject* o, at::ScalarType type, long device) {
        t = tensor(o);
        if (!on(t, type, device) || t->dim() != 3) return false;
        tokens = t->size(0); heads = t->size(1); D = t->size(2);
        token = tokens > 1 ? t->stride(0) : 0;
        head = heads > 1 ? t->stride(1) : 0;
        return D > 0 && t->stride(2) == 1;
    }
};

struct Call {
    PyObject* const* a;
    long device;
    void* stream;
    Call(PyObject* const* args, Py_ssize_t n)
        : a(args), device(PyLong_AsLong(args[n - 2])), stream(PyLong_AsVoidPtr(args[n - 1])) {}
    bool none(int i) const { return a[i] == Py_None; }
    // Numbers and flags, before the library is called: what is none leaves its error for call() to clear.
    bool number(int i, float* to) const {
        *to = static_cast<float>(PyFloat_AsDouble(a[i]));
        return !PyErr_Occurred();
    }
    bool flag(int i, int* to) const { return (*to = PyObject_IsTrue(a[i])) >= 0; }
};

// Runs f (Call -> status) if the argument count is right; no exception leaves.
template <int N, class F>
PyObject* call(PyObject* const* args, Py_ssize_t n, const F& f) {
    long status = kNotInOrder;
    if (n == N) {
        try {
            status = f(Call(args, n));
        } catch (...) {
            status = kNotInOrder;
        }
        if (PyErr_Occurred()) {
            PyErr_Clear();
            status = kNotInOrder;
        }
    }
    return PyLong_FromLong(status);
}

// int4_linear(x, w_int4, w_scale, bias, out, device, stream)
PyObject* int4_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<7>(args, n, [](const Call& c) -> long {
        const at::Tensor *x = tensor(c.a[0]), *w = tensor(c.a[1]), *s = tensor(c.a[2]), *out = tensor(c.a[4]);
        if (!x || x->dim() != 2 || !s || s->dim() != 2 || s->size(1) == 0) return kNotInOrder;
        const at::ScalarType type = x->scalar_type();
        const int64_t M = x->size(0), K = x->size(1), N = s->size(0), group = K / s->size(1);
        // (no values, K = 0, would be no work to the library, and the output nobody's)
        if (code(type) < 0 || group <= 0 || group * s->size(1) != K || !dense(x, type, c.device, {M, K}) ||
            !dense(s, at::kHalf, c.device, {N, s->size(1)}) || !dense(w, at::kByte, c.device, {N, (K + 127) / 128 * 64}) ||
            !dense(out, type, c.device, {M, N}) || M > INT32_MAX || K > INT32_MAX || N > INT32_MAX)
            return kNotInOrder;
        const at::Tensor* bias = nullptr;
        if (!c.none(3) && !dense(bias = tensor(c.a[3]), type, c.device, {N})) return kNotInOrder;
        return forge_int4_linear(at_<uint16_t>(x), at_<uint8_t>(w), at_<uint16_t>(s), at_<uint16_t>(bias), at_<uint16_t>(out),
                                 static_cast<int>(M), static_cast<int>(K), static_cast<int>(N), static_cast<int>(group),
                                 code(type), c.stream);
    });
}

// qk_norm_rope(q, k, v, q_weight, k_weight, cos, sin, positions, q_out, k_out, k_cache, v_cache, slots, eps,
// interleaved, device, stream): with k_out, with v, k_cache, v_cache and slots, or with both
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<17>(args, n, [](const Call& c) -> long {
        const at::Tensor* q0 = tensor(c.a[0]);
        if (!q0) return kNotInOrder;
        const at::ScalarType type = q0->scalar_type();
        Heads q, k, v = {};
        float eps;
        int interleaved;
        if (!c.number(13, &eps) || !c.flag(14, &interleaved)) return kNotInOrder;
        if (code(type) < 0 || !q.take(c.a[0], type, c.device) || !k.take(c.a[1], type, c.device)) return kNotInOrder;
        const int64_t T = q.tokens, D = q.D;
        const at::Tensor *qw = nullptr, *kw = nullptr, *cos = tensor(c.a[5]), *sin = tensor(c.a[6]), *pos = tensor(c.a[7]);
        const at::Tensor *q_out = tensor(c.a[8]), *k_out = nullptr, *kc = nullptr, *vc = nullptr, *slots = nullptr;
        if (!cos || cos->dim() != 2) return kNotInOrder;
        const int64_t P = cos->size(0), half = cos->size(1);
        if (k.tokens != T || k.D != D || !dense(cos, at::kFloat, c.device, {P, half}) || !dense(sin, at::kFloat, c.device, {P, half}) ||
            !dense(pos, at::kInt, c.device, {T}) || !dense(q_out, type, c.device, {T, q.heads, D}) || P > INT32_MAX ||
            T > INT32_MAX || D > 256 || half > 128)
            return kNotInOrder;
        if (!c.none(3) && !dense(qw = tensor(c.a[3]), type, c.device, {D})) return kNotInOrder;
        if (!c.none(4) && !dense(kw = tensor(c.a[4]), type, c.device, {D})) return kNotInOrder;
        int64_t rows = 0;
        if (c.none(9) && c.none(10)) return kNotInOrder;
        if (!c.none(9) && !dense(k_out = tensor(c.a[9]), type, c.device, {T, k.heads, D})) return kNotInOrder;
        if (!c.none(10)) {
            kc = tensor(c.a[10]);
            if (!kc || kc->dim() != 4 || !v.take(c.a[2], type, c.device) || v.tokens != T || v.heads != k.heads || v.D != D)
                return kNotInOrder;
            const int64_t pages = kc->size(0), page = kc->size(1);
            rows = pages * page;
            if (!dense(kc, type, c.device, {pages, page, k.heads, D}) ||
                !dense(vc = tensor(c.a[11]), type, c.device, {pages, page, k.heads, D}) ||
                !dense(slots = tensor(c.a[12]), at::kInt, c.device, {T}))
                return kNotInOrder;
        }
        return forge_qk_norm_rope(
            at_<uint16_t>(q.t), at_<uint16_t>(k.t), at_<uint16_t>(v.t), at_<uint16_t>(qw), at_<uint16_t>(kw), at_<float>(cos),
            at_<float>(sin), at_<int32_t>(pos), at_<uint16_t>(q_out), at_<uint16_t>(k_out), at_<uint16_t>(kc),
            at_<uint16_t>(vc), at_<int32_t>(slots), rows, static_cast<int>(T), static_cast<int>(q.heads),
            static_cast<int>(k.heads), static_cast<int>(D), static_cast<int>(2 * half), static_cast<int>(P), q.token, q.head,
            k.token, k.head, v.token, v.head, eps, interleaved, code(type), c.stream);
    });
}

// prompt_attention(q, k, v, cu_seqlens, out, scale, causal, device, stream)
PyObject* prompt_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<9>(args, n, [](const Call& c) -> long {
        const at::Tensor *q0 = tensor(c.a[0]), *cu = tensor(c.a[3]), *out = tensor(c.a[4]);
        if (!q0 || !cu || cu->dim() != 1 || cu->size(0) < 2) return kNotInOrder;
        const at::ScalarType type = q0->scalar_type();
        Heads q, k, v;
        float scale;
        int causal;
        if (!c.number(5, &scale) || !c.flag(6, &causal)) return kNotInOrder;
        if (code(type) < 0 || !q.take(c.a[0], type, c.device) || !k.take(c.a[1], type, c.device) ||
            !v.take(c.a[2], type, c.device))
            return kNotInOrder;
        const int64_t T = q.tokens, seqs = cu->size(0) - 1;
        if (k.tokens != T || v.tokens != T || k.D != q.D || v.D != q.D || k.heads != v.heads || k.heads == 0 || T > INT32_MAX ||
            seqs > INT32_MAX || !dense(cu, at::kInt, c.device, {seqs + 1}) || !dense(out, type, c.device, {T, q.heads, q.D}))
            return kNotInOrder;
        return forge_prompt_attention(at_<uint16_t>(q.t), at_<uint16_t>(k.t), at_<uint16_t>(v.t), at_<int32_t>(cu),
                                      at_<uint16_t>(out), static_cast<int>(seqs), static_cast<int>(T),
                                      static_cast<int>(q.heads), static_cast<int>(k.heads), static_cast<int>(q.D), q.token, q.head,
                                      k.token, k.head, v.token, v.head, scale, causal, code(type), c.stream);
    });
}

// cache_attention(q, k_cache, v_cache, page_table, cache_lens, tree, workspace, out, scale, device, stream)
PyObject* cache_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<11>(args, n, [](const Call& c) -> long {
        const at::Tensor *q = tensor(c.a[0]), *kc = tensor(c.a[1]), *vc = tensor(c.a[2]), *table = tensor(c.a[3]);
        const at::Tensor *lens = tensor(c.a[4]), *tree = nullptr, *ws = nullptr, *out = tensor(c.a[7]);
        if (!q || q->dim() != 4 || !kc || kc->dim() != 4 || !table || table->dim() != 2) return kNotInOrder;
        const at::ScalarType type = q->scalar_type();
        const int64_t B = q->size(0), T = q->size(1), Hq = q->size(2), D = q->size(3);
        const int64_t pages = kc->size(0), page = kc->size(1), Hkv = kc->size(2), width = table->size(1);
        float scale;
        if (!c.number(8, &scale)) return kNotInOrder;
        if (code(type) < 0 || T < 1 || T > 64 || D < 1 || !dense(q, type, c.device, {B, T, Hq, D}) || !dense(kc, type, c.device, {pages, page, Hkv, D}) ||
            !dense(vc, type, c.device, {pages, page, Hkv, D}) || !dense(table, at::kInt, c.device, {B, width}) ||
            !dense(lens, at::kInt, c.device, {B}) || !dense(out, type, c.device, {B, T, Hq, D}) || B > INT32_MAX ||
            Hq > INT32_MAX || pages > INT32_MAX || page > INT32_MAX || width > INT32_MAX)
            return kNotInOrder;
        if (!c.none(5) && !dense(tree = tensor(c.a[5]), at::kLong, c.device, {B, T})) return kNotInOrder;
        if (!c.none(6) && (!on(ws = tensor(c.a[6]), at::kByte, c.device) || !ws->is_contiguous())) return kNotInOrder;
        return forge_cache_attention(at_<uint16_t>(q), at_<uint16_t>(kc), at_<uint16_t>(vc), at_<int32_t>(table),
                                     at_<int32_t>(lens), at_<int64_t>(tree), at_<uint16_t>(out), static_cast<int>(B), static_cast<int>(T),
                                     static_cast<int>(Hq), static_cast<int>(Hkv), static_cast<int>(D), static_cast<int>(pages),
                                     static_cast<int>(page), static_cast<int>(width), scale, code(type), at_<void>(ws),
                                     ws ? static_cast<size_t>(ws->numel()) : 0, c.stream);
    });
}

// (pages, heads, page size, bytes of a position) of a 4-bit cache for heads of D values.
bool cache4(const at::Tensor* t, long device, int64_t heads, int64_t D) {
    if (!t || t->dim() != 4 || D < 1 || D > 256) return false;
    const int64_t units = D <= 64 ? 2 : D <= 96 ? 3 : D <= 128 ? 4 : D <= 192 ? 6 : 8;
    return dense(t, at::kByte, device, {t->size(0), heads, t->size(2), 32 * units + 8}) && t->size(0) <= INT32_MAX && t->size(2) <= INT32_MAX;
}

// cache4_write(k, v, cache, slots, device, stream)
PyObject* cache4_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<6>(args, n, [](const Call& c) -> long {
        const at::Tensor *k0 = tensor(c.a[0]), *cache = tensor(c.a[2]), *slots = tensor(c.a[3]);
        if (!k0) return kNotInOrder;
        const at::ScalarType type = k0->scalar_type();
        Heads k, v;
        if (code(type) < 0 || !k.take(c.a[0], type, c.device) || !v.take(c.a[1], type, c.device) || v.tokens != k.tokens ||
            v.heads != k.heads || v.D != k.D || k.heads == 0 || k.heads > INT32_MAX || k.tokens > INT32_MAX || !cache4(cache, c.device, k.heads, k.D) ||
            !dense(slots, at::kInt, c.device, {k.tokens}))
            return kNotInOrder;
        return forge_cache4_write(at_<uint16_t>(k.t), at_<uint16_t>(v.t), at_<uint8_t>(cache), at_<int32_t>(slots),
                                  static_cast<int>(k.tokens), static_cast<int>(k.heads), static_cast<int>(k.D),
                                  static_cast<int>(cache->size(0)), static_cast<int>(cache->size(2)), k.token, k.head, v.token, v.head,
                                  code(type), c.stream);
    });
}

// cache4_read(cache, slots, k_out, v_out, D, dtype, device, stream)
PyObject* cache4_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<8>(args, n, [](const Call& c) -> long {
        const at::Tensor *cache = tensor(c.a[0]), *slots = tensor(c.a[1]), *k = tensor(c.a[2]), *v = tensor(c.a[3]);
        if (!k || k->dim() != 3) return kNotInOrder;
        const at::ScalarType type = k->scalar_type();
        const int64_t T = k->size(0), heads = k->size(1), D = k->size(2);
        if (!THPDtype_Check(c.a[5]) || reinterpret_cast<THPDtype*>(c.a[5])->scalar_type != type || !PyLong_CheckExact(c.a[4]) ||
            PyLong_AsLongLong(c.a[4]) != D || code(type) < 0 || heads == 0 || heads > INT32_MAX || T > INT32_MAX || !cache4(cache, c.device, heads, D) ||
            !dense(slots, at::kInt, c.device, {T}) || !dense(k, type, c.device, {T, heads, D}) || !dense(v, type, c.device, {T, heads, D}))
            return kNotInOrder;
        return forge_cache4_read(at_<uint8_t>(cache), at_<int32_t>(slots), at_<uint16_t>(k), at_<uint16_t>(v), static_cast<int>(T),
                                 static_cast<int>(heads), static_cast<int>(D), static_cast<int>(cache->size(0)),
                                 static_cast<int>(cache->size(2)), code(type), c.stream);
    });
}

// A call of cache4_attention: q, cache, page_table, cache_lens and tree in a[0..4], checked.
struct Attend4 {
    const at::Tensor *q, *cache, *table, *lens, *tree;
    bool take(const Call& c) {
        q = tensor(c.a[0]); cache = tensor(c.a[1]); table = tensor(c.a[2]); lens = tensor(c.a[3]); tree = nullptr;
        if (!q || q->dim() != 4 || !cache || cache->dim() != 4 || !table || table->dim() != 2) return false;
        const at::ScalarType type = q->scalar_type();
        const int64_t B = q->size(0), T = q->size(1), Hq = q->size(2), D = q->size(3), Hkv = cache->size(1), width = table->size(1);
        return code(type) >= 0 && T >= 1 && T <= 64 && D >= 1 && Hkv >= 1 && dense(q, type, c.device, {B, T, Hq, D}) && cache4(cache, c.device, Hkv, D) &&
               dense(table, at::kInt, c.device, {B, width}) && dense(lens, at::kInt, c.device, {B}) && B <= INT32_MAX && Hq <= INT32_MAX &&
               Hkv <= INT32_MAX && width <= INT32_MAX && (c.none(4) || dense(tree = tensor(c.a[4]), at::kLong, c.device, {B, T}));
    }
    long run(const Call& c, const at::Tensor& out, const at::Tensor* ws, float scale) const {
        return forge_cache4_attention(at_<uint16_t>(q), at_<uint8_t>(cache), at_<int32_t>(table), at_<int32_t>(lens), at_<int64_t>(tree),
                                      at_<uint16_t>(out), static_cast<int>(q->size(0)), static_cast<int>(q->size(1)), static_cast<int>(q->size(2)),
                                      static_cast<int>(cache->size(1)), static_cast<int>(q->size(3)), static_cast<int>(cache->size(0)),
                                      static_cast<int>(cache->size(2)), static_cast<int>(table->size(1)), scale, code(q->scalar_type()),
                                      at_<void>(ws), ws ? ws->nbytes() : 0, c.stream);
    }
};

// cache4_attention(q, cache, page_table, cache_lens, tree, workspace, out, scale, device, stream)
PyObject* cache4_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<10>(args, n, [](const Call& c) -> long {
        Attend4 f;
        const at::Tensor *ws = nullptr, *out = tensor(c.a[6]);
        float scale;
        if (!c.number(7, &scale) || !f.take(c) || !out || !dense(out, f.q->scalar_type(), c.device, {f.q->size(0), f.q->size(1), f.q->size(2), f.q->size(3)}))
            return kNotInOrder;
        if (!c.none(5) && (!on(ws = tensor(c.a[5]), at::kByte, c.device) || !ws->is_contiguous())) return kNotInOrder;
        return f.run(c, *out, ws, scale);
    });
}

// The tensors that a call has made, if its status is 0.
template <size_t N>
PyObject* made_or(PyObject* status, at::Tensor (&made)[N]) {
    if (!status || PyLong_AsLong(status) != 0) return status;
    PyObject* tuple = PyTuple_New(N);
    if (!tuple) return nullptr;
    Py_DECREF(status);
    for (size_t i = 0; i < N; i++) PyTuple_SET_ITEM(tuple, i, THPVariable_Wrap(std::move(made[i])));
    return tuple;
}

// cache4_attention_new(q, cache, page_table, cache_lens, tree, scale, device, stream): the output, or a status
PyObject* cache4_attention_new(PyObject*, PyObject* const* args, Py_ssize_t n) {
    at::Tensor made[1];
    return made_or(call<8>(args, n, [&](const Call& c) -> long {
        Attend4 f;
        float scale;
        if (!c.number(5, &scale) || !f.take(c) || f.q->numel() == 0) return kNotInOrder;
        const size_t size = forge_cache4_attention_workspace_size(static_cast<int>(f.q->size(0)), static_cast<int>(f.q->size(1)),
                                                                  static_cast<int>(f.q->size(2)), static_cast<int>(f.cache->size(1)),
                                                                  static_cast<int>(f.q->size(3)), f.table->size(1) * f.cache->size(2));
        made[0] = at::empty(f.q->sizes(), f.q->options());
        at::Tensor ws;
        if (size) ws = at::empty({static_cast<int64_t>(size)}, f.cache->options());
        return f.run(c, made[0], size ? &ws : nullptr, scale);
    }), made);
}

// A call of beam_select: logits, scores and ended in a[0..2], the count and the end token, checked.
struct Beams {
    const at::Tensor *x, *scores, *ended;
    int64_t B, W, V;
    long count, end;
    int kind;
    bool take(const Call& c, PyObject* count_of, PyObject* end_of) {
        x = tensor(c.a[0]); scores = tensor(c.a[1]); ended = nullptr;
        if (!x || x->dim() != 3 || !PyLong_CheckExact(count_of) || !PyLong_CheckExact(end_of)) return false;
        const at::ScalarType type = x->scalar_type();
        kind = type == at::kFloat ? FORGE_FP32 : code(type);
        B = x->size(0); W = x->size(1); V = x->size(2);
        count = PyLong_AsLong(count_of); end = PyLong_AsLong(end_of);
        return !PyErr_Occurred() && kind >= 0 && on(x, type, c.device) && B >= 1 && W >= 1 && V >= 1 && B <= INT32_MAX && W <= INT32_MAX &&
               V <= INT32_MAX && (V == 1 || x->stride(2) == 1) && count >= 1 && count <= 64 && end >= INT32_MIN && end <= INT32_MAX &&
               dense(scores, at::kFloat, c.device, {B, W}) && (c.none(2) || dense(ended = tensor(c.a[2]), at::kBool, c.device, {B, W}));
    }
    long run(const Call& c, const at::Tensor& os, const at::Tensor& ob, const at::Tensor& ot, const at::Tensor& ws) const {
        return forge_beam_select(at_<void>(x), at_<float>(scores), at_<uint8_t>(ended), static_cast<int>(end), at_<float>(os),
                                 at_<int32_t>(ob), at_<int32_t>(ot), static_cast<int>(B), static_cast<int>(W), static_cast<int>(V),
                                 static_cast<int>(count), x->stride(0), x->stride(1), kind, at_<void>(ws), ws.nbytes(), c.stream);
    }
};

// beam_select(logits, scores, ended, out_scores, out_beams, out_tokens, workspace, count, end_token, device, stream)
PyObject* beam_select(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<11>(args, n, [](const Call& c) -> long {
        Beams f;
        const at::Tensor *os = tensor(c.a[3]), *ob = tensor(c.a[4]), *ot = tensor(c.a[5]), *ws = tensor(c.a[6]);
        if (!f.take(c, c.a[7], c.a[8]) || !dense(os, at::kFloat, c.device, {f.B, f.count}) || !dense(ob, at::kInt, c.device, {f.B, f.count}) ||
            !dense(ot, at::kInt, c.device, {f.B, f.count}) || !on(ws, at::kByte, c.device) || !ws->is_contiguous())
            return kNotInOrder;
        return f.run(c, *os, *ob, *ot, *ws);
    });
}

// beam_select_new(logits, scores, ended, count, end_token, device, stream): the outputs, or a status
PyObject* beam_select_new(PyObject*, PyObject* const* args, Py_ssize_t n) {
    at::Tensor made[3];
    return made_or(call<7>(args, n, [&](const Call& c) -> long {
        Beams f;
        if (!f.take(c, c.a[3], c.a[4])) return kNotInOrder;
        const size_t size = forge_beam_select_workspace_size(static_cast<int>(f.B), static_cast<int>(f.W), static_cast<int>(f.V), static_cast<int>(f.count));
        if (size == 0) return kNotInOrder;
        made[0] = at::empty({f.B, f.count}, f.scores->options());
        for (int i : {1, 2}) made[i] = at::empty({f.B, f.count}, f.scores->options().dtype(at::kInt));
        return f.run(c, made[0], made[1], made[2], at::empty({static_cast<int64_t>(size)}, f.scores->options().dtype(at::kByte)));
    }), made);
}

// A call of fork_pages: its inputs in a[0..3] and the page size, checked.
struct Fork {
    const at::Tensor *table, *lens, *parents, *refs;
    int64_t rows, width, group, pages;
    long page;
    bool take(const Call& c, PyObject* page_size) {
        table = tensor(c.a[0]); lens = tensor(c.a[1]); parents = tensor(c.a[2]); refs = tensor(c.a[3]);
        if (!table || table->dim() != 2 || !parents || parents->dim() != 2 || !refs || refs->dim() != 1 || !PyLong_CheckExact(page_size)) return false;
        rows = table->size(0); width = table->size(1); group = parents->size(1); pages = refs->size(0);
        page = PyLong_AsLong(page_size);
        return !PyErr_Occurred() && page >= 1 && page <= INT32_MAX && rows >= 1 && rows <= INT32_MAX && width >= 1 && width <= INT32_MAX &&
               pages >= 1 && pages <= INT32_MAX && group >= 1 && parents->size(0) * group == rows && dense(table, at::kInt, c.device, {rows, width}) &&
               dense(lens, at::kInt, c.device, {rows}) && dense(refs, at::kInt, c.device, {pages}) &&
               dense(parents, at::kInt, c.device, {parents->size(0), group});
    }
    long run(const Call& c, const at::Tensor* const (&o)[6], const at::Tensor& ws) const {
        auto p = [](const at::Tensor* t) { return at_<int32_t>(t); };
        return forge_fork_pages(p(table), p(lens), p(parents), p(refs), p(o[0]), p(o[1]), p(o[2]), p(o[3]), p(o[4]), p(o[5]),
                                static_cast<int>(rows), static_cast<int>(group), static_cast<int>(width), static_cast<int>(pages),
                                static_cast<int>(page), at_<void>(ws), ws.nbytes(), c.stream);
    }
};

// fork_pages(page_table, cache_lens, parents, refs, table, lens, refs, slots, src, dst, workspace, page_size, device, stream)
PyObject* fork_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<14>(args, n, [](const Call& c) -> long {
        Fork f;
        const at::Tensor *o[6], *ws = tensor(c.a[10]);
        if (!f.take(c, c.a[11]) || !on(ws, at::kByte, c.device) || !ws->is_contiguous()) return kNotInOrder;
        for (int i = 0; i < 6; i++) o[i] = tensor(c.a[4 + i]);
        if (!dense(o[0], at::kInt, c.device, {f.rows, f.width}) || !dense(o[2], at::kInt, c.device, {f.pages})) return kNotInOrder;
        for (int i : {1, 3, 4, 5})
            if (!dense(o[i], at::kInt, c.device, {f.rows})) return kNotInOrder;
        return f.run(c, o, *ws);
    });
}

// `sizes` int32 values of one allocation, from element `first` on, as a tensor of its own. (Seven allocations took 5 us.)
at::Tensor part_of(const at::Tensor& all, int64_t first, c10::IntArrayRef sizes) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(first);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
}

// fork_pages_new(page_table, cache_lens, parents, refs, page_size, device, stream): the outputs, or a status
PyObject* fork_pages_new(PyObject*, PyObject* const* args, Py_ssize_t n) {
    at::Tensor made[6];
    return made_or(call<7>(args, n, [&](const Call& c) -> long {
        Fork f;
        if (!f.take(c, c.a[4]) || f.rows > INT32_MAX || f.pages > INT32_MAX) return kNotInOrder;
        const size_t size = forge_fork_pages_workspace_size(static_cast<int>(f.rows), static_cast<int>(f.pages));
        if (size == 0) return kNotInOrder;
        int64_t total = 0;
        auto place = [&](int64_t n) {                                // in steps of 256 bytes
            const int64_t at = total;
            total += (n + 63) / 64 * 64;
            return at;
        };
        const int64_t table = place(f.rows * f.width), refs = place(f.pages), row = place(f.rows);
        for (int i = 1; i < 4; i++) place(f.rows);
        const int64_t scratch = place((static_cast<int64_t>(size) + 3) / 4), step = (f.rows + 63) / 64 * 64;
        const at::Tensor all = at::empty({total}, f.table->options());
        made[0] = part_of(all, table, {f.rows, f.width});
        made[1] = part_of(all, row, {f.rows});
        made[2] = part_of(all, refs, {f.pages});
        for (int i = 1; i < 4; i++) made[2 + i] = part_of(all, row + i * step, {f.rows});
        const at::Tensor ws = part_of(all, scratch, {(static_cast<int64_t>(size) + 3) / 4});
        const at::Tensor* o[6];
        for (int i = 0; i < 6; i++) o[i] = &made[i];
        return f.run(c, o, ws);
    }), made);
}

// copy_pages(caches, src, dst, device, stream)
PyObject* copy_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return call<5>(args, n, [](const Call& c) -> long {
        constexpr int kMost = 256;
        const at::Tensor *src = tensor(c.a[1]), *dst = tensor(c.a[2]);
        const bool list = PyList_CheckExact(c.a[0]);
        if (!src || !dst || (!list && !PyTuple_CheckExact(c.a[0]))) return kNotInOrder;
        const Py_ssize_t count = list ? PyList_GET_SIZE(c.a[0]) : PyTuple_GET_SIZE(c.a[0]);
        if (count < 1 || count > kMost || !on(src, at::kInt, c.device) || !on(dst, at::kInt, c.device) || !src->is_contiguous() ||
            !dst->is_contiguous() || !src->sizes().equals(dst->sizes()) || src->numel() > INT32_MAX)
            return kNotInOrder;
        void* at[kMost];
        int64_t pages = 0, bytes = 0;
        for (Py_ssize_t i = 0; i < count; i++) {
            const at::Tensor* t = tensor(list ? PyList_GET_ITEM(c.a[0], i) : PyTuple_GET_ITEM(c.a[0], i));
            if (!t || !on(t, t->scalar_type(), c.device) || !t->is_contiguous() || t->dim() < 1 || t->size(0) < 1) return kNotInOrder;
            if (i == 0) {
                pages = t->size(0);
                bytes = static_cast<int64_t>(t->nbytes());
            }
            if (t->size(0) != pages || static_cast<int64_t>(t->nbytes()) != bytes) return kNotInOrder;
            at[i] = t->data_ptr();
        }
        if (pages > INT32_MAX || bytes == 0) return kNotInOrder;
        return forge_copy_pages(at, static_cast<int>(count), bytes / pages, static_cast<int>(pages), at_<int32_t>(src), at_<int32_t>(dst),
                                static_cast<int>(src->numel()), c.stream);
    });
}

#define FASTCALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FASTCALL(int4_linear), FASTCALL(qk_norm_rope), FASTCALL(prompt_attention), FASTCALL(cache_attention),
                         FASTCALL(cache4_write), FASTCALL(cache4_read), FASTCALL(cache4_attention), FASTCALL(cache4_attention_new),
                         FASTCALL(beam_select), FASTCALL(beam_select_new),                         FASTCALL(fork_pages), FASTCALL(fork_pages_new), FASTCALL(copy_pages),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "forge_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_forge_torch() { return PyModule_Create(&module); }

// The decoder-attention calls from PyTorch tensors: ops.py hands its arguments over as they are, and a call
// whose operands are all in order goes straight to the C ABI. Anything else returns kNotInOrder and nothing has
// happened; ops.py then looks for what is wrong and raises. Through attributes and ctypes the checks and the
// call of these operators took 7 to 16 us, longer than their kernels at the smallest sizes (3 to 7 us).
//
// Every function takes its tensors (or None) first and ends in the current device's index and its current
// stream's handle; it returns the C ABI's status, or kNotInOrder.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

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

#define FASTCALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FASTCALL(int4_linear), FASTCALL(qk_norm_rope), FASTCALL(prompt_attention), FASTCALL(cache_attention),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "forge_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_forge_torch() { return PyModule_Create(&module); }

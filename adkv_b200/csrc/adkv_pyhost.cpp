// Host side of adkv_b200.gemv.decode_attn in native code: argument checks, output allocation and the call into the C ABI
// of libadkv_b200.so for the form that a decode loop uses -- plain contiguous CUDA tensors on the current device, no mask,
// no checkpoints.  Whatever is not of that form, an argument error included, is left to the Python code: `decode` then
// returns None and has done nothing.
//
// A step of one short sequence is bound by this path: the device needs 9.4 us of it (batch 1, 128 tokens), the checks,
// attribute look-ups and 30-argument ctypes call of the Python path took 24 us.
//
// The same for gemv.decode_attn_prefix, step.norm_rope_qkv and step.process_logits, whose Python paths take 42, 25 and 17 us.
#include <ATen/EmptyTensor.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <climits>

#include "../../include/adkv_b200.h"

namespace {

using decode_fn = decltype(&adkv_decode_attn);
decode_fn g_decode = nullptr;   // the entry point of the library that _lib.py loaded
decltype(&adkv_decode_attn_prefix) g_prefix = nullptr;
decltype(&adkv_decode_attn_prefix_scratch_bytes) g_prefix_scratch = nullptr;
decltype(&adkv_norm_rope_qkv) g_rope = nullptr;
decltype(&adkv_process_logits) g_logits = nullptr;

// A tensor whose memory is what its metadata says: no subclass, no wrapper of a transform, no lazy conjugate or negative.
const at::Tensor *plain(PyObject *o)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    constexpr c10::DispatchKeySet odd({c10::DispatchKey::Conjugate, c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor,
                                       c10::DispatchKey::Python, c10::DispatchKey::Functionalize,
                                       c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched,
                                       c10::DispatchKey::BatchedNestedTensor, c10::DispatchKey::NestedTensor});
    if (!t.defined() || t.layout() != at::kStrided || t.key_set().has_any(odd) || !t.has_storage()) return nullptr;
    return &t;
}

struct Device {
    c10::DeviceIndex index;
    const at::Tensor *tensor(PyObject *o, at::ScalarType type) const
    {
        const at::Tensor *t = plain(o);
        if (!t || !t->is_cuda() || t->get_device() != index || t->scalar_type() != type || !t->is_contiguous()) return nullptr;
        return t;
    }
    const void *data(PyObject *o, at::ScalarType type, int64_t numel) const
    {
        const at::Tensor *t = tensor(o, type);
        return t && t->numel() == numel ? t->data_ptr() : nullptr;
    }
    bool params(PyObject *o, int64_t numel, adkv_params &p) const
    {
        if (!PyTuple_Check(o) && !PyList_Check(o)) return false;
        if (PySequence_Fast_GET_SIZE(o) != 5) return false;
        const void **at[5] = {&p.zp_init, &p.scale_init, &p.alpha, &p.beta, &p.target};
        for (int i = 0; i < 5; ++i)
            if (!(*at[i] = data(PySequence_Fast_GET_ITEM(o, i), at::kHalf, numel))) return false;
        return true;
    }
};

// Something between a call and the backend wants to see every tensor that is made (a dispatch mode, a transform): the Python path's business.
bool watched()
{
    constexpr c10::DispatchKeySet keys({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::Functionalize,
                                        c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode});
    return c10::impl::tls_local_dispatch_key_set().included_.has_any(keys);
}

// A tensor on the current device, as at::empty makes it but without its way through the dispatcher (0.5 us); not while watched().
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type)
{
    return at::detail::empty_generic(sizes, c10::GetAllocator(at::kCUDA), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

// A tuple of tensors, or None.
PyObject *results(std::initializer_list<at::Tensor> tensors)
{
    PyObject *t = PyTuple_New(Py_ssize_t(tensors.size()));
    Py_ssize_t i = 0;
    for (const at::Tensor &x : tensors) {
        PyObject *o = t ? THPVariable_Wrap(x) : nullptr;
        if (!o) {
            Py_XDECREF(t);
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}

bool as_int(PyObject *o, int &v)
{
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    const long n = PyLong_AsLongAndOverflow(o, &overflow);
    if (overflow || n < 0 || n >= INT_MAX) return false;
    v = int(n);
    return true;
}

bool as_float(PyObject *o, float &v)
{
    if (PyFloat_CheckExact(o)) v = float(PyFloat_AS_DOUBLE(o));
    else return false;
    return true;
}

// decode(q, k_cache, v_cache, k_new, v_new, k_params, v_params, T, scaling, scale_min, scale_max, bits, out, k_tail, v_tail,
// flags) -> the output tensor, an error code of the library, or None
PyObject *decode(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (n != 16 || !g_decode) Py_RETURN_NONE;
    try {
        const at::Tensor *kc = plain(a[1]), *vc = plain(a[2]);
        if (!kc || !vc || !kc->is_cuda() || kc->dim() != 6 || kc->size(4) != 4 || kc->size(5) != 4) Py_RETURN_NONE;
        const Device dev{kc->get_device()};
        if (dev.index != c10::cuda::current_device()) Py_RETURN_NONE;
        if (!dev.tensor(a[1], at::kByte) || !dev.tensor(a[2], at::kByte) || vc->sizes() != kc->sizes()) Py_RETURN_NONE;
        const int64_t B = kc->size(0), Hkv = kc->size(1), cap = kc->size(2), D = 4 * kc->size(3);
        const at::Tensor *q = dev.tensor(a[0], at::kHalf);
        if (!q || q->dim() != 4 || q->size(2) != 1 || q->size(0) != B || q->size(3) != D) Py_RETURN_NONE;
        const int64_t Hq = q->size(1);
        if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || B > INT_MAX || Hq > INT_MAX || cap > INT_MAX || D > 512) Py_RETURN_NONE;
        const void *kn = dev.data(a[3], at::kHalf, B * Hkv * D), *vn = dev.data(a[4], at::kHalf, B * Hkv * D);
        adkv_params kp, vp;
        int T, bits, flags;
        float scaling, smin, smax;
        if (!kn || !vn || !dev.params(a[5], Hkv * D, kp) || !dev.params(a[6], Hkv * D, vp) || !as_int(a[7], T) ||
            !as_float(a[8], scaling) || !as_float(a[9], smin) || !as_float(a[10], smax) || !as_int(a[11], bits) ||
            (bits != 2 && bits != 4) || T / (32 / bits) >= cap || !as_int(a[15], flags))
            Py_RETURN_NONE;
        void *tail[2] = {nullptr, nullptr};
        if ((a[13] == Py_None) != (a[14] == Py_None)) Py_RETURN_NONE;
        if (a[13] != Py_None) {
            if (flags & ADKV_FLAG_HALF_STATE) Py_RETURN_NONE;
            for (int i = 0; i < 2; ++i) {
                const at::Tensor *t = dev.tensor(a[13 + i], at::kFloat);
                if (!t || t->dim() != 4 || t->size(0) != B || t->size(1) != Hkv || t->size(2) != 2 || t->size(3) != D) Py_RETURN_NONE;
                tail[i] = t->data_ptr();
            }
        }
        void *const stream = c10::cuda::getCurrentCUDAStream(dev.index).stream();
        const void *const qp = q->data_ptr();
        void *const kcp = kc->data_ptr(), *const vcp = vc->data_ptr();
        // Everything that may fail comes before the launch, the Python object of the result too: a step that has been
        // launched must not be left to the Python code, which would launch it again.
        void *op;
        PyObject *result;
        if (a[12] == Py_None) {
            const at::Tensor out = at::empty({B, Hq, D}, kc->options().dtype(at::kHalf));
            if (!out.is_cuda() || !out.has_storage()) Py_RETURN_NONE;
            op = out.data_ptr();
            result = THPVariable_Wrap(out);
            if (!result) {
                PyErr_Clear();
                Py_RETURN_NONE;
            }
        } else {
            const at::Tensor *t = dev.tensor(a[12], at::kHalf);
            if (!t || t->dim() != 3 || t->size(0) != B || t->size(1) != Hq || t->size(2) != D) Py_RETURN_NONE;
            op = t->data_ptr();
            result = a[12];
            Py_INCREF(result);
        }
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = g_decode(qp, kcp, vcp, kn, vn, &kp, &vp, tail[0], tail[1], nullptr, 0, op, int(B), int(Hq), int(Hkv), T, int(D),
                      int(cap), bits, scaling, smin, smax, unsigned(flags), stream);
        Py_END_ALLOW_THREADS
        if (!rc) return result;
        Py_DECREF(result);
        return PyLong_FromLong(rc);
    } catch (...) {   // out of memory and the like: the Python code meets it again and raises what it raises
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

// decode_prefix(q, (address of the adkv_prefix, its heads, bits), k_cache, v_cache, k_new, v_new, k_params, v_params, T, scaling, scale_min,
// scale_max, k_tail, v_tail, flags, out, scratch) -> the output tensor, an error code of the library, or None
PyObject *decode_prefix(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (n != 17 || !g_prefix || watched()) Py_RETURN_NONE;
    try {
        const at::Tensor *kc = plain(a[2]), *vc = plain(a[3]);
        if (!kc || !vc || !kc->is_cuda() || kc->dim() != 6 || kc->size(4) != 4 || kc->size(5) != 4) Py_RETURN_NONE;
        const Device dev{kc->get_device()};
        if (dev.index != c10::cuda::current_device()) Py_RETURN_NONE;
        if (!dev.tensor(a[2], at::kByte) || !dev.tensor(a[3], at::kByte) || vc->sizes() != kc->sizes()) Py_RETURN_NONE;
        const int64_t B = kc->size(0), Hkv = kc->size(1), cap = kc->size(2), D = 4 * kc->size(3);
        const at::Tensor *q = dev.tensor(a[0], at::kHalf);
        if (!q || q->dim() != 4 || q->size(2) != 1 || q->size(0) != B || q->size(3) != D) Py_RETURN_NONE;
        const int64_t Hq = q->size(1);
        if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || B > INT_MAX || Hq > INT_MAX || cap > INT_MAX || D != 128) Py_RETURN_NONE;
        // (address, heads, bits, device) of the prefix, checked when it was made
        int heads, bits, index;
        if (!PyTuple_CheckExact(a[1]) || PyTuple_GET_SIZE(a[1]) != 4 || !as_int(PyTuple_GET_ITEM(a[1], 1), heads) || !as_int(PyTuple_GET_ITEM(a[1], 2), bits) ||
            !as_int(PyTuple_GET_ITEM(a[1], 3), index) || heads != Hkv || index != dev.index)
            Py_RETURN_NONE;
        const adkv_prefix *prefix = static_cast<const adkv_prefix *>(PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[1], 0)));
        if (!prefix) { PyErr_Clear(); Py_RETURN_NONE; }
        const void *kn = dev.data(a[4], at::kHalf, B * Hkv * D), *vn = dev.data(a[5], at::kHalf, B * Hkv * D);
        adkv_params kp, vp;
        int T = 0, flags;
        float scaling, smin, smax;
        if (!kn || !vn || !dev.params(a[6], Hkv * D, kp) || !dev.params(a[7], Hkv * D, vp) || !as_float(a[9], scaling) || !as_float(a[10], smin) ||
            !as_float(a[11], smax) || !as_int(a[14], flags))
            Py_RETURN_NONE;
        const void *lens = nullptr;
        if (PyLong_CheckExact(a[8])) {
            if (!as_int(a[8], T)) Py_RETURN_NONE;
        } else if (!(lens = dev.data(a[8], at::kInt, B))) {
            Py_RETURN_NONE;
        }
        if (T / (32 / bits) >= cap) Py_RETURN_NONE;
        void *tail[2];
        for (int i = 0; i < 2; ++i) {
            const at::Tensor *t = dev.tensor(a[12 + i], at::kFloat);
            if (!t || t->dim() != 4 || t->size(0) != B || t->size(1) != Hkv || t->size(2) != 2 || t->size(3) != D) Py_RETURN_NONE;
            tail[i] = t->data_ptr();
        }
        void *const stream = c10::cuda::getCurrentCUDAStream(dev.index).stream();
        const long long need = g_prefix_scratch(int(B), int(Hq), int(Hkv), prefix->tokens, prefix->interval);
        if (need < 0) Py_RETURN_NONE;
        at::Tensor own;
        void *scratch;
        long long room = need;
        if (a[16] == Py_None) {
            own = fresh({need}, at::kByte);
            scratch = own.data_ptr();
        } else {
            const at::Tensor *t = plain(a[16]);
            if (!t || !t->is_cuda() || t->get_device() != dev.index || !t->is_contiguous()) Py_RETURN_NONE;
            scratch = t->data_ptr();
            room = t->numel() * t->element_size();
        }
        const void *const qp = q->data_ptr();
        void *const kcp = kc->data_ptr(), *const vcp = vc->data_ptr();
        void *op;
        PyObject *result;   // before the launch, as in decode
        if (a[15] == Py_None) {
            const at::Tensor out = at::empty({B, Hq, D}, kc->options().dtype(at::kHalf));
            if (!out.is_cuda() || !out.has_storage()) Py_RETURN_NONE;
            op = out.data_ptr();
            result = THPVariable_Wrap(out);
            if (!result) {
                PyErr_Clear();
                Py_RETURN_NONE;
            }
        } else {
            const at::Tensor *t = dev.tensor(a[15], at::kHalf);
            if (!t || t->dim() != 3 || t->size(0) != B || t->size(1) != Hq || t->size(2) != D) Py_RETURN_NONE;
            op = t->data_ptr();
            result = a[15];
            Py_INCREF(result);
        }
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = g_prefix(qp, prefix, kcp, vcp, kn, vn, &kp, &vp, tail[0], tail[1], lens, T, op, scratch, room, int(B), int(Hq), int(Hkv), int(D), int(cap),
                      bits, scaling, smin, smax, unsigned(flags), stream);
        Py_END_ALLOW_THREADS
        if (!rc) return result;
        Py_DECREF(result);
        return PyLong_FromLong(rc);
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

int element_type(at::ScalarType t) { return t == at::kHalf ? ADKV_T_F16 : t == at::kBFloat16 ? ADKV_T_BF16 : t == at::kFloat ? ADKV_T_F32 : -1; }

// norm_rope(qkv, n_heads, n_kv_heads, cos, sin, start, positions, q_weight, k_weight, eps, interleaved, dtype) -> (q, k, v), an error code, or
// None
PyObject *norm_rope(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (n != 12 || !g_rope || watched()) Py_RETURN_NONE;
    try {
        const at::Tensor *x = plain(a[0]), *cos = plain(a[3]), *sin = plain(a[4]);
        int Hq, Hkv, start;
        float eps;
        if (!x || !cos || !sin || !x->is_cuda() || x->dim() != 3 || !as_int(a[1], Hq) || !as_int(a[2], Hkv) || !as_int(a[5], start) || !as_float(a[9], eps) ||
            !PyBool_Check(a[10]))
            Py_RETURN_NONE;
        const Device dev{x->get_device()};
        if (dev.index != c10::cuda::current_device()) Py_RETURN_NONE;
        const int64_t B = x->size(0), T = x->size(1), heads = int64_t(Hq) + 2 * int64_t(Hkv), width = x->size(2);
        if (Hq <= 0 || Hkv <= 0 || B <= 0 || T <= 0 || B > INT_MAX / T || width % heads) Py_RETURN_NONE;
        const int64_t D = width / heads;
        const at::ScalarType type = x->scalar_type();
        at::ScalarType to = type;
        if (a[11] != Py_None) {
            if (!THPDtype_Check(a[11])) Py_RETURN_NONE;
            to = reinterpret_cast<THPDtype *>(a[11])->scalar_type;
        }
        const int in_type = element_type(type), out_type = element_type(to);
        if ((D != 64 && D != 128 && D != 256 && D != 512) || in_type < 0 || (to != type && to != at::kHalf)) Py_RETURN_NONE;
        const uintptr_t step = 4 * x->element_size();
        if (x->stride(2) != 1 || x->stride(0) % 4 || x->stride(1) % 4 || reinterpret_cast<uintptr_t>(x->data_ptr()) % step) Py_RETURN_NONE;
        for (const at::Tensor *t : {cos, sin})
            if (!t->is_cuda() || t->get_device() != dev.index || t->scalar_type() != at::kFloat || t->dim() != 2 || t->stride(1) != 1) Py_RETURN_NONE;
        if (cos->sizes() != sin->sizes() || cos->stride(0) != sin->stride(0)) Py_RETURN_NONE;
        const int64_t rows = cos->size(0), rot = 2 * cos->size(1);
        if (rot <= 0 || rot > D || rot % 8 || rows > INT_MAX) Py_RETURN_NONE;
        const void *positions = nullptr;
        bool each = false;
        if (a[6] != Py_None) {
            const at::Tensor *t = dev.tensor(a[6], at::kInt);
            if (!t || start) Py_RETURN_NONE;
            each = t->dim() == 2;
            if (t->dim() < 1 || t->dim() > 2 || t->size(0) != B || (each && t->size(1) != T)) Py_RETURN_NONE;
            positions = t->data_ptr();
        } else if (start + T > rows) {
            Py_RETURN_NONE;
        }
        const void *weight[2] = {nullptr, nullptr};
        for (int i = 0; i < 2; ++i)
            if (a[7 + i] != Py_None) {
                const at::Tensor *t = dev.tensor(a[7 + i], type);
                if (!t || t->dim() != 1 || t->size(0) != D || reinterpret_cast<uintptr_t>(t->data_ptr()) % step) Py_RETURN_NONE;
                weight[i] = t->data_ptr();
            }
        const at::Tensor q = fresh({B, Hq, T, D}, to), k = fresh({B, Hkv, T, D}, to), v = fresh({B, Hkv, T, D}, to);
        void *const stream = c10::cuda::getCurrentCUDAStream(dev.index).stream();
        int rc;
        const void *const xp = x->data_ptr(), *const cp = cos->data_ptr(), *const sp = sin->data_ptr();
        const int64_t sb = x->stride(0), st = x->stride(1), table = cos->stride(0);
        const bool pairs = a[10] == Py_True;
        Py_BEGIN_ALLOW_THREADS
        rc = g_rope(xp, sb, st, in_type, q.data_ptr(), k.data_ptr(), v.data_ptr(), out_type, weight[0], weight[1], eps, cp, sp, table, int(rows), int(rot),
                    positions, each, start, int(B), int(T), Hq, Hkv, int(D), pairs, stream);
        Py_END_ALLOW_THREADS
        if (rc) return PyLong_FromLong(rc);
        return results({q, k, v});   // if that fails the call is made again: it only writes its results
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

// logits(logits, history, history_lens, repetition, presence, frequency, bias, mask) -> (out, tokens), an error code, or None; out is new
PyObject *logits(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (n != 8 || !g_logits || watched()) Py_RETURN_NONE;
    try {
        const at::Tensor *x = plain(a[0]);
        if (!x || !x->is_cuda() || x->dim() != 2 || x->stride(1) != 1) Py_RETURN_NONE;
        const Device dev{x->get_device()};
        const int64_t B = x->size(0), V = x->size(1);
        const int type = element_type(x->scalar_type());
        if (dev.index != c10::cuda::current_device() || type < 0 || B <= 0 || B > 65535 || V <= 0 || V > 0x7fff0000) Py_RETURN_NONE;
        const auto rows = [&](PyObject *o, at::ScalarType t, int64_t least) -> const at::Tensor * {   // [B, least or more], rows in one piece
            const at::Tensor *m = plain(o);
            if (!m || !m->is_cuda() || m->get_device() != dev.index || m->scalar_type() != t || m->dim() != 2 || m->size(0) != B || m->size(1) < least ||
                m->stride(1) != 1)
                return nullptr;
            return m;
        };
        const at::Tensor *history = nullptr, *mask = nullptr;
        const void *lens = nullptr, *per_row[3];
        float all_rows[3];
        if (a[1] != Py_None && !(history = rows(a[1], at::kInt, 1))) Py_RETURN_NONE;
        if (history && history->size(1) > INT_MAX) Py_RETURN_NONE;
        if (a[2] != Py_None && (!history || !(lens = dev.data(a[2], at::kInt, B)))) Py_RETURN_NONE;
        for (int i = 0; i < 3; ++i) {
            per_row[i] = nullptr;
            all_rows[i] = 0.f;
            if (as_float(a[3 + i], all_rows[i])) continue;
            const at::Tensor *t = dev.tensor(a[3 + i], at::kFloat);
            if (!t || t->dim() != 1 || t->size(0) != B) Py_RETURN_NONE;
            per_row[i] = t->data_ptr();
        }
        if (!per_row[0] && !(all_rows[0] > 0.f)) Py_RETURN_NONE;
        const void *bias = nullptr;
        int64_t bias_stride = 0;
        if (a[6] != Py_None) {
            const at::Tensor *t = plain(a[6]);
            if (t && t->dim() == 1) {
                bias = dev.data(a[6], at::kFloat, V);
            } else if ((t = rows(a[6], at::kFloat, V)) && t->size(1) == V) {
                bias = t->data_ptr();
                bias_stride = t->stride(0);
            }
            if (!bias) Py_RETURN_NONE;
        }
        if (a[7] != Py_None && !(mask = rows(a[7], at::kInt, (V + 31) / 32))) Py_RETURN_NONE;
        const at::Tensor out = fresh({B, V}, x->scalar_type()), tokens = fresh({B}, at::kInt);
        void *const stream = c10::cuda::getCurrentCUDAStream(dev.index).stream();
        const void *const xp = x->data_ptr(), *const hp = history ? history->data_ptr() : nullptr, *const mp = mask ? mask->data_ptr() : nullptr;
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = g_logits(xp, x->stride(0), out.data_ptr(), V, type, tokens.data_ptr(), hp, hp ? history->stride(0) : 0, hp ? int(history->size(1)) : 0, lens,
                      per_row[0], all_rows[0], per_row[1], all_rows[1], per_row[2], all_rows[2], bias, bias_stride, mp, mp ? mask->stride(0) : 0, int(B),
                      int(V), stream);
        Py_END_ALLOW_THREADS
        if (rc) return PyLong_FromLong(rc);
        return results({out, tokens});
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

// bind_more(address of adkv_decode_attn_prefix, its scratch size, adkv_norm_rope_qkv, adkv_process_logits)
PyObject *bind_more(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    if (n != 4) Py_RETURN_NONE;
    g_prefix = reinterpret_cast<decltype(g_prefix)>(PyLong_AsVoidPtr(a[0]));
    g_prefix_scratch = reinterpret_cast<decltype(g_prefix_scratch)>(PyLong_AsVoidPtr(a[1]));
    g_rope = reinterpret_cast<decltype(g_rope)>(PyLong_AsVoidPtr(a[2]));
    g_logits = reinterpret_cast<decltype(g_logits)>(PyLong_AsVoidPtr(a[3]));
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

PyObject *bind(PyObject *, PyObject *addr)
{
    g_decode = reinterpret_cast<decode_fn>(PyLong_AsVoidPtr(addr));
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
    {"decode_prefix", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode_prefix)), METH_FASTCALL, nullptr},
    {"norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm_rope)), METH_FASTCALL, nullptr},
    {"logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(logits)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_O, nullptr},
    {"bind_more", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind_more)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_adkv_pyhost", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__adkv_pyhost(void) { return PyModule_Create(&module); }

// The library's hot entry points for torch tensors, as a CPython module (hbq_host): what a decode step calls tens of
// thousands of times a second.  A call through ctypes costs more than its kernel: building the argument objects, two
// trips through Python's allocator and torch.empty, the stream query -- 20 us of host time for a 3 us quantizer, 43 us
// for one linear layer (quantizer + product) whose kernels take 9 to 27 us; through this module 12 us for the layer.
//
// Each function takes the plain case -- exact torch.Tensor objects (or parameters) of ordinary dense CUDA storage,
// contiguous, of the dtypes and shapes the kernel reads -- and returns None for anything else: the caller then runs its
// general path, which also raises the errors.  A negative return code of the library comes back as an int.  The module
// does not load the library itself: bind() is given the entry points of the copy that the process uses.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include "../../include/hbq_b200.h"

namespace {

// What this module was compiled for (build.py compares it with the process that is about to load it).
__attribute__((used)) const char built_for[] = HBQ_HOST_TAG;

decltype(&hbq_quantize) p_quantize = nullptr;
decltype(&hbq_gemm) p_gemm = nullptr;
decltype(&hbq_gemm_workspace_bytes) p_gemm_workspace_bytes = nullptr;
decltype(&hbq_gemm_w4) p_gemm_w4 = nullptr;
decltype(&hbq_rope_rotate) p_rope_rotate = nullptr;
decltype(&hbq_qk_norm_rope) p_qk_norm_rope = nullptr;
decltype(&hbq_attention_run) p_attention_run = nullptr;
decltype(&hbq_attention_workspace_bytes) p_attention_workspace_bytes = nullptr;

// The tensor behind `o` when it is a plain dense CUDA tensor: no Python subclass, no functorch wrapper, no fake or
// lazily conjugated / negated tensor (any of them brings a dispatch key of its own).
const at::Tensor* dense_cuda(PyObject* o)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda()) return nullptr;
    const c10::DispatchKeySet ordinary = c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
                                         c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA) | c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView);
    if ((t.key_set().raw_repr() & ~ordinary.raw_repr()) != 0 || !t.has_storage()) return nullptr;
    return &t;
}
// ... and contiguous
const at::Tensor* plain_cuda(PyObject* o)
{
    const at::Tensor* t = dense_cuda(o);
    return t && t->is_contiguous() ? t : nullptr;
}

bool to_i64(PyObject* o, int64_t* v)
{
    *v = PyLong_AsLongLong(o);
    return !(*v == -1 && PyErr_Occurred());
}

const hbq_format* to_format(PyObject* o)
{
    if (!PyBytes_CheckExact(o) || PyBytes_GET_SIZE(o) != (Py_ssize_t)sizeof(hbq_format)) {
        PyErr_SetString(PyExc_TypeError, "format must be the bytes of an hbq_format");
        return nullptr;
    }
    return reinterpret_cast<const hbq_format*>(PyBytes_AS_STRING(o));
}

// An optional fp16 vector of n elements beside `like`; false when it is something the general path has to convert.
bool plain_bias(PyObject* o, const at::Tensor& like, int64_t n, const void** p)
{
    *p = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* b = plain_cuda(o);
    if (!b || b->scalar_type() != at::kHalf || b->numel() != n || b->device() != like.device()) return false;
    *p = b->data_ptr();
    return true;
}

// Library calls run without the interpreter lock, as through ctypes: a launch may wait for room in the launch queue.
template <class F>
int unlocked(F f)
{
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

PyObject* result(int rc, const at::Tensor& t) { return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(t); }

// bind(quantize, gemm, gemm_workspace_bytes, gemm_w4, rope_rotate, qk_norm_rope, attention_run,
// attention_workspace_bytes): addresses of the library's entry points
PyObject* host_bind(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    int64_t a[8];
    if (n != 8) { PyErr_SetString(PyExc_TypeError, "bind takes eight addresses"); return nullptr; }
    for (int i = 0; i < 8; ++i)
        if (!to_i64(args[i], &a[i])) return nullptr;
    p_quantize = reinterpret_cast<decltype(p_quantize)>(a[0]);
    p_gemm = reinterpret_cast<decltype(p_gemm)>(a[1]);
    p_gemm_workspace_bytes = reinterpret_cast<decltype(p_gemm_workspace_bytes)>(a[2]);
    p_gemm_w4 = reinterpret_cast<decltype(p_gemm_w4)>(a[3]);
    p_rope_rotate = reinterpret_cast<decltype(p_rope_rotate)>(a[4]);
    p_qk_norm_rope = reinterpret_cast<decltype(p_qk_norm_rope)>(a[5]);
    p_attention_run = reinterpret_cast<decltype(p_attention_run)>(a[6]);
    p_attention_workspace_bytes = reinterpret_cast<decltype(p_attention_workspace_bytes)>(a[7]);
    Py_RETURN_NONE;
}

// quantize(x, format, out_dtype): the fake-quantised tensor; out_dtype: -1 as x, 0 fp16, 1 bf16
PyObject* host_quantize(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int64_t od;
    if (n != 3 || !to_i64(args[2], &od)) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "quantize(x, format, out_dtype)"); return nullptr; }
    const hbq_format* f = to_format(args[1]);
    if (!f) return nullptr;
    const at::Tensor* x = plain_cuda(args[0]);
    if (!x || x->dim() < 1 || x->numel() == 0 || (f->kind == HBQ_KIND_MXFP && f->per_tensor_scale)) Py_RETURN_NONE;
    const auto st = x->scalar_type();
    if (st != at::kHalf && st != at::kBFloat16) Py_RETURN_NONE;
    const int in = st == at::kHalf ? HBQ_DTYPE_F16 : HBQ_DTYPE_BF16, out = od < 0 ? in : (int)od;
    const c10::cuda::OptionalCUDAGuard guard(x->device());
    const at::Tensor deq = at::empty(x->sizes(), x->options().dtype(out == HBQ_DTYPE_F16 ? at::kHalf : at::kBFloat16));
    const int64_t K = x->size(-1), rows = x->numel() / K;
    const void* xp = x->data_ptr();
    void* dp = deq.data_ptr();
    void* stream = at::cuda::getCurrentCUDAStream(x->device().index()).stream();
    return result(unlocked([&] { return p_quantize(xp, in, rows, K, f, dp, out, nullptr, nullptr, stream); }), deq);
    END_HANDLE_TH_ERRORS
}

// gemm(a, b, mode, group_k, group_n, bias, b_is_nk): a [M, K] x b [N, K] or [K, N], fp16
PyObject* host_gemm(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int64_t mode, gk, gn, nk;
    if (n != 7 || !to_i64(args[2], &mode) || !to_i64(args[3], &gk) || !to_i64(args[4], &gn) || !to_i64(args[6], &nk)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "gemm(a, b, mode, group_k, group_n, bias, b_is_nk)");
        return nullptr;
    }
    const at::Tensor *a = plain_cuda(args[0]), *b = plain_cuda(args[1]);
    if (!a || !b || a->scalar_type() != at::kHalf || b->scalar_type() != at::kHalf || a->dim() != 2 || b->dim() != 2 ||
        a->device() != b->device())
        Py_RETURN_NONE;
    const int64_t M = a->size(0), K = a->size(1), N = b->size(nk ? 0 : 1);
    const void* bias;
    if (b->size(nk ? 1 : 0) != K || M == 0 || N == 0 || K == 0 || !plain_bias(args[5], *a, N, &bias)) Py_RETURN_NONE;
    const c10::cuda::OptionalCUDAGuard guard(a->device());
    const at::Tensor c = at::empty({M, N}, a->options());
    const int64_t wb = p_gemm_workspace_bytes(M, N, K, (int)nk, (int)mode, (int)gk, (int)gn);
    at::Tensor ws;
    if (wb > 0) ws = at::empty({wb}, a->options().dtype(at::kByte));
    const void *ap = a->data_ptr(), *bp = b->data_ptr();
    void *cp = c.data_ptr(), *wp = wb > 0 ? ws.data_ptr() : nullptr;
    void* stream = at::cuda::getCurrentCUDAStream(a->device().index()).stream();
    return result(unlocked([&] { return p_gemm(ap, bp, cp, M, N, K, (int)nk, (int)mode, (int)gk, (int)gn, bias, wp, wb, stream); }), c);
    END_HANDLE_TH_ERRORS
}

// gemm_w4(x, data, N, K, format, container_bits, bias, workspace): x [M, K] fp16 times a prepacked weight, into a new tensor
PyObject* host_gemm_w4(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    int64_t N, K, bits;
    if (n != 8 || !to_i64(args[2], &N) || !to_i64(args[3], &K) || !to_i64(args[5], &bits)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "gemm_w4(x, data, N, K, format, container_bits, bias, workspace)");
        return nullptr;
    }
    const hbq_format* f = to_format(args[4]);
    if (!f) return nullptr;
    const at::Tensor *x = plain_cuda(args[0]), *d = plain_cuda(args[1]), *ws = plain_cuda(args[7]);
    const void* bias;
    if (!x || !d || !ws || x->scalar_type() != at::kHalf || x->dim() != 2 || x->size(1) != K || x->size(0) == 0 ||
        x->device() != d->device() || ws->device() != d->device() || !plain_bias(args[6], *x, N, &bias))
        Py_RETURN_NONE;
    const int64_t M = x->size(0);
    const c10::cuda::OptionalCUDAGuard guard(x->device());
    const at::Tensor c = at::empty({M, N}, x->options());
    const void *xp = x->data_ptr(), *dp = d->data_ptr();
    void *cp = c.data_ptr(), *wp = ws->data_ptr();
    const int64_t wb = ws->numel();
    void* stream = at::cuda::getCurrentCUDAStream(x->device().index()).stream();
    return result(unlocked([&] { return p_gemm_w4(xp, dp, cp, M, N, K, f, (int)bits, bias, wp, wb, stream); }), c);
    END_HANDLE_TH_ERRORS
}

bool to_float(PyObject* o, float* v)
{
    const double d = PyFloat_AsDouble(o);
    *v = (float)d;
    return !(d == -1.0 && PyErr_Occurred());
}
bool records(const at::Tensor& t) { return t.requires_grad() && c10::GradMode::is_enabled(); }
bool half_type(const at::Tensor& t, int* dtype)
{
    const auto st = t.scalar_type();
    *dtype = st == at::kHalf ? HBQ_DTYPE_F16 : HBQ_DTYPE_BF16;
    return st == at::kHalf || st == at::kBFloat16;
}
// The last axis dense; strides of axes of one element do not matter and read as 0.
bool strides_of(const at::Tensor& t, int64_t* s)
{
    const int n = (int)t.dim() - 1;
    for (int i = 0; i < n; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    return t.size(n) == 1 || t.stride(n) == 1;
}

// x [T, H, D] or [B, T, H, D] of ordinary layout, and a new tensor for its result
bool heads_of(PyObject* o, const at::Tensor*& x, hbq_heads* h, int64_t* B, int64_t* T, int64_t* D)
{
    x = dense_cuda(o);
    if (!x || (x->dim() != 3 && x->dim() != 4) || x->numel() == 0 || records(*x)) return false;
    const int k = (int)x->dim() - 3;
    int64_t s[3] = {0, 0, 0};
    if (!strides_of(*x, s)) return false;
    *B = k ? x->size(0) : 1; *T = x->size(k); *D = x->size(k + 2);
    h->data = x->data_ptr();
    h->heads = x->size(k + 1);
    for (int i = 0; i < 3; ++i) h->stride[i] = i - 1 + k >= 0 ? s[i - 1 + k] : 0;
    h->out_stride[2] = *D; h->out_stride[1] = h->heads * *D; h->out_stride[0] = *T * h->heads * *D;
    return true;
}
bool rotary_of(PyObject* freq, PyObject* pos, PyObject* inter, PyObject* fac, const at::Tensor& x, int64_t B, int64_t T, int64_t D,
               hbq_rotary* r)
{
    const at::Tensor *f = plain_cuda(freq), *p = dense_cuda(pos);
    if (!f || !p || f->scalar_type() != at::kDouble || f->dim() != 1 || f->numel() == 0 || 2 * f->numel() > D || f->device() != x.device() ||
        p->device() != x.device() || records(*f))
        return false;
    const auto st = p->scalar_type();
    if ((st != at::kLong && st != at::kInt) || p->dim() < 1 || p->dim() > 2 || p->size(-1) != T || (p->dim() == 2 && p->size(0) != 1 && p->size(0) != B))
        return false;
    r->inv_freq = static_cast<const double*>(f->data_ptr());
    r->positions = p->data_ptr();
    r->positions_64 = st == at::kLong;
    r->pos_stride[0] = p->dim() == 2 && p->size(0) > 1 ? p->stride(0) : 0;
    r->pos_stride[1] = p->stride(-1);
    r->rot = (int32_t)(2 * f->numel());
    const int i = PyObject_IsTrue(inter);
    if (i < 0) { PyErr_Clear(); return false; }
    r->interleaved = i;
    if (!to_float(fac, &r->factor)) { PyErr_Clear(); return false; }
    return true;
}

// rope_rotate(x, inv_freq, positions, interleaved, factor): the turned heads, in a new tensor
PyObject* host_rope_rotate(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 5) { PyErr_SetString(PyExc_TypeError, "rope_rotate(x, inv_freq, positions, interleaved, factor)"); return nullptr; }
    const at::Tensor* x;
    hbq_heads h = {};
    hbq_rotary r = {};
    int64_t B, T, D;
    int dtype;
    if (!heads_of(args[0], x, &h, &B, &T, &D) || !half_type(*x, &dtype) || !rotary_of(args[1], args[2], args[3], args[4], *x, B, T, D, &r)) Py_RETURN_NONE;
    const c10::cuda::OptionalCUDAGuard guard(x->device());
    const at::Tensor out = at::empty(x->sizes(), x->options());
    h.out = out.data_ptr();
    void* stream = at::cuda::getCurrentCUDAStream(x->device().index()).stream();
    return result(unlocked([&] { return p_rope_rotate(&h, &r, dtype, B, T, D, stream); }), out);
    END_HANDLE_TH_ERRORS
}

// qk_norm_rope(q, k, q_weight, k_weight, eps, inv_freq, positions, interleaved, factor): the pair of normed and turned heads
PyObject* host_qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 9) { PyErr_SetString(PyExc_TypeError, "qk_norm_rope(q, k, q_weight, k_weight, eps, inv_freq, positions, interleaved, factor)"); return nullptr; }
    const at::Tensor* x[2];
    hbq_heads h[2] = {};
    hbq_rotary r = {};
    int64_t B[2], T[2], D[2];
    int dtype[2];
    float eps;
    for (int i = 0; i < 2; ++i) {
        if (!heads_of(args[i], x[i], &h[i], &B[i], &T[i], &D[i]) || !half_type(*x[i], &dtype[i])) Py_RETURN_NONE;
        const at::Tensor* w = plain_cuda(args[2 + i]);
        if (!w || w->scalar_type() != x[i]->scalar_type() || w->dim() != 1 || w->numel() != D[i] || w->device() != x[0]->device() || records(*w)) Py_RETURN_NONE;
        h[i].weight = w->data_ptr();
    }
    if (!to_float(args[4], &eps)) { PyErr_Clear(); Py_RETURN_NONE; }
    if (B[0] != B[1] || T[0] != T[1] || D[0] != D[1] || dtype[0] != dtype[1] || x[0]->dim() != x[1]->dim() || x[0]->device() != x[1]->device() ||
        !rotary_of(args[5], args[6], args[7], args[8], *x[0], B[0], T[0], D[0], &r))
        Py_RETURN_NONE;
    const c10::cuda::OptionalCUDAGuard guard(x[0]->device());
    const at::Tensor oq = at::empty(x[0]->sizes(), x[0]->options()), ok = at::empty(x[1]->sizes(), x[1]->options());
    h[0].out = oq.data_ptr(); h[1].out = ok.data_ptr();
    void* stream = at::cuda::getCurrentCUDAStream(x[0]->device().index()).stream();
    const int rc = unlocked([&] { return p_qk_norm_rope(&h[0], &h[1], &r, dtype[0], B[0], T[0], D[0], eps, stream); });
    if (rc) return PyLong_FromLong(rc);
    PyObject *a = THPVariable_Wrap(oq), *b = THPVariable_Wrap(ok);
    PyObject* both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
    Py_XDECREF(a); Py_XDECREF(b);
    return both;
    END_HANDLE_TH_ERRORS
}

// An optional int32 vector of B elements beside `like`
bool counts_of(PyObject* o, const at::Tensor& like, int64_t B, const int32_t** p)
{
    *p = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* t = plain_cuda(o);
    if (!t || t->scalar_type() != at::kInt || t->dim() != 1 || t->numel() != B || t->device() != like.device()) return false;
    *p = static_cast<const int32_t*>(t->data_ptr());
    return true;
}

// attention(q, k, v, prefix_k, prefix_v, window, sinks, scale, lengths, starts): a new tensor [B, L, H, D]
PyObject* host_attention(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    hbq_attention p = {};
    if (n != 10 || !to_i64(args[5], &p.window) || !to_i64(args[6], &p.sinks) || !to_float(args[7], &p.scale)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "attention(q, k, v, prefix_k, prefix_v, window, sinks, scale, lengths, starts)");
        return nullptr;
    }
    const at::Tensor *q = dense_cuda(args[0]), *k = dense_cuda(args[1]), *v = dense_cuda(args[2]);
    int dtype;
    if (!q || !k || !v || q->dim() != 4 || k->dim() != 4 || v->dim() != 4 || q->numel() == 0 || !half_type(*q, &dtype) ||
        k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->device() != q->device() || v->device() != q->device() ||
        records(*q) || records(*k) || records(*v) || k->sizes() != v->sizes())
        Py_RETURN_NONE;
    p.B = q->size(0); p.L = q->size(1); p.H = q->size(2); p.D = q->size(3); p.Hkv = k->size(1); p.S = k->size(2);
    if (k->size(0) != p.B || k->size(3) != p.D || p.Hkv == 0 || p.H % p.Hkv || !strides_of(*q, p.q_stride) || !strides_of(*k, p.k_stride) ||
        !strides_of(*v, p.v_stride) || !counts_of(args[8], *q, p.B, &p.lengths) || !counts_of(args[9], *q, p.B, &p.starts))
        Py_RETURN_NONE;
    p.q = q->data_ptr(); p.k = k->data_ptr(); p.v = v->data_ptr();
    p.dtype = dtype;
    if (args[3] != Py_None) {
        const at::Tensor *pk = dense_cuda(args[3]), *pv = dense_cuda(args[4]);
        if (!pk || !pv || pk->dim() != 3 || pk->sizes() != pv->sizes() || pk->size(0) != p.Hkv || pk->size(2) != p.D ||
            pk->scalar_type() != q->scalar_type() || pv->scalar_type() != q->scalar_type() || pk->device() != q->device() ||
            pv->device() != q->device() || records(*pk) || records(*pv) || !strides_of(*pk, p.pk_stride) || !strides_of(*pv, p.pv_stride))
            Py_RETURN_NONE;
        p.P = pk->size(1);
        p.prefix_k = pk->data_ptr(); p.prefix_v = pv->data_ptr();
    }
    const c10::cuda::OptionalCUDAGuard guard(q->device());
    const at::Tensor out = at::empty({p.B, p.L, p.H, p.D}, q->options());
    p.out = out.data_ptr();
    p.out_stride[2] = p.D; p.out_stride[1] = p.H * p.D; p.out_stride[0] = p.L * p.H * p.D;
    const int64_t wb = p_attention_workspace_bytes(&p);
    at::Tensor ws;
    if (wb > 0) ws = at::empty({wb}, q->options().dtype(at::kByte));
    void *wp = wb > 0 ? ws.data_ptr() : nullptr, *stream = at::cuda::getCurrentCUDAStream(q->device().index()).stream();
    return result(unlocked([&] { return p_attention_run(&p, wp, wb, stream); }), out);
    END_HANDLE_TH_ERRORS
}

// current_stream(device_index): the handle of torch's current stream there
PyObject* host_current_stream(PyObject*, PyObject* o)
{
    HANDLE_TH_ERRORS
    int64_t i;
    if (!to_i64(o, &i)) return nullptr;
    return PyLong_FromVoidPtr(at::cuda::getCurrentCUDAStream((c10::DeviceIndex)i).stream());
    END_HANDLE_TH_ERRORS
}

#define HBQ_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(host_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {HBQ_FAST(bind), HBQ_FAST(quantize), HBQ_FAST(gemm), HBQ_FAST(gemm_w4), HBQ_FAST(rope_rotate), HBQ_FAST(qk_norm_rope), HBQ_FAST(attention),
                         {"current_stream", host_current_stream, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "hbq_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_hbq_host() { return PyModule_Create(&module); }

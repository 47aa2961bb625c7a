// CPython fast paths of the tensor-level wrappers in ops.py: check, allocate, take the current stream, call the C ABI.
//
// A decoding program makes one such call per linear layer and token, and a call's kernel runs for 5 to 15 us; the
// wrappers written in Python (attribute checks, a device guard, a stream object, a ctypes call of a dozen arguments) took
// 15 to 20 us of host time each, so the device waited for the host. The functions here take the same tensors and do the
// same work in about 2 us plus the launch.
//
// Every function returns None when an operand is not in the plain form the kernels take (wrong type, device, layout or
// size, a tensor subclass, a shape without work): the Python wrapper then goes through its own checks, which raise what
// they always raised. An error of the library itself is raised as the binding's LatentQError.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/SavedTensorHooks.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/InferenceMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>

#include "../../include/latentq.h"

namespace {

PyObject *g_error = nullptr;  // LatentQError

constexpr c10::DispatchKeySet kWrappedKeys({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched,
                                            c10::DispatchKey::Functionalize, c10::DispatchKey::Python, c10::DispatchKey::ZeroTensor,
                                            c10::DispatchKey::Conjugate, c10::DispatchKey::Negative});

constexpr int64_t kWorkspaceBytes = 64 << 20;  // what ops.py keeps for each device, stream and host thread

// A plain tensor (Tensor or Parameter, no other subclass) on a GPU, contiguous, of the given type. The wrappers of function
// transforms (vmap, functional gradients, functionalisation) have the Python type of a plain tensor and no memory of their own.
const at::Tensor *plain(PyObject *o, at::ScalarType type) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.key_set().has_any(kWrappedKeys) || !t.has_storage()) return nullptr;
    return t.is_cuda() && t.scalar_type() == type && t.is_contiguous() ? &t : nullptr;
}

const at::Tensor *bf16(PyObject *o) { return plain(o, at::kBFloat16); }

// Packed codes of an [N, K] matrix
const at::Tensor *codes4(PyObject *o, int64_t N, int64_t K) {
    const at::Tensor *t = plain(o, at::kChar);
    if (!t) t = plain(o, at::kByte);
    return t && t->numel() == N * K / 2 ? t : nullptr;
}

const at::Tensor *sized(const at::Tensor *t, int64_t n) { return t && t->numel() == n ? t : nullptr; }

struct W4 {
    const at::Tensor *codes, *scales, *zeros;
    bool load(PyObject *const *o, int64_t N, int64_t K) {
        if (N <= 0 || K <= 0) return false;
        codes = codes4(o[0], N, K);
        scales = sized(bf16(o[1]), N * K / LQ_GROUP);
        zeros = sized(bf16(o[2]), N * K / LQ_GROUP);
        return codes && scales && zeros;
    }
};

int64_t integer(PyObject *o) { return PyLong_AsLongLong(o); }

// The wrapper is to look at the call. An argument that could not be converted has left its error, which the wrapper's own conversions
// and checks take the place of.
PyObject *none() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

PyObject *fail(const char *who, int rc) {
    PyErr_Format(g_error ? g_error : PyExc_RuntimeError, "%s failed (%d): %s", who, rc, lq_last_error());
    return nullptr;
}

// The device of `t` made current, and its current stream
struct On {
    c10::OptionalDeviceGuard guard;
    void *stream;
    explicit On(const at::Tensor &t) {
        guard.reset_device(t.device());
        stream = (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
    }
};

bool same_device(const at::Tensor *a, const at::Tensor *b) { return a->device() == b->device(); }

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &like) {
    return at::empty(shape, like.options().dtype(type));
}

// The shape of x with its last dimension replaced
at::Tensor make_rows(const at::Tensor &x, int64_t last, at::ScalarType type) {
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = last;
    return make(shape, type, x);
}

// Several results of a call in one allocation, each a tensor by itself: an allocation is a microsecond of the host's time. `at`: the bytes before it,
// moved past it; those of 8 bytes an element first.
at::Tensor take(const at::Tensor &bytes, int64_t &at, at::IntArrayRef shape, at::ScalarType type) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(bytes.storage()), bytes.key_set(), c10::scalarTypeToTypeMeta(type));
    const int64_t size = (int64_t)c10::elementSize(type);
    t.unsafeGetTensorImpl()->set_storage_offset(at / size);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    at += c10::multiply_integers(shape) * size;
    return t;
}

// Token rows of an operand whose last dimension is `width`: 0 if there are none or the width differs
int64_t rows_of(const at::Tensor *x, int64_t width) {
    return x && x->dim() >= 1 && width > 0 && x->size(-1) == width ? x->numel() / width : 0;
}

bool aligned16(const at::Tensor *t) { return ((uintptr_t)t->data_ptr() & 15) == 0; }

// A workspace argument: None, or bytes on the operand's device
bool workspace(PyObject *o, const at::Tensor *x, void **p, int64_t *bytes) {
    *p = nullptr;
    *bytes = 0;
    if (o == Py_None) return true;
    const at::Tensor *t = plain(o, at::kByte);
    if (!t || !same_device(t, x)) return false;
    *p = t->data_ptr();
    *bytes = t->numel();
    return true;
}

PyObject *wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

#define LQ_CALL(name, ...)                              \
    do {                                                \
        int rc_;                                        \
        Py_BEGIN_ALLOW_THREADS                          \
        rc_ = name(__VA_ARGS__);                        \
        Py_END_ALLOW_THREADS                            \
        if (rc_ != LQ_OK) return fail(#name, rc_);      \
    } while (0)

// bias argument: None, or bf16 [N]; false if it is neither
bool bias_of(PyObject *o, int64_t N, const void **p) {
    *p = nullptr;
    if (o == Py_None) return true;
    const at::Tensor *t = sized(bf16(o), N);
    if (!t) return false;
    *p = t->data_ptr();
    return true;
}

#define LQ_ARGS(n) \
    if (nargs != (n)) { PyErr_SetString(PyExc_TypeError, "wrong number of arguments"); return nullptr; }

// Whether something looks at calls that autograd itself does not: a trace being recorded, an open forward-mode level, an active
// function transform
bool watched() {
    const c10::DispatchKeySet included = c10::impl::tls_local_dispatch_key_set().included_;
    return torch::jit::tracer::isTracing() || torch::autograd::ForwardADLevel::try_get_by_idx(0) ||
           included.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) || included.has(c10::DispatchKey::FuncTorchDynamicLayerBackMode);
}

// x, codes, scales, zeros, N, K, bias, workspace -> y
PyObject *linear4(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(8)
    const int64_t N = integer(a[4]), K = integer(a[5]);
    const at::Tensor *x = bf16(a[0]);
    const int64_t M = rows_of(x, K);
    W4 w;
    const void *bias;
    void *ws;
    int64_t ws_bytes;
    if (M <= 0 || !w.load(a + 1, N, K) || !same_device(x, w.codes) || !bias_of(a[6], N, &bias) || !workspace(a[7], x, &ws, &ws_bytes))
        return none();
    On on(*x);
    at::Tensor y = make_rows(*x, N, at::kBFloat16);
    LQ_CALL(lq_a16w4_fwd_ws, x->data_ptr(), w.codes->data_ptr(), w.scales->data_ptr(), w.zeros->data_ptr(), bias, y.data_ptr(), M, N,
            K, LQ_GROUP, ws, ws_bytes, on.stream);
    return wrap(std::move(y));
}

// x, codes, scales, zeros, N, K, bias -> y, for a layer in inference: the whole call where nothing watches and the tokens
// are few enough to need no workspace
PyObject *linear4_eval(PyObject *self, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(7)
    const int64_t K = integer(a[5]);
    const at::Tensor *x = bf16(a[0]);
    if (!x || K <= 0 || x->numel() > 16 * K || watched()) return none();
    PyObject *all[8] = {a[0], a[1], a[2], a[3], a[4], a[5], a[6], Py_None};
    return linear4(self, all, 8);
}

// dy, codes, scales, zeros, N, K, workspace -> dx
PyObject *dx4(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(7)
    const int64_t N = integer(a[4]), K = integer(a[5]);
    const at::Tensor *dy = bf16(a[0]);
    const int64_t M = rows_of(dy, N);
    W4 w;
    void *ws;
    int64_t ws_bytes;
    if (M <= 0 || !w.load(a + 1, N, K) || !same_device(dy, w.codes) || !workspace(a[6], dy, &ws, &ws_bytes)) return none();
    On on(*dy);
    at::Tensor dx = make_rows(*dy, K, at::kBFloat16);
    LQ_CALL(lq_a16w4_dx_ws, dy->data_ptr(), w.codes->data_ptr(), w.scales->data_ptr(), w.zeros->data_ptr(), dx.data_ptr(), M, N, K,
            LQ_GROUP, ws, ws_bytes, on.stream);
    return wrap(std::move(dx));
}

// x, gate (codes, scales, zeros), up (codes, scales, zeros), N, K, save, workspace -> h, or (h, g, u)
PyObject *gate_up(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(11)
    const int64_t N = integer(a[7]), K = integer(a[8]);
    const bool save = a[9] == Py_True;
    const at::Tensor *x = bf16(a[0]);
    const int64_t M = rows_of(x, K);
    W4 g, u;
    void *ws;
    int64_t ws_bytes;
    if (M <= 0 || !g.load(a + 1, N, K) || !u.load(a + 4, N, K) || !same_device(x, g.codes) || !same_device(x, u.codes) ||
        !workspace(a[10], x, &ws, &ws_bytes))
        return none();
    On on(*x);
    at::Tensor h = make_rows(*x, N, at::kBFloat16), go, uo;
    if (save) go = make_rows(*x, N, at::kBFloat16), uo = make_rows(*x, N, at::kBFloat16);
    LQ_CALL(lq_a16w4_gate_up_silu_ws, x->data_ptr(), g.codes->data_ptr(), g.scales->data_ptr(), g.zeros->data_ptr(),
            u.codes->data_ptr(), u.scales->data_ptr(), u.zeros->data_ptr(), h.data_ptr(), save ? go.data_ptr() : nullptr,
            save ? uo.data_ptr() : nullptr, M, N, K, LQ_GROUP, ws, ws_bytes, on.stream);
    if (!save) return wrap(std::move(h));
    return Py_BuildValue("NNN", wrap(std::move(h)), wrap(std::move(go)), wrap(std::move(uo)));
}

// dy, codes, scales, zeros, N, K, g, u -> (dg, du)
PyObject *dx_silu(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(8)
    const int64_t N = integer(a[4]), K = integer(a[5]);
    const at::Tensor *dy = bf16(a[0]), *g = bf16(a[6]), *u = bf16(a[7]);
    const int64_t M = rows_of(dy, N);
    W4 w;
    if (M <= 0 || !w.load(a + 1, N, K) || !same_device(dy, w.codes) || rows_of(g, K) != M || rows_of(u, K) != M ||
        !same_device(dy, g) || !same_device(dy, u))
        return none();
    On on(*dy);
    at::Tensor dg = make_rows(*dy, K, at::kBFloat16), du = make_rows(*dy, K, at::kBFloat16);
    LQ_CALL(lq_a16w4_dx_silu_bwd, dy->data_ptr(), w.codes->data_ptr(), w.scales->data_ptr(), w.zeros->data_ptr(), g->data_ptr(),
            u->data_ptr(), dg.data_ptr(), du.data_ptr(), M, N, K, LQ_GROUP, on.stream);
    return Py_BuildValue("NN", wrap(std::move(dg)), wrap(std::move(du)));
}

// dy1, w1 (3), dy2, w2 (3), N, K, workspace -> dx
PyObject *dx_pair(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(11)
    const int64_t N = integer(a[8]), K = integer(a[9]);
    const at::Tensor *d1 = bf16(a[0]), *d2 = bf16(a[4]);
    const int64_t M = rows_of(d1, N);
    W4 w1, w2;
    void *ws;
    int64_t ws_bytes;
    if (M <= 0 || rows_of(d2, N) != M || !w1.load(a + 1, N, K) || !w2.load(a + 5, N, K) || !same_device(d1, w1.codes) ||
        !same_device(d1, d2) || !same_device(d1, w2.codes) || !workspace(a[10], d1, &ws, &ws_bytes))
        return none();
    On on(*d1);
    at::Tensor dx = make_rows(*d1, K, at::kBFloat16);
    LQ_CALL(lq_a16w4_dx_pair_ws, d1->data_ptr(), w1.codes->data_ptr(), w1.scales->data_ptr(), w1.zeros->data_ptr(), d2->data_ptr(),
            w2.codes->data_ptr(), w2.scales->data_ptr(), w2.zeros->data_ptr(), dx.data_ptr(), M, N, K, LQ_GROUP, ws,
            ws_bytes, on.stream);
    return wrap(std::move(dx));
}

// x8, w8, sx, sw (fp32 or bf16), bias -> y
PyObject *linear8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(5)
    const at::Tensor *x = plain(a[0], at::kChar), *w = plain(a[1], at::kChar), *sx = plain(a[2], at::kFloat), *sw = plain(a[3], at::kFloat);
    const bool fp32 = sw != nullptr;
    if (!sw) sw = bf16(a[3]);
    if (!x || !w || !sx || !sw || w->dim() != 2 || w->numel() == 0) return none();
    const int64_t N = w->size(0), K = w->size(1), M = rows_of(x, K);
    const void *bias;
    if (M <= 0 || sx->numel() != M || sw->numel() != N || !bias_of(a[4], N, &bias) || !same_device(x, w) || !same_device(x, sx) ||
        !same_device(x, sw))
        return none();
    On on(*x);
    at::Tensor y = make_rows(*x, N, at::kBFloat16);
    if (fp32)
        LQ_CALL(lq_a8w8_fwd, x->data_ptr(), w->data_ptr(), (const float *)sx->data_ptr(), (const float *)sw->data_ptr(), bias,
                y.data_ptr(), nullptr, M, N, K, on.stream);
    else
        LQ_CALL(lq_a8w8_fwd_qs, x->data_ptr(), w->data_ptr(), (const float *)sx->data_ptr(), sw->data_ptr(), bias, y.data_ptr(),
                nullptr, M, N, K, on.stream);
    return wrap(std::move(y));
}

// x, w8, qscales, bias, per_token -> y: the forward of an 8-bit layer in inference (quantise the activations, int8 product)
PyObject *infer8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(5)
    const at::Tensor *x = bf16(a[0]), *w = plain(a[1], at::kChar), *qs = bf16(a[2]);
    if (!x || !w || !qs || w->dim() != 2 || w->numel() == 0) return none();
    const int64_t N = w->size(0), K = w->size(1), M = rows_of(x, K);
    const void *bias;
    if (M <= 0 || K % 8 || qs->numel() != N || !bias_of(a[3], N, &bias) || !same_device(x, w) || !same_device(x, qs)) return none();
    On on(*x);
    at::Tensor y = make_rows(*x, N, at::kBFloat16);
    if (aligned16(x) && aligned16(w) && lq_a8w8_infer_takes(M, N, K)) {
        LQ_CALL(lq_a8w8_infer, x->data_ptr(), w->data_ptr(), qs->data_ptr(), bias, y.data_ptr(), a[4] == Py_True, M, N, K, on.stream);
        return wrap(std::move(y));
    }
    // what the quantiser leaves for the product, in one allocation: x8 [M, K], sx [M], the quantiser's scratch
    const int64_t at_sx = (M * K + 15) / 16 * 16, at_work = at_sx + (M * 4 + 15) / 16 * 16;
    at::Tensor scratch = make({at_work + LQ_ACT_WORK_FLOATS * 4}, at::kByte, *x);
    uint8_t *p = (uint8_t *)scratch.data_ptr();
    int8_t *x8 = (int8_t *)p;
    float *sx = (float *)(p + at_sx), *work = (float *)(p + at_work);
    if (a[4] == Py_True)
        LQ_CALL(lq_act_quant_i8_per_token, x->data_ptr(), x8, sx, M, K, on.stream);
    else
        LQ_CALL(lq_act_quant_i8_dynamic, x->data_ptr(), x8, sx, work, M, K, 0, on.stream);
    LQ_CALL(lq_a8w8_fwd_qs, x8, w->data_ptr(), sx, qs->data_ptr(), bias, y.data_ptr(), nullptr, M, N, K, on.stream);
    return wrap(std::move(y));
}

// The same for a layer in inference: None where something watches
PyObject *infer8_eval(PyObject *self, PyObject *const *a, Py_ssize_t nargs) {
    return watched() ? none() : infer8(self, a, nargs);
}

// dy, w8, qscales, workspace -> dx
PyObject *dx8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(4)
    const at::Tensor *dy = bf16(a[0]), *w = plain(a[1], at::kChar), *qs = bf16(a[2]);
    if (!dy || !w || !qs || w->dim() != 2 || w->numel() == 0) return none();
    const int64_t N = w->size(0), K = w->size(1), M = rows_of(dy, N);
    void *ws;
    int64_t ws_bytes;
    if (M <= 0 || qs->numel() != N || N % 64 || K % 128 || !aligned16(dy) || !aligned16(w) || !same_device(dy, w) || !same_device(dy, qs) ||
        !workspace(a[3], dy, &ws, &ws_bytes))
        return none();
    On on(*dy);
    at::Tensor dx = make_rows(*dy, K, at::kBFloat16);
    LQ_CALL(lq_a8w8_dx_ws, dy->data_ptr(), w->data_ptr(), qs->data_ptr(), dx.data_ptr(), M, N, K, ws, ws_bytes, on.stream);
    return wrap(std::move(dx));
}

// x, alpha_bf16 -> (x8, sx, work)
PyObject *quant8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(2)
    const at::Tensor *x = bf16(a[0]);
    if (!x || x->dim() != 2 || x->numel() == 0) return none();
    const int64_t M = x->size(0), K = x->size(1);
    On on(*x);
    at::Tensor x8 = make(x->sizes(), at::kChar, *x), sx = make({M}, at::kFloat, *x), work = make({LQ_ACT_WORK_FLOATS}, at::kFloat, *x);
    LQ_CALL(lq_act_quant_i8_dynamic, x->data_ptr(), (int8_t *)x8.data_ptr(), (float *)sx.data_ptr(), (float *)work.data_ptr(), M, K,
            a[1] == Py_True, on.stream);
    return Py_BuildValue("NNN", wrap(std::move(x8)), wrap(std::move(sx)), wrap(std::move(work)));
}

// x -> (x8, sx)
PyObject *quant8_token(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(1)
    const at::Tensor *x = bf16(a[0]);
    if (!x || x->dim() != 2 || x->numel() == 0 || x->size(1) % 8) return none();
    const int64_t M = x->size(0), K = x->size(1);
    On on(*x);
    at::Tensor x8 = make(x->sizes(), at::kChar, *x), sx = make({M}, at::kFloat, *x);
    LQ_CALL(lq_act_quant_i8_per_token, x->data_ptr(), (int8_t *)x8.data_ptr(), (float *)sx.data_ptr(), M, K, on.stream);
    return Py_BuildValue("NN", wrap(std::move(x8)), wrap(std::move(sx)));
}

// x8, scale, per_token -> x
PyObject *dequant8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(3)
    const at::Tensor *x8 = plain(a[0], at::kChar), *scale = plain(a[1], at::kFloat);
    if (!x8 || !scale || x8->dim() != 2 || x8->numel() == 0 || x8->size(1) % 16 || !aligned16(x8) || !same_device(x8, scale)) return none();
    const bool per_token = a[2] == Py_True;
    const int64_t M = x8->size(0), K = x8->size(1);
    if (scale->numel() != (per_token ? M : 1)) return none();
    On on(*x8);
    at::Tensor x = make(x8->sizes(), at::kBFloat16, *x8);
    LQ_CALL(lq_act_dequant_i8, (const int8_t *)x8->data_ptr(), (const float *)scale->data_ptr(), per_token, x.data_ptr(), M, K, on.stream);
    return wrap(std::move(x));
}

// The operands of a weight gradient: 2-D, the same tokens, sizes the GEMM takes
bool dw_operands(PyObject *const *a, const at::Tensor **dy, const at::Tensor **x, int k_mult) {
    *dy = bf16(a[0]);
    *x = bf16(a[1]);
    return *dy && *x && (*dy)->dim() == 2 && (*x)->dim() == 2 && (*dy)->size(0) == (*x)->size(0) && (*dy)->size(0) > 0 &&
           (*dy)->size(1) > 0 && (*dy)->size(1) % 8 == 0 && (*x)->size(1) > 0 && (*x)->size(1) % k_mult == 0 &&
           aligned16(*dy) && aligned16(*x) && same_device(*dy, *x);
}

// dy, x -> dW
PyObject *weight_grad(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(2)
    const at::Tensor *dy, *x;
    if (!dw_operands(a, &dy, &x, 8)) return none();
    const int64_t M = dy->size(0), N = dy->size(1), K = x->size(1);
    On on(*dy);
    at::Tensor dw = make({N, K}, at::kBFloat16, *dy);
    LQ_CALL(lq_weight_grad, dy->data_ptr(), x->data_ptr(), dw.data_ptr(), M, N, K, on.stream);
    return wrap(std::move(dw));
}

// dy, x, g -> g, dW added onto it
PyObject *weight_grad_acc(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(3)
    const at::Tensor *dy, *x, *g = bf16(a[2]);
    if (!dw_operands(a, &dy, &x, 8)) return none();
    const int64_t M = dy->size(0), N = dy->size(1), K = x->size(1);
    if (!g || g->dim() != 2 || g->size(0) != N || g->size(1) != K || !same_device(dy, g) || !aligned16(g)) return none();
    On on(*dy);
    LQ_CALL(lq_weight_grad_acc, dy->data_ptr(), x->data_ptr(), g->data_ptr(), M, N, K, on.stream);
    Py_INCREF(a[2]);
    return a[2];
}

// dy, x, q, scale, seed, offset -> q, dW added to the int8 accumulator
PyObject *weight_grad_acc8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(6)
    const at::Tensor *dy, *x, *q = plain(a[2], at::kChar), *scale = bf16(a[3]);
    if (!dw_operands(a, &dy, &x, 16)) return none();
    const int64_t M = dy->size(0), N = dy->size(1), K = x->size(1);
    if (!q || q->dim() != 2 || q->size(0) != N || q->size(1) != K || !sized(scale, N) || !same_device(dy, q) || !same_device(dy, scale))
        return none();
    const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[4]), offset = PyLong_AsUnsignedLongLongMask(a[5]);
    On on(*dy);
    LQ_CALL(lq_weight_grad_acc8, dy->data_ptr(), x->data_ptr(), (int8_t *)q->data_ptr(), scale->data_ptr(), M, N, K, nullptr, seed, offset,
            on.stream);
    Py_INCREF(a[2]);
    return a[2];
}

// dw, q, scale, accumulate, seed, offset -> q
PyObject *gradq8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(6)
    const at::Tensor *dw = bf16(a[0]), *q = plain(a[1], at::kChar), *scale = bf16(a[2]);
    if (!dw || dw->dim() != 2 || dw->numel() == 0 || !q || q->sizes() != dw->sizes() || !sized(scale, dw->size(0)) ||
        !same_device(dw, q) || !same_device(dw, scale))
        return none();
    const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[4]), offset = PyLong_AsUnsignedLongLongMask(a[5]);
    On on(*dw);
    LQ_CALL(lq_gradq8_quant, dw->data_ptr(), (int8_t *)q->data_ptr(), scale->data_ptr(), a[3] == Py_True, dw->size(0), dw->size(1),
            nullptr, seed, offset, on.stream);
    Py_INCREF(a[1]);
    return a[1];
}

// The operands every form of the optimizer step shares: grad, state1, state2, scale1, max1, scale2, max2
struct Adam {
    const at::Tensor *grad, *s1, *s2, *blocks[4];
    float *f[4];
    int64_t n, block;
    bool load(PyObject *const *o) {
        grad = bf16(o[0]);
        if (!grad || grad->numel() == 0) return false;
        n = grad->numel();
        s1 = sized(plain(o[1], at::kByte), n);
        s2 = sized(plain(o[2], at::kByte), n);
        if (!s1 || !s2 || !same_device(grad, s1) || !same_device(grad, s2)) return false;
        int64_t nblk = 0;
        for (int i = 0; i < 4; ++i) {
            const at::Tensor *t = plain(o[3 + i], at::kFloat);
            if (!t || !same_device(grad, t) || (i ? t->numel() != nblk : (nblk = t->numel()) == 0)) return false;
            blocks[i] = t;
            f[i] = (float *)t->data_ptr();
        }
        block = n / nblk;
        return n % nblk == 0;
    }
    uint8_t *p1() const { return (uint8_t *)s1->data_ptr(); }
    uint8_t *p2() const { return (uint8_t *)s2->data_ptr(); }
};

bool doubles(PyObject *const *o, double *v, int n) {
    for (int i = 0; i < n; ++i) {
        v[i] = PyFloat_AsDouble(o[i]);
        if (v[i] == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            return false;
        }
    }
    return true;
}

// grad, state1, state2, scale1, max1, scale2, max2, beta1, beta2, eps, step_size, param -> param
PyObject *adam8_param(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(12)
    Adam s;
    double v[4];
    const at::Tensor *p = bf16(a[11]);
    if (!s.load(a) || !doubles(a + 7, v, 4) || !sized(p, s.n) || !same_device(p, s.grad)) return none();
    On on(*s.grad);
    LQ_CALL(lq_adam8_update, s.grad->data_ptr(), p->data_ptr(), nullptr, s.p1(), s.p2(), s.f[0], s.f[1], s.f[2], s.f[3], s.n, (int)s.block,
            v[0], v[1], v[2], v[3], on.stream);
    Py_INCREF(a[11]);
    return a[11];
}

// Steps of several parameters that one launch will run: what is queued, on which stream, and the tensors it works on
#define ADAM_STATE(s) (s).s1, (s).s2, (s).blocks[0], (s).blocks[1], (s).blocks[2], (s).blocks[3]
struct AdamQueue {
    void *items = nullptr;
    void *stream = nullptr;
    c10::Device device{c10::kCPU};
    std::vector<at::Tensor> keep;
    ~AdamQueue() { lq_adam8_queue_free(items); }
    static constexpr const char *kName = "adam8_queue";

    // The queue to append to, or null to run the step now: no queue given, or one of another stream or device. The tensors
    // stay referenced until the queue is run.
    static void *take(PyObject *o, const On &on, const at::Tensor &like, std::initializer_list<const at::Tensor *> used) {
        if (!PyCapsule_IsValid(o, kName)) return nullptr;
        AdamQueue *q = static_cast<AdamQueue *>(PyCapsule_GetPointer(o, kName));
        if (q->keep.empty()) {
            q->stream = on.stream;
            q->device = like.device();
        }
        if (q->stream != on.stream || q->device != like.device()) return nullptr;
        for (const at::Tensor *t : used) q->keep.push_back(*t);
        return q->items;
    }
};

// -> a queue
PyObject *adam8_queue(PyObject *, PyObject *const *, Py_ssize_t nargs) {
    LQ_ARGS(0)
    AdamQueue *q = new AdamQueue;
    if (lq_adam8_queue_new(&q->items) != LQ_OK) {
        delete q;
        return PyErr_NoMemory();
    }
    PyObject *o = PyCapsule_New(q, AdamQueue::kName, [](PyObject *c) { delete static_cast<AdamQueue *>(PyCapsule_GetPointer(c, AdamQueue::kName)); });
    if (!o) delete q;
    return o;
}

// queue ->: runs what is in it
PyObject *adam8_run(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(1)
    AdamQueue *q = static_cast<AdamQueue *>(PyCapsule_GetPointer(a[0], AdamQueue::kName));
    if (!q) return nullptr;
    if (q->keep.empty()) return none();
    c10::OptionalDeviceGuard guard(q->device);
    std::vector<at::Tensor> keep;  // until the launches are out
    keep.swap(q->keep);
    LQ_CALL(lq_adam8_queue_run, q->items, q->stream);
    return none();
}

// grad ... max2, beta1, beta2, eps, step_size, codes, scales, zeros, N, K, seed, offset, queue -> new codes
PyObject *adam8_sr(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(19)
    Adam s;
    double v[4];
    const int64_t N = integer(a[14]), K = integer(a[15]);
    W4 w;
    if (!s.load(a) || !doubles(a + 7, v, 4) || !w.load(a + 11, N, K) || s.n != N * K || !same_device(s.grad, w.codes)) return none();
    const uint64_t seed = PyLong_AsUnsignedLongLongMask(a[16]), offset = PyLong_AsUnsignedLongLongMask(a[17]);
    On on(*s.grad);
    at::Tensor out = at::empty_like(*w.codes);
    void *queue = AdamQueue::take(a[18], on, *s.grad, {s.grad, w.codes, &out, w.scales, w.zeros, ADAM_STATE(s)});
    LQ_CALL(lq_adam8_sr_step_queued, s.grad->data_ptr(), w.codes->data_ptr(), out.data_ptr(), w.scales->data_ptr(), w.zeros->data_ptr(), s.p1(),
            s.p2(), s.f[0], s.f[1], s.f[2], s.f[3], N, K, LQ_GROUP, (int)s.block, v[0], v[1], v[2], v[3], seed, offset, on.stream, queue);
    return wrap(std::move(out));
}

// (k1, b1, k2, b2, k3) of a residual curve
struct Curve {
    int k1, k2, k3;
    float b1, b2;
    bool load(PyObject *o) {
        if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 5) return false;
        double v[5];
        for (int i = 0; i < 5; ++i) {
            PyObject *e = PyTuple_GET_ITEM(o, i);
            if (!doubles(&e, v + i, 1)) return false;
        }
        k1 = (int)v[0]; k2 = (int)v[2]; k3 = (int)v[4];
        b1 = (float)v[1]; b2 = (float)v[3];
        return true;
    }
};

// grad ... max2, beta1, beta2, eps, step_size, codes, scales, zeros, N, K, residual, dequant curve, quant curve, queue -> codes
PyObject *adam8_w4(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(20)
    Adam s;
    double v[4];
    const int64_t N = integer(a[14]), K = integer(a[15]);
    W4 w;
    Curve d, q;
    const at::Tensor *r = plain(a[16], at::kInt);
    if (!s.load(a) || !doubles(a + 7, v, 4) || !w.load(a + 11, N, K) || s.n != N * K || !sized(r, N * K / 8) || !d.load(a[17]) ||
        !q.load(a[18]) || !same_device(s.grad, w.codes) || !same_device(s.grad, r))
        return none();
    On on(*s.grad);
    void *queue = AdamQueue::take(a[19], on, *s.grad, {s.grad, w.codes, r, w.scales, w.zeros, ADAM_STATE(s)});
    LQ_CALL(lq_adam8_latent_w4_step_queued, s.grad->data_ptr(), w.codes->data_ptr(), (int32_t *)r->data_ptr(), w.scales->data_ptr(),
            w.zeros->data_ptr(), s.p1(), s.p2(), s.f[0], s.f[1], s.f[2], s.f[3], N, K, LQ_GROUP, (int)s.block, d.k1, d.b1, d.k2, d.b2,
            d.k3, q.k1, q.b1, q.k2, q.b2, q.k3, v[0], v[1], v[2], v[3], on.stream, queue);
    Py_INCREF(a[11]);
    return a[11];
}

// grad ... max2, beta1, beta2, eps, step_size, codes, qscales, residual, dequant curve, quant curve, queue -> codes
PyObject *adam8_w8(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(17)
    Adam s;
    double v[4];
    Curve d, q;
    const at::Tensor *c = plain(a[11], at::kChar), *qs = bf16(a[12]), *r = plain(a[13], at::kInt);
    if (!s.load(a) || !doubles(a + 7, v, 4) || !c || c->dim() != 2 || c->numel() != s.n || c->size(1) % 8 || !sized(qs, c->size(0)) ||
        !sized(r, s.n / 8) || !d.load(a[14]) || !q.load(a[15]) || !same_device(s.grad, c) || !same_device(s.grad, qs) || !same_device(s.grad, r))
        return none();
    On on(*s.grad);
    void *queue = AdamQueue::take(a[16], on, *s.grad, {s.grad, c, r, qs, ADAM_STATE(s)});
    LQ_CALL(lq_adam8_latent_w8_step_queued, s.grad->data_ptr(), (int8_t *)c->data_ptr(), (int32_t *)r->data_ptr(), qs->data_ptr(), s.p1(), s.p2(),
            s.f[0], s.f[1], s.f[2], s.f[3], c->size(0), c->size(1), (int)s.block, d.k1, d.b1, d.k2, d.b2, d.k3, q.k1, q.b1, q.k2, q.b2,
            q.k3, v[0], v[1], v[2], v[3], on.stream, queue);
    Py_INCREF(a[11]);
    return a[11];
}

// ---- paged 8-bit cache of keys and values
// Its calls have no derivative: an operand that requires a gradient, and any call under an open forward-mode level, are the wrapper's,
// which refuses those that would lose one.
bool wants_gradient(const at::Tensor *t) { return t->requires_grad() && c10::GradMode::is_enabled(); }

// Rows [tokens, heads, dim] of a 16-bit type in the strides the kernels take, without a gradient to keep
struct Rows16 {
    const at::Tensor *t = nullptr;
    int dtype = 0;  // as the C entry points number them
    bool load(PyObject *o) {
        if (!THPVariable_CheckExact(o)) return false;
        const at::Tensor &x = THPVariable_Unpack(o);
        const bool f16 = x.scalar_type() == at::kHalf;
        if (!x.is_cuda() || (!f16 && x.scalar_type() != at::kBFloat16) || x.dim() != 3 || x.numel() == 0 || !x.has_storage()) return false;
        if (x.key_set().has_any(kWrappedKeys) || x.stride(2) != 1 || x.stride(0) % 8 || x.stride(1) % 8 || !aligned16(&x)) return false;
        if (wants_gradient(&x)) return false;
        t = &x;
        dtype = f16;
        return true;
    }
    // rows of their own, to be written: the heads of a token beside each other, or the tokens of a head (the wrapper looks at others)
    bool separate() const {
        const auto within = [this](int inner, int outer) {
            return (t->size(inner) == 1 || t->stride(inner) >= t->size(2)) && (t->size(outer) == 1 || t->stride(outer) >= t->stride(inner) * (t->size(inner) - 1) + t->size(2));
        };
        return within(1, 0) || within(0, 1);
    }
};

struct Cache8 {
    const at::Tensor *kc, *vc, *ks, *vs;
    int64_t blocks, heads, dim;
    bool load(PyObject *const *a) {
        kc = plain(a[0], at::kByte);
        vc = plain(a[1], at::kByte);
        ks = plain(a[2], at::kFloat);
        vs = plain(a[3], at::kFloat);
        if (!kc || !vc || !ks || !vs || kc->dim() != 4 || vc->dim() != 5 || ks->dim() != 2 || vs->dim() != 2) return false;
        blocks = kc->size(0);
        heads = kc->size(1);
        dim = kc->size(3);
        return blocks > 0 && heads > 0 && kc->size(2) == LQ_KV_BLOCK && (dim == 64 || dim == 96 || dim == 128 || dim == 256) &&
               vc->sizes() == at::IntArrayRef({blocks, heads, LQ_KV_BLOCK / 4, dim, 4}) && ks->sizes() == at::IntArrayRef({blocks, heads}) &&
               vs->sizes() == ks->sizes() && same_device(kc, vc) && same_device(kc, ks) && same_device(kc, vs) && aligned16(kc) && aligned16(vc) && !wants_gradient(ks) &&
               !wants_gradient(vs);
    }
};

// block_table, seq_lens; cu_tokens and max_tokens (None: what the rows allow)
struct Sequences {
    const at::Tensor *table, *lens;
    const int32_t *cu = nullptr;
    int64_t batch, width, most;
    bool load(PyObject *o_table, PyObject *o_lens, PyObject *o_cu, PyObject *o_most, int64_t tokens, const at::Tensor *like) {
        table = plain(o_table, at::kInt);
        lens = plain(o_lens, at::kInt);
        if (!table || !lens || table->dim() != 2 || lens->dim() != 1 || !same_device(table, like) || !same_device(lens, like)) return false;
        batch = table->size(0);
        width = table->size(1);
        if (batch == 0 || width == 0 || lens->size(0) != batch) return false;
        most = tokens;
        if (o_cu != Py_None) {
            const at::Tensor *c = plain(o_cu, at::kInt);
            if (!c || c->dim() != 1 || c->size(0) != batch + 1 || !same_device(c, like)) return false;
            cu = (const int32_t *)c->data_ptr();
        } else {
            if (tokens % batch) return false;
            most = tokens / batch;
        }
        if (o_most == Py_None) return true;
        const int64_t given = integer(o_most);
        if (given <= 0 || (!cu && given < most)) return false;
        most = std::min(most, given);
        return true;
    }
};

// k, v, cache (4), block_table, seq_lens, q, cos, sin, cu_tokens, max_tokens, q_out -> the rotated q, or True without one
PyObject *kv8_append(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(14)
    if (watched()) return none();
    Rows16 k, v, q, o;
    Cache8 c;
    Sequences s;
    const bool with_q = a[8] != Py_None, rotates = a[9] != Py_None;
    if (!k.load(a[0]) || !v.load(a[1]) || !c.load(a + 2) || !same_device(k.t, c.kc) || !same_device(v.t, c.kc) || k.dtype != v.dtype ||
        k.t->size(1) != c.heads || k.t->size(2) != c.dim || v.t->sizes() != k.t->sizes() || rotates != (a[10] != Py_None) || (with_q && !rotates) ||
        (!with_q && a[13] != Py_None))
        return none();
    const int64_t tokens = k.t->size(0);
    if (!s.load(a[6], a[7], a[11], a[12], tokens, c.kc)) return none();
    const at::Tensor *cos = rotates ? plain(a[9], at::kFloat) : nullptr, *sin = rotates ? plain(a[10], at::kFloat) : nullptr;
    if (rotates && (!cos || !sin || cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->numel() == 0 || cos->size(1) % 8 || 2 * cos->size(1) > c.dim ||
                    !same_device(cos, c.kc) || !same_device(sin, c.kc) || !aligned16(cos) || !aligned16(sin) || wants_gradient(cos) || wants_gradient(sin)))
        return none();
    if (with_q && (!q.load(a[8]) || !same_device(q.t, c.kc) || q.dtype != k.dtype || q.t->size(0) != tokens || q.t->size(2) != c.dim)) return none();
    if (a[13] != Py_None && (!o.load(a[13]) || !same_device(o.t, c.kc) || o.dtype != k.dtype || o.t->sizes() != q.t->sizes() || !o.separate())) return none();
    On on(*c.kc);
    at::Tensor made;
    if (with_q && !o.t) {
        made = make(q.t->sizes(), q.t->scalar_type(), *q.t);
        o.t = &made;
    }
    LQ_CALL(lq_kv8_append, k.t->data_ptr(), k.t->stride(0), k.t->stride(1), v.t->data_ptr(), v.t->stride(0), v.t->stride(1),
            with_q ? q.t->data_ptr() : nullptr, with_q ? q.t->stride(0) : 0, with_q ? q.t->stride(1) : 0, with_q ? o.t->data_ptr() : nullptr,
            with_q ? o.t->stride(0) : 0, with_q ? o.t->stride(1) : 0, rotates ? (const float *)cos->data_ptr() : nullptr,
            rotates ? (const float *)sin->data_ptr() : nullptr, rotates ? cos->size(0) : 0, rotates ? (int)(2 * cos->size(1)) : 0, c.kc->data_ptr(),
            c.vc->data_ptr(), (float *)c.ks->data_ptr(), (float *)c.vs->data_ptr(), c.blocks, (const int32_t *)s.table->data_ptr(), s.width,
            (const int32_t *)s.lens->data_ptr(), s.cu, s.batch, tokens, s.most, with_q ? (int)q.t->size(1) : 0, (int)c.heads, (int)c.dim, k.dtype, on.stream);
    if (!with_q) Py_RETURN_TRUE;
    if (made.defined()) return wrap(std::move(made));
    Py_INCREF(a[13]);
    return a[13];
}

// What attention writes: the caller's rows (o, from an operand that is not None), or some that are made
bool given_rows(PyObject *o_out, Rows16 &o, const Rows16 &q) {
    return o_out == Py_None || (o.load(o_out) && same_device(o.t, q.t) && o.dtype == q.dtype && o.t->sizes() == q.t->sizes() && o.separate());
}
PyObject *attended(PyObject *o_out, at::Tensor &made, at::Tensor &lse) {
    PyObject *out = o_out;
    if (made.defined()) out = wrap(std::move(made));
    else Py_INCREF(out);
    return lse.defined() ? Py_BuildValue("NN", out, wrap(std::move(lse))) : out;
}

// q, cache (4), block_table, seq_lens, cu_tokens, max_tokens, max_len, scale, causal, window, return_lse, out, workspace -> out, or (out, lse);
// without a workspace where one is wanted: its bytes, and nothing is done
PyObject *kv8_attention(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(16)
    if (watched()) return none();
    Rows16 q, o;
    Cache8 c;
    Sequences s;
    if (!q.load(a[0]) || !c.load(a + 1) || !same_device(q.t, c.kc) || q.t->size(2) != c.dim || q.t->size(1) % c.heads) return none();
    const int64_t tokens = q.t->size(0), heads = q.t->size(1);
    if (!s.load(a[5], a[6], a[7], a[8], tokens, c.kc)) return none();
    int64_t max_len = s.width * LQ_KV_BLOCK;
    if (a[9] != Py_None) {
        const int64_t given = integer(a[9]);
        if (given < 0) return none();
        max_len = std::min(max_len, given);
    }
    const double scale = a[10] == Py_None ? 1.0 / std::sqrt((double)c.dim) : PyFloat_AsDouble(a[10]);
    const int64_t window = a[12] == Py_None ? 0 : integer(a[12]);
    const int causal = PyObject_IsTrue(a[11]), with_lse = PyObject_IsTrue(a[13]);
    if (PyErr_Occurred() || !(scale > 0.0 && scale <= 3.4e38) || window < 0) return none();
    void *ws;
    int64_t ws_bytes;
    if (!given_rows(a[14], o, q) || !workspace(a[15], q.t, &ws, &ws_bytes)) return none();
    On on(*c.kc);
    if (!ws) {
        int kernel, parts;
        int64_t needed;
        const bool ahead = window && !causal;
        if (const int rc = lq_kv8_attention_plan(s.batch, tokens, s.most, ahead ? std::min(max_len, window + s.most + LQ_KV_BLOCK) : max_len, (int)heads, (int)c.heads,
                                                 (int)c.dim, ahead ? 0 : window, kWorkspaceBytes, 0, &kernel, &parts, &needed))
            return fail("lq_kv8_attention_plan", rc);
        if (needed) return PyLong_FromLongLong(needed);
    }
    at::Tensor made, lse;
    if (!o.t) {
        made = make(q.t->sizes(), q.t->scalar_type(), *q.t);
        o.t = &made;
    }
    if (with_lse) lse = make({tokens, heads}, at::kFloat, *q.t);
    LQ_CALL(lq_kv8_attention, q.t->data_ptr(), q.t->stride(0), q.t->stride(1), c.kc->data_ptr(), c.vc->data_ptr(), (const float *)c.ks->data_ptr(),
            (const float *)c.vs->data_ptr(), c.blocks, (const int32_t *)s.table->data_ptr(), s.width, (const int32_t *)s.lens->data_ptr(), s.cu, s.batch, tokens,
            s.most, max_len, (int)heads, (int)c.heads, (int)c.dim, q.dtype, (float)scale, causal, window, o.t->data_ptr(), o.t->stride(0), o.t->stride(1),
            with_lse ? (float *)lse.data_ptr() : nullptr, ws, ws_bytes, on.stream);
    return attended(a[14], made, lse);
}

// q, cache (4), block_table, seq_lens, shared, cu_tokens, max_tokens, max_len, scale, causal, return_lse, out -> out, or (out, lse)
PyObject *kv8_attention_shared(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(15)
    if (watched()) return none();
    Rows16 q, o;
    Cache8 c;
    Sequences s;
    if (!q.load(a[0]) || !c.load(a + 1) || !same_device(q.t, c.kc) || q.t->size(2) != c.dim || q.t->size(1) % c.heads) return none();
    const int64_t tokens = q.t->size(0), heads = q.t->size(1);
    if (!s.load(a[5], a[6], a[8], a[9], tokens, c.kc)) return none();
    const int64_t shared = integer(a[7]), room = s.width * LQ_KV_BLOCK;
    int64_t max_len = INT64_MAX;  // (not known)
    if (a[10] != Py_None) {
        const int64_t given = integer(a[10]);
        if (given < 0) return none();
        if (given <= room) max_len = given;
    }
    const double scale = a[11] == Py_None ? 1.0 / std::sqrt((double)c.dim) : PyFloat_AsDouble(a[11]);
    const int causal = PyObject_IsTrue(a[12]), with_lse = PyObject_IsTrue(a[13]);
    if (PyErr_Occurred() || !(scale > 0.0 && scale <= 3.4e38) || shared < 0 || shared > s.width || !given_rows(a[14], o, q)) return none();
    On on(*c.kc);
    int prefix, own;
    int64_t needed;
    if (const int rc = lq_kv8_attention_shared_plan(s.batch, tokens, s.most, max_len, (int)heads, (int)c.heads, (int)c.dim, shared, kWorkspaceBytes, 0, &prefix, &own, &needed))
        return fail("lq_kv8_attention_shared_plan", rc);
    if (!prefix)
        if (const int rc = lq_kv8_attention_plan(s.batch, tokens, s.most, std::min(max_len, room), (int)heads, (int)c.heads, (int)c.dim, 0, kWorkspaceBytes, 0, &prefix, &own, &needed))
            return fail("lq_kv8_attention_plan", rc);
    at::Tensor ws;
    if (needed) ws = make({needed}, at::kByte, *q.t);
    at::Tensor made, lse;
    if (!o.t) {
        made = make(q.t->sizes(), q.t->scalar_type(), *q.t);
        o.t = &made;
    }
    if (with_lse) lse = make({tokens, heads}, at::kFloat, *q.t);
    LQ_CALL(lq_kv8_attention_shared, q.t->data_ptr(), q.t->stride(0), q.t->stride(1), c.kc->data_ptr(), c.vc->data_ptr(), (const float *)c.ks->data_ptr(),
            (const float *)c.vs->data_ptr(), c.blocks, (const int32_t *)s.table->data_ptr(), s.width, (const int32_t *)s.lens->data_ptr(), s.cu, s.batch, tokens,
            s.most, max_len, shared, (int)heads, (int)c.heads, (int)c.dim, q.dtype, (float)scale, causal, o.t->data_ptr(), o.t->stride(0), o.t->stride(1),
            with_lse ? (float *)lse.data_ptr() : nullptr, needed ? ws.data_ptr() : nullptr, needed, on.stream);
    return attended(a[14], made, lse);
}

// cache (4), blocks, dtype as the C entry points number them -> (k, v)
PyObject *kv8_read(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(6)
    if (watched()) return none();
    Cache8 c;
    const at::Tensor *b = plain(a[4], at::kInt);
    const int64_t dtype = integer(a[5]);
    if (!c.load(a) || !b || b->dim() != 1 || b->numel() == 0 || !same_device(b, c.kc) || dtype < 0 || dtype > 2) return none();
    On on(*c.kc);
    const at::ScalarType type = dtype == 0 ? at::kBFloat16 : dtype == 1 ? at::kHalf : at::kFloat;
    at::Tensor k = make({b->numel(), LQ_KV_BLOCK, c.heads, c.dim}, type, *c.kc), v = make(k.sizes(), type, *c.kc);
    LQ_CALL(lq_kv8_read, c.kc->data_ptr(), c.vc->data_ptr(), (const float *)c.ks->data_ptr(), (const float *)c.vs->data_ptr(), c.blocks,
            (const int32_t *)b->data_ptr(), b->numel(), (int)c.heads, (int)c.dim, (int)dtype, k.data_ptr(), v.data_ptr(), on.stream);
    return Py_BuildValue("NN", wrap(std::move(k)), wrap(std::move(v)));
}

// block_table, seq_lens, free_blocks, free_count, change, rows (None: no positions and slots), shared -> (cu_tokens, positions, slots, status)
PyObject *kv8_resize(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(7)
    if (watched()) return none();
    const at::Tensor *t[5];
    for (int i = 0; i < 5; ++i) {
        t[i] = plain(a[i], at::kInt);
        if (!t[i] || !same_device(t[i], t[0])) return none();
    }
    if (t[0]->dim() != 2 || t[0]->numel() == 0 || t[1]->dim() != 1 || t[2]->dim() != 1 || t[3]->sizes() != at::IntArrayRef({1}) || t[4]->sizes() != t[1]->sizes() ||
        t[1]->size(0) != t[0]->size(0))
        return none();
    const int64_t batch = t[0]->size(0), rows = a[5] == Py_None ? -1 : integer(a[5]), shared = integer(a[6]);
    if (PyErr_Occurred() || (a[5] != Py_None && rows < 0) || rows > INT32_MAX || shared < 0 || shared > t[0]->size(1)) return none();
    On on(*t[0]);
    const int64_t n = std::max(rows, (int64_t)0);
    const at::Tensor all = make({16 * n + 4 * (batch + 2)}, at::kByte, *t[0]);
    int64_t at = 0;
    at::Tensor positions, slots;
    if (rows >= 0) {
        positions = take(all, at, {rows}, at::kLong);
        slots = take(all, at, {rows}, at::kLong);
    }
    at::Tensor cu = take(all, at, {batch + 1}, at::kInt), status = take(all, at, {1}, at::kInt);
    LQ_CALL(lq_kv8_resize, (int32_t *)t[0]->data_ptr(), t[0]->size(1), (int32_t *)t[1]->data_ptr(), (int32_t *)t[2]->data_ptr(), t[2]->size(0), (int32_t *)t[3]->data_ptr(),
            (const int32_t *)t[4]->data_ptr(), batch, shared, rows, (int32_t *)cu.data_ptr(), rows >= 0 ? (int64_t *)positions.data_ptr() : nullptr,
            rows >= 0 ? (int64_t *)slots.data_ptr() : nullptr, (int32_t *)status.data_ptr(), on.stream);
    if (rows < 0) return Py_BuildValue("NOON", wrap(std::move(cu)), Py_None, Py_None, wrap(std::move(status)));
    return Py_BuildValue("NNNN", wrap(std::move(cu)), wrap(std::move(positions)), wrap(std::move(slots)), wrap(std::move(status)));
}

// Rows [rows, vocab] of logits with their entries beside each other
struct Logits {
    const at::Tensor *t = nullptr;
    int dtype = 0;
    bool load(PyObject *o) {
        if (!THPVariable_CheckExact(o)) return false;
        const at::Tensor &x = THPVariable_Unpack(o);
        if (!x.is_cuda() || x.dim() != 2 || x.numel() == 0 || !x.has_storage() || x.key_set().has_any(kWrappedKeys) || x.stride(1) != 1) return false;
        dtype = x.scalar_type() == at::kBFloat16 ? 0 : x.scalar_type() == at::kHalf ? 1 : x.scalar_type() == at::kFloat ? 2 : -1;
        t = &x;
        return dtype >= 0;
    }
};

// logits, tokens, cu_tokens, draft_logits, accept_draws, sample_draws (None or tensors), temperature, batch, max_tokens (None), change (None or a tensor) -> (out, accepted)
PyObject *verify_drafts(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(10)
    if (watched()) return none();
    Logits l, d;
    const at::Tensor *tokens = plain(a[1], at::kLong), *cu = nullptr, *accept = nullptr, *sample = nullptr, *change = nullptr;
    if (!l.load(a[0]) || !tokens || !same_device(tokens, l.t)) return none();
    const int64_t rows = l.t->size(0), vocab = l.t->size(1);
    if (tokens->sizes() != at::IntArrayRef({rows}) || rows > 65535) return none();
    int64_t batch = rows;
    if (a[2] != Py_None) {
        cu = plain(a[2], at::kInt);
        if (!cu || cu->dim() != 1 || cu->size(0) < 2 || !same_device(cu, l.t) || a[7] != Py_None) return none();
        batch = cu->size(0) - 1;
    } else if (a[7] != Py_None) {
        batch = integer(a[7]);
        if (batch <= 0 || rows % batch) return none();
    }
    int64_t most = cu ? rows : rows / batch;
    if (a[8] != Py_None) {
        const int64_t given = integer(a[8]);
        if (given <= 0 || (!cu && given < most)) return none();
        most = std::min(most, given);
    }
    const double temperature = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred() || !(temperature == 0.0 || (temperature >= 0x1p-60 && temperature <= 0x1p60))) return none();
    const bool draws = temperature != 0.0;
    if (a[3] != Py_None && (!d.load(a[3]) || d.dtype != l.dtype || d.t->sizes() != l.t->sizes() || !same_device(d.t, l.t))) return none();
    if (a[4] != Py_None && (!(accept = plain(a[4], at::kFloat)) || accept->sizes() != at::IntArrayRef({rows}) || !same_device(accept, l.t))) return none();
    if (a[5] != Py_None && (!(sample = plain(a[5], at::kFloat)) || sample->sizes() != at::IntArrayRef({batch}) || !same_device(sample, l.t))) return none();
    if (a[9] != Py_None && (!(change = plain(a[9], at::kInt)) || change->sizes() != at::IntArrayRef({batch}) || !same_device(change, l.t))) return none();
    if (draws && (!sample || (!accept && most > 1))) return none();
    On on(*l.t);
    int slices;
    int64_t needed;
    if (const int rc = lq_verify_drafts_plan(batch, rows, vocab, !draws, d.t != nullptr, 0, &slices, &needed)) return fail("lq_verify_drafts_plan", rc);
    const at::Tensor all = make({8 * batch * most + 4 * batch}, at::kByte, *l.t), ws = make({needed}, at::kByte, *l.t);
    int64_t at = 0;
    at::Tensor out = take(all, at, {batch, most}, at::kLong), accepted = take(all, at, {batch}, at::kInt);
    LQ_CALL(lq_verify_drafts, l.t->data_ptr(), l.t->stride(0), d.t ? d.t->data_ptr() : nullptr, d.t ? d.t->stride(0) : 0, (const int64_t *)tokens->data_ptr(),
            cu ? (const int32_t *)cu->data_ptr() : nullptr, batch, rows, vocab, most, l.dtype, temperature, accept ? (const float *)accept->data_ptr() : nullptr,
            sample ? (const float *)sample->data_ptr() : nullptr, (int64_t *)out.data_ptr(), (int32_t *)accepted.data_ptr(),
            change ? (int32_t *)change->data_ptr() : nullptr, ws.data_ptr(), needed, on.stream);
    return Py_BuildValue("NN", wrap(std::move(out)), wrap(std::move(accepted)));
}

// device index -> the current stream's handle
PyObject *current_stream(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(1)
    return PyLong_FromVoidPtr((void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA((c10::DeviceIndex)integer(a[0])).stream());
}

PyObject *set_error(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(1)
    Py_INCREF(a[0]);
    Py_XSETREF(g_error, a[0]);
    return none();
}

// x -> whether a layer in training can take its short way: activations in plain form, autograd records, and nothing looks at the call
// that is given the tensors of the Function over rows otherwise (a trace, a transform, hooks on saved tensors, a dispatch mode)
PyObject *records_plainly(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    LQ_ARGS(1)
    const at::Tensor *x = bf16(a[0]);
    return PyBool_FromLong(x && x->dim() >= 1 && x->numel() > 0 && c10::GradMode::is_enabled() && !c10::InferenceMode::is_enabled() &&
                           !watched() && !c10::impl::dispatch_mode_enabled() && at::SavedTensorDefaultHooks::get_tls_state().stack.empty());
}

#define LQ_METHOD(f) {#f, (PyCFunction)(void (*)(void))guarded<f>, METH_FASTCALL, nullptr}

// Until a thread has touched the thread-local storage of the library loaded last, its every access to that of another library (the tensor
// library's dispatch state and modes are full of them) goes the slow way through the C library's __tls_get_addr (glibc before 2.39, its bug
// 19924). This library is loaded at the first call of a program, behind those others, and a store brings the calling thread up to date:
// torch.empty_like on the GPU 1.15 -> 0.90 us, seven layers on four tokens, 1536 columns, 38 -> 35, six steps of the optimizer 69 -> 62.
thread_local volatile char touched;

// A C++ exception (out of memory, say) leaves as the Python exception the tensor library would raise
template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    touched = 1;
    PyObject *r = F(self, a, n);
    if (r && PyErr_Occurred()) {  // an argument that is no number
        Py_DECREF(r);
        return nullptr;
    }
    return r;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    LQ_METHOD(linear4), LQ_METHOD(linear4_eval), LQ_METHOD(dx4), LQ_METHOD(gate_up), LQ_METHOD(dx_silu), LQ_METHOD(dx_pair), LQ_METHOD(linear8), LQ_METHOD(infer8),
    LQ_METHOD(infer8_eval), LQ_METHOD(dx8), LQ_METHOD(quant8), LQ_METHOD(quant8_token), LQ_METHOD(dequant8), LQ_METHOD(weight_grad),
    LQ_METHOD(weight_grad_acc), LQ_METHOD(weight_grad_acc8), LQ_METHOD(gradq8), LQ_METHOD(adam8_param), LQ_METHOD(adam8_sr),
    LQ_METHOD(adam8_queue), LQ_METHOD(adam8_run), LQ_METHOD(adam8_w4), LQ_METHOD(adam8_w8), LQ_METHOD(kv8_append), LQ_METHOD(kv8_attention), LQ_METHOD(kv8_attention_shared), LQ_METHOD(kv8_read), LQ_METHOD(kv8_resize), LQ_METHOD(verify_drafts), LQ_METHOD(current_stream),
    LQ_METHOD(records_plainly), LQ_METHOD(set_error), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lqbind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lqbind() { return PyModule_Create(&module); }

// Host path of the quantised linear layers in eager mode: what Linear.forward does between the model's call and the
// kernels -- argument checks, the memory of the result and of the int8 rows, the launches -- without the Python
// interpreter.  A layer of a few hundred tokens runs for 5 to 20 microseconds on the GPU, less than the two dozen Python
// calls and two ctypes calls of the general path take (77 x 3072 x 3072: 31 us a forward that way, 11 us this way).
//
//   bind(path)                  the kernels' library
//   linear(...)                 one layer: Linear.forward with its optional prologue, gate and residual
//   fanout(...)                 several layers that read the same tokens, quantised once
//   vector_fanout(...)          several small-batch layers that read the same rows, in one launch
//   adapters(...)               layers that read the same rows, with a low-rank adapter for each of them
//   block_norm(...)             what lies between two blocks, and the next one's projections where they are given
//
// Every function takes the cases it can decide on cheaply and returns None for all others (tensors of other types,
// devices or layouts, operands that need a cast or a copy, errors): the caller then goes the general way in Python, which
// also words the errors.  Nothing is kept between calls.
//
// Everything that belongs to Python (arguments, the tensors' sizes and pointers) is read first; the allocations and the
// launches then run without the interpreter's lock, as behind ctypes and torch's own operators: a full hardware queue or an
// allocator that has to give memory back makes this thread wait, not the others.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/autocast_mode.h>
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/i8f.h"
#include "../../../include/i8f_blocks.h"
#include "../quant_lora_entry.hpp"
#include "../w8a16_rotated.hpp"

namespace {

// ---- the kernels' library -----------------------------------------------------------------
#define I8F_ENTRY_POINTS(X)                                                                                              \
    X(i8f_quant_rowwise) X(i8f_quant_rowwise_prologue) X(i8f_quant_rowwise_norm_modulate) X(i8f_quant_rowwise_rms_norm)  \
    X(i8f_quant_rowwise_concat_gelu) X(i8f_rotate128) X(i8f_linear_w8a8_gated) X(i8f_linear_w8a8_grouped) X(i8f_linear_w8a16_small_m) \
    X(i8f_linear_w8a16_small_m_grouped) X(i8f_internal_w8a16_rotated) X(i8f_linear_w8a8_lora) X(i8f_internal_quant_lora)    \
    X(i8f_adapters_by_side) X(i8f_adapters_down) X(i8f_adapters_down_workspace_bytes) X(i8f_linear_w8a8_adapters) X(i8f_linear_w8a8_adapters_workspace_bytes) X(i8f_linear_w8a16_small_m_adapters) X(i8f_block_norm)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
    I8F_ENTRY_POINTS(X)
#undef X
    bool bound = false;
} lib;

PyObject *bind(PyObject *, PyObject *arg) {
    const char *path = PyUnicode_AsUTF8(arg);
    if (!path) return nullptr;
    void *h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (!h) return PyErr_Format(PyExc_RuntimeError, "cannot load %s: %s", path, dlerror());
#define X(name)                                                                                                    \
    if (!(lib.name = (decltype(lib.name))dlsym(h, #name)))                                                         \
        return PyErr_Format(PyExc_RuntimeError, "%s has no %s: build it again", path, #name);
    I8F_ENTRY_POINTS(X)
#undef X
    lib.bound = true;
    Py_RETURN_NONE;
}

// ---- arguments -----------------------------------------------------------------------------
int code_of(at::ScalarType t) {
    return t == at::kBFloat16 ? I8F_BF16 : t == at::kHalf ? I8F_F16 : t == at::kFloat ? I8F_F32 : -1;
}

// A plain torch.Tensor or Parameter (subclasses -- fake and wrapped tensors among them -- are the general path's).
const at::Tensor *tensor(PyObject *o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool aligned16(const at::Tensor &t) { return (uintptr_t)t.const_data_ptr() % 16 == 0; }

// The rows of t, all but its last dimension flattened, if they are a matrix of contiguous rows at one stride.
bool rows_of(const at::Tensor &t, int64_t &M, int64_t &K, int64_t &ld) {
    const int64_t d = t.dim();
    if (d < 1) return false;
    const auto sizes = t.sizes(), strides = t.strides();
    K = sizes[d - 1], M = 1, ld = K;
    if (K < 1 || (K > 1 && strides[d - 1] != 1)) return false;
    int64_t expect = -1;  // stride that the next outer dimension has to have
    for (int64_t i = d - 2; i >= 0; --i) {
        if (sizes[i] == 1) continue;
        if (sizes[i] == 0) return false;
        if (expect < 0) ld = strides[i];
        else if (strides[i] != expect) return false;
        expect = strides[i] * sizes[i];
        M *= sizes[i];
    }
    return ld >= K;
}

// A vector per leading index of x, shared by its tokens: [K], or [..., 1, K] with x's leading dimensions.
// K: the last dimension of what it is applied to (x itself or the layer's output).
bool broadcasts_over_tokens(const at::Tensor &x, int64_t K, const at::Tensor &v) {
    if (v.scalar_type() != x.scalar_type() || v.device() != x.device() || !v.is_contiguous() || x.dim() < 2) return false;
    if (v.dim() == 1) return v.size(0) == K;
    if (v.dim() != x.dim() || v.size(-1) != K || v.size(-2) != 1) return false;
    for (int64_t i = 0; i < x.dim() - 2; ++i)
        if (v.size(i) != x.size(i)) return false;
    return true;
}

// Weight, scale and bias of a layer as the kernels take them.
struct Layer {
    const int8_t *w = nullptr;
    const float *ws = nullptr;
    float ws_host = 0.0f;
    int mode = I8F_SCALE_TENSOR, bias_code = I8F_BF16;
    const void *bias = nullptr;
    int64_t N = 0, K = 0;
};

bool layer_of(PyObject *weight, PyObject *scale, PyObject *bias, bool per_row, const at::Device &dev, Layer &l) {
    const at::Tensor *w = tensor(weight);
    if (!w || w->scalar_type() != at::kChar || w->dim() != 2 || w->device() != dev || !w->is_contiguous()) return false;
    l.w = (const int8_t *)w->const_data_ptr(), l.N = w->size(0), l.K = w->size(1);
    if (l.N < 1) return false;
    if (PyFloat_Check(scale)) {
        if (per_row) return false;
        l.ws_host = (float)PyFloat_AS_DOUBLE(scale);
    } else {
        const at::Tensor *s = tensor(scale);
        if (!s || s->scalar_type() != at::kFloat || s->device() != dev || !s->is_contiguous() || s->numel() < 1) return false;
        if (per_row && s->numel() != l.N) return false;
        l.ws = (const float *)s->const_data_ptr();
        l.mode = per_row && s->numel() != 1 ? I8F_SCALE_ROW : I8F_SCALE_TENSOR;  // (one scale: element 0 counts)
    }
    if (bias != Py_None) {
        const at::Tensor *b = tensor(bias);
        if (!b || b->device() != dev || !b->is_contiguous() || b->numel() != l.N || (l.bias_code = code_of(b->scalar_type())) < 0) return false;
        l.bias = b->const_data_ptr();
    }
    return true;
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType t, const at::Device &dev) {
    return at::detail::empty_cuda(size, t, dev, std::nullopt);
}

// The size of a layer's output on x's tokens: x's leading dimensions and N columns.
using Size = c10::SmallVector<int64_t, 6>;
Size output_size(const at::Tensor &x, int64_t N) {
    Size size(x.sizes().begin(), x.sizes().end());
    size.back() = N;
    return size;
}

// The interpreter's lock is released while one of these lives.  (Taking it again ends the thread where the interpreter has
// been shut down meanwhile, by an unwinding that has to be let out of here.)
struct WithoutGil {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutGil() noexcept(false) { PyEval_RestoreThread(state); }
};

struct Stream {
    void *handle;
    bool ok;
    explicit Stream(const at::Device &dev) : handle(nullptr), ok(dev.is_cuda() && dev.index() == c10::hip::current_device()) {
        if (ok) handle = (void *)c10::hip::getCurrentHIPStream(dev.index()).stream();
    }
};

struct Owned {  // a new reference
    PyObject *p = nullptr;
    ~Owned() { Py_XDECREF(p); }
};

// ---- 16 rows or fewer: W8A16 ----------------------------------------------------------------
PyObject *small_m(const at::Tensor &x, int64_t M, int64_t K, int64_t ld, const Layer &l, bool rotate, void *stream) {
    const at::ScalarType type = x.scalar_type();
    const at::Device dev = x.device();
    const int dt = code_of(type);
    const void *xp = x.const_data_ptr();
    const Size size = output_size(x, l.N);
    at::Tensor rotated, y;
    bool done = false;
    {
        const WithoutGil released;
        y = empty(size, type, dev);
        void *out = y.data_ptr();
        done = rotate && !lib.i8f_internal_w8a16_rotated(xp, dt, M, K, ld, l.w, l.ws, l.ws_host, l.mode, l.bias, l.bias_code, out, l.N, stream);
        bool ready = true;
        if (rotate && !done) {
            rotated = empty({M, K}, type, dev);
            ready = !lib.i8f_rotate128(xp, dt, M, K, ld, rotated.data_ptr(), stream);
            xp = rotated.const_data_ptr(), ld = K;
        }
        if (ready && !done) done = !lib.i8f_linear_w8a16_small_m(xp, dt, M, K, ld, l.w, l.ws, l.ws_host, l.mode, l.bias, l.bias_code, out, l.N, stream);
    }
    if (!done) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
}

// ---- a dynamic LoRA on the layer ---------------------------------------------------------------
// Its first product by the launch that quantises x, the second inside the GEMM.  Two launches: with the BLAS library's call
// between them and the interpreter's part of it all, the host took 63 us a layer and the GPU waited for it below 2000 rows.
//
// linear_lora(x, weight, scale, bias, per_row, order, lora_A, lora_B, lora_alpha): a layer of more than 16 rows with the factors
// of a dynamic LoRA, no rotation, nothing in front and nothing behind.
PyObject *linear_lora(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 9) return PyErr_Format(PyExc_TypeError, "linear_lora takes 9 arguments, got %zd", n);
    const at::Tensor *xt = tensor(a[0]), *A = tensor(a[6]), *B = tensor(a[7]);
    if (!lib.bound || !xt || !A || !B || A->dim() != 2 || !xt->is_cuda()) Py_RETURN_NONE;
    const at::Tensor &x = *xt;
    const int64_t R = A->size(0);  // (the GEMM's LoRA epilogue takes ranks in steps of 16 up to 64)
    int64_t M, K, ld;
    if (R % 16 || R < 16 || R > 64 || !rows_of(x, M, K, ld)) Py_RETURN_NONE;
    // (every 16 rows read the factor once more: 16384 rows are as many as were measured.  There a 3072 x 3072 layer of rank 16 takes
    // 160 us where the quantiser, the BLAS library's product and the GEMM take 174, of rank 64 178 and 181, 4096 x 4096 277 either way)
    if (M > 16384 || K % 128 || K > (R > 32 ? 4096 : 6144) || ld % 8) Py_RETURN_NONE;
    Layer l;
    const at::ScalarType type = x.scalar_type();
    if ((type != at::kBFloat16 && type != at::kHalf) || !layer_of(a[1], a[2], a[3], a[4] == Py_True, x.device(), l)) Py_RETURN_NONE;
    for (const at::Tensor *f : {A, B})
        if (f->scalar_type() != type || f->device() != x.device() || f->dim() != 2 || !f->is_contiguous() || !aligned16(*f)) Py_RETURN_NONE;
    if (A->size(1) != K || B->size(0) != l.N || B->size(1) != R) Py_RETURN_NONE;
    if (K != l.K || l.N % 8 || !aligned16(x) || (uintptr_t)l.w % 16 || (l.mode == I8F_SCALE_ROW && (uintptr_t)l.ws % 16) || (uintptr_t)l.bias % 16 ||
        l.N * K >= (1ll << 31))
        Py_RETURN_NONE;
    if (at::autocast::is_autocast_enabled(at::kCUDA)) Py_RETURN_NONE;  // (the product's type is then the context's)
    float alpha = 0.0f;
    const bool has_alpha = a[8] != Py_None;
    if (has_alpha) {
        if (!PyFloat_CheckExact(a[8]) && !PyLong_CheckExact(a[8])) Py_RETURN_NONE;
        alpha = (float)PyFloat_AsDouble(a[8]);
        if (PyErr_Occurred()) return nullptr;
    }
    const Stream st(x.device());
    if (!st.ok) Py_RETURN_NONE;
    const int order = (int)PyLong_AsLong(a[5]);
    const at::Device dev = x.device();
    const Size size = output_size(x, l.N);
    const int dt = code_of(type);
    const void *xp = x.const_data_ptr(), *ap = A->const_data_ptr(), *bp = B->const_data_ptr();
    at::Tensor scratch, y;
    int rc;
    {
        const WithoutGil released;
        const int64_t q_bytes = (M * K + 255) / 256 * 256, t_bytes = (2 * M * R + 255) / 256 * 256;
        scratch = empty({q_bytes + t_bytes + 4 * M}, at::kByte, dev);
        int8_t *q = (int8_t *)scratch.data_ptr();
        void *t = q + q_bytes;
        float *qs = (float *)(q + q_bytes + t_bytes);
        y = empty(size, type, dev);
        rc = lib.i8f_internal_quant_lora(xp, dt, M, K, ld, ap, R, q, qs, t, st.handle);
        if (!rc)
            rc = lib.i8f_linear_w8a8_lora(q, qs, l.w, l.ws, l.ws_host, l.mode, l.bias, l.bias_code, t, bp, R, has_alpha, alpha, y.data_ptr(), dt, M,
                                          l.N, K, order, st.handle);
    }
    if (rc) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
}

constexpr int MAX_FANOUT = 8;

PyObject *list_of(at::Tensor *y, Py_ssize_t count) {
    PyObject *out = PyList_New(count);
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject *o = THPVariable_Wrap(std::move(y[i]));
        if (!o) {
            Py_DECREF(out);
            return nullptr;
        }
        PyList_SET_ITEM(out, i, o);
    }
    return out;
}

// The layers' products of the same int8 rows: layers of one form, a launch for as many as the library puts together.
int project(const Layer *l, int count, int8_t *q, float *qs, int64_t M, int64_t K, int dt, int order, at::Tensor *y, void *work, int64_t work_bytes,
            void *stream) {
    int rc = 0;
    for (int first = 0, next; !rc && first < count; first = next) {
        i8f_linear_group g[I8F_MAX_LINEAR_GROUPS] = {};
        int bias_code = -1;
        for (next = first; next < count && next - first < I8F_MAX_LINEAR_GROUPS; ++next) {
            const Layer &o = l[next];
            if (o.N != l[first].N || o.mode != l[first].mode || (o.bias && bias_code >= 0 && o.bias_code != bias_code)) break;
            if (o.bias) bias_code = o.bias_code;
            i8f_linear_group &e = g[next - first];
            e.a = q, e.a_scale = qs, e.w = o.w, e.w_scale = o.ws, e.w_scale_host = o.ws_host, e.bias = o.bias, e.out = y[next].data_ptr(), e.M = M;
            e.rows_per_gate = 1;
        }
        rc = lib.i8f_linear_w8a8_grouped(g, next - first, l[first].mode, bias_code < 0 ? (int)I8F_BF16 : bias_code, dt, l[first].N, K, order, work,
                                         work_bytes, stream);
    }
    return rc;
}

// The W8A8 form of linear and fanout, whose arguments these are; a gate or a residual for one layer only.
PyObject *w8a8(PyObject *const *a, const at::Tensor &x, int64_t M, int64_t K, int64_t ld, const Layer *l, int count, const Stream &st) {
    const int dt = code_of(x.scalar_type()), order = (int)PyLong_AsLong(a[7]), kind = (int)PyLong_AsLong(a[8]);
    const bool rotate = a[5] == Py_True, fused_add = a[13] == Py_True, gated = a[14] != Py_None, with_residual = a[15] != Py_None;
    if (count != 1 && (gated || with_residual)) Py_RETURN_NONE;

    // the operation in front of the layer and its operands
    const at::Tensor *s = nullptr, *t = nullptr, *w = nullptr;
    int64_t V = 1, Kall = K, Kb = 0, ldb = 0;
    float eps = 0.0f;
    if (kind == I8F_PRO_NORM_MODULATE || kind == I8F_PRO_RMS_NORM) {
        eps = (float)PyFloat_AsDouble(a[11]);
        if (PyErr_Occurred()) return nullptr;
    }
    if (kind == I8F_PRO_MODULATE || kind == I8F_PRO_NORM_MODULATE || kind == I8F_PRO_RMS_NORM) {
        s = a[9] == Py_None ? nullptr : tensor(a[9]), t = a[10] == Py_None ? nullptr : tensor(a[10]);
        if ((a[9] != Py_None && !s) || (a[10] != Py_None && !t) || (kind != I8F_PRO_RMS_NORM && !(s && t))) Py_RETURN_NONE;
        for (const at::Tensor *v : {s, t}) {
            if (!v) continue;
            if (!broadcasts_over_tokens(x, K, *v) || !aligned16(*v)) Py_RETURN_NONE;
            V = v->numel() / K;
        }
        if (s && t && s->sizes() != t->sizes()) Py_RETURN_NONE;
        if (V < 1 || M % V) Py_RETURN_NONE;
        if (kind != I8F_PRO_MODULATE && (K > 16384 || K % 16 || (M > 1 && ld % 8) || !aligned16(x))) Py_RETURN_NONE;
        if (kind == I8F_PRO_RMS_NORM && a[12] != Py_None) {
            w = tensor(a[12]);
            if (!w || w->scalar_type() != x.scalar_type() || w->dim() != 1 || w->size(0) != K || w->device() != x.device() || !w->is_contiguous() ||
                !aligned16(*w))
                Py_RETURN_NONE;
        }
    } else if (kind == I8F_PRO_CONCAT_GELU) {
        s = tensor(a[9]);
        int64_t Mb;
        if (!s || s->scalar_type() != x.scalar_type() || s->device() != x.device() || s->dim() != x.dim() || !rows_of(*s, Mb, Kb, ldb)) Py_RETURN_NONE;
        for (int64_t i = 0; i + 1 < x.dim(); ++i)
            if (s->size(i) != x.size(i)) Py_RETURN_NONE;
        Kall = K + Kb;
        if (K % 16 || Kb % 16 || Kall > 16384 || (M > 1 && (ld % 8 || ldb % 8)) || !aligned16(x) || !aligned16(*s) || (rotate && Kb % 128)) Py_RETURN_NONE;
    } else if (kind == I8F_PRO_SILU_GATE) {
        s = tensor(a[9]);
        if (!s || s->scalar_type() != x.scalar_type() || s->device() != x.device() || s->sizes() != x.sizes() || !s->is_contiguous()) Py_RETURN_NONE;
    } else if (kind != I8F_PRO_NONE && kind != I8F_PRO_GELU_TANH && kind != I8F_PRO_GELU_ERF) {
        Py_RETURN_NONE;
    }
    for (int i = 0; i < count; ++i)
        if (l[i].K != Kall) Py_RETURN_NONE;

    // what follows the layer
    const at::Tensor *gate = nullptr, *res = nullptr, *work = nullptr;
    int64_t gate_rows = 1;
    if (gated) {
        gate = tensor(a[14]);
        if (!gate || !broadcasts_over_tokens(x, l[0].N, *gate)) Py_RETURN_NONE;
        const int64_t vecs = gate->numel() / l[0].N;
        if (vecs < 1 || M % vecs) Py_RETURN_NONE;
        gate_rows = M / vecs;
    }
    if (with_residual) {
        res = tensor(a[15]);
        if (!res || res->scalar_type() != x.scalar_type() || res->device() != x.device() || res->dim() != x.dim() || !res->is_contiguous() ||
            res->numel() != M * l[0].N || res->size(-1) != l[0].N)
            Py_RETURN_NONE;
        for (int64_t i = 0; i + 1 < x.dim(); ++i)
            if (res->size(i) != x.size(i)) Py_RETURN_NONE;
    }
    Owned work_object;
    if (a[16] != Py_None) {   // (the narrowest layer has the fewest tiles: what it cannot use, none can)
        int64_t narrowest = l[0].N;
        for (int i = 1; i < count; ++i) narrowest = l[i].N < narrowest ? l[i].N : narrowest;
        work_object.p = PyObject_CallFunction(a[16], "OLLL", a[0], (long long)M, (long long)narrowest, (long long)Kall);
        if (!work_object.p) return nullptr;
        if (work_object.p != Py_None && !(work = tensor(work_object.p))) Py_RETURN_NONE;
    }

    const at::ScalarType type = x.scalar_type();
    const at::Device dev = x.device();
    Size size[MAX_FANOUT];
    for (int i = 0; i < count; ++i) size[i] = output_size(x, l[i].N);
    const auto address = [](const at::Tensor *o) { return o ? o->const_data_ptr() : nullptr; };
    const void *xp = x.const_data_ptr(), *sp = address(s), *tp = address(t), *wp = address(w), *gate_p = address(gate), *res_p = address(res);
    void *work_p = work ? work->data_ptr() : nullptr;
    const int64_t work_bytes = work ? work->numel() : 0;
    at::Tensor scratch, y[MAX_FANOUT];
    int rc;
    {
        const WithoutGil released;
        // one piece of memory for the int8 rows and, behind them, their scales; it goes back to the allocator when the call
        // returns, for work behind these kernels on the same stream
        const int64_t q_bytes = (M * Kall + 255) / 256 * 256;
        scratch = empty({q_bytes + 4 * M}, at::kByte, dev);
        int8_t *q = (int8_t *)scratch.data_ptr();
        float *qs = (float *)(q + q_bytes);
        for (int i = 0; i < count; ++i) y[i] = empty(size[i], type, dev);
        const int rb = rotate ? 128 : 0;
        switch (kind) {
        case I8F_PRO_NONE: rc = lib.i8f_quant_rowwise(xp, dt, M, K, ld, rb, q, qs, st.handle); break;
        case I8F_PRO_NORM_MODULATE:
            rc = lib.i8f_quant_rowwise_norm_modulate(xp, dt, M, K, ld, eps, sp, tp, M / V, fused_add, rb, q, qs, st.handle);
            break;
        case I8F_PRO_RMS_NORM: rc = lib.i8f_quant_rowwise_rms_norm(xp, dt, M, K, ld, eps, wp, sp, tp, M / V, fused_add, rb, q, qs, st.handle); break;
        case I8F_PRO_CONCAT_GELU: rc = lib.i8f_quant_rowwise_concat_gelu(xp, dt, M, K, ld, sp, Kb, ldb, rb, q, qs, st.handle); break;
        case I8F_PRO_SILU_GATE: rc = lib.i8f_quant_rowwise_prologue(xp, dt, M, K, ld, kind, sp, nullptr, 1, rb, q, qs, st.handle); break;
        default:
            rc = lib.i8f_quant_rowwise_prologue(xp, dt, M, K, ld, kind == I8F_PRO_MODULATE && fused_add ? (int)I8F_PRO_MODULATE_FUSED : kind, sp, tp,
                                                M / V, rb, q, qs, st.handle);
        }
        if (!rc && count == 1)
            rc = lib.i8f_linear_w8a8_gated(q, qs, l[0].w, l[0].ws, l[0].ws_host, l[0].mode, l[0].bias, l[0].bias_code, gate_p, gate_rows, res_p,
                                           y[0].data_ptr(), dt, M, l[0].N, l[0].K, order, work_p, work_bytes, st.handle);
        if (!rc && count > 1) rc = project(l, count, q, qs, M, Kall, dt, order, y, work_p, work_bytes, st.handle);
    }
    if (rc) Py_RETURN_NONE;
    return count == 1 ? THPVariable_Wrap(std::move(y[0])) : list_of(y, count);
}

// linear(x, weight, scale, bias, per_row, rotate, small_rows, order, kind, mod_scale, mod_shift, eps, norm_weight, fused_add,
//        gate, residual, workspace): kind, an i8f_prologue, names what is applied to x inside the quantiser; workspace(x, M, N,
// K) gives the memory of the K split, which the layers of one call share, or None.  It is called once a W8A8 call has passed
// every check, never for 16 rows or fewer or for a call that goes the general way, which asks for its own: the memory stays
// with the stream, or with the graph that is being captured, together with the kernel that clears it.
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 17) return PyErr_Format(PyExc_TypeError, "linear takes 17 arguments, got %zd", n);
    const at::Tensor *xt = tensor(a[0]);
    if (!lib.bound || !xt || !xt->is_cuda()) Py_RETURN_NONE;
    const at::Tensor &x = *xt;
    const int dt = code_of(x.scalar_type());
    const bool per_row = a[4] == Py_True, rotate = a[5] == Py_True;
    int64_t M, K, ld;
    Layer l;
    if ((dt != I8F_BF16 && dt != I8F_F16) || !rows_of(x, M, K, ld) || !layer_of(a[1], a[2], a[3], per_row, x.device(), l)) Py_RETURN_NONE;
    const Stream st(x.device());
    if (!st.ok || (rotate && K % 128)) Py_RETURN_NONE;
    if (M <= PyLong_AsLongLong(a[6])) {
        if (PyLong_AsLong(a[8]) != I8F_PRO_NONE || a[14] != Py_None || a[15] != Py_None || K != l.K) Py_RETURN_NONE;
        return small_m(x, M, K, ld, l, rotate, st.handle);
    }
    return w8a8(a, x, M, K, ld, &l, 1, st);
}

// fanout(the arguments of linear): weight, scale, bias and per_row are tuples with an entry for each layer; a list of outputs.
// Not for 16 rows or fewer.
PyObject *fanout(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 17) return PyErr_Format(PyExc_TypeError, "fanout takes 17 arguments, got %zd", n);
    const at::Tensor *xt = tensor(a[0]);
    if (!lib.bound || !xt || !xt->is_cuda()) Py_RETURN_NONE;
    const at::Tensor &x = *xt;
    const int dt = code_of(x.scalar_type());
    const Py_ssize_t count = PyTuple_Check(a[1]) ? PyTuple_GET_SIZE(a[1]) : 0;
    int64_t M, K, ld;
    if ((dt != I8F_BF16 && dt != I8F_F16) || count < 2 || count > MAX_FANOUT || x.dim() < 2 || !rows_of(x, M, K, ld)) Py_RETURN_NONE;
    for (int i = 2; i <= 4; ++i)
        if (!PyTuple_Check(a[i]) || PyTuple_GET_SIZE(a[i]) != count) Py_RETURN_NONE;
    Layer l[MAX_FANOUT];
    for (Py_ssize_t i = 0; i < count; ++i)
        if (!layer_of(PyTuple_GET_ITEM(a[1], i), PyTuple_GET_ITEM(a[2], i), PyTuple_GET_ITEM(a[3], i), PyTuple_GET_ITEM(a[4], i) == Py_True, x.device(), l[i]))
            Py_RETURN_NONE;
    const Stream st(x.device());
    if (!st.ok || (a[5] == Py_True && K % 128) || M <= PyLong_AsLongLong(a[6])) Py_RETURN_NONE;
    return w8a8(a, x, M, K, ld, l, (int)count, st);
}

// vector_fanout(x, weights, scales, biases, per_row, rotate): tuples with one entry per layer -> list of outputs
PyObject *vector_fanout(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 6) return PyErr_Format(PyExc_TypeError, "vector_fanout takes 6 arguments, got %zd", n);
    const at::Tensor *xt = tensor(a[0]);
    if (!lib.bound || !xt || !xt->is_cuda()) Py_RETURN_NONE;
    const at::Tensor &x = *xt;
    const int dt = code_of(x.scalar_type());
    int64_t M, K, ld;
    const Stream st(x.device());
    const Py_ssize_t count = PyTuple_Check(a[1]) ? PyTuple_GET_SIZE(a[1]) : 0;
    const bool rotate = a[5] == Py_True;
    if (!st.ok || (dt != I8F_BF16 && dt != I8F_F16) || !rows_of(x, M, K, ld) || M > 16 || count < 2 || count > I8F_MAX_LINEAR_GROUPS ||
        (rotate && K % 128))
        Py_RETURN_NONE;
    for (int i = 2; i <= 4; ++i)
        if (!PyTuple_Check(a[i]) || PyTuple_GET_SIZE(a[i]) != count) Py_RETURN_NONE;
    Layer l[I8F_MAX_LINEAR_GROUPS];
    int bias_code = -1;
    for (Py_ssize_t i = 0; i < count; ++i) {
        if (!layer_of(PyTuple_GET_ITEM(a[1], i), PyTuple_GET_ITEM(a[2], i), PyTuple_GET_ITEM(a[3], i), PyTuple_GET_ITEM(a[4], i) == Py_True,
                      x.device(), l[i]) ||
            l[i].K != K || l[i].mode != l[0].mode)
            Py_RETURN_NONE;
        if (l[i].bias) {
            if (bias_code >= 0 && bias_code != l[i].bias_code) Py_RETURN_NONE;
            bias_code = l[i].bias_code;
        }
    }
    const at::ScalarType type = x.scalar_type();
    const at::Device dev = x.device();
    const void *xp = x.const_data_ptr();
    Size size[I8F_MAX_LINEAR_GROUPS];
    for (Py_ssize_t i = 0; i < count; ++i) size[i] = output_size(x, l[i].N);
    at::Tensor rotated, y[I8F_MAX_LINEAR_GROUPS];
    bool done = true;
    {
        const WithoutGil released;
        if (rotate) {
            rotated = empty({M, K}, type, dev);
            done = !lib.i8f_rotate128(xp, dt, M, K, ld, rotated.data_ptr(), st.handle);
            xp = rotated.const_data_ptr(), ld = K;
        }
        i8f_small_m_group g[I8F_MAX_LINEAR_GROUPS];
        for (Py_ssize_t i = 0; i < count; ++i) {
            y[i] = empty(size[i], type, dev);
            g[i] = {xp, M, K, ld, l[i].w, l[i].ws, l[i].ws_host, l[i].bias, y[i].data_ptr(), l[i].N};
        }
        if (done)
            done = !lib.i8f_linear_w8a16_small_m_grouped(g, (int)count, dt, l[0].mode, bias_code < 0 ? (int)I8F_BF16 : bias_code, st.handle);
    }
    if (!done) Py_RETURN_NONE;
    return list_of(y, count);
}

// Whether an operand has or asks for a derivative that these operators do not have: the general path words the refusal.
bool wants_gradient(const at::Tensor *t) { return t && ((t->requires_grad() && c10::GradMode::is_enabled()) || t->_fw_grad(0).defined()); }

// v has the shape of t's leading dimensions, all of them but the last or fewer: the rows of t to an element of v, 0 if it has not.
int64_t rows_to_element(const at::Tensor &t, const at::Tensor &v) {
    const int64_t lead = t.dim() - 1;
    if (v.dim() > lead) return 0;
    for (int64_t i = 0; i < v.dim(); ++i)
        if (v.size(i) != t.size(i)) return 0;
    int64_t rows = 1;
    for (int64_t i = v.dim(); i < lead; ++i) rows *= t.size(i);
    return rows;
}

// adapters(x, ids, weights, scales, biases, per_row, rotate, small_rows, banks): tuples with an entry for each layer, a bank being (down,
// up, scale, first_rank, count, max_rank, in features, out features) -> list of outputs.
PyObject *adapters(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 9) return PyErr_Format(PyExc_TypeError, "adapters takes 9 arguments, got %zd", n);
    const at::Tensor *xt = tensor(a[0]), *ids = tensor(a[1]);
    if (!lib.bound || !xt || !ids || !xt->is_cuda()) Py_RETURN_NONE;
    const at::Tensor &x = *xt;
    const int dt = code_of(x.scalar_type());
    const Py_ssize_t count = PyTuple_Check(a[2]) ? PyTuple_GET_SIZE(a[2]) : 0;
    const bool rotate = a[6] == Py_True;
    int64_t M, K, ld;
    const Stream st(x.device());
    if (!st.ok || (dt != I8F_BF16 && dt != I8F_F16) || wants_gradient(xt) || !rows_of(x, M, K, ld) || count < 1 || count > I8F_MAX_ADAPTED_LAYERS ||
        (rotate && K % 128))
        Py_RETURN_NONE;
    if (ids->scalar_type() != at::kInt || ids->device() != x.device() || !ids->is_contiguous()) Py_RETURN_NONE;
    const int64_t per = rows_to_element(x, *ids);
    if (per < 1) Py_RETURN_NONE;
    for (int i : {3, 4, 5, 8})
        if (!PyTuple_Check(a[i]) || PyTuple_GET_SIZE(a[i]) != count) Py_RETURN_NONE;
    const bool few = M <= PyLong_AsLongLong(a[7]);
    i8f_adapted_layer l[I8F_MAX_ADAPTED_LAYERS] = {};
    Size size[I8F_MAX_ADAPTED_LAYERS];
    int64_t bytes = 0, t_at[I8F_MAX_ADAPTED_LAYERS], side_at[I8F_MAX_ADAPTED_LAYERS], work_bytes = 0;
    bool by_side = !few;
    const auto take = [&](int64_t b) {   // a piece of the scratch memory
        const int64_t at = bytes;
        bytes += (b + 255) / 256 * 256;
        return at;
    };
    const int64_t q_at = few ? (rotate ? take(2 * M * K) : 0) : take(M * K), qs_at = few ? 0 : take(4 * M);
    for (Py_ssize_t i = 0; i < count; ++i) {
        Layer o;
        if (!layer_of(PyTuple_GET_ITEM(a[2], i), PyTuple_GET_ITEM(a[3], i), PyTuple_GET_ITEM(a[4], i), PyTuple_GET_ITEM(a[5], i) == Py_True, x.device(), o) || o.K != K)
            Py_RETURN_NONE;
        PyObject *bank = PyTuple_GET_ITEM(a[8], i);
        if (!PyTuple_Check(bank) || PyTuple_GET_SIZE(bank) != 8) Py_RETURN_NONE;
        // (a factor's rows are padded in memory: 249 to 256 columns look the same there)
        if (PyLong_AsLongLong(PyTuple_GET_ITEM(bank, 6)) != K || PyLong_AsLongLong(PyTuple_GET_ITEM(bank, 7)) != o.N) Py_RETURN_NONE;
        const at::Tensor *down = tensor(PyTuple_GET_ITEM(bank, 0)), *up = tensor(PyTuple_GET_ITEM(bank, 1)), *scale = tensor(PyTuple_GET_ITEM(bank, 2)),
                         *first = tensor(PyTuple_GET_ITEM(bank, 3));
        i8f_adapters &ad = l[i].adapters;
        ad.count = PyLong_AsLongLong(PyTuple_GET_ITEM(bank, 4)), ad.max_rank = PyLong_AsLongLong(PyTuple_GET_ITEM(bank, 5));
        if (!down || !up || !scale || !first || down->scalar_type() != x.scalar_type() || down->device() != x.device() || down->dim() != 2 || down->size(1) != (K + 7) / 8 * 8 ||
            up->scalar_type() != x.scalar_type() || up->device() != x.device() || up->numel() != down->size(0) * o.N || scale->numel() != ad.count ||
            first->numel() != ad.count + 1)
            Py_RETURN_NONE;
        ad.down = down->const_data_ptr(), ad.up = up->const_data_ptr(), ad.scale = (const float *)scale->const_data_ptr();
        ad.first_rank = (const int32_t *)first->const_data_ptr(), ad.ids = (const int32_t *)ids->const_data_ptr(), ad.rows_per_id = per;
        l[i].w = o.w, l[i].w_scale = o.ws, l[i].w_scale_host = o.ws_host, l[i].scale_mode = o.mode, l[i].bias = o.bias, l[i].bias_dtype = o.bias_code, l[i].N = o.N;
        size[i] = output_size(x, o.N);
        by_side = by_side && lib.i8f_adapters_by_side(M, o.N, K, per);
        const int64_t need = few ? 0 : lib.i8f_linear_w8a8_adapters_workspace_bytes(M, o.N, K);
        work_bytes = need > work_bytes ? need : work_bytes;
    }
    for (Py_ssize_t i = 0; i < count; ++i) t_at[i] = take(2 * M * l[i].adapters.max_rank), side_at[i] = by_side ? take(4 * M * l[i].N) : 0;
    // (the memory of the first products is free when the projections start)
    int64_t ranks = 0;
    for (Py_ssize_t i = 0; i < count; ++i) ranks += l[i].adapters.max_rank;
    const int64_t down_bytes = lib.i8f_adapters_down_workspace_bytes(M, K, ranks, aligned16(x) && (M <= 1 || ld % 8 == 0)), more = down_bytes > work_bytes ? down_bytes : work_bytes;
    const int64_t work_at = more ? take(more) : 0;
    const at::ScalarType type = x.scalar_type();
    const at::Device dev = x.device();
    const void *xp = x.const_data_ptr();
    at::Tensor scratch, y[I8F_MAX_ADAPTED_LAYERS];
    int rc;
    {
        const WithoutGil released;
        scratch = empty({bytes + 256}, at::kByte, dev);
        char *base = (char *)scratch.data_ptr();
        for (Py_ssize_t i = 0; i < count; ++i) {
            y[i] = empty(size[i], type, dev);
            l[i].t = base + t_at[i], l[i].side = by_side ? (float *)(base + side_at[i]) : nullptr, l[i].out = y[i].data_ptr();
        }
        if (few) {
            rc = lib.i8f_adapters_down(xp, dt, M, K, ld, l, (int)count, 0, nullptr, nullptr, nullptr, 0, st.handle);
            if (!rc && rotate) {
                rc = lib.i8f_rotate128(xp, dt, M, K, ld, base + q_at, st.handle);
                xp = base + q_at, ld = K;
            }
            if (!rc) rc = lib.i8f_linear_w8a16_small_m_adapters(xp, dt, M, K, ld, l, (int)count, st.handle);
        } else {
            int8_t *q = (int8_t *)base + q_at;
            float *qs = (float *)(base + qs_at);
            rc = lib.i8f_adapters_down(xp, dt, M, K, ld, l, (int)count, rotate ? 128 : 0, q, qs, down_bytes ? base + work_at : nullptr, down_bytes, st.handle);
            if (!rc) rc = lib.i8f_linear_w8a8_adapters(q, qs, l, (int)count, dt, M, K, work_bytes ? base + work_at : nullptr, work_bytes, st.handle);
        }
    }
    if (rc) Py_RETURN_NONE;
    return list_of(y, count);
}

// An operand of block_norm's vectors: [K], or y's dimensions with ones from some dimension on; *rows of y to a vector.
bool block_vector(const at::Tensor &y, PyObject *o, const void **p, int64_t *rows) {
    if (o == Py_None) return true;
    const at::Tensor *v = tensor(o);
    const int64_t lead = y.dim() - 1, K = y.size(lead);
    if (!v || wants_gradient(v) || v->scalar_type() != y.scalar_type() || v->device() != y.device() || !v->is_contiguous() || v->dim() < 1 || v->size(-1) != K) return false;
    int64_t shared = 0;
    if (v->dim() != 1) {
        if (v->dim() != y.dim()) return false;
        while (shared < lead && v->size(shared) == y.size(shared)) ++shared;
        for (int64_t i = shared; i < lead; ++i)
            if (v->size(i) != 1) return false;
    }
    *rows = 1;
    for (int64_t i = shared; i < lead; ++i) *rows *= y.size(i);
    *p = v->const_data_ptr();
    return true;
}

// One of block_norm's norms: kind, weight, bias, eps at a[0..3]
bool block_norm_of(const at::Tensor &y, PyObject *const *a, int *kind, const void **weight, const void **bias, int *dtype, float *eps) {
    *dtype = code_of(y.scalar_type());
    if (a[0] == Py_None) *kind = I8F_NORM_NONE;
    else if (PyUnicode_Check(a[0]) && PyUnicode_CompareWithASCIIString(a[0], "rms") == 0) *kind = I8F_NORM_RMS;
    else if (PyUnicode_Check(a[0]) && PyUnicode_CompareWithASCIIString(a[0], "layer") == 0) *kind = I8F_NORM_LAYER;
    else return false;
    *eps = (float)PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred() || !(*eps >= 0.0f)) return false;
    int found = -1;
    for (int i = 1; i <= 2; ++i) {
        if (a[i] == Py_None) continue;
        const at::Tensor *v = tensor(a[i]);
        if (!v || *kind == I8F_NORM_NONE || wants_gradient(v) || v->dim() != 1 || v->size(0) != y.size(-1) || v->device() != y.device() || !v->is_contiguous()) return false;
        const int code = code_of(v->scalar_type());
        if ((code != *dtype && code != I8F_F32) || (found >= 0 && code != found)) return false;
        found = code;
        *(i == 1 ? weight : bias) = v->const_data_ptr();
    }
    if (found >= 0) *dtype = found;
    return true;
}

// block_norm(y, residual, post_norm, post_weight, post_bias, post_eps, gate, gate_tanh, residual_scale, branch_scale, pre_norm, pre_weight,
//            pre_bias, pre_eps, mod_scale, mod_shift, weights, scales, biases, per_row, rotate, order, workspace): weights is None -> (x,
// h); tuples with an entry for each layer -> (x, list of the layers' outputs), not for 16 rows or fewer
PyObject *block_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 23) return PyErr_Format(PyExc_TypeError, "block_norm takes 23 arguments, got %zd", n);
    const at::Tensor *yt = tensor(a[0]), *rt = tensor(a[1]);
    if (!lib.bound || !yt || !rt || !yt->is_cuda()) Py_RETURN_NONE;
    const at::Tensor &y = *yt, &r = *rt;
    const int dt = code_of(y.scalar_type());
    int64_t M, K, Mr, Kr;
    i8f_block_norm_args g = {};
    const Stream st(y.device());
    if (!st.ok || dt < 0 || wants_gradient(yt) || wants_gradient(rt) || r.scalar_type() != y.scalar_type() || r.device() != y.device() || r.sizes() != y.sizes() ||
        !rows_of(y, M, K, g.ldy) || !rows_of(r, Mr, Kr, g.ldr) || K < 1)
        Py_RETURN_NONE;
    g.rows_per_gate = g.rows_per_scale = g.rows_per_shift = 1;
    if (!block_norm_of(y, a + 2, &g.post_norm, &g.post_weight, &g.post_bias, &g.post_dtype, &g.post_eps) ||
        !block_norm_of(y, a + 10, &g.pre_norm, &g.pre_weight, &g.pre_bias, &g.pre_dtype, &g.pre_eps) || !block_vector(y, a[6], &g.gate, &g.rows_per_gate) ||
        !block_vector(y, a[14], &g.mod_scale, &g.rows_per_scale) || !block_vector(y, a[15], &g.mod_shift, &g.rows_per_shift))
        Py_RETURN_NONE;
    g.gate_tanh = PyObject_IsTrue(a[7]) == 1;
    g.residual_scale = (float)PyFloat_AsDouble(a[8]), g.branch_scale = (float)PyFloat_AsDouble(a[9]);
    if (PyErr_Occurred()) return nullptr;
    g.y = y.const_data_ptr(), g.residual = r.const_data_ptr(), g.M = M, g.K = K, g.dtype = dt;
    const bool with_h = g.pre_norm != I8F_NORM_NONE || g.mod_scale || g.mod_shift;
    const Py_ssize_t count = PyTuple_Check(a[16]) ? PyTuple_GET_SIZE(a[16]) : 0;
    Layer l[MAX_FANOUT];
    Size size[MAX_FANOUT];
    Owned work_object;
    const at::Tensor *work = nullptr;
    if (a[16] != Py_None) {
        if (count < 1 || count > MAX_FANOUT || !with_h || dt == I8F_F32 || y.dim() < 2 || M <= 16) Py_RETURN_NONE;
        g.rotate_block = a[20] == Py_True ? 128 : 0;
        if (g.rotate_block && K % 128) Py_RETURN_NONE;
        int64_t narrowest = -1;
        for (int i = 17; i <= 19; ++i)
            if (!PyTuple_Check(a[i]) || PyTuple_GET_SIZE(a[i]) != count) Py_RETURN_NONE;
        for (Py_ssize_t i = 0; i < count; ++i) {
            if (!layer_of(PyTuple_GET_ITEM(a[16], i), PyTuple_GET_ITEM(a[17], i), PyTuple_GET_ITEM(a[18], i), PyTuple_GET_ITEM(a[19], i) == Py_True, y.device(), l[i]) ||
                l[i].K != K)
                Py_RETURN_NONE;
            size[i] = output_size(y, l[i].N);
            narrowest = narrowest < 0 || l[i].N < narrowest ? l[i].N : narrowest;
        }
        if (a[22] != Py_None) {
            work_object.p = PyObject_CallFunction(a[22], "OLLL", a[0], (long long)M, (long long)narrowest, (long long)K);
            if (!work_object.p) return nullptr;
            if (work_object.p != Py_None && !(work = tensor(work_object.p))) Py_RETURN_NONE;
        }
    }
    const int order = (int)PyLong_AsLong(a[21]);
    const at::ScalarType type = y.scalar_type();
    const at::Device dev = y.device();
    const Size shape(y.sizes().begin(), y.sizes().end());
    void *work_p = work ? work->data_ptr() : nullptr;
    const int64_t work_bytes = work ? work->numel() : 0;
    at::Tensor x, h, scratch, outs[MAX_FANOUT];
    int rc;
    {
        const WithoutGil released;
        x = empty(shape, type, dev);
        g.x_out = x.data_ptr();
        if (count) {
            const int64_t q_bytes = (M * K + 255) / 256 * 256;
            scratch = empty({q_bytes + 4 * M}, at::kByte, dev);
            g.q = (int8_t *)scratch.data_ptr(), g.scale = (float *)(g.q + q_bytes);
            for (Py_ssize_t i = 0; i < count; ++i) outs[i] = empty(size[i], type, dev);
        } else if (with_h) {
            h = empty(shape, type, dev);
            g.h = h.data_ptr();
        }
        rc = lib.i8f_block_norm(&g, st.handle);
        if (!rc && count) rc = project(l, (int)count, g.q, g.scale, M, K, dt, order, outs, work_p, work_bytes, st.handle);
    }
    if (rc) Py_RETURN_NONE;
    Owned first, second;
    first.p = THPVariable_Wrap(std::move(x));
    if (count) second.p = list_of(outs, count);
    else if (with_h) second.p = THPVariable_Wrap(std::move(h));
    else Py_INCREF(Py_None), second.p = Py_None;
    if (!first.p || !second.p) return nullptr;
    return PyTuple_Pack(2, first.p, second.p);
}

// No C++ exception leaves an entry point: an allocator that has nothing left, say, becomes the general path's to report.
template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    try {
        PyObject *r = F(self, a, n);
        if (PyErr_Occurred()) {  // an operand that is no number: the general path words it
            PyErr_Clear();
            Py_XDECREF(r);
            Py_RETURN_NONE;
        }
        return r;
    } catch (const std::exception &) {
        Py_RETURN_NONE;
    }
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, "bind(path): load the kernels' library"},
    {"linear", (PyCFunction)(void (*)(void))guarded<linear>, METH_FASTCALL, "one quantised layer, or None"},
    {"fanout", (PyCFunction)(void (*)(void))guarded<fanout>, METH_FASTCALL, "several quantised layers of the same tokens, or None"},
    {"linear_lora", (PyCFunction)(void (*)(void))guarded<linear_lora>, METH_FASTCALL, "one quantised layer with a dynamic LoRA, or None"},
    {"vector_fanout", (PyCFunction)(void (*)(void))guarded<vector_fanout>, METH_FASTCALL, "several small-batch layers, or None"},
    {"adapters", (PyCFunction)(void (*)(void))guarded<adapters>, METH_FASTCALL, "quantised layers with an adapter for each row, or None"},
    {"block_norm", (PyCFunction)(void (*)(void))guarded<block_norm>, METH_FASTCALL, "what lies between two blocks, or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_i8f_host", "Native host path of the INT8 linear layers.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__i8f_host(void) { return PyModule_Create(&module); }

// Native call path of the operators (extension module lib/_b200q_host.so).
//
// An operator call on the ordinary arguments - CUDA tensors on the current device, contiguous, the dtypes and shapes the
// kernels read as they are - is checked, given its outputs and launched here, in a few microseconds of host time.  Every
// other call (a shape that does not match, a dtype to convert, a CPU tensor, a refused backend, an error code) makes the
// function return None, and the Python body of the operator takes it from the start: it holds all conversions and all
// error messages.  Nothing is kept between calls; outputs and scratch come from torch's caching allocator, which orders
// their reuse by stream.
//
// Why native: the Python route (validation, data_ptr() and ctypes conversions, current_stream()) costs about 17 us for a
// matvec whose kernel takes 5 us, and 25 us for an attention call of 13 us (host time per call, one B200 box).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <vector>

namespace {

using at::Tensor;

// addresses of the C ABI functions, handed over by the ctypes loader (the library itself is loaded there)
int (*p_qmatvec)(int, const void*, const uint8_t*, const void*, const void*, const void*, void*, int, int64_t, int64_t, int, int,
                 int, void*) = nullptr;
int (*p_gate_up)(int, const void*, const uint8_t*, const uint8_t*, const void*, const void*, const void*, const void*, void*, void*,
                 void*, const void*, const void*, int, float, void*, void*, int, int64_t, int64_t, int, int, int, void*) = nullptr;
int (*p_scratch_next)(void*, size_t) = nullptr;
size_t (*p_scratch_bytes)(int, int64_t, int) = nullptr;
size_t (*p_attn_ws)(int, int, int, int) = nullptr;
int (*p_attn_launches)(int, int, int) = nullptr;
int (*p_attn)(int, const void*, const uint8_t*, const uint8_t*, const void*, const void*, const int32_t*, const int32_t*, void*,
              void*, size_t, int, int, int, int, int, int64_t, int, int, float, int, int, void*) = nullptr;
int (*p_attn_window)(int, const void*, const uint8_t*, const uint8_t*, const void*, const void*, const int32_t*, const int32_t*,
                     void*, void*, size_t, int, int, int, int, int, int64_t, int, int, float, int, int, int, int, void*) = nullptr;

size_t (*p_plain_ws)(int, int, int, int) = nullptr;
int (*p_plain_attn)(const void*, const void*, const void*, const int32_t*, const int32_t*, void*, void*, size_t, int, int, int, int, int,
                    int64_t, int, float, int, void*) = nullptr;
int (*p_plain_checked)(const void*, const void*, const void*, const int32_t*, const int32_t*, void*, void*, size_t, int, int, int, int, int,
                       int64_t, int, float, int, int32_t*, void*) = nullptr;
int (*p_quant_pair)(int, const void*, const void*, uint8_t*, uint8_t*, void*, void*, int64_t, int, int, int, void*) = nullptr;
int (*p_dequant_pair)(int, const uint8_t*, const uint8_t*, const void*, const void*, void*, void*, int64_t, int, int, void*) = nullptr;

int (*p_head_rope)(const void*, const void*, void*, void*, const int64_t*, const void*, const void*, int, float, const float*, const float*,
                   const int32_t*, int64_t, int, int, int64_t, int, int, int, int, void*) = nullptr;
int (*p_append)(const void*, int64_t, const float*, const float*, int64_t, int, int, const int32_t*, const int32_t*, const int32_t*, int, int,
                const void*, const void*, int, float, void*, int, void*, void*, void*, void*, int64_t, int, int, int, int, int64_t, int, int,
                void*) = nullptr;
size_t (*p_lora_ws)(int64_t, int64_t, int) = nullptr;
int (*p_lora)(int, const void*, const uint8_t*, const void*, const void*, const void*, void*, const void*, const void*, const float*, const int32_t*,
              const int32_t*, int, int64_t, int64_t, int, int, int, int, int, void*, size_t, void*) = nullptr;
size_t (*p_reserve_ws)(int, int64_t) = nullptr;
size_t (*p_copy_ws)(int, int64_t) = nullptr;
size_t (*p_fork_ws)(int, int) = nullptr;
size_t (*p_compact_ws)(int64_t) = nullptr;
int (*p_reserve)(int32_t*, int64_t, int32_t*, const int32_t*, const int32_t*, int, int, int, int, void*, size_t, void*) = nullptr;
int (*p_release)(int32_t*, int64_t, int32_t*, int32_t*, const int32_t*, int, int, int, void*) = nullptr;
int (*p_copy_pages)(void* const*, int, int64_t, void* const*, int, int64_t, const int32_t*, const int32_t*, int, int64_t, int, void*, size_t,
                    void*) = nullptr;
int (*p_fork)(void* const*, int, int64_t, void* const*, int, int64_t, int32_t*, int64_t, int32_t*, int32_t*, const int32_t*, const int32_t*, int,
              int, int, int, void*, size_t, void*) = nullptr;
int (*p_compact)(void* const*, int, int64_t, void* const*, int, int64_t, int32_t*, int64_t, int32_t*, int, int, int, int32_t*, void*, size_t,
                 void*) = nullptr;

constexpr int kMaxDevices = 64;
constexpr int kErrUnsupported = -2, kErrWorkspace = -4;      // B200Q_ERR_*
constexpr int kMinNormRows = 5;      // from this many rows on the library runs the rmsnorm as a launch of its own

PyObject* none() { Py_RETURN_NONE; }

const Tensor* as_tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool safe_mode() {
    const char* v = std::getenv("MLX_METAL_CI_SAFE_MODE");
    return v != nullptr && std::strcmp(v, "1") == 0;
}

int dtype_code(at::ScalarType t) {
    return t == at::kHalf ? 0 : t == at::kBFloat16 ? 1 : t == at::kFloat ? 2 : -1;
}
bool act_dtype(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

bool on(const Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev && t.is_contiguous(); }
bool is_matrix(const Tensor& t, int64_t r, int64_t c) { return t.dim() == 2 && t.size(0) == r && t.size(1) == c; }

// codes [n, row bytes of k], scales and zero points [n, groups] in one dtype
struct Matrix {
    const Tensor *w, *s, *z;
    int64_t n;
};
bool matrix(Matrix& m, PyObject* w, PyObject* s, PyObject* z, int bits, int64_t k, int64_t group, int dev) {
    m.w = as_tensor(w);
    m.s = as_tensor(s);
    m.z = z == Py_None ? nullptr : as_tensor(z);
    if (m.w == nullptr || m.s == nullptr || (m.z == nullptr && z != Py_None)) return false;
    if (m.w->dim() != 2 || m.w->scalar_type() != at::kByte || !on(*m.w, dev)) return false;
    m.n = m.w->size(0);
    if (m.n <= 0 || m.w->size(1) * (bits == 4 ? 2 : 1) != k) return false;
    const int64_t groups = (k + group - 1) / group;
    if (dtype_code(m.s->scalar_type()) < 0 || !on(*m.s, dev) || !is_matrix(*m.s, m.n, groups)) return false;
    return m.z == nullptr || (m.z->scalar_type() == m.s->scalar_type() && on(*m.z, dev) && is_matrix(*m.z, m.n, groups));
}
const void* ptr(const Tensor* t) { return t == nullptr ? nullptr : t->const_data_ptr(); }
const uint8_t* codes(const Tensor* t) { return static_cast<const uint8_t*>(t->const_data_ptr()); }

const int32_t* i32(const Tensor* t) { return static_cast<const int32_t*>(ptr(t)); }

Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, int dev) {
    return at::detail::empty_cuda(shape, dtype, at::Device(at::kCUDA, dev), std::nullopt);
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
// the device of the first tensor when it is the current one (the library launches on the current device), else -1
int current_device_of(const Tensor* t) {
    if (t == nullptr || !t->is_cuda()) return -1;
    const int dev = t->get_device();
    return dev == c10::cuda::current_device() ? dev : -1;
}
bool one_of(PyObject* s, std::initializer_list<const char*> names) {
    if (!PyUnicode_Check(s)) return false;
    for (const char* n : names)
        if (PyUnicode_CompareWithASCIIString(s, n) == 0) return true;
    return false;
}
// a plain int (not a bool or a float that Python's own arithmetic would treat differently)
bool as_int(PyObject* o, int64_t* v) {
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    *v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow == 0;
}

// matvec(bits, x, w, scales, zeros, group_size, backend) -> y or None
PyObject* matvec(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    int64_t bits, group;
    if (p_qmatvec == nullptr || n_args != 7 || !as_int(a[0], &bits) || !as_int(a[5], &group) || group <= 0) return none();
    if (!one_of(a[6], {"cuda", "auto", "metal", "metal_tiled", "metal_parallel"}) || safe_mode()) return none();
    const Tensor* x = as_tensor(a[1]);
    const int dev = current_device_of(x);
    if (dev < 0 || !x->is_contiguous() || !act_dtype(x->scalar_type())) return none();
    if (!(x->dim() == 2 || (x->dim() == 3 && x->size(1) == 1))) return none();
    const int64_t B = x->size(0), K = x->size(x->dim() - 1);
    Matrix m;
    if (B <= 0 || B > INT32_MAX || K <= 0 || !matrix(m, a[2], a[3], a[4], (int)bits, K, group, dev)) return none();
    Tensor y = empty({B, m.n}, x->scalar_type(), dev), scratch;
    const size_t scratch_bytes = p_scratch_bytes((int)B, K, dtype_code(x->scalar_type()));
    if (scratch_bytes) scratch = empty({(int64_t)scratch_bytes}, at::kByte, dev);
    p_scratch_next(scratch_bytes ? scratch.mutable_data_ptr() : nullptr, scratch_bytes);      // the call below takes it, always
    const int rc = p_qmatvec((int)bits, x->const_data_ptr(), codes(m.w), ptr(m.s), ptr(m.z), nullptr, y.mutable_data_ptr(), (int)B, m.n,
                             K, (int)group, dtype_code(x->scalar_type()), dtype_code(m.s->scalar_type()), stream_of(dev));
    return rc == 0 ? THPVariable_Wrap(std::move(y)) : none();
}

// mlp_block(x, residual, norm_weight, gw, gs, gz, uw, us, uz, dw, ds, dz, bits, group_size, eps) -> out or None
PyObject* mlp_block(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    int64_t bits, group;
    if (p_gate_up == nullptr || n_args != 15 || !as_int(a[12], &bits) || !as_int(a[13], &group) || group <= 0 ||
        (bits != 4 && bits != 8) || !PyFloat_Check(a[14]) || safe_mode())
        return none();
    const Tensor *x = as_tensor(a[0]), *res = as_tensor(a[1]), *nw = as_tensor(a[2]);
    const int dev = current_device_of(x);
    if (dev < 0 || res == nullptr || nw == nullptr || x->dim() != 3 || x->sizes() != res->sizes() || !x->is_contiguous() ||
        !on(*res, dev) || !on(*nw, dev) || !act_dtype(x->scalar_type()) || res->scalar_type() != x->scalar_type() ||
        dtype_code(nw->scalar_type()) < 0)
        return none();
    const int64_t D = x->size(2), rows = x->size(0) * x->size(1);
    if (rows <= 0 || rows > INT32_MAX || nw->dim() != 1 || nw->size(0) != D) return none();
    Matrix g, u, d;
    if (!matrix(g, a[3], a[4], a[5], (int)bits, D, group, dev) || !matrix(u, a[6], a[7], a[8], (int)bits, D, group, dev) || u.n != g.n ||
        !matrix(d, a[9], a[10], a[11], (int)bits, g.n, group, dev) || d.n != D || u.s->scalar_type() != g.s->scalar_type() ||
        (u.z != nullptr && u.z->scalar_type() != g.s->scalar_type()))
        return none();
    const int act = dtype_code(x->scalar_type());
    void* st = stream_of(dev);
    // one scratch block: z [rows, D], the SwiGLU rows [rows, inter], and the normalised rows where the library wants them
    const int64_t zb = (rows * D * 2 + 255) / 256 * 256, mb = (rows * g.n * 2 + 255) / 256 * 256;
    const bool want_normed = rows >= kMinNormRows;
    const size_t xb = std::max(p_scratch_bytes((int)rows, D, act), p_scratch_bytes((int)rows, g.n, act));
    Tensor scratch = empty({zb + mb + (want_normed ? zb : 0) + (int64_t)xb}, at::kByte, dev);
    uint8_t* z = static_cast<uint8_t*>(scratch.mutable_data_ptr());
    uint8_t *mlp = z + zb, *normed = want_normed ? mlp + mb : nullptr;
    Tensor out = empty(x->sizes(), x->scalar_type(), dev);
    void* xs = xb ? z + zb + mb + (want_normed ? zb : 0) : nullptr;
    const float eps = (float)PyFloat_AS_DOUBLE(a[14]);
    p_scratch_next(xs, xb);
    int rc = p_gate_up((int)bits, x->const_data_ptr(), codes(g.w), codes(u.w), ptr(g.s), ptr(u.s), ptr(g.z), ptr(u.z), nullptr, nullptr,
                       mlp, res->const_data_ptr(), nw->const_data_ptr(), dtype_code(nw->scalar_type()), eps, z, normed, (int)rows, g.n,
                       D, (int)group, act, dtype_code(g.s->scalar_type()), st);
    if (rc != 0) return none();
    p_scratch_next(xs, xb);
    rc = p_qmatvec((int)bits, mlp, codes(d.w), ptr(d.s), ptr(d.z), z, out.mutable_data_ptr(), (int)rows, D, g.n, (int)group, act,
                   dtype_code(d.s->scalar_type()), st);
    return rc == 0 ? THPVariable_Wrap(std::move(out)) : none();
}

PyObject *s_bits, *s_group_size, *s_shape, *s_kq, *s_vq, *s_ks, *s_vs, *s_bt, *s_len;

// Owned attribute, released at scope end.
struct Attr {
    PyObject* o;
    Attr(PyObject* obj, PyObject* name) : o(PyObject_GetAttr(obj, name)) {
        if (o == nullptr) PyErr_Clear();
    }
    ~Attr() { Py_XDECREF(o); }
    Attr(const Attr&) = delete;
};

// paged_attention(q, cache, scale or None, sink_tokens, window_size) -> out or None
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    int64_t sink, window;
    if (p_attn == nullptr || n_args != 5 || !as_int(a[3], &sink) || !as_int(a[4], &window)) return none();
    const Tensor* q = as_tensor(a[0]);
    const int dev = current_device_of(q);
    if (dev < 0 || q->dim() != 4 || q->size(1) != 1 || !q->is_contiguous() || !act_dtype(q->scalar_type())) return none();
    const int64_t B = q->size(0), Hq = q->size(2), D = q->size(3);
    Attr bits_o(a[1], s_bits), group_o(a[1], s_group_size), shape(a[1], s_shape), kq_o(a[1], s_kq), vq_o(a[1], s_vq), ks_o(a[1], s_ks),
        vs_o(a[1], s_vs), bt_o(a[1], s_bt), len_o(a[1], s_len);
    int64_t bits, group, dims[4];
    if (bits_o.o == nullptr || group_o.o == nullptr || shape.o == nullptr || kq_o.o == nullptr || vq_o.o == nullptr ||
        ks_o.o == nullptr || vs_o.o == nullptr || bt_o.o == nullptr || len_o.o == nullptr)
        return none();
    if (!as_int(bits_o.o, &bits) || !as_int(group_o.o, &group) || (bits != 4 && bits != 8) || group <= 0 || !PyTuple_Check(shape.o) ||
        PyTuple_GET_SIZE(shape.o) != 4)
        return none();
    for (int i = 0; i < 4; ++i)
        if (!as_int(PyTuple_GET_ITEM(shape.o, i), &dims[i]) || dims[i] <= 0) return none();
    const int64_t pages = dims[0], P = dims[1], Hkv = dims[2];
    const Tensor *kq = as_tensor(kq_o.o), *vq = as_tensor(vq_o.o), *ks = as_tensor(ks_o.o), *vs = as_tensor(vs_o.o),
                 *bt = as_tensor(bt_o.o), *len = as_tensor(len_o.o);
    if (!kq || !vq || !ks || !vs || !bt || !len || !on(*kq, dev) || !on(*vq, dev) || !on(*ks, dev) || !on(*vs, dev) || !on(*bt, dev) ||
        !on(*len, dev))
        return none();
    const int64_t slots = pages * P * Hkv, dp = bits == 4 ? (D + 1) / 2 : D, gd = (D + group - 1) / group;
    if (B <= 0 || Hq <= 0 || D <= 0 || D > 128 || D != dims[3] || Hq < Hkv || Hq % Hkv != 0 || kq->scalar_type() != at::kByte ||
        vq->scalar_type() != at::kByte || kq->numel() != slots * dp || vq->numel() != slots * dp || ks->numel() != slots * gd ||
        vs->numel() != slots * gd || dtype_code(ks->scalar_type()) < 0 || vs->scalar_type() != ks->scalar_type() ||
        bt->scalar_type() != at::kInt || bt->dim() != 2 || bt->size(0) != B || len->scalar_type() != at::kInt || len->numel() != B ||
        B > INT32_MAX || Hq > INT32_MAX || P > INT32_MAX || bt->size(1) > INT32_MAX || bt->size(1) <= 0)
        return none();
    double scale = 1.0 / std::sqrt((double)D);
    if (a[2] != Py_None) {
        if (!PyFloat_Check(a[2])) return none();
        scale = PyFloat_AS_DOUBLE(a[2]);
    }
    Tensor out = empty(q->sizes(), q->scalar_type(), dev);
    // scratch for split-KV partial results; the one-launch cluster kernel of small dense batches needs none
    Tensor ws;
    size_t ws_bytes = 0;
    if (window > 0 || p_attn_launches((int)B, (int)Hkv, 0) > 1) {
        ws_bytes = p_attn_ws((int)B, (int)Hq, (int)Hkv, (int)D);
        ws = empty({(int64_t)ws_bytes}, at::kByte, dev);
    }
    void* wp = ws_bytes ? ws.mutable_data_ptr() : nullptr;
    const int act = dtype_code(q->scalar_type()), sdt = dtype_code(ks->scalar_type()), mb = (int)bt->size(1);
    const int rc = window > 0
        ? p_attn_window((int)bits, q->const_data_ptr(), codes(kq), codes(vq), ptr(ks), ptr(vs), i32(bt), i32(len), out.mutable_data_ptr(), wp,
                        ws_bytes, (int)B, (int)Hq, (int)Hkv, (int)D, (int)P, pages, mb, (int)group, (float)scale, act, sdt, (int)sink,
                        (int)window, stream_of(dev))
        : p_attn((int)bits, q->const_data_ptr(), codes(kq), codes(vq), ptr(ks), ptr(vs), i32(bt), i32(len), out.mutable_data_ptr(), wp,
                 ws_bytes, (int)B, (int)Hq, (int)Hkv, (int)D, (int)P, pages, mb, (int)group, (float)scale, act, sdt, stream_of(dev));
    return rc == 0 ? THPVariable_Wrap(std::move(out)) : none();
}

// Queries and waits on a stream are refused to every thread while one captures a graph in the default mode, unless the thread asks
// for the relaxed one.
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
// Memory that a kernel on the stream may still write to goes back to its allocator when the stream has ended; if even the wait
// fails it is kept for good.
void release_after_stream(Tensor word, cudaStream_t st) {
    cudaError_t err;
    Py_BEGIN_ALLOW_THREADS
    const RelaxedCapture relaxed;
    err = cudaStreamSynchronize(st);
    Py_END_ALLOW_THREADS
    if (err != cudaSuccess) new Tensor(std::move(word));
}

// plain_attention(q, K, V, block_table, lengths, scale or None) -> out or None: fp16 / bf16 pages.  The lengths are
// range-checked on the host, as the operator promises.  The split-KV kernel reports on them at its start, into pinned memory that
// the host polls while the GPU goes on (a copy on the stream took 10 of 42 us per call at 16 sequences: it kept the kernel from
// starting under the one before).  Elsewhere they are copied out ahead of the kernels, which clamp what they read,
// and the host waits for that copy once the kernels are enqueued.
PyObject* plain_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (p_plain_attn == nullptr || n_args != 6 || safe_mode()) return none();
    const Tensor *q = as_tensor(a[0]), *k = as_tensor(a[1]), *v = as_tensor(a[2]), *bt = as_tensor(a[3]), *len = as_tensor(a[4]);
    const int dev = current_device_of(q);
    if (dev < 0 || dev >= kMaxDevices || !k || !v || !bt || !len || q->dim() != 4 || q->size(1) != 1 || !q->is_contiguous() ||
        !act_dtype(q->scalar_type()))
        return none();
    const int64_t B = q->size(0), Hq = q->size(2), D = q->size(3);
    if (!on(*k, dev) || !on(*v, dev) || !on(*bt, dev) || !on(*len, dev) || k->dim() != 4 || k->sizes() != v->sizes() ||
        k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->size(3) != D || bt->dim() != 2 ||
        bt->size(0) != B || bt->scalar_type() != at::kInt || len->scalar_type() != at::kInt || len->dim() != 1 || len->size(0) != B)
        return none();
    const int64_t pages = k->size(0), P = k->size(1), Hkv = k->size(2), mb = bt->size(1);
    if (B <= 0 || Hq <= 0 || D <= 0 || D > 128 || pages <= 0 || P <= 0 || Hkv <= 0 || mb <= 0 || Hq % Hkv != 0 || B > INT32_MAX ||
        Hq > INT32_MAX || P * mb > INT32_MAX)
        return none();
    double scale = 1.0 / std::sqrt((double)D);
    if (a[5] != Py_None) {
        if (!PyFloat_Check(a[5])) return none();
        scale = PyFloat_AS_DOUBLE(a[5]);
    }
    cudaStream_t st = (cudaStream_t)stream_of(dev);
    cudaStreamCaptureStatus capture;
    if (cudaStreamIsCapturing(st, &capture) != cudaSuccess || capture != cudaStreamCaptureStatusNone) return none();
    Tensor out = empty(q->sizes(), q->scalar_type(), dev);
    const size_t ws_bytes = p_plain_ws((int)B, (int)Hq, (int)Hkv, (int)mb);
    Tensor ws = empty({(int64_t)std::max<size_t>(ws_bytes, 16)}, at::kByte, dev);
    if (D == 128 && P == 16) {
        Tensor word = at::detail::empty_cpu({1}, at::kInt, std::nullopt, std::nullopt, /*pin_memory=*/true, std::nullopt);
        volatile int32_t* verdict = static_cast<volatile int32_t*>(word.mutable_data_ptr());
        *verdict = 0;
        const int rc = p_plain_checked(q->const_data_ptr(), k->const_data_ptr(), v->const_data_ptr(), static_cast<const int32_t*>(bt->const_data_ptr()),
                                       static_cast<const int32_t*>(len->const_data_ptr()), out.mutable_data_ptr(), ws.mutable_data_ptr(), ws_bytes,
                                       (int)B, (int)Hq, (int)Hkv, (int)D, (int)P, pages, (int)mb, (float)scale, dtype_code(q->scalar_type()),
                                       const_cast<int32_t*>(verdict), st);
        if (rc == 0) {
            Py_BEGIN_ALLOW_THREADS
            // the stream is asked now and then, so that a kernel that never ran (an earlier error) ends the wait
            const RelaxedCapture relaxed;
            for (uint32_t i = 1; *verdict == 0; ++i) {
                if (i % 4096 == 0 && cudaStreamQuery(st) != cudaErrorNotReady) break;
                __builtin_ia32_pause();
            }
            Py_END_ALLOW_THREADS
            if (*verdict == 0) release_after_stream(word, st);
            return *verdict == 1 ? THPVariable_Wrap(std::move(out)) : none();      // 2: the Python body raises
        }
        if (rc != kErrUnsupported && rc != kErrWorkspace) {      // nothing is launched with these two; else the main kernel may be
            release_after_stream(word, st);
            return none();
        }
    }
    static thread_local cudaEvent_t copied[kMaxDevices] = {};      // one per thread and device that ever calls this
    if (copied[dev] == nullptr && cudaEventCreateWithFlags(&copied[dev], cudaEventDisableTiming) != cudaSuccess) return none();
    Tensor host = at::detail::empty_cpu({B}, at::kInt, std::nullopt, std::nullopt, /*pin_memory=*/true, std::nullopt);
    if (cudaMemcpyAsync(host.mutable_data_ptr(), len->const_data_ptr(), (size_t)B * 4, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaEventRecord(copied[dev], st) != cudaSuccess) {
        release_after_stream(host, st);
        return none();
    }
    const int rc = p_plain_attn(q->const_data_ptr(), k->const_data_ptr(), v->const_data_ptr(), static_cast<const int32_t*>(bt->const_data_ptr()),
                                static_cast<const int32_t*>(len->const_data_ptr()), out.mutable_data_ptr(), ws.mutable_data_ptr(), ws_bytes,
                                (int)B, (int)Hq, (int)Hkv, (int)D, (int)P, pages, (int)mb, (float)scale, dtype_code(q->scalar_type()), st);
    cudaError_t err;
    Py_BEGIN_ALLOW_THREADS
    const RelaxedCapture relaxed;
    err = cudaEventSynchronize(copied[dev]);
    Py_END_ALLOW_THREADS
    if (err != cudaSuccess) release_after_stream(host, st);
    if (rc != 0 || err != cudaSuccess) return none();
    const int32_t* n = static_cast<const int32_t*>(host.const_data_ptr());
    for (int64_t b = 0; b < B; ++b)
        if (n[b] < 0 || n[b] > mb * P) return none();              // the Python body raises
    return THPVariable_Wrap(std::move(out));
}

PyObject* tuple_of(std::initializer_list<Tensor*> ts) {
    PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (Tensor* t : ts) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(std::move(*t)));
    return out;
}

// quantize_kv(K, V, bits, group_size) -> (k codes, v codes, k scales, v scales) or None; K, V [..., D] of one shape
PyObject* quantize_kv(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    int64_t bits, group;
    if (p_quant_pair == nullptr || n_args != 4 || !as_int(a[2], &bits) || !as_int(a[3], &group) || (bits != 4 && bits != 8) || group <= 0)
        return none();
    const Tensor *k = as_tensor(a[0]), *v = as_tensor(a[1]);
    const int dev = current_device_of(k);
    if (dev < 0 || v == nullptr || k->dim() < 1 || k->sizes() != v->sizes() || !on(*k, dev) || !on(*v, dev) || !act_dtype(k->scalar_type()) ||
        v->scalar_type() != k->scalar_type() || k->numel() == 0)
        return none();
    const int64_t D = k->size(-1);
    if (D > INT32_MAX || group > INT32_MAX) return none();
    std::vector<int64_t> shape(k->sizes().begin(), k->sizes().end());
    shape.back() = bits == 4 ? (D + 1) / 2 : D;
    Tensor kc = empty(shape, at::kByte, dev), vc = empty(shape, at::kByte, dev);
    shape.back() = (D + group - 1) / group;
    Tensor ks = empty(shape, at::kHalf, dev), vs = empty(shape, at::kHalf, dev);
    const auto u8 = [](Tensor& t) { return static_cast<uint8_t*>(t.mutable_data_ptr()); };
    const int rc = p_quant_pair((int)bits, k->const_data_ptr(), v->const_data_ptr(), u8(kc), u8(vc), ks.mutable_data_ptr(),
                                vs.mutable_data_ptr(), k->numel() / D, (int)D, (int)group, dtype_code(k->scalar_type()), stream_of(dev));
    return rc == 0 ? tuple_of({&kc, &vc, &ks, &vs}) : none();
}

// dequantize_kv(k codes, v codes, k scales, v scales, bits, group_size, shape) -> (K, V) fp16 of `shape`, or None
PyObject* dequantize_kv(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    int64_t bits, group;
    if (p_dequant_pair == nullptr || n_args != 7 || !as_int(a[4], &bits) || !as_int(a[5], &group) || (bits != 4 && bits != 8) ||
        group <= 0 || !PyTuple_Check(a[6]))
        return none();
    const Tensor *kc = as_tensor(a[0]), *vc = as_tensor(a[1]), *ks = as_tensor(a[2]), *vs = as_tensor(a[3]);
    const int dev = current_device_of(kc);
    if (dev < 0 || !vc || !ks || !vs || !on(*kc, dev) || !on(*vc, dev) || !on(*ks, dev) || !on(*vs, dev) || kc->scalar_type() != at::kByte ||
        vc->scalar_type() != at::kByte || ks->scalar_type() != at::kHalf || vs->scalar_type() != at::kHalf)
        return none();
    std::vector<int64_t> shape((size_t)PyTuple_GET_SIZE(a[6]));
    int64_t n = 1;
    for (size_t i = 0; i < shape.size(); ++i) {
        if (!as_int(PyTuple_GET_ITEM(a[6], i), &shape[i]) || shape[i] <= 0) return none();
        n *= shape[i];
    }
    if (shape.empty() || shape.back() > INT32_MAX || group > INT32_MAX) return none();
    const int64_t D = shape.back(), rows = n / D, dp = bits == 4 ? (D + 1) / 2 : D, gd = (D + group - 1) / group;
    if (kc->numel() != rows * dp || vc->numel() != rows * dp || ks->numel() != rows * gd || vs->numel() != rows * gd) return none();
    Tensor k = empty(shape, at::kHalf, dev), v = empty(shape, at::kHalf, dev);
    const int rc = p_dequant_pair((int)bits, codes(kc), codes(vc), ptr(ks), ptr(vs), k.mutable_data_ptr(), v.mutable_data_ptr(), rows, (int)D,
                                  (int)group, stream_of(dev));
    return rc == 0 ? tuple_of({&k, &v}) : none();
}

// What the rotation operators share: tables, positions, norm weights and layout on one device.
struct Rotation {
    const Tensor *cos, *sin, *pos, *qw, *kw;
    int w_dtype = 2, half = 0;
    float eps = 0.0f;
};
bool rotation(Rotation& r, PyObject* cos, PyObject* sin, PyObject* pos, PyObject* qw, PyObject* kw, PyObject* eps, PyObject* layout, int64_t D,
              int dev) {
    r.cos = as_tensor(cos);
    r.sin = as_tensor(sin);
    r.pos = as_tensor(pos);
    r.qw = as_tensor(qw);
    r.kw = as_tensor(kw);
    if (!r.cos || !r.sin || !r.pos || (!r.qw && qw != Py_None) || (!r.kw && kw != Py_None) || !PyFloat_Check(eps)) return false;
    r.eps = (float)PyFloat_AS_DOUBLE(eps);
    r.half = one_of(layout, {"half"}) ? 1 : 0;
    if (!(r.eps >= 0.0f) || (!r.half && !one_of(layout, {"interleaved"}))) return false;
    if (!on(*r.cos, dev) || !on(*r.sin, dev) || !on(*r.pos, dev) || r.cos->dim() != 2 || r.cos->sizes() != r.sin->sizes() ||
        r.cos->scalar_type() != at::kFloat || r.sin->scalar_type() != at::kFloat || r.pos->scalar_type() != at::kInt)
        return false;
    if (r.cos->size(0) <= 0 || r.cos->size(1) <= 0 || 2 * r.cos->size(1) > D || D > 1024) return false;
    for (const Tensor* w : {r.qw, r.kw}) {
        if (w == nullptr) continue;
        if (!on(*w, dev) || w->dim() != 1 || w->size(0) != D || dtype_code(w->scalar_type()) < 0) return false;
        r.w_dtype = dtype_code(w->scalar_type());
    }
    return r.qw == nullptr || r.kw == nullptr || r.qw->scalar_type() == r.kw->scalar_type();
}
const float* f32(const Tensor* t) { return static_cast<const float*>(t->const_data_ptr()); }

// stride of the tokens of x [..., H, D] with contiguous heads when the leading dimensions (one or two) have one; else false
bool token_stride(const Tensor& x, int64_t* stride) {
    const int64_t n = x.dim();
    if (x.stride(n - 1) != 1 && x.size(n - 1) != 1) return false;
    if (n == 4 && x.size(0) != 1 && x.stride(0) != x.size(1) * x.stride(1)) return false;
    *stride = x.stride(n - 3);
    return true;
}

// head_rope(q, k or None, q_weight or None, k_weight or None, cos, sin, positions, eps, layout) -> (q, k or None) or None
PyObject* head_rope(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (p_head_rope == nullptr || n_args != 9) return none();
    const Tensor *q = as_tensor(a[0]), *k = as_tensor(a[1]);
    const int dev = current_device_of(q);
    if (dev < 0 || (k == nullptr && a[1] != Py_None) || (q->dim() != 3 && q->dim() != 4) || !act_dtype(q->scalar_type())) return none();
    const int64_t n = q->dim(), Hq = q->size(n - 2), D = q->size(n - 1), Hkv = k == nullptr ? 0 : k->size(n - 2);
    int64_t T = 1, qs = 0, ks = 0;
    for (int64_t i = 0; i < n - 2; ++i) T *= q->size(i);
    Rotation r;
    if (T <= 0 || Hq <= 0 || D <= 0 || Hq > INT32_MAX || Hkv > INT32_MAX || !token_stride(*q, &qs) ||
        !rotation(r, a[4], a[5], a[6], a[2], a[3], a[7], a[8], D, dev))
        return none();
    if (r.pos->sizes() != q->sizes().slice(0, n - 2)) return none();
    if (k != nullptr && (!k->is_cuda() || k->get_device() != dev || k->dim() != n || k->scalar_type() != q->scalar_type() || Hkv <= 0 ||
                         k->size(n - 1) != D || k->sizes().slice(0, n - 2) != q->sizes().slice(0, n - 2) || !token_stride(*k, &ks)))
        return none();
    Tensor qo = empty(q->sizes(), q->scalar_type(), dev), ko;
    if (k != nullptr) ko = empty(k->sizes(), k->scalar_type(), dev);
    const int64_t strides[8] = {qs, q->stride(n - 2), Hq * D, D, ks, k == nullptr ? 0 : k->stride(n - 2), Hkv * D, D};
    const int rc = p_head_rope(q->const_data_ptr(), ptr(k), qo.mutable_data_ptr(), k == nullptr ? nullptr : ko.mutable_data_ptr(), strides,
                               ptr(r.qw), ptr(r.kw), r.w_dtype, r.eps, f32(r.cos), f32(r.sin), i32(r.pos), r.cos->size(0),
                               (int)(2 * r.cos->size(1)), r.half, T, (int)Hq, (int)Hkv, (int)D, dtype_code(q->scalar_type()), stream_of(dev));
    if (rc != 0) return none();
    PyObject* out = PyTuple_New(2);
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(qo)));
    if (k == nullptr) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 1, k == nullptr ? Py_None : THPVariable_Wrap(std::move(ko)));
    return out;
}

// What both append operators share, a: qkv, cos, sin, positions, n_heads, sequences or None, q_weight, k_weight, eps, layout; pages and
// scales (null for plain pages) of the shape `dims`.
PyObject* append_rows(PyObject* const* a, const Tensor* bt, const Tensor* kp, const Tensor* vp, const Tensor* ks, const Tensor* vs, const int64_t* dims,
                      int64_t bits, int64_t group) {
    int64_t Hq;
    if (!as_int(a[4], &Hq)) return none();
    const int64_t pages = dims[0], P = dims[1], Hkv = dims[2], D = dims[3];
    if (pages <= 0 || P <= 0 || Hkv <= 0 || D <= 0) return none();
    const Tensor *x = as_tensor(a[0]), *seq = as_tensor(a[5]);
    const int dev = current_device_of(x);
    if (dev < 0 || bt == nullptr || (seq == nullptr && a[5] != Py_None) || x->dim() != 2 || !act_dtype(x->scalar_type()) || Hq <= 0 ||
        Hq > INT32_MAX || Hkv > INT32_MAX || P > INT32_MAX || x->size(0) <= 0 || x->size(1) != (Hq + 2 * Hkv) * D || x->stride(1) != 1 ||
        x->stride(0) < x->size(1))
        return none();
    const int64_t T = x->size(0);
    Rotation r;
    if (!rotation(r, a[1], a[2], a[3], a[6], a[7], a[8], a[9], D, dev) || r.pos->dim() != 1 || r.pos->size(0) != T) return none();
    if (!on(*bt, dev) || bt->scalar_type() != at::kInt || bt->dim() != 2 || bt->size(0) <= 0 || bt->size(1) <= 0 || bt->size(0) > INT32_MAX ||
        bt->size(1) > INT32_MAX)
        return none();
    if (seq == nullptr ? T != bt->size(0) : !on(*seq, dev) || seq->scalar_type() != at::kInt || seq->dim() != 1 || seq->size(0) != T) return none();
    const bool plain = bits == 16;
    if (!plain && ((bits != 4 && bits != 8) || group <= 0 || group > INT32_MAX)) return none();
    const int64_t slots = pages * P * Hkv, width = bits == 4 ? (D + 1) / 2 : D;
    for (const Tensor* t : {kp, vp})
        if (t == nullptr || !on(*t, dev) || t->scalar_type() != (plain ? x->scalar_type() : at::kByte) || t->dim() != 4 || t->size(0) != pages ||
            t->size(1) != P || t->size(2) != Hkv || t->size(3) != width)
            return none();
    for (const Tensor* t : {ks, vs})
        if (!plain && (t == nullptr || !on(*t, dev) || t->scalar_type() != at::kHalf || t->dim() != 4 || t->size(0) != pages || t->size(1) != P ||
                       t->size(2) != Hkv || t->numel() != slots * ((D + group - 1) / group)))
            return none();
    Tensor out = empty({T, Hq, D}, x->scalar_type(), dev);
    const auto w = [](const Tensor* t) { return t == nullptr ? nullptr : t->mutable_data_ptr(); };
    const int rc = p_append(x->const_data_ptr(), x->stride(0), f32(r.cos), f32(r.sin), r.cos->size(0), (int)(2 * r.cos->size(1)), r.half,
                            i32(r.pos), i32(seq), i32(bt), (int)bt->size(0), (int)bt->size(1), ptr(r.qw), ptr(r.kw), r.w_dtype, r.eps,
                            out.mutable_data_ptr(), (int)bits, w(kp), w(vp), plain ? nullptr : w(ks), plain ? nullptr : w(vs), T, (int)Hq,
                            (int)Hkv, (int)D, (int)P, pages, plain ? 0 : (int)group, dtype_code(x->scalar_type()), stream_of(dev));
    return rc == 0 ? THPVariable_Wrap(std::move(out)) : none();
}

// norm_rope_append(qkv, cos, sin, positions, n_heads, sequences, q_weight, k_weight, eps, layout, cache) -> q or None: quantised pages
PyObject* norm_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (p_append == nullptr || n_args != 11) return none();
    Attr bits_o(a[10], s_bits), group_o(a[10], s_group_size), shape(a[10], s_shape), kq(a[10], s_kq), vq(a[10], s_vq), ks(a[10], s_ks), vs(a[10], s_vs),
        bt(a[10], s_bt);
    for (PyObject* o : {bits_o.o, group_o.o, shape.o, kq.o, vq.o, ks.o, vs.o, bt.o})
        if (o == nullptr) return none();
    int64_t bits, group, dims[4];
    if (!as_int(bits_o.o, &bits) || !as_int(group_o.o, &group) || (bits != 4 && bits != 8) || !PyTuple_Check(shape.o) || PyTuple_GET_SIZE(shape.o) != 4)
        return none();
    for (int i = 0; i < 4; ++i)
        if (!as_int(PyTuple_GET_ITEM(shape.o, i), &dims[i])) return none();
    return append_rows(a, as_tensor(bt.o), as_tensor(kq.o), as_tensor(vq.o), as_tensor(ks.o), as_tensor(vs.o), dims, bits, group);
}

// norm_rope_append_pages(..., layout, K_pages, V_pages, block_table) -> q or None: plain pages
PyObject* norm_rope_append_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (p_append == nullptr || n_args != 13) return none();
    const Tensor *kp = as_tensor(a[10]), *vp = as_tensor(a[11]);
    if (kp == nullptr || kp->dim() != 4) return none();
    const int64_t dims[4] = {kp->size(0), kp->size(1), kp->size(2), kp->size(3)};
    return append_rows(a, as_tensor(a[12]), kp, vp, nullptr, nullptr, dims, 16, 0);
}

PyObject *s_a, *s_b, *s_scaling, *s_ranks, *s_kz, *s_vz;

// lora_linear(bits, x, w, scales, zeros, group_size, backend, adapters, adapter_ids, residual or None) -> y or None
PyObject* lora_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    int64_t bits, group;
    if (p_lora == nullptr || n_args != 10 || !as_int(a[0], &bits) || !as_int(a[5], &group) || group <= 0 || (bits != 4 && bits != 8)) return none();
    if (!one_of(a[6], {"cuda", "auto", "metal", "metal_tiled", "metal_parallel"}) || safe_mode()) return none();
    const Tensor *x = as_tensor(a[1]), *ids = as_tensor(a[8]), *res = as_tensor(a[9]);
    const int dev = current_device_of(x);
    if (dev < 0 || ids == nullptr || (res == nullptr && a[9] != Py_None) || !x->is_contiguous() || !act_dtype(x->scalar_type()) ||
        (x->dim() != 2 && x->dim() != 3))
        return none();
    const int64_t n = x->dim(), K = x->size(n - 1), rows = n == 2 ? x->size(0) : x->size(0) * x->size(1);
    Matrix m;
    if (rows <= 0 || rows > INT32_MAX || K <= 0 || !matrix(m, a[2], a[3], a[4], (int)bits, K, group, dev)) return none();
    if (!on(*ids, dev) || ids->scalar_type() != at::kInt || ids->sizes() != x->sizes().slice(0, n - 1)) return none();
    if (res != nullptr && (!on(*res, dev) || res->scalar_type() != x->scalar_type() || res->dim() != n || res->numel() != rows * m.n ||
                           res->sizes().slice(0, n - 1) != x->sizes().slice(0, n - 1)))
        return none();
    Attr fa(a[7], s_a), fb(a[7], s_b), fs(a[7], s_scaling), fr(a[7], s_ranks);
    if (fa.o == nullptr || fb.o == nullptr || fs.o == nullptr || fr.o == nullptr) return none();
    const Tensor *la = as_tensor(fa.o), *lb = as_tensor(fb.o), *ls = as_tensor(fs.o), *lr = as_tensor(fr.o);
    if (la == nullptr || lb == nullptr || (ls == nullptr && fs.o != Py_None) || (lr == nullptr && fr.o != Py_None)) return none();
    if (!on(*la, dev) || !on(*lb, dev) || la->scalar_type() != x->scalar_type() || lb->scalar_type() != x->scalar_type() || la->dim() != 3 ||
        lb->dim() != 3 || la->size(2) != K || lb->size(1) != m.n || la->size(0) != lb->size(0) || la->size(1) != lb->size(2) || la->numel() == 0 ||
        la->size(0) > INT32_MAX || la->size(1) > INT32_MAX)
        return none();
    const int64_t L = la->size(0), R = la->size(1);
    if (ls != nullptr && (!on(*ls, dev) || ls->scalar_type() != at::kFloat || ls->dim() != 1 || ls->size(0) != L)) return none();
    if (lr != nullptr && (!on(*lr, dev) || lr->scalar_type() != at::kInt || lr->dim() != 1 || lr->size(0) != L)) return none();
    const int act = dtype_code(x->scalar_type());
    void* st = stream_of(dev);
    // one scratch block for the adapters' rows and for the matvec
    const size_t lora_bytes = (p_lora_ws(rows, m.n, (int)R) + 255) / 256 * 256, mat_bytes = p_scratch_bytes((int)rows, K, act);
    Tensor scratch = empty({(int64_t)(lora_bytes + mat_bytes)}, at::kByte, dev);
    uint8_t* low = static_cast<uint8_t*>(scratch.mutable_data_ptr());
    std::vector<int64_t> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = m.n;
    Tensor y = empty(shape, x->scalar_type(), dev);
    p_scratch_next(mat_bytes ? low + lora_bytes : nullptr, mat_bytes);      // the call below takes it, always
    const int rc = p_lora((int)bits, x->const_data_ptr(), codes(m.w), ptr(m.s), ptr(m.z), ptr(res), y.mutable_data_ptr(), la->const_data_ptr(),
                          lb->const_data_ptr(), ls == nullptr ? nullptr : f32(ls), i32(lr), i32(ids), (int)rows, m.n, K, (int)group, (int)L, (int)R, act,
                          dtype_code(m.s->scalar_type()), low, lora_bytes, st);
    return rc == 0 ? THPVariable_Wrap(std::move(y)) : none();
}

// ---- pages of the caches of all layers ----
// The tensors of one call: two groups of one shape each, (codes or values) and scales.
struct Layers {
    std::vector<void*> base[2];
    const Tensor* like[2] = {nullptr, nullptr};
    int64_t slot[2] = {0, 0};
    std::vector<PyObject*> owned;      // attributes, released with the struct: the caches hold them meanwhile
    ~Layers() {
        for (PyObject* o : owned) Py_DECREF(o);
    }
};
bool add_layer_tensor(Layers& l, int group, PyObject* o, int dev) {
    const Tensor* t = as_tensor(o);
    if (t == nullptr || !on(*t, dev) || t->dim() != 4 || t->numel() == 0) return false;
    const Tensor*& like = l.like[group];
    if (like == nullptr) like = t;
    else if (t->sizes() != like->sizes() || t->scalar_type() != like->scalar_type()) return false;
    l.base[group].push_back(const_cast<void*>(t->const_data_ptr()));
    return true;
}
// caches: a list or tuple of pairs of tensors or of quantised caches, all of one kind
bool layers_of(Layers& l, PyObject* caches, int64_t num_pages, int64_t page_size, int dev) {
    if (!PyList_Check(caches) && !PyTuple_Check(caches)) return false;
    PyObject** items = PySequence_Fast_ITEMS(caches);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(caches);
    if (n <= 0 || n > 4096) return false;
    l.owned.reserve(6 * n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* c = items[i];
        if (PyTuple_CheckExact(c)) {
            if (PyTuple_GET_SIZE(c) != 2 || !add_layer_tensor(l, 0, PyTuple_GET_ITEM(c, 0), dev) || !add_layer_tensor(l, 0, PyTuple_GET_ITEM(c, 1), dev))
                return false;
            continue;
        }
        const struct { PyObject* name; int group; } want[6] = {{s_kq, 0}, {s_vq, 0}, {s_ks, 1}, {s_vs, 1}, {s_kz, -1}, {s_vz, -1}};
        for (const auto& w : want) {
            PyObject* o = PyObject_GetAttr(c, w.name);
            if (o == nullptr) {
                PyErr_Clear();
                return false;
            }
            l.owned.push_back(o);
            if (w.group < 0 ? o != Py_None : !add_layer_tensor(l, w.group, o, dev)) return false;
        }
    }
    if (l.like[1] != nullptr && l.base[1].size() != l.base[0].size()) return false;
    for (int g = 0; g < 2; ++g) {
        const Tensor* t = l.like[g];
        if (t == nullptr) continue;
        if (t->size(0) != num_pages || t->size(1) != page_size) return false;
        l.slot[g] = t->size(2) * t->size(3) * (int64_t)t->element_size();
    }
    return l.like[0] != nullptr;
}
int32_t* w32(const Tensor* t) { return static_cast<int32_t*>(t->mutable_data_ptr()); }
bool index_vector(const Tensor* t, int dev) { return t != nullptr && on(*t, dev) && t->dim() == 1 && t->scalar_type() == at::kInt && t->size(0) <= INT32_MAX; }
// counts, page size, block table and (where asked for) lengths of a page call
struct Pool {
    const Tensor *refs, *table, *lengths;
    int64_t pages, P, B, blocks;
    int dev;
};
bool pool_of(Pool& p, PyObject* refs, PyObject* page_size, PyObject* table, PyObject* lengths) {
    p.refs = as_tensor(refs);
    p.table = as_tensor(table);
    p.lengths = lengths == nullptr ? nullptr : as_tensor(lengths);
    p.dev = current_device_of(p.refs);
    if (p.dev < 0 || !index_vector(p.refs, p.dev) || !as_int(page_size, &p.P) || p.P <= 0 || p.P > INT32_MAX || p.refs->size(0) <= 0) return false;
    if (p.table == nullptr || !on(*p.table, p.dev) || p.table->dim() != 2 || p.table->scalar_type() != at::kInt || p.table->numel() == 0) return false;
    p.pages = p.refs->size(0);
    p.B = p.table->size(0);
    p.blocks = p.table->size(1);
    if (p.B > INT32_MAX || p.blocks > INT32_MAX) return false;
    return lengths == nullptr || (index_vector(p.lengths, p.dev) && p.lengths->size(0) == p.B);
}
PyObject* done(int rc) {
    if (rc != 0) return none();
    Py_RETURN_TRUE;
}

// reserve_pages(ref_counts, page_size, block_table, lengths, new tokens: int or tensor) -> True or None
PyObject* reserve_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    Pool p;
    if (p_reserve == nullptr || n_args != 5 || !pool_of(p, a[0], a[1], a[2], a[3])) return none();
    int64_t uniform = 0;
    const Tensor* per_row = as_tensor(a[4]);
    if (per_row != nullptr ? !index_vector(per_row, p.dev) || per_row->size(0) != p.B : !as_int(a[4], &uniform) || uniform < 0 || uniform > INT32_MAX)
        return none();
    const size_t bytes = p_reserve_ws((int)p.B, p.pages);
    Tensor ws = empty({(int64_t)bytes}, at::kByte, p.dev);
    return done(p_reserve(w32(p.refs), p.pages, w32(p.table), i32(p.lengths), i32(per_row), (int)uniform, (int)p.B, (int)p.blocks, (int)p.P,
                          ws.mutable_data_ptr(), bytes, stream_of(p.dev)));
}

// release_sequences(ref_counts, page_size, block_table, lengths, rows) -> True or None
PyObject* release_sequences(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    Pool p;
    if (p_release == nullptr || n_args != 5 || !pool_of(p, a[0], a[1], a[2], a[3])) return none();
    const Tensor* rows = as_tensor(a[4]);
    if (!index_vector(rows, p.dev) || rows->size(0) == 0) return none();
    return done(p_release(w32(p.refs), p.pages, w32(p.table), w32(p.lengths), i32(rows), (int)rows->size(0), (int)p.B, (int)p.blocks, stream_of(p.dev)));
}

// fork_sequences(caches, ref_counts, page_size, block_table, lengths, parents, children) -> True or None
PyObject* fork_sequences(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    Pool p;
    if (p_fork == nullptr || n_args != 7 || !pool_of(p, a[1], a[2], a[3], a[4])) return none();
    const Tensor *parents = as_tensor(a[5]), *children = as_tensor(a[6]);
    Layers l;
    if (!index_vector(parents, p.dev) || !index_vector(children, p.dev) || parents->size(0) == 0 || parents->size(0) != children->size(0) ||
        !layers_of(l, a[0], p.pages, p.P, p.dev))
        return none();
    const int n = (int)parents->size(0);
    const size_t bytes = p_fork_ws(n, (int)p.B);
    Tensor ws = empty({(int64_t)bytes}, at::kByte, p.dev);
    return done(p_fork(l.base[0].data(), (int)l.base[0].size(), l.slot[0], l.base[1].data(), (int)l.base[1].size(), l.slot[1], w32(p.refs), p.pages,
                       w32(p.table), w32(p.lengths), i32(parents), i32(children), n, (int)p.B, (int)p.blocks, (int)p.P, ws.mutable_data_ptr(), bytes,
                       stream_of(p.dev)));
}

// compact_pages(caches, ref_counts, page_size, block_table) -> remap or None
PyObject* compact_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    Pool p;
    Layers l;
    if (p_compact == nullptr || n_args != 4 || !pool_of(p, a[1], a[2], a[3], nullptr) || !layers_of(l, a[0], p.pages, p.P, p.dev)) return none();
    const size_t bytes = p_compact_ws(p.pages);
    Tensor ws = empty({(int64_t)bytes}, at::kByte, p.dev), remap = empty({p.pages}, at::kInt, p.dev);
    const int rc = p_compact(l.base[0].data(), (int)l.base[0].size(), l.slot[0], l.base[1].data(), (int)l.base[1].size(), l.slot[1], w32(p.refs), p.pages,
                             w32(p.table), (int)p.B, (int)p.blocks, (int)p.P, w32(&remap), ws.mutable_data_ptr(), bytes, stream_of(p.dev));
    return rc == 0 ? THPVariable_Wrap(std::move(remap)) : none();
}

// copy_pages(caches, src, dst) -> True or None
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (p_copy_pages == nullptr || n_args != 3) return none();
    const Tensor *src = as_tensor(a[1]), *dst = as_tensor(a[2]);
    const int dev = current_device_of(src);
    if (dev < 0 || !index_vector(src, dev) || !index_vector(dst, dev) || src->size(0) == 0 || src->size(0) != dst->size(0) ||
        (!PyList_Check(a[0]) && !PyTuple_Check(a[0])) || PySequence_Fast_GET_SIZE(a[0]) == 0)
        return none();
    // the pool's size is the first tensor's
    PyObject* first = PySequence_Fast_ITEMS(a[0])[0];
    Attr quantised(PyTuple_CheckExact(first) ? Py_None : first, s_kq);
    const Tensor* t = PyTuple_CheckExact(first) && PyTuple_GET_SIZE(first) == 2 ? as_tensor(PyTuple_GET_ITEM(first, 0))
                      : quantised.o != nullptr                                 ? as_tensor(quantised.o)
                                                                                : nullptr;
    Layers l;
    if (t == nullptr || t->dim() != 4 || t->size(0) > INT32_MAX || t->size(1) > INT32_MAX || !layers_of(l, a[0], t->size(0), t->size(1), dev))
        return none();
    const int n = (int)src->size(0);
    const size_t bytes = p_copy_ws(n, t->size(0));
    Tensor ws = empty({(int64_t)bytes}, at::kByte, dev);
    return done(p_copy_pages(l.base[0].data(), (int)l.base[0].size(), l.slot[0], l.base[1].data(), (int)l.base[1].size(), l.slot[1], i32(src), i32(dst), n,
                             t->size(0), (int)t->size(1), ws.mutable_data_ptr(), bytes, stream_of(dev)));
}

// bind({symbol: address}): the C ABI functions to call
PyObject* bind(PyObject*, PyObject* table) {
    const struct { const char* name; void** slot; } want[] = {
        {"b200q_qmatvec", (void**)&p_qmatvec}, {"b200q_gate_up_swiglu", (void**)&p_gate_up},
        {"b200q_scratch_next", (void**)&p_scratch_next}, {"b200q_scratch_bytes", (void**)&p_scratch_bytes},
        {"b200q_paged_gqa_workspace_bytes", (void**)&p_attn_ws}, {"b200q_attention_stage_launches", (void**)&p_attn_launches},
        {"b200q_paged_gqa_decode", (void**)&p_attn}, {"b200q_paged_gqa_decode_window", (void**)&p_attn_window},
        {"b200q_paged_fp16_gqa_workspace_bytes", (void**)&p_plain_ws}, {"b200q_paged_fp16_gqa_decode", (void**)&p_plain_attn},
        {"b200q_paged_fp16_gqa_decode_checked", (void**)&p_plain_checked},
        {"b200q_lora_qmatvec_workspace_bytes", (void**)&p_lora_ws}, {"b200q_lora_qmatvec", (void**)&p_lora},
        {"b200q_reserve_pages_workspace_bytes", (void**)&p_reserve_ws}, {"b200q_copy_pages_workspace_bytes", (void**)&p_copy_ws},
        {"b200q_fork_sequences_workspace_bytes", (void**)&p_fork_ws}, {"b200q_compact_pages_workspace_bytes", (void**)&p_compact_ws},
        {"b200q_reserve_pages", (void**)&p_reserve}, {"b200q_release_sequences", (void**)&p_release},
        {"b200q_copy_pages", (void**)&p_copy_pages}, {"b200q_fork_sequences", (void**)&p_fork}, {"b200q_compact_pages", (void**)&p_compact},
        {"b200q_head_rope", (void**)&p_head_rope}, {"b200q_norm_rope_kv_append", (void**)&p_append},
        {"b200q_quantize_kv_pair", (void**)&p_quant_pair}, {"b200q_dequantize_kv_pair", (void**)&p_dequant_pair},
    };
    for (const auto& w : want) {
        PyObject* v = PyDict_GetItemString(table, w.name);
        void* p = v == nullptr ? nullptr : PyLong_AsVoidPtr(v);
        if (p == nullptr) {
            PyErr_Format(PyExc_KeyError, "%s", w.name);
            return nullptr;
        }
        *w.slot = p;
    }
    return none();
}

// C++ exceptions (out of memory, a CUDA error) become Python ones, as torch's own functions raise them
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return F(self, args, n);
    END_HANDLE_TH_ERRORS
}
#define FAST(fn) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<fn>))

PyMethodDef methods[] = {
    {"bind", bind, METH_O, "bind({symbol: address})"},
    {"matvec", FAST(matvec), METH_FASTCALL, nullptr},
    {"mlp_block", FAST(mlp_block), METH_FASTCALL, nullptr},
    {"quantize_kv", FAST(quantize_kv), METH_FASTCALL, nullptr},
    {"dequantize_kv", FAST(dequantize_kv), METH_FASTCALL, nullptr},
    {"head_rope", FAST(head_rope), METH_FASTCALL, nullptr},
    {"norm_rope_append", FAST(norm_rope_append), METH_FASTCALL, nullptr},
    {"norm_rope_append_pages", FAST(norm_rope_append_pages), METH_FASTCALL, nullptr},
    {"lora_linear", FAST(lora_linear), METH_FASTCALL, nullptr},
    {"reserve_pages", FAST(reserve_pages), METH_FASTCALL, nullptr},
    {"release_sequences", FAST(release_sequences), METH_FASTCALL, nullptr},
    {"fork_sequences", FAST(fork_sequences), METH_FASTCALL, nullptr},
    {"compact_pages", FAST(compact_pages), METH_FASTCALL, nullptr},
    {"copy_pages", FAST(copy_pages), METH_FASTCALL, nullptr},
    {"plain_attention", FAST(plain_attention), METH_FASTCALL, nullptr},
    {"paged_attention", FAST(paged_attention), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_b200q_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__b200q_host() {
    const struct { const char* name; PyObject** slot; } names[] = {
        {"bits", &s_bits}, {"group_size", &s_group_size}, {"original_page_shape", &s_shape},
        {"k_pages_q", &s_kq}, {"v_pages_q", &s_vq}, {"k_scales", &s_ks}, {"v_scales", &s_vs}, {"block_table", &s_bt}, {"lengths", &s_len},
        {"a", &s_a}, {"b", &s_b}, {"scaling", &s_scaling}, {"ranks", &s_ranks}, {"k_zeros", &s_kz}, {"v_zeros", &s_vz},
    };
    for (const auto& n : names)
        if ((*n.slot = PyUnicode_InternFromString(n.name)) == nullptr) return nullptr;
    return PyModule_Create(&module_def);
}

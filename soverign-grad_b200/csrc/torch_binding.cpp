// Native side of the Python package's hot calls: takes torch tensors and the package's own objects, allocates the
// outputs, and calls the C ABI of include/sgq.h.
//
// Why it exists: a decode-sized forward takes 5-10 us on the GPU, and the Python form of the call (attribute walks,
// contiguous / float checks, a ctypes call with sixteen converted arguments, the stream lookup) took 15-20 us on the
// host, so an eager token loop was bound by the host at every small size.  Arguments are parsed by hand
// (METH_FASTCALL), the GIL is released around the library call as ctypes does.
//
// No computation happens here, and nothing falls back: unusual inputs are converted by the same torch operations the
// Python code used (contiguous, float).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <utility>
#include <vector>

#include "../../include/sgq.h"
#include "../../include/sgq_decoder.h"

namespace {

PyObject* g_error_class = nullptr;      // SgqError(status, what, detail)
PyObject* g_tensor_class = nullptr;     // QuantizedTensor(qdata, scales, scheme, original_shape, group_size, bits)
PyObject* g_workspace_class = nullptr;  // Workspace: .buf, .get(nbytes)

PyObject *s_qdata, *s_scales, *s_scheme, *s_shape, *s_group, *s_bits, *s_buf, *s_get;
PyObject *s_k_codes, *s_k_scales, *s_v_codes, *s_v_scales;

// A reference that is given back at the end of the scope.
struct Ref {
    PyObject* p;
    explicit Ref(PyObject* o = nullptr) : p(o) {}
    ~Ref() { Py_XDECREF(p); }
    Ref(const Ref&) = delete;
    Ref& operator=(const Ref&) = delete;
    PyObject* release() { PyObject* o = p; p = nullptr; return o; }
    explicit operator bool() const { return p != nullptr; }
};

struct PythonError {};      // a Python exception is set

[[noreturn]] void raise(PyObject* type, const char* msg) {
    PyErr_SetString(type, msg);
    throw PythonError();
}

void check(int status, const char* what) {
    if (status == SGQ_OK) return;
    Ref args(Py_BuildValue("(iss)", status, (std::string(what) + " failed: " + sgq_status_string(status)).c_str(), sgq_last_error()));
    Ref exc(args ? PyObject_CallObject(g_error_class, args.p) : nullptr);
    if (exc) PyErr_SetObject(g_error_class, exc.p);
    throw PythonError();
}

int64_t as_int(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError();
    return v;
}

const at::Tensor& as_tensor(PyObject* o) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "a torch tensor is needed here");
    return THPVariable_Unpack(o);
}

// fp32, contiguous, on the GPU; the tensor itself where it already is
at::Tensor f32_cuda(PyObject* o) {
    const at::Tensor& t = as_tensor(o);
    if (!t.is_cuda()) raise(PyExc_ValueError, "this library computes on CUDA tensors only");
    if (t.scalar_type() == at::kFloat && t.is_contiguous()) return t;
    return t.contiguous().to(at::kFloat);
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// What a QuantizedTensor holds.  Its scheme is read for INT8 only and its group for INT4 only: what a checkpoint loader left
// in the other one does not matter.
struct Quantized {
    at::Tensor qdata, scales;
    int64_t scheme = SGQ_PER_TENSOR, group = 0, bits, rows = 0, cols = 0, numel = 1;
    size_t dims;
    Ref shape;
    explicit Quantized(PyObject* q) {
        Ref d(PyObject_GetAttr(q, s_qdata)), s(PyObject_GetAttr(q, s_scales)), b(PyObject_GetAttr(q, s_bits));
        shape.p = PyObject_GetAttr(q, s_shape);
        if (!d || !s || !b || !shape) throw PythonError();
        qdata = as_tensor(d.p);
        scales = as_tensor(s.p);
        bits = as_int(b.p);
        Ref v(PyObject_GetAttr(q, bits == 4 ? s_group : s_scheme));
        if (!v) throw PythonError();
        (bits == 4 ? group : scheme) = as_int(v.p);
        Ref seq(PySequence_Fast(shape.p, "original_shape is a sequence"));
        if (!seq) throw PythonError();
        dims = static_cast<size_t>(PySequence_Fast_GET_SIZE(seq.p));
        for (size_t i = 0; i < dims; ++i) {
            const int64_t v = as_int(PySequence_Fast_GET_ITEM(seq.p, i));
            if (i == 0) rows = v;
            if (i == 1) cols = v;
            numel *= v;
        }
    }
    // a single scale counts as per tensor whatever the scheme says (src/quantization.cpp:91)
    int scheme_now() const { return scheme == SGQ_PER_TENSOR || scales.numel() == 1 ? SGQ_PER_TENSOR : SGQ_PER_ROW; }
};

// The scratch of a call: what the caller's workspace gives for `need` bytes (None: nothing), or a buffer of this call.  The
// package's own Workspace is read directly while its buffer is large enough; any other object, a class derived from it
// included, is asked through its get().
struct Scratch {
    at::Tensor buf;
    void* ptr = nullptr;
    size_t bytes = 0;
    Scratch(PyObject* workspace, size_t need, const at::Tensor& like) {
        if (need == 0) return;
        if (workspace == Py_None) {
            buf = empty({static_cast<int64_t>(need)}, at::kByte, like);
        } else {
            Ref b;
            if (reinterpret_cast<PyObject*>(Py_TYPE(workspace)) == g_workspace_class) {
                b.p = PyObject_GetAttr(workspace, s_buf);
                if (!b) throw PythonError();
            }
            if (b && b.p != Py_None && static_cast<size_t>(as_tensor(b.p).numel()) >= need) {
                buf = as_tensor(b.p);
            } else {
                Ref n(PyLong_FromSize_t(need));
                Ref given(n ? PyObject_CallMethodOneArg(workspace, s_get, n.p) : nullptr);
                if (!given) throw PythonError();
                if (given.p == Py_None) return;
                buf = as_tensor(given.p);
            }
        }
        ptr = buf.data_ptr();
        bytes = static_cast<size_t>(buf.numel());
    }
};

// Calls into the library without the GIL, as ctypes does.
template <typename F>
int without_gil(F&& f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        return F(args, n);
    } catch (const PythonError&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

float* fptr(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

// bias as N fp32 values, or an empty tensor
at::Tensor bias_of(PyObject* o, int64_t N) {
    if (o == Py_None) return at::Tensor();
    at::Tensor b = f32_cuda(o);
    if (b.numel() != N) raise(PyExc_RuntimeError, "Incompatible shapes for broadcasting!");      // src/ops.cpp:60
    return b;
}

// quantized_matmul(x, q, bias, layout, path, out, workspace, ldy, workspace_limit)
PyObject* quantized_matmul(PyObject* const* a, Py_ssize_t n) {
    if (n != 9) raise(PyExc_TypeError, "quantized_matmul takes nine arguments");
    const at::Tensor x = f32_cuda(a[0]);
    if (x.dim() != 2) raise(PyExc_RuntimeError, "matmul currently requires 2D tensors!");
    const Quantized q(a[1]);
    const int layout = static_cast<int>(as_int(a[3])), path = static_cast<int>(as_int(a[4]));
    if (q.dims != 2) raise(PyExc_RuntimeError, "matmul currently requires 2D tensors!");                     // src/ops.cpp:380-382
    const int64_t K = layout == SGQ_LAYOUT_KN ? q.rows : q.cols, N = layout == SGQ_LAYOUT_KN ? q.cols : q.rows, M = x.size(0);
    if (x.size(1) != K) raise(PyExc_RuntimeError, "Matrix inner dimensions must match for matmul!");         // src/ops.cpp:387-389
    const at::Tensor bias = bias_of(a[2], N);
    at::Tensor out;
    int64_t ldy = N;
    if (a[5] == Py_None) {
        out = empty({M, N}, at::kFloat, x);
    } else {
        out = as_tensor(a[5]);
        ldy = a[7] == Py_None ? out.stride(0) : as_int(a[7]);
    }
    size_t need = sgq_linear_workspace_bytes(static_cast<int>(q.bits), M, K, N, layout, path);
    const bool limited = a[8] != Py_None;
    const size_t limit = limited ? static_cast<size_t>(as_int(a[8])) : 0;
    if (limited && need > limit) need = limit;
    Scratch ws(a[6], need, x);
    if (limited && ws.bytes > limit) ws.bytes = limit;
    void* s = stream();
    const float* b = bias.defined() ? fptr(bias) : nullptr;
    check(without_gil([&] {
              return q.bits == 4 ? sgq_linear_int4(fptr(x), M, K, N, static_cast<const uint8_t*>(q.qdata.data_ptr()), fptr(q.scales), layout,
                                                   q.group, b, fptr(out), ldy, path, ws.ptr, ws.bytes, s)
                                 : sgq_linear_int8(fptr(x), M, K, N, static_cast<const int8_t*>(q.qdata.data_ptr()), fptr(q.scales), layout,
                                                   q.scheme_now(), b, fptr(out), ldy, path, ws.ptr, ws.bytes, s);
          }),
          "sgq_linear");
    if (a[5] != Py_None) {
        Py_INCREF(a[5]);
        return a[5];
    }
    return THPVariable_Wrap(std::move(out));
}

// quantized_matmul_backward_x(dy, q, layout, path, workspace)
PyObject* backward_x(PyObject* const* a, Py_ssize_t n) {
    if (n != 5) raise(PyExc_TypeError, "quantized_matmul_backward_x takes five arguments");
    const at::Tensor dy = f32_cuda(a[0]);
    const Quantized q(a[1]);
    const int layout = static_cast<int>(as_int(a[2])), path = static_cast<int>(as_int(a[3]));
    if (q.dims != 2) raise(PyExc_RuntimeError, "matmul currently requires 2D tensors!");
    const int64_t K = layout == SGQ_LAYOUT_KN ? q.rows : q.cols, N = layout == SGQ_LAYOUT_KN ? q.cols : q.rows;
    if (dy.dim() != 2 || dy.size(1) != N) raise(PyExc_RuntimeError, "Matrix inner dimensions must match for matmul!");
    const int64_t M = dy.size(0);
    at::Tensor dx = empty({M, K}, at::kFloat, dy);
    Scratch ws(a[4], sgq_linear_backward_x_workspace_bytes(static_cast<int>(q.bits), M, K, N, layout, path), dy);
    void* s = stream();
    check(without_gil([&] {
              return q.bits == 4 ? sgq_linear_int4_backward_x(fptr(dy), M, K, N, static_cast<const uint8_t*>(q.qdata.data_ptr()),
                                                              fptr(q.scales), layout, q.group, fptr(dx), K, path, ws.ptr, ws.bytes, s)
                                 : sgq_linear_int8_backward_x(fptr(dy), M, K, N, static_cast<const int8_t*>(q.qdata.data_ptr()),
                                                              fptr(q.scales), layout, q.scheme_now(), fptr(dx), K, path, ws.ptr, ws.bytes, s);
          }),
          "sgq_linear_backward_x");
    return THPVariable_Wrap(std::move(dx));
}

// linear_w8a8(x, q, bias, want_parts).  Every shape is checked here, before the device: the library below sees pointers and
// M, K, N only, and a narrower x, packed INT4 codes or a short bias would be read past their end.
PyObject* linear_w8a8(PyObject* const* a, Py_ssize_t n) {
    if (n != 4) raise(PyExc_TypeError, "linear_w8a8 takes four arguments");
    const at::Tensor& given = as_tensor(a[0]);
    const Quantized q(a[1]);
    if (given.dim() != 2 || q.dims != 2) raise(PyExc_RuntimeError, "matmul currently requires 2D tensors!");
    if (q.bits != 8) raise(PyExc_RuntimeError, "linear_w8a8 needs an INT8 weight stored [N,K]");
    const int64_t N = q.rows, K = q.cols, M = given.size(0);
    if (given.size(1) != K) raise(PyExc_RuntimeError, "Matrix inner dimensions must match for matmul!");
    if (a[2] != Py_None && as_tensor(a[2]).numel() != N) raise(PyExc_RuntimeError, "Incompatible shapes for broadcasting!");
    const int parts_asked = PyObject_IsTrue(a[3]);
    if (parts_asked < 0) throw PythonError();
    const at::Tensor x = f32_cuda(a[0]), bias = bias_of(a[2], N);
    at::Tensor y = empty({M, N}, at::kFloat, x), xq, sx, acc;
    const bool parts = parts_asked == 1;
    if (parts) {
        xq = empty({M, K}, at::kChar, x);
        sx = empty({M}, at::kFloat, x);
        acc = empty({M, N}, at::kInt, x);
    }
    const size_t need = sgq_linear_w8a8_workspace_bytes(M, K, N);
    at::Tensor ws = empty({static_cast<int64_t>(need > 256 ? need : 256)}, at::kByte, x);
    void* s = stream();
    check(without_gil([&] {
              return sgq_linear_w8a8(fptr(x), M, K, N, static_cast<const int8_t*>(q.qdata.data_ptr()), fptr(q.scales), q.scheme_now(),
                                     bias.defined() ? fptr(bias) : nullptr, fptr(y), N,
                                     parts ? static_cast<int8_t*>(xq.data_ptr()) : nullptr, parts ? fptr(sx) : nullptr,
                                     parts ? static_cast<int32_t*>(acc.data_ptr()) : nullptr, ws.data_ptr(),
                                     static_cast<size_t>(ws.numel()), s);
          }),
          "sgq_linear_w8a8");
    if (!parts) return THPVariable_Wrap(std::move(y));
    return Py_BuildValue("(NNNN)", THPVariable_Wrap(y), THPVariable_Wrap(xq), THPVariable_Wrap(sx), THPVariable_Wrap(acc));
}

// A QuantizedTensor object; `shape` as the package keeps it (a plain tuple)
PyObject* wrap_quantized(const at::Tensor& x, at::Tensor& qdata, at::Tensor& scales, int64_t scheme, int64_t group, int64_t bits) {
    Ref shape(PyTuple_New(x.dim()));
    if (!shape) throw PythonError();
    for (int64_t i = 0; i < x.dim(); ++i) PyTuple_SET_ITEM(shape.p, i, PyLong_FromLongLong(x.size(i)));
    Ref q(THPVariable_Wrap(qdata)), s(THPVariable_Wrap(scales)), sch(PyLong_FromLongLong(scheme)), g(PyLong_FromLongLong(group)),
        b(PyLong_FromLongLong(bits));
    PyObject* args[6] = {q.p, s.p, sch.p, shape.p, g.p, b.p};
    PyObject* r = PyObject_Vectorcall(g_tensor_class, args, 6, nullptr);
    if (!r) throw PythonError();
    return r;
}

// quantize_int8(x, scheme)
PyObject* quantize_int8(PyObject* const* a, Py_ssize_t n) {
    if (n != 2) raise(PyExc_TypeError, "quantize_int8 takes two arguments");
    const at::Tensor x = f32_cuda(a[0]);
    const int64_t scheme = as_int(a[1]), numel = x.numel();
    const bool tensor = scheme == SGQ_PER_TENSOR || x.dim() < 2;        // src/quantization.cpp:22
    const int64_t rows = tensor ? 1 : x.size(0), cols = tensor ? numel : (rows ? numel / rows : 0);
    at::Tensor codes = empty(x.sizes(), at::kChar, x), scales = empty({rows}, at::kFloat, x);
    void* s = stream();
    check(without_gil([&] {
              return sgq_quantize_int8(fptr(x), rows, cols, tensor ? SGQ_PER_TENSOR : SGQ_PER_ROW, static_cast<int8_t*>(codes.data_ptr()),
                                       fptr(scales), s);
          }),
          "sgq_quantize_int8");
    return wrap_quantized(x, codes, scales, scheme, numel, 8);
}

// quantize_int4(x, group_size)
PyObject* quantize_int4(PyObject* const* a, Py_ssize_t n) {
    if (n != 2) raise(PyExc_TypeError, "quantize_int4 takes two arguments");
    const at::Tensor x = f32_cuda(a[0]);
    const int64_t asked = as_int(a[1]), group = asked <= 0 ? 32 : asked, numel = x.numel();
    at::Tensor packed = empty({(numel + 1) / 2}, at::kByte, x), scales = empty({(numel + group - 1) / group}, at::kFloat, x);
    void* s = stream();
    check(without_gil([&] {
              return sgq_quantize_int4(fptr(x), numel, group, static_cast<uint8_t*>(packed.data_ptr()), fptr(scales), s);
          }),
          "sgq_quantize_int4");
    return wrap_quantized(x, packed, scales, SGQ_PER_TENSOR, group, 4);
}

// dequantize(q): either bit width
PyObject* dequantize(PyObject* const* a, Py_ssize_t n) {
    if (n != 1) raise(PyExc_TypeError, "dequantize takes one argument");
    const Quantized q(a[0]);
    std::vector<int64_t> sizes;
    Ref seq(PySequence_Fast(q.shape.p, "original_shape is a sequence"));
    if (!seq) throw PythonError();
    for (size_t i = 0; i < q.dims; ++i) sizes.push_back(as_int(PySequence_Fast_GET_ITEM(seq.p, i)));
    at::Tensor out = empty(sizes, at::kFloat, q.qdata);
    void* s = stream();
    if (q.bits == 4) {
        check(without_gil([&] {
                  return sgq_dequantize_int4(static_cast<const uint8_t*>(q.qdata.data_ptr()), fptr(q.scales), q.numel, q.group, fptr(out), s);
              }),
              "sgq_dequantize_int4");
    } else {
        const int scheme = q.scheme_now();
        const int64_t rows = scheme == SGQ_PER_TENSOR ? 1 : q.rows, cols = rows ? q.numel / rows : 0;
        check(without_gil([&] {
                  return sgq_dequantize_int8(static_cast<const int8_t*>(q.qdata.data_ptr()), fptr(q.scales), rows, cols, scheme, fptr(out), s);
              }),
              "sgq_dequantize_int8");
    }
    return THPVariable_Wrap(std::move(out));
}

// ---- the INT8 key/value cache.  Every shape is checked before the device: the library sees pointers and sizes only. ----

// A KVCacheInt8: k_codes / v_codes int8 [batch, kv heads, max_seq, head_dim], k_scales / v_scales fp32 [batch, kv heads, max_seq].
struct Cache8 {
    at::Tensor t[4];
    sgqd_cache_int8 c = {};
    explicit Cache8(PyObject* o) {
        PyObject* names[4] = {s_k_codes, s_k_scales, s_v_codes, s_v_scales};
        for (int i = 0; i < 4; ++i) {
            Ref a(PyObject_GetAttr(o, names[i]));
            if (!a) throw PythonError();
            t[i] = as_tensor(a.p);
        }
        if (t[0].dim() != 4) raise(PyExc_RuntimeError, "cache codes must be [batch, kv heads, max_seq, head_dim]");
        const auto rows = t[0].sizes().slice(0, 3);
        for (int i = 0; i < 4; i += 2) {
            if (t[i].scalar_type() != at::kChar || t[i].sizes() != t[0].sizes()) raise(PyExc_RuntimeError, "cache codes must be int8 of one shape");
            if (t[i + 1].scalar_type() != at::kFloat || t[i + 1].sizes() != rows) raise(PyExc_RuntimeError, "cache scales must be fp32 [batch, kv heads, max_seq]");
            if (!t[i].is_contiguous() || !t[i + 1].is_contiguous()) raise(PyExc_RuntimeError, "cache tensors must be contiguous");
        }
        c.batch = t[0].size(0); c.n_kv_heads = t[0].size(1); c.max_seq = t[0].size(2); c.head_dim = t[0].size(3);
        if (c.n_kv_heads <= 0 || c.max_seq <= 0 || c.head_dim <= 0) raise(PyExc_RuntimeError, "the cache has no heads, positions or values");
        c.k_codes = static_cast<int8_t*>(t[0].data_ptr()); c.k_scales = static_cast<float*>(t[1].data_ptr());
        c.v_codes = static_cast<int8_t*>(t[2].data_ptr()); c.v_scales = static_cast<float*>(t[3].data_ptr());
    }
    void on(const c10::Device& d) const {
        for (const at::Tensor& x : t)
            if (x.device() != d) raise(PyExc_ValueError, "all tensors must be on one GPU");
    }
};

// Rows of `width` values spaced evenly: [batch, tokens, width], or [batch, width] where tokens may be 1.  stride < 0: they are not.
struct Rows {
    at::Tensor t;
    int64_t batch, tokens, width, stride = -1;
    explicit Rows(const at::Tensor& x, bool two) : t(x) {
        if (t.dim() == 2 && two) t = t.unsqueeze(1);
        if (t.dim() != 3) raise(PyExc_RuntimeError, two ? "rows must be [batch, width] or [batch, 1, width]" : "rows must be [batch, tokens, width]");
        batch = t.size(0); tokens = t.size(1); width = t.size(2);
        if (t.scalar_type() != at::kFloat || (t.stride(2) != 1 && width > 1)) return;
        const int64_t step = tokens > 1 ? t.stride(1) : (batch > 1 ? t.stride(0) : width);
        if (batch > 1 && tokens > 1 && t.stride(0) != tokens * step) return;
        if (step < width || (step & 3) || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)) return;
        stride = step;
    }
};

// Optional DEVICE int32 vector: nullptr for None
struct Ints {
    at::Tensor t;
    const int32_t* p = nullptr;
    int64_t n = 0;
    Ints(PyObject* o, const char* what) {
        if (o == Py_None) return;
        t = as_tensor(o);
        if (t.scalar_type() != at::kInt || t.dim() > 1 || (t.dim() == 1 && t.size(0) > 1 && t.stride(0) != 1)) raise(PyExc_RuntimeError, what);
        n = t.numel();
        p = static_cast<const int32_t*>(t.data_ptr());
    }
};

// What the three calls that rotate have in common: qkv, tables, positions; all on one GPU.
struct Rotary {
    const Cache8& cache;
    Rows qkv;
    at::Tensor cos, sin;
    Ints pos;
    int64_t heads;
    Rotary(PyObject* q, const Cache8& c, PyObject* cos_o, PyObject* sin_o, PyObject* pos_o, PyObject* heads_o, bool two)
        : cache(c), qkv(as_tensor(q), two), cos(as_tensor(cos_o)), sin(as_tensor(sin_o)), pos(pos_o, "pos must be an int32 vector"),
          heads(as_int(heads_o)) {
        const int64_t hd = c.c.head_dim, kv = c.c.n_kv_heads;
        if (heads <= 0 || heads % kv) raise(PyExc_RuntimeError, "n_heads must be a multiple of the cache's heads");
        if (qkv.width != (heads + 2 * kv) * hd) raise(PyExc_RuntimeError, "qkv rows must hold n_heads + 2 * kv heads of head_dim values");
        if (qkv.batch != c.c.batch) raise(PyExc_RuntimeError, "qkv and the cache differ in batch");
        if (two && qkv.tokens != 1) raise(PyExc_RuntimeError, "one new token per sequence");
        if (cos.dim() != 2 || cos.sizes() != sin.sizes() || cos.size(1) != hd / 2 || cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat ||
            !cos.is_contiguous() || !sin.is_contiguous())
            raise(PyExc_RuntimeError, "cos and sin must be fp32 [rows, head_dim / 2]");
        if (!pos.p && pos.n == 0 && c.c.batch > 0) raise(PyExc_RuntimeError, "pos must be an int32 vector");
        if (pos.n != 1 && pos.n != c.c.batch) raise(PyExc_RuntimeError, "pos must have one element, or one per sequence");
        if (!qkv.t.is_cuda()) raise(PyExc_ValueError, "this library computes on CUDA tensors only");
        const c10::Device d = qkv.t.device();
        c.on(d);
        if (cos.device() != d || sin.device() != d || pos.t.device() != d) raise(PyExc_ValueError, "all tensors must be on one GPU");
    }
    int64_t pos_stride() const { return pos.n == 1 ? 0 : 1; }
    // rows for reading: evenly spaced fp32, copied where they are not
    void readable() {
        if (qkv.stride < 0) qkv = Rows(qkv.t.to(at::kFloat).clone(at::MemoryFormat::Contiguous), false);
    }
};

// rope_kv_store_int8(qkv, cache, cos, sin, pos, n_heads, q_out, rope_offset, n_new)
PyObject* rope_kv_store_int8(PyObject* const* a, Py_ssize_t n) {
    if (n != 9) raise(PyExc_TypeError, "rope_kv_store_int8 takes nine arguments");
    const Cache8 cache(a[1]);
    const bool in_place = a[6] == Py_None;
    const at::Tensor q_out = in_place ? at::Tensor() : as_tensor(a[6]);
    const Ints offset(a[7], "rope_offset must be one int32"), n_new(a[8], "n_new must be an int32 vector");
    if (a[7] != Py_None && offset.n != 1) raise(PyExc_RuntimeError, "rope_offset must be one int32");
    if (a[8] != Py_None && n_new.n != cache.c.batch) raise(PyExc_RuntimeError, "n_new must have one element per sequence");
    Rotary r(a[0], cache, a[2], a[3], a[4], a[5], false);
    const c10::Device d = r.qkv.t.device();
    if ((offset.p && offset.t.device() != d) || (n_new.p && n_new.t.device() != d) || (!in_place && q_out.device() != d))
        raise(PyExc_ValueError, "all tensors must be on one GPU");
    const int64_t dim = r.heads * cache.c.head_dim;
    if (in_place && r.qkv.stride < 0) raise(PyExc_RuntimeError, "in place, qkv must be evenly spaced fp32 rows aligned to 16 bytes");
    const c10::cuda::CUDAGuard guard(d);
    r.readable();
    float* q_ptr = fptr(r.qkv.t);
    int64_t q_stride = r.qkv.stride;
    if (!in_place) {
        const Rows q(q_out, false);
        if (q.batch != r.qkv.batch || q.tokens != r.qkv.tokens || q.width != dim || q.stride < 0)
            raise(PyExc_RuntimeError, "q_out must be evenly spaced fp32 rows [batch, tokens, n_heads * head_dim] aligned to 16 bytes");
        q_ptr = fptr(q.t);
        q_stride = q.stride;
    }
    void* s = stream();
    check(without_gil([&] {
              return sgqd_rope_kv_store_int8(fptr(r.qkv.t), r.qkv.stride, r.qkv.tokens, r.heads, fptr(r.cos), fptr(r.sin), r.cos.size(0), r.pos.p,
                                             r.pos_stride(), n_new.p, offset.p, q_ptr, q_stride, &cache.c, s);
          }),
          "sgqd_rope_kv_store_int8");
    PyObject* given = in_place ? a[0] : a[6];
    Py_INCREF(given);
    return given;
}

// kv_load_int8(cache, rows, batch, k_out, v_out, row0)
PyObject* kv_load_int8(PyObject* const* a, Py_ssize_t n) {
    if (n != 6) raise(PyExc_TypeError, "kv_load_int8 takes six arguments");
    const Cache8 cache(a[0]);
    const int64_t rows = as_int(a[1]), batch = a[2] == Py_None ? cache.c.batch : as_int(a[2]), row0 = as_int(a[5]);
    if (rows < 0 || rows > cache.c.max_seq) raise(PyExc_RuntimeError, "rows must lie inside the cache");
    if (batch < 0 || (batch != cache.c.batch && cache.c.batch != 1)) raise(PyExc_RuntimeError, "batch must be the cache's, or the cache one sequence");
    if ((a[3] == Py_None) != (a[4] == Py_None)) raise(PyExc_RuntimeError, "give both outputs or neither");
    if (row0 < 0 || (a[3] == Py_None && row0 != 0)) raise(PyExc_RuntimeError, "row0 goes with outputs of the caller's");
    at::Tensor out[2];
    int64_t out_rows = rows;
    if (a[3] != Py_None) {
        out[0] = as_tensor(a[3]);
        out[1] = as_tensor(a[4]);
        for (const at::Tensor& o : out) {
            if (o.dim() != 4 || o.scalar_type() != at::kFloat || !o.is_contiguous() || o.sizes() != out[0].sizes() || o.size(0) != batch ||
                o.size(1) != cache.c.n_kv_heads || o.size(3) != cache.c.head_dim || row0 > o.size(2) - rows)
                raise(PyExc_RuntimeError, "outputs must be contiguous fp32 [batch, kv heads, row0 + rows or more, head_dim]");
        }
        out_rows = out[0].size(2);
    }
    const c10::Device d = cache.t[0].device();
    if (!d.is_cuda()) raise(PyExc_ValueError, "this library computes on CUDA tensors only");
    cache.on(d);
    const c10::cuda::CUDAGuard guard(d);
    if (a[3] == Py_None) {
        for (at::Tensor& o : out) o = empty({batch, cache.c.n_kv_heads, rows, cache.c.head_dim}, at::kFloat, cache.t[0]);
    } else if (out[0].device() != d || out[1].device() != d) {
        raise(PyExc_ValueError, "all tensors must be on one GPU");
    }
    void* s = stream();
    check(without_gil([&] { return sgqd_kv_load_int8(&cache.c, rows, batch, fptr(out[0]), fptr(out[1]), out_rows, row0, s); }), "sgqd_kv_load_int8");
    return Py_BuildValue("(NN)", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]));
}

// What the decode calls have in common behind the arguments `first` and `first + 1`: out, prepared
struct DecodeOut {
    at::Tensor out, planes;
    PyObject* given;
    int64_t stride;
    uint8_t* p = nullptr;
    size_t bytes = 0;
    DecodeOut(PyObject* out_o, PyObject* planes_o, const Rotary& r) : given(out_o == Py_None ? nullptr : out_o) {
        const int64_t batch = r.cache.c.batch, dim = r.heads * r.cache.c.head_dim;
        const c10::Device d = r.qkv.t.device();
        if (given) {
            out = as_tensor(out_o);
            if (out.dim() != 2 || out.size(0) != batch || out.size(1) != dim || out.scalar_type() != at::kFloat || out.stride(1) != 1 ||
                (batch > 1 && out.stride(0) < dim))
                raise(PyExc_RuntimeError, "out must be fp32 rows [batch, n_heads * head_dim]");
            if (out.device() != d) raise(PyExc_ValueError, "all tensors must be on one GPU");
        }
        if (planes_o != Py_None) {
            planes = as_tensor(planes_o);
            if (planes.scalar_type() != at::kByte || !planes.is_contiguous()) raise(PyExc_RuntimeError, "prepared must be a uint8 buffer");
            if (planes.device() != d) raise(PyExc_ValueError, "all tensors must be on one GPU");
            p = static_cast<uint8_t*>(planes.data_ptr());
            bytes = static_cast<size_t>(planes.numel());
        }
        if (!given) out = empty({batch, dim}, at::kFloat, r.qkv.t);
        stride = batch > 1 ? out.stride(0) : dim;
    }
    PyObject* result() {
        if (!given) return THPVariable_Wrap(std::move(out));
        Py_INCREF(given);
        return given;
    }
};

// attn_decode_int8(qkv, cache, cos, sin, pos, n_heads, out, prepared, workspace)
PyObject* attn_decode_int8(PyObject* const* a, Py_ssize_t n) {
    if (n != 9) raise(PyExc_TypeError, "attn_decode_int8 takes nine arguments");
    const Cache8 cache(a[1]);
    Rotary r(a[0], cache, a[2], a[3], a[4], a[5], true);
    const c10::cuda::CUDAGuard guard(r.qkv.t.device());
    r.readable();
    DecodeOut o(a[6], a[7], r);
    const Scratch ws(a[8], sgqd_attn_decode_int8_workspace_bytes(cache.c.batch, r.heads, cache.c.n_kv_heads, cache.c.head_dim, cache.c.max_seq), r.qkv.t);
    if (ws.buf.defined() && ws.buf.device() != r.qkv.t.device()) raise(PyExc_ValueError, "all tensors must be on one GPU");
    void* s = stream();
    check(without_gil([&] {
              return sgqd_attn_decode_int8(fptr(r.qkv.t), r.qkv.stride, r.heads, fptr(r.cos), fptr(r.sin), r.cos.size(0), r.pos.p, r.pos_stride(), &cache.c,
                                           fptr(o.out), o.stride, o.p, o.bytes, ws.ptr, ws.bytes, s);
          }),
          "sgqd_attn_decode_int8");
    return o.result();
}

// attn_decode_prefix_int8(qkv, cache, prefix, prefix_len, cos, sin, pos, n_heads, out, prepared, workspace)
PyObject* attn_decode_prefix_int8(PyObject* const* a, Py_ssize_t n) {
    if (n != 11) raise(PyExc_TypeError, "attn_decode_prefix_int8 takes eleven arguments");
    const Cache8 cache(a[1]), prefix(a[2]);
    const Ints len(a[3], "prefix_len must be one int32");
    if (len.n != 1) raise(PyExc_RuntimeError, "prefix_len must be one int32");
    if (prefix.c.batch != 1 || prefix.c.n_kv_heads != cache.c.n_kv_heads || prefix.c.head_dim != cache.c.head_dim)
        raise(PyExc_RuntimeError, "the prefix is one sequence with the cache's heads");
    Rotary r(a[0], cache, a[4], a[5], a[6], a[7], true);
    const c10::Device d = r.qkv.t.device();
    prefix.on(d);
    if (len.t.device() != d) raise(PyExc_ValueError, "all tensors must be on one GPU");
    const c10::cuda::CUDAGuard guard(d);
    r.readable();
    DecodeOut o(a[8], a[9], r);
    const Scratch ws(a[10], sgqd_attn_decode_prefix_int8_workspace_bytes(cache.c.batch, r.heads, cache.c.n_kv_heads, cache.c.head_dim, cache.c.max_seq,
                                                                           prefix.c.max_seq),
                     r.qkv.t);
    if (ws.buf.defined() && ws.buf.device() != d) raise(PyExc_ValueError, "all tensors must be on one GPU");
    void* s = stream();
    check(without_gil([&] {
              return sgqd_attn_decode_prefix_int8(fptr(r.qkv.t), r.qkv.stride, r.heads, fptr(r.cos), fptr(r.sin), r.cos.size(0), r.pos.p, r.pos_stride(),
                                                  &cache.c, &prefix.c, len.p, fptr(o.out), o.stride, o.p, o.bytes, ws.ptr, ws.bytes, s);
          }),
          "sgqd_attn_decode_prefix_int8");
    return o.result();
}

// set_classes(SgqError, QuantizedTensor, Workspace)
PyObject* set_classes(PyObject* const* a, Py_ssize_t n) {
    if (n != 3) raise(PyExc_TypeError, "set_classes takes three arguments");
    PyObject** const classes[] = {&g_error_class, &g_tensor_class, &g_workspace_class};
    for (int i = 0; i < 3; ++i) {
        Py_INCREF(a[i]);
        Py_XDECREF(*classes[i]);
        *classes[i] = a[i];
    }
    Py_RETURN_NONE;
}

#define SGQ_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<name>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {
    SGQ_METHOD(quantized_matmul), SGQ_METHOD(backward_x), SGQ_METHOD(linear_w8a8), SGQ_METHOD(quantize_int8),
    SGQ_METHOD(quantize_int4),    SGQ_METHOD(dequantize), SGQ_METHOD(rope_kv_store_int8), SGQ_METHOD(kv_load_int8),
    SGQ_METHOD(attn_decode_int8), SGQ_METHOD(attn_decode_prefix_int8), SGQ_METHOD(set_classes), {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_sgq_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sgq_torch(void) {
    s_qdata = PyUnicode_InternFromString("qdata");
    s_scales = PyUnicode_InternFromString("scales");
    s_scheme = PyUnicode_InternFromString("scheme");
    s_shape = PyUnicode_InternFromString("original_shape");
    s_group = PyUnicode_InternFromString("group_size");
    s_bits = PyUnicode_InternFromString("bits");
    s_buf = PyUnicode_InternFromString("buf");
    s_get = PyUnicode_InternFromString("get");
    s_k_codes = PyUnicode_InternFromString("k_codes");
    s_k_scales = PyUnicode_InternFromString("k_scales");
    s_v_codes = PyUnicode_InternFromString("v_codes");
    s_v_scales = PyUnicode_InternFromString("v_scales");
    return PyModule_Create(&g_module);
}

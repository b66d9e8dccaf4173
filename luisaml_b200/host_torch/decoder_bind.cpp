// Python binding of include/lcml_decoder.h for torch tensors
// (luisaml_b200._decoder_bind, called by luisaml_b200/decoder.py).
//
// A decode step's kernels take a few microseconds; reading shapes, strides and
// pointers of a dozen tensors from Python costs more than that. Here the same
// checks and the descriptor take about a microsecond. Outputs and scratch come
// from torch's caching allocator, work goes to torch's current stream of the
// tensors' device. Refused arguments raise ValueError, a failing library call
// luisaml_b200.LcmlError; no C++ exception leaves a function.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "lcml_decoder.h"

namespace {

struct Refused {
    std::string what;
};
struct Failed {
    int status;
};
struct Raised {};  // a Python error is already set

PyObject *g_lcml_error = nullptr;

void need(bool ok, const char *what) {
    if (!ok) throw Refused{what};
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) throw Refused{std::string(name) + ": not a torch tensor"};
    return THPVariable_Unpack(o);
}

const at::Tensor *maybe(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return LCML_DTYPE_FLOAT;
        case at::kHalf: return LCML_DTYPE_FLOAT16;
        case at::kBFloat16: return LCML_DTYPE_BFLOAT16;
        default: return 0;
    }
}

int dtype_of(const at::Tensor &t, const char *name) {
    const int c = dtype_code(t.scalar_type());
    if (c == 0) throw Refused{std::string(name) + ": unsupported dtype " + at::toString(t.scalar_type())};
    return c;
}

double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

int64_t integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised{};
    return v != 0;
}

void check(int status) {
    if (status != LCML_OK) throw Failed{status};
}

// The device all tensors are on.
template <typename... Ts>
c10::Device device_of(const at::Tensor &first, const Ts *...rest) {
    need(first.is_cuda(), "luisaml_b200 ops take CUDA tensors");
    const c10::Device d = first.device();
    need(((rest == nullptr || rest->device() == d) && ...), "tensors on different devices");
    return d;
}

// The operators have no backward: a graph through them would end without a word.
template <typename... Ts>
void no_gradient(const Ts *...t) {
    if (at::GradMode::is_enabled())
        need(((t == nullptr || !t->requires_grad()) && ...), "no gradient flows through this operator: detach its inputs or call it under torch.no_grad()");
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType t, c10::Device d) { return at::detail::empty_cuda(size, t, d, std::nullopt); }

PyObject *wrap(const at::Tensor &t) {
    PyObject *o = THPVariable_Wrap(t);
    if (o == nullptr) throw Raised{};
    return o;
}

PyObject *same(PyObject *o) {
    Py_INCREF(o);
    return o;
}

lcml_kv_cache cache_of(const at::Tensor &k, const at::Tensor &v, const at::Tensor &ks, const at::Tensor &vs) {
    need(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == at::kByte && v.scalar_type() == at::kByte && k.is_contiguous() && v.is_contiguous(),
         "k_cache and v_cache are uint8 [pages, kv_heads, page_size, head_dim], contiguous");
    need(ks.dim() == 3 && ks.sizes() == vs.sizes() && ks.size(0) == k.size(0) && ks.size(1) == k.size(1) && ks.size(2) > 0 &&
             k.size(2) % ks.size(2) == 0 && ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.is_contiguous() && vs.is_contiguous(),
         "k_scale and v_scale are float32 [pages, kv_heads, page_size // scale_block], contiguous");
    need(k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX && k.size(3) <= INT32_MAX, "cache extents exceed 32 bits");
    lcml_kv_cache c{};
    c.k = static_cast<uint8_t *>(k.data_ptr());
    c.v = static_cast<uint8_t *>(v.data_ptr());
    c.k_scale = static_cast<float *>(ks.data_ptr());
    c.v_scale = static_cast<float *>(vs.data_ptr());
    c.num_pages = k.size(0);
    c.kv_heads = static_cast<int32_t>(k.size(1));
    c.page_size = static_cast<int32_t>(k.size(2));
    c.head_dim = static_cast<int32_t>(k.size(3));
    c.scale_block = static_cast<int32_t>(k.size(2) / ks.size(2));
    return c;
}

lcml_kv_batch batch_of(const at::Tensor &table, const at::Tensor &cu, const at::Tensor &lengths, int64_t total) {
    need(table.scalar_type() == at::kInt && cu.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt && table.dim() == 2 && cu.dim() == 1 &&
             lengths.dim() == 1 && table.size(0) == lengths.size(0) && cu.size(0) == lengths.size(0) + 1,
         "block_table [batch, columns], cu_tokens [batch + 1] and the lengths [batch] are int32");
    need((table.size(1) <= 1 || table.stride(1) == 1) && (table.size(0) <= 1 || table.stride(0) >= table.size(1)) && cu.is_contiguous() &&
             lengths.is_contiguous(),
         "block_table's rows, cu_tokens and the lengths are contiguous");
    need(table.size(1) <= INT32_MAX && lengths.size(0) <= INT32_MAX, "batch extents exceed 32 bits");
    lcml_kv_batch b{};
    b.batch = static_cast<int32_t>(lengths.size(0));
    b.table_cols = static_cast<int32_t>(table.size(1));
    b.block_table = static_cast<const int32_t *>(table.data_ptr());
    b.table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
    b.cu_tokens = static_cast<const int32_t *>(cu.data_ptr());
    b.lengths = static_cast<const int32_t *>(lengths.data_ptr());
    b.total_tokens = total;
    return b;
}

lcml_stream_t stream_of(c10::Device d) { return reinterpret_cast<lcml_stream_t>(c10::cuda::getCurrentCUDAStream(d.index()).stream()); }

// rmsnorm_quantize(x, weight, residual, eps, scale, out, scale_out, h_out)
PyObject *rmsnorm_quantize(PyObject *const *o) {
    const at::Tensor &x = tensor(o[0], "x"), &w = tensor(o[1], "weight");
    const at::Tensor *r = maybe(o[2], "residual"), *s = maybe(o[4], "scale"), *out = maybe(o[5], "out"), *s_out = maybe(o[6], "scale_out"),
                     *h_out = maybe(o[7], "h_out");
    need(x.dim() == 2, "rmsnorm_quantize: x is [rows, cols]");
    no_gradient(&x, &w, r, s);
    const c10::Device dev = device_of(x, &w, r, s, out, s_out, h_out);
    lcml_rmsnorm_desc d{};
    const int64_t rows = d.rows = x.size(0), cols = d.cols = x.size(1);
    d.x_dtype = dtype_of(x, "x");
    d.weight_dtype = dtype_of(w, "weight");
    need(d.weight_dtype == d.x_dtype || d.weight_dtype == LCML_DTYPE_FLOAT, "rmsnorm_quantize: weight is of x's type or float32");
    need(w.dim() == 1 && w.size(0) == cols && w.is_contiguous(), "rmsnorm_quantize: weight is [cols], contiguous");
    auto row_stride = [&](const at::Tensor &t) -> int64_t {
        need(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && (cols <= 1 || t.stride(1) == 1) && (rows <= 1 || t.stride(0) >= cols),
             "rmsnorm_quantize: x, residual and h_out share x's shape and type, with contiguous rows that do not overlap");
        return rows > 1 ? t.stride(0) : cols;
    };
    c10::cuda::CUDAGuard guard(dev);
    at::Tensor made_h, made_q, made_s;
    PyObject *po = o[5], *ps = s ? o[4] : o[6], *ph = o[7];
    d.ldx = row_stride(x);
    d.x = x.data_ptr();
    if (r) {
        d.ldr = row_stride(*r);
        d.residual = r->data_ptr();
        if (!h_out) {
            made_h = empty(x.sizes(), x.scalar_type(), dev);
            h_out = &made_h;
        }
    }
    if (h_out) {
        d.ldh = row_stride(*h_out);
        d.h_out = h_out->data_ptr();
    }
    if (!out) {
        made_q = empty(x.sizes(), at::kByte, dev);
        out = &made_q;
    }
    need(out->sizes() == x.sizes() && out->scalar_type() == at::kByte && out->is_contiguous(), "rmsnorm_quantize: out is uint8 [rows, cols], contiguous");
    if (s) {
        need(!s_out, "rmsnorm_quantize: give scale or scale_out, not both");
        need(s->numel() == 1 && s->scalar_type() == at::kFloat, "rmsnorm_quantize: scale is one float32");
        d.scale = static_cast<const float *>(s->data_ptr());
    } else {
        if (!s_out) {
            made_s = empty({rows}, at::kFloat, dev);
            s_out = &made_s;
        }
        need(s_out->dim() == 1 && s_out->size(0) == rows && s_out->scalar_type() == at::kFloat && s_out->is_contiguous(),
             "rmsnorm_quantize: scale_out is float32 [rows]");
        d.scale_out = static_cast<float *>(s_out->data_ptr());
    }
    d.weight = w.data_ptr();
    d.eps = static_cast<float>(number(o[3]));
    d.q = static_cast<uint8_t *>(out->data_ptr());
    check(lcml_rmsnorm_quantize(&d, stream_of(dev)));
    PyObject *a = made_q.defined() ? wrap(made_q) : same(po);
    PyObject *b = made_s.defined() ? wrap(made_s) : same(ps);
    PyObject *c = made_h.defined() ? wrap(made_h) : same(ph);
    PyObject *t = PyTuple_New(3);
    PyTuple_SET_ITEM(t, 0, a);
    PyTuple_SET_ITEM(t, 1, b);
    PyTuple_SET_ITEM(t, 2, c);
    return t;
}

// kv_cache_write(k_cache, v_cache, k_scale, v_scale, k, v, block_table, cu_tokens, start)
PyObject *kv_cache_write(PyObject *const *o) {
    const at::Tensor &kc = tensor(o[0], "k_cache"), &vc = tensor(o[1], "v_cache"), &ks = tensor(o[2], "k_scale"), &vs = tensor(o[3], "v_scale"),
                     &k = tensor(o[4], "k"), &v = tensor(o[5], "v"), &table = tensor(o[6], "block_table"), &cu = tensor(o[7], "cu_tokens"),
                     &start = tensor(o[8], "start");
    no_gradient(&k, &v, &ks, &vs);
    const c10::Device dev = device_of(kc, &vc, &ks, &vs, &k, &v, &table, &cu, &start);
    const lcml_kv_cache c = cache_of(kc, vc, ks, vs);
    const int dt = dtype_of(k, "k");
    need(k.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.size(1) == c.kv_heads && k.size(2) == c.head_dim &&
             k.stride(2) == 1 && v.stride(2) == 1,
         "k and v are [tokens, kv_heads, head_dim] of one type, with contiguous rows");
    const lcml_kv_batch b = batch_of(table, cu, start, k.size(0));
    c10::cuda::CUDAGuard guard(dev);
    check(lcml_kv_cache_write(&c, &b, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), dt, stream_of(dev)));
    Py_RETURN_NONE;
}

// kv_cache_read(k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, start, total, dtype)
PyObject *kv_cache_read(PyObject *const *o) {
    const at::Tensor &kc = tensor(o[0], "k_cache"), &vc = tensor(o[1], "v_cache"), &ks = tensor(o[2], "k_scale"), &vs = tensor(o[3], "v_scale"),
                     &table = tensor(o[4], "block_table"), &cu = tensor(o[5], "cu_tokens"), &start = tensor(o[6], "start");
    const int64_t total = integer(o[7]);
    need(THPDtype_Check(o[8]), "kv_cache_read: dtype is a torch dtype");
    const at::ScalarType t = reinterpret_cast<THPDtype *>(o[8])->scalar_type;
    const int dt = dtype_code(t);
    need(dt != 0, "kv_cache_read: dtype is float32, float16 or bfloat16");
    need(total >= 0, "kv_cache_read: negative total");
    no_gradient(&ks, &vs);
    const c10::Device dev = device_of(kc, &vc, &ks, &vs, &table, &cu, &start);
    const lcml_kv_cache c = cache_of(kc, vc, ks, vs);
    const lcml_kv_batch b = batch_of(table, cu, start, total);
    c10::cuda::CUDAGuard guard(dev);
    const at::Tensor k = empty({total, c.kv_heads, c.head_dim}, t, dev), v = empty({total, c.kv_heads, c.head_dim}, t, dev);
    if (total > 0) check(lcml_kv_cache_read(&c, &b, k.data_ptr(), v.data_ptr(), dt, stream_of(dev)));
    PyObject *a = wrap(k), *e = wrap(v);
    PyObject *r = PyTuple_New(2);
    PyTuple_SET_ITEM(r, 0, a);
    PyTuple_SET_ITEM(r, 1, e);
    return r;
}

// kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_tokens, kv_len, max_tokens, scale, causal, window, softcap, out, lse,
//              workspace, variant, size_only)
PyObject *kv_attention(PyObject *const *o) {
    const at::Tensor &q = tensor(o[0], "q"), &kc = tensor(o[1], "k_cache"), &vc = tensor(o[2], "v_cache"), &ks = tensor(o[3], "k_scale"),
                     &vs = tensor(o[4], "v_scale"), &table = tensor(o[5], "block_table"), &cu = tensor(o[6], "cu_tokens"), &len = tensor(o[7], "kv_len");
    const at::Tensor *out = maybe(o[13], "out"), *lse = maybe(o[14], "lse"), *ws = maybe(o[15], "workspace");
    no_gradient(&q, &ks, &vs);
    const c10::Device dev = device_of(q, &kc, &vc, &ks, &vs, &table, &cu, &len, out, lse, ws);
    const lcml_kv_cache c = cache_of(kc, vc, ks, vs);
    need(q.dim() == 3 && q.size(2) == c.head_dim && q.stride(2) == 1, "kv_attention: q is [tokens, q_heads, head_dim] with contiguous rows");
    need(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "kv_attention: q is float16 or bfloat16");
    const lcml_kv_batch b = batch_of(table, cu, len, q.size(0));
    lcml_kv_attention_desc d{};
    d.cache = &c;
    d.batch = &b;
    d.q = q.data_ptr();
    d.q_token_stride = q.stride(0);
    d.q_head_stride = q.stride(1);
    need(q.size(1) <= INT32_MAX, "kv_attention: too many heads");
    d.q_heads = static_cast<int32_t>(q.size(1));
    d.dtype = dtype_code(q.scalar_type());
    d.max_tokens = o[8] == Py_None ? q.size(0) : integer(o[8]);
    d.softmax_scale = o[9] == Py_None ? 1.0f / std::sqrt(static_cast<float>(c.head_dim)) : static_cast<float>(number(o[9]));
    d.causal = truth(o[10]);
    const int64_t window = integer(o[11]);
    need(window <= INT32_MAX && window >= INT32_MIN, "kv_attention: window exceeds 32 bits");
    d.window = static_cast<int32_t>(window);
    d.softcap = static_cast<float>(number(o[12]));
    d.variant = static_cast<int>(integer(o[16]));
    c10::cuda::CUDAGuard guard(dev);
    const int64_t bytes = lcml_kv_attention_workspace_size(&d);
    if (bytes < 0) throw Failed{LCML_ERR_INVALID_ARGUMENT};
    if (truth(o[17])) return PyLong_FromLongLong(bytes);
    at::Tensor made, made_ws;
    if (!out) {
        made = empty(q.sizes(), q.scalar_type(), dev);
        out = &made;
    }
    need(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && out->stride(2) == 1,
         "kv_attention: out has q's shape and type, with contiguous rows");
    d.out = out->data_ptr();
    d.out_token_stride = out->stride(0);
    d.out_head_stride = out->stride(1);
    if (lse) {
        need(lse->dim() == 2 && lse->size(0) == q.size(0) && lse->size(1) == q.size(1) && lse->scalar_type() == at::kFloat && lse->is_contiguous(),
             "kv_attention: lse is float32 [tokens, q_heads]");
        d.lse = static_cast<float *>(lse->data_ptr());
    }
    if (bytes > 0) {
        if (!ws) {
            made_ws = empty({bytes}, at::kByte, dev);
            ws = &made_ws;
        }
        need(ws->is_contiguous() && static_cast<int64_t>(ws->nbytes()) >= bytes, "kv_attention: the workspace is too small");
        d.workspace = ws->data_ptr();
    }
    check(lcml_kv_attention(&d, stream_of(dev)));
    return made.defined() ? wrap(made) : same(o[13]);
}

// Runs F on exactly N positional arguments; every error becomes a Python one.
template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Raised &) {
    } catch (const Refused &e) {
        PyErr_SetString(PyExc_ValueError, e.what.c_str());
    } catch (const Failed &e) {
        PyObject *x = PyObject_CallFunction(g_lcml_error, "is", e.status, lcml_last_error());
        if (x != nullptr) {
            PyErr_SetObject(g_lcml_error, x);
            Py_DECREF(x);
        }
    } catch (const c10::OutOfMemoryError &e) {
        PyObject *m = PyImport_ImportModule("torch");
        PyObject *x = m ? PyObject_GetAttrString(m, "OutOfMemoryError") : nullptr;
        if (x != nullptr) PyErr_SetString(x, e.what_without_backtrace());
        Py_XDECREF(x);
        Py_XDECREF(m);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
constexpr PyCFunction fast() {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>));
}

PyMethodDef methods[] = {
    {"rmsnorm_quantize", fast<rmsnorm_quantize, 8>(), METH_FASTCALL, nullptr},
    {"kv_cache_write", fast<kv_cache_write, 9>(), METH_FASTCALL, nullptr},
    {"kv_cache_read", fast<kv_cache_read, 9>(), METH_FASTCALL, nullptr},
    {"kv_attention", fast<kv_attention, 18>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decoder_bind", "Binding of lcml_decoder.h for torch tensors.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}// namespace

PyMODINIT_FUNC PyInit__decoder_bind() {
    PyObject *capi = PyImport_ImportModule("luisaml_b200._capi");
    if (capi == nullptr) return nullptr;
    g_lcml_error = PyObject_GetAttrString(capi, "LcmlError");
    Py_DECREF(capi);
    if (g_lcml_error == nullptr) return nullptr;
    return PyModule_Create(&module);
}

// Python binding of include/lcml_decoder.h and include/lcml_decode_step.h for torch tensors
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

#include "lcml_decode_step.h"

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
//              workspace, variant, size_only, sinks)
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
    const int64_t sinks = integer(o[18]);
    need(sinks >= 0 && sinks <= INT32_MAX, "kv_attention: sinks is negative or exceeds 32 bits");
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
    check(lcml_kv_attention_sinks(&d, static_cast<int32_t>(sinks), stream_of(dev)));
    return made.defined() ? wrap(made) : same(o[13]);
}

// An int32 output of n values: the one given, or a new one.
at::Tensor int_output(const at::Tensor *given, int64_t n, c10::Device dev, const char *what) {
    if (given == nullptr) return empty({n}, at::kInt, dev);
    need(given->dim() == 1 && given->size(0) == n && given->scalar_type() == at::kInt && given->is_contiguous(), what);
    return *given;
}

// kv_plan(new_tokens, held, block_table, free_pages, free_count, ended, page_size, total, kv_len, free_count_out)
// -> (cu_tokens, start, kv_len, positions, slots, free_count)
PyObject *kv_plan(PyObject *const *o) {
    const at::Tensor &fresh = tensor(o[0], "new_tokens"), &held = tensor(o[1], "held"), &table = tensor(o[2], "block_table"), &free = tensor(o[3], "free_pages"),
                     &count = tensor(o[4], "free_count");
    const at::Tensor *ended = maybe(o[5], "ended"), *len_out = maybe(o[8], "kv_len"), *count_out = maybe(o[9], "free_count_out");
    const c10::Device dev = device_of(fresh, &held, &table, &free, &count, ended, len_out, count_out);
    const int64_t page_size = integer(o[6]), total = integer(o[7]), batch = fresh.dim() == 1 ? fresh.size(0) : -1;
    need(batch >= 0 && fresh.scalar_type() == at::kInt && held.scalar_type() == at::kInt && held.dim() == 1 && held.size(0) == batch && fresh.is_contiguous() &&
             held.is_contiguous(),
         "kv_plan: new_tokens and held are int32 [batch], contiguous");
    need(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == batch && (table.size(1) <= 1 || table.stride(1) == 1) &&
             (batch <= 1 || table.stride(0) >= table.size(1)),
         "kv_plan: block_table is int32 [batch, columns] with contiguous rows");
    need(free.scalar_type() == at::kInt && free.dim() == 1 && free.is_contiguous() && count.scalar_type() == at::kInt && count.numel() == 1,
         "kv_plan: free_pages is int32 [pages], contiguous, and free_count one int32");
    need(ended == nullptr || ((ended->scalar_type() == at::kBool || ended->scalar_type() == at::kByte) && ended->dim() == 1 && ended->size(0) == batch && ended->is_contiguous()),
         "kv_plan: ended is bool or uint8 [batch], contiguous");
    need(page_size > 0 && page_size <= INT32_MAX && total >= 0 && table.size(1) <= INT32_MAX && batch <= INT32_MAX, "kv_plan: an extent is negative or exceeds 32 bits");
    c10::cuda::CUDAGuard guard(dev);
    // One allocation for all outputs that are not given: views of it cost a tenth of an allocation each.
    const int64_t row = (batch + 4) / 4 * 4, tokens = (total + 3) / 4 * 4;
    const at::Tensor all = empty({3 * row + 4 + 2 * tokens}, at::kInt, dev);
    auto part = [&](int64_t from, int64_t n) {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
        t.unsafeGetTensorImpl()->set_storage_offset(from);
        t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
        return t;
    };
    const at::Tensor cu = part(0, batch + 1), start = part(row, batch), positions = part(3 * row + 4, total), slots = part(3 * row + 4 + tokens, total);
    const at::Tensor len = len_out ? int_output(len_out, batch, dev, "kv_plan: kv_len is int32 [batch], contiguous") : part(2 * row, batch),
                     left = count_out ? int_output(count_out, 1, dev, "kv_plan: free_count_out is int32 [1]") : part(3 * row, 1);
    lcml_kv_plan_desc d{};
    d.batch = static_cast<int32_t>(batch);
    d.page_size = static_cast<int32_t>(page_size);
    d.table_cols = static_cast<int32_t>(table.size(1));
    d.table_stride = batch > 1 ? table.stride(0) : table.size(1);
    d.block_table = static_cast<int32_t *>(table.data_ptr());
    d.new_tokens = static_cast<const int32_t *>(fresh.data_ptr());
    d.held = static_cast<const int32_t *>(held.data_ptr());
    d.ended = ended ? static_cast<const uint8_t *>(ended->data_ptr()) : nullptr;
    d.free_pages = static_cast<int32_t *>(free.data_ptr());
    d.free_capacity = free.size(0);
    d.free_count = static_cast<const int32_t *>(count.data_ptr());
    d.total_tokens = total;
    d.cu_tokens = static_cast<int32_t *>(cu.data_ptr());
    d.start = static_cast<int32_t *>(start.data_ptr());
    d.kv_len = static_cast<int32_t *>(len.data_ptr());
    d.positions = static_cast<int32_t *>(positions.data_ptr());
    d.slots = static_cast<int32_t *>(slots.data_ptr());
    d.free_count_out = static_cast<int32_t *>(left.data_ptr());
    check(lcml_kv_plan(&d, stream_of(dev)));
    const at::Tensor *out[6] = {&cu, &start, &len, &positions, &slots, &left};
    PyObject *t = PyTuple_New(6);
    if (t == nullptr) throw Raised{};
    for (int i = 0; i < 6; ++i) {
        PyObject *x = i == 2 && len_out ? same(o[8]) : (i == 5 && count_out ? same(o[9]) : THPVariable_Wrap(*out[i]));
        if (x == nullptr) {
            Py_DECREF(t);
            throw Raised{};
        }
        PyTuple_SET_ITEM(t, i, x);
    }
    return t;
}

// qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, q_out, k_out) -> (q_out, k_out)
PyObject *qk_norm_rope(PyObject *const *o) {
    const at::Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k"), &pos = tensor(o[2], "positions"), &freq = tensor(o[3], "inv_freq");
    const at::Tensor *qw = maybe(o[4], "q_weight"), *kw = maybe(o[5], "k_weight"), *q_out = maybe(o[8], "q_out"), *k_out = maybe(o[9], "k_out");
    no_gradient(&q, &k, &freq, qw, kw);
    const c10::Device dev = device_of(q, &k, &pos, &freq, qw, kw, q_out, k_out);
    lcml_qk_norm_rope_desc d{};
    d.dtype = dtype_of(q, "q");
    need(q.dim() == 3 && k.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.scalar_type() == k.scalar_type() && q.size(1) <= INT32_MAX &&
             k.size(1) <= INT32_MAX && q.size(2) <= INT32_MAX,
         "qk_norm_rope: q and k are [tokens, heads, head_dim] of one type");
    const int64_t dim = q.size(2);
    need(pos.scalar_type() == at::kInt && pos.dim() == 1 && pos.size(0) == q.size(0) && pos.is_contiguous(), "qk_norm_rope: positions is int32 [tokens], contiguous");
    need((freq.scalar_type() == at::kFloat || freq.scalar_type() == at::kDouble) && freq.dim() == 1 && freq.is_contiguous() && freq.size(0) <= dim / 2,
         "qk_norm_rope: inv_freq is float32 or float64 [rotary / 2], contiguous, rotary at most head_dim");
    d.weight_dtype = LCML_DTYPE_FLOAT;
    for (const at::Tensor *w : {qw, kw}) {
        if (w == nullptr) continue;
        need(w->dim() == 1 && w->size(0) == dim && w->is_contiguous() && (w->scalar_type() == q.scalar_type() || w->scalar_type() == at::kFloat),
             "qk_norm_rope: q_weight and k_weight are [head_dim], contiguous, of q's type or float32");
        d.weight_dtype = dtype_of(*w, "weight");
    }
    need(qw == nullptr || kw == nullptr || qw->scalar_type() == kw->scalar_type(), "qk_norm_rope: q_weight and k_weight have one type");
    c10::cuda::CUDAGuard guard(dev);
    at::Tensor made_q, made_k;
    if (!q_out) {
        made_q = empty(q.sizes(), q.scalar_type(), dev);
        q_out = &made_q;
    }
    if (!k_out) {
        made_k = empty(k.sizes(), k.scalar_type(), dev);
        k_out = &made_k;
    }
    need(q_out->sizes() == q.sizes() && q_out->scalar_type() == q.scalar_type() && k_out->sizes() == k.sizes() && k_out->scalar_type() == k.scalar_type(),
         "qk_norm_rope: q_out and k_out have the shape and type of q and k");
    for (const at::Tensor *t : {&q, &k, q_out, k_out}) need(dim <= 1 || t->stride(2) == 1, "qk_norm_rope: heads are contiguous");
    d.tokens = q.size(0);
    d.q_heads = static_cast<int32_t>(q.size(1));
    d.k_heads = static_cast<int32_t>(k.size(1));
    d.head_dim = static_cast<int32_t>(dim);
    d.rotary = static_cast<int32_t>(2 * freq.size(0));
    d.interleaved = truth(o[7]);
    d.q = q.data_ptr();
    d.k = k.data_ptr();
    d.q_token_stride = q.stride(0), d.q_head_stride = q.stride(1), d.k_token_stride = k.stride(0), d.k_head_stride = k.stride(1);
    d.q_out = q_out->data_ptr();
    d.k_out = k_out->data_ptr();
    d.q_out_token_stride = q_out->stride(0), d.q_out_head_stride = q_out->stride(1), d.k_out_token_stride = k_out->stride(0), d.k_out_head_stride = k_out->stride(1);
    d.q_weight = qw ? qw->data_ptr() : nullptr;
    d.k_weight = kw ? kw->data_ptr() : nullptr;
    d.eps = static_cast<float>(number(o[6]));
    d.positions = static_cast<const int32_t *>(pos.data_ptr());
    d.inv_freq = freq.data_ptr();
    d.inv_freq_dtype = freq.scalar_type() == at::kDouble ? LCML_DTYPE_DOUBLE : LCML_DTYPE_FLOAT;
    check(lcml_qk_norm_rope(&d, stream_of(dev)));
    PyObject *t = PyTuple_New(2);
    if (t == nullptr) throw Raised{};
    for (int i = 0; i < 2; ++i) {
        const at::Tensor &made = i ? made_k : made_q;
        PyObject *x = made.defined() ? THPVariable_Wrap(made) : same(o[8 + i]);
        if (x == nullptr) {
            Py_DECREF(t);
            throw Raised{};
        }
        PyTuple_SET_ITEM(t, i, x);
    }
    return t;
}

// sample(logits, uniform, temperature, top_k, top_p, min_p, out, logprob) -> tokens
PyObject *sample(PyObject *const *o) {
    const at::Tensor &x = tensor(o[0], "logits"), &u = tensor(o[1], "uniform");
    const at::Tensor *t = maybe(o[2], "temperature"), *k = maybe(o[3], "top_k"), *p = maybe(o[4], "top_p"), *m = maybe(o[5], "min_p"), *out = maybe(o[6], "out"),
                     *lp = maybe(o[7], "logprob");
    no_gradient(&x, &u, t, p, m);
    const c10::Device dev = device_of(x, &u, t, k, p, m, out, lp);
    lcml_sample_desc d{};
    d.dtype = dtype_of(x, "logits");
    need(x.dim() == 2, "sample: logits is [rows, vocab]");
    const int64_t rows = x.size(0);
    need((x.size(1) <= 1 || x.stride(1) == 1) && (rows <= 1 || x.stride(0) >= x.size(1)), "sample: rows of logits are contiguous and do not overlap");
    auto row_values = [&](const at::Tensor *v, at::ScalarType type, const char *what) {
        need(v == nullptr || (v->dim() == 1 && v->size(0) == rows && v->scalar_type() == type && v->is_contiguous()), what);
        return v == nullptr ? nullptr : v->data_ptr();
    };
    d.rows = rows;
    d.vocab = x.size(1);
    d.logits = x.data_ptr();
    d.ld = rows > 1 ? x.stride(0) : x.size(1);
    d.uniform = static_cast<const float *>(row_values(&u, at::kFloat, "sample: uniform is float32 [rows], contiguous"));
    d.temperature = static_cast<const float *>(row_values(t, at::kFloat, "sample: temperature is float32 [rows], contiguous"));
    d.top_k = static_cast<const int32_t *>(row_values(k, at::kInt, "sample: top_k is int32 [rows], contiguous"));
    d.top_p = static_cast<const float *>(row_values(p, at::kFloat, "sample: top_p is float32 [rows], contiguous"));
    d.min_p = static_cast<const float *>(row_values(m, at::kFloat, "sample: min_p is float32 [rows], contiguous"));
    d.logprob = static_cast<float *>(row_values(lp, at::kFloat, "sample: logprob is float32 [rows], contiguous"));
    c10::cuda::CUDAGuard guard(dev);
    const at::Tensor tokens = int_output(out, rows, dev, "sample: out is int32 [rows], contiguous");
    d.tokens = static_cast<int32_t *>(tokens.data_ptr());
    check(lcml_sample(&d, stream_of(dev)));
    return out ? same(o[6]) : wrap(tokens);
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
    {"kv_attention", fast<kv_attention, 19>(), METH_FASTCALL, nullptr},
    {"kv_plan", fast<kv_plan, 10>(), METH_FASTCALL, nullptr},
    {"qk_norm_rope", fast<qk_norm_rope, 10>(), METH_FASTCALL, nullptr},
    {"sample", fast<sample, 8>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decoder_bind", "Binding of lcml_decoder.h and lcml_decode_step.h for torch tensors.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}// namespace

PyMODINIT_FUNC PyInit__decoder_bind() {
    PyObject *capi = PyImport_ImportModule("luisaml_b200._capi");
    if (capi == nullptr) return nullptr;
    g_lcml_error = PyObject_GetAttrString(capi, "LcmlError");
    Py_DECREF(capi);
    if (g_lcml_error == nullptr) return nullptr;
    return PyModule_Create(&module);
}

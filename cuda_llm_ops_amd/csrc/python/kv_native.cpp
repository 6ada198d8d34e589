// CPython module `_kv_native`: argument checks and calls of the paged KV cache's
// functions (cuda_llm_ops_amd/kv_cache.py, and the block-scaled form of
// flash_gqa.decode_flash_gqa_paged) over the C ABI of include/fgqa_kv.h.
//
// A single-token step is 4 to 14 us of GPU work and reads some fifty properties
// of up to a dozen tensors.  Reading them here instead of in Python took small
// calls in a row from 10.4 to 4.8 us (append), 8.5 to 4.4 (weights), 18.0 to 13.0
// (eviction) and 18.4 to 12.9 (decode), where the GPU is what takes the time.
//
// Functions take positional arguments from those Python functions, which hold the
// signatures and documentation; they raise ValueError for what the call does not
// take, and FgqaError for a status of the C ABI.  One returns NotImplemented when its
// tensors live on another device than the current one (the caller makes that
// current and calls again).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstring>
#include <initializer_list>
#include <utility>
#include <vector>

#include "../host/kv_apart.h"
#include "fgqa_kv.h"

namespace {

PyObject* g_get_device = nullptr;   // () -> current device's index
PyObject* g_get_stream = nullptr;   // (index) -> its current stream's handle
PyObject* g_error = nullptr;        // FgqaError(status, where)

// A Python exception is set.
struct Raised {};

[[noreturn]] void refuse(const char* format, ...) {
    va_list args;
    va_start(args, format);
    PyErr_FormatV(PyExc_ValueError, format, args);
    va_end(args);
    throw Raised{};
}

bool is_tensor(PyObject* o) { return THPVariable_Check(o); }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!is_tensor(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
        throw Raised{};
    }
    return THPVariable_Unpack(o);
}

// What int(o) gives; *outside: it does not fit 64 bits.
int64_t integer(PyObject* o) {
    PyObject* n = PyNumber_Long(o);
    if (n == nullptr) throw Raised{};
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(n, &overflow);
    Py_DECREF(n);
    if (overflow != 0) return overflow > 0 ? INT64_MAX : INT64_MIN;
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

void* address(const at::Tensor& t) { return t.data_ptr(); }
bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(address(t)) & 15u) == 0; }

// Head dim contiguous, 16-byte aligned base, strides in multiples of 8 elements.
bool kernel_ready(const at::Tensor& t) {
    const auto st = t.strides();
    if (st.back() != 1 || !aligned16(t)) return false;
    for (size_t i = 0; i + 1 < st.size(); ++i)
        if (st[i] & 7) return false;
    return true;
}

at::Tensor ready(const at::Tensor& t) { return kernel_ready(t) ? t : t.contiguous(); }

// No two elements of t share memory (an expanded tensor's do).
bool rows_apart(const at::Tensor& t) {
    if (t.is_contiguous()) return true;
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
    std::sort(dims.begin(), dims.end());
    int64_t end = 1;   // elements that the dims so far span
    for (const auto& d : dims) {
        if (d.first < end) return false;
        end += d.first * (d.second - 1);
    }
    return true;
}

void check_written(const at::Tensor& t) {
    if (!rows_apart(t)) refuse("a tensor that is written must not overlap itself (expanded dims)");
}

void check_written_scales(PyObject* k_scale, PyObject* v_scale) {
    if (is_tensor(k_scale)) check_written(THPVariable_Unpack(k_scale));
    if (is_tensor(v_scale)) check_written(THPVariable_Unpack(v_scale));
}

// The address ranges of a and b overlap.
bool meet(const at::Tensor& a, const at::Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    auto end = [](const at::Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return reinterpret_cast<uintptr_t>(address(t)) + (uintptr_t)(last + 1) * t.element_size();
    };
    return reinterpret_cast<uintptr_t>(address(a)) < end(b) && reinterpret_cast<uintptr_t>(address(b)) < end(a);
}

// Elements of a and b share memory: exactly for views of equal strides (interleaved
// ones are two memories), by their address ranges for others.  Neither overlaps itself.
bool share(const at::Tensor& a, const at::Tensor& b) {
    if (!meet(a, b)) return false;
    if (a.sizes() != b.sizes()) return true;
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return true;
    return fgqa::plan::views_meet(reinterpret_cast<uintptr_t>(address(a)), reinterpret_cast<uintptr_t>(address(b)),
                                  a.sizes().data(), a.strides().data(), (int)a.dim(), (int64_t)a.element_size());
}

// t and the caches or block scales o (others are numbers) share address ranges.
bool meet_any(const at::Tensor& t, std::initializer_list<PyObject*> o) {
    for (PyObject* x : o)
        if (is_tensor(x) && meet(t, THPVariable_Unpack(x))) return true;
    return false;
}

// Caches and block scales that are written: K's and V's lie apart.
void check_apart(const at::Tensor& k, const at::Tensor& v, PyObject* k_scale, PyObject* v_scale) {
    if (share(k, v)) refuse("k_cache and v_cache must be apart");
    if (is_tensor(k_scale) && is_tensor(v_scale) && share(THPVariable_Unpack(k_scale), THPVariable_Unpack(v_scale)))
        refuse("k_scale and v_scale must be apart");
}

// All tensors of a call live on one GPU.
struct Device {
    int64_t index = -1;
    bool first = true;
    void add(const at::Tensor& t) {
        const int64_t at = t.is_cuda() ? t.get_device() : -1;
        if (first) {
            if (at < 0) refuse("Flash GQA tensors must live on the GPU");
            index = at;
            first = false;
        } else if (at != index) {
            refuse("all tensors must be on cuda:%lld, got one on %s", (long long)index, t.device().str().c_str());
        }
    }
    void add_if(PyObject* o) {
        if (is_tensor(o)) add(THPVariable_Unpack(o));
    }
    // The index is the current device's; its stream in *stream.
    bool current(void** stream) const {
        PyObject* now = PyObject_CallNoArgs(g_get_device);
        if (now == nullptr) throw Raised{};
        const bool same = PyLong_AsLongLong(now) == index;
        if (same) {
            PyObject* s = PyObject_CallOneArg(g_get_stream, now);
            Py_DECREF(now);
            if (s == nullptr) throw Raised{};
            *stream = reinterpret_cast<void*>(PyLong_AsUnsignedLongLong(s));
            Py_DECREF(s);
        } else {
            Py_DECREF(now);
        }
        if (PyErr_Occurred()) throw Raised{};
        return same;
    }
};

// Autograd learns that t was written (inference tensors have no version).
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written_if(PyObject* o) {
    if (is_tensor(o)) written(THPVariable_Unpack(o));
}

PyObject* not_here() { Py_RETURN_NOTIMPLEMENTED; }

void raise_status(int status, const char* where) {
    if (status == FGQA_OK) return;
    PyObject* e = PyObject_CallFunction(g_error, "is", status, where);
    if (e != nullptr) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

template <typename Args>
void launch(int (*f)(const Args*, void*), const Args& a, void* stream, const char* where) {
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f(&a, stream);
    Py_END_ALLOW_THREADS
    raise_status(status, where);
}

// ---------------------------------------------------------------- the cache
const char* const kCacheShape = "must be [num_pages, page_size, Hkv, D]";

void check_cache(const at::Tensor& t, const char* name, int* dtype) {
    const auto type = t.scalar_type();
    *dtype = type == at::kBFloat16 ? FGQA_KV_BF16 : type == at::kFloat8_e4m3fn ? FGQA_KV_FP8_E4M3
             : type == at::kChar   ? FGQA_KV_INT8
                                   : -1;
    if (*dtype < 0) refuse("%s must be bf16, float8_e4m3fn or int8", name);
    if (t.dim() != 4) refuse("%s %s", name, kCacheShape);
    const auto n = t.sizes();
    const auto st = t.strides();
    if (n[1] < 1 || n[1] > INT_MAX || (n[1] & (n[1] - 1))) refuse("page_size must be a power of two");
    if (n[3] != 128 || n[2] < 1) refuse("head_dim must be 128 on this path");
    if (n[0] > INT_MAX || n[2] > INT_MAX) refuse("%s has too many pages or heads", name);
    if (st[3] != 1) refuse("the caches' head_dim must be contiguous");
    const int64_t mask = *dtype == FGQA_KV_BF16 ? 7 : 15;
    if (!aligned16(t) || ((st[0] | st[1] | st[2]) & mask))
        refuse("%s must be 16-byte aligned, with strides in multiples of 16 bytes", name);
}

// A tensor of one element stands for a number, unless it is all block scales of a
// cache of one page and head.
bool may_be_number(PyObject* o) { return !is_tensor(o) || THPVariable_Unpack(o).numel() == 1; }
bool may_be_blocks(PyObject* o, const at::Tensor& cache) {
    if (!is_tensor(o)) return false;
    const at::Tensor& s = THPVariable_Unpack(o);
    return s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == cache.size(0) && s.size(1) == cache.size(2) &&
           s.device() == cache.device();
}

PyObject* blocks_or_none(const float* scales, PyObject* o) { return scales != nullptr ? o : Py_None; }

// k_scale or v_scale: block scales (returned) or one for the cache.
float* check_scale(PyObject* o, bool as_number, const at::Tensor& cache, int dtype, const char* name, float* whole,
                   int64_t (&st)[2]) {
    *whole = 1.f;
    st[0] = st[1] = 0;
    if (is_tensor(o) && !as_number) {
        const at::Tensor& s = THPVariable_Unpack(o);
        if (dtype == FGQA_KV_BF16) refuse("bf16 caches have no block scales");
        if (s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != cache.size(0) || s.size(1) != cache.size(2))
            refuse("%s must be an fp32 [num_pages, Hkv] tensor", name);
        st[0] = s.stride(0);
        st[1] = s.stride(1);
        return static_cast<float*>(address(s));
    }
    if (dtype == FGQA_KV_INT8) refuse("int8 caches need %s as an fp32 [num_pages, Hkv] tensor", name);
    const double v = number(o);
    if (!std::isfinite(v) || !std::isfinite((float)v)) refuse("%s must be finite", name);
    if (dtype == FGQA_KV_BF16 && v != 1.0) refuse("bf16 caches have no scale");
    *whole = (float)v;
    return nullptr;
}

// v null: a call that reads K only.
fgqa_kv_cache check_caches(const at::Tensor& k, const at::Tensor* v, PyObject* k_scale, PyObject* v_scale) {
    fgqa_kv_cache c;
    std::memset(&c, 0, sizeof c);
    int dtype = 0;
    check_cache(k, "k_cache", &dtype);
    // (both scales in one way)
    const bool numbers = dtype != FGQA_KV_INT8 && may_be_number(k_scale) && (v == nullptr || may_be_number(v_scale)) &&
                         !(dtype == FGQA_KV_FP8_E4M3 && may_be_blocks(k_scale, k) &&
                           (v == nullptr || may_be_blocks(v_scale, *v)));
    if (v != nullptr) {
        if (v->scalar_type() != k.scalar_type() || v->sizes() != k.sizes())
            refuse("k_cache and v_cache must share dtype and shape");
        check_cache(*v, "v_cache", &dtype);
        if (!numbers && is_tensor(k_scale) != is_tensor(v_scale) && dtype != FGQA_KV_INT8)
            refuse("k_scale and v_scale must both be tensors or both numbers");
        c.v_scales = check_scale(v_scale, numbers, *v, dtype, "v_scale", &c.v_scale, c.v_scales_stride);
        c.v = address(*v);
        for (int i = 0; i < 3; ++i) c.v_stride[i] = v->stride(i);
    }
    c.k_scales = check_scale(k_scale, numbers, k, dtype, "k_scale", &c.k_scale, c.k_scales_stride);
    c.k = address(k);
    for (int i = 0; i < 3; ++i) c.k_stride[i] = k.stride(i);
    c.kv_dtype = dtype;
    c.num_pages = (int32_t)k.size(0);
    c.page_size = (int32_t)k.size(1);
    c.num_kv_heads = (int32_t)k.size(2);
    c.head_dim = 128;
    return c;
}

// A block table's stride of rows; its width in *pages.
int64_t check_table(const at::Tensor& t, int64_t B, const char* name, int64_t* pages) {
    if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != B || (t.stride(1) != 1 && t.size(1) > 1 && B > 0))
        refuse("%s must be an int32 [B, max_pages] tensor with contiguous rows", name);
    *pages = t.size(1);
    return B > 1 ? t.stride(0) : t.size(1);
}

int32_t* check_lens(const at::Tensor& t, int64_t B, const char* name) {
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != B || !t.is_contiguous())
        refuse("%s must be a contiguous int32 [B] tensor", name);
    return static_cast<int32_t*>(address(t));
}

int32_t* int32s(const at::Tensor& t) { return static_cast<int32_t*>(address(t)); }
float* floats(const at::Tensor& t) { return static_cast<float*>(address(t)); }

int32_t check_batch(int64_t B) {
    if (B > INT_MAX) refuse("the batch is too large");
    return (int32_t)B;
}

// Tokens of a block table's row, as far as an int goes.
int64_t table_tokens(int64_t pages, const fgqa_kv_cache& c) {
    return pages > INT_MAX / c.page_size ? INT_MAX : pages * c.page_size;
}

int32_t check_max_seqlen(PyObject* o, int64_t tokens, int64_t otherwise) {
    if (o == Py_None) return (int32_t)otherwise;
    const int64_t n = integer(o);
    if (n < 0 || n > tokens) refuse("max_seqlen must be between 0 and the block table's tokens");
    return (int32_t)n;
}

// Tokens of a row of weights.
int64_t check_weights(const at::Tensor& t, int64_t B, int64_t heads, const char* name) {
    if (t.scalar_type() != at::kFloat || t.dim() != 3 || t.size(0) != B || t.size(1) != heads || t.size(2) > INT_MAX ||
        (t.stride(2) != 1 && t.size(2) > 1 && t.numel() > 1))
        refuse("%s must be an fp32 [B, Hkv, W] tensor with contiguous rows", name);
    return t.size(2);
}

// ---------------------------------------------------------------- functions
// append(k, v, k_cache, v_cache, block_table, seqlens, new_lens, k_scale, v_scale)
PyObject* append(PyObject* const* o) {
    const at::Tensor &k = tensor(o[0], "k"), &v = tensor(o[1], "v");
    const at::Tensor &kc = tensor(o[2], "k_cache"), &vc = tensor(o[3], "v_cache");
    const at::Tensor &table = tensor(o[4], "block_table"), &lens = tensor(o[5], "seqlens");
    if (k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16) refuse("append expects bf16 tokens");
    fgqa_kv_append_args a;
    std::memset(&a, 0, sizeof a);
    a.cache = check_caches(kc, &vc, o[7], o[8]);
    if (k.dim() != 4 || v.sizes() != k.sizes() || k.size(2) != kc.size(2) || k.size(3) != 128)
        refuse("K and V must be [B, N, Hkv, D] matching the caches");
    if (k.size(1) > INT_MAX) refuse("too many new tokens");
    const int64_t B = a.batch = check_batch(k.size(0));
    int64_t pages;
    a.block_table_stride = check_table(table, B, "block_table", &pages);
    if (pages > INT_MAX) refuse("block_table has too many pages");
    a.seqlens = check_lens(lens, B, "seqlens");
    if (o[6] != Py_None) a.new_lens = check_lens(tensor(o[6], "new_lens"), B, "new_lens");
    if (a.cache.k_scales == nullptr && !(a.cache.k_scale > 0.f && a.cache.v_scale > 0.f))
        refuse("k_scale and v_scale must be positive");
    check_written(kc);
    check_written(vc);
    PyObject *const ks = blocks_or_none(a.cache.k_scales, o[7]), *const vs = blocks_or_none(a.cache.v_scales, o[8]);
    check_written_scales(ks, vs);
    check_apart(kc, vc, ks, vs);
    for (const at::Tensor* t : {&k, &v})
        if (meet(*t, kc) || meet(*t, vc)) refuse("K and V must be apart from the caches");
    Device dev;
    for (const at::Tensor* t : {&k, &v, &kc, &vc, &table, &lens}) dev.add(*t);
    for (PyObject* x : {o[6], ks, vs}) dev.add_if(x);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    const at::Tensor kr = ready(k), vr = ready(v);
    a.k_new = address(kr);
    a.v_new = address(vr);
    for (int i = 0; i < 3; ++i) {
        a.k_new_stride[i] = kr.stride(i);
        a.v_new_stride[i] = vr.stride(i);
    }
    a.block_table = int32s(table);
    a.max_new = (int32_t)k.size(1);
    a.max_pages = (int32_t)pages;
    launch(fgqa_kv_append, a, stream, "fgqa_kv_append");
    for (const at::Tensor* t : {&kc, &vc}) written(*t);
    for (PyObject* x : {ks, vs}) written_if(x);
    Py_RETURN_NONE;
}

// decode(q, k_cache, v_cache, block_table, seqlens, scale, k_scale, v_scale, out, lse, max_seqlen, split_tokens, workspace, prepare)
// -> out; or, prepare: (argument block's bytes, out, device's index, what it
// points at and this call allocated).
PyObject* decode(PyObject* const* o) {
    const at::Tensor &q = tensor(o[0], "q"), &kc = tensor(o[1], "k_cache"), &vc = tensor(o[2], "v_cache");
    const at::Tensor &table = tensor(o[3], "block_table"), &lens = tensor(o[4], "seqlens");
    if (q.scalar_type() != at::kBFloat16) refuse("paged decode expects a bf16 query");
    if (q.dim() != 3) refuse("expected q [B,Hq,D] and k_cache/v_cache [num_pages, page_size, Hkv, D]");
    fgqa_decode_blocks_args a;
    std::memset(&a, 0, sizeof a);
    a.cache = check_caches(kc, &vc, o[6], o[7]);
    const int64_t B = a.batch = check_batch(q.size(0));
    const int64_t Hq = q.size(1);
    if (q.size(2) != 128) refuse("the caches' head_dim must match Q");
    if (Hq < 1 || Hq > INT_MAX || Hq % kc.size(2) != 0) refuse("Query heads must be divisible by KV heads");
    int64_t pages;
    a.block_table_stride = check_table(table, B, "block_table", &pages);
    a.seqlens = check_lens(lens, B, "seqlens");
    const int64_t tokens = table_tokens(pages, a.cache);
    a.max_seqlen = check_max_seqlen(o[10], tokens, tokens);
    const int64_t split = integer(o[11]);
    if (split < 0 || split > INT_MAX) refuse("split_tokens must not be negative (and be below 2^31)");
    at::Tensor out, work;
    if (o[8] != Py_None) {
        out = tensor(o[8], "out");
        if (out.scalar_type() != at::kBFloat16 || out.sizes() != q.sizes() || !kernel_ready(out))
            refuse("out must be a bf16 [B, Hq, D] tensor with contiguous rows");
        check_written(out);
    }
    if (o[9] != Py_None) {
        const at::Tensor& lse = tensor(o[9], "lse");
        if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != B || lse.size(1) != Hq || !lse.is_contiguous())
            refuse("lse must be a contiguous fp32 [B, Hq] tensor");
        a.lse = floats(lse);
    }
    if (o[12] != Py_None) {
        work = tensor(o[12], "workspace");
        if (!work.is_contiguous()) refuse("workspace must be contiguous");   // (its bytes are all there)
        a.workspace = address(work);
        a.workspace_bytes = (size_t)work.numel() * work.element_size();
    }
    Device dev;
    for (const at::Tensor* t : {&q, &kc, &vc, &table, &lens}) dev.add(*t);
    for (PyObject* x : {blocks_or_none(a.cache.k_scales, o[6]), blocks_or_none(a.cache.v_scales, o[7]), o[8], o[9], o[12]})
        dev.add_if(x);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    const at::Tensor qr = ready(q);
    if (!out.defined()) out = at::empty(q.sizes(), q.options());
    a.q = address(qr);
    a.o = address(out);
    for (int i = 0; i < 2; ++i) {
        a.q_stride[i] = qr.stride(i);
        a.o_stride[i] = out.stride(i);
    }
    a.block_table = int32s(table);
    a.num_q_heads = (int32_t)Hq;
    a.scale = o[5] == Py_None ? (float)(1.0 / std::sqrt(128.0)) : (float)number(o[5]);
    a.split_tokens = (int32_t)split;
    if (!work.defined() && B > 0) {
        size_t bytes = 0;
        raise_status(fgqa_decode_blocks_workspace_bytes(&a, &bytes), "fgqa_decode_blocks_workspace_bytes");
        if (bytes > 0) {
            work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
            a.workspace = address(work);
            a.workspace_bytes = bytes;
        }
    }
    if (o[13] == Py_True)
        return Py_BuildValue("(y#NLNN)", reinterpret_cast<const char*>(&a), (Py_ssize_t)sizeof a, THPVariable_Wrap(out),
                             (long long)dev.index, THPVariable_Wrap(qr),
                             work.defined() ? THPVariable_Wrap(work) : (Py_INCREF(Py_None), Py_None));
    launch(fgqa_decode_blocks, a, stream, "fgqa_decode_blocks");
    return THPVariable_Wrap(out);
}

// weights(q, k_cache, lse, block_table, seqlens, weights, scale, k_scale, max_seqlen)
PyObject* weights(PyObject* const* o) {
    const at::Tensor &q = tensor(o[0], "q"), &kc = tensor(o[1], "k_cache"), &lse = tensor(o[2], "lse");
    const at::Tensor &table = tensor(o[3], "block_table"), &lens = tensor(o[4], "seqlens"), &w = tensor(o[5], "weights");
    if (q.scalar_type() != at::kBFloat16 || q.dim() != 3) refuse("expected a bf16 query [B, Hq, D]");
    fgqa_kv_weights_args a;
    std::memset(&a, 0, sizeof a);
    a.cache = check_caches(kc, nullptr, o[7], nullptr);
    const int64_t B = a.batch = check_batch(q.size(0));
    const int64_t Hq = q.size(1);
    if (q.size(2) != 128) refuse("the cache's head_dim must match Q");
    if (Hq < 1 || Hq > INT_MAX || Hq % kc.size(2) != 0) refuse("Query heads must be divisible by KV heads");
    if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != B || lse.size(1) != Hq || !lse.is_contiguous())
        refuse("lse must be a contiguous fp32 [B, Hq] tensor");
    const int64_t W = check_weights(w, B, kc.size(2), "weights");
    int64_t pages;
    a.block_table_stride = check_table(table, B, "block_table", &pages);
    a.seqlens = check_lens(lens, B, "seqlens");
    const int64_t tokens = table_tokens(pages, a.cache);
    a.max_seqlen = check_max_seqlen(o[8], tokens, std::min(tokens, W));
    if (W < a.max_seqlen) refuse("weights must hold max_seqlen tokens");
    check_written(w);
    PyObject* const ks = blocks_or_none(a.cache.k_scales, o[7]);
    if (meet(w, lse) || meet(w, q) || meet(w, table) || meet(w, lens) || meet_any(w, {o[1], ks})) refuse("weights must be apart from the inputs");
    Device dev;
    for (const at::Tensor* t : {&q, &kc, &lse, &table, &lens, &w}) dev.add(*t);
    dev.add_if(ks);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    const at::Tensor qr = ready(q);
    a.q = address(qr);
    a.lse = floats(lse);
    a.weights = floats(w);
    for (int i = 0; i < 2; ++i) {
        a.q_stride[i] = qr.stride(i);
        a.weights_stride[i] = w.stride(i);
    }
    a.block_table = int32s(table);
    a.num_q_heads = (int32_t)Hq;
    a.scale = o[6] == Py_None ? (float)(1.0 / std::sqrt(128.0)) : (float)number(o[6]);
    launch(fgqa_kv_weights, a, stream, "fgqa_kv_weights");
    written(w);
    Py_RETURN_NONE;
}

// evict(k_cache, v_cache, block_table, seqlens, weights, new_block_table, budget, recent, k_scale, v_scale,
//       new_seqlens, new_weights, kept, max_seqlen) -> (new_seqlens, new_weights, kept)
PyObject* evict(PyObject* const* o) {
    const at::Tensor &kc = tensor(o[0], "k_cache"), &vc = tensor(o[1], "v_cache"), &table = tensor(o[2], "block_table");
    const at::Tensor &lens = tensor(o[3], "seqlens"), &w = tensor(o[4], "weights");
    const at::Tensor& new_table = tensor(o[5], "new_block_table");
    fgqa_kv_evict_args a;
    std::memset(&a, 0, sizeof a);
    a.cache = check_caches(kc, &vc, o[8], o[9]);
    const int64_t heads = kc.size(2), budget = integer(o[6]), recent = integer(o[7]);
    if (budget < 1 || budget > INT_MAX || recent < 0)
        refuse("budget must be positive (and below 2^31) and recent not negative");
    if (lens.dim() != 1) refuse("seqlens must be a contiguous int32 [B] tensor");
    const int64_t B = a.batch = check_batch(lens.size(0));
    a.seqlens = check_lens(lens, B, "seqlens");
    const int64_t W = check_weights(w, B, heads, "weights");
    int64_t pages, new_pages;
    a.block_table_stride = check_table(table, B, "block_table", &pages);
    a.new_block_table_stride = check_table(new_table, B, "new_block_table", &new_pages);
    const int64_t tokens = table_tokens(pages, a.cache);
    a.max_seqlen = check_max_seqlen(o[13], tokens, std::min(tokens, W));
    if (W < a.max_seqlen) refuse("weights must hold max_seqlen tokens");
    const int64_t new_tokens = table_tokens(new_pages, a.cache);
    // without a max_seqlen, tokens past the weights' rows are kept as recent ones are
    // (no new pages at all, with weights of no tokens: nothing is kept)
    a.max_tokens = o[13] == Py_None && new_tokens > 0 ? (int32_t)std::min<int64_t>(tokens, 1 << 30) : a.max_seqlen;
    if (new_tokens < std::min<int64_t>(budget, a.max_seqlen))
        refuse("new_block_table must have pages for min(budget, max_seqlen) tokens");
    a.new_tokens = (int32_t)new_tokens;
    check_written(kc);
    check_written(vc);
    PyObject *const ks = blocks_or_none(a.cache.k_scales, o[8]), *const vs = blocks_or_none(a.cache.v_scales, o[9]);
    check_written_scales(ks, vs);
    check_apart(kc, vc, ks, vs);
    if (meet_any(w, {o[0], o[1], ks, vs})) refuse("weights must be apart from the caches and scales");
    at::Tensor given[3];   // new_seqlens, new_weights, kept
    if (o[10] != Py_None) {
        given[0] = tensor(o[10], "new_seqlens");
        check_lens(given[0], B, "new_seqlens");
    }
    if (o[11] != Py_None) {
        given[1] = tensor(o[11], "new_weights");
        if (check_weights(given[1], B, heads, "new_weights") != W) refuse("new_weights must have weights' shape");
        check_written(given[1]);
    }
    if (o[12] != Py_None) {
        given[2] = tensor(o[12], "kept");
        const at::Tensor& t = given[2];
        if (t.scalar_type() != at::kInt || t.dim() != 3 || t.size(0) != B || t.size(1) != heads || t.size(2) != budget ||
            !t.is_contiguous())
            refuse("kept must be a contiguous int32 [B, Hkv, budget] tensor");
    }
    for (int i = 0; i < 3; ++i) {
        if (!given[i].defined()) continue;
        bool met = meet(given[i], w) || meet(given[i], lens) || meet(given[i], table) || meet(given[i], new_table) ||
                   meet_any(given[i], {o[0], o[1], ks, vs});
        for (int j = 0; j < i; ++j) met = met || (given[j].defined() && meet(given[i], given[j]));
        if (met) refuse("new_seqlens, new_weights and kept must be apart from each other and from the inputs");
    }
    Device dev;
    for (const at::Tensor* t : {&w, &kc, &vc, &table, &lens, &new_table}) dev.add(*t);
    for (PyObject* x : {ks, vs, o[10], o[11], o[12]}) dev.add_if(x);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    if (!given[0].defined()) given[0] = at::empty({B}, lens.options());
    if (!given[1].defined()) given[1] = at::empty({B, heads, W}, w.options());
    if (!given[2].defined()) given[2] = at::empty({B, heads, budget}, lens.options());
    a.weights = floats(w);
    a.new_weights = floats(given[1]);
    for (int i = 0; i < 2; ++i) {
        a.weights_stride[i] = w.stride(i);
        a.new_weights_stride[i] = given[1].stride(i);
    }
    a.block_table = int32s(table);
    a.new_block_table = int32s(new_table);
    a.new_seqlens = int32s(given[0]);
    a.kept = int32s(given[2]);
    a.weights_len = (int32_t)W;
    a.budget = (int32_t)budget;
    a.recent = (int32_t)std::min(recent, budget);
    launch(fgqa_kv_evict, a, stream, "fgqa_kv_evict");
    for (const at::Tensor* t : {&kc, &vc}) written(*t);
    for (PyObject* x : {ks, vs, o[10], o[11], o[12]}) written_if(x);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(given[0]), THPVariable_Wrap(given[1]), THPVariable_Wrap(given[2]));
}

// bind(get_device, get_stream, FgqaError)
PyObject* bind(PyObject* const* o) {
    PyObject** to[] = {&g_get_device, &g_get_stream, &g_error};
    for (int i = 0; i < 3; ++i) {
        Py_INCREF(o[i]);
        Py_XSETREF(*to[i], o[i]);
    }
    Py_RETURN_NONE;
}

// Runs f on exactly kArgs arguments; no C++ exception leaves it.
template <PyObject* (*f)(PyObject* const*), int kArgs>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != kArgs) {
        PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
        return nullptr;
    }
    try {
        return f(args);
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

template <PyObject* (*f)(PyObject* const*), int kArgs>
constexpr PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<f, kArgs>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<append, 9>("append"),   method<decode, 14>("decode"), method<weights, 9>("weights"),
                           method<evict, 14>("evict"),    method<bind, 3>("bind"),      {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_kv_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_native() { return PyModule_Create(&g_module); }

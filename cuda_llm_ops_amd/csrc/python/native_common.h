// Argument checks that the native module's functions share (see kv_native.cpp).
#pragma once

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

namespace fgqa_native {

inline PyObject* g_get_device = nullptr;   // () -> current device's index
inline PyObject* g_get_stream = nullptr;   // (index) -> its current stream's handle
inline PyObject* g_error = nullptr;        // FgqaError(status, where)

// A Python exception is set.
struct Raised {};

[[noreturn]] inline void refuse(const char* format, ...) {
    va_list args;
    va_start(args, format);
    PyErr_FormatV(PyExc_ValueError, format, args);
    va_end(args);
    throw Raised{};
}

inline bool is_tensor(PyObject* o) { return THPVariable_Check(o); }

inline const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!is_tensor(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
        throw Raised{};
    }
    return THPVariable_Unpack(o);
}

// What int(o) gives; *outside: it does not fit 64 bits.
inline int64_t integer(PyObject* o) {
    PyObject* n = PyNumber_Long(o);
    if (n == nullptr) throw Raised{};
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(n, &overflow);
    Py_DECREF(n);
    if (overflow != 0) return overflow > 0 ? INT64_MAX : INT64_MIN;
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

inline double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

inline void* address(const at::Tensor& t) { return t.data_ptr(); }
inline bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(address(t)) & 15u) == 0; }

// Head dim contiguous, 16-byte aligned base, strides in multiples of 8 elements.
inline bool kernel_ready(const at::Tensor& t) {
    const auto st = t.strides();
    if (st.back() != 1 || !aligned16(t)) return false;
    for (size_t i = 0; i + 1 < st.size(); ++i)
        if (st[i] & 7) return false;
    return true;
}

inline at::Tensor ready(const at::Tensor& t) { return kernel_ready(t) ? t : t.contiguous(); }

// No two elements of t share memory (an expanded tensor's do).
inline bool rows_apart(const at::Tensor& t) {
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

inline void check_written(const at::Tensor& t) {
    if (!rows_apart(t)) refuse("a tensor that is written must not overlap itself (expanded dims)");
}

inline void check_written_scales(PyObject* k_scale, PyObject* v_scale) {
    if (is_tensor(k_scale)) check_written(THPVariable_Unpack(k_scale));
    if (is_tensor(v_scale)) check_written(THPVariable_Unpack(v_scale));
}

// The address ranges of a and b overlap.
inline bool meet(const at::Tensor& a, const at::Tensor& b) {
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
inline bool share(const at::Tensor& a, const at::Tensor& b) {
    if (!meet(a, b)) return false;
    if (a.sizes() != b.sizes()) return true;
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return true;
    return fgqa::plan::views_meet(reinterpret_cast<uintptr_t>(address(a)), reinterpret_cast<uintptr_t>(address(b)),
                                  a.sizes().data(), a.strides().data(), (int)a.dim(), (int64_t)a.element_size());
}

// t and the caches or block scales o (others are numbers) share address ranges.
inline bool meet_any(const at::Tensor& t, std::initializer_list<PyObject*> o) {
    for (PyObject* x : o)
        if (is_tensor(x) && meet(t, THPVariable_Unpack(x))) return true;
    return false;
}

// Caches and block scales that are written: K's and V's lie apart.
inline void check_apart(const at::Tensor& k, const at::Tensor& v, PyObject* k_scale, PyObject* v_scale) {
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
inline void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
inline void written_if(PyObject* o) {
    if (is_tensor(o)) written(THPVariable_Unpack(o));
}

inline PyObject* not_here() { Py_RETURN_NOTIMPLEMENTED; }

inline void raise_status(int status, const char* where) {
    if (status == FGQA_OK) return;
    PyObject* e = PyObject_CallFunction(g_error, "is", status, where);
    if (e != nullptr) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

template <typename Args>
inline void launch(int (*f)(const Args*, void*), const Args& a, void* stream, const char* where) {
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f(&a, stream);
    Py_END_ALLOW_THREADS
    raise_status(status, where);
}

// ---------------------------------------------------------------- the cache
inline const char* const kCacheShape = "must be [num_pages, page_size, Hkv, D]";

inline void check_cache(const at::Tensor& t, const char* name, int* dtype) {
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
inline bool may_be_number(PyObject* o) { return !is_tensor(o) || THPVariable_Unpack(o).numel() == 1; }
inline bool may_be_blocks(PyObject* o, const at::Tensor& cache) {
    if (!is_tensor(o)) return false;
    const at::Tensor& s = THPVariable_Unpack(o);
    return s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == cache.size(0) && s.size(1) == cache.size(2) &&
           s.device() == cache.device();
}

inline PyObject* blocks_or_none(const float* scales, PyObject* o) { return scales != nullptr ? o : Py_None; }

// k_scale or v_scale: block scales (returned) or one for the cache.
inline float* check_scale(PyObject* o, bool as_number, const at::Tensor& cache, int dtype, const char* name, float* whole,
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
inline fgqa_kv_cache check_caches(const at::Tensor& k, const at::Tensor* v, PyObject* k_scale, PyObject* v_scale) {
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
inline int64_t check_table(const at::Tensor& t, int64_t B, const char* name, int64_t* pages) {
    if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != B || (t.stride(1) != 1 && t.size(1) > 1 && B > 0))
        refuse("%s must be an int32 [B, max_pages] tensor with contiguous rows", name);
    *pages = t.size(1);
    return B > 1 ? t.stride(0) : t.size(1);
}

inline int32_t* check_lens(const at::Tensor& t, int64_t B, const char* name) {
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != B || !t.is_contiguous())
        refuse("%s must be a contiguous int32 [B] tensor", name);
    return static_cast<int32_t*>(address(t));
}

inline int32_t* int32s(const at::Tensor& t) { return static_cast<int32_t*>(address(t)); }
inline float* floats(const at::Tensor& t) { return static_cast<float*>(address(t)); }

inline int32_t check_batch(int64_t B) {
    if (B > INT_MAX) refuse("the batch is too large");
    return (int32_t)B;
}

// Tokens of a block table's row, as far as an int goes.
inline int64_t table_tokens(int64_t pages, const fgqa_kv_cache& c) {
    return pages > INT_MAX / c.page_size ? INT_MAX : pages * c.page_size;
}

inline int32_t check_max_seqlen(PyObject* o, int64_t tokens, int64_t otherwise) {
    if (o == Py_None) return (int32_t)otherwise;
    const int64_t n = integer(o);
    if (n < 0 || n > tokens) refuse("max_seqlen must be between 0 and the block table's tokens");
    return (int32_t)n;
}

// Tokens of a row of weights.
inline int64_t check_weights(const at::Tensor& t, int64_t B, int64_t heads, const char* name) {
    if (t.scalar_type() != at::kFloat || t.dim() != 3 || t.size(0) != B || t.size(1) != heads || t.size(2) > INT_MAX ||
        (t.stride(2) != 1 && t.size(2) > 1 && t.numel() > 1))
        refuse("%s must be an fp32 [B, Hkv, W] tensor with contiguous rows", name);
    return t.size(2);
}

}  // namespace fgqa_native

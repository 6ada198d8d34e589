// CPython module `_kv_native`: argument checks and calls of the paged KV cache's
// functions (cuda_llm_ops_amd/kv_cache.py, and the block-scaled form of
// flash_gqa.decode_flash_gqa_paged) over the C ABI of include/fgqa_kv.h, and, in
// files of their own (native_functions.h), of the other functions that it serves.
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
#include "native_common.h"
#include "native_functions.h"

using namespace fgqa_native;

namespace {

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

PyMethodDef g_methods[] = {method<append, 9>("append"),
                           method<decode, 14>("decode"),
                           method<weights, 9>("weights"),
                           method<evict, 14>("evict"),
                           method<rope, 11>("rope"),
                           method<rope_backward, 11>("rope_backward"),
                           method<fgqa_native::fork, 13>("fork"),
                           method<compact, 9>("compact"),
                           method<decode_shared, 14>("decode_shared"),
                           method<bind, 3>("bind"),
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_kv_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_native() { return PyModule_Create(&g_module); }

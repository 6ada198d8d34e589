// Argument checks and calls of the functions over include/fgqa_pages.h (see kv_native.cpp).
#include "fgqa_pages.h"
#include "native_common.h"
#include "native_functions.h"

namespace fgqa_native {
namespace {

// A list of pages that are in use elsewhere, or null.
const uint8_t* check_held(PyObject* o, const fgqa_kv_cache& c) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, "held");
    if ((t.scalar_type() != at::kBool && t.scalar_type() != at::kByte) || t.dim() != 1 || t.size(0) != c.num_pages || !t.is_contiguous())
        refuse("held must be a contiguous bool or uint8 [num_pages] tensor");
    return static_cast<const uint8_t*>(address(t));
}

// A tensor that is written lies apart from others: inputs, caches and what else is written.
void check_out(const at::Tensor& t, const char* name, std::initializer_list<PyObject*> inputs) {
    check_written(t);
    if (meet_any(t, inputs)) refuse("%s must be apart from the inputs and the other outputs", name);
}

template <typename Args>
at::Tensor workspace_of(int (*bytes_of)(const Args*, size_t*), Args* a, const at::Tensor& like, const char* where) {
    size_t bytes = 0;
    raise_status(bytes_of(a, &bytes), where);
    if (bytes == 0) return at::Tensor();   // (NULL and 0: none is needed)
    at::Tensor work = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
    a->workspace = address(work);
    a->workspace_bytes = bytes;
    return work;
}

}  // namespace

// fork(k_cache, v_cache, block_table, seqlens, parents, new_lens, held, width, k_scale, v_scale, new_block_table, new_seqlens,
//      num_free) -> (new_block_table, new_seqlens, num_free)
PyObject* fork(PyObject* const* o) {
    const at::Tensor &kc = tensor(o[0], "k_cache"), &vc = tensor(o[1], "v_cache"), &table = tensor(o[2], "block_table");
    const at::Tensor& lens = tensor(o[3], "seqlens");
    fgqa_kv_fork_args a;
    std::memset(&a, 0, sizeof a);
    a.cache = check_caches(kc, &vc, o[8], o[9]);
    if (lens.dim() != 1) refuse("seqlens must be a contiguous int32 [B] tensor");
    a.batch = check_batch(lens.size(0));
    a.seqlens = check_lens(lens, a.batch, "seqlens");
    int64_t pages;
    a.block_table_stride = check_table(table, a.batch, "block_table", &pages);
    int64_t N = a.batch;
    if (o[4] != Py_None) {
        const at::Tensor& parents = tensor(o[4], "parents");
        if (parents.dim() != 1) refuse("parents must be a contiguous int32 tensor of one dim");
        N = parents.size(0);
        a.parents = check_lens(parents, N, "parents");
    }
    a.new_batch = check_batch(N);
    if (o[5] != Py_None) {
        const at::Tensor& news = tensor(o[5], "new_lens");
        if (news.scalar_type() != at::kInt || news.dim() != 1 || news.size(0) != N || !news.is_contiguous())
            refuse("new_lens must be a contiguous int32 tensor with an element for each new row");
        a.new_lens = int32s(news);
    }
    a.held = check_held(o[6], a.cache);
    if (pages > INT_MAX) refuse("block_table has too many pages");
    a.max_pages = (int32_t)pages;
    check_written(kc);
    check_written(vc);
    PyObject *const ks = blocks_or_none(a.cache.k_scales, o[8]), *const vs = blocks_or_none(a.cache.v_scales, o[9]);
    check_written_scales(ks, vs);
    check_apart(kc, vc, ks, vs);
    for (PyObject* x : {o[2], o[3], o[4], o[5], o[6]})
        if (is_tensor(x) && meet_any(THPVariable_Unpack(x), {o[0], o[1], ks, vs})) refuse("the caches must be apart from the other inputs");
    at::Tensor new_table, new_lens, num_free;
    int64_t width = pages;
    if (o[7] != Py_None) {
        width = integer(o[7]);
        if (width < 0 || width > INT_MAX) refuse("max_pages must not be negative (and be below 2^31)");
    }
    if (o[10] != Py_None) {
        new_table = tensor(o[10], "new_block_table");
        a.new_block_table_stride = check_table(new_table, N, "new_block_table", &width);
        if (o[7] != Py_None && width != integer(o[7])) refuse("new_block_table must have max_pages columns");
        check_out(new_table, "new_block_table", {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[11], o[12], ks, vs});
    }
    if (width > INT_MAX) refuse("new_block_table has too many pages");
    if (o[11] != Py_None) {
        new_lens = tensor(o[11], "new_seqlens");
        check_lens(new_lens, N, "new_seqlens");
        check_out(new_lens, "new_seqlens", {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[12], ks, vs});
    }
    if (o[12] != Py_None) {
        num_free = tensor(o[12], "num_free");
        check_lens(num_free, 1, "num_free");
        check_out(num_free, "num_free", {o[0], o[1], o[2], o[3], o[4], o[5], o[6], ks, vs});
    }
    Device dev;
    for (const at::Tensor* t : {&kc, &vc, &table, &lens}) dev.add(*t);
    for (PyObject* x : {o[4], o[5], o[6], o[10], o[11], o[12], ks, vs}) dev.add_if(x);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    if (!new_table.defined()) {
        new_table = at::empty({N, width}, table.options());
        a.new_block_table_stride = width;
    }
    if (!new_lens.defined()) new_lens = at::empty({N}, lens.options());
    if (!num_free.defined()) num_free = at::empty({1}, lens.options());
    a.block_table = int32s(table);
    a.new_block_table = int32s(new_table);
    a.new_seqlens = int32s(new_lens);
    a.num_free = int32s(num_free);
    a.new_max_pages = (int32_t)width;
    const at::Tensor work = workspace_of(fgqa_kv_fork_workspace_bytes, &a, lens, "fgqa_kv_fork_workspace_bytes");
    launch(fgqa_kv_fork, a, stream, "fgqa_kv_fork");
    for (const at::Tensor* t : {&kc, &vc}) written(*t);
    for (PyObject* x : {ks, vs, o[10], o[11], o[12]}) written_if(x);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(new_table), THPVariable_Wrap(new_lens), THPVariable_Wrap(num_free));
}

// compact(k_cache, v_cache, block_table, seqlens, held, k_scale, v_scale, new_block_table, num_used)
// -> (new_block_table, num_used)
PyObject* compact(PyObject* const* o) {
    const at::Tensor &kc = tensor(o[0], "k_cache"), &vc = tensor(o[1], "v_cache"), &table = tensor(o[2], "block_table");
    const at::Tensor& lens = tensor(o[3], "seqlens");
    fgqa_kv_compact_args a;
    std::memset(&a, 0, sizeof a);
    a.cache = check_caches(kc, &vc, o[5], o[6]);
    if (lens.dim() != 1) refuse("seqlens must be a contiguous int32 [B] tensor");
    a.batch = check_batch(lens.size(0));
    a.seqlens = check_lens(lens, a.batch, "seqlens");
    int64_t pages;
    a.block_table_stride = check_table(table, a.batch, "block_table", &pages);
    if (pages > INT_MAX) refuse("block_table has too many pages");
    a.max_pages = (int32_t)pages;
    a.held = check_held(o[4], a.cache);
    check_written(kc);
    check_written(vc);
    PyObject *const ks = blocks_or_none(a.cache.k_scales, o[5]), *const vs = blocks_or_none(a.cache.v_scales, o[6]);
    check_written_scales(ks, vs);
    check_apart(kc, vc, ks, vs);
    for (PyObject* x : {o[2], o[3], o[4]})
        if (is_tensor(x) && meet_any(THPVariable_Unpack(x), {o[0], o[1], ks, vs})) refuse("the caches must be apart from the other inputs");
    at::Tensor new_table, num_used;
    if (o[7] != Py_None) {
        new_table = tensor(o[7], "new_block_table");
        int64_t width;
        a.new_block_table_stride = check_table(new_table, a.batch, "new_block_table", &width);
        if (width != pages) refuse("new_block_table must have block_table's shape");
        check_out(new_table, "new_block_table", {o[0], o[1], o[2], o[3], o[4], o[8], ks, vs});
    }
    if (o[8] != Py_None) {
        num_used = tensor(o[8], "num_used");
        check_lens(num_used, 1, "num_used");
        check_out(num_used, "num_used", {o[0], o[1], o[2], o[3], o[4], ks, vs});
    }
    Device dev;
    for (const at::Tensor* t : {&kc, &vc, &table, &lens}) dev.add(*t);
    for (PyObject* x : {o[4], o[7], o[8], ks, vs}) dev.add_if(x);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    if (!new_table.defined()) {
        new_table = at::empty(table.sizes(), table.options());
        a.new_block_table_stride = pages;
    }
    if (!num_used.defined()) num_used = at::empty({1}, lens.options());
    a.block_table = int32s(table);
    a.new_block_table = int32s(new_table);
    a.num_used = int32s(num_used);
    const at::Tensor work = workspace_of(fgqa_kv_compact_workspace_bytes, &a, lens, "fgqa_kv_compact_workspace_bytes");
    launch(fgqa_kv_compact, a, stream, "fgqa_kv_compact");
    for (const at::Tensor* t : {&kc, &vc}) written(*t);
    for (PyObject* x : {ks, vs, o[7], o[8]}) written_if(x);
    return Py_BuildValue("(NN)", THPVariable_Wrap(new_table), THPVariable_Wrap(num_used));
}

// decode_shared(q, k_cache, v_cache, block_table, seqlens, group_starts, shared_lens, scale, k_scale, v_scale, out, lse,
//               max_seqlen, workspace) -> out
PyObject* decode_shared(PyObject* const* o) {
    const at::Tensor &q = tensor(o[0], "q"), &kc = tensor(o[1], "k_cache"), &vc = tensor(o[2], "v_cache");
    const at::Tensor &table = tensor(o[3], "block_table"), &lens = tensor(o[4], "seqlens");
    const at::Tensor &starts = tensor(o[5], "group_starts"), &shared = tensor(o[6], "shared_lens");
    if (q.scalar_type() != at::kBFloat16) refuse("paged decode expects a bf16 query");
    if (q.dim() != 3) refuse("expected q [B,Hq,D] and k_cache/v_cache [num_pages, page_size, Hkv, D]");
    fgqa_decode_shared_args a;
    std::memset(&a, 0, sizeof a);
    a.cache = check_caches(kc, &vc, o[8], o[9]);
    const int64_t B = a.batch = check_batch(q.size(0));
    const int64_t Hq = q.size(1);
    if (q.size(2) != 128) refuse("the caches' head_dim must match Q");
    if (Hq < 1 || Hq > INT_MAX || Hq % kc.size(2) != 0) refuse("Query heads must be divisible by KV heads");
    int64_t pages;
    a.block_table_stride = check_table(table, B, "block_table", &pages);
    a.seqlens = check_lens(lens, B, "seqlens");
    if (shared.dim() != 1) refuse("shared_lens must be a contiguous int32 tensor of one dim");
    const int64_t N = shared.size(0);
    if (N > 4096) refuse("at most 4096 groups");
    a.num_groups = (int32_t)N;
    a.shared_lens = check_lens(shared, N, "shared_lens");
    if (starts.scalar_type() != at::kInt || starts.dim() != 1 || starts.size(0) != N + 1 || !starts.is_contiguous())
        refuse("group_starts must be a contiguous int32 tensor of one element more than shared_lens");
    a.group_starts = int32s(starts);
    const int64_t tokens = table_tokens(pages, a.cache);
    a.max_seqlen = check_max_seqlen(o[12], tokens, tokens);
    at::Tensor out, work;
    if (o[10] != Py_None) {
        out = tensor(o[10], "out");
        if (out.scalar_type() != at::kBFloat16 || out.sizes() != q.sizes() || !kernel_ready(out))
            refuse("out must be a bf16 [B, Hq, D] tensor with contiguous rows");
        check_out(out, "out", {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[8], o[9], o[11], o[13]});
    }
    if (o[11] != Py_None) {
        const at::Tensor& lse = tensor(o[11], "lse");
        if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != B || lse.size(1) != Hq || !lse.is_contiguous())
            refuse("lse must be a contiguous fp32 [B, Hq] tensor");
        check_out(lse, "lse", {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[8], o[9], o[13]});
        a.lse = floats(lse);
    }
    if (o[13] != Py_None) {
        work = tensor(o[13], "workspace");
        if (!work.is_contiguous()) refuse("workspace must be contiguous");
        check_out(work, "workspace", {o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[8], o[9]});
        a.workspace = address(work);
        a.workspace_bytes = (size_t)work.numel() * work.element_size();
    }
    Device dev;
    for (const at::Tensor* t : {&q, &kc, &vc, &table, &lens, &starts, &shared}) dev.add(*t);
    for (PyObject* x : {blocks_or_none(a.cache.k_scales, o[8]), blocks_or_none(a.cache.v_scales, o[9]), o[10], o[11], o[13]})
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
    a.scale = o[7] == Py_None ? (float)(1.0 / std::sqrt(128.0)) : (float)number(o[7]);
    if (!work.defined() && B > 0) work = workspace_of(fgqa_decode_shared_workspace_bytes, &a, q, "fgqa_decode_shared_workspace_bytes");
    launch(fgqa_decode_shared, a, stream, "fgqa_decode_shared");
    for (PyObject* x : {o[10], o[11]}) written_if(x);
    return THPVariable_Wrap(out);
}

}  // namespace fgqa_native

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

}  // namespace fgqa_native

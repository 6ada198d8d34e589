// Argument checks and calls of cuda_llm_ops_amd/qk_rope.py over the C ABI of
// include/fgqa_rope.h (see kv_native.cpp).
#include "fgqa_rope.h"
#include "native_common.h"
#include "native_functions.h"

namespace fgqa_native {
namespace {

// Strides {b, s, h} of a [B, S, H, D] or [T, H, D] tensor (one batch of T tokens); 0 for dims of one element.
struct Strides {
    int64_t at[3];
    explicit Strides(const at::Tensor& t) {
        const int first = 4 - (int)t.dim();
        for (int i = 0; i < 3; ++i) at[i] = i < first || t.size(i - first) <= 1 ? 0 : t.stride(i - first);
    }
    void put(int64_t (&to)[3]) const { std::copy(at, at + 3, to); }
};

bool rows_ready(const at::Tensor& t) {
    const Strides s(t);
    return (t.stride(-1) == 1 || t.numel() == 0) && aligned16(t) && ((s.at[0] | s.at[1] | s.at[2]) & 7) == 0;
}

at::Tensor ready_rows(const at::Tensor& t) { return rows_ready(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Rows of a and of b (of equal leading dims and head dims) share memory.
bool rows_meet(const at::Tensor& a, const at::Tensor& b) {
    if (!meet(a, b)) return false;
    const Strides x(a), y(b);
    if (x.at[0] != y.at[0] || x.at[1] != y.at[1]) return true;
    const int first = 4 - (int)a.dim();
    auto bytes = [&](const at::Tensor& t, const Strides& s) {
        return ((t.size(2 - first) - 1) * s.at[2] + t.size(3 - first)) * (int64_t)t.element_size();
    };
    return fgqa::plan::blocks_meet(reinterpret_cast<uintptr_t>(address(a)), bytes(a, x), reinterpret_cast<uintptr_t>(address(b)),
                                   bytes(b, y), first ? 1 : a.size(0), x.at[0] * 2, a.size(1 - first), x.at[1] * 2);
}

bool same_rows(const at::Tensor& a, const at::Tensor& b) {
    const Strides x(a), y(b);
    return address(a) == address(b) && std::equal(x.at, x.at + 3, y.at);
}

void check_rows(const at::Tensor& q, const at::Tensor& k, const char* qn, const char* kn) {
    if (q.scalar_type() != at::kBFloat16 || k.scalar_type() != at::kBFloat16) refuse("%s and %s must be bf16", qn, kn);
    if ((q.dim() != 4 && q.dim() != 3) || k.dim() != q.dim()) refuse("%s and %s must both be [B, S, H, D] or [T, H, D]", qn, kn);
    for (int i = 0; i < q.dim(); ++i)
        if (i != q.dim() - 2 && q.size(i) != k.size(i)) refuse("%s and %s must agree in all but their heads", qn, kn);
    if (q.size(-2) < 1 || k.size(-2) < 1) refuse("%s and %s must have heads", qn, kn);
    for (int i = 0; i < q.dim(); ++i)
        if (q.size(i) > INT_MAX || k.size(i) > INT_MAX) refuse("%s or %s is too large", qn, kn);
}

// What both directions read but q and k; o: positions, inv_freq, q_weight, k_weight, eps, axes, interleaved.
fgqa_rope_args check_shared(PyObject* const* o, const at::Tensor& q, const at::Tensor& k) {
    fgqa_rope_args a;
    std::memset(&a, 0, sizeof a);
    const int first = 4 - (int)q.dim();
    a.batch = first ? 1 : (int32_t)q.size(0);
    a.seqlen = (int32_t)q.size(1 - first);
    a.num_q_heads = (int32_t)q.size(-2);
    a.num_kv_heads = (int32_t)k.size(-2);
    a.head_dim = (int32_t)q.size(-1);
    if (a.head_dim < 16 || a.head_dim > 256 || a.head_dim % 16) refuse("the head dim must be a multiple of 16 up to 256");
    a.num_axes = 1;
    if ((o[0] == Py_None) != (o[1] == Py_None)) refuse("positions and inv_freq must both be given, or neither");
    if (o[0] != Py_None) {
        const at::Tensor &pos = tensor(o[0], "positions"), &freq = tensor(o[1], "inv_freq");
        if (freq.scalar_type() != at::kFloat || freq.dim() != 1 || !freq.is_contiguous())
            refuse("inv_freq must be a contiguous fp32 [R / 2] tensor");
        if (freq.size(0) % 8 || 2 * freq.size(0) > a.head_dim)
            refuse("inv_freq must have a multiple of 8 elements, at most half of the head dim");
        a.rotary_dim = (int32_t)(2 * freq.size(0));
        a.inv_freq = floats(freq);
        if (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) refuse("positions must be int32 or int64");
        // [A, B, S], [B, S] or [S] of [B, S, H, D]; [A, T] or [T] of [T, H, D]
        const int lead = 2 - first, extra = (int)pos.dim() - lead;
        if (extra > 1 || (first ? extra < 0 : extra < -1)) refuse("positions must be %s", first ? "[T] or [A, T]" : "[S], [B, S] or [A, B, S]");
        if (pos.size(-1) != a.seqlen || (!first && pos.dim() >= 2 && pos.size(-2) != a.batch))
            refuse("positions must match the tokens of q and k");
        if (extra == 1) {
            if (pos.size(0) < 1 || pos.size(0) > INT_MAX) refuse("positions must have at least one axis");
            a.num_axes = (int32_t)pos.size(0);
            a.positions_stride[0] = pos.stride(0);
        }
        if (!first && pos.dim() >= 2) a.positions_stride[1] = pos.stride(-2);
        a.positions_stride[2] = pos.stride(-1);
        a.positions = address(pos);
        a.positions_int64 = pos.scalar_type() == at::kLong;
        if (o[5] != Py_None) {
            const at::Tensor& axes = tensor(o[5], "axes");
            if (axes.scalar_type() != at::kInt || axes.dim() != 1 || axes.size(0) != freq.size(0) || !axes.is_contiguous())
                refuse("axes must be a contiguous int32 tensor of inv_freq's size");
            a.axes = int32s(axes);
        } else if (a.num_axes > 1) {
            refuse("positions of several axes need axes");
        }
    } else if (o[5] != Py_None) {
        refuse("axes need positions");
    }
    if ((o[2] == Py_None) != (o[3] == Py_None)) refuse("q_weight and k_weight must both be given, or neither");
    if (o[2] != Py_None) {
        const at::Tensor &qw = tensor(o[2], "q_weight"), &kw = tensor(o[3], "k_weight");
        for (const at::Tensor* w : {&qw, &kw})
            if ((w->scalar_type() != at::kBFloat16 && w->scalar_type() != at::kFloat) || w->scalar_type() != qw.scalar_type() ||
                w->dim() != 1 || w->size(0) != a.head_dim || !w->is_contiguous())
                refuse("q_weight and k_weight must be contiguous [D] tensors, both bf16 or both fp32");
        a.q_weight = address(qw);
        a.k_weight = address(kw);
        a.weights_bf16 = qw.scalar_type() == at::kBFloat16;
    }
    const double eps = number(o[4]);
    if (!(eps >= 0.0) || !std::isfinite((float)eps)) refuse("eps must be finite and not negative");
    a.eps = (float)eps;
    const int inter = PyObject_IsTrue(o[6]);
    if (inter < 0) throw Raised{};
    a.interleaved = inter;
    return a;
}

void add_shared(Device* dev, PyObject* const* o) {
    for (int i : {0, 1, 2, 3, 5}) dev->add_if(o[i]);
}

}  // namespace

// rope(q, k, positions, inv_freq, q_weight, k_weight, eps, axes, interleaved, q_out, k_out) -> (q_out, k_out)
PyObject* rope(PyObject* const* o) {
    const at::Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k");
    check_rows(q, k, "q", "k");
    fgqa_rope_args a = check_shared(o + 2, q, k);
    at::Tensor out[2];
    const at::Tensor* in[2] = {&q, &k};
    for (int i = 0; i < 2; ++i) {
        if (o[9 + i] == Py_None) continue;
        const char* name = i ? "k_out" : "q_out";
        out[i] = tensor(o[9 + i], name);
        if (out[i].scalar_type() != at::kBFloat16 || out[i].sizes() != in[i]->sizes() || !rows_ready(out[i]))
            refuse("%s must be bf16 of its input's shape, with contiguous, 16-byte aligned rows", name);
        check_written(out[i]);
        if (meet_any(out[i], {o[2], o[3], o[4], o[5], o[7]})) refuse("%s must be apart from positions, frequencies and weights", name);
    }
    for (int i = 0; i < 2; ++i) {
        if (!out[i].defined()) continue;
        bool met = rows_meet(out[i], *in[1 - i]) || (!same_rows(out[i], *in[i]) && rows_meet(out[i], *in[i]));
        met = met || (out[1 - i].defined() && rows_meet(out[i], out[1 - i]));
        if (met) refuse("q_out and k_out must be their inputs, or apart from them and from each other");
    }
    Device dev;
    dev.add(q);
    dev.add(k);
    add_shared(&dev, o + 2);
    dev.add_if(o[9]);
    dev.add_if(o[10]);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    // (a copied input is not its output any more)
    const at::Tensor qr = ready_rows(q), kr = ready_rows(k);
    for (int i = 0; i < 2; ++i)
        if (!out[i].defined()) out[i] = at::empty(in[i]->sizes(), in[i]->options());
    a.q = address(qr);
    a.k = address(kr);
    a.q_out = address(out[0]);
    a.k_out = address(out[1]);
    Strides(qr).put(a.q_stride);
    Strides(kr).put(a.k_stride);
    Strides(out[0]).put(a.q_out_stride);
    Strides(out[1]).put(a.k_out_stride);
    launch(fgqa_qk_norm_rope, a, stream, "fgqa_qk_norm_rope");
    written_if(o[9]);
    written_if(o[10]);
    return Py_BuildValue("(NN)", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]));
}

// rope_backward(grad_q, grad_k, q, k, positions, inv_freq, q_weight, k_weight, eps, axes, interleaved)
// -> (of q, of k, of q_weight, of k_weight)
PyObject* rope_backward(PyObject* const* o) {
    const at::Tensor &gq = tensor(o[0], "grad_q"), &gk = tensor(o[1], "grad_k");
    check_rows(gq, gk, "grad_q", "grad_k");
    fgqa_rope_backward_args a;
    std::memset(&a, 0, sizeof a);
    a.fwd = check_shared(o + 4, gq, gk);
    const bool norm = a.fwd.q_weight != nullptr;
    if (norm || o[2] != Py_None || o[3] != Py_None) {
        const at::Tensor &q = tensor(o[2], "q"), &k = tensor(o[3], "k");
        check_rows(q, k, "q", "k");
        if (q.sizes() != gq.sizes() || k.sizes() != gk.sizes()) refuse("grad_q and grad_k must have q's and k's shapes");
    }
    Device dev;
    dev.add(gq);
    dev.add(gk);
    for (int i : {2, 3}) dev.add_if(o[i]);
    add_shared(&dev, o + 4);
    void* stream = nullptr;
    if (!dev.current(&stream)) return not_here();
    const at::Tensor gqr = ready_rows(gq), gkr = ready_rows(gk);
    const at::Tensor dq = at::empty(gq.sizes(), gq.options()), dk = at::empty(gk.sizes(), gk.options());
    a.grad_q_out = address(gqr);
    a.grad_k_out = address(gkr);
    a.grad_q = address(dq);
    a.grad_k = address(dk);
    Strides(gqr).put(a.grad_q_out_stride);
    Strides(gkr).put(a.grad_k_out_stride);
    Strides(dq).put(a.grad_q_stride);
    Strides(dk).put(a.grad_k_stride);
    at::Tensor qr, kr, qw, kw, work;
    if (norm) {
        qr = ready_rows(THPVariable_Unpack(o[2]));
        kr = ready_rows(THPVariable_Unpack(o[3]));
        a.fwd.q = address(qr);
        a.fwd.k = address(kr);
        Strides(qr).put(a.fwd.q_stride);
        Strides(kr).put(a.fwd.k_stride);
        qw = at::empty({a.fwd.head_dim}, gq.options().dtype(at::kFloat));
        kw = at::empty({a.fwd.head_dim}, gq.options().dtype(at::kFloat));
        a.grad_q_weight = floats(qw);
        a.grad_k_weight = floats(kw);
        size_t bytes = 0;
        raise_status(fgqa_qk_norm_rope_backward_workspace_bytes(&a, &bytes), "fgqa_qk_norm_rope_backward_workspace_bytes");
        if (bytes > 0) {
            work = at::empty({(int64_t)bytes}, gq.options().dtype(at::kByte));
            a.workspace = address(work);
            a.workspace_bytes = bytes;
        }
    }
    launch(fgqa_qk_norm_rope_backward, a, stream, "fgqa_qk_norm_rope_backward");
    auto wrapped = [](const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : (Py_INCREF(Py_None), Py_None); };
    return Py_BuildValue("(NNNN)", wrapped(dq), wrapped(dk), wrapped(qw), wrapped(kw));
}

}  // namespace fgqa_native
